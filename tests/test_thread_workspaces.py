"""Calls of two launches with a workspace between them: every thread and stream has its own."""
import threading
import types

import pytest
import torch

from leone_b200.ops.cuda import CudaOps
from leone_b200.ops.int8 import Int8Products, PerThread
from tests.fewer_bits import Step, quantize4, quantize8

from leone_b200.cache import packed

DEV = "cuda:0"
BF16 = torch.bfloat16


def _in_threads(count, work):
    """``work(i)`` in ``count`` threads at once; what they returned.  All run until the last has begun."""
    results, errors, gate = [None] * count, [], threading.Barrier(count, timeout=60)

    def run(i):
        try:
            gate.wait()
            results[i] = work(i)
            gate.wait()
        except BaseException as e:                           # noqa: BLE001 (raised again below)
            errors.append(e)
            gate.abort()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]
    return results


def test_threads_and_streams_have_workspaces_of_their_own(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ops = CudaOps.__new__(CudaOps)
    ops.device, ops._pinned_stream, ops._workspaces = torch.device("cpu"), 7, PerThread()
    products = Int8Products.__new__(Int8Products)
    products.ops, products.buffers = types.SimpleNamespace(device=torch.device("cpu")), PerThread()

    def both(_):
        return ops._workspace("parts", 1000), products.tokens(5, 64, 7)[0]

    (a, x), (b, y) = _in_threads(2, both)
    assert a.data_ptr() != b.data_ptr() and x.data_ptr() != y.data_ptr()
    # of one thread: the same again, another for another stream, a larger one where it is outgrown
    first, codes = both(0)
    again, more = both(0)
    assert first is again and codes is more
    assert products.tokens(5, 64, 8)[0] is not codes and products.tokens(100, 64, 7)[0].shape[0] >= 100
    assert ops._workspace("parts", 1 << 17).numel() >= 1 << 17 and ops._workspace("other", 1000) is not first


@pytest.mark.gpu
def test_products_of_two_threads_on_one_stream():
    """Between a product's rounding of its tokens and its sums another thread's rounding may run."""
    from leone_b200.ops.int8 import quantize_matrix
    ops = CudaOps(DEV, BF16)
    ops.bind_status(torch.zeros(4, dtype=torch.int32, device=DEV))
    gen = torch.Generator(DEV).manual_seed(1)
    m, n, k = 48, 512, 4096
    w = ops.prepare_matrix_int8(*quantize_matrix(torch.randn((n, k), generator=gen, device=DEV)))
    xs = [(torch.randn((m, k), generator=gen, device=DEV) * (1 + 30 * i)).to(BF16) for i in range(4)]
    want = []
    for x in xs:
        want.append(torch.empty((m, n), device=DEV))
        ops.linear(x, w, want[-1])
        a, s = quantize8(x.double())
        exact = (a @ w.weight.double().T) * s * w.scales.double()
        # a sum, two scales and their products: five roundings
        assert ((want[-1].double() - exact).abs() <= exact.abs() * 5 * 2.0 ** -24 + 1e-30).all()
    torch.cuda.synchronize()

    def work(i):
        outs = torch.zeros((300, m, n), device=DEV)
        for out in outs:
            ops.linear(xs[i], w, out)
        return outs

    for outs, right in zip(_in_threads(4, work), want):
        torch.cuda.synchronize()
        assert (outs == right).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lens,splits", [([(1, 3000)], 33), ([(30, 2000)], 9)])
def test_split_attention_of_two_threads_on_one_stream(lens, splits):
    """Between the blocks that share a sequence's keys and what merges their parts another thread's blocks may run."""
    ops = CudaOps(DEV, BF16)
    ops.bind_status(torch.zeros(4, dtype=torch.int32, device=DEV))
    ops.force_decode4_splits = ops.force_prompt4_splits = splits
    n_q, n_kv, d = 8, 2, 128
    cases = []
    for seed in range(3):
        step = Step(lens, 16, DEV, seed=seed)
        gen = torch.Generator(DEV).manual_seed(seed)
        pools = [packed.pack_pages(*quantize4(torch.randn((step.pages, n_kv, 16, d), generator=gen, device=DEV).double()), v)
                 for v in (False, True)]
        qkv = torch.randn((step.ctx.n_tokens, (n_q + 2 * n_kv) * d), generator=gen, device=DEV).to(BF16)
        cases.append((step, qkv, step.view(*pools)))

    def call(step, qkv, view, out):
        ops.attention(step.ctx, qkv, out, n_q, n_kv, d, d ** -0.5, None, view)
        return out

    shape = (cases[0][1].shape[0], n_q * d)
    want = [call(*c, torch.zeros(shape, dtype=BF16, device=DEV)) for c in cases]
    torch.cuda.synchronize()

    def work(i):
        outs = torch.zeros((300, *shape), dtype=BF16, device=DEV)
        for out in outs:
            call(*cases[i], out)
        return outs

    for outs, right in zip(_in_threads(3, work), want):
        torch.cuda.synchronize()
        assert torch.equal(outs, right.expand_as(outs))


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_gates_without_the_epilogue_on_two_streams_at_once(captured):
    """Where gate and up lie side by side before the gate (32-bit runs), they lie in the stream's own workspace, or the graph's."""
    from leone_b200.ops.int8 import quantize_matrix
    ops = CudaOps(DEV, torch.float32)
    ops.bind_status(torch.zeros(4, dtype=torch.int32, device=DEV))
    gen = torch.Generator(DEV).manual_seed(3)
    m, k, inter = 700, 256, 1000
    gate, up = (quantize_matrix(torch.randn((inter, k), generator=gen, device=DEV)) for _ in range(2))
    w = ops.prepare_gate_up_int8(*gate, *up)
    xs = [torch.randn((m, k), generator=gen, device=DEV) for _ in range(2)]
    want = [torch.empty((m, inter), device=DEV) for _ in range(2)]
    for x, y in zip(xs, want):
        ops.linear_swiglu(x, w, y)
    streams, outs, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros_like(y) for y in want], []
    torch.cuda.synchronize()
    if captured:
        for x, y in zip(xs, outs):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=streams[0]):
                ops.linear_swiglu(x, w, y)
    for _ in range(20):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if captured:
                    graphs[i].replay()
                else:
                    for _ in range(4):
                        ops.linear_swiglu(xs[i], w, outs[i])
        torch.cuda.synchronize()
        for y, z in zip(outs, want):
            assert torch.equal(y, z)
    del graphs
