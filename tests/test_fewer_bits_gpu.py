"""Pages in 4 bits and products in 8 bits together, as a layer and an engine use them."""
import math

import pytest
import torch

from leone_b200.cache import packed
from leone_b200.ops.int8 import quantize_matrix
from tests.fewer_bits import Step, attention64, quantize4, quantize8, rotate, values4
from tests.tiny import make_folder

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, FP32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _ops(dtype):
    from leone_b200.ops.cuda import CudaOps
    ops = CudaOps(DEV, dtype)
    ops.bind_status(torch.zeros(4, dtype=torch.int32, device=DEV))
    return ops


@pytest.mark.parametrize("dtype,n_q,n_kv,d,hidden", [(BF16, 8, 2, 128, 512), (BF16, 14, 2, 64, 384), (FP32, 4, 2, 64, 256), (FP32, 6, 3, 32, 96)])
def test_a_layer(dtype, n_q, n_kv, d, hidden):
    """Three steps of an attention layer (prompts, a mixed step, decode rows): each operator against its 64-bit form on what the operator
    before it left, with what earlier steps left in the pages."""
    from leone_b200.parts.rotary import build_rotary_table
    ops = _ops(dtype)
    half = torch.finfo(dtype).eps / 2
    cols = (n_q + 2 * n_kv) * d
    w_qkv, w_o = (torch.randn(s, generator=_gen(i), device=DEV) * 0.05 for i, s in enumerate([(cols, hidden), (hidden, n_q * d)]))
    qkv8, o8 = (quantize_matrix(w) for w in (w_qkv, w_o))
    m_qkv, m_o = ops.prepare_matrix_int8(*qkv8), ops.prepare_matrix_int8(*o8)
    q_norm, k_norm = (1 + 0.1 * torch.randn((2, d), generator=_gen(5), device=DEV)).unbind(0)
    table = build_rotary_table(256, d, 10000.0).to(DEV)
    pools = [torch.full((12, n_kv, 16, packed.row_bytes(d)), 0xFF, dtype=torch.uint8, device=DEV) for _ in range(2)]
    rows = torch.full((2, 8), -1, dtype=torch.int32, device=DEV)
    rows[0, :4] = torch.tensor([7, 2, 11, 0])
    rows[1, :3] = torch.tensor([5, 9, 3])
    done = [0, 0]
    for new in ((21, 1), (1, 18), (1, 1)):
        step = Step([(n, p) for n, p in zip(new, done)], 16, DEV)
        step.table = rows
        n = step.ctx.n_tokens
        x = torch.randn((n, hidden), generator=_gen(n + done[0]), device=DEV).to(dtype)
        stream = torch.randn((n, hidden), generator=_gen(n + 9), device=DEV)
        qkv, attn, out = torch.empty((n, cols), dtype=dtype, device=DEV), torch.empty((n, n_q * d), dtype=dtype, device=DEV), stream.clone()
        view = step.view(*pools)
        ops.linear(x, m_qkv, qkv)
        before = qkv.double().unflatten(1, (n_q + 2 * n_kv, d))
        ops.qk_norm_rope_write(step.ctx, qkv, n_q, n_kv, d, q_norm, k_norm, 1e-6, table, d, view)
        ops.attention(step.ctx, qkv, attn, n_q, n_kv, d, d ** -0.5, None, view)
        ops.linear(attn, m_o, out, residual=out)

        a, s = quantize8(x.double())
        want = (a @ qkv8[0].double().T) * s * qkv8[1].double()
        assert ((before.flatten(1) - want).abs() <= want.abs() * (half + 2.0 ** -21) + 1e-30).all()
        k = before[:, n_q:n_q + n_kv]
        k = rotate(k * k_norm.double() * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6), step.pos, 10000.0, "half_split", d)
        page, slot = rows[step.seq, step.pos // 16].long(), step.pos % 16
        held = []
        for pool, new_rows, values in ((pools[0], k, False), (pools[1], before[:, n_q + n_kv:], True)):
            got = packed.unpack_pages(pool, d, values)
            codes, sc, z = quantize4(new_rows)
            assert torch.equal(got[0][page, :, slot].long(), codes) and torch.equal(got[1][page, :, slot].double(), sc)
            assert torch.equal(got[2][page, :, slot].double(), z)
            held.append(values4(*got))
        q = qkv[:, :n_q * d].double().unflatten(1, (n_q, d))
        want, top_s, top_v = attention64(q, *held, step.lens, rows, 16, d ** -0.5, 0)
        # (the bound of a prompt portion, the widest of the kernels': see test_cache4_gpu.py)
        loose = top_v * (2 * top_s * (2.0 ** -11 + (d + 4) * 10 * 2.0 ** -23) + 3 * 2.0 ** -8) if dtype == BF16 else \
            top_v * (2 * (d + 4) * 2.0 ** -23 * top_s + 80 * 2.0 ** -23)
        assert ((attn.double().unflatten(1, (n_q, d)) - want).abs() <= loose.double()[..., None] + want.abs() * half + 1e-30).all()
        a, s = quantize8(attn.double())
        want = (a @ o8[0].double().T) * s * o8[1].double() + stream.double()
        assert ((out.double() - want).abs() <= (want.abs() + stream.abs()) * 2.0 ** -21 + 1e-30).all()
        assert step.ctx.status.tolist() == [0, 0, 0, 0]
        done = [p + n for p, n in zip(done, new)]
    assert ops.status.tolist() == [0, 0, 0, 0]


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return make_folder(tmp_path_factory.mktemp("models"), "C")


def _engine(folder, dtype, **kw):
    from leone_b200.engine.engine import Engine
    return Engine.from_folder(folder, dtype=dtype, **{**dict(page_tokens=16, num_pages=40, max_requests=4, max_batch_tokens=128), **kw})


BITS = [dict(cache_bits=4), dict(weight_bits=8), dict(cache_bits=4, weight_bits=8)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bits", BITS)
def test_engine_computes_what_the_stand_ins_compute(folder, dtype, bits):
    """Prompts in portions and tokens after them, against the engine on the 64-bit stand-ins.  The two differ where a rounding before
    a code falls otherwise (one step of one element), so in 32 bits the logits' difference is measured against the distance that the
    options themselves make, which is that of every element's rounding.  In bfloat16 the roundings of weights and activations to
    8 significant bits make a distance of the same size as those to 8-bit integers do, so it cannot be: there the bound is what
    some dozen roundings of 2^-8 of each of two layers can add up to."""
    from leone_b200.engine.engine import Engine
    from tests.test_fewer_bits_engine import FewerBitsOps
    prompt = [(11 * i) % 300 for i in range(60)]
    trace = [[("a", prompt[:33], list(range(33)))], [("a", prompt[33:40], list(range(7))), ("b", prompt[:30], [29])],
             [("a", [prompt[40]], [0]), ("b", [prompt[30]], [0])]]
    got = _engine(folder, dtype, **bits)
    plain = Engine.from_folder(folder, dtype="float32", device="cpu", ops=FewerBitsOps(), page_tokens=16, num_pages=40, max_requests=4,
                               max_batch_tokens=128, **bits)
    full = _engine(folder, dtype)
    for entries in trace:
        a, b, c = got.step(entries).double().cpu(), plain.step(entries).double(), full.step(entries).double().cpu()
        away, off = float((b - c).norm() / c.norm()), float((a - b).norm() / b.norm())
        assert off < (0.35 * away if dtype == "float32" else 24 * 2.0 ** -8), (off, away)


@pytest.mark.parametrize("bits", BITS)
def test_generate_with_graphs_and_reused_pages(folder, bits):
    from leone_b200 import generate
    prompts = [[(7 * i + n) % 300 for i in range(n)] for n in (5, 40, 17)]
    outs = []
    for kw in (dict(use_graphs=False), dict(), dict(decode_quantum=4)):
        eng = _engine(folder, "float32", **bits)
        outs.append(generate(eng, prompts, 10, eos_token_id=-1, **kw))
        again = generate(eng, prompts, 10, eos_token_id=-1, **kw)          # over pages that hold the first run's rows
        assert again == outs[-1]
        assert eng.cache.free_pages()[0] == 40
    assert outs[0] == outs[1] == outs[2]
    with_bf16 = generate(folder, prompts, 10, dtype="bfloat16", eos_token_id=-1, **bits)
    assert [len(t) for t in with_bf16] == [10, 10, 10]


def test_captured_decode_steps_in_bfloat16_stay_near_eager_ones(folder):
    prompts = {"a": list(range(1, 50)), "b": list(range(60, 80))}
    logits = []
    for graph in (False, True):
        eng = _engine(folder, "bfloat16", cache_bits=4, weight_bits=8)
        eng.step([(r, p, []) for r, p in prompts.items()])
        rows = []
        for token in (3, 4, 5):
            if graph:
                rows.append(eng.decode_logits(list(prompts), [token, token]).clone())
            else:
                rows.append(eng.step([(r, [token], [0]) for r in prompts]))
        logits.append(torch.stack(rows).double())
        assert eng.ops.launches > 0
    # the same kernels but for how many ways the keys are split: roundings of bfloat16 that fall otherwise
    assert float((logits[0] - logits[1]).norm() / logits[0].norm()) < 0.03


@pytest.mark.parametrize("bits", BITS)
def test_steps_of_a_head_size_that_tuned_kernels_take(tmp_path, bits):
    """Prompts, a mixed step, decode steps and captured ones of heads of 64 in bfloat16, whose decode steps prepare q and k in the attention
    kernel where the cache is in the run dtype: against the engine on the 64-bit stand-ins.

    The two differ by bfloat16's roundings, bounded as above, and by the codes that these move.  A rounding moves an element by half a
    step of 2^-8, and its group's offset and scale by a step, against codes whose step is 1/15 of the group's width (1/254 of the
    row's with 8 bits, whose scale is not rounded): 2^-9 to 2^-8 of up to 15 steps three times, 0.09 to 0.12 of a step for the largest
    elements and half of that on average, so about one element in twelve to twenty falls on the next code.  One step in one of twelve
    elements is in the mean square what rounding to codes makes itself (a step squared over 12): the distance of the options to the run
    without them, once more."""
    from leone_b200 import generate
    from leone_b200.engine.engine import Engine
    from tests.test_fewer_bits_engine import FewerBitsOps
    folder = make_folder(tmp_path, "D")
    prompt = [(11 * i) % 250 for i in range(90)]
    trace = [[("a", prompt[:60], list(range(60)))], [("b", [prompt[3]], [0]), ("a", prompt[60:70], list(range(10)))]] + \
        [[("a", [prompt[70 + i]], [0]), ("b", [prompt[i]], [0])] for i in range(4)]
    got = _engine(folder, "bfloat16", **bits)
    plain = Engine.from_folder(folder, dtype="float32", device="cpu", ops=FewerBitsOps(), page_tokens=16, num_pages=40, max_requests=4,
                               max_batch_tokens=128, **bits)
    without = _engine(folder, "float32")
    for i, entries in enumerate(trace):
        want = plain.step(entries).double()
        away = float((without.step(entries).double().cpu() - want).norm() / want.norm())
        have = (got.decode_logits([r for r, _, _ in entries], [t[0] for _, t, _ in entries]) if i > 3 else got.step(entries)).double().cpu()
        assert float((have - want).norm() / want.norm()) < 24 * 2.0 ** -8 + away
    prompts = [[(7 * i + n) % 250 for i in range(n)] for n in (5, 40, 17)]
    outs = [generate(_engine(folder, "bfloat16", **bits), prompts, 10, eos_token_id=-1, **kw) for kw in (dict(), dict(decode_quantum=4))]
    assert outs[0] == outs[1] and [len(t) for t in outs[0]] == [10, 10, 10]


def test_a_captured_product_survives_larger_ones():
    """A graph keeps the buffers of codes it was captured with, also when a larger product has outgrown them."""
    ops = _ops(BF16)
    x = torch.randn((4, 256), generator=_gen(1), device=DEV).to(BF16)
    w = ops.prepare_matrix_int8(*quantize_matrix(torch.randn((96, 256), generator=_gen(2), device=DEV)))
    want, out = torch.empty((4, 96), dtype=BF16, device=DEV), torch.empty((4, 96), dtype=BF16, device=DEV)
    ops.linear(x, w, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear(x, w, out)
    big = torch.randn((700, 256), generator=_gen(3), device=DEV).to(BF16)
    for _ in range(3):
        ops.linear(big, w, torch.empty((700, 96), dtype=BF16, device=DEV))
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_products_on_two_streams_at_once():
    ops = _ops(BF16)
    inputs = [torch.randn((300, 1024), generator=_gen(i), device=DEV).to(BF16) for i in range(2)]
    w = ops.prepare_matrix_int8(*quantize_matrix(torch.randn((512, 1024), generator=_gen(7), device=DEV)))
    want = [torch.empty((300, 512), dtype=BF16, device=DEV) for _ in range(2)]
    for x, y in zip(inputs, want):
        ops.linear(x, w, y)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros_like(y) for y in want]
    for _ in range(20):
        for s, x, y in zip(streams, inputs, outs):
            with torch.cuda.stream(s):
                ops.linear(x, w, y)
    torch.cuda.synchronize()
    for y, z in zip(outs, want):
        assert torch.equal(y, z)
