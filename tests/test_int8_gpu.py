"""Products in 8 bits against 64-bit forms."""
import math

import pytest
import torch

from leone_b200.ops.cuda import KernelError
from leone_b200.ops.int8 import NARROW, PAIRS, STREAM, quantize_matrix
from tests.fewer_bits import quantize8

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops_of():
    from leone_b200.ops.cuda import CudaOps
    made = {}

    def get(dtype):
        if dtype not in made:
            made[dtype] = CudaOps(DEV, dtype)
            made[dtype].bind_status(torch.zeros(4, dtype=torch.int32, device=DEV))
        return made[dtype]
    yield get
    torch.cuda.synchronize()
    for ops in made.values():
        assert ops.status.tolist() == [0, 0, 0, 0]


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _inputs(m, n, k, dtype, seed):
    x = torch.randn((m, k), generator=_gen(seed), device=DEV)
    x[:, ::61] *= 15
    return x.to(dtype), *quantize_matrix(torch.randn((n, k), generator=_gen(seed + 1), device=DEV) * 0.02)


def _want(x, codes, scales):
    a, s = quantize8(x.double())
    return (a @ codes.double().T) * s * scales.double()


def _check(got, want, also, dtype):
    """The integer sum is exact; sum, two scales, a product each, then what is added (`also`): six roundings of 32 bits, one to the type."""
    bound = (want.abs() + also.abs()) * (6 * 2.0 ** -24 + torch.finfo(dtype).eps / 2) + 1e-37
    err = (got.double() - want).abs()
    assert (err <= bound).all(), f"worst {float((err / bound).max())} of the bound at {int((err / bound).argmax())}"


SIZES = [(1, 4096, 2048), (8, 64, 16), (3, 32, 4096), (17, 1000, 272), (33, 4096, 144), (77, 2048, 6144), (128, 96, 1040), (129, 6144, 4096),
         (300, 31, 128), (513, 2100, 528), (5, 24576, 256), (2048, 256, 12288)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("bias", [False, True])
def test_linear(ops_of, m, n, k, dtype, bias):
    ops = ops_of(dtype)
    x, codes, scales = _inputs(m, n, k, dtype, m + n)
    b = torch.randn(n, generator=_gen(3), device=DEV) if bias else None
    w = ops.prepare_matrix_int8(codes, scales, b)
    zero = torch.zeros((), device=DEV, dtype=torch.float64) if b is None else b.double()
    want = _want(x, codes, scales)
    out = torch.full((m, n), 9.0, dtype=dtype, device=DEV)
    ops.linear(x, w, out)
    _check(out, want + zero, zero, dtype)
    wide = torch.full((m, n), 9.0, dtype=FP32, device=DEV)
    ops.linear(x, w, wide)
    _check(wide, want + zero, zero, FP32)
    residual = torch.randn((m, n), generator=_gen(4), device=DEV)
    stream = residual.clone()
    ops.linear(x, w, stream, residual=stream)
    _check(stream, want + zero + residual.double(), residual.double().abs() + zero.abs(), FP32)


@pytest.mark.parametrize("form", [(form, width) for form in (NARROW, PAIRS) for width in (32, 64, 96, 128, 192, 224, 256)]
                         + [(STREAM, splits) for splits in range(1, 9)])
def test_forms(ops_of, form):
    """Every tile width on single SMs and on pairs and every split of the stream, whatever the rule would take."""
    ops = ops_of(BF16)
    sizes = [(1, 400, 272), (17, 1056, 1040), (32, 96, 4096), (7, 4000, 128)] if form[0] == STREAM else \
        [(1, 400, 272), (130, 1056, 1040), (257, 96, 4096)]
    for m, n, k in sizes:
        x, codes, scales = _inputs(m, n, k, BF16, m)
        w = ops.prepare_matrix_int8(codes, scales)
        out, wide = torch.empty((m, n), dtype=BF16, device=DEV), torch.empty((m, n), device=DEV)
        residual = torch.randn((m, n), generator=_gen(8), device=DEV)
        stream = residual.clone()
        ops.int8.force = form
        try:
            ops.linear(x, w, out)
            ops.linear(x, w, wide)
            ops.linear(x, w, stream, residual=stream)
        finally:
            ops.int8.force = None
        want = _want(x, codes, scales)
        _check(out, want, want * 0, BF16)
        _check(wide, want, want * 0, FP32)
        _check(stream, want + residual.double(), residual.double(), FP32)


GATES = [None, (1.0, 7.0, 1.0, 0.0), (1.595769, math.inf, 0.0, 0.044715)]


@pytest.mark.parametrize("m,inter,k", [(1, 48, 64), (8, 12288, 128), (40, 16, 4096), (200, 1040, 272), (9, 24, 96), (700, 512, 1024)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", GATES)
def test_linear_swiglu(ops_of, m, inter, k, dtype, shape):
    ops = ops_of(dtype)
    x, codes, scales = _inputs(m, 2 * inter, k, dtype, m + inter)
    scales *= 8
    bias = torch.randn(2 * inter, generator=_gen(3), device=DEV)
    half = lambda t: (t[:inter], t[inter:])  # noqa: E731
    w = ops.prepare_gate_up_int8(codes[:inter], scales[:inter], codes[inter:], scales[inter:], *half(bias))
    out = torch.full((m, inter), 9.0, dtype=dtype, device=DEV)
    ops.linear_swiglu(x, w, out, gate_shape=shape)
    sums = _want(x, codes, scales)
    y = sums + bias.double()
    # gate and up are off by six roundings of the parts that they are sums of, which may cancel: with |d (g sigmoid(z)) / dg| <= 1 + |z| / 4
    # (z = slope g (1 + cubic g^2), of which these shapes' slope and cubic term add at most a factor of 3 + |z|)
    parts = (sums.abs() + bias.double().abs()) * 6 * 2.0 ** -24
    g, u = y[:, :inter], y[:, inter:]
    slope, limit, shift, cubic = shape or (1.0, math.inf, 0.0, 0.0)
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    z = slope * g * (1 + cubic * g * g)
    want = g * torch.sigmoid(z) * (u + shift)
    if dtype == FP32 or w.gate_up_layout == "stacked":
        # gate and up stand in the run's type in between: half a step of each, of which the gate's moves its sigmoid's argument too
        t = torch.finfo(dtype).eps / 2
        rel = 2 * t + 3 * t * z.abs() + 2.0 ** -20 * (1 + z.abs())
    else:
        t, rel = 2.0 ** -8, 2.0 ** -19 * (1 + z.abs())
    cancelled = (g * torch.sigmoid(z)).abs() * parts[:, inter:] + (u + shift).abs() * parts[:, :inter] * (3 + z.abs())
    spread = (g * torch.sigmoid(z)).abs() * ((u + shift).abs() + u.abs())
    assert ((out.double() - want).abs() <= spread * rel + want.abs() * t + 1e-6 * spread + cancelled + 1e-30).all()


def test_rows_that_are_zero_or_not_finite(ops_of):
    for dtype in (BF16, FP32):
        ops = ops_of(dtype)
        x, codes, scales = _inputs(6, 64, 128, dtype, 1)
        x[0] = 0
        x[1, 5] = math.inf
        x[2, 127] = math.nan
        x[3] *= 1e-38                                         # 127 / max has no fp32
        x[4, 0] = 3e38
        w = ops.prepare_matrix_int8(codes, scales)
        out = torch.empty((6, 64), dtype=dtype, device=DEV)
        ops.linear(x, w, out)
        assert (out[0] == 0).all() and out[1].isnan().all() and out[2].isnan().all()
        rest = [3, 4, 5]
        want = _want(x[rest], codes, scales)
        _check(out[rest], want, want * 0 + 1e-39, dtype)


def test_codes_at_the_border_of_two(ops_of):
    """Values that lie exactly between two codes go to the even one, and their neighbours in fp32 to their own side."""
    ops = ops_of(FP32)
    k = 256
    half = torch.arange(-126, 127, device=DEV, dtype=FP32) + 0.5
    x = torch.zeros((3, k), device=DEV)
    x[:, 0] = 127.0
    x[0, 1:254], x[1, 1:254] = half, torch.nextafter(half, torch.full_like(half, 1e9))
    x[2, 1:254] = torch.nextafter(half, torch.full_like(half, -1e9))
    w = ops.prepare_matrix_int8(torch.eye(k, device=DEV, dtype=torch.int8).contiguous(), torch.ones(k, device=DEV))
    out = torch.empty((3, k), device=DEV)
    ops.linear(x, w, out)
    assert torch.equal(out.double(), torch.round(x.double()))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("k,lead", [(16, 0), (2048, 0), (2048, 1), (4112, 8), (16384, 0), (16400, 0), (20000, 0)])
def test_codes_of_tokens(ops_of, dtype, k, lead):
    """Rows as the kernels round them, for every form that the rounding has."""
    ops = ops_of(dtype)
    x = torch.randn((5, k + 16), generator=_gen(k), device=DEV).to(dtype)[:, lead:lead + k]
    codes, scales = torch.empty((5, k), dtype=torch.int8, device=DEV), torch.empty(5, device=DEV)
    assert ops.int8.calls.leone_quantize_rows(0 if dtype == FP32 else 1, x, 5, k, x.stride(0), codes, scales, ops._stream()) == 0
    want, s = quantize8(x.double())
    assert torch.equal(codes.double(), want) and torch.equal(scales, s[:, 0].float())


def test_strided_inputs_and_outputs(ops_of):
    ops = ops_of(BF16)
    x, codes, scales = _inputs(20, 100, 64, BF16, 2)
    w = ops.prepare_matrix_int8(codes, scales)
    wide = torch.full((20, 131), 5.0, dtype=BF16, device=DEV)
    rows = torch.randn((20, 200), generator=_gen(1), device=DEV).to(BF16)
    rows[:, 7:71] = x
    ops.linear(rows[:, 7:71], w, wide[:, 3:103])
    plain = torch.empty((20, 100), dtype=BF16, device=DEV)
    ops.linear(x, w, plain)
    assert torch.equal(wide[:, 3:103], plain)
    assert (wide[:, :3] == 5).all() and (wide[:, 103:] == 5).all()


def test_refusals(ops_of):
    ops = ops_of(BF16)
    x, codes, scales = _inputs(4, 64, 128, BF16, 2)
    out = torch.empty((4, 64), dtype=BF16, device=DEV)
    w = ops.prepare_matrix_int8(codes, scales)
    for args, match in [((codes[:, :120], scales), "contiguous"), ((codes[:, :120].contiguous(), scales), "multiple of 16"),
                        ((codes.float(), scales), "int8"), ((codes, scales[:5]), "one per row"), ((codes, scales.double()), "fp32"),
                        ((codes.cpu(), scales.cpu()), "lies on")]:
        with pytest.raises(KernelError, match=match):
            ops.prepare_matrix_int8(*args)
    with pytest.raises(KernelError, match="one number per row"):
        ops.prepare_matrix_int8(codes, scales, torch.zeros(3, device=DEV))
    with pytest.raises(KernelError, match="chain"):
        ops.linear(x[:, :64], w, out)
    with pytest.raises(KernelError, match="dtype"):
        ops.linear(x.half(), w, out)
    with pytest.raises(KernelError, match="output shape"):
        ops.linear_swiglu(x, w, out)
    with pytest.raises(KernelError, match="gate and up"):
        ops.linear_swiglu(x, w, out[:, :32].contiguous())
    with pytest.raises(KernelError, match="differ"):
        ops.prepare_gate_up_int8(codes, scales, codes[:32], scales[:32])
    ops.linear(x[:0], w, out[:0])                              # no tokens: nothing to do


@pytest.mark.parametrize("m,n,k", [(3, 4096, 8192), (100, 2048, 8192), (300, 2048, 4096)])
def test_two_graphs_at_once(ops_of, m, n, k):
    """Two captured products of one width, replayed beside one another on two streams, and two eager ones: each has its own tokens."""
    ops = ops_of(BF16)
    cases = []
    for seed in (1, 2):
        x, codes, scales = _inputs(m, n, k, BF16, seed)
        w, want = ops.prepare_matrix_int8(codes, scales), torch.empty((m, n), dtype=BF16, device=DEV)
        ops.linear(x, w, want)
        cases.append((x, w, torch.empty_like(want), want))
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for x, w, got, _ in cases:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=streams[0]):
            ops.linear(x, w, got)
        graphs.append(graph)
    for eager in (False, True):
        for _ in range(20):
            for case in cases:
                case[2].zero_()
            torch.cuda.synchronize()
            for stream, graph, (x, w, got, _) in zip(streams, graphs, cases):
                with torch.cuda.stream(stream):
                    if eager:
                        ops.linear(x, w, got)
                    else:
                        graph.replay()
            torch.cuda.synchronize()
            for _, _, got, want in cases:
                assert torch.equal(got, want)
    del graphs
