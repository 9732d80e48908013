"""Products of 8-bit integers: a tile's width moves no bit of a result."""
import pytest
import torch

from leone_b200.ops.int8 import MAX_K, NARROW, PAIRS, Int8Products
from tests.test_int8_gpu import BF16, DEV, _check, _gen, _inputs, _want, ops_of  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", [NARROW, PAIRS])
@pytest.mark.parametrize("m,n,k", [(1, 400, 272), (129, 9760, 1024), (257, 96, 4096), (300, 1056, 1040), (130, 1600, 144)])
def test_every_width(ops_of, form, m, n, k):  # noqa: F811
    """All widths that the rule chooses from, with a bias, onto a residual and through the gates: the sums are exact and the epilogue is one, so
    that results are equal bit for bit, and those of one width are right."""
    ops = ops_of(BF16)
    x, codes, scales = _inputs(m, n, k, BF16, m)
    bias = torch.randn(n, generator=_gen(3), device=DEV)
    plain, biased = ops.prepare_matrix_int8(codes, scales), ops.prepare_matrix_int8(codes, scales, bias)
    half = n // 2
    gates = [ops.prepare_gate_up_int8(codes[:half], scales[:half], codes[half:], scales[half:], *b) for b in ((), (bias[:half], bias[half:]))] \
        if half % 16 == 0 else []
    residual = torch.randn((m, n), generator=_gen(8), device=DEV)

    def results(width):
        outs = [torch.full((m, n), 9.0, dtype=dtype, device=DEV) for dtype in (BF16, torch.float32, BF16, torch.float32)] + [residual.clone()]
        ops.int8.force = (form, width)
        try:
            for w, out in zip((plain, plain, biased, biased), outs):
                ops.linear(x, w, out)
            ops.linear(x, biased, outs[4], residual=outs[4])
            for w in gates:
                for shape in (None, (1.0, 7.0, 1.0, 0.0)):
                    outs.append(torch.full((m, half), 9.0, dtype=BF16, device=DEV))
                    ops.linear_swiglu(x, w, outs[-1], gate_shape=shape)
        finally:
            ops.int8.force = None
        return outs

    first = results(64)
    want = _want(x, codes, scales)
    _check(first[0], want, want * 0, BF16)
    _check(first[1], want, want * 0, torch.float32)
    _check(first[3], want + bias.double(), bias.double(), torch.float32)
    for width in range(32, 257, 32):
        for a, b in zip(first, results(width)):
            assert torch.equal(a, b), width


def test_the_rule_takes_160_weight_rows(ops_of):  # noqa: F811
    products: Int8Products = ops_of(BF16).int8
    assert products.choose(129, 9760, 1024) == (PAIRS, 160)


@pytest.mark.parametrize("m,n,k", [(1, 96, 256), (5, 96, 256), (140, 400, 272)])
def test_rows_that_are_one(ops_of, m, n, k):  # noqa: F811
    """A row that is broadcast over the tokens, and rows that overlap, as products in the run dtype take them."""
    ops = ops_of(BF16)
    x, codes, scales = _inputs(m, n, k, BF16, m)
    w = ops.prepare_matrix_int8(codes, scales)
    for rows in (x[:1].expand(m, k), x.flatten().as_strided((m, k), (16 if m > 1 else 0, 1)) if m * k >= 16 * m + k else x[:1]):
        out = torch.empty((rows.shape[0], n), dtype=BF16, device=DEV)
        ops.linear(rows, w, out)
        want = _want(rows, codes, scales)
        _check(out, want, want * 0, BF16)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_the_largest_sums(ops_of, m):  # noqa: F811
    """The widest matrix that is taken, all codes 127: sums of 2.11e9 stay in 32 bits, in every form."""
    ops = ops_of(BF16)
    k, n = MAX_K, 96
    x = torch.full((m, k), 2.0, dtype=BF16, device=DEV)
    x[:, 1::2] *= torch.where(torch.arange(m, device=DEV) % 2 == 0, 1.0, -1.0).to(BF16)[:, None]         # (odd rows: 0)
    codes = torch.full((n, k), 127, dtype=torch.int8, device=DEV)
    codes[1] = -127
    w = ops.prepare_matrix_int8(codes, torch.ones(n, device=DEV))
    out = torch.full((m, n), 9.0, device=DEV)
    ops.linear(x, w, out)
    want = torch.full((m, n), 127.0 * k * 2.0, dtype=torch.float64, device=DEV)
    want[:, 1] *= -1
    want[1::2] = 0
    assert ((out.double() - want).abs() <= want.abs() * 4 * 2.0 ** -24).all()


@pytest.mark.parametrize("m", [5, 60, 200])
@pytest.mark.parametrize("n", [96, 100, 33])
def test_strided_rows_in_every_form(ops_of, m, n):  # noqa: F811
    """Tokens, outputs and residuals that are columns of wider rows, on odd elements: as the same without gaps, and nothing beside them."""
    ops = ops_of(BF16)
    k = 208
    x, codes, scales = _inputs(m, n, k, BF16, 2)
    w = ops.prepare_matrix_int8(codes, scales, torch.randn(n, generator=_gen(1), device=DEV))
    rows = torch.randn((m, k + 31), generator=_gen(2), device=DEV).to(BF16)
    rows[:, 7:7 + k] = x
    for dtype, residual in ((BF16, False), (torch.float32, False), (torch.float32, True)):
        start = torch.randn((m, n), generator=_gen(3), device=DEV).to(dtype)
        plain, wide = start.clone(), torch.full((m, n + 31), 5.0, dtype=dtype, device=DEV)
        wide[:, 3:3 + n] = start
        into = wide[:, 3:3 + n]
        ops.linear(x, w, plain, residual=plain if residual else None)
        ops.linear(rows[:, 7:7 + k], w, into, residual=into if residual else None)
        assert torch.equal(into, plain)
        assert (wide[:, :3] == 5).all() and (wide[:, 3 + n:] == 5).all()
        want = _want(x, codes, scales) + w.bias.double() + (start.double() if residual else 0)
        _check(plain, want, w.bias.double().abs() + start.double().abs(), dtype)
    if n == 96:
        gate = ops.prepare_gate_up_int8(codes[:48], scales[:48], codes[48:], scales[48:])
        plain = torch.empty((m, 48), dtype=BF16, device=DEV)
        ops.linear_swiglu(x, gate, plain)
        flat = torch.full((m * 48 + 9,), 5.0, dtype=BF16, device=DEV)
        ops.linear_swiglu(rows[:, 7:7 + k], gate, flat[3:-6].view(m, 48))
        assert torch.equal(flat[3:-6].view(m, 48), plain) and (flat[:3] == 5).all() and (flat[-6:] == 5).all()
