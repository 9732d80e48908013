"""Attention over pages in 4 bits in bfloat16: how far outputs are off in relation to their size, row by row.

Rounding to bfloat16 moves a number by 2^-7 / 12^(1/2) of its power of two in the mean square, 0.0016 of the numbers of a row.  Decode rounds
the weights times their scale and the output, portions round the values, the weights and the output; keys are exact or fp16 (an eighth
of that of a score's products).  Of many keys these are independent: 2^(1/2) 0.0016 of a call's outputs for decode and 3^(1/2) 0.0016 for
portions, a fourth more for the chance.  In a row where one key has all the weight, the weight's rounding is at most 2^-8 of every
element alike.  Sums in 32 bits are of 2^-23 and do not count.
"""
import pytest
import torch

from leone_b200.cache import packed
from tests.fewer_bits import Step, attention64, quantize4, values4
from tests.test_cache4_gpu import BF16, DECODE, DEV, PROMPT, _attention_case, _gen, ops_of  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

ROW = 2.0 ** -8 + 1.25 * 2 ** 0.5 * 0.0016
CALL = {"decode": 1.25 * 2 ** 0.5 * 0.0016, "prompt": 1.25 * 3 ** 0.5 * 0.0016}


def _errors(out, want):
    """Of every row (token, head), and of all of them; NaN counts as wrong."""
    off, size = (out - want).square(), want.square()
    rows = (off.sum(-1) / size.sum(-1)).sqrt()
    return float(rows.nan_to_num(9).max()), float((off.sum() / size.sum()).sqrt())


def _right(kind, out, want):
    row, call = _errors(out, want)
    # (of few rows one may be all of the call)
    return row < ROW and call < (CALL[kind] if want.shape[0] * want.shape[1] >= 200 else ROW)


@pytest.mark.parametrize("splits", [0, 1, 2, 7, 8, 9, 33, 64])
@pytest.mark.parametrize("n_q,n_kv,d,lens,page,window", DECODE)
def test_decode(ops_of, n_q, n_kv, d, lens, page, window, splits):  # noqa: F811
    ops = ops_of(BF16)
    ops.force_decode4_splits = splits
    try:
        *_, out, want, _, _ = _attention_case(ops, BF16, n_q, n_kv, d, lens, page, window, seed=d + n_q)
    finally:
        ops.force_decode4_splits = 0
    assert _right("decode", out, want), _errors(out, want)


@pytest.mark.parametrize("spread", [1, 3])
@pytest.mark.parametrize("splits", [0, 1, 2, 5, 64])
@pytest.mark.parametrize("n_q,n_kv,d,lens,page,window", PROMPT)
def test_prompt(ops_of, n_q, n_kv, d, lens, page, window, splits, spread):  # noqa: F811
    ops = ops_of(BF16)
    ops.force_prompt4_splits = splits
    try:
        *_, out, want, _, _ = _attention_case(ops, BF16, n_q, n_kv, d, lens, page, window, seed=d + n_q, stride=8, scale=spread * d ** -0.5)
    finally:
        ops.force_prompt4_splits = 0
    assert _right("prompt", out, want), _errors(out, want)


def _plain(q, k, v, scale):
    """One sequence's last token: q [n_q, d], k and v [keys, n_kv, d]."""
    g = q.shape[0] // k.shape[1]
    score = torch.einsum("hd,khd->hk", q, k.repeat_interleave(g, 1)) * scale
    return torch.einsum("hk,khd->hd", torch.softmax(score, 1), v.repeat_interleave(g, 1))


def test_the_bounds_see_what_is_wrong():
    """An output of zeros, a 64th of 9,000 keys left out, keys rounded to bfloat16: each is out of bounds, by the plain form alone."""
    gen = torch.Generator("cuda:0").manual_seed(1)
    q, k, v = (torch.randn(shape, generator=gen, device="cuda:0", dtype=torch.float64) for shape in ((8, 128), (9000, 1, 128), (9000, 1, 128)))
    k[..., ::19] *= 4
    want = _plain(q, k, v, 128 ** -0.5)[None]
    assert not _right("decode", torch.zeros_like(want), want)
    kept = torch.ones(9000, dtype=torch.bool, device="cuda:0")
    kept[5000:5140] = False
    assert not _right("decode", _plain(q, k[kept], v[kept], 128 ** -0.5)[None], want)
    q = torch.randn((400, 128), generator=gen, device="cuda:0", dtype=torch.float64)
    want, off = (_plain(q, x, v, 3 * 128 ** -0.5)[None] for x in (k, k.bfloat16().double()))
    assert not _right("prompt", off, want)
    assert _right("prompt", _plain(q, k.half().double(), v, 3 * 128 ** -0.5)[None], want)


@pytest.mark.parametrize("power", [-60, -57, -30, 30, 52])
@pytest.mark.parametrize("d,lens,splits", [(64, [(1, 300), (1, 40)], 1), (128, [(1, 300), (1, 700)], 1), (128, [(1, 900)], 9), (64, [(60, 300)], 1),
                                           (128, [(60, 300)], 2)])
def test_values_of_any_size(ops_of, d, lens, splits, power):  # noqa: F811
    """Values of 2^-60 to 2^52, whose scales are an eighth of them and more: the error in relation to the output is the same."""
    ops = ops_of(BF16)
    step = Step(lens, 16, DEV, seed=1)
    pools, plain = [], []
    for values, size in ((False, 1.0), (True, 2.0 ** power)):
        coded = quantize4(torch.randn((step.pages, 2, 16, d), generator=_gen(3 + values), device=DEV).double() * size)
        pools.append(packed.pack_pages(*coded, values))
        plain.append(values4(*coded))
    n = step.ctx.n_tokens
    qkv = torch.randn((n, 8 * d), generator=_gen(9), device=DEV).to(BF16)
    out = torch.zeros((n, 4 * d), dtype=BF16, device=DEV)
    ops.force_decode4_splits = ops.force_prompt4_splits = splits
    try:
        ops.attention(step.ctx, qkv, out, 4, 2, d, d ** -0.5, None, step.view(*pools))
    finally:
        ops.force_decode4_splits = ops.force_prompt4_splits = 0
    want, *_ = attention64(qkv[:, :4 * d].double().unflatten(1, (4, d)), *plain, lens, step.table, 16, d ** -0.5, 0)
    out = out.double().view_as(want)
    assert _right("prompt" if n > len(lens) else "decode", out * 2.0 ** -power, want * 2.0 ** -power), _errors(out, want)
