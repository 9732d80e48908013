"""Pages in 4 bits: append, read and attention against plain 64-bit forms."""
import math

import pytest
import torch

from leone_b200.cache import packed
from leone_b200.ops.cuda import KernelError
from leone_b200.parts.rotary import build_rotary_table
from tests.fewer_bits import Step, attention64, quantize4, rotate, values4

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
    return get


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _pools(step, n_kv, d, fill=0):
    return [torch.full((step.pages, n_kv, step.page_tokens, packed.row_bytes(d)), fill, dtype=torch.uint8, device=DEV) for _ in range(2)]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


APPENDS = [
    # dtype, d, n_q, n_kv, norm, pairing, rotary elements, page tokens, lens
    (BF16, 128, 16, 8, True, "half_split", 128, 16, [(1, 700)]),
    (BF16, 128, 32, 8, True, "half_split", 128, 16, [(75, 0), (1, 30), (40, 9)]),
    (BF16, 128, 3, 1, True, "adjacent", 128, 48, [(33, 47), (1, 0)]),
    (BF16, 64, 14, 2, False, "half_split", 64, 32, [(5, 3), (17, 40)]),
    (BF16, 64, 4, 4, True, "adjacent", 32, 16, [(20, 1)]),                    # a part of a head rotates
    (BF16, 256, 8, 2, True, "half_split", 256, 16, [(9, 100)]),
    (BF16, 128, 8, 2, True, None, 0, 16, [(30, 2)]),                          # no rotation
    (FP32, 64, 12, 4, False, "adjacent", 64, 16, [(30, 77), (2, 0)]),
    (FP32, 128, 2, 1, True, "half_split", 128, 16, [(1, 0), (1, 15), (1, 16), (50, 3)]),
    (FP32, 16, 4, 2, True, "half_split", 16, 16, [(21, 2), (7, 0)]),
    (FP32, 96, 4, 2, True, "half_split", 96, 16, [(11, 6)]),
    (FP32, 512, 2, 1, True, "half_split", 512, 16, [(3, 14)]),
    (BF16, 192, 4, 2, True, "adjacent", 192, 16, [(6, 10)]),
]


@pytest.mark.parametrize("dtype,d,n_q,n_kv,norm,pairing,rot,page,lens", APPENDS)
@pytest.mark.parametrize("wdtype", [FP32, BF16])
def test_append_and_read(ops_of, dtype, d, n_q, n_kv, norm, pairing, rot, page, lens, wdtype):
    ops = ops_of(dtype)
    step = Step(lens, page, DEV, seed=d)
    n = step.ctx.n_tokens
    rows = torch.randn((n, (n_q + 2 * n_kv) * d), generator=_gen(d + n), device=DEV)
    rows[:, ::37] *= 9
    rows = rows.to(dtype)
    weights = (1 + 0.1 * torch.randn((2, d), generator=_gen(2), device=DEV)).to(wdtype) if norm else (None, None)
    k_pool, v_pool = _pools(step, n_kv, d, fill=0xA5)
    view = step.view(k_pool, v_pool)
    table = build_rotary_table(int(step.pos.max()) + 1, rot, 10000.0).to(DEV) if rot else None
    got = rows.clone()
    kw = {} if pairing is None else {"pairing": pairing}
    eps = 2.0 ** -20
    ops.qk_norm_rope_write(step.ctx, got, n_q, n_kv, d, weights[0], weights[1], eps, table, rot, view, **kw)

    q, k, v = rows.double().unflatten(1, (n_q + 2 * n_kv, d)).split([n_q, n_kv, n_kv], 1)
    if norm:
        q, k = (x * w.double() * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) for x, w in ((q, weights[0]), (k, weights[1])))
    partner = torch.zeros_like(q)
    if rot:
        turned = q[..., :rot]
        partner[..., :rot] = torch.cat([turned[..., rot // 2:], turned[..., :rot // 2]], -1) if pairing == "half_split" else \
            turned.unflatten(-1, (-1, 2)).flip(-1).flatten(-2)
    pair = (q.abs() + partner.abs()).flatten(1)
    if rot:
        q, k = (rotate(x, step.pos, 10000.0, pairing, rot) for x in (q, k))
    # Queries, in units of 2^-24: an element before the rotation is off by half of the roundings of a sum of squares (nine or less for
    # lanes of a warp; d / 32 + 5 in the form of any size, which is in 64 bits), four for the reciprocal root and its argument, and two
    # products, an element after it by a product's and a sum's more of its pair's two elements: 13 (|a| + |b|) with all of them,
    # and one rounding to the type.
    want = q.flatten(1)
    bound = want.abs() * _half_step(dtype) + pair * 13 * 2.0 ** -24 + 1e-30
    assert ((got[:, :n_q * d].double() - want).abs() <= bound).all()
    assert torch.equal(got[:, n_q * d:], rows[:, n_q * d:])                    # keys and values are not written back
    held = []
    for pool, x, values in ((k_pool, k, False), (v_pool, v, True)):
        codes, s, z = packed.unpack_pages(pool, d, values)
        have = (codes[step.page, :, step.slot], s[step.page, :, step.slot], z[step.page, :, step.slot])
        want_codes, want_s, want_z = quantize4(x)
        assert torch.equal(have[0].long(), want_codes)
        assert torch.equal(have[1].double(), want_s) and torch.equal(have[2].double(), want_z)
        # off by at most half a scale
        err = (values4(*have) - x).abs().unflatten(-1, (s.shape[-1], -1))
        assert (err <= want_s[..., None] * (0.5 + 2.0 ** -20) + 1e-300).all()
        # no other byte moved
        other = torch.ones(pool.shape[:3], dtype=torch.bool, device=DEV)
        other[step.page, :, step.slot] = False
        fill = packed.unpack_pages(torch.full_like(pool, 0xA5), d, values)
        for a, b in zip((codes, s, z), fill):
            assert torch.equal(a[other].float(), b[other].float())
        held.append(values4(*have))
    k_out, v_out = torch.full((2, n, n_kv * d), 7.0, dtype=dtype, device=DEV)
    ops.read_packed_rows(step.ctx, view, n_kv, d, k_out, v_out)
    for out, x in zip((k_out, v_out), held):
        assert torch.equal(out, x.flatten(1).float().to(dtype))
    assert step.ctx.status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("d", [64, 128, 32])
def test_append_of_odd_groups(ops_of, dtype, d):
    """Constant groups, zeros, the smallest and largest numbers, infinities and NaN."""
    ops = ops_of(dtype)
    step = Step([(9, 3)], 16, DEV)
    x = torch.randn((9, 3, d), generator=_gen(5), device=DEV)
    x[0] = 0.0
    x[1] = -2.7
    x[2] *= 1e-38
    x[3, :, 0] = math.inf
    x[4, :, d - 1] = math.nan
    x[5, :, 0], x[5, :, 1] = 3.3e38, -3.3e38
    x[6] = 5e-39                                             # no normal number
    x[7, :, 3] = -math.inf
    x[8] = 1000.0 + x[8]
    rows = x.to(dtype).flatten(1)
    pools = _pools(step, 1, d)
    ops.qk_norm_rope_write(step.ctx, rows.clone(), 1, 1, d, None, None, 1e-6, None, 0, step.view(*pools))
    want = quantize4(rows.double().unflatten(1, (3, d)))
    for i, (pool, values) in enumerate(zip(pools, (False, True))):
        codes, s, z = (t[step.page, 0, step.slot] for t in packed.unpack_pages(pool, d, values))
        assert torch.equal(codes.long(), want[0][:, 1 + i])
        torch.testing.assert_close(s.double(), want[1][:, 1 + i], rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(z.double(), want[2][:, 1 + i], rtol=0, atol=0, equal_nan=True)
    assert step.ctx.status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("pairing", ["half_split", "adjacent"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype,d,n_kv", [(BF16, 128, 3), (FP32, 128, 2), (BF16, 64, 5), (FP32, 64, 1)])
def test_append_of_many_rows(ops_of, dtype, d, n_kv, norm, pairing):
    """So many rows that codes next to a border and scales in doubt are among them, and rows that no norm is at ease with."""
    ops = ops_of(dtype)
    step = Step([(1501, 0), (900, 333)], 16, DEV, seed=d)
    n, n_q = step.ctx.n_tokens, 1
    x = torch.randn((n, n_q + 2 * n_kv, d), generator=_gen(n_kv), device=DEV)
    x[3] = 0.0
    x[4] = 1.5
    x[5] *= 1e-18
    x[6] *= 1e18
    x[7, :, 1:] *= 1e-7
    x[8] = torch.arange(d, device=DEV) / 16
    x[9] *= 1e-30
    x[1600] = -0.25
    rows = x.to(dtype).flatten(1)
    weights = (1 + 0.1 * torch.randn((2, d), generator=_gen(2), device=DEV)).to(dtype) if norm else (None, None)
    pools = _pools(step, n_kv, d)
    table = build_rotary_table(int(step.pos.max()) + 1, d, 10000.0).to(DEV)
    eps = 2.0 ** -20
    ops.qk_norm_rope_write(step.ctx, rows.clone(), n_q, n_kv, d, weights[0], weights[1], eps, table, d, step.view(*pools),
                           pairing=pairing)
    k, v = rows.double().unflatten(1, (n_q + 2 * n_kv, d))[:, n_q:].split(n_kv, 1)
    if norm:
        k = k * weights[1].double() * torch.rsqrt(k.square().mean(-1, keepdim=True) + eps)
    k = rotate(k, step.pos, 10000.0, pairing, d)
    for pool, want, values in ((pools[0], k, False), (pools[1], v, True)):
        have = [t[step.page, :, step.slot] for t in packed.unpack_pages(pool, d, values)]
        codes, s, z = quantize4(want)
        assert torch.equal(have[1].double(), s) and torch.equal(have[2].double(), z)
        assert torch.equal(have[0].long(), codes)
    assert step.ctx.status.tolist() == [0, 0, 0, 0]


def test_append_and_read_report_bad_metadata(ops_of):
    ops = ops_of(BF16)
    d, n_kv = 128, 2
    rows = torch.randn((3, 4 * d + 2 * d), generator=_gen(1), device=DEV).to(BF16)
    table = build_rotary_table(64, d, 10000.0).to(DEV)
    for spoil, code in (("page", 2), ("far page", 2), ("sequence", 5), ("position", 3)):
        step = Step([(3, 17)], 16, DEV)
        if spoil == "page":
            step.table[0, 1] = -1
        if spoil == "far page":
            step.table[0, 1] = step.pages
        if spoil == "sequence":
            step.ctx.seq_of_token[1] = 1
        if spoil == "position":
            step.ctx.positions[2] = 64
        pools = _pools(step, n_kv, d, fill=3)
        ops.qk_norm_rope_write(step.ctx, rows.clone(), 2, n_kv, d, None, None, 1e-6, table, d, step.view(*pools))
        assert int(step.ctx.status[0]) == code, spoil
        step.ctx.status.zero_()
        out = torch.full((2, 3, n_kv * d), 5.0, dtype=BF16, device=DEV)
        ops.read_packed_rows(step.ctx, step.view(*pools), n_kv, d, *out)
        assert int(step.ctx.status[0]) == (2 if spoil == "position" else code), spoil


def _attention_case(ops, dtype, n_q, n_kv, d, lens, page, window, seed=0, stale=True, stride=0, scale=None):
    step = Step(lens, page, DEV, seed=seed, window=window)
    pools, plain = [], []
    for values in (False, True):
        x = torch.randn((step.pages, n_kv, page, d), generator=_gen(seed + 3 + values), device=DEV).double()
        if not values:
            x[..., ::19] *= 4
        codes, s, z = quantize4(x)
        plain.append(values4(codes, s, z))
        pool = packed.pack_pages(codes, s, z, values)
        if stale:
            # rows that hold no token of a sequence are NaN: nothing of them may reach a result
            owned = torch.zeros((step.pages, page), dtype=torch.bool, device=DEV)
            for i, (new, past) in enumerate(lens):
                p = torch.arange(max(0, past - window + 1) if window else 0, new + past, device=DEV)
                owned[step.table[i, p // page].long(), p % page] = True
            broken = packed.pack_pages(codes, torch.where(owned[:, None, :, None], s, math.nan),
                                       torch.where(owned[:, None, :, None], z, math.nan), values)
            pool = broken
        pools.append(pool)
    n = step.ctx.n_tokens
    cols = (n_q + 2 * n_kv) * d + stride
    qkv = torch.randn((n, cols), generator=_gen(seed + 9), device=DEV).to(dtype)
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((n, n_q * d), 77.0, dtype=dtype, device=DEV)
    ops.attention(step.ctx, qkv, out, n_q, n_kv, d, scale, window or None, step.view(*pools))
    want, top_s, top_v = attention64(qkv[:, :n_q * d].double().unflatten(1, (n_q, d)), *plain, lens, step.table, page, scale, window)
    assert step.ctx.status.tolist() == [0, 0, 0, 0]
    return step, qkv, pools, out.unflatten(1, (n_q, d)).double(), want, top_s.double(), top_v.double()


def _bounds(dtype, step, d, n_q, want, top_s, top_v, tensor_cores):
    """How far an output may be off, per (token, head).

    Scores: d products summed in fp32, relative to sum |q k| at most (d + 4) 2^-23 (a tensor core's additions truncate).  On tensor cores
    a form may have codes as 128 + code, 9 times the largest code, and take the offset out again: 10 times that.  A score's error moves each
    weight by that much relative to itself, twice (the sum too).  Weights and sums: (keys + 8) 2^-23.  On tensor cores a weight times its
    scale is rounded to bfloat16: a half step of the weighted codes around their middle, 8 s <= 0.54 (max - min) of 2^-8 each; again
    codes of 128 + code in the sums.  Then one rounding to the type."""
    keys = torch.tensor(step.ctx.ctx_lens, device=DEV).double()[step.seq]
    score = (d + 4) * 2.0 ** -23 * top_s * (10 if tensor_cores else 1)
    weight = (keys + 8)[:, None] * 2.0 ** -23 * (10 if tensor_cores else 1)
    off = top_v * (2 * score + 2 * weight + (0.54 * 2 * 2.0 ** -8 if tensor_cores else 0))
    return off[..., None] + want.abs() * _half_step(dtype) + 1e-30


ANY = [
    # dtype, n_q, n_kv, d, lens, page, window
    (FP32, 4, 2, 16, [(5, 0), (1, 40)], 16, 0),
    (FP32, 12, 4, 64, [(3, 77), (1, 0), (20, 5)], 16, 0),
    (FP32, 16, 1, 128, [(1, 200), (2, 31)], 32, 0),                           # 16 query heads a cached one
    (FP32, 3, 1, 96, [(33, 30)], 16, 20),
    (FP32, 2, 2, 512, [(4, 60)], 48, 0),
    (FP32, 64, 8, 128, [(1, 300), (7, 100)], 16, 64),
    (BF16, 6, 2, 32, [(9, 50), (1, 0)], 16, 0),
    (BF16, 20, 1, 96, [(1, 130)], 16, 0),
    (BF16, 4, 2, 256, [(17, 100)], 16, 33),
]


@pytest.mark.parametrize("dtype,n_q,n_kv,d,lens,page,window", ANY)
def test_attention_any_size(ops_of, dtype, n_q, n_kv, d, lens, page, window):
    step, _, _, out, want, top_s, top_v = _attention_case(ops_of(dtype), dtype, n_q, n_kv, d, lens, page, window, seed=d)
    assert ((out - want).abs() <= _bounds(dtype, step, d, n_q, want, top_s, top_v, False)).all()


@pytest.mark.parametrize("splits", [1, 2, 5, 64])
@pytest.mark.parametrize("dtype,n_q,n_kv,d,lens,page,window", ANY + [(FP32, 8, 2, 128, [(1, 3000), (1, 0), (2, 31)], 16, 0),
                                                                     (BF16, 11, 1, 96, [(1, 700), (3, 90)], 32, 50)])
def test_attention_any_size_split(ops_of, dtype, n_q, n_kv, d, lens, page, window, splits):
    ops = ops_of(dtype)
    ops.force_any4_splits = splits
    try:
        step, qkv, pools, out, want, top_s, top_v = _attention_case(ops, dtype, n_q, n_kv, d, lens, page, window, seed=d, stride=3)
    finally:
        ops.force_any4_splits = 0
    # the parts' weights are three roundings more
    bound = _bounds(dtype, step, d, n_q, want, top_s, top_v, False) + (top_v * 3 * 2.0 ** -23)[..., None]
    assert ((out - want).abs() <= bound).all()


def test_attention_any_size_split_reports_bad_metadata(ops_of):
    ops = ops_of(FP32)
    n_q, n_kv, d = 4, 2, 64
    for spoil, status in (("page", [2, 0, -1, 32]), ("sequence", [5, 0, 9, 0]), ("position", [3, 0, -1, 0])):
        step, qkv, pools, *_ = _attention_case(ops, FP32, n_q, n_kv, d, [(1, 200), (1, 90)], 16, 0)
        if spoil == "page":
            step.table[0, 2] = -1
        if spoil == "sequence":
            step.ctx.seq_of_token[0] = 9
        if spoil == "position":
            step.ctx.positions[0] = -1
        out = torch.full((2, n_q * d), 5.0, device=DEV)
        ops.force_any4_splits = 3
        try:
            ops.attention(step.ctx, qkv, out, n_q, n_kv, d, 0.1, None, step.view(*pools))
        finally:
            ops.force_any4_splits = 0
        assert step.ctx.status.tolist() == status
        if spoil != "page":
            assert not out[0].any() and out[1].any()


DECODE = [
    # n_q, n_kv, d, lens, page, window
    (16, 8, 128, [(1, 511)], 16, 0),
    (32, 8, 128, [(1, 0), (1, 15), (1, 16), (1, 17), (1, 700)], 16, 0),
    (14, 2, 64, [(1, 100), (1, 1100), (1, 3)], 16, 500),
    (12, 1, 128, [(1, 300), (1, 64)], 48, 0),                                 # two tiles of heads
    (40, 2, 64, [(1, 300), (1, 1)], 16, 0),                                   # two groups of heads
    (5, 5, 128, [(1, 200)] * 40, 32, 33),
    (3, 1, 64, [(1, 2047)], 16, 16),
    (8, 1, 128, [(1, 9000)], 16, 0),
    (64, 8, 128, [(1, 130 + 7 * i) for i in range(20)], 16, 0),
]


@pytest.mark.parametrize("splits", [0, 1, 2, 7, 8, 9, 33, 64])
@pytest.mark.parametrize("n_q,n_kv,d,lens,page,window", DECODE)
def test_attention_decode(ops_of, n_q, n_kv, d, lens, page, window, splits):
    ops = ops_of(BF16)
    ops.force_decode4_splits = splits
    try:
        step, qkv, pools, out, want, top_s, top_v = _attention_case(ops, BF16, n_q, n_kv, d, lens, page, window, seed=d + n_q)
    finally:
        ops.force_decode4_splits = 0
    assert ((out - want).abs() <= _bounds(BF16, step, d, n_q, want, top_s, top_v, True)).all()


def test_attention_decode_in_an_order_and_in_a_graph(ops_of):
    ops = ops_of(BF16)
    lens = [(1, 37 * i) for i in range(50)]
    step, qkv, pools, out, want, top_s, top_v = _attention_case(ops, BF16, 16, 8, 128, lens, 16, 0)
    view = step.view(*pools)
    step.ctx.seq_order = torch.arange(49, -1, -1, dtype=torch.int32, device=DEV)
    again = torch.zeros((50, 16 * 128), dtype=BF16, device=DEV)
    ops.attention(step.ctx, qkv, again, 16, 8, 128, 128 ** -0.5, None, view)
    assert torch.equal(again.double().view_as(out), out)
    graph, got = torch.cuda.CUDAGraph(), torch.zeros_like(again)
    with torch.cuda.graph(graph):
        ops.attention(step.ctx, qkv, got, 16, 8, 128, 128 ** -0.5, None, view)
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(got, again)
    step.ctx.seq_order = step.ctx.seq_order[:3]
    with pytest.raises(KernelError, match="order"):
        ops.attention(step.ctx, qkv, again, 16, 8, 128, 128 ** -0.5, None, view)


def test_attention_decode_reports_a_bad_page(ops_of):
    ops = ops_of(BF16)
    for bad in (-1, 10 ** 6):
        step, qkv, pools, *_ = _attention_case(ops, BF16, 4, 2, 128, [(1, 200), (1, 90)], 16, 0)
        step.table[0, 3] = bad
        out = torch.zeros((2, 4 * 128), dtype=BF16, device=DEV)
        ops.attention(step.ctx, qkv, out, 4, 2, 128, 0.1, None, step.view(*pools))
        assert step.ctx.status.tolist() == [2, 0, bad if bad > 0 else -1, 48]


PROMPT = [
    # n_q, n_kv, d, lens, page, window
    (16, 8, 128, [(2, 0)], 16, 0),
    (32, 8, 128, [(300, 0), (77, 500), (2, 129)], 16, 0),
    (14, 2, 64, [(1, 100), (1, 700), (333, 1100)], 16, 500),                  # a mixed step
    (4, 4, 128, [(129, 127), (128, 128), (1, 0), (130, 0)], 32, 0),           # (a single row that does not lead)
    (40, 2, 64, [(65, 300), (3, 1)], 16, 0),
    (128, 1, 128, [(9, 200)], 16, 0),                                         # a query tile of one token
    (8, 2, 64, [(500, 30)], 48, 33),
    (6, 2, 128, [(40, 1000), (700, 0)], 16, 128),
    (5, 1, 128, [(31, 2000)], 16, 16),
]


@pytest.mark.parametrize("splits", [0, 1, 2, 5, 64])
@pytest.mark.parametrize("n_q,n_kv,d,lens,page,window", PROMPT)
def test_attention_prompt(ops_of, n_q, n_kv, d, lens, page, window, splits):
    ops = ops_of(BF16)
    ops.force_prompt4_splits = splits
    try:
        step, qkv, pools, out, want, top_s, top_v = _attention_case(ops, BF16, n_q, n_kv, d, lens, page, window, seed=d + n_q, stride=8)
    finally:
        ops.force_prompt4_splits = 0
    # keys and values stand as bfloat16 operands: a half step of each, the keys' in the scores (twice: the sum too)
    half = 2.0 ** -8
    extra = top_v * (2 * half * top_s + half)
    assert ((out - want).abs() <= _bounds(BF16, step, d, n_q, want, top_s, top_v, True) + extra[..., None]).all()


def test_attention_prompt_behind_an_odd_number_of_rows(ops_of):
    """Three leading rows, seven heads, three splits: an odd number of parts stands before the portion's."""
    ops = ops_of(BF16)
    n_q, n_kv, d = 7, 1, 64
    ops.force_prompt4_splits = 3
    try:
        step, qkv, pools, out, want, top_s, top_v = _attention_case(ops, BF16, n_q, n_kv, d, [(1, 30), (1, 7), (1, 100), (40, 700)], 16, 0)
    finally:
        ops.force_prompt4_splits = 0
    half = 2.0 ** -8
    extra = top_v * (2 * half * top_s + half)
    assert ((out - want).abs() <= _bounds(BF16, step, d, n_q, want, top_s, top_v, True) + extra[..., None]).all()


@pytest.mark.parametrize("lens,splits", [([(1, 9000)], 33), ([(40, 5000)], 18)])
def test_attention_of_two_graphs_at_once(ops_of, lens, splits):
    """Two captured calls that split their keys, replayed beside one another on two streams, and two eager ones: neither writes into the
    other's parts."""
    ops = ops_of(BF16)
    n_q, n_kv, d = 8, 2, 128
    ops.force_decode4_splits = ops.force_prompt4_splits = splits
    try:
        cases = []
        for seed in (1, 2):
            step, qkv, pools, out, *_ = _attention_case(ops, BF16, n_q, n_kv, d, lens, 16, 0, seed=seed)
            view, got = step.view(*pools), torch.zeros((qkv.shape[0], n_q * d), dtype=BF16, device=DEV)
            cases.append((step, qkv, view, got, out.flatten(1).to(BF16)))

        def call(step, qkv, view, got, _):
            ops.attention(step.ctx, qkv, got, n_q, n_kv, d, d ** -0.5, None, view)

        streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
        for case in cases:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=streams[0]):
                call(*case)
            graphs.append(graph)
        for eager in (False, True):
            for _ in range(20):
                for case in cases:
                    case[3].zero_()
                torch.cuda.synchronize()
                for stream, graph, case in zip(streams, graphs, cases):
                    with torch.cuda.stream(stream):
                        if eager:
                            call(*case)
                        else:
                            graph.replay()
                torch.cuda.synchronize()
                for case in cases:
                    assert torch.equal(case[3], case[4])
        del graphs
    finally:
        ops.force_decode4_splits = ops.force_prompt4_splits = 0


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("splits", [1, 2])
def test_values_and_keys_that_are_nan(ops_of, d, window, many, splits):
    """A group of a cached value that is NaN makes the group's columns NaN for the rows that see it, and nothing else; a key that is NaN
    makes every row NaN that sees it."""
    ops = ops_of(BF16)
    n_q, n_kv, lens = 4, 2, [(150, 60), (1, 90)]
    step = Step(lens, 16, DEV, window=window)
    bad_v = [(0, 70 + i) for i in range(45)] if many else [(0, 100), (0, 203), (1, 90)]
    bad_k = [(0, 140)]
    pools, plain = [], []
    for values in (False, True):
        x = torch.randn((step.pages, n_kv, 16, d), generator=_gen(7 + values), device=DEV).double()
        codes, s, z = quantize4(x)
        for seq, key in bad_v if values else bad_k:
            page = int(step.table[seq, key // 16])
            if page >= 0:
                s[page, 1, key % 16, -1] = z[page, 1, key % 16, -1] = math.nan
        pools.append(packed.pack_pages(codes, s, z, values))
        plain.append(values4(codes, s, z))
    qkv = torch.randn((151, (n_q + 2 * n_kv) * d), generator=_gen(9), device=DEV).to(BF16)
    out = torch.zeros((151, n_q * d), dtype=BF16, device=DEV)
    ops.force_prompt4_splits = splits
    try:
        ops.attention(step.ctx, qkv, out, n_q, n_kv, d, d ** -0.5, window or None, step.view(*pools))
    finally:
        ops.force_prompt4_splits = 0
    got = out.view(151, n_q, d).isnan()
    want = torch.zeros_like(got)
    for seq, first, count, past in ((0, 0, 150, 60), (1, 150, 1, 90)):
        for t in range(count):
            p = past + t
            sees = lambda key: key <= p and (not window or key > p - window)  # noqa: E731
            if any(s == seq and sees(key) for s, key in bad_v):
                want[first + t, 2:, d - 64 if d > 64 else 0:] = True
            if any(s == seq and sees(key) for s, key in bad_k):
                want[first + t, 2:] = True
    if many and window:
        # (more than fit into the kernel's list: the keys behind it count as one range)
        assert (got | ~want).all() and not got[:, :2].any()
    else:
        assert torch.equal(got, want)
    assert step.ctx.status.tolist() == [0, 0, 0, 0]


def test_attention_prompt_reports_a_bad_page(ops_of):
    ops = ops_of(BF16)
    for bad in (-1, 10 ** 6):
        step, qkv, pools, *_ = _attention_case(ops, BF16, 4, 2, 128, [(20, 200), (30, 90)], 16, 0)
        step.table[0, 3] = bad
        out = torch.zeros((50, 4 * 128), dtype=BF16, device=DEV)
        ops.attention(step.ctx, qkv, out, 4, 2, 128, 0.1, None, step.view(*pools))
        assert step.ctx.status.tolist()[0] == 2 and step.ctx.status.tolist()[3] == 48


def test_attention_refusals(ops_of):
    ops = ops_of(BF16)
    step = Step([(1, 20)], 16, DEV)
    d, n_q, n_kv = 128, 4, 2
    pools = _pools(step, n_kv, d)
    qkv = torch.zeros((1, (n_q + 2 * n_kv) * d), dtype=BF16, device=DEV)
    out = torch.zeros((1, n_q * d), dtype=BF16, device=DEV)
    good = step.view(*pools)

    def refused(match, **kw):
        args = dict(ctx=step.ctx, qkv=qkv, out=out, n_q=n_q, n_kv=n_kv, d=d, cache=good)
        args.update(kw)
        with pytest.raises(KernelError, match=match):
            ops.attention(args["ctx"], args["qkv"], args["out"], args["n_q"], args["n_kv"], args["d"], 0.1, None, args["cache"],
                          **({"fuse": {}} if "fuse" in kw else {}))

    refused("pool layout", cache=step.view(pools[0].view(torch.int8), pools[1]))
    refused("pool layout", cache=step.view(pools[0], None))
    refused("pool layout", cache=step.view(pools[0][:, :, :, :64], pools[1]))
    refused("pool layout", cache=step.view(pools[0].transpose(0, 1), pools[1].transpose(0, 1)))
    refused("output layout", out=out[:, :64])
    refused("written before", fuse=True)
    refused("query rows", n_q=3, out=out[:, :3 * d].contiguous())
    odd = Step([(1, 20)], 24, DEV)
    refused("pool layout", cache=odd.view(*_pools(odd, n_kv, d)))
    with pytest.raises(KernelError, match="cannot be held"):
        ops.qk_norm_rope_write(step.ctx, torch.zeros((1, 3 * 20), dtype=BF16, device=DEV), 1, 1, 20, None, None, 1e-6, None, 0, good)
    bad = step.view(*pools)
    bad.block_table = step.table.long()
    refused("block table", cache=bad)
    bad.block_table = step.table[:0]
    refused("row of the block table", cache=bad)
    with pytest.raises(KernelError, match="position for every token"):
        ops.qk_norm_rope_write(step.ctx, qkv.repeat(2, 1), n_q, n_kv, d, None, None, 1e-6, None, 0, good)
