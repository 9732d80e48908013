"""Pages in 4 bits: what the kernels do at the edges of what they take, against plain 64-bit forms."""
import pytest
import torch

from leone_b200.cache import packed
from leone_b200.parts.rotary import build_rotary_table
from tests.fewer_bits import Step, attention64, quantize4, values4

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


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype,d,n_q,n_kv,new", [
    (BF16, 128, 16, 8, 5),         # few tokens: blocks of 8 heads
    (FP32, 64, 2, 3, 7),           # an odd number of cached heads, a block of all kinds
    (BF16, 128, 32, 8, 700),       # many tokens: a block of all of a token's heads
    (FP32, 128, 1, 1, 900),
    (BF16, 64, 40, 20, 600),       # two blocks a token, the second of keys and values
    (BF16, 96, 4, 2, 9),           # the form of any size
])
def test_append_behind_the_rotation_table(ops_of, dtype, d, n_q, n_kv, new, norm):
    """Tokens whose position the rotation table does not reach, on pages that they have: the status says so, their queries and keys
    stay as they were, their values are written, and nothing beside them."""
    ops = ops_of(dtype)
    past, reach = 30, 30 + new // 2                          # half of the tokens lie behind the table
    step = Step([(new, past)], 16, DEV, seed=d)
    rows = torch.randn((new, (n_q + 2 * n_kv) * d), generator=_gen(d + new), device=DEV).to(dtype)
    weights = (1 + 0.1 * torch.randn((2, d), generator=_gen(2), device=DEV)) if norm else (None, None)
    guard = 3                                                # pages in front of the pools and behind them
    whole = [torch.full((step.pages + 2 * guard, n_kv, 16, packed.row_bytes(d)), 0xA5, dtype=torch.uint8, device=DEV) for _ in range(2)]
    pools = [w[guard:guard + step.pages] for w in whole]
    table = build_rotary_table(reach, d, 10000.0).to(DEV)
    got, full = rows.clone(), rows.clone()
    ops.qk_norm_rope_write(step.ctx, got, n_q, n_kv, d, *weights, 1e-6, table, d, step.view(*pools))
    assert step.ctx.status[0] == 3 and int(step.ctx.status[1]) >= new // 2
    step.ctx.status.zero_()
    want = [torch.full_like(w, 0xA5) for w in whole]
    longer = build_rotary_table(past + new, d, 10000.0).to(DEV)
    ops.qk_norm_rope_write(step.ctx, full, n_q, n_kv, d, *weights, 1e-6, longer, d, step.view(*(w[guard:guard + step.pages] for w in want)))
    assert step.ctx.status[0] == 0
    inside = step.pos < reach
    assert torch.equal(got[inside], full[inside]) and torch.equal(got[~inside], rows[~inside])
    for have, w, values in zip(whole, want, (False, True)):
        assert (have[:guard] == 0xA5).all() and (have[-guard:] == 0xA5).all()
        fill = packed.unpack_pages(torch.full_like(pools[0], 0xA5), d, values)
        for a, b, untouched in zip(*(packed.unpack_pages(t[guard:guard + step.pages], d, values) for t in (have, w)), fill):
            a, b, untouched = a.float(), b.float(), untouched.float()
            if not values:
                b[step.page[~inside], :, step.slot[~inside]] = untouched[step.page[~inside], :, step.slot[~inside]]
            assert torch.equal(a, b)
    # and they are the right ones
    v = rows.double().unflatten(1, (n_q + 2 * n_kv, d))[:, n_q + n_kv:]
    codes, s, z = (t[step.page, :, step.slot] for t in packed.unpack_pages(pools[1], d, True))
    for a, b in zip((codes.long(), s.double(), z.double()), quantize4(v)):
        assert torch.equal(a, b)


def _nan_pattern(ops, n_q, n_kv, d, lens, window, bad, runs=1, splits=0):
    """Prompt attention over pages whose last cached head has NaN in the last group of the values `bad` [(sequence, key)]: the outputs'
    NaN, and which of them there have to be, ``[tokens, n_q, d]``."""
    step = Step(lens, 16, DEV, window=window)
    pools = []
    for values in (False, True):
        codes, s, z = quantize4(torch.randn((step.pages, n_kv, 16, d), generator=_gen(7 + values), device=DEV).double())
        for seq, key in bad if values else ():
            page = int(step.table[seq, key // 16])
            if page >= 0:
                s[page, -1, key % 16, -1] = z[page, -1, key % 16, -1] = float("nan")
        pools.append(packed.pack_pages(codes, s, z, values))
    n = step.ctx.n_tokens
    qkv = torch.randn((n, (n_q + 2 * n_kv) * d), generator=_gen(9), device=DEV).to(BF16)
    got = []
    ops.force_prompt4_splits = splits
    try:
        for _ in range(runs):
            out = torch.zeros((n, n_q * d), dtype=BF16, device=DEV)
            ops.attention(step.ctx, qkv, out, n_q, n_kv, d, d ** -0.5, window or None, step.view(*pools))
            got.append(out.view(n, n_q, d).isnan())
    finally:
        ops.force_prompt4_splits = 0
    assert step.ctx.status.tolist() == [0, 0, 0, 0]
    sees = torch.zeros(n, dtype=torch.bool, device=DEV)
    for seq, key in bad:
        sees |= (step.seq == seq) & (step.pos >= key) & ((step.pos < key + window) if window else True)
    want = torch.zeros((n, n_q, d), dtype=torch.bool, device=DEV)
    want[:, n_q - n_q // n_kv:, max(0, d - 64):] = sees[:, None, None]
    return got, want


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_values_on_both_sides_of_a_window(ops_of, d, splits):
    """A block of 128 tokens whose first 40 and last 40 keys have NaN, more than it lists: rows whose window lies between see none."""
    bad = [(0, 64 + 128 * block + i) for block in range(2) for i in (*range(40), *range(88, 128))]
    got, want = _nan_pattern(ops_of(BF16), 2, 2, d, [(256, 64)], 16, bad, splits=splits)
    assert torch.equal(got[0], want)
    assert want[:40, 1].any(-1).all() and not want[56:88].any()


@pytest.mark.parametrize("d", [64, 128])
def test_nan_values_that_only_the_second_query_tile_sees(ops_of, d):
    """Blocks of two query tiles of 32 tokens, the second of which reads a tile of keys that the first does not: NaN in that tile, many
    of them or one, is not the first's."""
    lens = [(640, 20)] * 3 + [(500, 52)]                      # 68 query tiles of 32 tokens, for each of 8 cached heads
    for behind in ([129, 130, 180, 250], range(128, 256)):
        bad = [(seq, key + 128 * tile) for seq in range(4) for tile in (0, 2) for key in behind]
        got, want = _nan_pattern(ops_of(BF16), 32, 8, d, lens, 0, bad, runs=5)
        assert want.any() and not want.all()
        for g in got:
            assert torch.equal(g, want)


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["key", "channel"])
@pytest.mark.parametrize("power", [10, 16, 20])
def test_prompt_of_keys_of_unlike_size(ops_of, power, kind, d, splits):
    """One key, or one channel of every key, 2^10 and more times the rest: rows that do not see the key lose nothing by it, and the small
    channels count as they did.

    An output's roundings: its own to bfloat16 and its values' (an element each, off by 2^-7 / 12^(1/2) of the number's power of two,
    0.0016 of the numbers of a row by their squares), and the weights': the same again for many keys, at most 2^-8 of every element
    alike where one key has all the weight.  Keys are fp16: 2^-11 at most of a score's products, which are random, about 0.0003 for
    scores of a size of one.  So 0.0028 of a call's outputs and 2^-8 + 2^(1/2) 0.0016, a fourth more for the chance of 64 elements, of a row's."""
    ops = ops_of(BF16)
    n_q, n_kv, lens, large = 4, 2, [(200, 100), (60, 300)], [(0, 255), (1, 305)]
    step = Step(lens, 16, DEV, seed=power)
    x = [torch.randn((step.pages, n_kv, 16, d), generator=_gen(power + i), device=DEV).double() for i in range(2)]
    n = step.ctx.n_tokens
    qkv = torch.randn((n, (n_q + 2 * n_kv) * d), generator=_gen(5), device=DEV)
    if kind == "key":
        for seq, key in large:
            x[0][int(step.table[seq, key // 16]), :, key % 16] *= 2.0 ** power
    else:
        x[0][..., 5] = x[0][..., 5].abs() * 2.0 ** power
        qkv[:, 5:n_q * d:d] *= 2.0 ** -power
    qkv = qkv.to(BF16)
    pools, plain = [], []
    for t, values in zip(x, (False, True)):
        coded = quantize4(t)
        pools.append(packed.pack_pages(*coded, values))
        plain.append(values4(*coded))
    out = torch.zeros((n, n_q * d), dtype=BF16, device=DEV)
    ops.force_prompt4_splits = splits
    try:
        ops.attention(step.ctx, qkv, out, n_q, n_kv, d, d ** -0.5, None, step.view(*pools))
    finally:
        ops.force_prompt4_splits = 0
    q = qkv[:, :n_q * d].double().unflatten(1, (n_q, d))
    want, *_ = attention64(q, *plain, lens, step.table, 16, d ** -0.5, 0)
    off = (out.double().view_as(want) - want).square()
    counts = torch.ones((n, n_q), dtype=torch.bool, device=DEV)
    if kind == "key":
        # rows whose score with the large key is not far from the others' turn on its last bits
        for seq, key in large:
            k = plain[0][int(step.table[seq, key // 16]), :, key % 16].repeat_interleave(n_q // n_kv, 0)
            score = (q * k).sum(-1) * d ** -0.5
            counts &= ~((step.seq == seq) & (step.pos >= key))[:, None] | (score.abs() > 40)
        assert counts[:155].all() and counts.float().mean() > 0.9
    off, size = off[counts], want.square()[counts]
    assert (off.sum() / size.sum()).sqrt() < 1.25 * 3 ** 0.5 * 0.0016
    assert (off.sum(-1) / size.sum(-1)).sqrt().max() < 2.0 ** -8 + 1.25 * 2 ** 0.5 * 0.0016
    assert step.ctx.status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("spread", [1e-6, 2e-5, 1e-4, 1e-3])
@pytest.mark.parametrize("dtype,d,n_kv,tokens", [(FP32, 64, 2, 3000), (FP32, 128, 2, 3000), (FP32, 64, 8, 20), (BF16, 128, 4, 1500)])
def test_append_of_keys_that_are_nearly_equal(ops_of, dtype, d, n_kv, tokens, spread):
    """Groups of normed keys whose spread is small against their size: their rounding to 32 bits is a good part of a step, and codes are
    those of 64 bits all the same."""
    ops = ops_of(dtype)
    step = Step([(tokens, 3)], 16, DEV)
    x = 1 + torch.rand((tokens, 1 + 2 * n_kv, d), generator=_gen(tokens), device=DEV) * spread
    # the least of a normed head lies just above 1.5, a number of bfloat16
    weights = torch.full((2, d), 1.5 * (1 + 0.7 * spread), device=DEV)
    if dtype == BF16:                                        # equal elements, and weights that are not
        x = torch.randn((tokens, 1 + 2 * n_kv, 1), generator=_gen(1), device=DEV).expand_as(x).abs() + 0.1
        weights = 1.5 * (1 + 0.2 * spread + 2.0 ** -20 + torch.rand((2, d), generator=_gen(2), device=DEV) * spread)
    rows = x.to(dtype).flatten(1)
    pools = [torch.zeros((step.pages, n_kv, 16, packed.row_bytes(d)), dtype=torch.uint8, device=DEV) for _ in range(2)]
    eps = 2.0 ** -30
    ops.qk_norm_rope_write(step.ctx, rows.clone(), 1, n_kv, d, weights[0], weights[1], eps, None, 0, step.view(*pools))
    k = rows.double().unflatten(1, (1 + 2 * n_kv, d))[:, 1:1 + n_kv]
    k = k * weights[1].double() * torch.rsqrt(k.square().mean(-1, keepdim=True) + eps)
    have = [t[step.page, :, step.slot] for t in packed.unpack_pages(pools[0], d, False)]
    codes, s, z = quantize4(k)
    assert torch.equal(have[1].double(), s) and torch.equal(have[2].double(), z)
    assert torch.equal(have[0].long(), codes)
    assert (s.amax() < 2 * spread) and len(codes.unique()) >= 8 and step.ctx.status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("dtype,d,n_q,n_kv", [(BF16, 128, 32, 8), (FP32, 128, 4, 8), (BF16, 96, 16, 8)])
def test_pages_behind_4_gib(ops_of, dtype, d, n_q, n_kv):
    """Pools of more than 2^32 bytes: append, read, decode rows and portions on their last pages, bit for bit as in small pools."""
    ops = ops_of(dtype)
    n_q = max(n_q, n_kv)
    lens = [(1, 300), (1, 20), (70, 200)]
    step = Step(lens, 16, DEV, seed=4)
    pages = (1 << 32) // (n_kv * 16 * packed.row_bytes(d)) + 1 + step.pages
    far = Step(lens, 16, DEV, seed=4)
    far.table = torch.where(step.table >= 0, step.table + (pages - step.pages), step.table)
    small = [packed.pack_pages(*quantize4(torch.randn((step.pages, n_kv, 16, d), generator=_gen(i), device=DEV).double()), bool(i)) for i in range(2)]
    large = [torch.zeros((pages, *t.shape[1:]), dtype=torch.uint8, device=DEV) for t in small]
    assert large[0].numel() > 1 << 32
    for a, b in zip(large, small):
        a[-step.pages:] = b
    n = step.ctx.n_tokens
    rows = torch.randn((n, (n_q + 2 * n_kv) * d), generator=_gen(9), device=DEV).to(dtype)
    table = build_rotary_table(400, d, 10000.0).to(DEV)
    results = []
    for s, pools in ((step, small), (far, large)):
        qkv, view = rows.clone(), s.view(*pools)
        ops.qk_norm_rope_write(s.ctx, qkv, n_q, n_kv, d, None, None, 1e-6, table, d, view)
        held = torch.zeros((2, n, n_kv * d), dtype=dtype, device=DEV)
        ops.read_packed_rows(s.ctx, view, n_kv, d, *held)
        out = torch.zeros((n, n_q * d), dtype=dtype, device=DEV)
        ops.attention(s.ctx, qkv, out, n_q, n_kv, d, d ** -0.5, None, view)
        assert s.ctx.status.tolist() == [0, 0, 0, 0]
        results.append((qkv, held, out, *(p[-step.pages:] for p in pools)))
    for a, b in zip(*results):
        assert torch.equal(a, b) and a.any()
    assert not large[0][:1000].any() and not large[1][:1000].any()


@pytest.mark.parametrize("splits", [1, 4, 8, 33])
@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (128, 20)])
def test_decode_rows_without_a_key(ops_of, d, window, splits):
    """Rows of a step that stand for no sequence (no keys, no pages) become zeros and report nothing; the others are as they were."""
    ops = ops_of(BF16)
    n_q, n_kv, lens = 6, 2, [(1, 200), (1, 10), (1, 90), (1, 33)]
    step = Step(lens, 16, DEV, seed=2, window=window)
    pools = [packed.pack_pages(*quantize4(torch.randn((step.pages, n_kv, 16, d), generator=_gen(i), device=DEV).double()), bool(i)) for i in range(2)]
    qkv = torch.randn((4, (n_q + 2 * n_kv) * d), generator=_gen(5), device=DEV).to(BF16)
    outs = []
    ops.force_decode4_splits = splits
    try:
        for empty in ((), (1, 3)):
            for i in empty:
                step.ctx.ctx_len[i], step.table[i] = 0, -1
            out = torch.full((4, n_q * d), 7.0, dtype=BF16, device=DEV)
            ops.attention(step.ctx, qkv, out, n_q, n_kv, d, d ** -0.5, window or None, step.view(*pools))
            outs.append(out)
    finally:
        ops.force_decode4_splits = 0
    assert torch.equal(outs[0][::2], outs[1][::2]) and not outs[1][1::2].any() and outs[0][1::2].any()
    assert step.ctx.status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (FP32, 64)])
def test_sequences_without_a_token(ops_of, dtype, d):
    """Sequences that bring no token to a step of portions: the others' outputs are as without them."""
    ops = ops_of(dtype)
    n_q, n_kv = 4, 2
    results = []
    for lens in ([(40, 100), (3, 20)], [(40, 100), (0, 60), (3, 20), (0, 5)]):
        step = Step(lens, 16, DEV, seed=3)
        # the same pages' contents for the same sequences, by their place in the table
        whole = [torch.randn((2, 12, n_kv, 16, d), generator=_gen(7 + i), device=DEV).double() for i in range(2)]
        pools = []
        for values, x in zip((False, True), whole):
            t = torch.zeros((step.pages, n_kv, 16, d), dtype=torch.float64, device=DEV)
            for which, seq in enumerate([i for i, (new, _) in enumerate(lens) if new]):
                pages = step.table[seq][step.table[seq] >= 0].long()
                t[pages] = x[which, :len(pages)]
            pools.append(packed.pack_pages(*quantize4(t), values))
        qkv = torch.randn((43, (n_q + 2 * n_kv) * d), generator=_gen(5), device=DEV).to(dtype)
        out = torch.full((43, n_q * d), 7.0, dtype=dtype, device=DEV)
        ops.force_prompt4_splits = ops.force_any4_splits = 1
        try:
            ops.attention(step.ctx, qkv, out, n_q, n_kv, d, d ** -0.5, None, step.view(*pools))
        finally:
            ops.force_prompt4_splits = ops.force_any4_splits = 0
        assert step.ctx.status.tolist() == [0, 0, 0, 0]
        results.append(out)
    assert torch.equal(*results) and not (results[0] == 7.0).all()
