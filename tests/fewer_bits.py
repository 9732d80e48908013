"""Plain 64-bit forms of pages in 4 bits and rows in 8 bits, and a step's context for the kernels' tests."""
import math

import numpy as np
import torch


def bf16_floor(x):
    """The largest bfloat16 not above x (fp64), in fp64: 8 significant bits, none below 2^-133."""
    bits = x.view(torch.int64)
    low = bits & ((1 << 45) - 1)
    normal = torch.where((low != 0) & (bits < 0), bits - low + (1 << 45), bits - low).view(torch.float64)
    small = torch.floor(x * 2.0 ** 133) * 2.0 ** -133
    return torch.where(torch.isfinite(x), torch.where(x.abs() < 2.0 ** -126, small, normal), x)


def quantize4(x):
    """fp64 [.., d] -> codes (int64), s, z (fp64 [.., groups]); groups with a NaN or an infinity: codes 0, s = z = NaN."""
    d = x.shape[-1]
    groups = -(-d // 64)
    x = x.unflatten(-1, (groups, d // groups))
    fine = torch.isfinite(x).all(-1)
    y = torch.where(fine[..., None], x, torch.zeros_like(x))
    z = bf16_floor(y.amin(-1))
    s = -bf16_floor(-(y.amax(-1) - z) / torch.full_like(z, 15))
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    fine &= (s <= 3.3895e38) & (z >= -3.3895e38)
    codes = torch.round((y - z[..., None]) / torch.where(s > 0, s, torch.full_like(s, math.inf))[..., None]).clamp(0, 15)
    codes = torch.where(fine[..., None], codes, torch.zeros_like(codes))
    nan = torch.full_like(s, math.nan)
    return codes.flatten(-2).long(), torch.where(fine, s, nan), torch.where(fine, z, nan)


def values4(codes, s, z):
    c = codes.double().unflatten(-1, (s.shape[-1], codes.shape[-1] // s.shape[-1]))
    return (z.double()[..., None] + s.double()[..., None] * c).flatten(-2)


def quantize8(x):
    """fp64 [rows, k] -> (codes, s [rows, 1])"""
    top = x.abs().amax(-1, keepdim=True)
    q = torch.round(x * 127 / torch.where(top > 0, top, torch.ones_like(top)))
    return q, top / 127


def rotate(x, pos, theta, pairing, rot):
    """x [n, heads, d] in fp64; the table's cos and sin are fp32."""
    freq = theta ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device=x.device) / rot)
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos().float().double()[:, None], angle.sin().float().double()[:, None]
    out = x.clone()
    if pairing == "half_split":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return out


class Step:
    """A step of sequences of ``lens = [(new, cached), ..]`` tokens over shuffled pages; ``spare`` pages belong to nobody."""

    def __init__(self, lens, page_tokens, device, seed=0, window=0, spare=2):
        from leone_b200.engine.batch import StepContext
        rng = np.random.default_rng(seed)
        new, past = (np.array(v) for v in zip(*lens))
        counts = [-(-(a + b) // page_tokens) for a, b in lens]
        self.pages, self.page_tokens, self.lens = sum(counts) + spare, page_tokens, lens
        ids = rng.permutation(self.pages)
        table = np.full((len(lens), max(counts) + 1), -1, dtype=np.int32)
        at = 0
        for i, n in enumerate(counts):
            gone = max(0, lens[i][1] - window + 1) // page_tokens if window else 0
            table[i, gone:n] = ids[at + gone:at + n]
            at += n
        c = self.ctx = StepContext()
        c.n_tokens, c.n_seqs = int(new.sum()), len(lens)
        c.q_lens, c.starts, c.ctx_lens = new, past, new + past
        c.max_q_len, c.max_ctx_len, c.decode_only = int(new.max()), int(c.ctx_lens.max()), bool(new.max() == 1)
        seq = np.repeat(np.arange(len(lens)), new)
        first = np.cumsum(new) - new
        pos = np.arange(new.sum()) - first[seq] + past[seq]
        ints = lambda t: torch.tensor(np.asarray(t), dtype=torch.int32, device=device)  # noqa: E731
        c.positions, c.seq_of_token = ints(pos), ints(seq)
        c.q_start, c.ctx_len = ints(np.concatenate([[0], np.cumsum(new)])), ints(c.ctx_lens)
        c.status = torch.zeros(4, dtype=torch.int32, device=device)
        self.table, self.pos, self.seq, self.first = ints(table), torch.tensor(pos, device=device), torch.tensor(seq, device=device), first
        # the page and slot of every token of the step
        self.page = self.table[self.seq, self.pos // page_tokens].long()
        self.slot = self.pos % page_tokens

    def view(self, k_pool, v_pool, **kw):
        from leone_b200.parts.base import PagedCacheView
        return PagedCacheView(k_pool, v_pool, self.table, self.page_tokens, bits=4, **kw)


def attention64(q, keys, vals, lens, table, page_tokens, scale, window):
    """q [n, n_q, d]; keys, vals [pages, n_kv, page_tokens, d], all fp64.  Returns the output and, per row, the largest absolute
    score before the softmax's shift and the largest absolute value, for bounds."""
    n, n_q, d = q.shape
    n_kv = keys.shape[1]
    out, top_s, top_v = torch.empty_like(q), torch.empty(n, n_q, device=q.device), torch.empty(n, n_q, device=q.device)
    at = 0
    for i, (new, past) in enumerate(lens):
        ctx = new + past
        pages = table[i, :-(-ctx // page_tokens)].long().clamp(min=0)
        p = torch.arange(past, ctx, device=q.device)[:, None]
        j = torch.arange(ctx, device=q.device)[None]
        seen = (j <= p) & ((p - j < window) if window else (j >= 0))
        lo = int((past - window + 1)) if window and past - window + 1 > 0 else 0
        for h in range(n_q):
            kv = h // (n_q // n_kv)
            k = keys[pages, kv].flatten(0, 1)[:ctx]
            v = vals[pages, kv].flatten(0, 1)[:ctx].clone()
            v[:lo] = 0                                      # rows that no query of this portion sees
            s = (q[at:at + new, h] @ k.T) * scale
            s = torch.where(seen, s, torch.full_like(s, -math.inf))
            out[at:at + new, h] = torch.softmax(s, 1) @ v
            top_s[at:at + new, h] = torch.where(seen, (q[at:at + new, h].abs() @ k.abs().T) * scale, torch.zeros_like(s)).amax(1).float()
            top_v[at:at + new, h] = v.abs().amax().float()
        at += new
    return out, top_s, top_v
