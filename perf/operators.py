"""Serving in fewer bits: a cache in 4 bits with the attention that reads it, and products in 8 bits.

A case names one operator and its sizes:

``append``   a step's rows [q heads | k heads | v heads]: per-head RMSNorm and rotation of q and k, keys and values into their pages
             in 4 bits; returns the rotated queries and the keys and values that the cache then holds.
``attend``   grouped-query attention of a step's queries over pages in 4 bits: decode rows, portions of prompts, both.
``product``  tokens rounded to 8 bits with a scale each, times a matrix in 8 bits with a scale for each row; into the run's type,
             onto a fp32 residual, or gate and up through SwiGLU.

4 bits: the elements of a head's row are cut into groups of at most 64; a group has a scale ``s`` and an offset ``z``, both
bfloat16: ``z`` the largest one not above the group's minimum, ``s`` the smallest one not below ``(max - z) / 15`` (0 where that is
no normal number), and an element's code is ``rint((x - z) / s)`` in 0 .. 15.  It stands for ``z + s * code``.
8 bits: ``s = max|x| / 127`` of the row, a code is ``rint(127 x / max|x|)``.
Codes are those of values in 64 bits: a value next to the border of two codes has the same code in every order of summing.

Every size is a user's: head counts, widths and lengths of the dense shapes of ``leone_b200.benchmark``, or generic.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
PAGE = 16                                  # the engine's default page


# -- the cases ------------------------------------------------------------------------------------------
def listed():
    return [
        # one conversation's next token: the smallest call, where only the latency counts
        {"name": "append-1", "do": "append", "dtype": "bf16", "requests": 1, "tokens": 1, "past": 700, "ragged": False, "n_q": 16,
         "n_kv": 8, "d": 128, "norm": True, "pairing": "half_split"},
        # a long prompt's keys and values go into the cache
        {"name": "append-2048", "do": "append", "dtype": "bf16", "requests": 1, "tokens": 2048, "past": 0, "ragged": False,
         "n_q": 32, "n_kv": 8, "d": 128, "norm": True, "pairing": "half_split"},
        # the 32-bit path, portions of three prompts behind what they cached before; smaller heads, adjacent pairs, no norm
        {"name": "append-3x111-fp32", "do": "append", "dtype": "fp32", "requests": 3, "tokens": 111, "past": 77, "ragged": True,
         "n_q": 12, "n_kv": 4, "d": 64, "norm": False, "pairing": "adjacent"},
        # one conversation's next token over a short context
        {"name": "decode-1x512", "do": "attend", "dtype": "bf16", "requests": 1, "tokens": 1, "past": 511, "decode": 0,
         "ragged": False, "n_q": 16, "n_kv": 8, "d": 128, "window": 0},
        # a busy server: 64 conversations with contexts of up to 2,048 tokens
        {"name": "decode-64-ragged", "do": "attend", "dtype": "bf16", "requests": 64, "tokens": 1, "past": 2047, "decode": 0,
         "ragged": True, "n_q": 32, "n_kv": 8, "d": 128, "window": 0},
        # one very long context: as many positions as the dense configurations have
        {"name": "decode-1x40960", "do": "attend", "dtype": "bf16", "requests": 1, "tokens": 1, "past": 40959, "decode": 0,
         "ragged": False, "n_q": 32, "n_kv": 8, "d": 128, "window": 0},
        # the fourth portion of a long prompt reads what the portions before it cached
        {"name": "prompt-2048-behind-6144", "do": "attend", "dtype": "bf16", "requests": 1, "tokens": 2048, "past": 6144,
         "decode": 0, "ragged": False, "n_q": 32, "n_kv": 8, "d": 128, "window": 0},
        # a server's mixed step with a sliding window: 17 decode rows and a portion of a prompt, seven query heads a cached one
        {"name": "mixed-17+333-window", "do": "attend", "dtype": "bf16", "requests": 1, "tokens": 333, "past": 1100, "decode": 17,
         "ragged": False, "n_q": 14, "n_kv": 2, "d": 64, "window": 500},
        # the smallest product: q, k and v of one token
        {"name": "product-1", "do": "product", "dtype": "bf16", "m": 1, "n": 4096, "k": 2048, "out": "run"},
        # gate and up of eight conversations that decode together
        {"name": "gated-8", "do": "product", "dtype": "bf16", "m": 8, "n": 24576, "k": 4096, "out": "gated"},
        # the way back onto the residual stream for a short prompt in the 32-bit path
        {"name": "residual-77-fp32", "do": "product", "dtype": "fp32", "m": 77, "n": 2048, "k": 6144, "out": "residual"},
        # gate and up of a long prompt
        {"name": "gated-2048", "do": "product", "dtype": "bf16", "m": 2048, "n": 24576, "k": 4096, "out": "gated"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    do = rng.choice(["append", "attend", "attend", "attend", "product", "product"])
    dtype = "fp32" if rng.random() < 0.2 else "bf16"
    if do == "product":
        k, n = 16 * _log(rng, 8, 768), 32 * _log(rng, 8, 768)
        out = rng.choice(["run", "gated", "residual"])
        return {"do": do, "dtype": dtype, "m": _log(rng, 1, 2048), "n": n, "k": k, "out": out}
    n_kv = rng.choice([1, 2, 4, 8])
    heads = {"n_q": n_kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "n_kv": n_kv, "d": rng.choice([64, 128, 128])}
    if do == "append":
        requests = _log(rng, 1, 16)
        return {"do": do, "dtype": dtype, "requests": requests, "tokens": _log(rng, 1, 2048 // requests), "past": _log(rng, 1, 4000) - 1,
                "ragged": rng.random() < 0.5, **heads, "norm": rng.random() < 0.7, "pairing": rng.choice(["half_split", "adjacent"])}
    window = rng.choice([0, 0, 0, _log(rng, 16, 2000)])
    kind = rng.choice(["decode", "decode", "prompt", "mixed"])
    if dtype == "fp32":                                      # what checks a model: short contexts
        return {"do": do, "dtype": dtype, "requests": _log(rng, 1, 4), "tokens": 1 if kind == "decode" else _log(rng, 2, 64),
                "past": _log(rng, 1, 500) - 1, "decode": 0, "ragged": True, **heads, "window": window}
    if kind == "decode":
        requests = _log(rng, 1, 64)
        return {"do": do, "dtype": dtype, "requests": requests, "tokens": 1, "past": _log(rng, 1, 128000 // requests) - 1, "decode": 0,
                "ragged": rng.random() < 0.5, **heads, "window": window}
    requests = _log(rng, 1, 4)
    return {"do": do, "dtype": dtype, "requests": requests, "tokens": _log(rng, 2, 2000 // requests), "past": _log(rng, 1, 4000) - 1,
            "decode": _log(rng, 1, 30) if kind == "mixed" else 0, "ragged": rng.random() < 0.5, **heads, "window": window}


def _lengths(case):
    """(new tokens, cached tokens) of every sequence; decode rows stand in front."""
    rng = random.Random(case["requests"] * 1000003 + case["tokens"] * 1009 + case["past"])
    few = lambda v, least: rng.randint(max(least, v // 32), v) if case["ragged"] and v > least else v  # noqa: E731
    lens = [(1, rng.randint(0, case["past"])) for _ in range(case.get("decode", 0))]
    return lens + [(few(case["tokens"], 1), few(case["past"], 0)) for _ in range(case["requests"])]


def _visible(case):
    """(pairs of a query and a key it sees, keys that some query of its sequence sees)."""
    pairs = keys = 0
    for new, past in _lengths(case):
        w = case["window"] or past + new
        pairs += sum(min(p + 1, w) for p in range(past, past + new))
        keys += min(past + new, w + new - 1)
    return pairs, keys


def work(case):
    item = 2 if case["dtype"] == "bf16" else 4
    if case["do"] == "product":
        m, n, k, out = case["m"], case["n"], case["k"], case["out"]
        wide = m * n * 8 if out == "residual" else m * (n // 2 if out == "gated" else n) * item
        return {"bytes": m * k * item + n * k + 4 * n + wide, "flops": 2 * m * n * k}
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    row = d // 2 + 4 * -(-d // 64)                             # bytes of a key or value in 4 bits
    tokens = sum(new for new, _ in _lengths(case))
    if case["do"] == "append":
        # rows in, queries out, 4-bit rows written, the values they stand for out, rotation
        return {"bytes": tokens * ((n_q + 2 * n_kv) * d * item + n_q * d * item + 2 * n_kv * (row + d * item) + 4 * d),
                "flops": tokens * (n_q + 2 * n_kv) * d * 10}
    pairs, keys = _visible(case)
    return {"bytes": 2 * keys * n_kv * row + 2 * tokens * n_q * d * item, "flops": 4 * pairs * n_q * d}


# -- 4 bits and 8 bits ----------------------------------------------------------------------------------
def _bf16_down(x):
    """The largest bfloat16 not above x (fp64), as fp64."""
    near = x.float()
    below = torch.where(near.double() > x, torch.nextafter(near, torch.full_like(near, -math.inf)), near)
    bits = below.view(torch.int32)
    low = bits & 0xFFFF
    return torch.where((low != 0) & (bits < 0), bits - low + 0x10000, bits - low).view(torch.float32).double()


def _quantize4(x):
    """fp64 [.., d] to (codes uint8 [.., d], s and z fp32 [.., groups])."""
    d = x.shape[-1]
    groups = -(-d // 64)
    x = x.unflatten(-1, (groups, d // groups))
    z = _bf16_down(x.amin(-1))
    s = -_bf16_down(-(x.amax(-1) - z) / torch.full_like(z, 15))        # (a tensor: the division by a number may be a product)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    steps = torch.where(s > 0, s, torch.full_like(s, math.inf))
    codes = torch.round((x - z[..., None]) / steps[..., None]).clamp(0, 15).to(torch.uint8)
    return codes.flatten(-2), s.float(), z.float()


def _values4(codes, s, z):
    """What the codes stand for, fp32 [.., d]."""
    c = codes.float().unflatten(-1, (s.shape[-1], codes.shape[-1] // s.shape[-1]))
    return (z[..., None] + s[..., None] * c).flatten(-2)


def _quantize8(x):
    """fp32 [rows, k] to (codes as fp32, s fp32 [rows, 1]); the quotient in 64 bits, whose border between two codes is where it is."""
    top = x.abs().amax(-1, keepdim=True)
    some = torch.where(top > 0, top, torch.full_like(top, math.inf)).double()
    return torch.round(x.double() * 127 / some).float(), top / torch.full_like(top, 127)


# -- inputs ---------------------------------------------------------------------------------------------
def _rows(gen, n, width, spread):
    """Activations: normal, with a few wide channels, as a model's stream has them."""
    x = torch.randn((n, width), generator=gen, device=DEVICE)
    wide = torch.rand(width, generator=gen, device=DEVICE) < 0.02
    return x * torch.where(wide, torch.full_like(x[0], spread), torch.ones_like(x[0]))


def _tables(lens, window, gen):
    """(block table int32 [sequences, columns], pages): shuffled pages; -1 behind a sequence and where a window has passed."""
    counts = [-(-(new + past) // PAGE) for new, past in lens]
    pages = sum(counts) + 3
    ids = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, (n, (new, past)) in enumerate(zip(counts, lens)):
        gone = max(0, past - window + 1) // PAGE if window else 0
        table[i, gone:n] = ids[at + gone:at + n]
        at += n
    return table, pages


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case, "dtype": dtype}
    if case["do"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        state["x"] = _rows(gen, m, k, 12.0).to(dtype)
        codes, scale = _quantize8(torch.randn((n, k), generator=gen, device=DEVICE) * 0.02)
        state["w"], state["w_scale"] = codes.to(torch.int8), scale[:, 0].contiguous()
        if case["out"] == "residual":
            state["residual"] = torch.randn((m, n), generator=gen, device=DEVICE) * 4
        if own:
            _own_product(state)
        return state
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    lens = _lengths(case)
    n = sum(new for new, _ in lens)
    longest = max(new + past for new, past in lens)
    table, pages = _tables(lens, case.get("window", 0), gen)
    new, past = (torch.tensor(v, device=DEVICE) for v in zip(*lens))
    state["seq"] = torch.repeat_interleave(torch.arange(len(lens), device=DEVICE), new)
    state["first"] = torch.cumsum(new, 0) - new
    state["pos"] = torch.arange(n, device=DEVICE) - state["first"][state["seq"]] + past[state["seq"]]
    state["table"], state["lens"], state["new_most"] = table, lens, max(v for v, _ in lens)
    cols = (n_q + 2 * n_kv) * d
    state["rows"] = _rows(gen, n, cols, 6.0).to(dtype)
    if case["do"] == "append":
        freq = 1000000.0 ** (-torch.arange(d // 2, dtype=torch.float64, device=DEVICE) * 2 / d)
        angle = torch.arange(longest, dtype=torch.float64, device=DEVICE)[:, None] * freq
        state["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        state["q_norm"], state["k_norm"] = (1 + 0.1 * torch.randn((2, d), generator=gen, device=DEVICE)).unbind(0)
    else:
        # what earlier steps cached: keys after norm and rotation, with some wide channels, and values
        wide = torch.where(torch.rand(d, generator=gen, device=DEVICE) < 0.05, 3.0, 1.0)
        state["k"] = _quantize4(torch.randn((pages, n_kv, PAGE, d), generator=gen, device=DEVICE).double() * wide)
        state["v"] = _quantize4(torch.randn((pages, n_kv, PAGE, d), generator=gen, device=DEVICE).double())
    if own:
        _own_cached(state, pages)
    return state


# -- the plain form -------------------------------------------------------------------------------------
def _rotated(x, cos, sin, pairing):
    """x [n, heads, d]; cos, sin [n, 1, d / 2]."""
    if pairing == "half_split":
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _append(state):
    case, dtype = state["case"], state["dtype"]
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    q, k, v = state["rows"].double().unflatten(1, (n_q + 2 * n_kv, d)).split([n_q, n_kv, n_kv], 1)
    cos, sin = (t[:, None] for t in state["rope"][state["pos"]].double().unbind(-1))

    def normed(x, w):
        return x * w * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()

    if case["norm"]:
        q, k = normed(q, state["q_norm"]), normed(k, state["k_norm"])
    q, k = _rotated(q, cos, sin, case["pairing"]), _rotated(k, cos, sin, case["pairing"])
    return q.flatten(1).to(dtype), _values4(*_quantize4(k)).flatten(1).to(dtype), _values4(*_quantize4(v)).flatten(1).to(dtype)


def _attend(state):
    case, dtype = state["case"], state["dtype"]
    n_q, n_kv, d, window = case["n_q"], case["n_kv"], case["d"], case["window"]
    seq, pos, first = state["seq"], state["pos"], state["first"]
    b, most = len(state["lens"]), state["new_most"]
    row = torch.arange(pos.numel(), device=DEVICE) - first[seq]
    q = torch.zeros((b, most, n_q, d), device=DEVICE)
    q[seq, row] = state["rows"][:, :n_q * d].float().unflatten(1, (n_q, d))
    at = torch.full((b, most), -1, device=DEVICE)
    at[seq, row] = pos
    pages = state["table"].clamp(min=0).long()
    # [sequences, cached heads, keys, d]
    k, v = (_values4(*(t[pages] for t in state[x])).transpose(1, 2).flatten(2, 3) for x in "kv")
    q = q.unflatten(2, (n_kv, n_q // n_kv)).permute(0, 2, 3, 1, 4).flatten(2, 3)               # [b, n_kv, g * most, d]
    score = (q @ k.transpose(2, 3)).unflatten(2, (n_q // n_kv, most)) * d ** -0.5
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = key <= at[..., None]
    if window:
        seen &= key > at[..., None] - window
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = (weight.flatten(2, 3) @ v).unflatten(2, (n_q // n_kv, most)).permute(0, 3, 1, 2, 4)  # [b, most, n_kv, g, d]
    return out[seq, row].flatten(1).to(dtype)


def _product(state):
    case, dtype = state["case"], state["dtype"]
    codes, scale = _quantize8(state["x"].float())
    y = codes @ state["w"].float().T * scale * state["w_scale"]
    if case["out"] == "residual":
        return y + state["residual"]
    if case["out"] == "gated":
        gate, up = y.chunk(2, 1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(dtype)


# -- the framework's calls ------------------------------------------------------------------------------
_OPS = {}


def _ops(dtype):
    if dtype not in _OPS:
        from leone_b200.ops.cuda import CudaOps
        _OPS[dtype] = CudaOps(DEVICE, dtype)
    return _OPS[dtype]


def _own_product(state):
    """The matrix as a program keeps it, and where the result goes."""
    case, ops = state["case"], _ops(state["dtype"])
    w, scale = state["w"], state["w_scale"]
    if case["out"] == "gated":
        half = case["n"] // 2
        state["matrix"] = ops.prepare_gate_up_int8(w[:half], scale[:half], w[half:], scale[half:])
    else:
        state["matrix"] = ops.prepare_matrix_int8(w, scale)
    cols = case["n"] // 2 if case["out"] == "gated" else case["n"]
    state["out"] = torch.empty((case["m"], cols), dtype=torch.float32 if case["out"] == "residual" else state["dtype"], device=DEVICE)


def _own_cached(state, pages):
    """A step's context and its pages in 4 bits."""
    import numpy as np
    from leone_b200.cache.packed import pack_pages, row_bytes
    from leone_b200.engine.batch import StepContext
    from leone_b200.parts.base import PagedCacheView
    case = state["case"]
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    new, past = (np.array(v) for v in zip(*state["lens"]))
    ctx = StepContext()
    ctx.n_tokens, ctx.n_seqs = int(new.sum()), len(new)
    ctx.q_lens, ctx.starts, ctx.ctx_lens = new, past, new + past
    ctx.max_q_len, ctx.max_ctx_len, ctx.decode_only = int(new.max()), int(ctx.ctx_lens.max()), bool(new.max() == 1)
    ints = lambda t: torch.as_tensor(t, dtype=torch.int32, device=DEVICE)  # noqa: E731
    ctx.positions, ctx.seq_of_token = ints(state["pos"]), ints(state["seq"])
    ctx.q_start, ctx.ctx_len = ints(np.concatenate([[0], np.cumsum(new)])), ints(ctx.ctx_lens)
    ctx.status = torch.zeros(4, dtype=torch.int32, device=DEVICE)
    if case["do"] == "append":
        pools = [torch.zeros((pages, n_kv, PAGE, row_bytes(d)), dtype=torch.uint8, device=DEVICE) for _ in range(2)]
        state["work"] = torch.empty_like(state["rows"])
        state["held"] = torch.empty((2, ctx.n_tokens, n_kv * d), dtype=state["dtype"], device=DEVICE)
    else:
        pools = [pack_pages(*state["k"], values=False), pack_pages(*state["v"], values=True)]
        state["out"] = torch.empty((ctx.n_tokens, n_q * d), dtype=state["dtype"], device=DEVICE)
    state["ctx"], state["cache"] = ctx, PagedCacheView(*pools, state["table"], PAGE, bits=4)


def _own_run(state):
    case, ops = state["case"], _ops(state["dtype"])
    if case["do"] == "product":
        if case["out"] == "gated":
            ops.linear_swiglu(state["x"], state["matrix"], state["out"])
        else:
            ops.linear(state["x"], state["matrix"], state["out"], residual=state.get("residual"))
        return state["out"]
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    ctx, cache = state["ctx"], state["cache"]
    if case["do"] == "attend":
        ops.attention(ctx, state["rows"], state["out"], n_q, n_kv, d, d ** -0.5, case["window"] or None, cache)
        return state["out"]
    rows = state["work"].copy_(state["rows"])                # queries are normed and rotated in place
    norm = (state["q_norm"], state["k_norm"]) if case["norm"] else (None, None)
    ops.qk_norm_rope_write(ctx, rows, n_q, n_kv, d, *norm, 1e-6, state["rope"], d, cache, pairing=case["pairing"])
    k, v = state["held"]
    ops.read_packed_rows(ctx, cache, n_kv, d, k, v)
    return rows[:, :n_q * d], k, v


def run(state):
    if own:
        return _own_run(state)
    return {"append": _append, "attend": _attend, "product": _product}[state["case"]["do"]](state)


# -- in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["do"] == "product":
        x = state["x"].double()
        top = x.abs().max(1, keepdim=True).values
        codes = (x * 127 / top.clamp(min=1e-300)).round()
        y = (codes @ state["w"].double().T) * (top / 127) * state["w_scale"].double()
        if case["out"] == "residual":
            return y + state["residual"].double()
        if case["out"] == "gated":
            half = case["n"] // 2
            return torch.nn.functional.silu(y[:, :half]) * y[:, half:]
        return y
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    rows = state["rows"].double().view(-1, n_q + 2 * n_kv, d)
    if case["do"] == "append":
        parts = list(rows.split([n_q, n_kv, n_kv], 1))
        for i, w in ((0, state["q_norm"]), (1, state["k_norm"])):
            x = parts[i]
            if case["norm"]:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * w.double()
            turn = torch.view_as_complex(state["rope"].double())[state["pos"]][:, None]
            if case["pairing"] == "half_split":
                y = torch.complex(x[..., :d // 2], x[..., d // 2:]) * turn
                parts[i] = torch.cat([y.real, y.imag], -1)
            else:
                parts[i] = torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)

        def held(x):
            g = x.unflatten(-1, (-(-d // 64), -1))
            lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
            m, e = torch.frexp(lo)                                # 8 significant bits, down and up
            z = torch.ldexp((m * 256).floor(), e - 8)
            m, e = torch.frexp((hi - z) / 15)
            s = torch.ldexp((m * 256).ceil(), e - 8)
            return (z + s * ((g - z) / s.clamp(min=1e-300)).round().clamp(0, 15)).flatten(1)

        return parts[0].flatten(1), held(parts[1]), held(parts[2])
    out = torch.empty((rows.shape[0], n_q, d), dtype=torch.float64, device=DEVICE)
    at = 0
    for i, (new, past) in enumerate(state["lens"]):
        ctx = new + past
        pages = state["table"][i, :-(-ctx // PAGE)].clamp(min=0).long()
        p = torch.arange(past, ctx, device=DEVICE)[:, None]
        j = torch.arange(ctx, device=DEVICE)[None]
        seen = (j <= p) & (p - j < (case["window"] or ctx))
        for h in range(n_kv):
            def held(codes, s, z):
                c, s, z = (t[pages, h].flatten(0, 1)[:ctx].double() for t in (codes, s, z))
                return z.repeat_interleave(d // z.shape[1], 1) + c * s.repeat_interleave(d // s.shape[1], 1)
            k, v = held(*state["k"]), held(*state["v"])
            for q_head in range(h * (n_q // n_kv), (h + 1) * (n_q // n_kv)):
                score = rows[at:at + new, q_head] @ k.T / math.sqrt(d)
                out[at:at + new, q_head] = torch.softmax(score.masked_fill(~seen, -math.inf), 1) @ v
        at += new
    return out.flatten(1)
