"""Pages that hold keys and values in 4 bits: their sizes, and their contents in plain tensors.

The kernels' definition is ``csrc/cache4.cuh``: the elements of a head's row in groups of at most 64, a scale ``s`` and an offset
``z`` (bfloat16) for each group, a code 0 .. 15 for each element, which stands for ``z + s * code``.  The reference caches f16 rows
only (crates/leone/src/kv.rs:14-31).  A pool is ``uint8 [pages, cached heads, page_tokens, row_bytes(d)]`` with pages of a multiple of
:data:`UNIT` tokens.  :func:`pack_pages` and :func:`unpack_pages` go between pools and plain codes, for what writes or reads pages
outside a step (tests, a request's pages from elsewhere).
"""
from __future__ import annotations

import torch

UNIT = 16          # tokens whose rows lie together; pages are multiples of it
MAX_DIM = 512


def attention_workspace(d: int) -> int:
    """Bytes that the parts of split attention over such pages take at most: of a step 148 tiles of 128 rows of prompt portions, three blocks
    an SM of up to 16 rows of decode, or 2,048 blocks of 8 rows of the kernel of any size; and the latter two twice more, for the
    captured decode steps and for the stream on which they are captured."""
    decode = 3 * 148 * 16 * 130 + 2048 * 8 * (d + 2)
    return 4 * (148 * 128 * 130 + 3 * decode)


def groups(d: int) -> int:
    """Groups of a head's row of ``d`` elements."""
    return -(-d // 64)


def row_bytes(d: int) -> int:
    """Bytes of a key's or value's row of ``d`` elements."""
    return d // 2 + 4 * groups(d)


def dim_ok(d: int) -> bool:
    """Whether rows of ``d`` elements can be held: every group a whole number of 8 elements."""
    return 0 < d <= MAX_DIM and d % (8 * groups(d)) == 0


def _places(d: int, values: bool) -> torch.Tensor:
    """``[UNIT, d / 8]``: the place in a unit (in 32-bit words) of every token's words."""
    g, words = groups(d), d // 8
    w = torch.arange(words)
    row = torch.arange(UNIT)
    place = w
    if values:
        row = (row & 8) | ((row & 7) >> 1) | ((row & 1) << 2)
    if d == 64 * g:
        group, i = w // 8, w % 8
        place = i * g + group if values else (i // 2) * 2 * g + 2 * group + i % 2
    place = place[None].expand(UNIT, words)
    if values and d == 64 * g and g == 2:
        place = place ^ (((row >> 1) & 1) << 3)[:, None]
    return row[:, None] * words + place


def _check_pool(page_tokens: int, d: int) -> None:
    if not dim_ok(d):
        raise ValueError(f"rows of {d} elements cannot be held in 4 bits: groups of at most 64 must be multiples of 8")
    if page_tokens <= 0 or page_tokens % UNIT:
        raise ValueError(f"pages in 4 bits hold a multiple of {UNIT} tokens, not {page_tokens}")


def pack_pages(codes: torch.Tensor, s: torch.Tensor, z: torch.Tensor, values: bool) -> torch.Tensor:
    """A pool of codes (uint8 ``[pages, heads, page_tokens, d]``, 0 .. 15) and their groups' scales and offsets
    (``[pages, heads, page_tokens, groups]``, bfloat16 numbers in any type); ``values``: the layout of the value pool."""
    pages, heads, tokens, d = codes.shape
    _check_pool(tokens, d)
    g, units = groups(d), tokens // UNIT
    if s.shape != (pages, heads, tokens, g) or z.shape != s.shape:
        raise ValueError(f"scales and offsets must be {(pages, heads, tokens, g)}")
    c = codes.to(torch.int32).unflatten(-1, (d // 8, 4, 2))                      # element 2 j in nibble j, 2 j + 1 in nibble j + 4
    shifts = 4 * torch.arange(4, dtype=torch.int32, device=codes.device)[:, None] + torch.tensor([0, 16], dtype=torch.int32,
                                                                                                device=codes.device)
    words = (c << shifts).sum((-1, -2), dtype=torch.int32).reshape(pages, heads, units, UNIT * (d // 8))
    placed = torch.empty_like(words)
    placed[..., _places(d, values).flatten().to(codes.device)] = words
    sz = torch.stack([s, z], -1).to(torch.bfloat16).contiguous().view(torch.int32).reshape(pages, heads, units, UNIT * g)
    unit = torch.cat([placed, sz], -1).contiguous()
    return unit.view(torch.uint8).reshape(pages, heads, tokens, row_bytes(d))


def unpack_pages(pool: torch.Tensor, d: int, values: bool):
    """``(codes, s, z)`` of a pool, as :func:`pack_pages` takes them (scales and offsets in bfloat16)."""
    pages, heads, tokens, width = pool.shape
    _check_pool(tokens, d)
    if pool.dtype != torch.uint8 or width != row_bytes(d):
        raise ValueError(f"a pool of rows of {d} elements is uint8 [.., {row_bytes(d)}], not {pool.dtype} [.., {width}]")
    g, units = groups(d), tokens // UNIT
    unit = pool.contiguous().reshape(pages, heads, units, UNIT * width).view(torch.int32)
    words = unit[..., :UNIT * (d // 8)][..., _places(d, values).flatten().to(pool.device)]
    sz = unit[..., UNIT * (d // 8):].contiguous().view(torch.bfloat16).reshape(pages, heads, tokens, g, 2)
    shifts = 4 * torch.arange(4, dtype=torch.int32, device=pool.device)[:, None] + torch.tensor([0, 16], dtype=torch.int32,
                                                                                               device=pool.device)
    codes = ((words[..., None, None] >> shifts) & 15).to(torch.uint8).reshape(pages, heads, tokens, d)
    return codes, sz[..., 0].contiguous(), sz[..., 1].contiguous()
