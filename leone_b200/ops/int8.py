"""Products of 8-bit integers: matrices with a scale for each row, tokens rounded on the way with a scale each.

``out[m, n] = sum_k a[m, k] w[n, k] * s_a[m] * s_w[n]``: the codes ``w`` and scales ``s_w`` of a matrix are made once
(:func:`quantize_matrix`), a token's when it is multiplied (``csrc/quantize8.cu``); the sums are exact integers on the tensor cores
and the two scales are applied in fp32.  The reference's quantised matrices are 4 to 8 bit blocks of GGUF files, multiplied in fp32
or with 8-bit activations on dp4a (crates/leone-cuda/cuda/ie_cuda.cu:1718-1931).
"""
from __future__ import annotations

import ctypes
import threading
from ctypes import addressof, c_float
from typing import Optional

import torch

from ..csrc.build import ensure_built
from .entry_points import EntryPoints

# the forms of a product: a stream over the weights for few tokens (gemm_int8.cu), single SMs (gemm_narrow.cu), pairs (gemm_pair.cu)
STREAM, NARROW, PAIRS = 0, 1, 2
MAX_K = 1 << 17            # sums of 127 * 127 * MAX_K stay in 32 bits


def quantize_matrix(w: torch.Tensor):
    """``(codes int8 [out, in], scales fp32 [out])`` of a matrix: ``s = max|row| / 127``, ``code = rint(127 w / max|row|)``.  A row of
    zeros has the scale 0; one that holds a NaN or an infinity has codes 0 and the scale NaN."""
    if w.dim() != 2:
        raise ValueError("a weight matrix is [out, in]")
    codes = torch.empty(w.shape, dtype=torch.int8, device=w.device)
    scales = torch.empty(w.shape[0], dtype=torch.float32, device=w.device)
    rows = max(1, (1 << 24) // max(w.shape[1], 1))          # in pieces: the 64-bit quotients take eight times a matrix's bytes
    for r in range(0, w.shape[0], rows):
        x = w[r:r + rows].float()
        top = x.abs().amax(1, keepdim=True)
        fine = torch.isfinite(x).all(1, keepdim=True)
        q = torch.round(x.double() * 127 / torch.where(fine & (top > 0), top, torch.ones_like(top)).double())
        codes[r:r + rows] = torch.where(fine, q, torch.zeros_like(q)).to(torch.int8)
        scales[r:r + rows] = torch.where(fine, top / torch.full_like(top, 127), torch.full_like(top, float("nan")))[:, 0]
    return codes, scales


class PerThread(threading.local):
    """``held``: a dictionary of the calling thread's own."""

    def __init__(self):
        self.held = {}


class Int8Matrix:
    """A matrix ``[out, in]`` in 8-bit integers with a scale for each row, and the fp32 bias ``[out]`` (or None) of its products."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor] = None):
        self.weight = codes
        self.scales = scales
        self.bias = bias
        self.out_features, self.in_features = codes.shape

    @property
    def shape(self):
        return self.weight.shape

    @property
    def dtype(self):
        return self.weight.dtype


class Int8Products:
    """The launches of a :class:`leone_b200.ops.cuda.CudaOps`."""

    def __init__(self, ops):
        self.ops = ops
        self.lib = ctypes.CDLL(ensure_built("bf16"))
        if ops.fast is None:
            self.lib.leone_bf16_set_pdl(1 if ops._pdl else 0)
        self.calls = EntryPoints(self.lib)
        self.sm_count = torch.cuda.get_device_properties(ops.device).multi_processor_count
        self.plans, self.buffers = {}, PerThread()

    force = None               # (form, splits or tile width) of every product, whatever the rule says (tests set it)

    def choose(self, m: int, n: int, k: int):
        """The form of a product: ``(STREAM, splits)``, ``(NARROW, tile width)`` or ``(PAIRS, tile width)``.  Times below with the rounding of
        the tokens, from cold caches.

        Up to 32 tokens the stream: 8 tokens 24576 x 4096 30.9 us (33.2 on narrow tiles), 4096 x 12288 21.2 (24.8).  Its splits of K until nine
        tenths of the SMs' places (two each) are taken, which clusters of up to 8 find.
        From there to 128 narrow tiles of the width of the lowest estimate, in us: 3.2, 0.012 for every tile past 64, for every
        round of tiles over the SMs and k-block 0.12 + 0.0007 a weight row (no less than the weights at 6 MB a us), and 0.02 a weight
        row for the last tile's epilogue.  64 tokens 24576 x 4096: 34.9 us with 64 rows, 35.0 with 96, 39.1 with 192, 41 with 32.
        From 129 on pairs, the width likewise: 2.3 + 0.016 a weight row and for every round over the pairs and k-block the longest of
        0.18, 0.0013 a weight row and the operands at 18 MB a us.  512 tokens 2048 x 6144: 30.9 us with 128 rows, 41.0 with 256;
        2,048 tokens 24576 x 4096: 133 with 224, 136 with 192 and 256, 152 with 128."""
        k_blocks, best = -(-k // 128), None
        if m <= 32:
            return STREAM, max(1, min(8, 2 * self.sm_count * 9 // 10 // -(-n // 128), k_blocks // 2))
        for w in range(256, 31, -32):
            tiles = -(-n // w)
            if m <= 128:
                cost = max(3.2 + 0.012 * max(0, min(tiles, self.sm_count) - 64) + -(-tiles // self.sm_count) * k_blocks * (0.12 + 0.0007 * w),
                           n * k / 6e6) + 0.02 * w
            else:
                pairs, tiles = self.sm_count // 2, tiles * -(-m // 256)
                block = max(0.18, 0.0013 * w, min(tiles, pairs) * (256 + w) * 128 / 18e6)
                cost = 2.3 + 0.016 * w + -(-tiles // pairs) * k_blocks * block
            if best is None or cost < 0.99 * best[0]:
                best = (cost, w)
        return (NARROW if m <= 128 else PAIRS), best[1]

    def run(self, x, w: Int8Matrix, out, epilogue, residual, gate_shape) -> int:
        """A product of ``x`` with ``w``; returns the number of launches."""
        ops = self.ops
        m, k = x.shape
        n = w.out_features
        plan = self.plans.get((m, n, k))
        if plan is None:
            plan = self.plans[m, n, k] = self.choose(m, n, k)
        form, width = self.force or plan
        step = x.stride(0) if m > 1 else k                   # elements between rows, 32 bits in the kernels
        if step >= 1 << 31:
            raise OverflowError(f"linear (8 bits): rows {step} elements apart")
        stream = ops._stream()
        codes, scales = self.tokens(m, k, stream)
        gs = None
        if gate_shape is not None:
            shape = (c_float * 4)(*[float(v) for v in gate_shape])
            gs = addressof(shape)
        code = self.calls.leone_linear_i8(1 if x.dtype == torch.bfloat16 else 0, x, step, codes, scales, w.weight, w.scales, out,
                                          residual, m, n, k, out.stride(0), epilogue, form, width, ops.status, self.sm_count, gs, w.bias,
                                          stream)
        if code != 0:
            from .cuda import _check
            _check(code, "linear (8 bits)")
        return 2

    def tokens(self, m: int, k: int, stream):
        """Codes and scales of ``m`` tokens for the call at hand.  A captured graph has its own (from the graph's pool), so that graphs may
        be replayed beside one another; every other call those of its width, thread and stream, which only grow.  (Between a call's
        two launches there may be one of another thread's on the same stream.)"""
        captured = torch.cuda.is_current_stream_capturing()
        buffers = self.buffers.held
        held = None if captured else buffers.get((k, stream))
        if held is not None and held[0].shape[0] >= m:
            return held
        rows = m if captured else -(-m // 64) * 64
        fresh = (torch.empty((rows, k), dtype=torch.int8, device=self.ops.device),
                 torch.empty(rows, dtype=torch.float32, device=self.ops.device))
        if not captured:
            buffers[k, stream] = fresh
        return fresh
