"""Products of 8-bit integers: matrices with a scale for each row, tokens rounded on the way with a scale each.

``out[m, n] = sum_k a[m, k] w[n, k] * s_a[m] * s_w[n]``: the codes ``w`` and scales ``s_w`` of a matrix are made once
(:func:`quantize_matrix`), a token's when it is multiplied (``csrc/quantize8.cu``); the sums are exact integers on the tensor cores
and the two scales are applied in fp32.  The reference's quantised matrices are 4 to 8 bit blocks of GGUF files, multiplied in fp32
or with 8-bit activations on dp4a (crates/leone-cuda/cuda/ie_cuda.cu:1718-1931).
"""
from __future__ import annotations

import ctypes
from ctypes import addressof, c_float
from typing import Optional

import torch

from ..csrc.build import ensure_built
from .entry_points import EntryPoints

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

    force = None               # (on pairs of SMs, tile width) of every product, whatever the rule says (tests set it)

    def choose(self, m: int, n: int, k: int, gated: bool):
        """``(on pairs of SMs, weight rows per tile)``."""
        if m > 128:
            return True, 256
        return False, 32 * max(1, min(8, -(-n // (32 * self.sm_count))))

    def run(self, x, w: Int8Matrix, out, epilogue, residual, gate_shape) -> int:
        """A product of ``x`` with ``w``; returns the number of launches."""
        from .cuda import _check, _dt
        m, k = x.shape
        n = w.out_features
        stream = self.ops._stream()
        codes = self.ops._scratch("int8_codes", m, k, torch.int8)
        scales = self.ops._scratch("int8_scales", m, 1, torch.float32)
        _check(self.ops.packed_calls.leone_quantize_rows(_dt(x.dtype), x, m, k, x.stride(0), codes, scales, stream), "quantize_rows")
        shape = None if gate_shape is None else (c_float * 4)(*[float(v) for v in gate_shape])
        gs = None if shape is None else addressof(shape)
        pairs, width = self.force or self.choose(m, n, k, epilogue == 3)
        entry = self.calls.leone_gemm_pair_i8 if pairs else self.calls.leone_gemm_narrow_i8
        _check(entry(codes, scales, w.weight, w.scales, out, residual, m, n, k, k, k, out.stride(0), epilogue, width, self.ops.status,
                     self.sm_count, gs, w.bias, stream), "gemm_int8")
        return 2
