// Rows of tokens in 8-bit integers with a scale each: s = max|x| / 127, code = rint(127 x / max|x|), so that s * code is off by at
// most half of s.  A row that holds a NaN or an infinity has codes 0 and the scale NaN: what is made of it is NaN.
//
// The quotient's rounding is that of 64 bits: in fp32 (two roundings) it is off by less than 1.25e-7 of itself, and a value that
// comes so near to the border of two codes (a few in a million) is divided again in 64 bits.
#include "common.cuh"

namespace leone {

constexpr int kQuantThreads = 256;

// Whether the quotient t, which is rounded to q, may lie on the other side of a border of two codes.
__device__ __forceinline__ bool at_border(float t, float q) { return fabsf(fabsf(t - q) - 0.5f) <= fabsf(t) * 1.25e-7f; }

template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
quantize_rows_kernel(const T* __restrict__ x, int ldx, int8_t* __restrict__ codes, float* __restrict__ scales, int k) {
  __shared__ float scratch[33];
  pdl_trigger();
  pdl_wait();
  const T* row = x + (size_t)blockIdx.x * ldx;
  int8_t* dst = codes + (size_t)blockIdx.x * k;
  float top = 0.f;
  int odd = 0;
  for (int c = threadIdx.x; c < k; c += kQuantThreads) {
    const float v = fabsf(to_float<T>(row[c]));
    odd |= !(v < INFINITY);
    top = fmaxf(top, v);
  }
  odd = __syncthreads_or(odd);
  top = block_max(top, scratch);
  if (odd) top = 0.f;
  const float inv = top > 0.f ? 127.f / top : 0.f;
  const bool wide = !(inv < INFINITY);                    // (a row of the smallest numbers)
  for (int c = threadIdx.x; c < k; c += kQuantThreads) {
    const float v = odd ? 0.f : to_float<T>(row[c]);
    float t = v * inv, q = rintf(t);
    if (at_border(t, q) || wide) q = (float)rint((double)v * 127.0 / (double)top);
    dst[c] = (int8_t)(int)q;
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = odd ? NAN : top / 127.f;
}

// The same where rows start on 16 bytes and have a multiple of 16 elements, up to 16,384: a thread holds 16 elements of the row from its
// only reading on, a block has just the threads that a row takes.  (2,048 rows of 4,096 in bfloat16 12.5 us, 17 in the form above.)
template <typename T>
__global__ void __launch_bounds__(1024)
quantize_rows16_kernel(const T* __restrict__ x, int ldx, int8_t* __restrict__ codes, float* __restrict__ scales, int k) {
  constexpr int kLoads = 16 * sizeof(T) / 16;
  __shared__ float top_s[32];
  pdl_trigger();
  pdl_wait();
  const int at = threadIdx.x * 16, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (blockDim.x + 31) >> 5;
  uint4 raw[kLoads];                                       // (kept as they come: the floats of 16 elements would cost half of the warps)
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    raw[i] = at < k ? reinterpret_cast<const uint4*>(x + (size_t)blockIdx.x * ldx + at)[i] : make_uint4(0, 0, 0, 0);
  const T* e = reinterpret_cast<const T*>(raw);
  // as bit patterns absolute values have the order of their numbers, with infinity and the NaNs above all
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) bits = max(bits, __float_as_uint(to_float<T>(e[i])) & 0x7fffffffu);
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (warps > 1) {
    if (lane == 0) top_s[warp] = __uint_as_float(bits);
    __syncthreads();
    bits = __reduce_max_sync(0xffffffffu, lane < warps ? __float_as_uint(top_s[lane]) : 0u);
  }
  const bool odd = bits >= 0x7f800000u;
  const float top = odd ? 0.f : __uint_as_float(bits);
  const float inv = top > 0.f ? 127.f / top : 0.f;
  const bool wide = !(inv < INFINITY);
  if (at < k) {
    uint32_t word[4] = {0, 0, 0, 0};
    unsigned close = 0;                                    // elements at the border of two codes
    if (!odd) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float t = to_float<T>(e[i]) * inv, q = rintf(t);
        if (at_border(t, q) || wide) close |= 1u << i;
        word[i >> 2] |= ((uint32_t)(int)q & 255u) << (8 * (i & 3));
      }
    }
    uint8_t* dst = reinterpret_cast<uint8_t*>(codes + (size_t)blockIdx.x * k + at);
    *reinterpret_cast<uint4*>(dst) = make_uint4(word[0], word[1], word[2], word[3]);
    while (close != 0) {                                   // (read again: a register cannot be chosen at run time)
      const int i = __ffs(close) - 1;
      close &= close - 1;
      const double v = to_float<T>(x[(size_t)blockIdx.x * ldx + at + i]);
      dst[i] = (uint8_t)(int8_t)(int)rint(v * 127.0 / (double)top);
    }
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = odd ? NAN : top / 127.f;
}

}  // namespace leone

using namespace leone;

// x [m, k] with ldx elements between rows (0: one row for all; rows may overlap); codes [m, k] without gaps, scales [m].
extern "C" int leone_quantize_rows(int dtype, const void* x, int m, int k, int ldx, void* codes, float* scales, cudaStream_t stream) {
  if (m <= 0) return 0;
  if (k <= 0 || ldx < 0) return kRefusedSize;
  const int item = dtype == 0 ? 4 : 2;
  if (k % 16 == 0 && k <= 16384 && ((long long)ldx * item) % 16 == 0 && (((uintptr_t)x | (uintptr_t)codes) & 15) == 0) {
    const dim3 threads((k / 16 + 31) / 32 * 32);
    if (dtype == 0)
      return launch_kernel(quantize_rows16_kernel<float>, dim3(m), threads, 0, stream, (const float*)x, ldx, (int8_t*)codes, scales, k);
    if (dtype == 1)
      return launch_kernel(quantize_rows16_kernel<__nv_bfloat16>, dim3(m), threads, 0, stream, (const __nv_bfloat16*)x, ldx,
                           (int8_t*)codes, scales, k);
  }
  if (dtype == 0)
    return launch_kernel(quantize_rows_kernel<float>, dim3(m), dim3(kQuantThreads), 0, stream, (const float*)x, ldx, (int8_t*)codes,
                         scales, k);
  if (dtype == 1)
    return launch_kernel(quantize_rows_kernel<__nv_bfloat16>, dim3(m), dim3(kQuantThreads), 0, stream, (const __nv_bfloat16*)x, ldx,
                         (int8_t*)codes, scales, k);
  return kRefusedDtype;
}
