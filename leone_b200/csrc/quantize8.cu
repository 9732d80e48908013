// Rows of tokens in 8-bit integers with a scale each: s = max|x| / 127, code = rint(127 x / max|x|), so that s * code is off by at
// most half of s.  A row that holds a NaN or an infinity has codes 0 and the scale NaN: what is made of it is NaN.
//
// The quotient's rounding is that of 64 bits: in fp32 it is off by less than 4e-5, and a value that comes within 1e-4 of the border
// of two codes (one in 5,000) is divided again in 64 bits.
#include "common.cuh"

namespace leone {

constexpr int kQuantThreads = 256;

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
    if (wide || fabsf(fabsf(t - q) - 0.5f) < 1e-4f) q = (float)rint((double)v * 127.0 / (double)top);
    dst[c] = (int8_t)(int)q;
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = odd ? NAN : top / 127.f;
}

}  // namespace leone

using namespace leone;

// x [m, k] with ldx elements between rows; codes [m, k] without gaps, scales [m].
extern "C" int leone_quantize_rows(int dtype, const void* x, int m, int k, int ldx, void* codes, float* scales, cudaStream_t stream) {
  if (m <= 0) return 0;
  if (k <= 0 || ldx < k) return kRefusedSize;
  if (dtype == 0)
    return launch_kernel(quantize_rows_kernel<float>, dim3(m), dim3(kQuantThreads), 0, stream, (const float*)x, ldx, (int8_t*)codes,
                         scales, k);
  if (dtype == 1)
    return launch_kernel(quantize_rows_kernel<__nv_bfloat16>, dim3(m), dim3(kQuantThreads), 0, stream, (const __nv_bfloat16*)x, ldx,
                         (int8_t*)codes, scales, k);
  return kRefusedDtype;
}
