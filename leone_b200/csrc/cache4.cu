// A step's keys and values into pages in 4 bits (cache4.cuh), what such pages hold, and attention over them at any size.
#include "cache4.cuh"

namespace leone {
namespace cache4 {

// Where token t's row of a cached head lies: its unit and its place there; false (and a status) where the step's metadata names no
// page.
struct Place {
  long long page;
  int slot;
};
__device__ __forceinline__ bool find_place(Place& place, int t, int pos, const int* seq_of_token, int n_seqs, const int* block_table,
                                           int table_width, int num_pages, int page_tokens, int* status, bool report) {
  const int s = seq_of_token[t];
  if (s < 0 || s >= n_seqs) {
    if (report) set_status(status, kBadSequence, t, s);
    return false;
  }
  const int blk = pos / page_tokens;
  const int page = (pos >= 0 && blk < table_width) ? block_table[(size_t)s * table_width + blk] : -1;
  if (page < 0 || page >= num_pages) {
    if (report) set_status(status, kBadPage, t, page, pos);
    return false;
  }
  place.page = page;
  place.slot = pos % page_tokens;
  return true;
}

// The largest float not above v, then the largest bfloat16 not above that: rounding down twice rounds down once.
__device__ __forceinline__ __nv_bfloat16 bf16_down(double v) { return __float2bfloat16_rd(__double2float_rd(v)); }
__device__ __forceinline__ __nv_bfloat16 bf16_up(double v) { return __float2bfloat16_ru(__double2float_ru(v)); }

// RMSNorm and rotation of q and k per head as in qk_norm_rope_write (elementwise.cu), queries back into qkv, keys and values into
// the pools in 4 bits.  One warp per (token, head).  Everything in 64 bits: the code of a key next to the border of two codes then
// does not depend on the order in which the head's squares are added.
template <typename T, typename TW>
__global__ void append_kernel(T* __restrict__ qkv, int n_tokens, int n_q, int n_kv, int d, const TW* __restrict__ q_w,
                              const TW* __restrict__ k_w, float eps, const float2* __restrict__ rope, int rotary_dim,
                              int max_positions, const int* __restrict__ positions, const int* __restrict__ seq_of_token,
                              const int* __restrict__ block_table, int table_width, int n_seqs, uint8_t* __restrict__ k_pool,
                              uint8_t* __restrict__ v_pool, int num_pages, int page_tokens, int adjacent, int* status) {
  extern __shared__ double row_s[];
  pdl_trigger();
  pdl_wait();
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = n_q + 2 * n_kv;
  const long long item = (long long)blockIdx.x * warps + warp;
  if (item >= (long long)n_tokens * heads) return;
  const int t = (int)(item / heads), h = (int)(item - (long long)t * heads);
  double* x = row_s + (size_t)warp * d;
  T* row = qkv + ((size_t)t * heads + h) * d;
  const bool is_q = h < n_q, is_k = !is_q && h < n_q + n_kv;
  const int pos = positions[t];
  if ((is_q || is_k) && rope != nullptr && (pos < 0 || pos >= max_positions)) {
    if (lane == 0) set_status(status, kBadPosition, t, pos);
    return;
  }
  Place place;
  if (!is_q && !find_place(place, t, pos, seq_of_token, n_seqs, block_table, table_width, num_pages, page_tokens, status, lane == 0))
    return;

  const TW* w = is_q ? q_w : (is_k ? k_w : nullptr);
  double ss = 0.0;
  for (int c = lane; c < d; c += 32) {
    const double v = (double)to_float<T>(row[c]);
    x[c] = v;
    ss = fma(v, v, ss);
  }
  if (w != nullptr) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const double factor = rsqrt(ss / d + (double)eps);
    for (int c = lane; c < d; c += 32) x[c] *= (double)to_float<TW>(w[c]) * factor;
  }
  __syncwarp();
  if ((is_q || is_k) && rope != nullptr) {
    const int half = rotary_dim >> 1;
    for (int i = lane; i < half; i += 32) {
      const float2 cs = rope[(size_t)pos * half + i];
      const int at = adjacent ? 2 * i : i, bt = adjacent ? 2 * i + 1 : i + half;
      const double a = x[at], b = x[bt];
      x[at] = a * cs.x - b * cs.y;
      x[bt] = a * cs.y + b * cs.x;
    }
    __syncwarp();
  }
  if (is_q) {
    for (int c = lane; c < d; c += 32) row[c] = from_float<T>((float)x[c]);
    return;
  }
  const int G = groups(d), size = d / G;
  uint8_t* unit = (is_k ? k_pool : v_pool) +
                  unit_at(place.page, n_kv, is_k ? h - n_q : h - n_q - n_kv, page_tokens, place.slot / kUnit * kUnit, d);
  const int slot = place.slot % kUnit;
  for (int g = 0; g < G; ++g) {
    double lo = INFINITY, hi = -INFINITY;
    bool odd = false;                                       // a NaN or an infinity
    for (int c = lane; c < size; c += 32) {
      const double v = x[g * size + c];
      odd |= !isfinite(v);
      lo = fmin(lo, v);
      hi = fmax(hi, v);
    }
    odd = __any_sync(0xffffffffu, odd);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo = fmin(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmax(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    __nv_bfloat16 z16 = bf16_down(lo);
    const double z = __bfloat162float(z16);
    __nv_bfloat16 s16 = bf16_up((hi - z) / 15.0);
    if (__bfloat162float(s16) < 1.17549435e-38f) s16 = __float2bfloat16_rn(0.f);
    odd |= !isfinite(z) || !isfinite(__bfloat162float(s16));
    if (odd) z16 = s16 = __ushort_as_bfloat16(0x7fc0);
    const double s = __bfloat162float(s16);
    for (int i = lane; i < size / 8; i += 32) {
      uint32_t word = 0;
      if (!odd && s > 0.0) {
        for (int e = 0; e < 8; ++e) {
          const double q = rint((x[g * size + 8 * i + e] - z) / s);
          word |= (uint32_t)fmin(fmax(q, 0.0), 15.0) << (4 * (e >> 1) + 16 * (e & 1));
        }
      }
      const int word_at = g * (size / 8) + i;
      *reinterpret_cast<uint32_t*>(unit + (is_k ? key_word_at(slot, word_at, d) : value_word_at(slot, word_at, d))) = word;
    }
    if (lane == 0)
      *reinterpret_cast<uint32_t*>(unit + scale_at(slot, g, d)) =
          (uint32_t)__bfloat16_as_ushort(s16) | (uint32_t)__bfloat16_as_ushort(z16) << 16;
  }
}

// One row into its page by one warp, everything in 64 bits: rows for which append_vec_kernel's 32 bits leave a code in doubt.  `row` in
// shared memory; w: the norm's weights or null; rope: the position's pairs or null.
template <typename T, typename TW, int D>
__device__ __noinline__ void append_exact(const T* row, const TW* w, float eps, const float2* rope, bool adjacent, bool is_k, int slot,
                                          uint8_t* unit) {
  constexpr int E = D / 32, G = D / 64, kGroupLanes = 32 / G, kWordLanes = 8 / E;
  const int lane = threadIdx.x & 31;
  double d[E], most = -INFINITY, least = INFINITY;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < E; ++i) d[i] = (double)to_float<T>(row[lane * E + i]);
  if (w != nullptr) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) ss = fma(d[i], d[i], ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const double factor = rsqrt(ss / D + (double)eps);
#pragma unroll
    for (int i = 0; i < E; ++i) d[i] *= (double)to_float<TW>(w[lane * E + i]) * factor;
  }
  if (rope != nullptr) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (adjacent) {
        if (i & 1) continue;
        const float2 cs = rope[(lane * E + i) >> 1];
        const double a = d[i], b = d[i + 1];
        d[i] = a * cs.x - b * cs.y;
        d[i + 1] = a * cs.y + b * cs.x;
      } else {
        const float2 cs = rope[(lane & 15) * E + i];
        const double other = __shfl_xor_sync(0xffffffffu, d[i], 16);
        d[i] = lane >= 16 ? other * cs.y + d[i] * cs.x : d[i] * cs.x - other * cs.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    odd |= !isfinite(d[i]);
    least = fmin(least, d[i]);
    most = fmax(most, d[i]);
  }
#pragma unroll
  for (int o = kGroupLanes / 2; o > 0; o >>= 1) {
    least = fmin(least, __shfl_xor_sync(0xffffffffu, least, o));
    most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
    odd |= __shfl_xor_sync(0xffffffffu, (int)odd, o) != 0;
  }
  __nv_bfloat16 z16 = bf16_down(least);
  const double z = __bfloat162float(z16);
  __nv_bfloat16 s16 = bf16_up((most - z) / 15.0);
  if (__bfloat162float(s16) < 1.17549435e-38f) s16 = __float2bfloat16_rn(0.f);
  odd |= !isfinite(z) || !isfinite(__bfloat162float(s16));
  if (odd) z16 = s16 = __ushort_as_bfloat16(0x7fc0);
  const double s = __bfloat162float(s16);
  // the word's lanes put their nibbles together (element 2 j in nibble j, 2 j + 1 in nibble j + 4), the first of them stores it
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const uint32_t code = !odd && s > 0.0 ? (uint32_t)fmin(fmax(rint((d[i] - z) / s), 0.0), 15.0) : 0u;
    word |= code << (4 * (i >> 1) + 16 * (i & 1));
  }
  word <<= 4 * (E / 2) * (lane % kWordLanes);
#pragma unroll
  for (int o = 1; o < kWordLanes; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
  const int w_at = lane / kWordLanes;
  if (lane % kWordLanes == 0)
    *reinterpret_cast<uint32_t*>(unit + (is_k ? key_word_at(slot, w_at, D) : value_word_at(slot, w_at, D))) = word;
  if (lane % kGroupLanes == 0)
    *reinterpret_cast<uint32_t*>(unit + scale_at(slot, lane / kGroupLanes, D)) =
        (uint32_t)__bfloat16_as_ushort(s16) | (uint32_t)__bfloat16_as_ushort(z16) << 16;
}

// The same for heads of 64 and 128 elements that rotate whole or not at all.  grid = (tokens, blocks of `per` heads); a block brings its
// rows into shared memory at once, then its warps take two heads each in turn, with the token's place, rotation and norm weights
// at hand: half a warp for a head, lane r with elements H r .. H r + H - 1 of the head's first half and of its second.  So a pair
// of the rotation lies in one lane whichever way elements pair, and a group of 64 is one half of 128 or all of 64.
//
// Codes are those of 64 bits.  Keys are normed and rotated in 64 bits and then rounded to 32 (kRounded of the value off), values
// are what they are; minima, maxima and quotients are of 32.  Where the ends of the range in which the minimum and the maximum lie give
// one z and one s, those are right.  A quotient that comes no nearer to a border of two codes than the roundings take it is rounded right;
// one that does is settled by the sign of x - z - (code + 1/2) s in 64 bits.  (Values in bfloat16 lie on a border more often than
// not in a row.)  Where z or s is in doubt, where a key's rounding is a quarter of a step and more, or something is not finite, the
// warp computes the row again, which a step hardly ever does: that code is never in the instruction cache, and a block waits 4 us for it.
// (With norm and rotation in 32 bits a row of keys in a hundred was in doubt: 2,048 tokens of 48 heads of 128 took 28.2 us, of 22 of 64
// 10.6, where this takes 20.6 and 8.6.  Their queries alone take 8.6, the bytes 6.8.)
constexpr float kRounded = 1.01f / 16777216.f;
constexpr float kToInteger = 12582912.f;           // 1.5 2^23: adding it rounds to an integer, which the low bits then hold
constexpr int kAppendWarps = 4;
constexpr int kAppendHeads = 48;                   // of a block, at most

// Over the 16 lanes of half a warp.
__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float half_min(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The largest number of 8 bits that is not above v, and the smallest that is not below v >= 0; v finite (of another a doubt is known).
__device__ __forceinline__ float eight_bits_down(float v) {
  const uint32_t b = __float_as_uint(v);
  return __uint_as_float((b + ((int)b < 0 ? 0xffffu : 0u)) & 0xffff0000u);
}
__device__ __forceinline__ float eight_bits_up(float v) { return __uint_as_float((__float_as_uint(v) + 0xffffu) & 0xffff0000u); }
__device__ __forceinline__ float reciprocal(float v) {                   // off by at most 2^-23 of itself
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
template <typename F> __device__ __forceinline__ void turn_pair(F& x, F& y, float2 c) {
  const F u = x * (F)c.x - y * (F)c.y;
  y = x * (F)c.y + y * (F)c.x;
  x = u;
}

// kFew: the form for up to two blocks an SM.  Its code is one copy for keys and values, and a block first goes through it over what happens
// to be in shared memory, with results that go nowhere, while the kernel before this one still works: a launch of a step finds the code
// in no cache, and waited longer for it than it ran.  An 8B layer's products with append and decode attention over 2,048 keys: one token 89.8
// us, 87.5 with one copy, 85.1 so; 8 tokens 95.6, 92.1, 89.9; 64 tokens (384 blocks) no less.  In a loop of its own, where the code stays, the
// append of one token takes 3.5 us so and 3.0 in the other form.
template <typename T, typename TW, int D, bool kFew>
__global__ void __launch_bounds__(32 * kAppendWarps, kFew ? 4 : 5)
append_vec_kernel(T* __restrict__ qkv, int n_q, int n_kv, const TW* __restrict__ q_w, const TW* __restrict__ k_w, float eps,
                  const float2* __restrict__ rope, int max_positions, const int* __restrict__ positions,
                  const int* __restrict__ seq_of_token, const int* __restrict__ block_table, int table_width, int n_seqs,
                  uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, int num_pages, int page_tokens, int adjacent, int per,
                  int* status) {
  constexpr int H = D / 32, G = D / 64, kWordLanes = 8 / H;
  constexpr unsigned kAll = 0xffffffffu;
  pdl_trigger();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, sub = threadIdx.x >> 4 & 1, r = threadIdx.x & 15;
  const int heads = n_q + 2 * n_kv;
  const int h0 = blockIdx.y * per, h1 = min(heads, h0 + per);
  struct __align__(sizeof(T) * H) Part { T e[H]; };        // a lane's elements of half a head
  extern __shared__ __align__(16) uint8_t rows_s[];
  T* tok = qkv + (size_t)t * heads * D;
#pragma unroll 1
  for (int pass = kFew ? 0 : 1; pass < 2; ++pass) {
    const bool dry = kFew && pass == 0;
    if (!dry) {
      pdl_wait();
      for (int i = threadIdx.x; i < (h1 - h0) * D * (int)sizeof(T) / 16; i += 32 * kAppendWarps) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(rows_s) + 16 * i;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(reinterpret_cast<const uint4*>(tok + (size_t)h0 * D) + i)
                     : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const int pos = dry ? 0 : positions[t];
    const bool in_table = rope == nullptr || dry || (pos >= 0 && pos < max_positions), rotate = rope != nullptr && in_table;
    if (!in_table && threadIdx.x == 0) set_status(status, kBadPosition, t, pos);
    const float2* turn = rotate ? rope + (size_t)pos * (D / 2) : nullptr;
    // the lane's pairs: element i of the first half with i of the second, or elements 2 i, 2 i + 1 of the first, then of the second
    float2 cs[H];
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const int pair = !adjacent ? H * r + i : H / 2 * r + i % (H / 2) + i / (H / 2) * (D / 4);
      cs[i] = rotate && !dry ? turn[pair] : make_float2(1.f, 0.f);
    }
    float wa[H], wb[H];
    auto weights = [&](const TW* from) {
#pragma unroll
      for (int i = 0; i < H; ++i) {
        wa[i] = dry ? 1.f : to_float<TW>(from[H * r + i]);
        wb[i] = dry ? 1.f : to_float<TW>(from[D / 2 + H * r + i]);
      }
    };
    const Part* rows = reinterpret_cast<const Part*>(rows_s) + r;                 // 32 for every head
    auto fetch = [&](int at, float (&a)[H], float (&b)[H]) {
      const Part x = rows[at * 32], y = rows[at * 32 + 16];
#pragma unroll
      for (int i = 0; i < H; ++i) {
        a[i] = to_float<T>(x.e[i]);
        b[i] = to_float<T>(y.e[i]);
      }
    };
    auto norm = [&](float (&a)[H], float (&b)[H]) {
      float sa = a[0] * a[0], sb = b[0] * b[0];
#pragma unroll
      for (int i = 1; i < H; ++i) {
        sa = fmaf(a[i], a[i], sa);
        sb = fmaf(b[i], b[i], sb);
      }
      const float f = rsqrtf(half_sum(sa + sb) * (1.f / D) + eps);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        a[i] = a[i] * wa[i] * f;
        b[i] = b[i] * wb[i] * f;
      }
    };
    auto rotated = [&](auto& a, auto& b) {                   // a pair and its turn: (x, y) (cos, sin)
      if (adjacent) {
#pragma unroll
        for (int i = 0; i < H / 2; ++i) {
          turn_pair(a[2 * i], a[2 * i + 1], cs[i]);
          turn_pair(b[2 * i], b[2 * i + 1], cs[H / 2 + i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < H; ++i) turn_pair(a[i], b[i], cs[i]);
      }
    };
    const int n_queries = max(0, min(h1, n_q) - h0), n_keys = max(0, min(h1, n_q + n_kv) - max(h0, n_q));
    const int n_values = h1 - h0 - n_queries - n_keys;
    int p = warp;                                            // two heads of one kind; the kinds' follow one another
    if (p < (n_queries + 1) / 2 && q_w != nullptr) weights(q_w);
    Place place{0, 0};
    const bool placed = h1 <= n_q || dry ||
                        find_place(place, t, pos, seq_of_token, n_seqs, block_table, table_width, num_pages, page_tokens,
                                                status, threadIdx.x == 0);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    for (; p < (n_queries + 1) / 2; p += kAppendWarps) {
      const bool real = 2 * p + sub < n_queries;
      const int at = real ? 2 * p + sub : 2 * p;
      float a[H], b[H];
      fetch(at, a, b);
      if (q_w != nullptr) norm(a, b);
      if (rotate) rotated(a, b);
      Part x, y;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        x.e[i] = from_float<T>(a[i]);
        y.e[i] = from_float<T>(b[i]);
      }
      if (real && in_table && !dry) {
        Part* to = reinterpret_cast<Part*>(tok + (size_t)(h0 + at) * D) + r;
        to[0] = x;
        to[16] = y;
      }
    }
    p -= (n_queries + 1) / 2;
    if (!placed) return;                                     // (in the pass that counts)
    const long long unit = unit_at(place.page, n_kv, 0, page_tokens, place.slot / kUnit * kUnit, D);
    const int slot = place.slot % kUnit, head_bytes = page_tokens * row_bytes(D);
    // of the lanes that share a word of the first half and one of the second, the first stores the one and the last the other
    const int w_at = r / kWordLanes + (r % kWordLanes == kWordLanes - 1 ? D / 16 : 0);
    const bool stores = r % kWordLanes == 0 || r % kWordLanes == kWordLanes - 1;
    auto store = [&](bool is_k, int first, int count) {      // heads first .. first + count - 1 of the block's
      const bool computed = is_k && (k_w != nullptr || rotate);
      const int word_at = is_k ? key_word_at(slot, w_at, D) : value_word_at(slot, w_at, D);
      for (; p < (count + 1) / 2; p += kAppendWarps) {
        if (is_k && !in_table) continue;                     // (their position is reported; values need none)
        const bool real = 2 * p + sub < count;
        const int at = first + (real ? 2 * p + sub : 2 * p);
        float a[H], b[H];
        double da[H], db[H];                                 // of keys
        bool doubt = false;
        fetch(at, a, b);
        if (computed) {
#pragma unroll
          for (int i = 0; i < H; ++i) {
            da[i] = a[i];
            db[i] = b[i];
          }
          if (k_w != nullptr) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < H; ++i) ss = fma(da[i], da[i], fma(db[i], db[i], ss));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(kAll, ss, o);
            ss = ss * (1.0 / D) + (double)eps;
            doubt |= !(ss > 1e-37 && ss < 1e37);
            double f = rsqrtf((float)ss);                    // two steps of Newton's take it to 64 bits
            f *= fma(-0.5 * ss * f, f, 1.5);
            f *= fma(-0.5 * ss * f, f, 1.5);
#pragma unroll
            for (int i = 0; i < H; ++i) {
              da[i] *= (double)wa[i] * f;
              db[i] *= (double)wb[i] * f;
            }
          }
          if (rotate) rotated(da, db);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            a[i] = (float)da[i];
            b[i] = (float)db[i];
          }
        }
        float lo[2], hi[2];                                  // of the halves
        lo[0] = hi[0] = a[0];
        lo[1] = hi[1] = b[0];
#pragma unroll
        for (int i = 0; i < H; ++i) {
          doubt |= !(fabsf(a[i]) < INFINITY) || !(fabsf(b[i]) < INFINITY);
          lo[0] = fminf(lo[0], a[i]);
          hi[0] = fmaxf(hi[0], a[i]);
          lo[1] = fminf(lo[1], b[i]);
          hi[1] = fmaxf(hi[1], b[i]);
        }
        if (G == 1) {
          lo[0] = fminf(lo[0], lo[1]);
          hi[0] = fmaxf(hi[0], hi[1]);
        }
        float z[2], s[2], inv[2], limit[2];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          lo[g] = half_min(lo[g]);
          hi[g] = half_max(hi[g]);
          const float err = computed ? fmaxf(fabsf(lo[g]), fabsf(hi[g])) * kRounded : 0.f;
          z[g] = eight_bits_down(__fsub_rd(lo[g], err));
          doubt |= z[g] != eight_bits_down(__fadd_ru(lo[g], err));
          // s is the smallest with 15 s >= hi - z; 15 s has 12 bits.  Of a value the rounded difference is on the side of 15 s that the
          // difference is on, or meets it; of a key it is off by the maximum's rounding and its own (and the margin's).
          const float range = hi[g] - z[g], margin = err + 2.f * kRounded * range;
          s[g] = eight_bits_up(range * (1.f / 15.f) * (1.f - 6e-7f));         // or the next
          if (15.f * s[g] < range) s[g] = __uint_as_float(__float_as_uint(s[g]) + 0x10000u);
          if (err != 0.f) {
            const float below = __uint_as_float(__float_as_uint(s[g]) - 0x10000u);
            doubt |= !(range - margin > 15.f * below && range + margin < 15.f * s[g]);
          } else if (range == 15.f * s[g]) {
            const float back = hi[g] - range;
            doubt |= (hi[g] - (range + back)) + (back - z[g]) != 0.f;
          }
          doubt |= (s[g] != 0.f && !(s[g] > 1e-37f && s[g] < 1e37f)) || !(fabsf(z[g]) < 3e38f);
          inv[g] = s[g] > 0.f ? reciprocal(s[g]) : 0.f;
          limit[g] = 0.5f - fmaf(err, inv[g] * 1.01f, 15.5f * 2.5e-7f);
          doubt |= limit[g] < 0.25f;                         // (one border has to be the only one in reach)
        }
        if (G == 1) {
          z[1] = z[0];
          s[1] = s[0];
          inv[1] = inv[0];
          limit[1] = limit[0];
        }
        float code[2][H];                                    // + kToInteger
        bool near = false;
#pragma unroll
        for (int i = 0; i < H; ++i)
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float gap = (g ? b[i] : a[i]) - z[g], c = fmaf(gap, inv[g], kToInteger);
            near |= fabsf(fmaf(gap, inv[g], kToInteger - c)) >= limit[g];
            code[g][i] = c;
          }
        if (near) {
#pragma unroll
          for (int i = 0; i < H; ++i)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const float x = g ? b[i] : a[i], q = (x - z[g]) * inv[g], low = floorf(q);
              if (fabsf(fabsf(q - low) - 0.5f) > 0.5f - limit[g] + 1e-5f) continue;      // (what made it near, and the product's rounding)
              const double gap = (computed ? (g ? db[i] : da[i]) : (double)x) - (double)z[g];
              const double side = fma(-(double)(low + 0.5f), (double)s[g], gap);
              code[g][i] = (side > 0.0 || (side == 0.0 && ((int)low & 1)) ? low + 1.f : low) + kToInteger;
            }
        }
        // the word's lanes put their nibbles together (element 2 j in nibble j, 2 j + 1 in nibble j + 4)
        uint32_t word[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          word[g] = 0;
#pragma unroll
          for (int i = 0; i < H; ++i)
            word[g] += (__float_as_uint(code[g][i]) - __float_as_uint(kToInteger)) << (4 * (i >> 1) + 16 * (i & 1));
          word[g] <<= 4 * (H / 2) * (r % kWordLanes);
        }
#pragma unroll
        for (int o = kWordLanes / 2; o > 1; o >>= 1) {
          word[0] |= __shfl_xor_sync(kAll, word[0], o);
          word[1] |= __shfl_xor_sync(kAll, word[1], o);
        }
        const uint32_t other = __shfl_xor_sync(kAll, r & 1 ? word[0] : word[1], 1), whole = (r & 1 ? word[1] : word[0]) | other;
        const unsigned again = __ballot_sync(kAll, doubt);
        uint8_t* pool = is_k ? k_pool + (size_t)(h0 + at - n_q) * head_bytes : v_pool + (size_t)(h0 + at - n_q - n_kv) * head_bytes;
        if (again == 0 || dry) {
          if (real && stores && !dry) *reinterpret_cast<uint32_t*>(pool + unit + word_at) = whole;
          if (real && r < G && !dry)
            *reinterpret_cast<uint32_t*>(pool + unit + scale_at(slot, r, D)) =
                __float_as_uint(r ? s[1] : s[0]) >> 16 | (__float_as_uint(r ? z[1] : z[0]) & 0xffff0000u);
          continue;
        }
        for (int u = 0; u < 2 && 2 * p + u < count; ++u) {
          const int h = first + 2 * p + u;
          append_exact<T, TW, D>(reinterpret_cast<const T*>(rows_s) + (size_t)h * D, is_k ? k_w : (const TW*)nullptr, eps,
                                 is_k ? turn : nullptr, adjacent != 0, is_k, slot,
                                 (is_k ? k_pool + (size_t)(h0 + h - n_q) * head_bytes
                                       : v_pool + (size_t)(h0 + h - n_q - n_kv) * head_bytes) + unit);
        }
      }
      p -= (count + 1) / 2;
    };
    if (in_table && k_w != nullptr && p < (n_keys + 1) / 2) weights(k_w);
    if constexpr (kFew) {
#pragma unroll 1
      for (int kind = 0; kind < 2; ++kind) {
        store(kind == 0, kind == 0 ? n_queries : n_queries + n_keys, kind == 0 ? n_keys : n_values);
      }
    } else {
      store(true, n_queries, n_keys);
      store(false, n_queries + n_keys, n_values);
    }
  }
}

// What the pages hold for the step's tokens: rows [n_tokens][n_kv * d] of keys and of values.  grid = (tokens, blocks of heads); a warp takes
// a cached head at a time, a lane a word of its key, then of its value.
constexpr int kReadWarps = 8;
template <typename T>
__global__ void __launch_bounds__(32 * kReadWarps)
read_kernel(T* __restrict__ k_out, T* __restrict__ v_out, int n_kv, int d, const int* __restrict__ positions,
            const int* __restrict__ seq_of_token, const int* __restrict__ block_table, int table_width, int n_seqs,
            const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool, int num_pages, int page_tokens, int* status) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, t = blockIdx.x;
  Place place;
  if (!find_place(place, t, positions[t], seq_of_token, n_seqs, block_table, table_width, num_pages, page_tokens, status,
                  threadIdx.x == 0))
    return;
  const int slot = place.slot % kUnit, size = d / groups(d), words = d / 8;
  for (int h = blockIdx.y * kReadWarps + (threadIdx.x >> 5); h < n_kv; h += gridDim.y * kReadWarps) {
    const long long item = (long long)t * n_kv + h;
    const long long unit = unit_at(place.page, n_kv, h, page_tokens, place.slot / kUnit * kUnit, d);
    for (int i = lane; i < 2 * words; i += 32) {
      const bool key = i < words;
      const int w = key ? i : i - words;
      const uint8_t* from = (key ? k_pool : v_pool) + unit;
      const uint32_t word = *reinterpret_cast<const uint32_t*>(from + (key ? key_word_at(slot, w, d) : value_word_at(slot, w, d)));
      const uint32_t sz = *reinterpret_cast<const uint32_t*>(from + scale_at(slot, 8 * w / size, d));
      __align__(16) T out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = from_float<T>(fmaf(scale_of(sz), (float)code_of(word, e), offset_of(sz)));
      uint4* dst = reinterpret_cast<uint4*>((key ? k_out : v_out) + item * d + 8 * w);       // (d is a multiple of 8)
#pragma unroll
      for (int e = 0; e < (int)sizeof(T) / 2; ++e) dst[e] = reinterpret_cast<const uint4*>(out)[e];
    }
  }
}

// Causal grouped-query attention over pages in 4 bits, any sizes, any cut: the formulas of attention_generic.cu.  One block per
// (token, cached head, up to kHeads of its query heads, split of the keys) walks its keys in tiles of 32: a tile's keys, then its values,
// are brought into shared memory in fp32; warp w has the scores of heads w and w + 4, a lane a key; thread c sums the outputs' columns
// c, c + 128, ..  A key's or value's number is read once for all heads (2,048 tokens behind 6,144, 32 heads on 8 of
// 128: 34 ms, 58 where it was read for each).  Where there are too few blocks for the SMs,
// `splits` of them share a token's keys and leave their (maximum, sum, unnormalised outputs) in scratch, [token][query head][split], for
// attention_any_merge_kernel (one sequence of 8,192 keys, 8 heads on 2
// of 128, 32 bits: 31 us with 64, 1,380 without).
constexpr int kAnyThreads = 128;
constexpr int kAnyKeys = 32;
__host__ __device__ constexpr int any_row(int d) { return d + 1; }      // floats between the tile's rows: lanes on different banks

template <typename T, int kHeads>
__global__ void __launch_bounds__(kAnyThreads)
attention_any_kernel(const T* __restrict__ qkv, int row_stride, T* __restrict__ out, int out_stride,
                     const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool, const int* __restrict__ block_table,
                     int table_width, const int* __restrict__ seq_of_token, const int* __restrict__ positions, int n_q, int n_kv,
                     int d, float scale, int window, int page_tokens, int num_pages, int n_seqs, int splits, float* __restrict__ part_o,
                     float* __restrict__ part_ml, int* status) {
  extern __shared__ float smem_f[];
  float* tile = smem_f;                                    // [32][any_row(d)]
  float* q_s = tile + kAnyKeys * any_row(d);               // [kHeads][d]
  float* p_s = q_s + kHeads * d;                           // [32][kHeads]
  float* alpha_s = p_s + kHeads * kAnyKeys;                // [kHeads]
  float* l_s = alpha_s + kHeads;                           // [kHeads]
  __shared__ long long unit_s[kAnyKeys];
  constexpr int kWarpHeads = (kHeads + 3) / 4;             // of a warp
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, g = n_q / n_kv, parts = (g + kHeads - 1) / kHeads;
  const int kvh = blockIdx.y / parts, part = blockIdx.y - kvh * parts;
  const int head0 = kvh * g + part * kHeads, heads = min(kHeads, g - part * kHeads);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pos = positions[t], s = seq_of_token[t];
  T* dst = out + (size_t)t * out_stride + (size_t)head0 * d;
  auto part_at = [&](int h) { return ((size_t)t * n_q + head0 + h) * splits + blockIdx.z; };
  if (s < 0 || s >= n_seqs || pos < 0) {
    if (tid == 0) set_status(status, s < 0 || s >= n_seqs ? kBadSequence : kBadPosition, t, s < 0 || s >= n_seqs ? s : pos);
    if (splits > 1) {
      if (tid < heads) *reinterpret_cast<float2*>(part_ml + 2 * part_at(tid)) = make_float2(-INFINITY, 0.f);
      return;
    }
    for (int c = tid; c < heads * d; c += kAnyThreads) dst[c] = from_float<T>(0.f);
    return;
  }
  const T* q = qkv + (size_t)t * row_stride + (size_t)head0 * d;
  for (int c = tid; c < kHeads * d; c += kAnyThreads) q_s[c] = c < heads * d ? to_float<T>(q[c]) : 0.f;
  for (int c = tid; c < kHeads * (kAnyKeys + 1); c += kAnyThreads) p_s[c] = 0.f;        // (and alpha_s: heads that are not there)
  const int G = groups(d), size = d / G, words = d / 8;
  const int first = window > 0 ? max(0, pos - window + 1) : 0;
  const int share = ((pos - first) / kAnyKeys + splits) / splits;               // tiles of a split, rounded up
  const long long lo = first + (long long)blockIdx.z * share * kAnyKeys;
  const int end = (int)min((long long)pos + 1, lo + (long long)share * kAnyKeys);
  float m_run[kWarpHeads], l_run[kWarpHeads];
#pragma unroll
  for (int u = 0; u < kWarpHeads; ++u) {
    m_run[u] = -INFINITY;
    l_run[u] = 0.f;
  }
  float acc[kHeads][kMaxDim / kAnyThreads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
#pragma unroll
    for (int i = 0; i < kMaxDim / kAnyThreads; ++i) acc[h][i] = 0.f;
  auto fetch = [&](const uint8_t* pool, bool keys, int j0) {
    for (int idx = tid; idx < kAnyKeys * words; idx += kAnyThreads) {
      const int r = idx / words, w = idx - r * words;
      float* to = tile + r * any_row(d) + 8 * w;
      if (unit_s[r] < 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) to[e] = 0.f;
        continue;
      }
      const int slot = (j0 + r) % page_tokens % kUnit;
      const uint8_t* unit = pool + unit_s[r];
      const uint32_t word = *reinterpret_cast<const uint32_t*>(unit + (keys ? key_word_at(slot, w, d) : value_word_at(slot, w, d)));
      const uint32_t sz = *reinterpret_cast<const uint32_t*>(unit + scale_at(slot, 8 * w / size, d));
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = fmaf(scale_of(sz), (float)code_of(word, e), offset_of(sz));
    }
  };
  for (int j0 = (int)min(lo, (long long)end); j0 < end; j0 += kAnyKeys) {
    __syncthreads();                                       // the tile before is done with
    if (tid < kAnyKeys) {
      const int j = j0 + tid;
      long long unit = -1;
      if (j < end) {
        const int blk = j / page_tokens;
        const int page = blk < table_width ? block_table[(size_t)s * table_width + blk] : -1;
        if (page < 0 || page >= num_pages) set_status(status, kBadPage, t, page, j);
        else unit = unit_at(page, n_kv, kvh, page_tokens, j % page_tokens / kUnit * kUnit, d);
      }
      unit_s[tid] = unit;
    }
    __syncthreads();
    fetch(k_pool, true, j0);
    __syncthreads();
    float dot[kWarpHeads];
#pragma unroll
    for (int u = 0; u < kWarpHeads; ++u) dot[u] = 0.f;
    if (warp < heads) {
      const float* k = tile + lane * any_row(d);
#pragma unroll 2
      for (int c = 0; c < d; c += 4) {
        const float k0 = k[c], k1 = k[c + 1], k2 = k[c + 2], k3 = k[c + 3];
#pragma unroll
        for (int u = 0; u < kWarpHeads; ++u) {
          const float4 v = *reinterpret_cast<const float4*>(q_s + (warp + 4 * u) * d + c);
          dot[u] = fmaf(v.w, k3, fmaf(v.z, k2, fmaf(v.y, k1, fmaf(v.x, k0, dot[u]))));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kWarpHeads; ++u) {
      const int h = warp + 4 * u;
      if (h >= heads) break;
      const bool here = unit_s[lane] >= 0;
      const float score = here ? dot[u] * scale : -INFINITY;
      // (fmaxf leaves out a NaN; the weight of its key is NaN all the same, and with it the sum)
      const float m_new = fmaxf(m_run[u], warp_max(score));
      const float p = here ? (m_new == -INFINITY ? (isnan(score) ? score : 0.f) : expf(score - m_new)) : 0.f;
      const float alpha = m_run[u] == -INFINITY ? (l_run[u] == 0.f ? 0.f : 1.f) : expf(m_run[u] - m_new);
      l_run[u] = l_run[u] * alpha + warp_sum(p);
      m_run[u] = m_new;
      p_s[lane * kHeads + h] = p;
      if (lane == 0) alpha_s[h] = alpha;
    }
    __syncthreads();
    fetch(v_pool, false, j0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMaxDim / kAnyThreads; ++i) {
      const int c = tid + i * kAnyThreads;
      if (c >= d) break;
#pragma unroll
      for (int h = 0; h < kHeads; ++h) acc[h][i] *= alpha_s[h];
#pragma unroll 4
      for (int r = 0; r < kAnyKeys; ++r) {
        const float v = tile[r * any_row(d) + c];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) acc[h][i] = fmaf(p_s[r * kHeads + h], v, acc[h][i]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kWarpHeads; ++u)
    if (warp + 4 * u < heads && lane == 0) {
      l_s[warp + 4 * u] = l_run[u];
      if (splits > 1) *reinterpret_cast<float2*>(part_ml + 2 * part_at(warp + 4 * u)) = make_float2(m_run[u], l_run[u]);
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMaxDim / kAnyThreads; ++i) {
    const int c = tid + i * kAnyThreads;
    if (c >= d) break;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (h >= heads) break;
      if (splits > 1) part_o[part_at(h) * d + c] = acc[h][i];
      // no key at all: 0; a sum that is NaN stays one
      else dst[(size_t)h * d + c] = from_float<T>(l_s[h] == 0.f ? 0.f : acc[h][i] / l_s[h]);
    }
  }
}

// grid = (tokens, heads): a head's parts, up to 64 of them, into its output.
template <typename T>
__global__ void __launch_bounds__(kAnyThreads)
attention_any_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, T* __restrict__ out, int out_stride,
                           int n_q, int d, int splits) {
  __shared__ float f_s[64];
  __shared__ float l_s;
  pdl_trigger();
  pdl_wait();
  const size_t base = ((size_t)blockIdx.x * n_q + blockIdx.y) * splits;
  const int tid = threadIdx.x;
  if (tid < 32) {
    float2 v[2];
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] = tid + 32 * i < splits ? *reinterpret_cast<const float2*>(part_ml + 2 * (base + tid + 32 * i)) : make_float2(-INFINITY, 0.f);
    const float top = warp_max(fmaxf(v[0].x, v[1].x));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // a part without a key has no sums (perhaps its outputs were not written); one whose scores are all NaN has sums that are
      f[i] = v[i].x == -INFINITY ? (v[i].y == 0.f ? 0.f : 1.f) : expf(v[i].x - top);
      f_s[tid + 32 * i] = f[i];
    }
    const float sum = warp_sum(fmaf(f[0], v[0].y, f[1] * v[1].y));
    if (tid == 0) l_s = sum;
  }
  __syncthreads();
  for (int c = tid; c < d; c += kAnyThreads) {
    float o = 0.f;
#pragma unroll 16
    for (int s = 0; s < splits; ++s) {
      const float f = f_s[s];
      o = fmaf(f, f != 0.f ? part_o[(base + s) * d + c] : 0.f, o);
    }
    out[(size_t)blockIdx.x * out_stride + (size_t)blockIdx.y * d + c] = from_float<T>(l_s == 0.f ? 0.f : o / l_s);
  }
}

}  // namespace cache4
}  // namespace leone

using namespace leone;

extern "C" void leone_packed_set_pdl(int enabled) { pdl_flag() = enabled ? 1 : 0; }

static bool pool_ok(int d, int n_kv, int page_tokens, int table_width, const void* k_pool, const void* v_pool) {
  return cache4::dim_ok(d) && n_kv > 0 && page_tokens > 0 && page_tokens % cache4::kUnit == 0 && table_width > 0 &&
         k_pool != nullptr && v_pool != nullptr;
}

// Arguments as leone_qk_norm_rope_write, the pools in 4 bits.
extern "C" int leone_append4(int dtype, void* qkv, int n_tokens, int n_q, int n_kv, int d, const void* q_w, const void* k_w,
                             int w_dtype, float eps, const float* rope, int rotary_dim, int max_positions, const int* positions,
                             const int* seq_of_token, const int* block_table, int table_width, int n_seqs, void* k_pool,
                             void* v_pool, int num_pages, int page_tokens, int adjacent, int* status, cudaStream_t stream) {
  if (n_tokens <= 0) return 0;
  if (n_q <= 0 || !pool_ok(d, n_kv, page_tokens, table_width, k_pool, v_pool)) return kRefusedSize;
  if (rope != nullptr && (rotary_dim <= 0 || rotary_dim > d || (rotary_dim & 1))) return kRefusedSize;
  if (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) return kRefusedAlignment;
  // Heads that rotate whole or not at all.  A block has two heads a warp for few tokens, all of a token's heads (up to 48) for many: 200
  // tokens of 48 heads 6.0 us in blocks of 8 heads, 6.3 in blocks of 48; 500 tokens 10.3 and 7.8.
  if ((d == 64 || d == 128) && (rope == nullptr || rotary_dim == d) && (q_w == nullptr) == (k_w == nullptr) && ((uintptr_t)qkv & 15) == 0 &&
      n_q + 2 * n_kv <= 65535) {
    const int heads = n_q + 2 * n_kv, most = n_tokens <= 200 ? 2 * cache4::kAppendWarps : cache4::kAppendHeads;
    const int blocks_of = (heads + most - 1) / most, per = (heads + blocks_of - 1) / blocks_of;
    const dim3 grid(n_tokens, blocks_of);
    const bool few = (long long)n_tokens * blocks_of <= 2 * 148;
    const size_t row_bytes = (size_t)per * d * (dtype == 0 ? 4 : 2);
#define LAUNCH_VEC(T, TW, D)                                                                                                        \
  return launch_kernel(few ? cache4::append_vec_kernel<T, TW, D, true> : cache4::append_vec_kernel<T, TW, D, false>, grid,           \
                       dim3(32 * cache4::kAppendWarps), row_bytes, stream, (T*)qkv, n_q, n_kv, (const TW*)q_w, (const TW*)k_w, eps, \
                       (const float2*)rope, max_positions, positions, seq_of_token, block_table, table_width, n_seqs,               \
                       (uint8_t*)k_pool, (uint8_t*)v_pool, num_pages, page_tokens, adjacent, per, status)
    if (d == 64) {
      if (dtype == 0 && w_dtype == 0) LAUNCH_VEC(float, float, 64);
      if (dtype == 1 && w_dtype == 0) LAUNCH_VEC(__nv_bfloat16, float, 64);
      if (dtype == 0 && w_dtype == 1) LAUNCH_VEC(float, __nv_bfloat16, 64);
      if (dtype == 1 && w_dtype == 1) LAUNCH_VEC(__nv_bfloat16, __nv_bfloat16, 64);
    } else {
      if (dtype == 0 && w_dtype == 0) LAUNCH_VEC(float, float, 128);
      if (dtype == 1 && w_dtype == 0) LAUNCH_VEC(__nv_bfloat16, float, 128);
      if (dtype == 0 && w_dtype == 1) LAUNCH_VEC(float, __nv_bfloat16, 128);
      if (dtype == 1 && w_dtype == 1) LAUNCH_VEC(__nv_bfloat16, __nv_bfloat16, 128);
    }
#undef LAUNCH_VEC
  }
  const int warps = 4;
  const long long blocks = ((long long)n_tokens * (n_q + 2 * n_kv) + warps - 1) / warps;
  if (blocks > 0x7fffffff) return kRefusedSize;
  const size_t smem = (size_t)warps * d * sizeof(double);
#define LAUNCH(T, TW)                                                                                                          \
  return launch_kernel(cache4::append_kernel<T, TW>, dim3((unsigned)blocks), dim3(warps * 32), smem, stream, (T*)qkv, n_tokens, \
                       n_q, n_kv, d, (const TW*)q_w, (const TW*)k_w, eps, (const float2*)rope, rotary_dim, max_positions,       \
                       positions, seq_of_token, block_table, table_width, n_seqs, (uint8_t*)k_pool, (uint8_t*)v_pool,           \
                       num_pages, page_tokens, adjacent, status)
  if (dtype == 0 && w_dtype == 0) LAUNCH(float, float);
  if (dtype == 1 && w_dtype == 0) LAUNCH(__nv_bfloat16, float);
  if (dtype == 0 && w_dtype == 1) LAUNCH(float, __nv_bfloat16);
  if (dtype == 1 && w_dtype == 1) LAUNCH(__nv_bfloat16, __nv_bfloat16);
#undef LAUNCH
  return kRefusedDtype;
}

extern "C" int leone_read4(int dtype, void* k_out, void* v_out, int n_tokens, int n_kv, int d, const int* positions,
                           const int* seq_of_token, const int* block_table, int table_width, int n_seqs, const void* k_pool,
                           const void* v_pool, int num_pages, int page_tokens, int* status, cudaStream_t stream) {
  if (n_tokens <= 0) return 0;
  if (!pool_ok(d, n_kv, page_tokens, table_width, k_pool, v_pool)) return kRefusedSize;
  if (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_out | (uintptr_t)v_out) & 15) return kRefusedAlignment;
  const int blocks = (n_kv + cache4::kReadWarps - 1) / cache4::kReadWarps;
  const dim3 grid(n_tokens, blocks < 65535 ? blocks : 65535);
#define LAUNCH(T)                                                                                                            \
  return launch_kernel(cache4::read_kernel<T>, grid, dim3(32 * cache4::kReadWarps), 0, stream, (T*)k_out, (T*)v_out,         \
                       n_kv, d, positions, seq_of_token, block_table, table_width, n_seqs, (const uint8_t*)k_pool, \
                       (const uint8_t*)v_pool, num_pages, page_tokens, status)
  if (dtype == 0) LAUNCH(float);
  if (dtype == 1) LAUNCH(__nv_bfloat16);
#undef LAUNCH
  return kRefusedDtype;
}

template <typename T, int kHeads>
static int launch_any(const void* qkv, int row_stride, void* out, int out_stride, const void* k_pool, const void* v_pool,
                      const int* block_table, int table_width, const int* seq_of_token, const int* positions, int n_tokens, int n_q,
                      int n_kv, int d, float scale, int window, int page_tokens, int num_pages, int n_seqs, int splits, float* scratch,
                      int* status, cudaStream_t stream) {
  using namespace cache4;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(attention_any_kernel<T, kHeads>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  const long long rows = (long long)n_kv * ((n_q / n_kv + kHeads - 1) / kHeads);
  if (rows > 65535) return kRefusedSize;
  const int smem = (kAnyKeys * any_row(d) + kHeads * (d + kAnyKeys + 2)) * 4;
  float* part_ml = splits > 1 ? scratch + (size_t)n_tokens * n_q * splits * d : nullptr;
  const int e = launch_kernel(attention_any_kernel<T, kHeads>, dim3(n_tokens, (unsigned)rows, splits), dim3(kAnyThreads), smem, stream,
                              (const T*)qkv, row_stride, (T*)out, out_stride, (const uint8_t*)k_pool, (const uint8_t*)v_pool,
                              block_table, table_width, seq_of_token, positions, n_q, n_kv, d, scale, window, page_tokens, num_pages,
                              n_seqs, splits, scratch, part_ml, status);
  if (e != 0 || splits == 1) return e;
  return launch_kernel(attention_any_merge_kernel<T>, dim3(n_tokens, n_q), dim3(kAnyThreads), 0, stream, (const float*)scratch,
                       (const float*)part_ml, (T*)out, out_stride, n_q, d, splits);
}

// Arguments as leone_attention_generic, the pools in 4 bits.  `splits`: blocks that share a token's keys, up to 64; more than one take
// n_tokens n_q splits (d + 2) floats of scratch.
extern "C" int leone_attention4_any(int dtype, const void* qkv, int row_stride, void* out, int out_stride, const void* k_pool,
                                    const void* v_pool, const int* block_table, int table_width, const int* seq_of_token,
                                    const int* positions, int n_tokens, int n_q, int n_kv, int d, float scale, int window,
                                    int page_tokens, int num_pages, int n_seqs, int splits, float* scratch, int* status,
                                    cudaStream_t stream) {
  if (n_tokens <= 0) return 0;
  if (n_q <= 0 || !pool_ok(d, n_kv, page_tokens, table_width, k_pool, v_pool) || n_q % n_kv != 0) return kRefusedSize;
  if (splits < 1 || splits > 64 || (splits > 1) != (scratch != nullptr) || n_q > 65535) return kRefusedSize;
  if (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)scratch) & 15) return kRefusedAlignment;
  const int g = n_q / n_kv;
#define LAUNCH(T, H)                                                                                                             \
  return launch_any<T, H>(qkv, row_stride, out, out_stride, k_pool, v_pool, block_table, table_width, seq_of_token, positions,   \
                          n_tokens, n_q, n_kv, d, scale, window, page_tokens, num_pages, n_seqs, splits, scratch, status, stream)
  if (dtype == 0 && g <= 2) LAUNCH(float, 2);
  if (dtype == 0 && g <= 4) LAUNCH(float, 4);
  if (dtype == 0) LAUNCH(float, 8);
  if (dtype == 1 && g <= 2) LAUNCH(__nv_bfloat16, 2);
  if (dtype == 1 && g <= 4) LAUNCH(__nv_bfloat16, 4);
  if (dtype == 1) LAUNCH(__nv_bfloat16, 8);
#undef LAUNCH
  return kRefusedDtype;
}
