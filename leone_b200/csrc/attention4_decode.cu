// Decode attention over pages in 4 bits (cache4.cuh): sequences with one query token each, head sizes 64 and 128, bfloat16 queries.
//
// Formulas as in attention_tiled.cu: kv_head = q_head / (n_q / n_kv); score = (q.k) * scale; online softmax in fp32; output = numerator
// / sum (crates/leone/src/cpu.rs:2299-2421).  A key is k = z + s c per group of 64 elements, so with codes c as the MMA's operand
//   q.k = sum over groups  s (q.c) + z sum(q)           and          sum_j p_j v_j = sum_j (p_j s_j) c_j + sum_j p_j z_j:
// nothing is multiplied per element.  P_j = p_j s_j is rounded to bfloat16; as
//   out = sum_j P_j c_j - 8 sum_j P_j + sum_j p_j (z_j + 8 s_j)
// its rounding weighs c_j - 8 only: half a step of at most 8 s, what a bfloat16 value would lose itself.  sum_j P_j is an MMA with ones.
//
// A code becomes a bfloat16 by one AND: as a bit pattern the integers 0 .. 255 are the numbers n 2^-133 (the subnormal ones and those of
// the smallest exponent have one step), so of a word a code in bits 0-3 is c 2^-133, one in bits 4-7 is 16 c 2^-133.  Queries
// are multiplied by 2^48 before (those that meet bits 4-7 by 2^44) and weights by 2^62, so that the sums lie in the middle of fp32's range,
// and the sums by 2^85 and 2^71 after; all are exact while queries stay below 2^79, scales of keys below 2^40 and scales of values between 2^-62
// and 2^57.  (128 + c by AND-OR, which needs
// a shift for every code but a word's first and the 128 taken out again, took 425 instructions for 16 keys of 128 where this takes 296.)
//
// Keys ride the MMA's M side and up to 8 query heads its N side (NT tiles of them), as in attention_tiled.cu.  The pages' layout is
// made so that a thread's operands are words that lie side by side: 16 keys are one piece of 1,152 bytes (576 with 64 elements) for
// keys and one for values, each fetched by one untiled copy of the TMA into a ring of kStages parts of kPart units that every warp
// has of its own, and read from there with 16- and 8-byte loads without bank conflicts.
//
// A block is 4 warps for one (sequence, cached head, up to 16 of its query heads, split of the keys); its warps take units in turn.
// Splits of up to 8 merge inside a thread-block cluster through distributed shared memory, more through scratch and a kernel.
//
// 32 query heads on 8 of 128, one call behind another: 166 sequences of 2,048 keys 87 us (4.5 TB/s of the copy's 6.5), 64 of them 45 us (512
// blocks where 444 run at once), 64 of up to 2,048 30 us, one of 40,960 19.4 us (2.4 TB/s).  Memory does not bound it: with every page in the
// L2 166 sequences take 92 us where they take 96 from memory.  Nor does a pipe: at 168 registers a thread 12 warps an SM, 2.5 a scheduler, find
// an instruction to issue in 48 % of the cycles (fixed latencies first, then memory, then the ALUs that mask codes, 46 % busy), so the
// chains of a part's instructions are what the time goes by, and their number.  Of 296 instructions for 16 keys the scores take 74, the
// outputs 105, maximum, weights and the ring 80.
// Slower or no faster: four blocks an SM with parts of two (64 sequences 41 us, of up to 2,048 34, one of 40,960 23), parts of one, keys
// dealt to warps as one line of all sequences, blocks that sort the sequences by length themselves.
#include "cache4.cuh"
#include "tc_common.cuh"

namespace leone {
namespace cache4 {

using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::mbar_wait;
using tc::smem_u32;

constexpr int kDecodeWarps = 4;
constexpr int kDecodeThreads = 32 * kDecodeWarps;
constexpr int kPart = 3;                    // units that a warp takes at once: their chains of instructions overlap
constexpr int kStages = 2;                  // parts in flight (parts of 2 with 3 in flight: 166 sequences of 2,048 keys 88.2 us, 86.7 so)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleAt = 8.f;          // the running maximum moves when a score exceeds it by this (log2): weights stay below 2^8

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {          // an 8x8 tile of 16-bit values across the warp
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// Loads of a stage: after the wait for it and before the next request into it, which are volatile too; free to move among the rest.
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;           // codes as c 2^-133 and as 16 c 2^-133
constexpr uint32_t kMinus8 = 0x80088008u;                              // -8 2^-133, twice
constexpr float kUp = 281474976710656.f;                              // 2^48
constexpr float kBack = 38685626227668133590597632.f;                 // 2^85
constexpr float kWeightUp = 4611686018427387904.f;                    // 2^62 (times weights of up to 2^8 and a scale of 2^57: a bfloat16)
constexpr float kWeightBack = 2361183241434822606848.f;               // 2^71
// Two bfloat16 times 2^48 and, where the word's codes of bits 4-7 meet them, times 2^44.
__device__ __forceinline__ uint32_t raised(uint32_t q, float by) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(q << 16) * by, __uint_as_float(q & 0xffff0000u) * by);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// One warp's running state over its units.  Lane = 4 * gid + tig; of every 16 x 8 accumulator a thread holds rows gid and gid + 8 and
// columns (heads) 2 tig, 2 tig + 1.
template <int D, int NT>
struct Warp4 {
  static constexpr int G = D / 64;
  static constexpr int kUnitBytes = kUnit * row_bytes(D);
  static constexpr int kScales = kUnit * (D / 2);
  uint32_t qb[G][NT][8];             // [pair of a word's 4][..]: queries of head gid, elements 64 g + 16 tig ..
  float qsum[G][NT][2];              // sums of the queries' group, times scale * log2 e
  float m_run[NT][2], limit[NT][2], l_run[NT][2], corr[G][NT][2];   // limit: scores past the maximum that move it; corr: sum p (z + 8 s)
  float base[NT][2];                 // minus the maximum, 0 before the first key: scores are taken relative to it
  float psum[G][NT][4];              // -8 sum P, as o (every row the same)
  float o[G][4][NT][4];              // O^T: rows = elements 64 g + 8 gid + 2 j (gid + 8: + 1)

  __device__ __forceinline__ void init(const __nv_bfloat16* q, int heads, float sl2, int lane) {
    const int gid = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + gid;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (h < heads) {
          const uint4* src = reinterpret_cast<const uint4*>(q + (size_t)h * D + 64 * g + 16 * tig);
          a = src[0];
          b = src[1];
        }
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          qb[g][nt][i] = raised(w[i], i & 1 ? kUp / 16 : kUp);         // odd pairs of a word are those in bits 4-7 and 12-15
          sum += __uint_as_float(w[i] << 16) + __uint_as_float(w[i] & 0xffff0000u);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);            // the whole group's, of head gid
        qsum[g][nt][0] = __shfl_sync(0xffffffffu, sum, 8 * tig) * sl2;
        qsum[g][nt][1] = __shfl_sync(0xffffffffu, sum, 8 * tig + 4) * sl2;
        corr[g][nt][0] = corr[g][nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          psum[g][nt][i] = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[g][j][nt][i] = 0.f;
        }
      }
      m_run[nt][0] = m_run[nt][1] = limit[nt][0] = limit[nt][1] = -INFINITY;
      base[nt][0] = base[nt][1] = l_run[nt][0] = l_run[nt][1] = 0.f;
    }
  }

  // The keys' words of a unit are multiplied with the queries: st = base + (its scores of keys gid and gid + 8) * scale * log2 e.
  __device__ __forceinline__ void scores(uint32_t k_s, float (&st)[NT][4], float back, int gid, int tig) {
    uint32_t w0[2 * G], w1[2 * G], p0[G], p1[G];
    const uint32_t at = k_s + gid * (D / 2) + tig * (8 * G);
    if constexpr (G == 2) {
      const uint4 a = lds128(at), b = lds128(at + 8 * (D / 2));
      w0[0] = a.x; w0[1] = a.y; w0[2] = a.z; w0[3] = a.w;
      w1[0] = b.x; w1[1] = b.y; w1[2] = b.z; w1[3] = b.w;
      const uint2 c = lds64(k_s + kScales + gid * 8);
      const uint2 d = lds64(k_s + kScales + gid * 8 + 64);
      p0[0] = c.x; p0[1] = c.y;
      p1[0] = d.x; p1[1] = d.y;
    } else {
      const uint2 a = lds64(at), b = lds64(at + 8 * (D / 2));
      w0[0] = a.x; w0[1] = a.y;
      w1[0] = b.x; w1[1] = b.y;
      p0[0] = lds32(k_s + kScales + gid * 4);
      p1[0] = lds32(k_s + kScales + gid * 4 + 32);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const uint32_t x = w0[2 * g + b] >> (8 * jj), y = w1[2 * g + b] >> (8 * jj);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_16816(acc[nt], x & kLow, y & kLow, x & kHigh, y & kHigh, qb[g][nt][4 * b + 2 * jj], qb[g][nt][4 * b + 2 * jj + 1]);
        }
      }
      const float z0 = offset_of(p0[g]), z1 = offset_of(p1[g]);
      const float f0 = scale_of(p0[g]) * back, f1 = scale_of(p1[g]) * back;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        st[nt][0] = fmaf(f0, acc[nt][0], fmaf(z0, qsum[g][nt][0], g == 0 ? base[nt][0] : st[nt][0]));
        st[nt][1] = fmaf(f0, acc[nt][1], fmaf(z0, qsum[g][nt][1], g == 0 ? base[nt][1] : st[nt][1]));
        st[nt][2] = fmaf(f1, acc[nt][2], fmaf(z1, qsum[g][nt][0], g == 0 ? base[nt][0] : st[nt][2]));
        st[nt][3] = fmaf(f1, acc[nt][3], fmaf(z1, qsum[g][nt][1], g == 0 ? base[nt][1] : st[nt][3]));
      }
    }
  }

  // A unit's values times the weights p of keys gid and gid + 8 join the outputs; keep0, keep1: whether those keys are seen.
  template <bool kWhole>
  __device__ __forceinline__ void outputs(uint32_t v_s, const float (&p)[NT][4], bool keep0, bool keep1, int gid, int tig) {
    uint2 v[4];
    uint32_t q0[G], q1[G];
    if constexpr (G == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = tig + 4 * i;
        v[i] = lds64(v_s + row * 64 + ((gid * 8) ^ (((row >> 1) & 1) << 5)));
      }
      const uint2 c = lds64(v_s + kScales + gid * 8);
      const uint2 d = lds64(v_s + kScales + gid * 8 + 64);
      q0[0] = c.x; q0[1] = c.y;
      q1[0] = d.x; q1[1] = d.y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i].x = lds32(v_s + (tig + 4 * i) * 32 + gid * 4);
      q0[0] = lds32(v_s + kScales + gid * 4);
      q1[0] = lds32(v_s + kScales + gid * 4 + 32);
    }
    if constexpr (!kWhole) {
#pragma unroll
      for (int g = 0; g < G; ++g) {                          // what stands in a row that is not seen may be anything, NaN too
        if (!keep0) q0[g] = 0;
        if (!keep1) q1[g] = 0;
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float s0 = scale_of(q0[g]), s1 = scale_of(q1[g]);
      const float z0 = fmaf(8.f, s0, offset_of(q0[g])), z1 = fmaf(8.f, s1, offset_of(q1[g]));
      const float r0 = s0 * kWeightUp, r1 = s1 * kWeightUp;
      uint32_t b[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(p[nt][0] * r0, p[nt][1] * r0);
        const __nv_bfloat162 hi = __floats2bfloat162_rn(p[nt][2] * r1, p[nt][3] * r1);
        corr[g][nt][0] = fmaf(p[nt][0], z0, fmaf(p[nt][2], z1, corr[g][nt][0]));
        corr[g][nt][1] = fmaf(p[nt][1], z0, fmaf(p[nt][3], z1, corr[g][nt][1]));
        b[nt][0] = transposed(*reinterpret_cast<const uint32_t*>(&lo));
        b[nt][1] = transposed(*reinterpret_cast<const uint32_t*>(&hi));
        mma_16816(psum[g][nt], kMinus8, kMinus8, kMinus8, kMinus8, b[nt][0], b[nt][1]);
      }
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = g == 0 ? v[i].x : v[i].y;
      // keys 2 tig, 2 tig + 1 and 2 tig + 8, 2 tig + 9 side by side: elements 2 j in x, 2 j + 1 in y
      uint32_t x01 = __byte_perm(w[0], w[1], 0x5410), y01 = __byte_perm(w[0], w[1], 0x7632);
      uint32_t x23 = __byte_perm(w[2], w[3], 0x5410), y23 = __byte_perm(w[2], w[3], 0x7632);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816(o[g][j][nt], x01 & kLow, y01 & kLow, x23 & kLow, y23 & kLow, b[nt][0], b[nt][1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_16816(o[g][j + 1][nt], x01 & kHigh, y01 & kHigh, x23 & kHigh, y23 & kHigh, b[nt][0], b[nt][1]);
        x01 >>= 8; y01 >>= 8; x23 >>= 8; y23 >>= 8;
      }
    }
  }

  // kPart units (a part of a stage: keys, then values) from position key0 on; keys in [k_lo, k_end) are seen but for units whose bit
  // of `gone` is set.  back: scale * log2 e * 2^85
  template <bool kWhole>
  __device__ __forceinline__ void part(uint32_t at, int key0, int k_lo, int k_end, unsigned gone, float back, int lane) {
    const int gid = lane >> 2, tig = lane & 3;
    float p[kPart][NT][4];
#pragma unroll
    for (int u = 0; u < kPart; ++u) scores(at + 2 * u * kUnitBytes, p[u], back, gid, tig);
    bool keep[kPart][2];
#pragma unroll
    for (int u = 0; u < kPart; ++u) keep[u][0] = keep[u][1] = true;
    if constexpr (!kWhole) {
#pragma unroll
      for (int u = 0; u < kPart; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = key0 + u * kUnit + gid + 8 * r;
          keep[u][r] = key >= k_lo && key < k_end && !(gone >> u & 1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            if (!keep[u][r]) p[u][nt][2 * r] = p[u][nt][2 * r + 1] = -INFINITY;
        }
    }
    float top[NT][2];
    bool moves = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[nt][h] = fmaxf(p[0][nt][h], p[0][nt][2 + h]);
#pragma unroll
        for (int u = 1; u < kPart; ++u) top[nt][h] = fmaxf(top[nt][h], fmaxf(p[u][nt][h], p[u][nt][2 + h]));
        moves |= top[nt][h] > limit[nt][h];
      }
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float t = top[nt][h];
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
          const float m_new = fmaxf(m_run[nt][h], t - base[nt][h]);
          if (m_run[nt][h] != -INFINITY && m_new > m_run[nt][h]) {        // (nothing is summed before the first key)
            const float alpha = ex2(m_run[nt][h] - m_new);
            l_run[nt][h] *= alpha;
#pragma unroll
            for (int g = 0; g < G; ++g) {
              corr[g][nt][h] *= alpha;
              psum[g][nt][h] *= alpha;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                o[g][j][nt][h] *= alpha;
                o[g][j][nt][2 + h] *= alpha;
              }
            }
          }
          m_run[nt][h] = m_new;
          const float to = m_new == -INFINITY ? 0.f : -m_new;
#pragma unroll
          for (int u = 0; u < kPart; ++u) {
            p[u][nt][h] += to - base[nt][h];
            p[u][nt][2 + h] += to - base[nt][h];
          }
          base[nt][h] = to;
          limit[nt][h] = m_new == -INFINITY ? -INFINITY : kRescaleAt;
        }
    }
#pragma unroll
    for (int u = 0; u < kPart; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[u][nt][i] = ex2(p[u][nt][i]);
        l_run[nt][0] += p[u][nt][0] + p[u][nt][2];
        l_run[nt][1] += p[u][nt][1] + p[u][nt][3];
      }
#pragma unroll
    for (int u = 0; u < kPart; ++u) outputs<kWhole>(at + (2 * u + 1) * kUnitBytes, p[u], keep[u][0], keep[u][1], gid, tig);
  }

  // This warp's (max, sum, unnormalised output) per head into mo [warps][8 NT][D] and ml [warps][8 NT][2].
  __device__ __forceinline__ void stash(float* mo, float* ml, int warp, int lane) {
    const int gid = lane >> 2, tig = lane & 3;
    auto over_rows = [](float v) {
      v += __shfl_xor_sync(0xffffffffu, v, 4);
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      return v + __shfl_xor_sync(0xffffffffu, v, 16);
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = warp * 8 * NT + nt * 8 + tig * 2 + h;
        const float l = over_rows(l_run[nt][h]);
        if (gid == 0) {
          ml[r * 2] = m_run[nt][h];
          ml[r * 2 + 1] = l;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float c = fmaf(psum[g][nt][h], kWeightBack, over_rows(corr[g][nt][h]));
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float2*>(mo + (size_t)r * D + 64 * g + 8 * gid + 2 * j) =
                make_float2(fmaf(o[g][j][nt][h], j & 1 ? kWeightBack / 16 : kWeightBack, c),
                            fmaf(o[g][j][nt][2 + h], j & 1 ? kWeightBack / 16 : kWeightBack, c));
        }
      }
  }
};

struct Pages {
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const int* block_table;
  int table_width, page_tokens, num_pages, n_kv;
};

template <int D, int NT> struct DecodeSmem {
  static constexpr int kUnitBytes = kUnit * row_bytes(D);
  static constexpr int kRing = kDecodeWarps * kStages * kPart * 2 * kUnitBytes;
  static constexpr int kRows = 8 * NT;
  static constexpr int kMerge = kDecodeWarps * kRows * (D + 2) * 4;
  static constexpr int kFirst = kRing > kMerge ? kRing : kMerge;              // the merge buffer lies over the rings
  static constexpr int kInbox = (kRows * D + 4 * 8 + 8 * kRows * 2) * 4;      // [splits][per] outputs, [splits][rows][2]
  static constexpr int kBytes = kFirst + kInbox + kDecodeWarps * kStages * 8;
};

template <int D, int NT>
__global__ void __launch_bounds__(kDecodeThreads, NT == 1 ? 3 : 2)
attention4_decode_kernel(const __nv_bfloat16* __restrict__ qkv, int row_stride, __nv_bfloat16* __restrict__ out, int out_stride,
                         Pages pa, const int* __restrict__ q_start, const int* __restrict__ ctx_len, int n_q, float scale, int window,
                         int splits, int in_cluster, const int* __restrict__ order, float* __restrict__ part_o,
                         float* __restrict__ part_ml, int* status) {
  using Smem = DecodeSmem<D, NT>;
  constexpr int kUnitBytes = Smem::kUnitBytes, kRows = Smem::kRows, kPartBytes = 2 * kPart * kUnitBytes;
  extern __shared__ __align__(128) uint8_t smem[];
  float* inbox_o = reinterpret_cast<float*>(smem + Smem::kFirst);
  float* inbox_ml = inbox_o + kRows * D + 4 * 8;
  __shared__ int gave_up;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring = smem_u32(smem) + warp * kStages * kPartBytes;
  const uint32_t bars = smem_u32(smem) + Smem::kFirst + Smem::kInbox + warp * kStages * 8;
  if (tid == 0) gave_up = 0;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(bars + 8 * s, 1);
    tc::mbar_fence_init();
  }
  pdl_trigger();
  if (in_cluster) cluster_arrive_relaxed();              // this block runs; waited for before another writes into its inbox
  __syncthreads();
  volatile int* giveup = &gave_up;

  const int g = n_q / pa.n_kv, groups_of = (g + 15) / 16;
  const int kvh = blockIdx.x / groups_of, hg = blockIdx.x - kvh * groups_of;
  const int head0 = kvh * g + hg * 16, heads = min(16, g - hg * 16);
  const int split = blockIdx.y;
  pdl_wait();
  const int seq = order != nullptr ? order[blockIdx.z] : blockIdx.z;
  const int row_token = q_start[seq];
  const int ctx = ctx_len[seq];
  const int k_lo = window > 0 ? max(0, ctx - window) : 0;
  const int first = k_lo / kUnit, total = (ctx + kUnit - 1) / kUnit - first;
  const int share = ((total + splits - 1) / splits + kPart - 1) / kPart * kPart;
  const int u0 = first + split * share, u1 = min(first + total, u0 + share);
  const int parts = u1 > u0 ? (u1 - u0 + kPart - 1) / kPart : 0;
  const int mine = (parts - warp + kDecodeWarps - 1) / kDecodeWarps;       // this warp's parts are warp, warp + 4, ..

  Warp4<D, NT> state;
  const float sl2 = scale * kLog2e, back = sl2 * kBack;
  const int* table = pa.block_table + (size_t)seq * pa.table_width;
  // where the units of the warp's parts i .. i + 32 / kPart - 1 lie in the pools, one a lane (-1: no page; the step fails by its status)
  auto places_from = [&](int i) {
    const int u = u0 + kPart * (warp + kDecodeWarps * (i + lane / kPart)) + lane % kPart;
    long long at = -1;
    if (u < u1) {
      const int blk = u * kUnit / pa.page_tokens;
      const int page = blk < pa.table_width ? table[blk] : -1;
      if (page < 0 || page >= pa.num_pages) set_status(status, kBadPage, row_token, page, u * kUnit);
      else at = unit_at(page, pa.n_kv, kvh, pa.page_tokens, u * kUnit - blk * pa.page_tokens, D);
    }
    return at;
  };
  long long places = places_from(0);
  unsigned gone = 0;                                       // bit kPart * stage + u: unit u of the stage's part has no page, or is past the last
  // Requests part i into its stage; the warp goes on together.
  auto request = [&](int i) {
    if (i >= mine) return;
    if (i > 0 && i % (32 / kPart) == 0) places = places_from(i);
    const int stage = i % kStages;
    const uint32_t bar = bars + 8 * stage, dst = ring + stage * kPartBytes;
    long long at[kPart];
    unsigned none = 0;
#pragma unroll
    for (int u = 0; u < kPart; ++u) {
      at[u] = __shfl_sync(0xffffffffu, places, i % (32 / kPart) * kPart + u);
      if (at[u] < 0) none |= 1u << u;
    }
    gone = (gone & ~(((1u << kPart) - 1) << (kPart * stage))) | none << (kPart * stage);
    if (lane == 0) {
      mbar_expect_tx(bar, (kPart - __popc(none)) * 2 * kUnitBytes);
#pragma unroll
      for (int u = 0; u < kPart; ++u) {
        if (at[u] < 0) continue;
        tc::bulk_load(dst + 2 * u * kUnitBytes, pa.k_pool + at[u], kUnitBytes, bar);
        tc::bulk_load(dst + (2 * u + 1) * kUnitBytes, pa.v_pool + at[u], kUnitBytes, bar);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) request(i);
  state.init(qkv + (size_t)row_token * row_stride + (size_t)head0 * D, heads, sl2, lane);
  int stage = 0;
  unsigned phase = 0;
  for (int i = 0; i < mine; ++i) {
    if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * stage, phase, giveup))) break;
    const uint32_t at = ring + stage * kPartBytes;
    const int key0 = (u0 + kPart * (warp + kDecodeWarps * i)) * kUnit;
    const unsigned lost = gone >> (kPart * stage) & ((1u << kPart) - 1);
    if (key0 >= k_lo && key0 + kPart * kUnit <= ctx && lost == 0) state.template part<true>(at, key0, k_lo, ctx, lost, back, lane);
    else state.template part<false>(at, key0, k_lo, ctx, lost, back, lane);
    __syncwarp();                                          // everyone has read the stage that the next request refills
    request(i + kStages);
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  __syncthreads();                                         // every warp is done with its ring: the merge buffer lies there
  if (gave_up) {
    if (tid == 0) set_status(status, kWaitTimeout, blockIdx.x, 7);
    const long long start = clock64();                     // copies that are still in flight land first
    while (clock64() - start < 200000) {}
    __syncthreads();
  }

  // the warps -> one (max, sum, output) per head of the block
  float* mo = reinterpret_cast<float*>(smem);              // [warps][kRows][D]
  float* ml = mo + kDecodeWarps * kRows * D;               // [warps][kRows][2]
  state.stash(mo, ml, warp, lane);
  __syncthreads();
  const int n_out = heads * D;
  // in a cluster block s finishes outputs [s per, s per + per): all store their parts of that range into its inbox
  const int per = ((n_out + splits - 1) / splits + 3) / 4 * 4;
  if (in_cluster) cluster_wait();
  for (int idx = tid * 4; idx < n_out; idx += kDecodeThreads * 4) {
    const int r = idx / D, c = idx - r * D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) m = fmaxf(m, ml[(w * kRows + r) * 2]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      const float mw = ml[(w * kRows + r) * 2];
      // a warp without a key has no sums; one whose scores are all NaN has sums that are, and no maximum
      const float f = mw == -INFINITY ? 1.f : ex2(mw - m);
      const float4 ow = *reinterpret_cast<const float4*>(mo + (size_t)(w * kRows + r) * D + c);
      l = fmaf(f, ml[(w * kRows + r) * 2 + 1], l);
      o.x = fmaf(f, ow.x, o.x);
      o.y = fmaf(f, ow.y, o.y);
      o.z = fmaf(f, ow.z, o.z);
      o.w = fmaf(f, ow.w, o.w);
    }
    if (in_cluster) {
      const int owner = idx / per;
      cluster_st_f32x4(cluster_map(smem_u32(inbox_o) + (uint32_t)(split * per + idx - owner * per) * 4, owner), o.x, o.y, o.z, o.w);
      if (c == 0)
        for (int s = 0; s < splits; ++s)
          cluster_st_f32x2(cluster_map(smem_u32(inbox_ml) + (uint32_t)(split * kRows + r) * 8, s), m, l);
    } else if (splits > 1) {
      const size_t p = ((size_t)seq * n_q + head0 + r) * splits + split;
      *reinterpret_cast<float4*>(part_o + p * D + c) = o;
      if (c == 0) *reinterpret_cast<float2*>(part_ml + p * 2) = make_float2(m, l);
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(out + (size_t)row_token * out_stride + (size_t)(head0 + r) * D + c);
      dst[0] = __floats2bfloat162_rn(o.x * inv, o.y * inv);
      dst[1] = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    }
  }
  if (!in_cluster) return;

  cluster_arrive_release();                                // every thread of every block of the cluster comes here
  cluster_wait_acquire();
  const int end = min(n_out, split * per + per) - split * per;
  for (int j = tid * 2; j < end; j += kDecodeThreads * 2) {
    const int idx = split * per + j, r = idx / D;
    float m = -INFINITY;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, inbox_ml[(s * kRows + r) * 2]);
    float l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float ms = inbox_ml[(s * kRows + r) * 2];
      const float f = ms == -INFINITY ? 1.f : ex2(ms - m);
      const float2 os = *reinterpret_cast<const float2*>(inbox_o + s * per + j);
      l = fmaf(f, inbox_ml[(s * kRows + r) * 2 + 1], l);
      o0 = fmaf(f, os.x, o0);
      o1 = fmaf(f, os.y, o1);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<__nv_bfloat162*>(out + (size_t)row_token * out_stride + (size_t)head0 * D + idx) =
        __floats2bfloat162_rn(o0 * inv, o1 * inv);
  }
}

constexpr int kMergeWays = 4;
constexpr int merge_ways(int splits) { return splits > 8 ? kMergeWays : 1; }
// The parts of more splits than a cluster holds, and those of prompt portions.  grid = (sequences or tokens, heads), merge_ways(splits)
// threads for two columns (one sequence of 40,960 keys in 37 splits: 21.7 us with four, 25.2 with one, which fetches 8 parts at a time);
// rows: where a sequence's row of the output is, or null for token i in row i.
__global__ void attention4_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                        __nv_bfloat16* __restrict__ out, int out_stride, const int* __restrict__ rows, int n_q, int d,
                                        int splits) {
  __shared__ float f_s[64];
  __shared__ float l_s;
  __shared__ float2 o_s[kMergeWays][64];
  pdl_trigger();
  pdl_wait();
  const int head = blockIdx.y, seq = blockIdx.x, tid = threadIdx.x;
  const size_t base = ((size_t)seq * n_q + head) * splits;
  if (tid < 32) {
    float m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = tid + 32 * i;
      const float2 v = s < splits ? *reinterpret_cast<const float2*>(part_ml + (base + s) * 2) : make_float2(-INFINITY, 0.f);
      m[i] = v.x;
      l[i] = v.y;
    }
    const float top = warp_max(fmaxf(m[0], m[1]));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // a part without a key has no outputs (perhaps none were written); one whose scores are all NaN has a sum that is
      const float f = m[i] == -INFINITY ? (l[i] == 0.f ? 0.f : 1.f) : ex2(m[i] - top);
      f_s[tid + 32 * i] = f;
      sum = fmaf(f, l[i], sum);
    }
    sum = warp_sum(sum);
    if (tid == 0) l_s = sum;
  }
  __syncthreads();
  // `ways` threads share two columns: 64 splits are 16 loads a thread, all in flight at once
  const int ways = blockDim.x / (d / 2), way = tid / (d / 2), c = (tid - way * (d / 2)) * 2;
  float o0 = 0.f, o1 = 0.f;
#pragma unroll 16
  for (int s = way; s < splits; s += ways) {
    const float f = f_s[s];
    float2 v = make_float2(0.f, 0.f);
    if (f != 0.f) v = *reinterpret_cast<const float2*>(part_o + (base + s) * d + c);
    o0 = fmaf(f, v.x, o0);
    o1 = fmaf(f, v.y, o1);
  }
  if (ways > 1) {
    o_s[way][c / 2] = make_float2(o0, o1);
    __syncthreads();
    if (way != 0) return;
    for (int w = 1; w < ways; ++w) {
      o0 += o_s[w][c / 2].x;
      o1 += o_s[w][c / 2].y;
    }
  }
  const float inv = l_s == 0.f ? 0.f : 1.f / l_s;
  *reinterpret_cast<__nv_bfloat162*>(out + (size_t)(rows == nullptr ? seq : rows[seq]) * out_stride + (size_t)head * d + c) =
      __floats2bfloat162_rn(o0 * inv, o1 * inv);
}

template <int D, int NT> int configure_decode() {
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(attention4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         DecodeSmem<D, NT>::kBytes);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  return 0;
}
template <int D, int NT>
int launch_decode(const __nv_bfloat16* qkv, int row_stride, __nv_bfloat16* out, int out_stride, const Pages& pa, const int* q_start,
                  const int* ctx_len, int n_seqs, int n_q, float scale, int window, int splits, int in_cluster, const int* order,
                  float* scratch, int* status, cudaStream_t stream) {
  const int r = configure_decode<D, NT>();
  if (r != 0) return r;
  const dim3 grid(pa.n_kv * ((n_q / pa.n_kv + 15) / 16), splits, n_seqs);
  float* part_ml = scratch == nullptr ? nullptr : scratch + (size_t)n_seqs * n_q * splits * D;
  if (in_cluster)
    return launch_kernel_cluster(attention4_decode_kernel<D, NT>, grid, dim3(kDecodeThreads), DecodeSmem<D, NT>::kBytes, stream,
                                 dim3(1, splits, 1), qkv, row_stride, out, out_stride, pa, q_start, ctx_len, n_q, scale, window,
                                 splits, 1, order, scratch, part_ml, status);
  const int e = launch_kernel(attention4_decode_kernel<D, NT>, grid, dim3(kDecodeThreads), DecodeSmem<D, NT>::kBytes, stream, qkv,
                              row_stride, out, out_stride, pa, q_start, ctx_len, n_q, scale, window, splits, 0, order, scratch,
                              part_ml, status);
  if (e != 0 || splits == 1) return e;
  return launch_kernel(attention4_merge_kernel, dim3(n_seqs, n_q), dim3(D / 2 * merge_ways(splits)), 0, stream, (const float*)scratch,
                       (const float*)part_ml, out, out_stride, q_start, n_q, D, splits);
}

}  // namespace cache4
}  // namespace leone

using namespace leone;

// One query token a sequence (row q_start[s] of qkv).  `splits`: blocks that share a sequence's keys, up to 8 with in_cluster, up to 64
// with scratch of n_seqs n_q splits (d + 2) floats; `order`: the sequences in the order in which their blocks start, or null.
extern "C" int leone_attention4_decode(const void* qkv, int row_stride, void* out, int out_stride, const void* k_pool,
                                       const void* v_pool, const int* block_table, int table_width, const int* q_start,
                                       const int* ctx_len, int n_seqs, int n_q, int n_kv, int d, float scale, int window,
                                       int page_tokens, int num_pages, int splits, int in_cluster, const int* order, float* scratch,
                                       int* status, cudaStream_t stream) {
  if (n_seqs <= 0) return 0;
  if ((d != 64 && d != 128) || n_q <= 0 || n_kv <= 0 || n_q % n_kv != 0 || n_seqs > 65535 || n_q > 65535) return kRefusedSize;
  if (page_tokens <= 0 || page_tokens % cache4::kUnit != 0 || table_width <= 0 || window < 0) return kRefusedSize;
  if (splits < 1 || splits > 64 || (in_cluster && (splits < 2 || splits > 8)) || (!in_cluster && splits > 1 && scratch == nullptr))
    return kRefusedSize;
  if (row_stride % 8 != 0 || out_stride % 2 != 0) return kRefusedAlignment;
  if (((uintptr_t)qkv | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)scratch) & 15 || ((uintptr_t)out & 3))
    return kRefusedAlignment;
  const cache4::Pages pa{(const uint8_t*)k_pool, (const uint8_t*)v_pool, block_table, table_width, page_tokens, num_pages, n_kv};
  const bool wide = n_q / n_kv > 8;
#define LAUNCH(D, NT)                                                                                                              \
  return cache4::launch_decode<D, NT>((const __nv_bfloat16*)qkv, row_stride, (__nv_bfloat16*)out, out_stride, pa, q_start, ctx_len, \
                                      n_seqs, n_q, scale, window, splits, in_cluster, order, scratch, status, stream)
  if (d == 64) {
    if (wide) LAUNCH(64, 2);
    LAUNCH(64, 1);
  }
  if (wide) LAUNCH(128, 2);
  LAUNCH(128, 1);
#undef LAUNCH
}

// What leone_attention4_prefill left in scratch becomes the output's rows 0 .. n_tokens - 1.
extern "C" int leone_attention4_merge(const float* part_o, const float* part_ml, void* out, int out_stride, int n_tokens, int n_q, int d,
                                      int splits, cudaStream_t stream) {
  if (n_tokens <= 0) return 0;
  if ((d != 64 && d != 128) || n_q <= 0 || n_q > 65535 || splits < 1 || splits > 64) return kRefusedSize;
  if (out_stride % 2 != 0 || ((uintptr_t)out & 3) || ((uintptr_t)part_o | (uintptr_t)part_ml) & 15) return kRefusedAlignment;
  return launch_kernel(cache4::attention4_merge_kernel, dim3(n_tokens, n_q), dim3(d / 2 * cache4::merge_ways(splits)), 0, stream, part_o, part_ml,
                       (__nv_bfloat16*)out, out_stride, (const int*)nullptr, n_q, d, splits);
}
