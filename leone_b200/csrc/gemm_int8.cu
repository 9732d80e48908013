// out[M,N] = x[M,K] * w[N,K]^T of 8-bit integers for few tokens: a stream over the weights.
//
// The swapped form of gemm_tc.cu for `kind::i8`: a tile of 128 weight rows rides the MMA's M side, up to 32 tokens its N side, a k-block is
// 128 integers.  One tile a block, two blocks an SM.  Where the tiles are fewer than the SMs' places, the `splits` blocks of a
// thread-block cluster share a tile's k-blocks; each pushes its int32 sums into the shared memory of the block that finishes the rows
// (chunks of 32 rows, chunk c belongs to rank c % splits), and after one cluster barrier the owners add them, exactly, and run the
// epilogue: float(sum) * w_scale[n] * x_scale[m], bias, then bf16, fp32, fp32 + residual, or the gate.
//
// Warp 0 loads (the weights of the first stages before it waits for the kernel before this one, which rounds the tokens), warp 1 issues
// tcgen05.mma, warps 2-5 finish.  Every wait is bounded.
#include "gemm_parts.cuh"

namespace leone {
namespace tc {

constexpr int kStreamThreads = 192;
constexpr int kStreamMaxStages = 8;
constexpr int kStreamK = 2 * kTileK;                       // integers of a k-block: 128 bytes
constexpr int kStreamTokens = 32;                          // the MMA's N
constexpr int kStreamABytes = kTileW * kStreamK, kStreamStage = kStreamABytes + kStreamTokens * kStreamK;
constexpr int kStreamLimit = 227 * 1024 / 2 - 1536;        // (the static part and what the system takes of each block)
// Slots of 32 rows that a block's inbox needs: one for every (chunk it owns, rank).
__host__ __device__ inline int stream_slots(int splits) { return splits > 1 ? (4 + splits - 1) / splits * splits : 0; }
__host__ __device__ inline int stream_columns(int m) { return (m + 7) / 8 * 8; }

__global__ void __launch_bounds__(kStreamThreads, 2)
gemm_int8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const GemmParams p,
                        const int stages) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  const uint32_t full0 = tiles + stages * kStreamStage, empty0 = full0 + 8 * kStreamMaxStages, acc_full = empty0 + 8 * kStreamMaxStages;
  int* inbox = reinterpret_cast<int*>(smem_raw + (acc_full + 16 - raw));               // [slot][column][row of the chunk]
  __shared__ uint32_t tmem_holder;
  __shared__ int gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.splits, rank = S > 1 ? (int)cluster_ctarank() : 0, tile = blockIdx.x / S;
  const int all = (p.K + kStreamK - 1) / kStreamK, share = (all + S - 1) / S;
  const int kb0 = min(all, rank * share), kb1 = min(all, kb0 + share);                  // (perhaps none)
  const int columns = stream_columns(p.M);

  if (threadIdx.x == 0) {
    gave_up = 0;
    for (int s = 0; s < stages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(acc_full, 1);
    mbar_fence_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_holder), kStreamTokens);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  volatile int* giveup = &gave_up;
  pdl_trigger();
  if (S > 1) cluster_arrive_relaxed();                     // this block runs; waited for before another writes into its inbox

  if (warp == 0) {
    if (elect_one()) {
      auto load_w = [&](int kb, int s) {
        mbar_expect_tx(full0 + 8 * s, kStreamStage);
        tma_load_2d(tiles + s * kStreamStage, &map_w, full0 + 8 * s, kb * kStreamK, tile * kTileW);
      };
      auto load_x = [&](int kb, int s) {
        tma_load_2d(tiles + s * kStreamStage + kStreamABytes, &map_x, full0 + 8 * s, kb * kStreamK, 0);
      };
      const int early = min(stages, kb1 - kb0);
      for (int i = 0; i < early; ++i) load_w(kb0 + i, i);
      for (int i = 0; i < p.l2_ahead && kb0 + early + i < kb1; ++i) tma_prefetch_2d(&map_w, (kb0 + early + i) * kStreamK, tile * kTileW);
      pdl_wait();
      for (int i = 0; i < early; ++i) load_x(kb0 + i, i);
      int s = 0;
      uint32_t phase = 0;
      for (int kb = kb0 + early; kb < kb1; ++kb) {
        if (!mbar_wait(empty0 + 8 * s, phase, giveup)) break;
        load_w(kb, s);
        load_x(kb, s);
        if (++s == stages) {
          s = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = instr_desc_i8(kTileW, kStreamTokens);
      int s = 0, kb = kb0;
      uint32_t phase = 0;
      for (; kb < kb1; ++kb) {
        if (!mbar_wait(full0 + 8 * s, phase, giveup)) break;
        const uint32_t a = desc_low(tiles + s * kStreamStage);
        umma_k128_i8(tmem, a, a + (kStreamABytes >> 4), idesc, kb > kb0 ? 1u : 0u);
        umma_commit(empty0 + 8 * s);
        if (++s == stages) {
          s = 0;
          phase ^= 1;
        }
      }
      if (kb == kb1) umma_commit(acc_full);                // (at once where this block has no k-blocks)
    }
  } else {
    const int quarter = warp & 3;
    const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16);
    pdl_wait();                                            // outputs, residual and the tokens' scales
    const bool ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, giveup));
    tc_fence_after();
    if (ok && S == 1) {
      const int n = tile * kTileW + quarter * 32 + lane;
      const float scale = n < p.N ? p.col_scale[n] : 0.f;
      for (int c = 0; c < columns; c += 8) {
        float r[8], v[8];
        fetch_residual<8>(p, r, n, 0, c);
        uint32_t sum[8];
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(sum[0]), "=r"(sum[1]), "=r"(sum[2]), "=r"(sum[3]), "=r"(sum[4]), "=r"(sum[5]), "=r"(sum[6]), "=r"(sum[7])
                     : "r"(taddr + c) : "memory");
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)(int)sum[j] * scale * (c + j < p.M ? p.row_scale[c + j] : 0.f);
        finish_swapped<8>(p, v, r, n, 0, c, lane, nullptr);
      }
    } else if (ok) {
      // a thread's row of sums goes to the block that finishes its chunk, slot (chunk / S, this block's rank)
      const uint32_t slot = smem_u32(inbox) + (uint32_t)((((quarter / S) * S + rank) * columns) * 32 + lane) * 4;
      const uint32_t dst = cluster_map(slot, (uint32_t)(quarter % S));
      cluster_wait();
      for (int c = 0; c < columns; c += 8) {
        uint32_t sum[8];
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(sum[0]), "=r"(sum[1]), "=r"(sum[2]), "=r"(sum[3]), "=r"(sum[4]), "=r"(sum[5]), "=r"(sum[6]), "=r"(sum[7])
                     : "r"(taddr + c) : "memory");
        tmem_ld_wait();
        // (a share without k-blocks has no sums)
#pragma unroll
        for (int j = 0; j < 8; ++j) cluster_st_f32(dst + (uint32_t)(c + j) * 128, __uint_as_float(kb0 < kb1 ? sum[j] : 0u));
      }
    } else if (S > 1) {
      cluster_wait();
    }
  }

  if (S > 1) {
    // Every thread of every block of the cluster comes here (all loops above are bounded).
    if (warp < 2) cluster_wait();
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2 && !*giveup) {
      for (int ch = rank; ch < kTileW / 32; ch += S) {
        const int n = tile * kTileW + ch * 32 + lane;
        const float scale = n < p.N ? p.col_scale[n] : 0.f;
        const int* mine = inbox + (size_t)((ch / S) * S) * columns * 32 + lane;
        for (int c = (warp - 2) * 2; c < p.M; c += 8) {
          float r[2], v[2];
          fetch_residual<2>(p, r, n, 0, c);
          int sum[2] = {0, 0};
          for (int s = 0; s < S; ++s) {
            sum[0] += mine[(s * columns + c) * 32];
            sum[1] += mine[(s * columns + c + 1) * 32];
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) v[j] = (float)sum[j] * scale * (c + j < p.M ? p.row_scale[c + j] : 0.f);
          finish_swapped<2>(p, v, r, n, 0, c, lane, nullptr);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (gave_up) {
    if (threadIdx.x == 0) set_status(p.status, kWaitTimeout, blockIdx.x, 8);
    // let tile copies that are still in flight land before the block's memory goes away
    const long long start = clock64();
    while (clock64() - start < 200000) {}
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kStreamTokens);
  }
}

static int launch_stream(const CUtensorMap& mw, const CUtensorMap& mx, const GemmParams& p, cudaStream_t stream) {
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(gemm_int8_stream_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamLimit);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  const int other = 1024 + 16 * kStreamMaxStages + 16 + stream_slots(p.splits) * stream_columns(p.M) * 128;
  const int k_blocks = (p.K + kStreamK - 1) / kStreamK, most = (k_blocks + p.splits - 1) / p.splits;
  int stages = (kStreamLimit - other) / kStreamStage;
  if (stages > kStreamMaxStages) stages = kStreamMaxStages;
  if (stages > most) stages = most;
  const size_t smem = (size_t)other + (size_t)stages * kStreamStage;
  const dim3 grid((unsigned)((p.N + kTileW - 1) / kTileW * p.splits));
  if (p.splits == 1)
    return launch_kernel(gemm_int8_stream_kernel, grid, dim3(kStreamThreads), smem, stream, mw, mx, p, stages);
  return launch_kernel_cluster(gemm_int8_stream_kernel, grid, dim3(kStreamThreads), smem, stream, dim3((unsigned)p.splits), mw, mx, p,
                               stages);
}

}  // namespace tc
}  // namespace leone

using namespace leone;
using namespace leone::tc;

// Arguments as leone_gemm_narrow_i8 (gemm_narrow.cu), up to 32 tokens; `splits`: blocks that share a tile's k-blocks, 1 to 8.
extern "C" int leone_gemm_stream_i8(const void* x, const float* x_scale, const void* w, const float* w_scale, void* out,
                                    const float* residual, int m, int n, int k, int ldx, int ldw, int ldc, int epilogue, int splits,
                                    int* status, const float* gate_shape, const float* bias, cudaStream_t stream) {
  if (m <= 0 || n <= 0) return 0;
  if (k <= 0 || (k % 16) != 0 || (ldx % 16) != 0 || (ldw % 16) != 0) return kRefusedAlignment;
  if (m > kStreamTokens || epilogue < 0 || epilogue > 3 || splits < 1 || splits > 8) return kRefusedSize;
  if ((epilogue == 2 && residual == nullptr) || (epilogue == 3 && (n % 32) != 0) || x_scale == nullptr || w_scale == nullptr)
    return kRefusedSize;
  CUtensorMap mw, mx;
  int r = make_tensor_map_2d_i8(&mw, w, (uint64_t)n, (uint64_t)k, (uint64_t)ldw, kTileW);
  if (r != 0) return r;
  r = make_tensor_map_2d_i8(&mx, x, (uint64_t)m, (uint64_t)k, (uint64_t)ldx, kStreamTokens);
  if (r != 0) return r;
  GemmParams p{out, residual, m, n, k, ldc, epilogue, splits, 0, nullptr, nullptr, status, nullptr,
               nullptr, nullptr, nullptr, 0, nullptr, 0, 0.f, 8};
  set_gate_shape(p, gate_shape);
  p.bias = bias;
  p.row_scale = x_scale;
  p.col_scale = w_scale;
  return launch_stream(mw, mx, p, stream);
}

extern "C" int leone_quantize_rows(int dtype, const void* x, int m, int k, int ldx, void* codes, float* scales, cudaStream_t stream);
extern "C" int leone_gemm_narrow_i8(const void*, const float*, const void*, const float*, void*, const float*, int, int, int, int, int,
                                    int, int, int, int*, int, const float*, const float*, cudaStream_t);
extern "C" int leone_gemm_pair_i8(const void*, const float*, const void*, const float*, void*, const float*, int, int, int, int, int, int,
                                  int, int, int*, int, const float*, const float*, cudaStream_t);

// Tokens x [m, k] (dtype 0 fp32, 1 bfloat16) rounded to `codes` [m, k] and `scales` [m], and their product with w: form 0 the stream
// (`shape`: splits), 1 narrow tiles, 2 pairs of SMs (`shape`: weight rows of a tile).
extern "C" int leone_linear_i8(int dtype, const void* x, int ldx, void* codes, float* scales, const void* w, const float* w_scale, void* out,
                               const float* residual, int m, int n, int k, int ldc, int epilogue, int form, int shape, int* status,
                               int sm_count, const float* gate_shape, const float* bias, cudaStream_t stream) {
  if (form < 0 || form > 2) return kRefusedSize;
  const int e = leone_quantize_rows(dtype, x, m, k, ldx, codes, scales, stream);
  if (e != 0) return e;
  if (form == 0)
    return leone_gemm_stream_i8(codes, scales, w, w_scale, out, residual, m, n, k, k, k, ldc, epilogue, shape, status, gate_shape, bias,
                                stream);
  return (form == 1 ? leone_gemm_narrow_i8 : leone_gemm_pair_i8)(codes, scales, w, w_scale, out, residual, m, n, k, k, k, ldc, epilogue,
                                                                 shape, status, sm_count, gate_shape, bias, stream);
}
