// Product of two microscaled 4-bit matrices on the tensor cores:
//   out[m, n] = g_a g_b sum_k (a s_a)[m, k] (b s_b)[n, k] + bias[n]
// with the codes, block scales and tensor scales of fp4.cuh, fp32
// accumulation and one rounding to the output's type.
//
// One operand gives the rows of a tile (P), the other its columns (Q).
// tcgen05.mma reads codes from shared memory and block scales from tensor
// memory; a stage of the ring holds 256 columns of K: rows of 128 bytes (one
// swizzle atom) and their scale tiles, 512 bytes for 128 rows and four
// blocks, which tcgen05.cp spreads over tensor memory just before the MMAs
// that read them.
//
// Roles (10 warps): warp 0 loads (one thread), warp 1 copies scales and
// issues MMAs, warps 2-9 run the epilogue, each a quarter of the
// tile's rows and half of its columns.
#include <type_traits>

#include "common.h"
#include "fp4.cuh"
#include "gemm_tile.cuh"
#include "ptx.cuh"

namespace dgxm {

constexpr int kGemmRows = 128;
constexpr int kGemmK = 256;               // columns of K a stage: 128 bytes of codes

struct __align__(64) Fp4GemmParams {
  CUtensorMap tmap_p, tmap_q;    // codes: dims (pitch, 1, rows, 1), boxes (128, 1, 128 or TN, 1)
  CUtensorMap tmap_sp, tmap_sq;  // scale tiles of 128 words: dims (128, groups, row tiles)
  CUtensorMap tmap_out;          // where `vec`: dims (n, 1, m, 1), boxes of 128 bytes x 32 rows
  const float* scale_a;          // the tensors' scales, or NULL
  const float* scale_b;
  const void* bias;              // n values of bias_dtype, or NULL
  void* out;
  int64_t ld_out;                // elements
  int p_rows, q_rows, k, k_tiles;
  int p_tiles, q_tiles, split;
  int q_is_tokens;               // P holds the weight's rows: the tile is the output transposed
  int out_dtype, bias_dtype, vec;
};

// A tile of kRows x TN outputs: one CTA's 128 rows, or (PAIR) a CTA pair's 256,
// each CTA loading its own 128 rows of P and its half of Q's rows.
template <int TN, int FORMAT, bool PAIR>
struct Fp4Tile {
  static constexpr int kRows = PAIR ? 2 * kGemmRows : kGemmRows;
  static constexpr int kQLoad = PAIR ? TN / 2 : TN;                // Q rows this CTA loads
  static constexpr int kAtoms = kGemmK / (4 * fp4_block(FORMAT));  // scale tiles of a stage, for 128 rows
  static constexpr int kQTiles = (TN + 127) / 128;                 // 128-row tiles of scales that Q's rows touch
  static constexpr int kPBytes = kGemmRows * 128;
  static constexpr int kQBytes = kQLoad * 128;
  static constexpr int kSfBytes = kAtoms * 512;
  static constexpr int kStageBytes = kPBytes + kQBytes + kSfBytes * (1 + kQTiles);
  // A split tile's partial sums in the CTA that finishes their rows, in the
  // place of the staging rows: (rank, four columns, row), 16 bytes each, an odd
  // number of rows apart (138 at the most for all ranks).
  static constexpr bool kSplits = !PAIR && TN <= 64;
  static constexpr int kPartBytes = kSplits ? (kGemmRows + 10) * TN * 4 : 0;
  static constexpr int kStagingBytes = kPartBytes > 8 * kGemmStageRows ? kPartBytes : 8 * kGemmStageRows;
  static constexpr int kStages = (kGemmSmemMax - 1024 - kGemmCtrlBytes - kStagingBytes) / kStageBytes;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kStagingBytes + kGemmCtrlBytes;
  // Tensor memory: accumulators, then scales, for each stage of the ring P's 4
  // columns and Q's 4 a 128-row tile for four blocks of K.  A copy of scales is
  // ordered before the MMAs that follow it, but not behind earlier ones that
  // read the same columns; those of a stage have completed when the stage is
  // filled again.  The room for that leaves 192 columns one accumulator, which
  // its tiles do not feel, where two, and a wait of the MMA warp's for its fewer
  // columns of scales, cost 5 % (512 x 5120 x 5120: 13.5 us, 14.2).
  static constexpr int kAccs = TN <= 128 ? 2 : 1;
  static constexpr int kSfCol = kAccs * TN, kSfCols = 4 * (1 + kQTiles);
  static_assert(kSfCol + kStages * kAtoms * kSfCols <= 512, "tensor memory");
  static_assert(kStageBytes % 1024 == 0, "swizzle atoms stay aligned");
  // Barriers
  static constexpr int kFull = 0, kEmpty = kStages, kAccFull = 2 * kStages, kAccEmpty = kAccFull + kAccs,
                       kDrain = kAccEmpty + kAccs, kBars = kDrain + 1;
  static_assert(kBars * 8 + 16 <= kGemmCtrlBytes, "control block");
};

// Instruction descriptor of the block-scaled 4-bit kinds: e2m1 operands,
// K-major, K = 64; scale type 0 ue4m3, 1 ue8m0; sf: which bytes of the scale
// words of A and B a K step starts at.
__host__ __device__ constexpr uint32_t fp4_idesc(int m, int n, int format, int sf) {
  return (static_cast<uint32_t>(sf) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         ((format == DGXM_FP4_MXFP4 ? 1u : 0u) << 23) | (static_cast<uint32_t>(m >> 7) << 27) |
         (static_cast<uint32_t>(sf) << 29);
}

// Shared-memory descriptor of a 512-byte scale tile: 32 rows of 16 bytes, no swizzle.
__device__ __forceinline__ uint64_t fp4_sf_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(128 >> 4) << 32) |
         (uint64_t(1) << 46);
}

// Scale tile -> four tensor-memory columns, the same in all four lane
// quarters (PAIR: each CTA's own tile into its own tensor memory).
template <bool PAIR>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (PAIR)
    asm volatile(DGXM_ELECT "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}\n" ::"r"(taddr), "l"(desc)
                 : "memory");
  else
    asm volatile(DGXM_ELECT "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}\n" ::"r"(taddr), "l"(desc)
                 : "memory");
}

#define DGXM_UMMA_FP4(group, kind)                                                                   \
  asm volatile(DGXM_ELECT                                                                             \
               "setp.ne.b32 p, %6, 0;\n\t"                                                           \
               "@q tcgen05.mma." group "." kind " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::            \
               "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) \
               : "memory")

template <int FORMAT, bool PAIR>
__device__ __forceinline__ void umma_fp4_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                            uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (FORMAT == DGXM_FP4_NVFP4) {
    if constexpr (PAIR) DGXM_UMMA_FP4("cta_group::2", "kind::mxf4nvf4.block_scale.scale_vec::4X");
    else DGXM_UMMA_FP4("cta_group::1", "kind::mxf4nvf4.block_scale.scale_vec::4X");
  } else {
    if constexpr (PAIR) DGXM_UMMA_FP4("cta_group::2", "kind::mxf4.block_scale.scale_vec::2X");
    else DGXM_UMMA_FP4("cta_group::1", "kind::mxf4.block_scale.scale_vec::2X");
  }
}

__device__ __forceinline__ float fp4_gemm_bias(const Fp4GemmParams& p, int n) {
  if (p.bias_dtype == DGXM_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
  if (p.bias_dtype == DGXM_DTYPE_F16) return __half2float(static_cast<const __half*>(p.bias)[n]);
  return static_cast<const float*>(p.bias)[n];
}

// A warp's 32 rows x NC columns of finished values (a row a lane) from row
// pr0 and column q0 of the output.
template <int NC, int ELT, typename P>
__device__ __forceinline__ void fp4_store_rows(const P& p, uint8_t* stage, const float (&v)[NC], int pr0,
                                               int q0, int lane) {
  constexpr int kEach = 16 / ELT;  // elements of a piece
  constexpr int kMost = 128 / ELT;
  constexpr int kCols = NC % kMost == 0 ? kMost : NC % (kMost / 2) == 0 ? kMost / 2 : NC;  // columns staged at one time
  static_assert(kCols <= kMost && NC % kCols == 0, "whole chunks");
  constexpr int kPieces = kCols / kEach;
#pragma unroll
  for (int c0 = 0; c0 < NC; c0 += kCols) {
    if (q0 + c0 >= p.q_rows) return;  // uniform over the warp
    if (kCols == kMost && p.vec) {
      if (lane == 0) tma_store_wait_read();  // the last chunk has left the staging rows
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = fp4_piece<ELT>(p, v + c0 + i * kEach);
    fp4_flush_rows<kCols, ELT>(p, stage, pr0, q0 + c0, lane);
  }
}

template <typename T>
__device__ __forceinline__ T fp4_narrow(float v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(v);
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return v;
}

// The finished values of one row of P, where that is a column of the output:
// neighbouring lanes store neighbouring values.
template <typename T, int NC>
__device__ __forceinline__ void fp4_store_column(const Fp4GemmParams& p, const float (&v)[NC], float bias, int n, int q0) {
  T* to = static_cast<T*>(p.out) + q0 * p.ld_out + n;
#pragma unroll
  for (int c = 0; c < NC; ++c, to += p.ld_out)
    if (q0 + c < p.q_rows) *to = fp4_narrow<T>(v[c] + bias);
}

// A split tile: this CTA's share of the rows, `rows` from row pr0, out of the
// partial sums.  A thread takes four columns of one row at a time; its bias
// came before (row j's, where the rows of P are output columns, or column e's).
template <typename T, int TN>
__device__ __forceinline__ void fp4_store_split(const Fp4GemmParams& p, const float* part, int share, int rows, int pr0,
                                                int q0, int thread, float ga, float gb, const float (&bias)[4]) {
  const float4* part4 = reinterpret_cast<const float4*>(part);
  const int pitch = share | 1;
  constexpr int kTimes = kGemmRows / 2 * (TN / 4) / 256 > 1 ? kGemmRows / 2 * (TN / 4) / 256 : 1;
#pragma unroll
  for (int j = 0; j < kTimes; ++j) {
    const int i = thread + 256 * j;
    if (i >= rows * (TN / 4)) return;
    // neighbouring lanes take neighbouring output columns
    const int row = p.q_is_tokens ? i % rows : i / (TN / 4), c = 4 * (p.q_is_tokens ? i / rows : i % (TN / 4));
    const int pr = pr0 + row, q = q0 + c;
    if (pr >= p.p_rows || q >= p.q_rows) continue;
    float4 sum = part4[c / 4 * pitch + row];
    for (int k = 1; k < p.split; ++k) {
      const float4 more = part4[(k * (TN / 4) + c / 4) * pitch + row];
      sum.x += more.x;
      sum.y += more.y;
      sum.z += more.z;
      sum.w += more.w;
    }
    const float v[4] = {sum.x * ga * gb, sum.y * ga * gb, sum.z * ga * gb, sum.w * ga * gb};
    const int64_t step = p.q_is_tokens ? p.ld_out : 1;
    T* to = static_cast<T*>(p.out) + (p.q_is_tokens ? q * p.ld_out + pr : pr * p.ld_out + q);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (q + e < p.q_rows) to[e * step] = fp4_narrow<T>(v[e] + bias[p.q_is_tokens ? j : e]);
  }
}

// One CTA a tile; or `split` CTAs of a cluster sharing a tile's K, each
// finishing a share of its rows: every CTA stores its partial sums into the
// shared memory of the row's owner (stores are not waited for, where loads
// from a peer cost their latency over and over: 1003 x 777 x 1000 took 18 us
// that way), and the owner sums them in rank order, so the result does not
// depend on timing; or PAIR: a CTA pair a tile, the even CTA issuing the
// M256 MMAs of both.
template <int TN, int FORMAT, bool PAIR>
__global__ void __launch_bounds__(kGemmThreads, 1) fp4_gemm_kernel(const __grid_constant__ Fp4GemmParams p) {
  using C = Fp4Tile<TN, FORMAT, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  uint8_t* staging = smem + C::kStages * C::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + C::kStagingBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int cta = PAIR ? rank : 0;
  const int share = PAIR ? 2 : p.split;  // CTAs of a tile
  const int first_tile = blockIdx.x / share, tile_step = gridDim.x / share;
  const int tiles = p.p_tiles * p.q_tiles;
  const int kt0 = PAIR ? 0 : rank * p.k_tiles / p.split;  // this CTA's share of K
  const int kt1 = PAIR ? p.k_tiles : (rank + 1) * p.k_tiles / p.split;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar(C::kFull + s), 1);
      mbar_init(bar(C::kEmpty + s), 1);
    }
    for (int a = 0; a < C::kAccs; ++a) {
      mbar_init(bar(C::kAccFull + a), 1);
      mbar_init(bar(C::kAccEmpty + a), PAIR ? 16 : 8);  // every epilogue warp
    }
    mbar_init(bar(C::kDrain), 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.tmap_p);
    tma_prefetch_desc(&p.tmap_q);
    tma_prefetch_desc(&p.tmap_sp);
    tma_prefetch_desc(&p.tmap_sq);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (PAIR || (C::kSplits && p.split > 1)) cluster_sync();  // the peers' barriers, and their shared memory, are there
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();  // the operands are there

  float ga = 1.f, gb = 1.f, split_bias[4] = {0.f, 0.f, 0.f, 0.f};  // the epilogue's
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < tiles; tile += tile_step) {
        int pt, qt;
        fp4_tile_coords(p, tile, pt, qt);
        for (int kt = kt0; kt < kt1; ++kt, ++it) {
          const int s = it % C::kStages;
          if (!mbar_wait(bar(C::kEmpty + s), ((it / C::kStages) & 1) ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t dst = base + s * C::kStageBytes;
          const uint32_t full = PAIR ? mapa_shared(bar(C::kFull + s), 0) : bar(C::kFull + s);
          if (cta == 0) mbar_expect_tx(bar(C::kFull + s), (PAIR ? 2 : 1) * C::kStageBytes);
          fp4_tma<PAIR>(dst, &p.tmap_p, full, kt * 128, 0, pt * C::kRows + cta * kGemmRows);
          fp4_tma<PAIR>(dst + C::kPBytes, &p.tmap_q, full, kt * 128, 0, qt * TN + cta * C::kQLoad);
          const uint32_t sf = dst + C::kPBytes + C::kQBytes;
          fp4_tma<PAIR>(sf, &p.tmap_sp, full, 0, kt * C::kAtoms, pt * (C::kRows / 128) + cta);
          fp4_tma<PAIR>(sf + C::kSfBytes, &p.tmap_sq, full, 0, kt * C::kAtoms, qt * TN / 128);
        }
      }
      if (!ok) {
        report_device_error(kErrProducerTimeout);
        *abort_flag = 1;
        // Let the loads already issued land before the CTA can exit.
        if (cta == 0) {
          const int first = it > C::kStages ? it - C::kStages : 0;
          for (int i = first; i < it; ++i) mbar_wait(bar(C::kFull + i % C::kStages), (i / C::kStages) & 1, nullptr);
        } else {
          for (int i = 0; i < 50; ++i) __nanosleep(1000);  // the odd CTA cannot test the even one's barriers
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ scales and MMAs
    if (cta == 0) {
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      int s = 0, parity = 0, u = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < tiles; tile += tile_step, ++u) {
        const int a = u % C::kAccs;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(C::kAccEmpty + a), ((u / C::kAccs) & 1) ^ 1, abort_flag)))) break;
        tc_fence_after();
        const uint32_t acc = tm + a * TN;
        int pt, qt;
        fp4_tile_coords(p, tile, pt, qt);
        const uint32_t q_col = qt * TN % 128 / 32;  // 0, or 2 where a tile starts in the middle of a tile of scales
        for (int kt = kt0; kt < kt1; ++kt) {
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(C::kFull + s), parity, abort_flag)))) break;
          tc_fence_after();
          const uint32_t sp = base + s * C::kStageBytes, sq = sp + C::kPBytes, sf = sq + C::kQBytes;
          const uint32_t tsf = tm + C::kSfCol + s * (C::kAtoms * C::kSfCols);
          const uint64_t dp = sdesc_sw128(sp, 16, 1024), dq = sdesc_sw128(sq, 16, 1024), df = fp4_sf_desc(sf);
          // K = 64 an MMA; the rest of the last tile is empty.
          const int steps = min(kGemmK, p.k - kt * kGemmK + 63) / 64;
#pragma unroll
          for (int kk = 0; kk < kGemmK / 64; ++kk) {
            constexpr int kPer = 4 / C::kAtoms;  // MMAs a scale tile serves
            const int i = kk / kPer;
            const uint32_t tp = tsf + i * C::kSfCols, tq = tp + 4;
            if (kk % kPer == 0) {
              tmem_cp_scales<PAIR>(tp, df + 32 * i);
#pragma unroll
              for (int j = 0; j < C::kQTiles; ++j)
                tmem_cp_scales<PAIR>(tq + 4 * j, df + ((1 + j) * C::kSfBytes + 512 * i) / 16);
            }
            if (kk < steps)
              umma_fp4_ss<FORMAT, PAIR>(acc, dp + 2 * kk, dq + 2 * kk,
                                        fp4_idesc(C::kRows, TN, FORMAT, kPer == 1 ? 0 : 2 * (kk % kPer)), tp,
                                        tq + q_col, (kt > kt0 || kk > 0) ? 1u : 0u);
          }
          fp4_commit<PAIR>(bar(C::kEmpty + s));
          if (++s == C::kStages) {
            s = 0;
            parity ^= 1;
          }
        }
        if (ok) fp4_commit<PAIR>(bar(C::kAccFull + a));
      }
      if (!ok) {
        report_device_error(kErrMmaTimeout);
        *abort_flag = 1;
      }
      // Every MMA issued has completed before tensor memory is released.
      fp4_commit<PAIR>(bar(C::kDrain));
      mbar_wait(bar(C::kDrain), 0, nullptr);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;
    constexpr int kCols = TN / 2;  // this warp's columns
    if (p.scale_a != nullptr) ga = *p.scale_a;
    if (p.scale_b != nullptr) gb = *p.scale_b;
    if (const float both = ga * gb; fabsf(both) >= 0x1p-126f && fabsf(both) <= 0x1p126f) {
      ga = 1.f;
      gb = both;
    }
    const uint64_t gab = pk2(gb, gb);
    const uint32_t acc_empty = PAIR ? mapa_shared(bar(C::kAccEmpty), 0) : bar(C::kAccEmpty);
    uint8_t* stage = staging + (warp - 2) * kGemmStageRows;
    int u = 0;
    for (int tile = first_tile; tile < tiles; tile += tile_step, ++u) {
      const int a = u % C::kAccs;
      int pt, qt;
      fp4_tile_coords(p, tile, pt, qt);
      const int pr0 = pt * C::kRows + cta * kGemmRows + quarter * 32;  // this warp's first row
      const int q0 = qt * TN + half * kCols;
      if (C::kSplits && p.split > 1) {
        const int share = (kGemmRows + p.split - 1) / p.split, rows = min(share, kGemmRows - rank * share);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = threadIdx.x - 64 + 256 * j;
          const int n = p.q_is_tokens ? pt * kGemmRows + rank * share + i % rows : qt * TN + 4 * (i % (TN / 4)) + j;
          if (p.bias != nullptr && n < (p.q_is_tokens ? p.p_rows : p.q_rows)) split_bias[j] = fp4_gemm_bias(p, n);
        }
      }
      float bias[(kCols + 31) / 32];  // column 32 i + lane, or (tokens) this lane's row
#pragma unroll
      for (int i = 0; i < (kCols + 31) / 32; ++i) {
        const int n = p.q_is_tokens ? pr0 + lane : q0 + 32 * i + lane;
        bias[i] = p.bias != nullptr && n < (p.q_is_tokens ? p.p_rows : p.q_rows) ? fp4_gemm_bias(p, n) : 0.f;
      }
      const bool got = __all_sync(0xffffffffu, mbar_wait(bar(C::kAccFull + a), (u / C::kAccs) & 1, abort_flag));
      if (!got) {
        report_device_error(kErrEpilogueTimeout);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      uint32_t r[kCols / 8][8];
      const uint32_t from = tmem + lane_off + a * TN + half * kCols;
#pragma unroll
      for (int c = 0; c < kCols / 8; ++c) tmem_ld8(from + 8 * c, r[c]);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < kCols / 8; ++c) reg_fence8(r[c]);
      // The accumulator is in registers: the next tile's MMAs may start.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        // relaxed: the reads of tensor memory are done (wait::ld), and a release
        // would first wait for the last tile's stores
        if constexpr (PAIR) mbar_arrive_cluster_relaxed(acc_empty + a * 8);
        else mbar_arrive(acc_empty + a * 8);
      }
      if (C::kSplits && p.split > 1) {
        const int share = (kGemmRows + p.split - 1) / p.split, pitch = share | 1;
        const uint32_t to = mapa_shared(smem_u32(staging), row / share) +
                            ((rank * (TN / 4) + half * (kCols / 4)) * pitch + row % share) * 16;
#pragma unroll
        for (int c = 0; c < kCols / 4; ++c) st_shared_cluster(to + c * pitch * 16, r[c / 2] + 4 * (c % 2));
        continue;
      }
      float v[kCols];
#pragma unroll
      for (int c = 0; c < kCols; ++c) v[c] = __uint_as_float(r[c / 8][c % 8]);
      if (ga != 1.f) {  // g_a g_b leaves fp32's range: one after the other
#pragma unroll
        for (int c = 0; c < kCols; ++c) v[c] *= ga;
      }
#pragma unroll
      for (int c = 0; c < kCols; c += 2) upk2(fmul2(pk2(v[c], v[c + 1]), gab), v[c], v[c + 1]);
      if (p.q_is_tokens) {  // neighbouring lanes hold neighbouring output columns
        if (const int n = pr0 + lane; n < p.p_rows) {
          if (p.out_dtype == DGXM_DTYPE_BF16) fp4_store_column<__nv_bfloat16>(p, v, bias[0], n, q0);
          else if (p.out_dtype == DGXM_DTYPE_F16) fp4_store_column<__half>(p, v, bias[0], n, q0);
          else fp4_store_column<float>(p, v, bias[0], n, q0);
        }
      } else {
        if (p.bias != nullptr) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) v[c] += __shfl_sync(0xffffffffu, bias[c / 32], c % 32);
        }
        if (p.out_dtype == DGXM_DTYPE_F32) fp4_store_rows<kCols, 4>(p, stage, v, pr0, q0, lane);
        else fp4_store_rows<kCols, 2>(p, stage, v, pr0, q0, lane);
      }
    }
    if (lane == 0) tma_store_wait_all();  // the staging rows outlive the stores
    __syncwarp();
  }
  tc_fence_before();
  if (PAIR || (C::kSplits && p.split > 1)) cluster_sync();  // both CTAs' MMAs drained; or every partial sum is in place
  else __syncthreads();
  if (C::kSplits && p.split > 1 && warp >= 2 && *abort_flag == 0) {
    if constexpr (C::kSplits) {
      const float* part = reinterpret_cast<const float*>(staging);
      int pt, qt;
      fp4_tile_coords(p, first_tile, pt, qt);
      const int share = (kGemmRows + p.split - 1) / p.split, rows = min(share, kGemmRows - rank * share);
      const int pr0 = pt * kGemmRows + rank * share, q0 = qt * TN, thread = threadIdx.x - 64;
      if (p.out_dtype == DGXM_DTYPE_BF16)
        fp4_store_split<__nv_bfloat16, TN>(p, part, share, rows, pr0, q0, thread, ga, gb, split_bias);
      else if (p.out_dtype == DGXM_DTYPE_F16)
        fp4_store_split<__half, TN>(p, part, share, rows, pr0, q0, thread, ga, gb, split_bias);
      else
        fp4_store_split<float, TN>(p, part, share, rows, pr0, q0, thread, ga, gb, split_bias);
    }
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// Packed scales: tiles of 128 words, `groups` of them in a row of tiles; a box
// is one stage's tiles of `tiles` row tiles.
static int fp4_scale_map(CUtensorMap* map, const void* scales, int64_t groups, int64_t row_tiles, int atoms, int tiles) {
  return encode_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, {128, (cuuint64_t)groups, (cuuint64_t)row_tiles},
                 {512, (cuuint64_t)groups * 512}, {128, (cuuint32_t)atoms, (cuuint32_t)tiles}, CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct Fp4Operand {
  const void *values, *scales;
  int64_t rows;
};

template <int TN, int FORMAT, bool PAIR>
static int fp4_gemm_launch(Fp4GemmParams& p, const Fp4Operand& po, const Fp4Operand& qo, cudaStream_t st) {
  using C = Fp4Tile<TN, FORMAT, PAIR>;
  static std::atomic<uint64_t> configured{0};
  DGXM_CUDA_TRY(set_smem_limit_once(fp4_gemm_kernel<TN, FORMAT, PAIR>, C::kSmemBytes, configured));
  const int64_t pitch = fp4_pitch(p.k), groups = fp4_groups(p.k, FORMAT);
  if (int rc = encode_map_4d(&p.tmap_p, po.values, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, pitch, 1, po.rows, 1, pitch, pitch,
                             pitch * po.rows, 128, kGemmRows))
    return rc;
  if (int rc = encode_map_4d(&p.tmap_q, qo.values, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, pitch, 1, qo.rows, 1, pitch, pitch,
                             pitch * qo.rows, 128, C::kQLoad))
    return rc;
  if (int rc = fp4_scale_map(&p.tmap_sp, po.scales, groups, (po.rows + 127) / 128, C::kAtoms, 1)) return rc;
  if (int rc = fp4_scale_map(&p.tmap_sq, qo.scales, groups, (qo.rows + 127) / 128, C::kAtoms, C::kQTiles)) return rc;
  if (p.vec && !p.q_is_tokens) {  // boxes of 128 bytes x 32 rows
    const int elt = p.out_dtype == DGXM_DTYPE_F32 ? 4 : 2;
    const cuuint64_t row = static_cast<cuuint64_t>(p.ld_out) * elt;
    if (int rc = encode_map_3d(&p.tmap_out, elt == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, p.out,
                         {(cuuint64_t)p.q_rows, 1, (cuuint64_t)p.p_rows}, {row, row}, {(cuuint32_t)(128 / elt), 1, 32},
                         CU_TENSOR_MAP_SWIZZLE_128B))
      return rc;
  }
  p.p_tiles = (p.p_rows + C::kRows - 1) / C::kRows;
  p.q_tiles = (p.q_rows + TN - 1) / TN;
  const int tiles = p.p_tiles * p.q_tiles, share = PAIR ? 2 : p.split;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = share;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  // One tile at a time; a split tile's cluster has one tile.
  cfg.gridDim = dim3(PAIR ? 2 * std::min(tiles, 74) : p.split > 1 ? tiles * p.split : std::min(tiles, 148));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  DGXM_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp4_gemm_kernel<TN, FORMAT, PAIR>, p));
  return DGXM_OK;
}

template <int FORMAT>
static int fp4_gemm_pick(Fp4GemmParams& p, const Fp4Operand& po, const Fp4Operand& qo, int tn, cudaStream_t st) {
  switch (tn) {
    case 16: return fp4_gemm_launch<16, FORMAT, false>(p, po, qo, st);
    case 32: return fp4_gemm_launch<32, FORMAT, false>(p, po, qo, st);
    case 64: return fp4_gemm_launch<64, FORMAT, false>(p, po, qo, st);
    case 128: return fp4_gemm_launch<128, FORMAT, false>(p, po, qo, st);
    case 192: return fp4_gemm_launch<192, FORMAT, false>(p, po, qo, st);
    default: return fp4_gemm_launch<256, FORMAT, true>(p, po, qo, st);
  }
}

// How a product is cut: the tile's columns (256: a CTA pair's 256 x 256),
// into how many CTAs its K is split, which operand gives the tile's rows.
struct Fp4Cut {
  int tn, split;
  bool q_is_tokens;
};

// The cut whose waves of tiles take the least time by what one wave took
// (microseconds a stage of K, a tile, and at the least; nvfp4, 9450 x 5120 x
// 256, 1024 and 5120, the narrow ones 1 .. 64 x 2560 .. 13824 x 256 .. 14336):
// narrow tiles where only they fill the SMs or more are not needed (1 x 5120 x
// 1024: 3.7 us with 16 columns, 4.1 with 64), wide ones, which load the least
// for what they compute, where those do too, and K split where even those are
// few (16 x 5120 x 5120: 7.8 and 6.4 us on 1 and 3 CTAs a tile; 16 x 5120 x
// 1024: 3.7 and 4.5).  The sums order the cuts and are not the times of calls:
// launches in a row took 10.1 us where they say 5.8 (65 x 5120 x 5120), 12.0
// for 6.6 (300 rows), 11.8 for 9.5 (512), 17.3 for 19.0 (1024), and 117 for 147
// (40000 x 5120 x 1024).  mxfp4, with half the copies of scales, takes the same
// cuts and 0.1 to 2.4 us less at K = 5120.  A second tile of 16 or 32 columns would begin at an odd
// column of scales in tensor memory, which the MMA cannot address.
static Fp4Cut fp4_cut(int64_t m, int64_t n, int k_tiles) {
  struct Kind {
    int tn, rows, at_once;
    double stage, tile, least;
  };
  static const Kind kinds[] = {{16, 128, 148, 0.26, 0.4, 0.4},  {32, 128, 148, 0.26, 0.5, 0.5},
                               {64, 128, 148, 0.25, 0.8, 1.0},  {128, 128, 148, 0.29, 0.8, 1.1},
                               {192, 128, 148, 0.42, 1.1, 2.2}, {256, 256, 74, 0.42, 1.75, 2.2}};
  // Clusters of a size that the SMs' groups hold at one time.
  static const int clusters[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
  Fp4Cut best{128, 1, false};
  double least = 1e30;
  const bool tokens = m <= n;  // with one tile of columns, the narrow side is Q
  for (const Kind& kind : kinds) {
    const int64_t narrow = m < n ? m : n;
    const bool one = kind.tn <= 64 && narrow <= kind.tn;  // tiles of 16 and 32 columns only as one
    if (kind.tn < 64 && !one) continue;
    const int64_t p_rows = one && tokens ? n : m, q_rows = one && tokens ? m : n;
    const int64_t tiles = (p_rows + kind.rows - 1) / kind.rows * ((q_rows + kind.tn - 1) / kind.tn);
    for (int split = 1; split <= (kind.tn <= 64 ? 8 : 1) && split <= k_tiles; ++split) {
      if (split > 1 && tiles > clusters[split]) continue;
      const int64_t waves = (tiles * split + kind.at_once - 1) / kind.at_once;
      const double us = waves * std::max((k_tiles + split - 1) / split * kind.stage + kind.tile, kind.least) +
                        (split > 1 ? 0.8 + 0.026 * kind.tn : 0.0);  // exchange within the cluster
      if (us < least) {
        least = us;
        best = {kind.tn, split, one && tokens};
      }
    }
  }
  return best;
}

}  // namespace dgxm

extern "C" int dgxm_fp4_matmul(const dgxm_fp4_gemm_desc* d, const void* a_values, const void* a_scales,
                               const float* a_scale, const void* b_values, const void* b_scales, const float* b_scale,
                               const void* bias, void* out, void* stream) {
  using namespace dgxm;
  if (d == nullptr) return fail(DGXM_ERR_INVALID, "NULL 4-bit product descriptor");
  if (d->format != DGXM_FP4_NVFP4 && d->format != DGXM_FP4_MXFP4)
    return fail(DGXM_ERR_UNSUPPORTED, "4-bit format %d (nvfp4 or mxfp4)", d->format);
  if (d->m < 0 || d->n < 0 || d->k <= 0 || d->m > (1 << 30) || d->n > (1 << 30))
    return fail(DGXM_ERR_INVALID, "product of (%lld, %lld) and (%lld, %lld)", (long long)d->m, (long long)d->k,
                (long long)d->n, (long long)d->k);
  // One tile's K takes 0.5 us a stage at the most: 33 ms here, well within the bounded waits' second.
  if (d->k > (1 << 24)) return fail(DGXM_ERR_UNSUPPORTED, "k %lld above 2^24", (long long)d->k);
  for (int t : {d->out_dtype, d->bias_dtype})
    if (t != DGXM_DTYPE_BF16 && t != DGXM_DTYPE_F16 && t != DGXM_DTYPE_F32)
      return fail(DGXM_ERR_UNSUPPORTED, "output or bias dtype %d (bf16, f16 or f32)", t);
  if (d->out_stride < d->n) return fail(DGXM_ERR_INVALID, "output row stride %lld below %lld columns",
                                        (long long)d->out_stride, (long long)d->n);
  if (d->m == 0 || d->n == 0) return DGXM_OK;
  const bool nv = d->format == DGXM_FP4_NVFP4;
  if (a_values == nullptr || a_scales == nullptr || b_values == nullptr || b_scales == nullptr || out == nullptr)
    return fail(DGXM_ERR_INVALID, "NULL operand or output");
  if (nv != (a_scale != nullptr) || nv != (b_scale != nullptr))
    return fail(DGXM_ERR_INVALID, "nvfp4 takes both tensors' fp32 scales, mxfp4 none");
  if ((reinterpret_cast<uintptr_t>(a_values) | reinterpret_cast<uintptr_t>(a_scales) |
       reinterpret_cast<uintptr_t>(b_values) | reinterpret_cast<uintptr_t>(b_scales)) % 16)
    return fail(DGXM_ERR_INVALID, "values and scales must be 16-byte aligned");
  const int out_elt = d->out_dtype == DGXM_DTYPE_F32 ? 4 : 2, bias_elt = d->bias_dtype == DGXM_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(out) % out_elt || reinterpret_cast<uintptr_t>(bias) % bias_elt ||
      (reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale)) % 4)
    return fail(DGXM_ERR_INVALID, "output, bias or scale is not aligned to its elements");
  const int64_t m = d->m, n = d->n;
  if ((m + 127) / 128 * ((n + 127) / 128) > (1 << 26)) return fail(DGXM_ERR_UNSUPPORTED, "too many output tiles");
  Fp4GemmParams p;
  memset(&p, 0, sizeof(p));
  p.k = static_cast<int>(d->k);
  p.k_tiles = static_cast<int>((d->k + kGemmK - 1) / kGemmK);
  const Fp4Cut cut = fp4_cut(m, n, p.k_tiles);
  p.q_is_tokens = cut.q_is_tokens;
  p.split = cut.split;
  p.p_rows = static_cast<int>(p.q_is_tokens ? n : m);
  p.q_rows = static_cast<int>(p.q_is_tokens ? m : n);
  const Fp4Operand a{a_values, a_scales, m}, b{b_values, b_scales, n};
  const Fp4Operand &po = p.q_is_tokens ? b : a, &qo = p.q_is_tokens ? a : b;
  p.scale_a = a_scale;
  p.scale_b = b_scale;
  p.bias = bias;
  p.out = out;
  p.ld_out = d->out_stride;
  p.out_dtype = d->out_dtype;
  p.bias_dtype = d->bias_dtype;
  p.vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && d->out_stride * out_elt % 16 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return nv ? fp4_gemm_pick<DGXM_FP4_NVFP4>(p, po, qo, cut.tn, st) : fp4_gemm_pick<DGXM_FP4_MXFP4>(p, po, qo, cut.tn, st);
}
