// Product of two microscaled 4-bit matrices on the tensor cores:
//   out[m, n] = g_a g_b sum_k (a s_a)[m, k] (b s_b)[n, k] + bias[n]
// with the codes, block scales and tensor scales of fp4.cuh, fp32
// accumulation and one rounding to the output's type.
//
// One operand gives the 128 rows of a tile (P), the other its TN columns (Q).
// tcgen05.mma reads codes from shared memory and block scales from tensor
// memory; a stage of the ring holds 256 columns of K: 128 + TN rows of 128
// bytes (one swizzle atom) and their scale tiles, 512 bytes for 128 rows and
// four blocks, which tcgen05.cp spreads over tensor memory just before the
// MMAs that read them.
//
// Roles (10 warps): warp 0 loads (one thread), warp 1 copies scales and
// issues MMAs (one thread), warps 2-9 run the epilogue, each a quarter of the
// tile's rows and half of its columns.
//
// A tile whose K is split runs as a cluster of `split` CTAs; each leaves its
// partial tile in its own shared memory and sums its share of the columns
// over the cluster in rank order, so the result does not depend on timing.
#include "common.h"
#include "fp4.cuh"
#include "ptx.cuh"

namespace dgxm {

constexpr int kGemmThreads = 10 * 32;
constexpr int kGemmRows = 128;
constexpr int kGemmK = 256;               // columns of K a stage: 128 bytes of codes
constexpr int kGemmSmemMax = 227 * 1024;
constexpr int kGemmCtrlBytes = 512;

struct __align__(64) Fp4GemmParams {
  CUtensorMap tmap_p, tmap_q;  // codes: dims (pitch, 1, rows, 1), boxes (128, 1, 128 or TN, 1)
  const uint8_t* sf_p;
  const uint8_t* sf_q;
  const float* scale_a;        // the tensors' scales, or NULL
  const float* scale_b;
  const void* bias;            // n values of bias_dtype, or NULL
  void* out;
  int64_t ld_out;              // elements
  int64_t groups;              // scale tiles in a row of tiles
  int p_rows, q_rows, k, k_tiles;
  int p_tiles, q_tiles, split;
  int q_is_tokens;             // P holds the weight's rows: the tile is the output transposed
  int out_dtype, bias_dtype, vec;
};

template <int TN, int FORMAT>
struct Fp4Tile {
  static constexpr int kAtoms = kGemmK / (4 * fp4_block(FORMAT));  // scale tiles of a stage, for 128 rows
  static constexpr int kQTiles = (TN + 127) / 128;                 // 128-row tiles of scales on the Q side
  static constexpr int kPBytes = kGemmRows * 128;
  static constexpr int kQBytes = TN * 128;
  static constexpr int kSfBytes = kAtoms * 512;
  static constexpr int kStageBytes = kPBytes + kQBytes + kSfBytes * (1 + kQTiles);
  static constexpr int kStages = (kGemmSmemMax - 1024 - kGemmCtrlBytes) / kStageBytes;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kGemmCtrlBytes;
  // Tensor memory: accumulators, then two buffers of scales (P's 4 columns a
  // tile, Q's 4 columns a tile and 128 rows).
  static constexpr int kAccs = TN <= 128 ? 2 : 1;
  static constexpr int kSfP = 4 * kAtoms, kSfQ = 4 * kAtoms * kQTiles;
  static constexpr int kSfCol = kAccs * TN;
  static_assert(kSfCol + 2 * (kSfP + kSfQ) <= 512, "tensor memory");
  static_assert(TN * kGemmRows * 4 <= kStages * kStageBytes, "a partial tile fits the ring");
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

// Scale tile -> four tensor-memory columns, the same in all four lane quarters.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

template <int FORMAT>
__device__ __forceinline__ void umma_fp4_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (FORMAT == DGXM_FP4_NVFP4)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// `bytes` (a multiple of 16) global -> this CTA's shared memory, counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ float ld_shared_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float fp4_gemm_bias(const Fp4GemmParams& p, int n) {
  if (p.bias_dtype == DGXM_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
  if (p.bias_dtype == DGXM_DTYPE_F16) return __half2float(static_cast<const __half*>(p.bias)[n]);
  return static_cast<const float*>(p.bias)[n];
}

__device__ __forceinline__ void fp4_gemm_store(const Fp4GemmParams& p, int64_t at, float v) {
  if (p.out_dtype == DGXM_DTYPE_BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
  else if (p.out_dtype == DGXM_DTYPE_F16) static_cast<__half*>(p.out)[at] = __float2half_rn(v);
  else static_cast<float*>(p.out)[at] = v;
}

// N accumulators (N <= 8) of one P row, columns q .. q + N - 1 of Q, finished and stored.
template <int N>
__device__ __forceinline__ void fp4_gemm_emit(const Fp4GemmParams& p, int pr, int q, float (&v)[N], float ga, float gb) {
  if (pr >= p.p_rows || q >= p.q_rows) return;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = v[i] * ga * gb;
  if (p.q_is_tokens) {  // neighbouring lanes hold neighbouring output columns
    const float b = p.bias != nullptr ? fp4_gemm_bias(p, pr) : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (q + i < p.q_rows) fp4_gemm_store(p, (q + i) * p.ld_out + pr, v[i] + b);
    return;
  }
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (q + i < p.q_rows) v[i] += fp4_gemm_bias(p, q + i);
  }
  const int64_t at = pr * p.ld_out + q;
  if constexpr (N == 8) {
    if (p.vec && q + 8 <= p.q_rows) {
      if (p.out_dtype == DGXM_DTYPE_F32) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else if (p.out_dtype == DGXM_DTYPE_BF16) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + at) =
            make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
      } else {
        *reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + at) =
            make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (q + i < p.q_rows) fp4_gemm_store(p, at + i, v[i]);
}

// Tiles run in groups of eight P tiles, Q outermost within a group, so that
// the CTAs resident at one time share a few panels of both operands.
__device__ __forceinline__ void fp4_tile_coords(const Fp4GemmParams& p, int tile, int& pt, int& qt) {
  const int per_group = 8 * p.q_tiles;
  const int g = tile / per_group, r = tile - g * per_group;
  const int rows = min(8, p.p_tiles - g * 8);
  pt = g * 8 + r % rows;
  qt = r / rows;
}

template <int TN, int FORMAT>
__global__ void __launch_bounds__(kGemmThreads, 1) fp4_gemm_kernel(const __grid_constant__ Fp4GemmParams p) {
  using C = Fp4Tile<TN, FORMAT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStageBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int first_tile = blockIdx.x / p.split, tile_step = gridDim.x / p.split;
  const int tiles = p.p_tiles * p.q_tiles;
  const int kt0 = rank * p.k_tiles / p.split, kt1 = (rank + 1) * p.k_tiles / p.split;  // this CTA's share of K

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar(C::kFull + s), 1);
      mbar_init(bar(C::kEmpty + s), 1);
    }
    for (int a = 0; a < C::kAccs; ++a) {
      mbar_init(bar(C::kAccFull + a), 1);
      mbar_init(bar(C::kAccEmpty + a), 8);  // every epilogue warp
    }
    mbar_init(bar(C::kDrain), 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.tmap_p);
    tma_prefetch_desc(&p.tmap_q);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

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
          const uint32_t dst = base + s * C::kStageBytes, full = bar(C::kFull + s);
          const int64_t left = p.groups - int64_t(kt) * C::kAtoms;
          const uint32_t sf_bytes = static_cast<uint32_t>(left < C::kAtoms ? left : C::kAtoms) * 512;
          const int q_sf = qt * TN / 128;  // first 128-row tile of Q's scales
          const bool second = C::kQTiles == 2 && (q_sf + 1) * 128 < p.q_rows;
          mbar_expect_tx(full, C::kPBytes + C::kQBytes + sf_bytes * (second ? 3 : 2));
          tma_load_4d(dst, &p.tmap_p, full, kt * 128, 0, pt * kGemmRows, 0);
          tma_load_4d(dst + C::kPBytes, &p.tmap_q, full, kt * 128, 0, qt * TN, 0);
          const uint32_t sf = dst + C::kPBytes + C::kQBytes;
          bulk_load(sf, p.sf_p + (pt * p.groups + int64_t(kt) * C::kAtoms) * 512, sf_bytes, full);
          bulk_load(sf + C::kSfBytes, p.sf_q + (q_sf * p.groups + int64_t(kt) * C::kAtoms) * 512, sf_bytes, full);
          if (second)
            bulk_load(sf + 2 * C::kSfBytes, p.sf_q + ((q_sf + 1) * p.groups + int64_t(kt) * C::kAtoms) * 512, sf_bytes,
                      full);
        }
      }
      if (!ok) {
        report_device_error(kErrProducerTimeout);
        *abort_flag = 1;
      }
      // Every load issued lands before the CTA can exit.
      const int first = it > C::kStages ? it - C::kStages : 0;
      for (int i = first; i < it; ++i) mbar_wait(bar(C::kFull + i % C::kStages), (i / C::kStages) & 1, nullptr);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ scales and MMAs
    if (lane == 0) {
      int it = 0, u = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < tiles; tile += tile_step, ++u) {
        const int a = u % C::kAccs;
        if (!(ok = mbar_wait(bar(C::kAccEmpty + a), ((u / C::kAccs) & 1) ^ 1, abort_flag))) break;
        tc_fence_after();
        const uint32_t acc = tmem + a * TN;
        for (int kt = kt0; kt < kt1; ++kt, ++it) {
          const int s = it % C::kStages;
          if (!(ok = mbar_wait(bar(C::kFull + s), (it / C::kStages) & 1, abort_flag))) break;
          tc_fence_after();
          const uint32_t sp = base + s * C::kStageBytes, sq = sp + C::kPBytes, sf = sq + C::kQBytes;
          const uint32_t tp = tmem + C::kSfCol + (it & 1) * (C::kSfP + C::kSfQ), tq = tp + C::kSfP;
          const int steps = min(kGemmK, p.k - kt * kGemmK + 63) / 64;  // K = 64 each; the rest of the last tile is empty
#pragma unroll
          for (int i = 0; i < C::kAtoms; ++i) {
            tmem_cp_scales(tp + 4 * i, fp4_sf_desc(sf + 512 * i));
#pragma unroll
            for (int j = 0; j < C::kQTiles; ++j)
              tmem_cp_scales(tq + 4 * (C::kQTiles * i + j), fp4_sf_desc(sf + (1 + j) * C::kSfBytes + 512 * i));
          }
          for (int kk = 0; kk < steps; ++kk) {
            const int i = FORMAT == DGXM_FP4_NVFP4 ? kk : kk >> 1;
            const uint32_t idesc = FORMAT == DGXM_FP4_NVFP4 || (kk & 1) == 0 ? fp4_idesc(kGemmRows, TN, FORMAT, 0)
                                                                            : fp4_idesc(kGemmRows, TN, FORMAT, 2);
            umma_fp4_ss<FORMAT>(acc, sdesc_sw128(sp + kk * 32, 16, 1024), sdesc_sw128(sq + kk * 32, 16, 1024), idesc,
                                tp + 4 * i, tq + 4 * C::kQTiles * i, (kt > kt0 || kk > 0) ? 1u : 0u);
          }
          umma_commit(bar(C::kEmpty + s));
        }
        if (ok) umma_commit(bar(C::kAccFull + a));
      }
      if (!ok) {
        report_device_error(kErrMmaTimeout);
        *abort_flag = 1;
      }
      umma_commit(bar(C::kDrain));
      mbar_wait(bar(C::kDrain), 0, nullptr);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;
    constexpr int kCols = TN / 2;  // this warp's columns
    const float ga = p.scale_a != nullptr ? *p.scale_a : 1.f, gb = p.scale_b != nullptr ? *p.scale_b : 1.f;
    int u = 0;
    for (int tile = first_tile; tile < tiles; tile += tile_step, ++u) {
      const int a = u % C::kAccs;
      int pt, qt;
      fp4_tile_coords(p, tile, pt, qt);
      const bool got = __all_sync(0xffffffffu, mbar_wait(bar(C::kAccFull + a), (u / C::kAccs) & 1, abort_flag));
      if (!got) {
        report_device_error(kErrEpilogueTimeout);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      uint32_t v[kCols / 8][8];
      const uint32_t from = tmem + lane_off + a * TN + half * kCols;
#pragma unroll
      for (int c = 0; c < kCols / 8; ++c) tmem_ld8(from + 8 * c, v[c]);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < kCols / 8; ++c) reg_fence8(v[c]);
      // The accumulator is in registers: the next tile's MMAs may start.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::kAccEmpty + a));
      if (p.split == 1) {
#pragma unroll
        for (int c = 0; c < kCols / 8; ++c) {
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[c][i]);
          fp4_gemm_emit<8>(p, pt * kGemmRows + row, qt * TN + half * kCols + 8 * c, f, ga, gb);
        }
      } else {
        // The ring is drained (its last MMAs have completed): it takes the
        // partial tile, column by column.
        float* part = reinterpret_cast<float*>(smem) + row;
#pragma unroll
        for (int c = 0; c < kCols / 8; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) part[(half * kCols + 8 * c + i) * kGemmRows] = __uint_as_float(v[c][i]);
      }
    }
  }
  tc_fence_before();
  if (p.split > 1) {
    cluster_sync();  // every partial tile is in place
    if (warp >= 2 && *abort_flag == 0) {
      const int t = threadIdx.x - 64, row = t & 127;
      const float ga = p.scale_a != nullptr ? *p.scale_a : 1.f, gb = p.scale_b != nullptr ? *p.scale_b : 1.f;
      int pt, qt;
      fp4_tile_coords(p, first_tile, pt, qt);
      const int per = TN / p.split;  // columns this CTA sums: 2 at the least
      for (int c = (t >> 7) * 8; c < per; c += 16) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        const int c0 = rank * per + c;
        for (int r = 0; r < p.split; ++r) {
          const uint32_t from = mapa_shared(base, r) + (c0 * kGemmRows + row) * 4;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < per) v[i] += ld_shared_cluster(from + i * kGemmRows * 4);
        }
        const int q = qt * TN + c0, pr = pt * kGemmRows + row;
        if (per >= 8) {
          fp4_gemm_emit<8>(p, pr, q, v, ga, gb);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float one[1] = {v[i]};
            if (i < per) fp4_gemm_emit<1>(p, pr, q + i, one, ga, gb);
          }
        }
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while a peer reads its partial tile
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int TN, int FORMAT>
static int fp4_gemm_launch(Fp4GemmParams& p, cudaStream_t st) {
  using C = Fp4Tile<TN, FORMAT>;
  static std::atomic<uint64_t> configured{0};
  DGXM_CUDA_TRY(set_smem_limit_once(fp4_gemm_kernel<TN, FORMAT>, C::kSmemBytes, configured));
  const int tiles = p.p_tiles * p.q_tiles;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(p.split > 1 ? tiles * p.split : std::min(tiles, 148));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DGXM_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp4_gemm_kernel<TN, FORMAT>, p));
  return DGXM_OK;
}

template <int FORMAT>
static int fp4_gemm_pick(Fp4GemmParams& p, int tn, cudaStream_t st) {
  switch (tn) {
    case 16: return fp4_gemm_launch<16, FORMAT>(p, st);
    case 32: return fp4_gemm_launch<32, FORMAT>(p, st);
    case 64: return fp4_gemm_launch<64, FORMAT>(p, st);
    case 128: return fp4_gemm_launch<128, FORMAT>(p, st);
    default: return fp4_gemm_launch<256, FORMAT>(p, st);
  }
}

}  // namespace dgxm

extern "C" int dgxm_fp4_matmul(const dgxm_fp4_gemm_desc* d, const void* a_values, const void* a_scales,
                               const float* a_scale, const void* b_values, const void* b_scales, const float* b_scale,
                               const void* bias, void* out, void* stream) {
  using namespace dgxm;
  if (d == nullptr) return fail(DGXM_ERR_INVALID, "NULL 4-bit product descriptor");
  if (d->format != DGXM_FP4_NVFP4 && d->format != DGXM_FP4_MXFP4)
    return fail(DGXM_ERR_UNSUPPORTED, "4-bit format %d (nvfp4 or mxfp4)", d->format);
  if (d->m < 0 || d->n < 0 || d->k <= 0 || d->m > (1 << 30) || d->n > (1 << 30) || d->k > (1 << 30))
    return fail(DGXM_ERR_INVALID, "product of (%lld, %lld) and (%lld, %lld)", (long long)d->m, (long long)d->k,
                (long long)d->n, (long long)d->k);
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
  Fp4GemmParams p;
  memset(&p, 0, sizeof(p));
  // The tile: the wider side gives the 128 rows, unless both fill 256 x 128.
  const int64_t m = d->m, n = d->n;
  const int64_t narrow = m < n ? m : n;
  const bool q_is_tokens = narrow <= 64 && m <= n;
  int tn = narrow <= 16 ? 16 : narrow <= 32 ? 32 : narrow <= 64 ? 64 : 128;
  if (tn == 128 && (m + 127) / 128 * ((n + 255) / 256) >= 148) tn = 256;
  const int64_t p_rows = q_is_tokens ? n : m, q_rows = q_is_tokens ? m : n;
  const int64_t p_tiles = (p_rows + 127) / 128, q_tiles = (q_rows + tn - 1) / tn;
  if (p_tiles * q_tiles > (1 << 28)) return fail(DGXM_ERR_UNSUPPORTED, "too many output tiles");
  p.p_rows = static_cast<int>(p_rows);
  p.q_rows = static_cast<int>(q_rows);
  p.k = static_cast<int>(d->k);
  p.k_tiles = static_cast<int>((d->k + kGemmK - 1) / kGemmK);
  p.p_tiles = static_cast<int>(p_tiles);
  p.q_tiles = static_cast<int>(q_tiles);
  p.split = 1;
  while (p.split < 8 && p.split * 2 <= p.k_tiles && p_tiles * q_tiles * p.split * 2 <= 148) p.split *= 2;
  p.q_is_tokens = q_is_tokens;
  p.groups = fp4_groups(d->k, d->format);
  const int64_t pitch = fp4_pitch(d->k);
  const void* pv = q_is_tokens ? b_values : a_values;
  const void* qv = q_is_tokens ? a_values : b_values;
  if (int rc = encode_map_4d(&p.tmap_p, pv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, pitch, 1, p_rows, 1, pitch, pitch,
                             pitch * p_rows, 128, kGemmRows))
    return rc;
  if (int rc = encode_map_4d(&p.tmap_q, qv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, pitch, 1, q_rows, 1, pitch, pitch,
                             pitch * q_rows, 128, tn))
    return rc;
  p.sf_p = static_cast<const uint8_t*>(q_is_tokens ? b_scales : a_scales);
  p.sf_q = static_cast<const uint8_t*>(q_is_tokens ? a_scales : b_scales);
  p.scale_a = a_scale;
  p.scale_b = b_scale;
  p.bias = bias;
  p.out = out;
  p.ld_out = d->out_stride;
  p.out_dtype = d->out_dtype;
  p.bias_dtype = d->bias_dtype;
  p.vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && d->out_stride * out_elt % 16 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return nv ? fp4_gemm_pick<DGXM_FP4_NVFP4>(p, tn, st) : fp4_gemm_pick<DGXM_FP4_MXFP4>(p, tn, st);
}
