// A 16-bit Linear with everything that follows it in a block in its epilogue,
// and its gradients:
//   pre = x W^T + bias,   out = residual + gate * act(pre)
//   dz = dout * gate * act'(pre),   dx = dz W,   dW = dz^T x,
//   dbias = sum dz,   dgate = sum dout * act(pre).
//
// All three products run in one kernel, D[p, q] = sum_k A[p, k] B[q, k], on
// tcgen05 with fp32 accumulators in tensor memory.  Either operand is K-major
// (contiguous in k) or MN-major (contiguous in its rows, as W is to dx and dz
// and x are to dW): only the TMA boxes and the descriptors' strides differ, so
// no operand is transposed in memory.
//
// Roles (10 warps), tile order, stores and the exchange of a split K are those
// of the 4-bit product (fp4_gemm.cu): warp 0 loads, warp 1 issues the MMAs,
// warps 2-9 run the epilogue.  Large products run on CTA pairs (256 x 256,
// M256 MMAs that read both CTAs' operands), others on single CTAs, and with
// few rows, or few tiles and a long K, the weight gives the rows of a tile.
//
// Large products are bound by power (9450 x 13824 x 5120 with GELU: 988 to 1034
// us in a row, 1.29 to 1.35 PFLOP/s), few rows by DRAM (2 x 30720 x 5120: 51 us,
// 6.1 TB/s), and what lies between by its few tiles, of 0.25 us a stage of K each
// (512 x 5120 x 4096: 21 to 24 us).
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "device_error.cuh"
#include "gemm_tile.cuh"
#include "ptx.cuh"

namespace dgxm {

constexpr int kLinK = 64;  // K a stage: one swizzle atom of 128 bytes

struct __align__(64) LinearParams {
  CUtensorMap tmap_a, tmap_b;  // K-major: dims (k, 1, rows), boxes (64, 1, 128 ..); MN-major: dims (rows, 1, k), boxes (64, 1, 64)
  CUtensorMap tmap_out;        // where `vec`: dims (q_rows, 1, p_rows), boxes of 128 bytes x 32 rows
  CUtensorMap tmap_res;        // where `res_bulk`: the same of the residual
  CUtensorMap tmap_pre;        // where `pre_vec`: the same of pre
  const void *bias, *gate, *residual;
  void *out, *pre;
  int64_t ld_out, ld_res, ld_pre;         // elements
  int64_t gate_sample, gate_row;          // elements between samples, rows
  int p_rows, q_rows, k_tiles, k;
  int p_tiles, q_tiles, split;
  int step, tn;                           // rows of A a tile takes, 128 (256) at the most, and rows of B
  int q_is_tokens;                        // the rows of A are output columns: the tile is the output transposed
  int out_dtype, bias_dtype, gate_dtype, pre_dtype, vec, res_bulk, pre_vec;
  int act, sample_rows, f16;
};

template <int TN, bool PAIR>
struct LinTile {
  static constexpr int kRows = PAIR ? 256 : 128;
  static constexpr int kQLoad = PAIR ? TN / 2 : TN;  // rows of B this CTA loads
  static constexpr int kABytes = 128 * 128, kBBytes = kQLoad * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr bool kSplits = TN <= 64;           // transposed tiles, stored by the lanes
  // Partial sums as in Fp4Tile, or a staging buffer for each epilogue warp.  (A
  // sixth stage of the ring is worth more than a second buffer: the loads'
  // latency bounds a stage.)
  static constexpr int kStagingBytes = kSplits ? (128 + 10) * TN * 4 : 8 * kGemmStageRows;
  static constexpr int kStages = (kGemmSmemMax - 1024 - kGemmCtrlBytes - kStagingBytes) / kStageBytes;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kStagingBytes + kGemmCtrlBytes;
  static constexpr int kFull = 0, kEmpty = kStages, kAccFull = 2 * kStages, kAccEmpty = kAccFull + 2,
                       kDrain = kAccEmpty + 2, kRes = kDrain + 1, kBars = kRes + 8;
  static_assert(kBars * 8 + 16 <= kGemmCtrlBytes, "control block");
  static_assert(kStageBytes % 1024 == 0, "swizzle atoms stay aligned");
  static constexpr int kTmem = TN < 32 ? 64 : 2 * TN;  // columns: a power of two, two accumulators
};

template <bool PAIR>
__device__ __forceinline__ void lin_umma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(DGXM_ELECT
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
                 "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
  else
    asm volatile(DGXM_ELECT
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
                 "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}

constexpr float kLinLog2e = 1.44269504f;

__device__ __forceinline__ float lin_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// 1 / (1 + e^-v); zero below -88, where it leaves the normal numbers.
__device__ __forceinline__ float lin_sigmoid(float v) { return lin_rcp(1.f + ex2_approx(-kLinLog2e * v)); }

constexpr float kGeluTanhA = 1.5957691216057308f;  // 2 sqrt(2 / pi): 1 + tanh(u) = 2 / (1 + e^-2u)
constexpr float kGeluTanhB = 0.044715f;

__device__ __forceinline__ float lin_act(float z, int act) {
  if (act == DGXM_ACT_SILU) return z * lin_sigmoid(z);
  if (act == DGXM_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == DGXM_ACT_GELU_TANH) return z * lin_sigmoid(kGeluTanhA * fmaf(kGeluTanhB * z * z, z, z));
  return z;
}

__device__ __forceinline__ float lin_value(const void* base, int dtype, int64_t at) {
  if (dtype == DGXM_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at]);
  if (dtype == DGXM_DTYPE_F16) return __half2float(static_cast<const __half*>(base)[at]);
  return static_cast<const float*>(base)[at];
}

__device__ __forceinline__ void lin_widen8(uint4 w, int dtype, float (&v)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float2 f;
    if (dtype == DGXM_DTYPE_BF16) f = make_float2(__uint_as_float(u[k] << 16), __uint_as_float(u[k] & 0xFFFF0000u));
    else f = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
    v[2 * k] = f.x;
    v[2 * k + 1] = f.y;
  }
}

// The first `count` of N neighbouring values.
template <int N, typename Use>
__device__ __forceinline__ void lin_each(const void* base, int dtype, int64_t at, int count, Use&& use) {
  if (dtype == DGXM_DTYPE_F32) {
    const float* from = static_cast<const float*>(base) + at;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < count) use(c, from[c]);
  } else if (const uint16_t* from = static_cast<const uint16_t*>(base) + at;
             count >= N && reinterpret_cast<uintptr_t>(from) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      float f[8];
      lin_widen8(reinterpret_cast<const uint4*>(from)[i], dtype, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) use(8 * i + k, f[k]);
    }
  } else {
    const bool bf16 = dtype == DGXM_DTYPE_BF16;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < count) {
        const uint16_t u = from[c];
        use(c, bf16 ? __uint_as_float(static_cast<uint32_t>(u) << 16) : __half2float(*reinterpret_cast<const __half*>(&u)));
      }
  }
}

__device__ __forceinline__ void lin_put(void* base, int dtype, int64_t at, float v) {
  if (dtype == DGXM_DTYPE_BF16) static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(v);
  else if (dtype == DGXM_DTYPE_F16) static_cast<__half*>(base)[at] = __float2half_rn(v);
  else static_cast<float*>(base)[at] = v;
}

// One operand's rows of a stage.  K-major: `rows` rows of 64 k.  MN-major:
// blocks of 64 rows, each 64 k of 128 bytes.
template <bool PAIR, bool MN, int ROWS>
__device__ __forceinline__ void lin_load(uint32_t dst, const void* map, uint32_t bar, int kt, int row) {
  if constexpr (MN) {
#pragma unroll
    for (int i = 0; i < ROWS / 64; ++i) fp4_tma<PAIR>(dst + i * 8192, map, bar, row + i * 64, 0, kt * kLinK);
  } else {
    fp4_tma<PAIR>(dst, map, bar, kt * kLinK, 0, row);
  }
}

// Descriptor of an operand's K step kk (16 k): K-major 32 bytes on in each row;
// MN-major 16 rows of 128 bytes on, blocks of 64 rows 8 KB apart.
template <bool MN>
__device__ __forceinline__ uint64_t lin_desc(uint32_t addr) {
  return MN ? sdesc_sw128(addr, 8192, 1024) : sdesc_sw128(addr, 16, 1024);
}
template <bool MN>
constexpr uint32_t kLinStep = MN ? 2048 / 16 : 32 / 16;

// What fp4_piece and fp4_flush_rows are told of `pre`.
struct LinPreOut {
  const CUtensorMap& tmap_out;
  void* out;
  int64_t ld_out;
  int p_rows, q_rows, out_dtype, vec;
};

// The residual of a warp's 32 rows x 128 bytes from row pr0 and column q0 into
// its staging rows as a bulk load leaves them, where its rows are off 16
// bytes: neighbouring lanes load neighbouring values.
template <int ELT>
__device__ __forceinline__ void lin_stage_residual(const LinearParams& p, uint8_t* buffer, int pr0, int q0, int lane) {
  using Elt = typename std::conditional<ELT == 4, uint32_t, uint16_t>::type;
  constexpr int kMost = 128 / ELT, kEach = 16 / ELT;
  const int rows = min(32, p.p_rows - pr0);
  const Elt* from = static_cast<const Elt*>(p.residual) + pr0 * p.ld_res + q0;
#pragma unroll 8
  for (int r = 0; r < rows; ++r)
#pragma unroll
    for (int c = lane; c < kMost; c += 32)
      if (q0 + c < p.q_rows)
        *reinterpret_cast<Elt*>(buffer + r * 128 + (((c / kEach) ^ (r & 7)) << 4) + (c % kEach) * ELT) = from[r * p.ld_res + c];
  __syncwarp();
}

// Column chunks of 128 output bytes of a tile, the even ones for the warps of
// half 0, the odd ones for half 1; a warp's own are numbered here.
template <int TN, int ELT>
struct LinChunks {
  static constexpr int kCols = 128 / ELT, kOwn = TN / kCols / 2 > 0 ? TN / kCols / 2 : 1;
  static __device__ __forceinline__ int column(int half, int i) { return (2 * i + half) * kCols; }
};

template <bool PAIR>
__device__ __forceinline__ void lin_release(uint32_t acc_empty, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) {
    if constexpr (PAIR) mbar_arrive_cluster_relaxed(acc_empty);
    else mbar_arrive(acc_empty);
  }
}

// The epilogue of a warp's 32 rows of a tile from row pr0, rows being tokens:
// bias and activation alone.  What else there can be stands apart
// (lin_epilogue_full, in kernels of its own): with those ways between them, the few instructions
// here miss the instruction cache at every jump (2000 cycles a chunk of 64
// columns instead of 300).
template <int TN, bool PAIR, int ELT, int ACT>
__device__ __forceinline__ void lin_epilogue(const LinearParams& p, uint8_t* stage, uint32_t tmem,
                                             uint32_t acc_empty, int pr0, int q_tile, int half, int lane,
                                             const float (&bias)[LinChunks<TN, ELT>::kOwn * LinChunks<TN, ELT>::kCols / 32]) {
  using K = LinChunks<TN, ELT>;
  constexpr int CC = K::kCols;
#pragma unroll
  for (int ch = 0; ch < K::kOwn; ++ch) {
    const int c0 = K::column(half, ch), q0 = q_tile + c0;
    const bool mine = c0 < p.tn && q0 < p.q_rows;  // uniform over the warp
    uint32_t r[CC / 8][8];
    if (mine) {
#pragma unroll
      for (int c = 0; c < CC / 8; ++c) tmem_ld8(tmem + c0 + 8 * c, r[c]);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < CC / 8; ++c) reg_fence8(r[c]);
    }
    if (ch == K::kOwn - 1) lin_release<PAIR>(acc_empty, lane);  // the accumulator is in registers
    if (!mine) continue;
    float v[CC];
#pragma unroll
    for (int c = 0; c < CC; ++c) v[c] = __uint_as_float(r[c / 8][c % 8]);
    if (p.bias != nullptr) {
#pragma unroll
      for (int c = 0; c < CC; ++c) v[c] += __shfl_sync(0xffffffffu, bias[(ch * CC + c) / 32], c % 32);
    }
    if (ACT != DGXM_ACT_NONE) {
#pragma unroll
      for (int c = 0; c < CC; ++c) v[c] = lin_act(v[c], ACT);
    }
    if (lane == 0) tma_store_wait_read();  // the last chunk has left the staging rows
    __syncwarp();
    uint8_t* const row_out = stage + lane * 128;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<uint4*>(row_out + ((i ^ (lane & 7)) << 4)) = fp4_piece<ELT>(p, v + i * (16 / ELT));
    fp4_flush_rows<CC, ELT>(p, stage, pr0, q0, lane);
  }
}

// The same with a gate, a residual or pre, sixteen columns at a time.
template <int TN, bool PAIR, int ELT>
__device__ __forceinline__ void lin_epilogue_full(const LinearParams& p, uint8_t* stage, uint32_t res_bar, int& res_phase,
                                               uint32_t tmem, uint32_t acc_empty, int pr0, int q_tile, int half, int lane) {
  using K = LinChunks<TN, ELT>;
  constexpr int CC = K::kCols;
  const int m = pr0 + lane;
  const int sample = min(m, p.p_rows - 1) / p.sample_rows, in_sample = m - sample * p.sample_rows;
  const char* const gate = static_cast<const char*>(p.gate);
  const bool one = p.gate_row == 0 && __all_sync(0xffffffffu, sample == __shfl_sync(0xffffffffu, sample, 0));
  const bool pre_staged = p.pre != nullptr && p.residual == nullptr;
  const LinPreOut to_pre{p.tmap_pre, p.pre, p.ld_pre, p.p_rows, p.q_rows, p.pre_dtype, p.pre_vec};
#pragma unroll 1
  for (int ch = 0; ch < K::kOwn; ++ch) {
    const int c0 = K::column(half, ch), q0 = q_tile + c0;
    if (!(c0 < p.tn && q0 < p.q_rows)) {  // uniform over the warp
      if (ch == K::kOwn - 1) lin_release<PAIR>(acc_empty, lane);
      continue;
    }
    float bias[2], gates[2];  // of column 32 i + lane
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = q0 + 32 * i + lane;
      const bool in = 32 * i < CC && n < p.q_rows;
      bias[i] = p.bias != nullptr && in ? lin_value(p.bias, p.bias_dtype, n) : 0.f;
      gates[i] = gate == nullptr ? 1.f : one && in ? lin_value(gate, p.gate_dtype, sample * p.gate_sample + n) : 0.f;
    }
    uint8_t* const row_out = stage + lane * 128;
    if (p.residual != nullptr) {
      if (p.res_bulk) {
        if (!mbar_wait(res_bar, res_phase, nullptr)) report_device_error(kErrEpilogueTimeout);
        res_phase ^= 1;
      } else if (ch > 0) {
        if (lane == 0) tma_store_wait_read();
        __syncwarp();
        lin_stage_residual<ELT>(p, stage, pr0, q0, lane);
      }
    } else {
      if (lane == 0) tma_store_wait_read();  // the last chunk has left the staging rows
      __syncwarp();
    }
    if (pre_staged) {  // pre by itself first
#pragma unroll 1
      for (int i = 0; i < CC / 16; ++i) {
        uint32_t r[2][8];
        tmem_ld8(tmem + c0 + 16 * i, r[0]);
        tmem_ld8(tmem + c0 + 16 * i + 8, r[1]);
        tmem_wait_ld();
        reg_fence8(r[0]);
        reg_fence8(r[1]);
        float v[16];
        const float b = i < 2 ? bias[0] : bias[1];
#pragma unroll
        for (int k = 0; k < 16; ++k)
          v[k] = __uint_as_float(r[k / 8][k % 8]) + __shfl_sync(0xffffffffu, b, (16 * i & 16) + k);
        *reinterpret_cast<uint4*>(row_out + (((2 * i) ^ (lane & 7)) << 4)) = fp4_piece<2>(to_pre, v);
        *reinterpret_cast<uint4*>(row_out + (((2 * i + 1) ^ (lane & 7)) << 4)) = fp4_piece<2>(to_pre, v + 8);
      }
      fp4_flush_rows<CC, 2>(to_pre, stage, pr0, q0, lane);
      if (lane == 0) tma_store_wait_read();
      __syncwarp();
    }
#pragma unroll 1
    for (int i = 0; i < CC / 16; ++i) {
      uint32_t r[2][8];
      tmem_ld8(tmem + c0 + 16 * i, r[0]);
      tmem_ld8(tmem + c0 + 16 * i + 8, r[1]);
      tmem_wait_ld();
      reg_fence8(r[0]);
      reg_fence8(r[1]);
      if (ch == K::kOwn - 1 && i == CC / 16 - 1) lin_release<PAIR>(acc_empty, lane);
      float v[16];
      const float b = i < 2 ? bias[0] : bias[1], g = i < 2 ? gates[0] : gates[1];
#pragma unroll
      for (int k = 0; k < 16; ++k)
        v[k] = __uint_as_float(r[k / 8][k % 8]) + __shfl_sync(0xffffffffu, b, (16 * i & 16) + k);
      if (p.pre != nullptr && !pre_staged && m < p.p_rows) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 piece = fp4_piece<2>(to_pre, v + 8 * h);
          const int n = q0 + 16 * i + 8 * h;
          uint16_t* at = static_cast<uint16_t*>(p.pre) + m * p.ld_pre + n;
          if (p.pre_vec && n + 8 <= p.q_rows) {
            *reinterpret_cast<uint4*>(at) = piece;
          } else {
            const uint32_t u[4] = {piece.x, piece.y, piece.z, piece.w};
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (n + k < p.q_rows) at[k] = static_cast<uint16_t>(u[k / 2] >> (16 * (k % 2)));
          }
        }
      }
      if (p.act == DGXM_ACT_SILU) {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = lin_act(v[k], DGXM_ACT_SILU);
      } else if (p.act == DGXM_ACT_GELU) {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = lin_act(v[k], DGXM_ACT_GELU);
      } else if (p.act == DGXM_ACT_GELU_TANH) {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = lin_act(v[k], DGXM_ACT_GELU_TANH);
      }
      if (gate == nullptr || one) {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] *= __shfl_sync(0xffffffffu, g, (16 * i & 16) + k);
      } else if (m < p.p_rows) {
        lin_each<16>(gate, p.gate_dtype, sample * p.gate_sample + in_sample * p.gate_row + q0 + 16 * i,
                     p.q_rows - q0 - 16 * i, [&](int k, float f) { v[k] *= f; });
      }
#pragma unroll
      for (int j = 0; j < ELT; ++j) {
        constexpr int kEach = 16 / ELT;
        uint4* const at = reinterpret_cast<uint4*>(row_out + (((i * ELT + j) ^ (lane & 7)) << 4));
        if (p.residual != nullptr) {
          const uint4 w = *at;
          if constexpr (ELT == 4) {
            v[4 * j] += __uint_as_float(w.x);
            v[4 * j + 1] += __uint_as_float(w.y);
            v[4 * j + 2] += __uint_as_float(w.z);
            v[4 * j + 3] += __uint_as_float(w.w);
          } else {
            float f[8];
            lin_widen8(w, p.out_dtype, f);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[8 * j + k] += f[k];
          }
        }
        *at = fp4_piece<ELT>(p, v + kEach * j);
      }
    }
    fp4_flush_rows<CC, ELT>(p, stage, pr0, q0, lane);
    const int next = K::column(half, ch + 1);
    if (p.res_bulk && ch + 1 < K::kOwn && next < p.tn && q_tile + next < p.q_rows) {
      tma_store_fence();  // rows that went by the lanes' stores have been written and read before the load writes them
      __syncwarp();
      if (lane == 0) {
        tma_store_wait_read();
        mbar_expect_tx(res_bar, kGemmStageRows);
        tma_load_4d(smem_u32(stage), &p.tmap_res, res_bar, q_tile + next, 0, pr0, 0);
      }
    }
  }
}

// The epilogue of a transposed tile out of the partial sums of the CTAs that
// share its K, this one having rows `rank` (128 / split) .. of it: four columns
// of a row a thread and turn of the loop, each way of the epilogue taken for the
// four together (8192 x 64 x 256 in tiles of 64 columns: 25 us with a thread's 32
// values unrolled, which miss the instruction cache, 15.5 one at a time, 12.5 one
// after another of four, 8.9; 64 x 5120 x 5120: 15.2 -> 12.4).
template <int TN>
__device__ __forceinline__ void lin_finish_share(const LinearParams& p, const float4* part, int rank, int pt, int qt) {
  const int most = (128 + p.split - 1) / p.split, rows = min(most, p.step - rank * most), pitch = most | 1;
  if (rows <= 0) return;
  const int down = 256 / rows, along = 256 - down * rows;  // from a thread's values to its next ones
  int c4 = (threadIdx.x - 64) / rows, r = threadIdx.x - 64 - c4 * rows;
  for (; c4 < TN / 4; c4 += down) {  // neighbouring lanes take neighbouring output columns
    const int n = pt * p.step + rank * most + r, m = qt * TN + 4 * c4;
    if (n < p.p_rows && m < p.q_rows) {
      const float4 own = part[c4 * pitch + r];
      float v[4] = {own.x, own.y, own.z, own.w};
      for (int k = 1; k < p.split; ++k) {
        const float4 more = part[(k * (TN / 4) + c4) * pitch + r];
        v[0] += more.x;
        v[1] += more.y;
        v[2] += more.z;
        v[3] += more.w;
      }
      const int count = min(4, p.q_rows - m);
      if (p.bias != nullptr) {
        const float bias = lin_value(p.bias, p.bias_dtype, n);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += bias;
      }
      if (p.pre != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < count) lin_put(p.pre, p.pre_dtype, (m + e) * p.ld_pre + n, v[e]);
      }
      if (p.act == DGXM_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lin_act(v[e], DGXM_ACT_SILU);
      } else if (p.act == DGXM_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lin_act(v[e], DGXM_ACT_GELU);
      } else if (p.act == DGXM_ACT_GELU_TANH) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lin_act(v[e], DGXM_ACT_GELU_TANH);
      }
      float by[4], more[4];
      if (p.gate != nullptr) {
        const int last = p.q_rows - 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = min(m + e, last), sample = at / p.sample_rows;
          by[e] = lin_value(p.gate, p.gate_dtype, sample * p.gate_sample + (at - sample * p.sample_rows) * p.gate_row + n);
        }
      }
      if (p.residual != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) more[e] = e < count ? lin_value(p.residual, p.out_dtype, (m + e) * p.ld_res + n) : 0.f;
      }
      if (p.gate != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= by[e];
      }
      if (p.residual != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += more[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < count) lin_put(p.out, p.out_dtype, (m + e) * p.ld_out + n, v[e]);
    }
    r += along;
    if (r >= rows) {
      r -= rows;
      ++c4;
    }
  }
}

// What follows a product by rows: ELT bytes of an output, the activation, or
// (kActFull) any of them with a gate, a residual or pre.  Kernels of their own:
// together in one they spill, and miss the instruction cache.
constexpr int kActFull = -1;

template <int TN, bool PAIR, bool AMN, bool BMN, int ELT, int ACT>
__global__ void __launch_bounds__(kGemmThreads, 1) linear_kernel(const __grid_constant__ LinearParams p) {
  using C = LinTile<TN, PAIR>;
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
  const int kt0 = PAIR ? 0 : static_cast<int>(static_cast<int64_t>(rank) * p.k_tiles / p.split);  // this CTA's share of K
  const int kt1 = PAIR ? p.k_tiles : static_cast<int>(static_cast<int64_t>(rank + 1) * p.k_tiles / p.split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar(C::kFull + s), 1);
      mbar_init(bar(C::kEmpty + s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar(C::kAccFull + a), 1);
      mbar_init(bar(C::kAccEmpty + a), PAIR ? 16 : 8);  // every epilogue warp
    }
    mbar_init(bar(C::kDrain), 1);
    for (int i = 0; i < 8; ++i) mbar_init(bar(C::kRes + i), 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.tmap_a);
    tma_prefetch_desc(&p.tmap_b);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), C::kTmem);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), C::kTmem);
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

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      const int q_load = PAIR ? p.tn / 2 : TN;  // rows of B that this CTA multiplies
      // (MN-major B comes in whole blocks of 64 rows)
      const uint32_t bytes = PAIR ? 2 * (C::kABytes + (BMN ? C::kQLoad : q_load) * 128) : (AMN ? 128 : p.step) * 128 + C::kBBytes;
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
          if (cta == 0) mbar_expect_tx(bar(C::kFull + s), bytes);
          lin_load<PAIR, AMN, 128>(dst, &p.tmap_a, full, kt, pt * p.step + cta * 128);
          lin_load<PAIR, BMN, C::kQLoad>(dst + C::kABytes, &p.tmap_b, full, kt, qt * p.tn + cta * q_load);
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
    // ------------------------------------------------------------ MMAs
    if (cta == 0) {
      // idesc: fp32 accumulator, one format for both operands, their majors
      const uint32_t idesc = __shfl_sync(0xffffffffu, idesc_make(C::kRows, PAIR ? p.tn : TN, p.f16 ? 0u : 1u, BMN) | (AMN ? 1u << 15 : 0u), 0);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      int s = 0, parity = 0, u = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < tiles; tile += tile_step, ++u) {
        const int a = u & 1;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(C::kAccEmpty + a), ((u >> 1) & 1) ^ 1, abort_flag)))) break;
        tc_fence_after();
        const uint32_t acc = tm + a * TN;
        for (int kt = kt0; kt < kt1; ++kt) {
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(C::kFull + s), parity, abort_flag)))) break;
          tc_fence_after();
          const uint32_t sa = base + s * C::kStageBytes;
          const uint64_t da = lin_desc<AMN>(sa), db = lin_desc<BMN>(sa + C::kABytes);
#pragma unroll
          for (int kk = 0; kk < kLinK / 16; ++kk)
            lin_umma<PAIR>(acc, da + kk * kLinStep<AMN>, db + kk * kLinStep<BMN>, idesc, (kt > kt0 || kk > 0) ? 1u : 0u);
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
    const uint32_t acc_empty = PAIR ? mapa_shared(bar(C::kAccEmpty), 0) : bar(C::kAccEmpty);
    uint8_t* stage = staging + (warp - 2) * kGemmStageRows;  // (not of a transposed tile)
    const uint32_t res_bar = bar(C::kRes + warp - 2);
    const bool by_rows = TN > 64;
    int u = 0, res_phase = 0;
    for (int tile = first_tile; tile < tiles; tile += tile_step, ++u) {
      const int a = u & 1;
      int pt, qt;
      fp4_tile_coords(p, tile, pt, qt);
      const int pr0 = pt * p.step + cta * 128 + quarter * 32;  // this warp's first row
      bool fetched = false;
      if (ACT == kActFull && by_rows && p.residual != nullptr) {  // the residual's first chunk comes while the MMAs run
        if (lane == 0) tma_store_wait_read();
        tma_store_fence();  // as between chunks
        __syncwarp();
        if (const int c0 = LinChunks<TN, ELT>::column(half, 0), q0 = qt * p.tn + c0; c0 < p.tn && q0 < p.q_rows) {
          if (!p.res_bulk) {
            lin_stage_residual<ELT>(p, stage, pr0, q0, lane);
          } else {
            fetched = true;
            if (lane == 0) {
              mbar_expect_tx(res_bar, kGemmStageRows);
              tma_load_4d(smem_u32(stage), &p.tmap_res, res_bar, q0, 0, pr0, 0);
            }
          }
        }
        __syncwarp();
      }
      // Bias of column 32 i + lane of this warp's chunks, one after the other.
      constexpr int kBias = LinChunks<TN, ELT>::kOwn * LinChunks<TN, ELT>::kCols / 32;
      float bias[kBias];
      if (ACT != kActFull && by_rows) {
        constexpr int kOwn = LinChunks<TN, ELT>::kCols;
#pragma unroll
        for (int i = 0; i < kBias; ++i) {
          const int n = qt * p.tn + LinChunks<TN, ELT>::column(half, 32 * i / kOwn) + 32 * i % kOwn + lane;
          bias[i] = p.bias != nullptr && n < p.q_rows ? lin_value(p.bias, p.bias_dtype, n) : 0.f;
        }
      }
      const bool got = __all_sync(0xffffffffu, mbar_wait(bar(C::kAccFull + a), (u >> 1) & 1, abort_flag));
      if (!got) {
        report_device_error(kErrEpilogueTimeout);
        *abort_flag = 1;
        if (fetched) mbar_wait(res_bar, res_phase, nullptr);  // the load lands before the CTA can exit
        if (by_rows || p.split > 1) break;  // (the others meet at every tile, and no wait takes long from here on)
      }
      tc_fence_after();
      if constexpr (TN > 64) {
        if (by_rows) {
          const uint32_t from = tmem + lane_off + a * TN;
          const uint32_t to = acc_empty + a * 8;
          if constexpr (ACT == kActFull)
            lin_epilogue_full<TN, PAIR, ELT>(p, stage, res_bar, res_phase, from, to, pr0, qt * p.tn, half, lane);
          else
            lin_epilogue<TN, PAIR, ELT, ACT>(p, stage, from, to, pr0, qt * p.tn, half, lane, bias);
          continue;
        }
      }
      if constexpr (TN <= 64) {  // transposed, maybe a share of K
        if (got) {
          const uint32_t from = tmem + lane_off + a * TN + half * kCols;
          uint32_t r[kCols / 8][8];
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c) tmem_ld8(from + 8 * c, r[c]);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c) reg_fence8(r[c]);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty + a * 8);
          const int rows = (128 + p.split - 1) / p.split, pitch = rows | 1;
          const uint32_t to = mapa_shared(smem_u32(staging), row / rows) +
                              ((rank * (TN / 4) + half * (kCols / 4)) * pitch + row % rows) * 16;
#pragma unroll
          for (int c = 0; c < kCols / 4; ++c) st_shared_cluster(to + c * pitch * 16, r[c / 2] + 4 * (c % 2));
        }
        if (p.split == 1) {
          named_barrier_sync(1, 256);  // the tile is in place
          if (got) lin_finish_share<TN>(p, reinterpret_cast<const float4*>(staging), 0, pt, qt);
          named_barrier_sync(1, 256);  // and read
        }
      }
    }
    if (lane == 0) tma_store_wait_all();  // the staging rows outlive the stores
    __syncwarp();
  }
  tc_fence_before();
  if (PAIR || (C::kSplits && p.split > 1)) cluster_sync();  // both CTAs' MMAs drained; or every partial sum is in place
  else __syncthreads();
  if constexpr (C::kSplits) {
    if (p.split > 1 && warp >= 2 && *abort_flag == 0) {
      int pt, qt;
      fp4_tile_coords(p, first_tile, pt, qt);
      lin_finish_share<TN>(p, reinterpret_cast<const float4*>(staging), rank, pt, qt);
    }
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem, C::kTmem);
    else tmem_dealloc(tmem, C::kTmem);
  }
}

// One operand of a product: rows x k, contiguous in k, or (mn) in its rows.
struct LinOperand {
  const void* ptr;
  int64_t rows, ld;
  bool mn;
};

static int lin_map(CUtensorMap* map, const LinOperand& o, int64_t k, int box_rows) {
  const cuuint64_t row = static_cast<cuuint64_t>(o.ld) * 2;
  if (o.mn)
    return encode_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, o.ptr, {(cuuint64_t)o.rows, 1, (cuuint64_t)k}, {row, row},
                   {64, 1, kLinK}, CU_TENSOR_MAP_SWIZZLE_128B);
  return encode_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, o.ptr, {(cuuint64_t)k, 1, (cuuint64_t)o.rows}, {row, row},
                 {kLinK, 1, (cuuint32_t)box_rows}, CU_TENSOR_MAP_SWIZZLE_128B);
}

static int lin_out_map(CUtensorMap* map, const void* base, int64_t ld, int elt, const LinearParams& p) {
  const cuuint64_t row = static_cast<cuuint64_t>(ld) * elt;
  return encode_map_3d(map, elt == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, base,
                 {(cuuint64_t)p.q_rows, 1, (cuuint64_t)p.p_rows}, {row, row}, {(cuuint32_t)(128 / elt), 1, 32},
                 CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int TN, bool PAIR, bool AMN, bool BMN, int ELT = 2, int ACT = DGXM_ACT_NONE>
static int lin_launch(LinearParams& p, const LinOperand& a, const LinOperand& b, cudaStream_t st) {
  using C = LinTile<TN, PAIR>;
  static std::atomic<uint64_t> configured{0};
  DGXM_CUDA_TRY(set_smem_limit_once(linear_kernel<TN, PAIR, AMN, BMN, ELT, ACT>, C::kSmemBytes, configured));
  if (int rc = lin_map(&p.tmap_a, a, p.k, PAIR ? 128 : p.step)) return rc;
  if (int rc = lin_map(&p.tmap_b, b, p.k, PAIR ? p.tn / 2 : TN)) return rc;
  const int elt = p.out_dtype == DGXM_DTYPE_F32 ? 4 : 2;
  const bool rows = !p.q_is_tokens && p.split == 1;
  p.vec = p.vec && rows;
  p.res_bulk = rows && p.residual != nullptr && reinterpret_cast<uintptr_t>(p.residual) % 16 == 0 && p.ld_res > 0 &&
               p.ld_res * elt % 16 == 0;
  // (a chunk of pre is 128 bytes of its own beside a 16-bit output only)
  p.pre_vec = rows && p.pre != nullptr && reinterpret_cast<uintptr_t>(p.pre) % 16 == 0 && p.ld_pre % 8 == 0;
  if (p.vec)
    if (int rc = lin_out_map(&p.tmap_out, p.out, p.ld_out, elt, p)) return rc;
  if (p.res_bulk)
    if (int rc = lin_out_map(&p.tmap_res, p.residual, p.ld_res, elt, p)) return rc;
  if (p.pre_vec)
    if (int rc = lin_out_map(&p.tmap_pre, p.pre, p.ld_pre, 2, p)) return rc;
  p.p_tiles = (p.p_rows + p.step - 1) / p.step;
  p.q_tiles = (p.q_rows + p.tn - 1) / p.tn;
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
  DGXM_CUDA_TRY(cudaLaunchKernelEx(&cfg, linear_kernel<TN, PAIR, AMN, BMN, ELT, ACT>, p));
  return DGXM_OK;
}

template <int TN, bool PAIR, int ELT>
static int lin_launch_act(LinearParams& p, const LinOperand& a, const LinOperand& b, cudaStream_t st) {
  if (p.gate != nullptr || p.residual != nullptr || p.pre != nullptr)
    return lin_launch<TN, PAIR, false, false, ELT, kActFull>(p, a, b, st);
  switch (p.act) {
    case DGXM_ACT_SILU: return lin_launch<TN, PAIR, false, false, ELT, DGXM_ACT_SILU>(p, a, b, st);
    case DGXM_ACT_GELU: return lin_launch<TN, PAIR, false, false, ELT, DGXM_ACT_GELU>(p, a, b, st);
    case DGXM_ACT_GELU_TANH: return lin_launch<TN, PAIR, false, false, ELT, DGXM_ACT_GELU_TANH>(p, a, b, st);
    default: return lin_launch<TN, PAIR, false, false, ELT, DGXM_ACT_NONE>(p, a, b, st);
  }
}

// How a product is cut: the tile's columns, whether a CTA pair has it, into how
// many CTAs its K is split, and whether the tile is transposed.
struct LinCut {
  int tn;
  bool pair;
  int split;
  bool q_is_tokens;  // with at most 64 columns
  int step;          // rows of a tile
};

// Tiles of up to 64 columns are transposed: the rows (m) are B's.  They serve
// few rows, and (64) products of few tiles, whose K is long enough to share.
// (MN-major operands come in blocks of 64 rows.)
static LinCut lin_cut(int64_t m, int64_t n, int k_tiles, bool a_mn, bool b_mn) {
  struct Kind {
    int tn;
    bool pair;
    double stage, tile, least;
  };
  // Microseconds a stage of K, a tile (transposed ones share its epilogue with the CTAs of a split K), and at the least, as
  // measured with all SMs at work (1024 and 2048 x 5120 x 5120 by rows, 1 .. 64 x 5120 x 5120, 256 x 804 x 8064 and
  // 8192 x 64 x 256 transposed); the sums order the cuts and are not the times of calls.  (A pair with 128 columns, 0.245,
  // 1.5 and 2.0, has no fewer passes than single CTAs ever, and a dearer one.)
  static const Kind kinds[] = {{16, false, 0.18, 1.3, 0.4},  {32, false, 0.19, 2.3, 0.5},  {64, false, 0.22, 4.5, 1.0},
                               {128, false, 0.24, 1.3, 1.6}, {192, true, 0.285, 1.7, 2.2}, {256, true, 0.315, 2.0, 2.5}};
  static const int clusters[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};  // that the SMs hold at one time
  LinCut best{128, false, 1, false, 128};
  double least = 1e30;
  for (const Kind& kind : kinds) {
    const bool swapped = kind.tn <= 64;
    if ((swapped && kind.tn < 64 && (a_mn || m > kind.tn)) || (b_mn && kind.pair && kind.tn % 128 != 0)) continue;
    const int64_t p_rows = swapped ? n : m, q_rows = swapped ? m : n;
    const int rows = kind.pair ? 256 : 128, at_once = kind.pair ? 74 : 148;
    const int64_t tiles = (p_rows + rows - 1) / rows * ((q_rows + kind.tn - 1) / kind.tn);
    for (int split = 1; split <= (swapped ? 8 : 1) && split <= k_tiles; ++split) {
      if (split > 1 && tiles > clusters[split]) continue;
      const int64_t waves = (tiles * split + at_once - 1) / at_once;
      const double us = waves * std::max((k_tiles + split - 1) / split * kind.stage + kind.tile / split, kind.least) +
                        (split > 1 ? 1.6 + 0.02 * kind.tn : 0.0);
      if (us < least) {
        least = us;
        best = {kind.tn, kind.pair, split, swapped, rows};
      }
    }
  }
  // A transposed product reads the weight once and DRAM bounds it: tiles of
  // fewer rows, so that every SM has as many as the others (2 x 30720 x 5120:
  // 240 tiles of 128 rows or 296 of 104 on 148 SMs).
  if (best.q_is_tokens && best.split == 1 && m <= best.tn) {
    const int64_t waves = ((n + 127) / 128 + 147) / 148;
    best.step = static_cast<int>(std::min<int64_t>(128, ((n + 148 * waves - 1) / (148 * waves) + 7) / 8 * 8));
  }
  return best;
}

// D (m x n) = A B^T with the epilogue in p; a gives the tokens' side.
static int lin_product(LinearParams& p, const LinOperand& a, const LinOperand& b, int64_t k, cudaStream_t st) {
  p.k = static_cast<int>(k);
  p.k_tiles = static_cast<int>((k + kLinK - 1) / kLinK);
  const LinCut cut = lin_cut(a.rows, b.rows, p.k_tiles, a.mn, b.mn);
  p.split = cut.split;
  p.q_is_tokens = cut.q_is_tokens;
  p.step = cut.step;
  p.tn = cut.tn;
  if (p.q_is_tokens && b.mn) p.step = 128;  // whole blocks of 64 rows are loaded there
  const LinOperand &po = p.q_is_tokens ? b : a, &qo = p.q_is_tokens ? a : b;
  p.p_rows = static_cast<int>(po.rows);
  p.q_rows = static_cast<int>(qo.rows);
  p.vec = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ld_out * (p.out_dtype == DGXM_DTYPE_F32 ? 4 : 2) % 16 == 0;
  const bool amn = po.mn, bmn = qo.mn;
  switch (cut.tn) {
    case 16: return amn ? lin_launch<16, false, true, false>(p, po, qo, st) : lin_launch<16, false, false, false>(p, po, qo, st);
    case 32: return amn ? lin_launch<32, false, true, false>(p, po, qo, st) : lin_launch<32, false, false, false>(p, po, qo, st);
    case 64:
      if (bmn) return lin_launch<64, false, true, true>(p, po, qo, st);  // (w's gradient: both are)
      return amn ? lin_launch<64, false, true, false>(p, po, qo, st) : lin_launch<64, false, false, false>(p, po, qo, st);
    default: break;
  }
  if (amn || bmn) {  // the gradients' products: 16-bit outputs and nothing more
    if (cut.pair) return amn ? lin_launch<256, true, true, true>(p, po, qo, st) : lin_launch<256, true, false, true>(p, po, qo, st);
    return amn ? lin_launch<128, false, true, true>(p, po, qo, st) : lin_launch<128, false, false, true>(p, po, qo, st);
  }
  const bool wide = p.out_dtype == DGXM_DTYPE_F32;
  if (cut.pair) return wide ? lin_launch_act<256, true, 4>(p, po, qo, st) : lin_launch_act<256, true, 2>(p, po, qo, st);
  return wide ? lin_launch_act<128, false, 4>(p, po, qo, st) : lin_launch_act<128, false, 2>(p, po, qo, st);
}

// ------------------------------------------------------------ matrices off 16 bytes
// Rows that no TMA box can start at are copied to a pitch of whole 16 bytes
// first, up to two matrices in one launch.
struct LinPackParams {
  struct {
    const uint16_t* from;
    uint16_t* to;
    int64_t ld, words;  // of the whole copy, 16 bytes each
    int cols, pitch;
  } of[2];
  int n;
};

__global__ void __launch_bounds__(256) linear_pack_kernel(const __grid_constant__ LinPackParams p) {
  pdl_launch_dependents();
  pdl_wait();
  for (int j = 0; j < p.n; ++j) {
    const auto& o = p.of[j];
    const int across = o.pitch / 8;
    for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < o.words; i += gridDim.x * 256LL) {
      const int64_t row = o.words <= 0xffffffffLL ? static_cast<uint32_t>(i) / static_cast<uint32_t>(across) : i / across;
      const int col = static_cast<int>(i - row * across) * 8;
      const uint16_t* from = o.from + row * o.ld + col;
      uint32_t v[8], w[4];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = col + k < o.cols ? from[k] : 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = v[2 * k] | v[2 * k + 1] << 16;
      *reinterpret_cast<uint4*>(o.to + row * o.pitch + col) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

static int64_t lin_pitch(int64_t cols) { return (cols + 7) / 8 * 8; }
static bool lin_on_words(const void* ptr, int64_t ld) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && ld % 8 == 0; }
static int64_t lin_packed_bytes(const void* ptr, int64_t ld, int64_t rows, int64_t cols) {
  return lin_on_words(ptr, ld) ? 0 : (rows * lin_pitch(cols) * 2 + 255) / 256 * 256;
}

// Matrices to be copied so that their rows lie on 16 bytes.
struct LinPacker {
  LinPackParams p;
  char* work;
  explicit LinPacker(char* w) : work(w) { memset(&p, 0, sizeof(p)); }
  void add(const void** ptr, int64_t* ld, int64_t rows, int64_t cols) {
    const int64_t bytes = lin_packed_bytes(*ptr, *ld, rows, cols);
    if (bytes == 0) return;
    auto& o = p.of[p.n++];
    o.from = static_cast<const uint16_t*>(*ptr);
    o.to = reinterpret_cast<uint16_t*>(work);
    o.ld = *ld;
    o.cols = static_cast<int>(cols);
    o.pitch = static_cast<int>(lin_pitch(cols));
    o.words = rows * (o.pitch / 8);
    *ptr = work;
    *ld = o.pitch;
    work += bytes;
  }
  int run(cudaStream_t st) {
    if (p.n == 0) return DGXM_OK;
    const int64_t words = std::max(p.of[0].words, p.n > 1 ? p.of[1].words : 0);
    DGXM_CUDA_TRY(launch_overlapped(linear_pack_kernel, static_cast<unsigned>(std::min<int64_t>((words + 255) / 256, 148 * 8)),
                                    256, 0, st, p));
    p.n = 0;
    return DGXM_OK;
  }
};

// ------------------------------------------------------------ dz and the sums over rows
// A thread takes eight columns of a run of rows of one sample; its sums of dz and dout act(pre), whichever are wanted, go
// to (run, one or two, n) partial sums, which a second kernel adds in the order of the runs.  DRAM bounds it: dout and pre
// read, dz written.  Rows come by asynchronous copies into a ring, three ahead (in registers the loop waits for a row when
// it moves it up), and values are taken in pairs.  9450 x 13824 gelu_tanh with a bias: 235 -> 133 us (784 MB, 5.9 TB/s).
constexpr int kDzSlots = 4, kDzLeast = 4;  // of rows under way; rows of the shortest run

struct LinDzParams {
  const void *dout, *pre, *gate;
  void *dz, *g_gate;  // g_gate: a token's own, contiguous
  float* partial;     // (runs, sum_bias + sum_gate, pitch), or NULL
  int64_t pitch;
  int64_t ld_dout, ld_pre, ld_dz, gate_sample, gate_row;
  int64_t runs;
  int n, sample_rows, sample_runs, run_rows, sum_bias, sum_gate;
  int dtype, dout_dtype, gate_dtype, vec, gate_vec;
};

// Eight values from column `col`, zeros past the last.
__device__ __forceinline__ void lin_read8(const void* base, int dtype, int64_t at, int col, int n, int vec, float (&v)[8]) {
  if (vec && col + 8 <= n) {
    if (dtype == DGXM_DTYPE_F32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
      const float4 a = p[0], b = p[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      lin_widen8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at), dtype, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < n ? lin_value(base, dtype, at + i) : 0.f;
  }
}

// z within the limits past which a sigmoid's tail is below fp32's steps, so that the slope of values at the ends of the
// range is 0 or 1 and no infinity times zero; a NaN stays.
__device__ __forceinline__ float lin_within(float z, float limit) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(limit));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(r) : "f"(-limit));
  return r;
}

__device__ __forceinline__ uint64_t lin_two(float v) { return pk2(v, v); }

// An activation and its slope, of two values.  With s = sigmoid(q), q = z or z A (1 + B z^2) (SiLU, GELU by tanh):
// z s, and s (1 + (1 - s) z q').
template <int ACT>
__device__ __forceinline__ void lin_both(float z0, float z1, uint64_t& act, uint64_t& slope) {
  if constexpr (ACT == DGXM_ACT_GELU) {
    float a[2], b[2];
    const float z[2] = {z0, z1};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float phi = 0.5f * (1.f + erff(z[i] * 0.70710678118654752f)), zc = lin_within(z[i], 32.f);
      a[i] = z[i] * phi;
      b[i] = fmaf(zc * 0.39894228040143268f, ex2_approx(-0.5f * kLinLog2e * zc * zc), phi);
    }
    act = pk2(a[0], a[1]);
    slope = pk2(b[0], b[1]);
  } else if constexpr (ACT == DGXM_ACT_NONE) {
    act = pk2(z0, z1);
    slope = lin_two(1.f);
  } else {
    constexpr bool kTanh = ACT == DGXM_ACT_GELU_TANH;
    constexpr float kLimit = kTanh ? 16.f : 128.f, kA = kTanh ? kGeluTanhA : 1.f;
    const uint64_t z = pk2(lin_within(z0, kLimit), lin_within(z1, kLimit)), one = lin_two(1.f);
    uint64_t e = fmul2(z, lin_two(-kLinLog2e * kA)), dq = lin_two(kA);
    if constexpr (kTanh) {
      const uint64_t zz = fmul2(z, z);
      e = fmul2(e, ffma2(zz, lin_two(kGeluTanhB), one));
      dq = ffma2(zz, lin_two(3.f * kGeluTanhB * kA), dq);
    }
    float e0, e1;
    upk2(e, e0, e1);
    upk2(fadd2(pk2(ex2_approx(e0), ex2_approx(e1)), one), e0, e1);
    const uint64_t s = pk2(lin_rcp(e0), lin_rcp(e1));
    act = fmul2(pk2(z0, z1), s);
    const uint64_t rest = fmul2(ffma2(s, lin_two(-1.f), one), z);
    slope = fmul2(s, kTanh ? ffma2(rest, dq, one) : fadd2(rest, one));
  }
}

// GATES: a gate's gradient is wanted.  The loop over rows stays one: a run of
// a small call passes it a few times only, and would wait for the instructions
// of unrolled rows instead (512 x 5120 gelu: 29 us unrolled, 10 us).
template <int ACT, bool GATES>
__global__ void __launch_bounds__(128) linear_dz_kernel(const __grid_constant__ LinDzParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int col = (blockIdx.y * 128 + threadIdx.x) * 8;
  if (col >= p.n) return;
  constexpr bool kPre = ACT != DGXM_ACT_NONE || GATES;
  const bool whole = p.vec && col + 8 <= p.n && p.dout_dtype == p.dtype, f16 = p.dtype == DGXM_DTYPE_F16;
  __shared__ uint4 ring[kDzSlots][1 + kPre][128];
  for (int64_t run = blockIdx.x; run < p.runs; run += gridDim.x) {
    const int64_t sample = run / p.sample_runs;
    const int first = static_cast<int>(run - sample * p.sample_runs) * p.run_rows;
    const int rows = min(p.run_rows, p.sample_rows - first);
    const int64_t m0 = sample * p.sample_rows + first;
    // Rows under way, in a ring; its slot is a thread's own, and refilled a row after it was read.
    auto fetch = [&](int r) {
      if (whole && r < rows) {
        const uint32_t to = smem_u32(&ring[r % kDzSlots][0][threadIdx.x]);
        cp_async16(to, static_cast<const uint16_t*>(p.dout) + (m0 + r) * p.ld_dout + col);
        if (kPre) cp_async16(to + 128 * 16, static_cast<const uint16_t*>(p.pre) + (m0 + r) * p.ld_pre + col);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int j = 0; j + 1 < kDzSlots; ++j) fetch(j);
    float gate[8];
    uint64_t sum[4], sum_gate[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      gate[2 * i] = gate[2 * i + 1] = 1.f;
      sum[i] = sum_gate[i] = 0;  // (two zeros)
    }
    if (p.gate != nullptr && p.gate_row == 0)
      lin_read8(p.gate, p.gate_dtype, sample * p.gate_sample + col, col, p.n, p.gate_vec, gate);
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
      const int64_t m = m0 + r;
      float d[8], z[8];
      if (whole) {
        cp_async_wait<kDzSlots - 2>();
        lin_widen8(ring[r % kDzSlots][0][threadIdx.x], p.dtype, d);
        if (kPre) lin_widen8(ring[r % kDzSlots][kPre][threadIdx.x], p.dtype, z);
      } else {
        lin_read8(p.dout, p.dout_dtype, m * p.ld_dout + col, col, p.n, p.vec, d);
        if (kPre) lin_read8(p.pre, p.dtype, m * p.ld_pre + col, col, p.n, p.vec, z);
      }
      fetch(r + kDzSlots - 1);
      if (p.gate != nullptr && p.gate_row != 0)
        lin_read8(p.gate, p.gate_dtype, sample * p.gate_sample + (first + r) * p.gate_row + col, col, p.n, p.gate_vec, gate);
      float of_gate[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t dd = pk2(d[2 * i], d[2 * i + 1]), gg = pk2(gate[2 * i], gate[2 * i + 1]);
        uint64_t dz = fmul2(dd, gg);
        if constexpr (kPre) {
          uint64_t act, slope;
          lin_both<ACT>(z[2 * i], z[2 * i + 1], act, slope);
          const uint64_t og = fmul2(dd, act);
          sum_gate[i] = fadd2(sum_gate[i], og);
          upk2(og, of_gate[2 * i], of_gate[2 * i + 1]);
          dz = fmul2(dz, slope);
        }
        sum[i] = fadd2(sum[i], dz);
        upk2(dz, d[2 * i], d[2 * i + 1]);
      }
      if (GATES && p.g_gate != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < p.n) lin_put(p.g_gate, p.gate_dtype, m * p.n + col + i, of_gate[i]);
      }
      if (p.dz != nullptr)  // (columns past the last, up to the pitch, are zeros)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dz) + m * p.ld_dz + col) =
            f16 ? make_uint4(pack_f16x2(d[0], d[1]), pack_f16x2(d[2], d[3]), pack_f16x2(d[4], d[5]), pack_f16x2(d[6], d[7]))
                : make_uint4(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]), pack_bf16x2(d[4], d[5]), pack_bf16x2(d[6], d[7]));
    }
    if (p.partial != nullptr) {
      auto put = [&](int64_t row, const uint64_t (&v)[4]) {  // the pitch is whole eights
        ulonglong2* to = reinterpret_cast<ulonglong2*>(p.partial + row * p.pitch + col);
        to[0] = make_ulonglong2(v[0], v[1]);
        to[1] = make_ulonglong2(v[2], v[3]);
      };
      const int64_t row = run * (p.sum_bias + p.sum_gate);
      if (p.sum_bias) put(row, sum);
      if (GATES && p.sum_gate) put(row + p.sum_bias, sum_gate);
    }
  }
}

template <bool GATES>
static auto lin_dz_pick(int act) {
  return act == DGXM_ACT_SILU   ? linear_dz_kernel<DGXM_ACT_SILU, GATES>
         : act == DGXM_ACT_GELU ? linear_dz_kernel<DGXM_ACT_GELU, GATES>
         : act == DGXM_ACT_NONE ? linear_dz_kernel<DGXM_ACT_NONE, GATES>
                                : linear_dz_kernel<DGXM_ACT_GELU_TANH, GATES>;
}

struct LinSumParams {
  const float* partial;
  void *g_bias, *g_gate;
  int64_t samples;
  int n, pitch, sample_runs, bias_dtype, gate_dtype, gate_form;
};

// A block takes 32 columns.  Its warps form groups of equal size, up to one a
// sample; a group shares out the runs of a sample, and then takes another.
__global__ void __launch_bounds__(1024) linear_sum_kernel(const __grid_constant__ LinSumParams p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float part[32][2][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane;
  const bool in = col < p.n, biases = p.g_bias != nullptr, gates = p.g_gate != nullptr;
  const int sums = biases + gates;
  int groups = 1;
  while (groups < 32 && groups < p.samples) groups *= 2;
  const int each = 32 / groups, group = warp / each, turn = warp % each;
  // The sums of `count` warps from `first` on, `step` apart, in order.
  auto join = [&](float& b, float& g, bool mine, int first, int step, int count) {
    part[warp][0][lane] = b;
    part[warp][1][lane] = g;
    __syncthreads();
    if (mine) {
      b = g = 0.f;
      for (int k = 0; k < count; ++k) {
        b += part[first + k * step][0][lane];
        g += part[first + k * step][1][lane];
      }
    }
    __syncthreads();
  };
  float bias = 0.f, shared = 0.f;
  for (int64_t s0 = 0; s0 < p.samples; s0 += groups) {
    const int64_t s = s0 + group;
    float b = 0.f, g = 0.f;
    const int64_t r0 = s * p.sample_runs + static_cast<int64_t>(p.sample_runs) * turn / each;
    const int64_t r1 = s * p.sample_runs + static_cast<int64_t>(p.sample_runs) * (turn + 1) / each;
    if (in && s < p.samples) {
#pragma unroll 4
      for (int64_t r = r0; r < r1; ++r) {
        if (biases) b += p.partial[r * sums * p.pitch + col];
        if (gates) g += p.partial[(r * sums + biases) * p.pitch + col];
      }
    }
    if (each > 1) join(b, g, turn == 0, warp, 1, each);
    if (turn != 0) continue;
    if (in && s < p.samples && gates && p.gate_form == DGXM_MOD_SAMPLE) lin_put(p.g_gate, p.gate_dtype, s * p.n + col, g);
    bias += b;
    shared += g;
  }
  if (groups > 1) join(bias, shared, warp == 0, 0, each, groups);
  if (warp != 0 || !in) return;
  if (gates && p.gate_form == DGXM_MOD_SHARED) lin_put(p.g_gate, p.gate_dtype, col, shared);
  if (biases) lin_put(p.g_bias, p.bias_dtype, col, bias);
}

// ------------------------------------------------------------ the C entries
static int lin_check(const dgxm_linear_desc* d) {
  if (d == nullptr) return fail(DGXM_ERR_INVALID, "NULL linear descriptor");
  const int64_t most = int64_t(1) << 30;
  if (d->m < 0 || d->n < 0 || d->k <= 0 || d->m > most || d->n > most)
    return fail(DGXM_ERR_INVALID, "product of (%lld, %lld) and (%lld, %lld)", (long long)d->m, (long long)d->k,
                (long long)d->n, (long long)d->k);
  // A stage of K takes 0.5 us at the most: the longest K waits well within the bounded waits' second.
  if (d->k > (1 << 24) || d->n > (1 << 24)) return fail(DGXM_ERR_UNSUPPORTED, "k %lld or n %lld above 2^24", (long long)d->k, (long long)d->n);
  if (d->dtype != DGXM_DTYPE_BF16 && d->dtype != DGXM_DTYPE_F16)
    return fail(DGXM_ERR_UNSUPPORTED, "dtype %d (bf16 or f16)", d->dtype);
  for (int t : {d->out_dtype, d->bias_dtype, d->gate_dtype})
    if (t != d->dtype && t != DGXM_DTYPE_F32)
      return fail(DGXM_ERR_UNSUPPORTED, "output, bias or gate dtype %d (the operands' or f32)", t);
  if (d->activation < DGXM_ACT_NONE || d->activation > DGXM_ACT_GELU_TANH)
    return fail(DGXM_ERR_UNSUPPORTED, "activation %d", d->activation);
  if (d->gate_form < DGXM_MOD_NONE || d->gate_form > DGXM_MOD_TOKEN)
    return fail(DGXM_ERR_INVALID, "modulation form %d", d->gate_form);
  if (d->gate_form != DGXM_MOD_NONE && (d->sample_rows <= 0 || (d->m > 0 && d->m % d->sample_rows != 0)))
    return fail(DGXM_ERR_INVALID, "%lld rows are no whole samples of %lld", (long long)d->m, (long long)d->sample_rows);
  if ((d->m > 1 && d->x_stride < d->k) || (d->n > 1 && d->w_stride < d->k) || (d->m > 1 && d->out_stride < d->n))
    return fail(DGXM_ERR_INVALID, "a row stride is below its row");
  if ((d->m + 127) / 128 * ((d->n + 127) / 128) > (1 << 26) || (d->m + 127) / 128 * ((d->k + 127) / 128) > (1 << 26) ||
      (d->n + 127) / 128 * ((d->k + 127) / 128) > (1 << 26))
    return fail(DGXM_ERR_UNSUPPORTED, "too many output tiles");
  return DGXM_OK;
}

static int lin_elt(int dtype) { return dtype == DGXM_DTYPE_F32 ? 4 : 2; }

static int lin_aligned(const void* ptr, int dtype, const char* what) {
  if (reinterpret_cast<uintptr_t>(ptr) % lin_elt(dtype)) return fail(DGXM_ERR_INVALID, "%s is not aligned to its elements", what);
  return DGXM_OK;
}

static void lin_gate_strides(const dgxm_linear_desc* d, int64_t* sample, int64_t* row) {
  *sample = d->gate_form == DGXM_MOD_SAMPLE || d->gate_form == DGXM_MOD_TOKEN ? d->gate_stride[0] : 0;
  *row = d->gate_form == DGXM_MOD_TOKEN ? d->gate_stride[1] : 0;
}

}  // namespace dgxm

extern "C" int64_t dgxm_linear_workspace(const dgxm_linear_desc* d, const void* x, const void* w) {
  using namespace dgxm;
  if (lin_check(d)) return -1;
  if (d->m == 0 || d->n == 0) return 0;
  return lin_packed_bytes(x, d->x_stride, d->m, d->k) + lin_packed_bytes(w, d->w_stride, d->n, d->k);
}

extern "C" int dgxm_linear(const dgxm_linear_desc* d, const void* x, const void* w, const void* bias, const void* gate,
                           const void* residual, void* out, void* pre, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  using namespace dgxm;
  if (int rc = lin_check(d)) return rc;
  if (d->m == 0 || d->n == 0) return DGXM_OK;
  if (x == nullptr || w == nullptr || out == nullptr) return fail(DGXM_ERR_INVALID, "NULL operand or output");
  if ((gate != nullptr) != (d->gate_form != DGXM_MOD_NONE)) return fail(DGXM_ERR_INVALID, "gate and gate_form do not match");
  if ((residual != nullptr && d->m > 1 && d->residual_stride < d->n && d->residual_stride != 0) ||
      (pre != nullptr && d->m > 1 && d->pre_stride < d->n))
    return fail(DGXM_ERR_INVALID, "a row stride is below its row");
  if (int rc = lin_aligned(x, d->dtype, "x")) return rc;
  if (int rc = lin_aligned(w, d->dtype, "w")) return rc;
  if (int rc = lin_aligned(bias, d->bias_dtype, "bias")) return rc;
  if (int rc = lin_aligned(gate, d->gate_dtype, "gate")) return rc;
  if (int rc = lin_aligned(residual, d->out_dtype, "residual")) return rc;
  if (int rc = lin_aligned(out, d->out_dtype, "out")) return rc;
  if (int rc = lin_aligned(pre, d->dtype, "pre")) return rc;
  const int64_t need = dgxm_linear_workspace(d, x, w);
  if (need > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < need))
    return fail(DGXM_ERR_INVALID, "workspace of %lld bytes (%lld needed)", (long long)workspace_bytes, (long long)need);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int64_t ldx = d->m > 1 ? d->x_stride : lin_pitch(d->k), ldw = d->n > 1 ? d->w_stride : lin_pitch(d->k);
  if (d->m == 1 && !lin_on_words(x, d->x_stride)) ldx = d->x_stride;
  if (d->n == 1 && !lin_on_words(w, d->w_stride)) ldw = d->w_stride;
  LinPacker pack(static_cast<char*>(workspace));
  pack.add(&x, &ldx, d->m, d->k);
  pack.add(&w, &ldw, d->n, d->k);
  if (int rc = pack.run(st)) return rc;
  LinearParams p;
  memset(&p, 0, sizeof(p));
  p.bias = bias;
  p.gate = gate;
  p.residual = residual;
  p.out = out;
  p.pre = pre;
  p.ld_out = d->m > 1 ? d->out_stride : lin_pitch(d->n);  // (of one row unused)
  p.ld_res = d->m > 1 ? d->residual_stride : lin_pitch(d->n);
  p.ld_pre = d->m > 1 ? d->pre_stride : lin_pitch(d->n);
  lin_gate_strides(d, &p.gate_sample, &p.gate_row);
  p.out_dtype = d->out_dtype;
  p.bias_dtype = d->bias_dtype;
  p.gate_dtype = d->gate_dtype;
  p.pre_dtype = d->dtype;
  p.act = d->activation;
  p.sample_rows = static_cast<int>(d->gate_form != DGXM_MOD_NONE ? d->sample_rows : d->m);
  p.f16 = d->dtype == DGXM_DTYPE_F16;
  return lin_product(p, {x, d->m, ldx, false}, {w, d->n, ldw, false}, d->k, st);
}

namespace dgxm {

// Where the gradient's intermediates lie in the workspace.
struct LinBackPlan {
  bool dz;      // dz is not dout itself
  int sums;     // over rows that are wanted, bias' and a gate's
  int64_t gate_sample, gate_row;
  int64_t runs, sample_runs, sample_rows, run_rows, dz_bytes, part_bytes, x_bytes, w_bytes, dout_bytes;
  int64_t total() const { return dz_bytes + part_bytes + x_bytes + w_bytes + dout_bytes; }
};

static int lin_check_back(const dgxm_linear_desc* d, const dgxm_linear_grads* g) {
  if (int rc = lin_check(d)) return rc;
  if (g == nullptr) return fail(DGXM_ERR_INVALID, "NULL gradients");
  // w's gradient is a product along m, bounded as k is.
  if (g->w != nullptr && d->m > (1 << 24)) return fail(DGXM_ERR_UNSUPPORTED, "w's gradient over m %lld, above 2^24", (long long)d->m);
  return DGXM_OK;
}

static LinBackPlan lin_back_plan(const dgxm_linear_desc* d, const dgxm_linear_grads* g, const void* dout, const void* x,
                                 const void* w) {
  LinBackPlan b;
  memset(&b, 0, sizeof(b));
  const bool products = g->x != nullptr || g->w != nullptr;
  b.dz = products && (d->activation != DGXM_ACT_NONE || d->gate_form != DGXM_MOD_NONE || d->out_dtype != d->dtype);
  b.sums = (g->bias != nullptr) + (g->gate != nullptr && d->gate_form != DGXM_MOD_TOKEN);
  // Runs end where a sample does only for the sake of its gate's sum, or of samples whose tokens' gates are not a step
  // apart: with a row a sample every run would be one row (9450 x 1 x 13824, a token's gate and a bias: 1.05 GB of partial
  // sums, 8 MB here).
  b.gate_sample = b.gate_row = 0;
  b.sample_rows = d->m;
  if (d->gate_form == DGXM_MOD_SAMPLE) {
    b.gate_sample = d->gate_stride[0];
    b.sample_rows = d->sample_rows;
  } else if (d->gate_form == DGXM_MOD_TOKEN) {
    b.gate_row = d->sample_rows == 1 ? d->gate_stride[0] : d->gate_stride[1];
    if (d->m > d->sample_rows && d->gate_stride[0] != d->sample_rows * b.gate_row) {
      b.gate_sample = d->gate_stride[0];
      b.sample_rows = d->sample_rows;
    }
  }
  // Runs of 64 rows, or shorter ones where those would leave the SMs without work (512 x 5120: 51 us in runs of 64, 10 in
  // runs of 4; 9450 x 13824 133 in runs of 64, 141 in runs of 4 and four times as long for their sums).
  const int64_t across = (lin_pitch(d->n) / 8 + 127) / 128;
  b.run_rows = std::max<int64_t>(kDzLeast, std::min<int64_t>(64, d->m * across / (148 * 8)));
  b.sample_runs = (b.sample_rows + b.run_rows - 1) / b.run_rows;
  b.runs = b.sample_rows > 0 ? d->m / b.sample_rows * b.sample_runs : 0;
  if (b.dz) b.dz_bytes = (d->m * lin_pitch(d->n) * 2 + 255) / 256 * 256;
  else if (products) b.dout_bytes = lin_packed_bytes(dout, d->out_stride, d->m, d->n);
  if (b.sums > 0) b.part_bytes = (b.runs * b.sums * lin_pitch(d->n) * 4 + 255) / 256 * 256;
  if (g->w != nullptr) b.x_bytes = lin_packed_bytes(x, d->x_stride, d->m, d->k);
  if (g->x != nullptr) b.w_bytes = lin_packed_bytes(w, d->w_stride, d->n, d->k);
  return b;
}

}  // namespace dgxm

extern "C" int64_t dgxm_linear_backward_workspace(const dgxm_linear_desc* d, const dgxm_linear_grads* g, const void* dout,
                                                  const void* x, const void* w) {
  using namespace dgxm;
  if (lin_check_back(d, g)) return -1;
  if (d->m == 0 || d->n == 0) return 0;
  return lin_back_plan(d, g, dout, x, w).total();
}

extern "C" int dgxm_linear_backward(const dgxm_linear_desc* d, const dgxm_linear_grads* g, const void* dout, const void* x,
                                    const void* w, const void* gate, const void* pre, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  using namespace dgxm;
  if (int rc = lin_check_back(d, g)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->m == 0 || d->n == 0) {  // sums of nothing
    if (g->x != nullptr && d->m > 0) DGXM_CUDA_TRY(cudaMemsetAsync(g->x, 0, d->m * d->k * 2, st));
    if (g->w != nullptr && d->n > 0) DGXM_CUDA_TRY(cudaMemsetAsync(g->w, 0, d->n * d->k * 2, st));
    if (g->bias != nullptr && d->n > 0) DGXM_CUDA_TRY(cudaMemsetAsync(g->bias, 0, d->n * lin_elt(d->bias_dtype), st));
    if (g->gate != nullptr && d->n > 0 && d->gate_form == DGXM_MOD_SHARED)
      DGXM_CUDA_TRY(cudaMemsetAsync(g->gate, 0, d->n * lin_elt(d->gate_dtype), st));
    return DGXM_OK;
  }
  if (dout == nullptr) return fail(DGXM_ERR_INVALID, "NULL upstream gradient");
  if ((g->x != nullptr && w == nullptr) || (g->w != nullptr && x == nullptr)) return fail(DGXM_ERR_INVALID, "NULL operand");
  if ((gate != nullptr) != (d->gate_form != DGXM_MOD_NONE) || (gate == nullptr && g->gate != nullptr))
    return fail(DGXM_ERR_INVALID, "gate, gate_form and the gate's gradient do not match");
  if (pre == nullptr && (d->activation != DGXM_ACT_NONE || g->gate != nullptr))
    return fail(DGXM_ERR_INVALID, "an activation's or a gate's gradient without pre");
  if (pre != nullptr && d->m > 1 && d->pre_stride < d->n) return fail(DGXM_ERR_INVALID, "a row stride is below its row");
  for (const void* q : {x, w, pre, static_cast<const void*>(g->x), static_cast<const void*>(g->w)})
    if (int rc = lin_aligned(q, d->dtype, "a tensor")) return rc;
  if (int rc = lin_aligned(dout, d->out_dtype, "dout")) return rc;
  if (int rc = lin_aligned(g->bias, d->bias_dtype, "the bias' gradient")) return rc;
  for (const void* q : {gate, static_cast<const void*>(g->gate)})
    if (int rc = lin_aligned(q, d->gate_dtype, "the gate or its gradient")) return rc;
  const LinBackPlan plan = lin_back_plan(d, g, dout, x, w);
  if (plan.total() > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < plan.total()))
    return fail(DGXM_ERR_INVALID, "workspace of %lld bytes (%lld needed)", (long long)workspace_bytes, (long long)plan.total());
  char* work = static_cast<char*>(workspace);
  const void* dz = dout;
  int64_t ld_dz = d->out_stride;
  const bool tok = d->gate_form == DGXM_MOD_TOKEN;
  if (plan.dz || plan.sums > 0 || (g->gate != nullptr && tok)) {
    LinDzParams q;
    memset(&q, 0, sizeof(q));
    q.dout = dout;
    q.pre = pre;
    q.gate = gate;
    if (plan.dz) {
      q.dz = work;
      q.ld_dz = lin_pitch(d->n);
      work += plan.dz_bytes;
    }
    if (plan.sums > 0) {
      q.partial = reinterpret_cast<float*>(work);
      work += plan.part_bytes;
    }
    q.pitch = lin_pitch(d->n);
    q.g_gate = tok ? g->gate : nullptr;
    q.ld_dout = d->out_stride;
    q.ld_pre = d->pre_stride;
    q.gate_sample = plan.gate_sample;
    q.gate_row = plan.gate_row;
    q.runs = plan.runs;
    q.n = static_cast<int>(d->n);
    q.sample_rows = static_cast<int>(plan.sample_rows);
    q.sample_runs = static_cast<int>(plan.sample_runs);
    q.run_rows = static_cast<int>(plan.run_rows);
    q.sum_bias = g->bias != nullptr;
    q.sum_gate = g->gate != nullptr && !tok;
    q.dtype = d->dtype;
    q.dout_dtype = d->out_dtype;
    q.gate_dtype = d->gate_dtype;
    q.vec = reinterpret_cast<uintptr_t>(dout) % 16 == 0 && d->out_stride * lin_elt(d->out_dtype) % 16 == 0 &&
            (pre == nullptr || (reinterpret_cast<uintptr_t>(pre) % 16 == 0 && d->pre_stride % 8 == 0));
    const int ge = lin_elt(d->gate_dtype);
    q.gate_vec = reinterpret_cast<uintptr_t>(gate) % 16 == 0 && q.gate_sample * ge % 16 == 0 && q.gate_row * ge % 16 == 0;
    const unsigned across = static_cast<unsigned>((lin_pitch(d->n) / 8 + 127) / 128);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(plan.runs, 1 << 20)), across);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    DGXM_CUDA_TRY(cudaLaunchKernelEx(&cfg, g->gate != nullptr ? lin_dz_pick<true>(d->activation) : lin_dz_pick<false>(d->activation), q));
    if (plan.sums > 0) {
      LinSumParams s;
      s.partial = q.partial;
      s.g_bias = g->bias;
      s.g_gate = tok ? nullptr : g->gate;
      s.samples = d->m / plan.sample_rows;
      s.n = q.n;
      s.pitch = static_cast<int>(q.pitch);
      s.sample_runs = q.sample_runs;
      s.bias_dtype = d->bias_dtype;
      s.gate_dtype = d->gate_dtype;
      s.gate_form = d->gate_form;
      DGXM_CUDA_TRY(launch_overlapped(linear_sum_kernel, (q.n + 31) / 32, 1024, 0, st, s));
    }
    if (plan.dz) {
      dz = q.dz;
      ld_dz = q.ld_dz;
    }
  }
  if (g->x == nullptr && g->w == nullptr) return DGXM_OK;
  LinPacker pack(work);
  int64_t ldw = d->w_stride, ldx = d->x_stride;
  if (!plan.dz) pack.add(&dz, &ld_dz, d->m, d->n);
  if (g->x != nullptr) pack.add(&w, &ldw, d->n, d->k);
  if (pack.p.n == 2)
    if (int rc = pack.run(st)) return rc;
  if (g->w != nullptr) pack.add(&x, &ldx, d->m, d->k);
  if (int rc = pack.run(st)) return rc;
  LinearParams p;
  memset(&p, 0, sizeof(p));
  p.out_dtype = p.bias_dtype = p.gate_dtype = p.pre_dtype = d->dtype;
  p.f16 = d->dtype == DGXM_DTYPE_F16;
  p.ld_out = d->k;
  if (g->x != nullptr) {
    p.out = g->x;
    p.sample_rows = static_cast<int>(d->m);
    if (int rc = lin_product(p, {dz, d->m, ld_dz, false}, {w, d->k, ldw, true}, d->n, st)) return rc;
  }
  if (g->w != nullptr) {
    p.out = g->w;
    p.sample_rows = static_cast<int>(d->n);
    if (int rc = lin_product(p, {dz, d->n, ld_dz, true}, {x, d->k, ldx, true}, d->m, st)) return rc;
  }
  return DGXM_OK;
}
