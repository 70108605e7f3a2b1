// What stands between two branches of a transformer block, in one pass, and
// its gradient:
//
//   m = branch, or (branch norm) branch / sqrt(mean(branch^2) + eps) * w2
//   r = x + g m
//   n = (r - mean r) / sqrt(var r + eps)   or   r / sqrt(mean(r^2) + eps)
//   y = (n w + b) (1 + s) + t
//
// and with upstream gradients dy of y and dr of r, and k = 1 / sqrt(...):
//
//   dt = sum dy,  ds = sum dy (n w + b),  dh = dy (1 + s),
//   dw = sum dh n,  db = sum dh,
//   R = dr + k (dh w - mean(dh w) - n mean(dh w n))   (RMS: no first mean)
//   dx = R,  dg = sum R m,  dm = R g,  dw2 = sum dm n2,
//   dbranch = dm, or k2 (dm w2 - n2 mean(dm w2 n2)).
//
// Every value is moved once and takes a few operations, so DRAM bounds both.
// A block holds a row, a thread the same columns of every row it sees: the
// modulation of a sample and the weights stay in its registers, and so do the
// sums over rows, which a second kernel adds in the order of the blocks.
// Means and variances are fp32 and the variance is that of the deviations, a
// second sum over the row; every output is rounded once.
#include "common.h"
#include "ptx.cuh"

namespace dgxm {

constexpr int kBnMaxWidth = 8192;  // six fp32 rows fit the shared memory of a block
constexpr int kBnMaxIn = 6;
// Streams of rows that a block reads: forward (x, branch, gate, scale, shift),
// backward (dy, dr, r, branch, gate, scale); the modulations where each token
// has its own.
enum { kBnX = 0, kBnBranch = 1, kBnGate = 2, kBnScale = 3, kBnShift = 4 };
enum { kBnDy = 0, kBnDr = 1, kBnR = 2, kBnBranchB = 3, kBnGateB = 4, kBnScaleB = 5 };

struct BlockNormParams {
  const char* in[kBnMaxIn];  // streams, NULL: absent
  int64_t in_sb[kBnMaxIn], in_sr[kBnMaxIn];  // bytes between samples, rows
  int in_f32[kBnMaxIn];      // a modulation of fp32 beside 16-bit tensors
  int in_off[kBnMaxIn];      // bytes into the stage
  int in_pitch[kBnMaxIn];    // bytes of a row in the stage, a multiple of 16
  int n_in, stage_bytes;
  // Values of a column that serve every row of a sample (gate, scale, shift), or all rows; NULL: absent
  const char *gate, *scale, *shift, *norm_w, *norm_b, *branch_w;
  int64_t gate_sb, scale_sb, shift_sb;  // bytes between samples
  int mod_f32, w_f32;
  char *out, *x_out;         // forward: y and r; backward: dbranch and dx
  int64_t out_sb, out_sr, x_out_sb, x_out_sr;  // bytes
  char *g_gate, *g_scale, *g_shift;  // backward, a row each token: contiguous
  float* partial;            // backward: (block + sample, 3, width)
  int want;                  // which of the three sums are wanted, a bit each
  int batch, seq, width, mode, branch_norm, gated;
  int64_t rows;
  float eps, inv_width;
};

template <typename T>
struct __align__(16) BnChunk {
  static constexpr int kN = 16 / static_cast<int>(sizeof(T));
  T v[kN];
};

// CH values from 16 bytes of T, or from fp32 (a modulation of fp32 beside 16-bit tensors).
template <typename T, int CH>
__device__ __forceinline__ void bn_read(const uint8_t* row, int chunk, int f32, float (&v)[CH]) {
  if (sizeof(T) == 4 || f32) {
    const float4* p = reinterpret_cast<const float4*>(row + static_cast<int64_t>(chunk) * CH * 4);
#pragma unroll
    for (int i = 0; i < CH / 4; ++i) {
      const float4 a = p[i];
      v[4 * i] = a.x, v[4 * i + 1] = a.y, v[4 * i + 2] = a.z, v[4 * i + 3] = a.w;
    }
  } else {
    const BnChunk<T> c = *reinterpret_cast<const BnChunk<T>*>(row + chunk * 16);
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = qk_widen(c.v[i]);
  }
}

// One value of a column vector of T or fp32.
template <typename T>
__device__ __forceinline__ float bn_value(const char* base, int f32, int col) {
  return f32 ? reinterpret_cast<const float*>(base)[col] : qk_widen(reinterpret_cast<const T*>(base)[col]);
}

template <typename T, int CH>
__device__ __forceinline__ void bn_vector(const char* base, int f32, int col, int width, float fill, float (&v)[CH]) {
#pragma unroll
  for (int i = 0; i < CH; ++i) v[i] = base != nullptr && col + i < width ? bn_value<T>(base, f32, col + i) : fill;
}

// Store CH values of a row from column `col` on.
template <typename T, int CH>
__device__ __forceinline__ void bn_store(char* row, int col, int width, const float (&v)[CH]) {
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if (col + i < width) reinterpret_cast<T*>(row)[col + i] = qk_narrow<T>(v[i]);
}

template <typename T, int CH>
__device__ __forceinline__ void bn_store_mod(char* row, int f32, int col, int width, const float (&v)[CH]) {
  if (f32) bn_store<float, CH>(row, col, width, v);
  else bn_store<T, CH>(row, col, width, v);
}

// Sums over the block, the same in every thread.  `red` alternates between
// two halves of N x 32 floats, so one barrier a sum is enough.
template <int N>
__device__ __forceinline__ void bn_block_sum(float (&v)[N], float* red, int& turn) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  float* half = red + (turn ^= 1) * (4 * 32);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) half[i * 32 + (threadIdx.x >> 5)] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = lane < warps ? half[i * 32 + lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
}

// Copy one row of every stream into the stage, value by value, and zeros up
// to whole chunks.
template <typename T>
__device__ __forceinline__ void bn_fill(const BlockNormParams& p, uint8_t* stage, int64_t b, int64_t l) {
  for (int s = 0; s < p.n_in; ++s) {
    if (p.in[s] == nullptr) continue;
    const char* from = p.in[s] + b * p.in_sb[s] + l * p.in_sr[s];
    uint8_t* to = stage + p.in_off[s];
    if (p.in_f32[s] || sizeof(T) == 4) {
      for (int c = threadIdx.x; c < p.in_pitch[s] / 4; c += blockDim.x)
        reinterpret_cast<float*>(to)[c] = c < p.width ? reinterpret_cast<const float*>(from)[c] : 0.f;
    } else {
      for (int c = threadIdx.x; c < p.in_pitch[s] / 2; c += blockDim.x)
        reinterpret_cast<uint16_t*>(to)[c] = c < p.width ? reinterpret_cast<const uint16_t*>(from)[c] : uint16_t(0);
    }
  }
}

// Thread t holds chunks t, t + blockDim, ... of each row, NV of them.
template <typename T, int NV>
__global__ void __launch_bounds__(1024) block_norm_kernel(const __grid_constant__ BlockNormParams p) {
  constexpr int CH = BnChunk<T>::kN;
  extern __shared__ __align__(16) uint8_t stage[];
  __shared__ float red[2 * 4 * 32];
  const int64_t first = blockIdx.x * p.rows / gridDim.x, last = (blockIdx.x + 1) * p.rows / gridDim.x;
  float g[NV][CH], a[NV][CH], c[NV][CH];
  int64_t sample = -1;
  int turn = 0;
  for (int64_t row = first; row < last; ++row) {
    const int64_t b = row / p.seq, l = row - b * p.seq;
    if (b != sample) {
      sample = b;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (threadIdx.x + k * blockDim.x) * CH;
        float w[CH], bias[CH], t[CH];
        bn_vector<T, CH>(p.gate ? p.gate + b * p.gate_sb : nullptr, p.mod_f32, col, p.width, 1.f, g[k]);
        bn_vector<T, CH>(p.scale ? p.scale + b * p.scale_sb : nullptr, p.mod_f32, col, p.width, 0.f, a[k]);
        bn_vector<T, CH>(p.shift ? p.shift + b * p.shift_sb : nullptr, p.mod_f32, col, p.width, 0.f, t);
        bn_vector<T, CH>(p.norm_w, p.w_f32, col, p.width, 1.f, w);
        bn_vector<T, CH>(p.norm_b, p.w_f32, col, p.width, 0.f, bias);
#pragma unroll
        for (int i = 0; i < CH; ++i) {  // y = n a + c
          a[k][i] += 1.f;
          c[k][i] = fmaf(bias[i], a[k][i], t[i]);
          a[k][i] *= w[i];
        }
      }
    }
    __syncthreads();
    bn_fill<T>(p, stage, b, l);
    __syncthreads();
    float root2 = 1.f;
    if (p.branch_norm) {
      float ss[1] = {0.f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int q = threadIdx.x + k * blockDim.x;
        if (q * CH >= p.width) continue;
        float m[CH];
        bn_read<T, CH>(stage + p.in_off[kBnBranch], q, 0, m);
#pragma unroll
        for (int i = 0; i < CH; ++i) ss[0] = fmaf(m[i], m[i], ss[0]);
      }
      bn_block_sum<1>(ss, red, turn);
      root2 = rsqrtf(fmaf(ss[0], p.inv_width, p.eps));
    }
    float r[NV][CH], sum[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = threadIdx.x + k * blockDim.x, col = q * CH;
      if (col >= p.width) continue;
      bn_read<T, CH>(stage + p.in_off[kBnX], q, 0, r[k]);
      if (p.in[kBnBranch] != nullptr) {
        float m[CH];
        bn_read<T, CH>(stage + p.in_off[kBnBranch], q, 0, m);
        if (p.branch_norm) {
          float w2[CH];
          bn_vector<T, CH>(p.branch_w, p.w_f32, col, p.width, 1.f, w2);
#pragma unroll
          for (int i = 0; i < CH; ++i) m[i] *= root2 * w2[i];
        }
        if (p.in[kBnGate] != nullptr) bn_read<T, CH>(stage + p.in_off[kBnGate], q, p.in_f32[kBnGate], g[k]);
#pragma unroll
        for (int i = 0; i < CH; ++i) r[k][i] = fmaf(g[k][i], m[i], r[k][i]);
        bn_store<T, CH>(p.x_out + b * p.x_out_sb + l * p.x_out_sr, col, p.width, r[k]);
      }
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (col + i < p.width) sum[0] += p.mode == DGXM_BLOCK_NORM_LAYER ? r[k][i] : r[k][i] * r[k][i];
    }
    if (p.mode == DGXM_BLOCK_NORM_NONE) continue;
    bn_block_sum<1>(sum, red, turn);
    float mean = 0.f;
    if (p.mode == DGXM_BLOCK_NORM_LAYER) {
      mean = sum[0] * p.inv_width;
      sum[0] = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if ((threadIdx.x + k * blockDim.x) * CH + i < p.width) sum[0] = fmaf(r[k][i] - mean, r[k][i] - mean, sum[0]);
      bn_block_sum<1>(sum, red, turn);
    }
    const float root = rsqrtf(fmaf(sum[0], p.inv_width, p.eps));
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = threadIdx.x + k * blockDim.x, col = q * CH;
      if (col >= p.width) continue;
      float y[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) y[i] = fmaf((r[k][i] - mean) * root, a[k][i], c[k][i]);
      if (p.in[kBnScale] != nullptr) {
        float s[CH];
        bn_read<T, CH>(stage + p.in_off[kBnScale], q, p.in_f32[kBnScale], s);
#pragma unroll
        for (int i = 0; i < CH; ++i) y[i] = fmaf(y[i], s[i], y[i]);
      }
      if (p.in[kBnShift] != nullptr) {
        float t[CH];
        bn_read<T, CH>(stage + p.in_off[kBnShift], q, p.in_f32[kBnShift], t);
#pragma unroll
        for (int i = 0; i < CH; ++i) y[i] += t[i];
      }
      bn_store<T, CH>(p.out + b * p.out_sb + l * p.out_sr, col, p.width, y);
    }
  }
}

// The gradient.  The sums over rows that a thread keeps for its columns are
//   0: sum e,  1: sum e n,  2: sum f n2
// with e = dy and f = R where the modulation serves a sample, so that the
// gradients of weights and modulations both follow from them, and e = dh,
// f = dm where each token has its own (n2 = branch without a branch norm).
template <typename T, int NV>
__global__ void __launch_bounds__(1024) block_norm_backward_kernel(const __grid_constant__ BlockNormParams p) {
  constexpr int CH = BnChunk<T>::kN;
  extern __shared__ __align__(16) uint8_t stage[];
  __shared__ float red[2 * 4 * 32];
  const int64_t first = blockIdx.x * p.rows / gridDim.x, last = (blockIdx.x + 1) * p.rows / gridDim.x;
  float g[NV][CH], a[NV][CH], w2[NV][CH], acc[3][NV][CH];
  int64_t sample = -1;
  int turn = 0;
  auto flush = [&]() {
    if (sample < 0 || p.partial == nullptr) return;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      if (!(p.want >> j & 1)) continue;
      float* to = p.partial + ((blockIdx.x + sample) * 3 + j) * p.width;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (const int col = (threadIdx.x + k * blockDim.x) * CH + i; col < p.width) to[col] = acc[j][k][i];
    }
  };
  for (int64_t row = first; row < last; ++row) {
    const int64_t b = row / p.seq, l = row - b * p.seq;
    if (b != sample) {
      flush();
      sample = b;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (threadIdx.x + k * blockDim.x) * CH;
        float w[CH];
        bn_vector<T, CH>(p.gate ? p.gate + b * p.gate_sb : nullptr, p.mod_f32, col, p.width, 1.f, g[k]);
        bn_vector<T, CH>(p.scale ? p.scale + b * p.scale_sb : nullptr, p.mod_f32, col, p.width, 0.f, a[k]);
        bn_vector<T, CH>(p.norm_w, p.w_f32, col, p.width, 1.f, w);
        bn_vector<T, CH>(p.branch_w, p.w_f32, col, p.width, 1.f, w2[k]);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          a[k][i] = (1.f + a[k][i]) * w[i];  // dh w = dy a
          acc[0][k][i] = acc[1][k][i] = acc[2][k][i] = 0.f;
        }
      }
    }
    __syncthreads();
    bn_fill<T>(p, stage, b, l);
    __syncthreads();
    float n[NV][CH], dn[NV][CH];
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = threadIdx.x + k * blockDim.x, col = q * CH;
      if (col >= p.width) continue;
      if (p.mode != DGXM_BLOCK_NORM_NONE) {
        bn_read<T, CH>(stage + p.in_off[kBnR], q, 0, n[k]);
#pragma unroll
        for (int i = 0; i < CH; ++i)
          sums[0] += p.mode == DGXM_BLOCK_NORM_LAYER ? n[k][i] : n[k][i] * n[k][i];
      }
      if (p.branch_norm) {
        float m[CH];
        bn_read<T, CH>(stage + p.in_off[kBnBranchB], q, 0, m);
#pragma unroll
        for (int i = 0; i < CH; ++i) sums[1] = fmaf(m[i], m[i], sums[1]);
      }
    }
    bn_block_sum<2>(sums, red, turn);
    const float root2 = p.branch_norm ? rsqrtf(fmaf(sums[1], p.inv_width, p.eps)) : 1.f;
    float mean = 0.f, root = 0.f, m1 = 0.f, m2 = 0.f;
    if (p.mode != DGXM_BLOCK_NORM_NONE) {
      if (p.mode == DGXM_BLOCK_NORM_LAYER) {
        mean = sums[0] * p.inv_width;
        float ss[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int i = 0; i < CH; ++i)
            if ((threadIdx.x + k * blockDim.x) * CH + i < p.width) ss[0] = fmaf(n[k][i] - mean, n[k][i] - mean, ss[0]);
        bn_block_sum<1>(ss, red, turn);
        sums[0] = ss[0];
      }
      root = rsqrtf(fmaf(sums[0], p.inv_width, p.eps));
      sums[0] = sums[1] = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int q = threadIdx.x + k * blockDim.x, col = q * CH;
        if (col >= p.width) continue;
        float dy[CH], e[CH], s[CH];
        bn_read<T, CH>(stage + p.in_off[kBnDy], q, 0, dy);
#pragma unroll
        for (int i = 0; i < CH; ++i) n[k][i] = (n[k][i] - mean) * root;
        if (p.in[kBnScaleB] != nullptr) bn_read<T, CH>(stage + p.in_off[kBnScaleB], q, p.in_f32[kBnScaleB], s);
        if (p.g_scale != nullptr) {  // a token's own: dy h
          float h[CH], bias[CH];
          bn_vector<T, CH>(p.norm_w, p.w_f32, col, p.width, 1.f, h);
          bn_vector<T, CH>(p.norm_b, p.w_f32, col, p.width, 0.f, bias);
#pragma unroll
          for (int i = 0; i < CH; ++i) h[i] = dy[i] * fmaf(n[k][i], h[i], bias[i]);
          bn_store_mod<T, CH>(p.g_scale + row * p.width * (p.mod_f32 ? 4 : sizeof(T)), p.mod_f32, col, p.width, h);
        }
        if (p.g_shift != nullptr)
          bn_store_mod<T, CH>(p.g_shift + row * p.width * (p.mod_f32 ? 4 : sizeof(T)), p.mod_f32, col, p.width, dy);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          e[i] = p.in[kBnScaleB] != nullptr ? dy[i] * (1.f + s[i]) : dy[i];
          dn[k][i] = e[i] * a[k][i];
          acc[0][k][i] += e[i];
          acc[1][k][i] = fmaf(e[i], n[k][i], acc[1][k][i]);
          if (col + i < p.width) {
            sums[0] += dn[k][i];
            sums[1] = fmaf(dn[k][i], n[k][i], sums[1]);
          }
        }
      }
      bn_block_sum<2>(sums, red, turn);
      m1 = p.mode == DGXM_BLOCK_NORM_LAYER ? sums[0] * p.inv_width : 0.f;
      m2 = sums[1] * p.inv_width;
    }
    float inner[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = threadIdx.x + k * blockDim.x, col = q * CH;
      if (col >= p.width) continue;
      float big[CH];
      if (p.in[kBnDr] != nullptr) bn_read<T, CH>(stage + p.in_off[kBnDr], q, 0, big);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (p.in[kBnDr] == nullptr) big[i] = 0.f;
        if (p.mode != DGXM_BLOCK_NORM_NONE) big[i] = fmaf(root, dn[k][i] - m1 - n[k][i] * m2, big[i]);
      }
      if (p.x_out != nullptr) bn_store<T, CH>(p.x_out + b * p.x_out_sb + l * p.x_out_sr, col, p.width, big);
      if (p.in[kBnBranchB] == nullptr) continue;
      float m[CH];
      bn_read<T, CH>(stage + p.in_off[kBnBranchB], q, 0, m);
      if (p.in[kBnGateB] != nullptr) bn_read<T, CH>(stage + p.in_off[kBnGateB], q, p.in_f32[kBnGateB], g[k]);
      if (p.g_gate != nullptr) {
        float dg[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) dg[i] = big[i] * m[i] * root2 * w2[k][i];
        bn_store_mod<T, CH>(p.g_gate + row * p.width * (p.mod_f32 ? 4 : sizeof(T)), p.mod_f32, col, p.width, dg);
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        m[i] *= root2;
        const float dm = big[i] * g[k][i];
        acc[2][k][i] = fmaf(p.in[kBnGateB] != nullptr ? dm : big[i], m[i], acc[2][k][i]);
        n[k][i] = m[i];
        dn[k][i] = dm * w2[k][i];
        if (col + i < p.width) inner[0] = fmaf(dn[k][i], m[i], inner[0]);
      }
      if (!p.branch_norm && p.out != nullptr)
        bn_store<T, CH>(p.out + b * p.out_sb + l * p.out_sr, col, p.width, dn[k]);
    }
    if (p.branch_norm) {
      bn_block_sum<1>(inner, red, turn);
      const float m3 = inner[0] * p.inv_width;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (threadIdx.x + k * blockDim.x) * CH;
        if (col >= p.width) continue;
#pragma unroll
        for (int i = 0; i < CH; ++i) dn[k][i] = root2 * (dn[k][i] - n[k][i] * m3);
        if (p.out != nullptr) bn_store<T, CH>(p.out + b * p.out_sb + l * p.out_sr, col, p.width, dn[k]);
      }
    }
  }
  flush();
}

// The gradients of weights and modulations from the blocks' sums.
struct BlockNormSumParams {
  const float* partial;
  const char *gate, *scale, *norm_w, *norm_b, *branch_w;
  int64_t gate_sb, scale_sb;
  void *g_gate, *g_scale, *g_shift, *g_norm_w, *g_norm_b, *g_branch_w;
  int gate_form, mod_form;  // of the modulations
  int want, dtype, mod_dtype, weight_dtype;
  int batch, seq, width, blocks;
  int64_t rows;
};

__device__ __forceinline__ float bn_any(const char* base, int dtype, int col, float fill) {
  if (base == nullptr) return fill;
  if (dtype == DGXM_DTYPE_F32) return reinterpret_cast<const float*>(base)[col];
  if (dtype == DGXM_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[col]);
  return __half2float(reinterpret_cast<const __half*>(base)[col]);
}

__device__ __forceinline__ void bn_put(void* base, int dtype, int64_t at, float v) {
  if (base == nullptr) return;
  if (dtype == DGXM_DTYPE_F32) static_cast<float*>(base)[at] = v;
  else if (dtype == DGXM_DTYPE_BF16) static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(base)[at] = __float2half_rn(v);
}

constexpr int kBnSumWarps = 32;

// A block takes 32 columns.  Its warps take the samples in turn where there
// are many, or else share out the blocks of each; warp 0 adds their sums in
// order.
__global__ void __launch_bounds__(kBnSumWarps * 32) block_norm_sum_kernel(const __grid_constant__ BlockNormSumParams p) {
  __shared__ float part[kBnSumWarps][6][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * 32 + lane;
  const bool in = col < p.width;
  const float w = in ? bn_any(p.norm_w, p.weight_dtype, col, 1.f) : 0.f;
  const float bias = in ? bn_any(p.norm_b, p.weight_dtype, col, 0.f) : 0.f;
  const float w2 = in ? bn_any(p.branch_w, p.weight_dtype, col, 1.f) : 0.f;
  const bool many = p.batch >= kBnSumWarps;
  float all[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // shift, scale, gate, norm_b, norm_w, branch_w over samples
  auto finish = [&](int b, const float (&s)[3]) {
    const float up = p.mod_form == DGXM_MOD_TOKEN || p.scale == nullptr || !in
                         ? 1.f
                         : 1.f + bn_any(p.scale + b * p.scale_sb, p.mod_dtype, col, 0.f);
    const float gate = p.gate_form == DGXM_MOD_TOKEN || p.gate == nullptr || !in
                           ? 1.f
                           : bn_any(p.gate + b * p.gate_sb, p.mod_dtype, col, 0.f);
    const float v[6] = {s[0], fmaf(w, s[1], bias * s[0]), w2 * s[2], up * s[0], up * s[1], gate * s[2]};
    if (in && p.mod_form == DGXM_MOD_SAMPLE) {
      bn_put(p.g_shift, p.mod_dtype, static_cast<int64_t>(b) * p.width + col, v[0]);
      bn_put(p.g_scale, p.mod_dtype, static_cast<int64_t>(b) * p.width + col, v[1]);
    }
    if (in && p.gate_form == DGXM_MOD_SAMPLE)
      bn_put(p.g_gate, p.mod_dtype, static_cast<int64_t>(b) * p.width + col, v[2]);
#pragma unroll
    for (int j = 0; j < 6; ++j) all[j] += v[j];
  };
  for (int b = many ? warp : 0; b < p.batch; b += many ? kBnSumWarps : 1) {
    float s[3] = {0.f, 0.f, 0.f};
    // The blocks that hold rows of this sample: block i has rows [i rows / blocks, (i + 1) rows / blocks).
    int64_t lo = 0, hi = 0;
    if (p.rows > 0) {
      const int64_t r0 = static_cast<int64_t>(b) * p.seq, r1 = r0 + p.seq - 1;
      lo = ((r0 + 1) * p.blocks - 1) / p.rows;
      hi = ((r1 + 1) * p.blocks - 1) / p.rows + 1;
    }
    const int64_t i0 = many ? lo : lo + (hi - lo) * warp / kBnSumWarps;
    const int64_t i1 = many ? hi : lo + (hi - lo) * (warp + 1) / kBnSumWarps;
    if (in) {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        if (!(p.want >> j & 1)) continue;
        const float* from = p.partial + ((i0 + b) * 3 + j) * p.width + col;
#pragma unroll 4
        for (int64_t i = i0; i < i1; ++i, from += 3 * static_cast<int64_t>(p.width)) s[j] += *from;
      }
    }
    if (many) {
      finish(b, s);
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j) part[warp][j][lane] = s[j];
      __syncthreads();
      if (warp == 0) {
        float t[3] = {0.f, 0.f, 0.f};
        for (int k = 0; k < kBnSumWarps; ++k)
#pragma unroll
          for (int j = 0; j < 3; ++j) t[j] += part[k][j][lane];
        finish(b, t);
      }
      __syncthreads();
    }
  }
  if (many) {
#pragma unroll
    for (int j = 0; j < 6; ++j) part[warp][j][lane] = all[j];
    __syncthreads();
    if (warp == 0)
#pragma unroll
      for (int j = 0; j < 6; ++j) {
        all[j] = 0.f;
        for (int k = 0; k < kBnSumWarps; ++k) all[j] += part[k][j][lane];
      }
  }
  if (warp != 0 || !in) return;
  if (p.mod_form == DGXM_MOD_SHARED) {
    bn_put(p.g_shift, p.mod_dtype, col, all[0]);
    bn_put(p.g_scale, p.mod_dtype, col, all[1]);
  }
  if (p.gate_form == DGXM_MOD_SHARED) bn_put(p.g_gate, p.mod_dtype, col, all[2]);
  bn_put(p.g_norm_b, p.weight_dtype, col, all[3]);
  bn_put(p.g_norm_w, p.weight_dtype, col, all[4]);
  bn_put(p.g_branch_w, p.weight_dtype, col, all[5]);
}

static int bn_check(const dgxm_block_norm_desc* d) {
  if (d == nullptr) return fail(DGXM_ERR_INVALID, "NULL block norm descriptor");
  if (d->batch < 0 || d->seq < 0) return fail(DGXM_ERR_INVALID, "negative sizes (%d, %d)", d->batch, d->seq);
  if (d->width <= 0 || d->width > kBnMaxWidth)
    return fail(DGXM_ERR_UNSUPPORTED, "width %d (1 to %d)", d->width, kBnMaxWidth);
  if (d->dtype != DGXM_DTYPE_BF16 && d->dtype != DGXM_DTYPE_F16 && d->dtype != DGXM_DTYPE_F32)
    return fail(DGXM_ERR_UNSUPPORTED, "dtype %d (bf16, f16 or f32)", d->dtype);
  for (int t : {d->weight_dtype, d->mod_dtype})
    if (t != d->dtype && t != DGXM_DTYPE_F32)
      return fail(DGXM_ERR_UNSUPPORTED, "weight or modulation dtype %d (the tensors' or f32)", t);
  if (d->norm_mode != DGXM_BLOCK_NORM_NONE && d->norm_mode != DGXM_BLOCK_NORM_LAYER && d->norm_mode != DGXM_BLOCK_NORM_RMS)
    return fail(DGXM_ERR_UNSUPPORTED, "norm mode %d", d->norm_mode);
  for (int f : {d->gate_form, d->mod_form})
    if (f < DGXM_MOD_NONE || f > DGXM_MOD_TOKEN) return fail(DGXM_ERR_INVALID, "modulation form %d", f);
  if (!(d->eps >= 0.f)) return fail(DGXM_ERR_INVALID, "eps must not be negative or NaN");
  if (d->norm_mode == DGXM_BLOCK_NORM_NONE && d->mod_form != DGXM_MOD_NONE)
    return fail(DGXM_ERR_INVALID, "a scale or shift without a norm");
  return DGXM_OK;
}

static int64_t bn_rows(const dgxm_block_norm_desc* d) { return static_cast<int64_t>(d->batch) * d->seq; }

// How a call is cut: chunks a thread, threads of a block, blocks.
struct BnCut {
  int chunks, threads, blocks;
};

static BnCut bn_cut(const dgxm_block_norm_desc* d, bool back) {
  const int ch = d->dtype == DGXM_DTYPE_F32 ? 4 : 8;
  const int total = (d->width + ch - 1) / ch;
  BnCut cut;
  cut.chunks = total <= 1024 ? 1 : 2;
  cut.threads = ((total + cut.chunks - 1) / cut.chunks + 31) / 32 * 32;
  const int per_sm = std::max(1, (back ? 1024 : 2048) / cut.threads);
  cut.blocks = static_cast<int>(std::min<int64_t>(bn_rows(d), 148 * std::min(per_sm, 16)));
  return cut;
}

static int64_t bn_partial_bytes(const dgxm_block_norm_desc* d) {
  return (bn_cut(d, true).blocks + static_cast<int64_t>(d->batch)) * 3 * d->width * 4;
}

// What both directions share of the parameters.
static void bn_common(const dgxm_block_norm_desc* d, BlockNormParams* p) {
  memset(p, 0, sizeof(*p));
  p->batch = d->batch;
  p->seq = d->seq;
  p->width = d->width;
  p->mode = d->norm_mode;
  p->branch_norm = d->branch_norm != 0;
  p->rows = bn_rows(d);
  p->eps = d->eps;
  p->inv_width = 1.f / d->width;
  p->mod_f32 = d->mod_dtype == DGXM_DTYPE_F32;
  p->w_f32 = d->weight_dtype == DGXM_DTYPE_F32;
}

static int bn_elt(int dtype) { return dtype == DGXM_DTYPE_F32 ? 4 : 2; }

static void bn_stream(BlockNormParams* p, int s, const void* base, const int64_t (&stride)[2], int dtype) {
  p->in[s] = static_cast<const char*>(base);
  p->in_sb[s] = stride[0] * bn_elt(dtype);
  p->in_sr[s] = stride[1] * bn_elt(dtype);
  p->in_f32[s] = dtype == DGXM_DTYPE_F32;
}

// Place the streams in the stage; whole chunks of the widest.
static void bn_layout(const dgxm_block_norm_desc* d, BlockNormParams* p, int n_in) {
  const int ch = d->dtype == DGXM_DTYPE_F32 ? 4 : 8;
  const int padded = (d->width + ch - 1) / ch * ch;
  p->n_in = n_in;
  int at = 0;
  for (int s = 0; s < n_in; ++s) {
    if (p->in[s] == nullptr) continue;
    p->in_off[s] = at;
    p->in_pitch[s] = padded * (p->in_f32[s] ? 4 : 2);
    at += p->in_pitch[s];
  }
  p->stage_bytes = at;
}

static int bn_aligned(std::initializer_list<const void*> ptrs, int elt, const char* what) {
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % elt) return fail(DGXM_ERR_INVALID, "%s not aligned to its elements", what);
  return DGXM_OK;
}

template <typename T, int NV>
static int bn_launch_as(bool back, const BnCut& cut, const BlockNormParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> done[2] = {};
  auto kernel = back ? block_norm_backward_kernel<T, NV> : block_norm_kernel<T, NV>;
  if (p.stage_bytes > 48 * 1024) DGXM_CUDA_TRY(set_smem_limit_once(kernel, 224 * 1024, done[back]));
  kernel<<<cut.blocks, cut.threads, p.stage_bytes, st>>>(p);
  DGXM_CUDA_TRY(cudaGetLastError());
  return DGXM_OK;
}

template <typename T>
static int bn_launch(bool back, const BnCut& cut, const BlockNormParams& p, cudaStream_t st) {
  if (cut.chunks == 1) return bn_launch_as<T, 1>(back, cut, p, st);
  return bn_launch_as<T, 2>(back, cut, p, st);

}

static int bn_run(const dgxm_block_norm_desc* d, bool back, const BnCut& cut, const BlockNormParams& p, cudaStream_t st) {
  if (d->dtype == DGXM_DTYPE_BF16) return bn_launch<__nv_bfloat16>(back, cut, p, st);
  if (d->dtype == DGXM_DTYPE_F16) return bn_launch<__half>(back, cut, p, st);
  return bn_launch<float>(back, cut, p, st);
}

}  // namespace dgxm

extern "C" int dgxm_block_norm(const dgxm_block_norm_desc* d, const void* x, const void* branch, const void* gate,
                               const void* scale, const void* shift, const void* norm_w, const void* norm_b,
                               const void* branch_w, void* x_out, void* out, void* stream) {
  using namespace dgxm;
  if (int rc = bn_check(d)) return rc;
  if (bn_rows(d) == 0) return DGXM_OK;  // empty tensors may be NULL
  const bool norm = d->norm_mode != DGXM_BLOCK_NORM_NONE;
  if ((branch == nullptr) != (x_out == nullptr)) return fail(DGXM_ERR_INVALID, "a branch and x_out come together");
  if (norm != (out != nullptr)) return fail(DGXM_ERR_INVALID, "out comes with a norm, and only then");
  if (!norm && branch == nullptr) return fail(DGXM_ERR_INVALID, "neither a norm nor a branch");
  if (branch == nullptr && (gate != nullptr || d->branch_norm || branch_w != nullptr))
    return fail(DGXM_ERR_INVALID, "a gate or a branch norm without a branch");
  if (branch_w != nullptr && !d->branch_norm) return fail(DGXM_ERR_INVALID, "branch_w without a branch norm");
  if (!norm && (norm_w != nullptr || norm_b != nullptr)) return fail(DGXM_ERR_INVALID, "norm weights without a norm");
  if (norm_b != nullptr && d->norm_mode == DGXM_BLOCK_NORM_RMS)
    return fail(DGXM_ERR_INVALID, "norm_b goes with the layer norm");
  if ((gate != nullptr) != (d->gate_form != DGXM_MOD_NONE)) return fail(DGXM_ERR_INVALID, "gate and gate_form do not match");
  if ((scale != nullptr || shift != nullptr) != (d->mod_form != DGXM_MOD_NONE))
    return fail(DGXM_ERR_INVALID, "scale, shift and mod_form do not match");
  if (x == nullptr) return fail(DGXM_ERR_INVALID, "NULL x");
  if (int rc = bn_aligned({x, branch, x_out, out}, bn_elt(d->dtype), "x, branch or an output is")) return rc;
  if (int rc = bn_aligned({gate, scale, shift}, bn_elt(d->mod_dtype), "a modulation is")) return rc;
  if (int rc = bn_aligned({norm_w, norm_b, branch_w}, bn_elt(d->weight_dtype), "a weight is")) return rc;
  BlockNormParams p;
  bn_common(d, &p);
  bn_stream(&p, kBnX, x, d->x_stride, d->dtype);
  bn_stream(&p, kBnBranch, branch, d->branch_stride, d->dtype);
  const int me = bn_elt(d->mod_dtype);
  if (d->gate_form == DGXM_MOD_TOKEN) {
    bn_stream(&p, kBnGate, gate, d->gate_stride, d->mod_dtype);
  } else if (gate != nullptr) {
    p.gate = static_cast<const char*>(gate);
    p.gate_sb = d->gate_form == DGXM_MOD_SAMPLE ? d->gate_stride[0] * me : 0;
  }
  if (d->mod_form == DGXM_MOD_TOKEN) {
    bn_stream(&p, kBnScale, scale, d->scale_stride, d->mod_dtype);
    bn_stream(&p, kBnShift, shift, d->shift_stride, d->mod_dtype);
  } else {
    p.scale = static_cast<const char*>(scale);
    p.shift = static_cast<const char*>(shift);
    p.scale_sb = d->mod_form == DGXM_MOD_SAMPLE ? d->scale_stride[0] * me : 0;
    p.shift_sb = d->mod_form == DGXM_MOD_SAMPLE ? d->shift_stride[0] * me : 0;
  }
  p.norm_w = static_cast<const char*>(norm_w);
  p.norm_b = static_cast<const char*>(norm_b);
  p.branch_w = static_cast<const char*>(branch_w);
  p.x_out = static_cast<char*>(x_out);
  p.out = static_cast<char*>(out);
  const int e = bn_elt(d->dtype);
  p.x_out_sb = d->x_out_stride[0] * e;
  p.x_out_sr = d->x_out_stride[1] * e;
  p.out_sb = d->out_stride[0] * e;
  p.out_sr = d->out_stride[1] * e;
  bn_layout(d, &p, 5);
  return bn_run(d, false, bn_cut(d, false), p, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t dgxm_block_norm_backward_workspace(const dgxm_block_norm_desc* d) {
  using namespace dgxm;
  if (bn_check(d)) return -1;
  return bn_rows(d) == 0 ? 0 : bn_partial_bytes(d);
}

extern "C" int dgxm_block_norm_backward(const dgxm_block_norm_desc* d, const dgxm_block_norm_grads* g, const void* dy,
                                        const void* dx_out, const void* x_out, const void* branch, const void* gate,
                                        const void* scale, const void* norm_w, const void* norm_b, const void* branch_w,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dgxm;
  if (int rc = bn_check(d)) return rc;
  if (g == nullptr) return fail(DGXM_ERR_INVALID, "NULL gradients");
  const bool norm = d->norm_mode != DGXM_BLOCK_NORM_NONE;
  const int64_t rows = bn_rows(d);
  if (rows > 0) {  // empty tensors may be NULL
    if (norm && g->x == nullptr) return fail(DGXM_ERR_INVALID, "NULL gradient of x");
    if (branch == nullptr && (gate != nullptr || d->branch_norm || branch_w != nullptr || g->branch != nullptr ||
                              g->gate != nullptr || g->branch_w != nullptr))
      return fail(DGXM_ERR_INVALID, "a gate, a branch norm or their gradients without a branch");
    if ((branch_w != nullptr || g->branch_w != nullptr) && !d->branch_norm)
      return fail(DGXM_ERR_INVALID, "branch_w without a branch norm");
    if (!norm && (norm_w != nullptr || norm_b != nullptr || g->norm_w != nullptr || g->norm_b != nullptr))
      return fail(DGXM_ERR_INVALID, "norm weights without a norm");
    if ((norm_b != nullptr || g->norm_b != nullptr) && d->norm_mode == DGXM_BLOCK_NORM_RMS)
      return fail(DGXM_ERR_INVALID, "norm_b goes with the layer norm");
    if ((gate != nullptr) != (d->gate_form != DGXM_MOD_NONE) || (gate == nullptr && g->gate != nullptr))
      return fail(DGXM_ERR_INVALID, "gate, gate_form and the gate's gradient do not match");
    if (d->mod_form == DGXM_MOD_NONE && (scale != nullptr || g->scale != nullptr || g->shift != nullptr))
      return fail(DGXM_ERR_INVALID, "scale, shift and mod_form do not match");
    if (g->scale != nullptr && scale == nullptr) return fail(DGXM_ERR_INVALID, "the gradient of a scale without the scale");
  }
  const int me = bn_elt(d->mod_dtype), we = bn_elt(d->weight_dtype), e = bn_elt(d->dtype);
  if (int rc = bn_aligned({dy, dx_out, x_out, branch, g->x, g->branch}, e, "a tensor is")) return rc;
  if (int rc = bn_aligned({gate, scale, g->gate, g->scale, g->shift}, me, "a modulation is")) return rc;
  if (int rc = bn_aligned({norm_w, norm_b, branch_w, g->norm_w, g->norm_b, g->branch_w}, we, "a weight is")) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  BlockNormParams p;
  bn_common(d, &p);
  const bool tok_gate = d->gate_form == DGXM_MOD_TOKEN, tok_mod = d->mod_form == DGXM_MOD_TOKEN;
  const bool sum_shift = !tok_mod && g->shift != nullptr, sum_scale = !tok_mod && g->scale != nullptr;
  const bool sum_gate = !tok_gate && g->gate != nullptr;
  p.want = ((sum_shift || g->norm_b != nullptr || (sum_scale && norm_b != nullptr)) ? 1 : 0) |
           ((sum_scale || g->norm_w != nullptr) ? 2 : 0) | ((sum_gate || g->branch_w != nullptr) ? 4 : 0);
  int blocks = 0;
  if (rows > 0) {  // else the sums of nothing
    if (norm && (dy == nullptr || x_out == nullptr)) return fail(DGXM_ERR_INVALID, "NULL upstream gradient or x_out");
    if (!norm && dx_out == nullptr) return fail(DGXM_ERR_INVALID, "neither a norm nor an upstream gradient of x_out");
    if (p.want) {
      const int64_t need = bn_partial_bytes(d);
      if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 4 || workspace_bytes < need)
        return fail(DGXM_ERR_INVALID, "workspace of %lld bytes (%lld needed)", (long long)workspace_bytes, (long long)need);
      p.partial = static_cast<float*>(workspace);
    }
    bn_stream(&p, kBnDy, norm ? dy : nullptr, d->dy_stride, d->dtype);
    bn_stream(&p, kBnDr, dx_out, d->dx_out_stride, d->dtype);
    bn_stream(&p, kBnR, norm ? x_out : nullptr, d->x_stride, d->dtype);
    const bool apart = gate != nullptr || d->branch_norm;  // the branch's gradient is not the stream's
    if (apart) bn_stream(&p, kBnBranchB, branch, d->branch_stride, d->dtype);
    if (tok_gate) {
      bn_stream(&p, kBnGateB, gate, d->gate_stride, d->mod_dtype);
      p.g_gate = static_cast<char*>(g->gate);
    } else {
      p.gate = static_cast<const char*>(gate);
      p.gate_sb = d->gate_form == DGXM_MOD_SAMPLE ? d->gate_stride[0] * me : 0;
    }
    if (tok_mod) {
      if (scale != nullptr) bn_stream(&p, kBnScaleB, scale, d->scale_stride, d->mod_dtype);
      p.g_scale = static_cast<char*>(g->scale);
      p.g_shift = static_cast<char*>(g->shift);
    } else {
      p.scale = static_cast<const char*>(scale);
      p.scale_sb = d->mod_form == DGXM_MOD_SAMPLE ? d->scale_stride[0] * me : 0;
    }
    p.norm_w = static_cast<const char*>(norm_w);
    p.norm_b = static_cast<const char*>(norm_b);
    p.branch_w = static_cast<const char*>(branch_w);
    p.x_out = static_cast<char*>(g->x);
    p.out = apart ? static_cast<char*>(g->branch) : nullptr;
    p.x_out_sb = d->x_out_stride[0] * e;
    p.x_out_sr = d->x_out_stride[1] * e;
    p.out_sb = d->out_stride[0] * e;
    p.out_sr = d->out_stride[1] * e;
    if (!apart && g->branch != nullptr) return fail(DGXM_ERR_INVALID, "the branch's gradient is that of x: pass NULL");
    bn_layout(d, &p, 6);
    const BnCut cut = bn_cut(d, true);
    blocks = cut.blocks;
    if (int rc = bn_run(d, true, cut, p, st)) return rc;
  }
  if (!p.want) return DGXM_OK;
  BlockNormSumParams sp;
  memset(&sp, 0, sizeof(sp));
  sp.partial = p.partial;
  sp.gate = tok_gate ? nullptr : static_cast<const char*>(gate);
  sp.scale = tok_mod ? nullptr : static_cast<const char*>(scale);
  sp.gate_sb = d->gate_form == DGXM_MOD_SAMPLE ? d->gate_stride[0] * me : 0;
  sp.scale_sb = d->mod_form == DGXM_MOD_SAMPLE ? d->scale_stride[0] * me : 0;
  sp.norm_w = static_cast<const char*>(norm_w);
  sp.norm_b = static_cast<const char*>(norm_b);
  sp.branch_w = static_cast<const char*>(branch_w);
  sp.g_gate = g->gate;
  sp.g_scale = g->scale;
  sp.g_shift = g->shift;
  sp.g_norm_w = g->norm_w;
  sp.g_norm_b = g->norm_b;
  sp.g_branch_w = g->branch_w;
  sp.gate_form = d->gate_form;
  sp.mod_form = d->mod_form;
  sp.want = p.want;
  sp.dtype = d->dtype;
  sp.mod_dtype = d->mod_dtype;
  sp.weight_dtype = d->weight_dtype;
  sp.batch = d->batch;
  sp.seq = d->seq;
  sp.width = d->width;
  sp.blocks = blocks;
  sp.rows = rows;
  block_norm_sum_kernel<<<(d->width + 31) / 32, kBnSumWarps * 32, 0, st>>>(sp);
  DGXM_CUDA_TRY(cudaGetLastError());
  return DGXM_OK;
}
