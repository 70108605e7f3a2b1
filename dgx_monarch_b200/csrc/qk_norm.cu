// RMSNorm of every query and key head with the rotary position embedding in
// the same pass, on local tensors of any stride, and its gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R (n w)
//   with R the rotation by the token's angles, and for an upstream gradient dy
//   g = R^T dy,  dw = sum over rows of g n,
//   dx = r (g w - n mean(g w n)).
//
// Both directions move each value once and compute a handful of operations
// on it, so DRAM bounds them.  A head row is held by a group of 8, 16 or 32
// lanes, eight values a lane (16 bytes of a 16-bit type), so a warp reads and
// writes whole 32-byte sectors whatever the strides, the sums of a row are
// shuffles within the group, and a row stays in registers between its load
// and its store.  One warp takes several heads of one token: the token's
// cosines and sines and the head weight are loaded once for all of them, and
// the loads of kFwdRows (kBwdRows) rows are in flight together.
//
// Everything between the load and the store is fp32 and is rounded once, to
// the tensors' type.  (The fused scatter of prologue.cu rounds after the
// norm and after the weight as well, as the separate modules it replaces do.)
#include "common.h"
#include "ptx.cuh"

namespace dgxm {

constexpr int kQkThreads = 256;
constexpr int kQkWarps = kQkThreads / 32;
constexpr int kFwdRows = 4;  // rows of a lane group in flight, forward
constexpr int kBwdRows = 2;  // backward: two tensors are read for each row

struct QkNormParams {
  // [0] q, [1] k; strides in elements: batch, row, head
  const char* x[2];
  const char* dy[2];
  char* out[2];  // forward: y; backward: dx
  const void* w[2];
  int64_t xs[2][3], ds[2][3], os[2][3];
  const float* rope;  // (seq, rot / 2, 2) cosines and sines, or NULL
  int64_t rope_sb;    // floats between batch items (0: shared)
  float* partial;     // backward: (grid, 2, head_dim) sums of g n, or NULL
  int heads[2], chunks[2];  // chunks: warps for one token's heads of the tensor
  uint32_t seq, items;      // items: batch * seq * (chunks of q + chunks of k)
  int dim, rot, halves, norm, w_f32, rope_vec;
  float eps, inv_dim;
};

template <typename T>
__device__ __forceinline__ float qk_widen(T v);
template <>
__device__ __forceinline__ float qk_widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float qk_widen(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float qk_widen(float v) { return v; }

template <typename T>
__device__ __forceinline__ T qk_narrow(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 qk_narrow(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half qk_narrow(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float qk_narrow(float v) { return v; }

// Eight values as they lie in memory.  VEC: 16-byte accesses (base and every
// stride a multiple of 16 bytes); otherwise one access a value.
template <typename T>
struct __align__(16) Qk8 {
  T v[8];
};

template <typename T, bool VEC>
__device__ __forceinline__ Qk8<T> qk_load(const char* base, int64_t elem) {
  Qk8<T> r;
  const T* p = reinterpret_cast<const T*>(base) + elem;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i)
      reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = p[i];
  }
  return r;
}

template <typename T, bool VEC>
__device__ __forceinline__ void qk_store(char* base, int64_t elem, const float (&y)[8]) {
  Qk8<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = qk_narrow<T>(y[i]);
  T* p = reinterpret_cast<T*>(base) + elem;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&r)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = r.v[i];
  }
}

template <int G>
__device__ __forceinline__ float qk_group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What one warp works on: `first` .. of the heads of tensor t at one token.
struct QkItem {
  int t, first;
  uint32_t b, l;
};

__device__ __forceinline__ QkItem qk_item(const QkNormParams& p, uint32_t item, int rows_per_item) {
  QkItem r;
  const uint32_t per = p.chunks[0] + p.chunks[1];
  const uint32_t token = item / per;
  int c = static_cast<int>(item - token * per);
  r.t = c >= p.chunks[0];
  if (r.t) c -= p.chunks[0];
  r.first = c * rows_per_item;
  r.b = token / p.seq;
  r.l = token - r.b * p.seq;
  return r;
}

// Lane `sub` of a group holds values e = 8 sub + i of its row.  The rotation
// of either order is y_e = x_e c_e + x_partner s_e with the sign in s_e:
//   adjacent: pair e / 2, partner e ^ 1, the even value's sine negative;
//   halves:   pair e mod rot / 2, partner e +- rot / 2, the first half's
//             sine negative.
// SIGN = -1 gives the transposed rotation.
template <int SIGN>
__device__ __forceinline__ void qk_angles(const QkNormParams& p, const QkItem& it, int sub, float (&c)[8],
                                          float (&s)[8]) {
  const float* row = p.rope + it.b * p.rope_sb + static_cast<int64_t>(it.l) * p.rot;
  const int e0 = 8 * sub, half = p.rot / 2;
  if (!p.halves) {
    if (p.rope_vec && e0 + 8 <= p.rot) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(row + e0) + i);
        c[4 * i] = c[4 * i + 1] = v.x;
        c[4 * i + 2] = c[4 * i + 3] = v.z;
        s[4 * i] = -SIGN * v.y;
        s[4 * i + 1] = SIGN * v.y;
        s[4 * i + 2] = -SIGN * v.w;
        s[4 * i + 3] = SIGN * v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const bool in = e0 + i < p.rot;
        c[i] = c[i + 1] = in ? __ldg(row + e0 + i) : 1.f;
        const float v = in ? __ldg(row + e0 + i + 1) : 0.f;
        s[i] = -SIGN * v;
        s[i + 1] = SIGN * v;
      }
    }
  } else if (p.rope_vec && half % 8 == 0 && e0 + 8 <= p.rot) {
    const bool low = e0 < half;
    const float4* v4 = reinterpret_cast<const float4*>(row + 2 * (low ? e0 : e0 - half));
    const float sg = low ? -SIGN : SIGN;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = __ldg(v4 + i);
      c[2 * i] = v.x;
      s[2 * i] = sg * v.y;
      c[2 * i + 1] = v.z;
      s[2 * i + 1] = sg * v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = e0 + i;
      const bool in = e < p.rot, low = e < half;
      const int a = low ? e : e - half;
      c[i] = in ? __ldg(row + 2 * a) : 1.f;
      const float v = in ? __ldg(row + 2 * a + 1) : 0.f;
      s[i] = low ? -SIGN * v : SIGN * v;
    }
  }
}

// Rotate a lane's eight values.  Values past `rot` stay as they are (a
// product with a zero sine would turn an infinite neighbour into NaN).  The
// halves order meets its partners in `buf`, the warp's 256 floats.
__device__ __forceinline__ void qk_rotate(const QkNormParams& p, int sub, int lane, const float (&c)[8],
                                          const float (&s)[8], float* buf, float (&y)[8]) {
  const int e0 = 8 * sub;
  float q[8];
  if (!p.halves) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = y[i ^ 1];
  } else {
    const int half = p.rot / 2;
    float* mine = buf + lane * 8;
    __syncwarp();
    reinterpret_cast<float4*>(mine)[0] = make_float4(y[0], y[1], y[2], y[3]);
    reinterpret_cast<float4*>(mine)[1] = make_float4(y[4], y[5], y[6], y[7]);
    __syncwarp();
    if (half % 4 == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = e0 + 4 * i;
        const int d = e < half ? half : e < p.rot ? -half : 0;
        const float4 v = *reinterpret_cast<const float4*>(mine + 4 * i + d);
        q[4 * i] = v.x;
        q[4 * i + 1] = v.y;
        q[4 * i + 2] = v.z;
        q[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        q[i] = mine[i + (e < half ? half : e < p.rot ? -half : 0)];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = fmaf(q[i], s[i], y[i] * c[i]);
    y[i] = e0 + i < p.rot ? v : y[i];
  }
}

template <typename T>
__device__ __forceinline__ void qk_weight(const QkNormParams& p, int t, int sub, bool in, float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (p.w[t] == nullptr || !in) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = p.w_f32 ? __ldg(static_cast<const float*>(p.w[t]) + 8 * sub + i)
                   : qk_widen<T>(static_cast<const T*>(p.w[t])[8 * sub + i]);
}

// One warp per (token, tensor, chunk of kFwdRows rows a lane group).
template <typename T, int G, bool VEC>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_kernel(const __grid_constant__ QkNormParams p) {
  constexpr int kGroups = 32 / G;
  __shared__ float stage[kQkWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t item = blockIdx.x * kQkWarps + warp;
  if (item >= p.items) return;
  const QkItem it = qk_item(p, item, kFwdRows * kGroups);
  const int sub = lane % G, group = lane / G, t = it.t;
  const bool in = 8 * sub < p.dim;
  const char* x = p.x[t];
  const int64_t x0 = it.b * p.xs[t][0] + it.l * p.xs[t][1] + 8 * sub;
  const int64_t o0 = it.b * p.os[t][0] + it.l * p.os[t][1] + 8 * sub;
  Qk8<T> raw[kFwdRows];
#pragma unroll
  for (int u = 0; u < kFwdRows; ++u) {
    const int h = it.first + u * kGroups + group;
    if (in && h < p.heads[t]) {
      raw[u] = qk_load<T, VEC>(x, x0 + h * p.xs[t][2]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[u].v[i] = qk_narrow<T>(0.f);
    }
  }
  float w[8], c[8], s[8];
  if (p.norm) qk_weight<T>(p, t, sub, in, w);
  if (p.rope != nullptr) qk_angles<1>(p, it, sub, c, s);
#pragma unroll
  for (int u = 0; u < kFwdRows; ++u) {
    if (it.first + u * kGroups >= p.heads[t]) break;  // uniform over the warp
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = qk_widen<T>(raw[u].v[i]);
    if (p.norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
      const float r = rsqrtf(fmaf(qk_group_sum<G>(ss), p.inv_dim, p.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * r * w[i];
    }
    if (p.rope != nullptr) qk_rotate(p, sub, lane, c, s, stage[warp], y);
    const int h = it.first + u * kGroups + group;
    if (in && h < p.heads[t]) qk_store<T, VEC>(p.out[t], o0 + h * p.os[t][2], y);
  }
}

// Gradients.  The blocks stride over the items; each lane adds g n of its
// eight columns over all the rows it meets, q's and k's apart, the block sums
// its warps in a fixed order, and qk_weight_grad_kernel sums the blocks: no
// atomics, so the same call gives the same bits.
template <typename T, int G, bool VEC>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_bwd_kernel(const __grid_constant__ QkNormParams p) {
  constexpr int kGroups = 32 / G;
  __shared__ float stage[kQkWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % G, group = lane / G;
  const bool in = 8 * sub < p.dim;
  float dw[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[0][i] = dw[1][i] = 0.f;
  const uint32_t step = gridDim.x * kQkWarps;
  for (uint32_t item = blockIdx.x * kQkWarps + warp; item < p.items; item += step) {
    const QkItem it = qk_item(p, item, kBwdRows * kGroups);
    const int t = it.t;
    const int64_t x0 = it.b * p.xs[t][0] + it.l * p.xs[t][1] + 8 * sub;
    const int64_t d0 = it.b * p.ds[t][0] + it.l * p.ds[t][1] + 8 * sub;
    const int64_t o0 = it.b * p.os[t][0] + it.l * p.os[t][1] + 8 * sub;
    Qk8<T> xr[kBwdRows], dr[kBwdRows];
#pragma unroll
    for (int u = 0; u < kBwdRows; ++u) {
      const int h = it.first + u * kGroups + group;
      if (in && h < p.heads[t]) {
        dr[u] = qk_load<T, VEC>(p.dy[t], d0 + h * p.ds[t][2]);
        if (p.norm) xr[u] = qk_load<T, VEC>(p.x[t], x0 + h * p.xs[t][2]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) xr[u].v[i] = dr[u].v[i] = qk_narrow<T>(0.f);
      }
    }
    float w[8], c[8], s[8];
    if (p.norm) qk_weight<T>(p, t, sub, in, w);
    if (p.rope != nullptr) qk_angles<-1>(p, it, sub, c, s);
#pragma unroll
    for (int u = 0; u < kBwdRows; ++u) {
      if (it.first + u * kGroups >= p.heads[t]) break;  // uniform over the warp
      const int h = it.first + u * kGroups + group;
      const bool mine = in && h < p.heads[t];
      float g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = qk_widen<T>(dr[u].v[i]);
      if (p.rope != nullptr) qk_rotate(p, sub, lane, c, s, stage[warp], g);
      if (p.norm) {
        float x[8], xx = 0.f, gx = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = qk_widen<T>(xr[u].v[i]);
          xx = fmaf(x[i], x[i], xx);
          gx = fmaf(g[i] * w[i], x[i], gx);
        }
        xx = qk_group_sum<G>(xx);
        gx = qk_group_sum<G>(gx);
        const float r = rsqrtf(fmaf(xx, p.inv_dim, p.eps));
        const float m = gx * r * p.inv_dim;  // mean(g w n)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n = x[i] * r;
          if (mine) dw[t][i] = fmaf(g[i], n, dw[t][i]);
          g[i] = r * fmaf(-n, m, g[i] * w[i]);
        }
      }
      if (mine) qk_store<T, VEC>(p.out[t], o0 + h * p.os[t][2], g);
    }
  }
  if (p.partial == nullptr) return;  // uniform over the grid
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = dw[t][i];
#pragma unroll
      for (int o = G; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (group == 0 && in) stage[warp][8 * sub + i] = v;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.dim; e += kQkThreads) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kQkWarps; ++k) v += stage[k][e];
      p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + t) * p.dim + e] = v;
    }
  }
}

struct QkWeightGradParams {
  const float* partial;
  void* out[2];
  int blocks, dim, dtype;
};

// Sum of the blocks' partial sums: 32 columns a block, eight warps over the
// rows, then the warps in order.
__global__ void __launch_bounds__(256) qk_weight_grad_kernel(const __grid_constant__ QkWeightGradParams p) {
  __shared__ float part[8][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * 32 + lane;  // over q | k
  float v = 0.f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (col < 2 * p.dim)
    for (int b = warp; b < p.blocks; b += 8) v += p.partial[static_cast<int64_t>(b) * 2 * p.dim + col];
  part[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || col >= 2 * p.dim) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v += part[k][lane];
  const int t = col >= p.dim, e = col - t * p.dim;
  if (p.out[t] == nullptr) return;
  if (p.dtype == DGXM_DTYPE_F32) static_cast<float*>(p.out[t])[e] = v;
  else if (p.dtype == DGXM_DTYPE_F16) static_cast<__half*>(p.out[t])[e] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p.out[t])[e] = __float2bfloat16_rn(v);
}

static int qk_group(int dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }

// Blocks of the backward kernel: six of 256 threads fit an SM's registers.
static int qk_bwd_blocks(const dgxm_qk_norm_desc* d, int rows_per_item, int sms, int64_t* items) {
  const int64_t per = (d->q_heads + rows_per_item - 1) / rows_per_item + (d->k_heads + rows_per_item - 1) / rows_per_item;
  *items = static_cast<int64_t>(d->batch) * d->seq * per;
  return static_cast<int>(std::min<int64_t>((*items + kQkWarps - 1) / kQkWarps, int64_t(sms) * 6));
}

static int qk_check(const dgxm_qk_norm_desc* d) {
  if (d == nullptr) return fail(DGXM_ERR_INVALID, "NULL Q/K norm descriptor");
  if (d->batch < 0 || d->seq < 0 || d->q_heads < 0 || d->k_heads < 0)
    return fail(DGXM_ERR_INVALID, "negative extents: batch %d, rows %d, heads %d / %d", d->batch, d->seq, d->q_heads,
                d->k_heads);
  if (d->head_dim <= 0 || d->head_dim % 8 || d->head_dim > 256)
    return fail(DGXM_ERR_UNSUPPORTED, "head_dim %d is not a multiple of 8 up to 256", d->head_dim);
  if (d->rot_dim < 0 || d->rot_dim % 2 || d->rot_dim > d->head_dim)
    return fail(DGXM_ERR_INVALID, "rot_dim %d is not even or above head_dim %d", d->rot_dim, d->head_dim);
  if (d->dtype != DGXM_DTYPE_BF16 && d->dtype != DGXM_DTYPE_F16 && d->dtype != DGXM_DTYPE_F32)
    return fail(DGXM_ERR_UNSUPPORTED, "dtype %d (bf16, f16 or f32)", d->dtype);
  if (d->weight_dtype != d->dtype && d->weight_dtype != DGXM_DTYPE_F32)
    return fail(DGXM_ERR_UNSUPPORTED, "weight dtype %d with dtype %d (the same, or f32)", d->weight_dtype, d->dtype);
  if (d->norm_mode != DGXM_NORM_NONE && d->norm_mode != DGXM_NORM_HEAD)
    return fail(DGXM_ERR_UNSUPPORTED, "norm mode %d (none or per head)", d->norm_mode);
  if (!(d->eps >= 0.f) || d->eps > 3e38f) return fail(DGXM_ERR_INVALID, "eps must be finite and not negative");
  return DGXM_OK;
}

// Fill the kernel parameters that both directions share; *vec says whether
// every access may be 16 bytes wide.
static int qk_params(const dgxm_qk_norm_desc* d, const void* const (&x)[2], const void* const (&dy)[2],
                     void* const (&out)[2], const void* const (&w)[2], const float* rope, int rows_per_item,
                     QkNormParams* p, bool* vec) {
  memset(p, 0, sizeof(*p));
  const int elt = d->dtype == DGXM_DTYPE_F32 ? 4 : 2;
  const bool back = dy[0] != nullptr || dy[1] != nullptr;
  uintptr_t bits = 0;
  for (int t = 0; t < 2; ++t) {
    p->heads[t] = t ? d->k_heads : d->q_heads;
    if (p->heads[t] == 0) continue;
    if (out[t] == nullptr || (back ? dy[t] == nullptr || (d->norm_mode != DGXM_NORM_NONE && x[t] == nullptr)
                                   : x[t] == nullptr))
      return fail(DGXM_ERR_INVALID, "NULL tensor for %s", t ? "k" : "q");
    p->x[t] = static_cast<const char*>(x[t]);
    p->dy[t] = static_cast<const char*>(dy[t]);
    p->out[t] = static_cast<char*>(out[t]);
    p->w[t] = d->norm_mode == DGXM_NORM_NONE ? nullptr : w[t];
    for (int i = 0; i < 3; ++i) {
      p->xs[t][i] = t ? d->k_stride[i] : d->q_stride[i];
      p->ds[t][i] = t ? d->dk_stride[i] : d->dq_stride[i];
      p->os[t][i] = t ? d->k_out_stride[i] : d->q_out_stride[i];
      bits |= static_cast<uintptr_t>(p->os[t][i] * elt);
      if (x[t] != nullptr) bits |= static_cast<uintptr_t>(p->xs[t][i] * elt);
      if (back) bits |= static_cast<uintptr_t>(p->ds[t][i] * elt);
    }
    bits |= reinterpret_cast<uintptr_t>(x[t]) | reinterpret_cast<uintptr_t>(dy[t]) | reinterpret_cast<uintptr_t>(out[t]);
    if ((reinterpret_cast<uintptr_t>(x[t]) | reinterpret_cast<uintptr_t>(dy[t]) | reinterpret_cast<uintptr_t>(out[t])) % elt ||
        reinterpret_cast<uintptr_t>(w[t]) % (d->weight_dtype == DGXM_DTYPE_F32 ? 4 : 2))
      return fail(DGXM_ERR_INVALID, "%s is not aligned to its elements", t ? "k" : "q");
  }
  if (reinterpret_cast<uintptr_t>(rope) % 4) return fail(DGXM_ERR_INVALID, "rope is not aligned to its elements");
  *vec = bits % 16 == 0;
  p->rope = d->rot_dim > 0 ? rope : nullptr;
  p->rope_sb = d->rope_batch_stride;
  p->rope_vec = reinterpret_cast<uintptr_t>(rope) % 16 == 0 && d->rot_dim % 4 == 0 && d->rope_batch_stride % 4 == 0;
  for (int t = 0; t < 2; ++t) p->chunks[t] = (p->heads[t] + rows_per_item - 1) / rows_per_item;
  const int64_t items = static_cast<int64_t>(d->batch) * d->seq * (p->chunks[0] + p->chunks[1]);
  if (items > (int64_t(1) << 31) - 1)
    return fail(DGXM_ERR_UNSUPPORTED, "%lld head groups in one call (up to 2^31 - 1)", (long long)items);
  p->seq = static_cast<uint32_t>(d->seq);
  p->items = static_cast<uint32_t>(items);
  p->dim = d->head_dim;
  p->rot = p->rope != nullptr ? d->rot_dim : 0;
  p->halves = d->rope_halves != 0;
  p->norm = d->norm_mode == DGXM_NORM_HEAD;
  p->w_f32 = d->weight_dtype == DGXM_DTYPE_F32;
  p->eps = d->eps;
  p->inv_dim = 1.f / d->head_dim;
  return DGXM_OK;
}

using QkKernel = void (*)(QkNormParams);

template <bool BACK, typename T, bool VEC>
static QkKernel qk_pick_group(int group) {
  if constexpr (BACK)
    return group == 8 ? qk_norm_rope_bwd_kernel<T, 8, VEC> : group == 16 ? qk_norm_rope_bwd_kernel<T, 16, VEC>
                                                                         : qk_norm_rope_bwd_kernel<T, 32, VEC>;
  else
    return group == 8 ? qk_norm_rope_kernel<T, 8, VEC> : group == 16 ? qk_norm_rope_kernel<T, 16, VEC>
                                                                     : qk_norm_rope_kernel<T, 32, VEC>;
}

template <bool BACK>
static QkKernel qk_pick(int dtype, int group, bool vec) {
  if (dtype == DGXM_DTYPE_BF16)
    return vec ? qk_pick_group<BACK, __nv_bfloat16, true>(group) : qk_pick_group<BACK, __nv_bfloat16, false>(group);
  if (dtype == DGXM_DTYPE_F16)
    return vec ? qk_pick_group<BACK, __half, true>(group) : qk_pick_group<BACK, __half, false>(group);
  return vec ? qk_pick_group<BACK, float, true>(group) : qk_pick_group<BACK, float, false>(group);
}

}  // namespace dgxm

extern "C" int dgxm_qk_norm_rope(const dgxm_qk_norm_desc* d, const void* q, const void* k, const void* norm_q_w,
                                 const void* norm_k_w, const float* rope, void* q_out, void* k_out, void* stream) {
  using namespace dgxm;
  if (int rc = qk_check(d)) return rc;
  if (d->batch == 0 || d->seq == 0 || d->q_heads + d->k_heads == 0) return DGXM_OK;
  const int group = qk_group(d->head_dim), rows = kFwdRows * (32 / group);
  QkNormParams p;
  bool vec = false;
  if (int rc = qk_params(d, {q, k}, {nullptr, nullptr}, {q_out, k_out}, {norm_q_w, norm_k_w}, rope, rows, &p, &vec))
    return rc;
  const unsigned blocks = (p.items + kQkWarps - 1) / kQkWarps;
  qk_pick<false>(d->dtype, group, vec)<<<blocks, kQkThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  DGXM_CUDA_TRY(cudaGetLastError());
  return DGXM_OK;
}

extern "C" int64_t dgxm_qk_norm_rope_backward_workspace(const dgxm_qk_norm_desc* d) {
  using namespace dgxm;
  if (qk_check(d)) return -1;
  int64_t items = 0;
  const int blocks = qk_bwd_blocks(d, kBwdRows * (32 / qk_group(d->head_dim)), 148, &items);
  return std::max<int64_t>(int64_t(blocks) * 2 * d->head_dim * 4, 4);
}

extern "C" int dgxm_qk_norm_rope_backward(const dgxm_qk_norm_desc* d, const void* dq, const void* dk, const void* q,
                                          const void* k, const void* norm_q_w, const void* norm_k_w,
                                          const float* rope, void* gq, void* gk, void* g_norm_q_w, void* g_norm_k_w,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dgxm;
  if (int rc = qk_check(d)) return rc;
  const int group = qk_group(d->head_dim), rows = kBwdRows * (32 / group);
  const bool weights = d->norm_mode == DGXM_NORM_HEAD && (g_norm_q_w != nullptr || g_norm_k_w != nullptr);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  QkNormParams p;
  memset(&p, 0, sizeof(p));
  int blocks = 0;
  if (d->batch > 0 && d->seq > 0 && d->q_heads + d->k_heads > 0) {
    bool vec = false;
    if ((d->q_heads > 0 && dq == nullptr) || (d->k_heads > 0 && dk == nullptr))
      return fail(DGXM_ERR_INVALID, "NULL upstream gradient");
    if (int rc = qk_params(d, {q, k}, {dq, dk}, {gq, gk}, {norm_q_w, norm_k_w}, rope, rows, &p, &vec)) return rc;
    int64_t items = 0;
    blocks = qk_bwd_blocks(d, rows, 148, &items);
    if (weights) {
      if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 4 ||
          workspace_bytes < int64_t(blocks) * 2 * d->head_dim * 4)
        return fail(DGXM_ERR_INVALID, "workspace of %lld bytes (%lld needed)", (long long)workspace_bytes,
                    (long long)blocks * 2 * d->head_dim * 4);
      p.partial = static_cast<float*>(workspace);
    }
    qk_pick<true>(d->dtype, group, vec)<<<blocks, kQkThreads, 0, st>>>(p);
    DGXM_CUDA_TRY(cudaGetLastError());
  }
  if (!weights) return DGXM_OK;
  QkWeightGradParams wp;
  wp.partial = p.partial;
  wp.out[0] = g_norm_q_w;
  wp.out[1] = g_norm_k_w;
  wp.blocks = blocks;
  wp.dim = d->head_dim;
  wp.dtype = d->weight_dtype;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((2 * d->head_dim + 31) / 32);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DGXM_CUDA_TRY(cudaLaunchKernelEx(&cfg, qk_weight_grad_kernel, wp));
  return DGXM_OK;
}
