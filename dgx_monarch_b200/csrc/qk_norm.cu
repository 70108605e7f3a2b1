// RMSNorm of every query and key head with the rotary position embedding in
// the same pass, on local tensors of any stride, and its gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = R (n w)
//   with R the rotation by the token's angles, and for an upstream gradient dy
//   g = R^T dy,  dw = sum over rows of g n,
//   dx = r (g w - n mean(g w n)).
//
// Both directions move each value once and compute a handful of operations
// on it, so DRAM bounds them as long as the instructions stay few and enough
// loads are under way.  A head row is held by a group of 8, 16 or 32 lanes,
// eight values a lane (16 bytes of a 16-bit type), so a warp reads and writes
// whole 32-byte sectors whatever the strides, and the sums of a row are
// shuffles within the group.  One warp takes a chunk of the heads of one
// token and tensor.  It sends for all their rows at once, by cp.async into
// shared memory, where each lane finds its own values (and the halves order
// its partners) again: loads in flight cost no registers, and the token's
// cosines and sines and the head weight, which serve every row of the chunk,
// are fetched and multiplied with one another meanwhile.  The forward's
// arithmetic runs on pairs of fp32, two rows at a time (72 us against 78 with
// single values, 9450 x 80 heads of 128 in bf16, halves); the gradient's, on more
// registers, on single values (108 us against 115 adjacent).
//
// Everything between the load and the store is fp32 and is rounded once, to
// the tensors' type.  (The fused scatter of prologue.cu rounds after the
// norm and after the weight as well, as the separate modules it replaces do.)
#include "common.h"
#include "ptx.cuh"

namespace dgxm {

// The rotation's order; kQkHalvesOff: halves that are no whole number of a
// lane's eight values.
constexpr int kQkNoTurn = 0, kQkAdjacent = 1, kQkHalves = 2, kQkHalvesOff = 3;

constexpr int kQkThreads = 128;
constexpr int kQkWarps = kQkThreads / 32;
constexpr int kQkRing = 4096;     // bytes of rows a warp has under way, of each tensor it reads
constexpr int kQkFwdPerSm = 8;    // blocks of an SM: 64 registers a thread, 128 KB of rows under way
constexpr int kQkBwdPerSm = 6;    // 80 registers a thread, 192 KB (5 blocks of 96 registers: 113 us against 108 adjacent, 118 against 121 halves)
// Up to here a gradient with weights is one launch of a cluster, beyond a second launch adds the blocks (us at 8, 40, 80
// and 160 warps of 128 bf16: 4.3, 5.3, 6.4, 8.6 against 4.9, 4.7, 4.7, 4.9; a launch and a workspace are 4.5 of host time).
constexpr int kQkClusterWarps = 64;
constexpr int kQkBwdBlocks = 148 * kQkBwdPerSm;  // as many as run at one time, each with one partial sum of dw

// Rows a lane group has under way.
template <typename T>
constexpr int kQkRows = kQkRing / (32 * 8 * static_cast<int>(sizeof(T)));

static_assert(kQkRows<float> % 2 == 0 && kQkRows<__half> % 2 == 0, "rows go in twos");
static_assert(kQkWarps * 2 * kQkRing <= 48 * 1024, "dynamic shared memory without an opt-in");
static_assert(2 * kQkRing >= 1024, "the warps' sums fit");

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
  void* gw[2];        // backward on one cluster: the weights' gradients themselves
  int gw_dtype, cluster;  // cluster: its blocks (the whole grid), or 0
  int heads[2], chunks[2];  // chunks: warps for one token's heads of the tensor
  uint32_t seq, tokens;     // tokens: batch * seq
  int rows;                 // rows of a chunk for each lane group of its warp
  int dim, rot, halves, norm, w_f32, rope_vec, w_vec;
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

// Eight values as they lie in memory.
template <typename T>
struct __align__(16) Qk8 {
  T v[8];
};

// A warp's rows in shared memory: row u of every lane group, 16-byte pieces
// of 32 lanes side by side (one piece a lane for a 16-bit type, two for fp32).
template <typename T>
__device__ __forceinline__ uint8_t* qk_slot(uint8_t* ring, int u, int lane, int piece) {
  constexpr int kPieces = static_cast<int>(sizeof(T)) / 2;
  return ring + ((u * kPieces + piece) * 32 + lane) * 16;
}

// Send for a lane's values of row u.  VEC: 16-byte accesses (base and every
// stride a multiple of 16 bytes); otherwise one access a value.
template <typename T, bool VEC>
__device__ __forceinline__ void qk_fetch(uint8_t* ring, int u, int lane, const char* base, int64_t elem) {
  const T* p = reinterpret_cast<const T*>(base) + elem;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
    if constexpr (VEC) {
      cp_async16(smem_u32(qk_slot<T>(ring, u, lane, i)), reinterpret_cast<const uint4*>(p) + i);
    } else {
      constexpr int kEach = 16 / static_cast<int>(sizeof(T));
      T* dst = reinterpret_cast<T*>(qk_slot<T>(ring, u, lane, i));
#pragma unroll
      for (int k = 0; k < kEach; ++k) dst[k] = p[i * kEach + k];
    }
  }
}

// All the chunk's rows of a lane; lanes past head_dim hold zeros (qk_blank).
template <typename T, bool VEC>
__device__ __forceinline__ void qk_fetch_rows(uint8_t* ring, int lane, const char* base, int64_t at, int64_t step,
                                              int n) {
#pragma unroll 4
  for (int u = 0; u < n; ++u, at += step) qk_fetch<T, VEC>(ring, u, lane, base, at);
}

template <typename T>
__device__ __forceinline__ void qk_blank_row(uint8_t* ring, int u, int lane) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
    *reinterpret_cast<uint4*>(qk_slot<T>(ring, u, lane, i)) = make_uint4(0u, 0u, 0u, 0u);
}

template <typename T>
__device__ __forceinline__ void qk_blank(uint8_t* ring, int lane) {
  for (int u = 0; u < kQkRows<T>; ++u) qk_blank_row<T>(ring, u, lane);
}

template <typename T>
__device__ __forceinline__ Qk8<T> qk_take(uint8_t* ring, int u, int lane) {
  Qk8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
    reinterpret_cast<uint4*>(&r)[i] = *reinterpret_cast<const uint4*>(qk_slot<T>(ring, u, lane, i));
  return r;
}

template <typename T>
__device__ __forceinline__ T qk_take1(uint8_t* ring, int u, int lane, int i) {
  constexpr int kEach = 16 / static_cast<int>(sizeof(T));
  return reinterpret_cast<const T*>(qk_slot<T>(ring, u, lane, i / kEach))[i % kEach];
}

template <typename T, bool VEC>
__device__ __forceinline__ void qk_store(T* p, const float (&y)[8]) {
  Qk8<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = qk_narrow<T>(y[i]);
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

// A lane's eight values as four pairs: (0, 2), (1, 3), (4, 6), (5, 7).  The
// adjacent rotation's partners of pair j are then pair j ^ 1 as it stands.
__device__ __forceinline__ void qk_pair(const float (&x)[8], uint64_t (&v)[4]) {
  v[0] = pk2(x[0], x[2]);
  v[1] = pk2(x[1], x[3]);
  v[2] = pk2(x[4], x[6]);
  v[3] = pk2(x[5], x[7]);
}

__device__ __forceinline__ void qk_unpair(const uint64_t (&v)[4], float (&x)[8]) {
  upk2(v[0], x[0], x[2]);
  upk2(v[1], x[1], x[3]);
  upk2(v[2], x[4], x[6]);
  upk2(v[3], x[5], x[7]);
}

template <typename T>
__device__ __forceinline__ void qk_pairs_of(const Qk8<T>& r, uint64_t (&v)[4]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = qk_widen<T>(r.v[i]);
  qk_pair(x, v);
}

__device__ __forceinline__ float qk_total(uint64_t a) {
  float lo, hi;
  upk2(a, lo, hi);
  return lo + hi;
}

// The token that a warp works on, and which heads of tensor t.
struct QkItem {
  int first;
  uint32_t b, l;
};

__device__ __forceinline__ QkItem qk_item(const QkNormParams& p, uint32_t item, uint32_t chunks, int rows) {
  QkItem r;
  const uint32_t token = item / chunks;
  r.first = static_cast<int>(item - token * chunks) * rows;
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
template <int ROT, int SIGN>
__device__ __forceinline__ void qk_angles(const QkNormParams& p, const QkItem& it, int sub, float (&c)[8],
                                          float (&s)[8]) {
  const float* row = p.rope + it.b * p.rope_sb + static_cast<int64_t>(it.l) * p.rot;
  const int e0 = 8 * sub, half = p.rot / 2;
  if constexpr (ROT == kQkAdjacent) {
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
  } else if (ROT == kQkHalves && p.rope_vec && e0 + 8 <= p.rot) {
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

// The lane's partners in the halves order, from the rows in shared memory.
// A value that is not rotated gets itself.
template <typename T, int ROT>
__device__ __forceinline__ void qk_halves(const QkNormParams& p, int sub, int lane, uint8_t* ring, int u,
                                          float (&f)[8]) {
  const int e0 = 8 * sub, half = p.rot / 2;
  if constexpr (ROT == kQkHalves) {
    const int d = e0 < half ? half / 8 : e0 < p.rot ? -(half / 8) : 0;
    const Qk8<T> r = qk_take<T>(ring, u, lane + d);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = qk_widen<T>(r.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = e0 + i, to = e < half ? e + half : e < p.rot ? e - half : e;
      f[i] = qk_widen<T>(qk_take1<T>(ring, u, lane - sub + to / 8, to % 8));
    }
  }
}

// y = x a + x_partner b; values past `rot` take x a alone (a product with a
// zero sine would turn an infinite neighbour into NaN).
template <typename T, int ROT>
__device__ __forceinline__ void qk_rotate(const QkNormParams& p, int sub, int lane, const uint64_t (&a)[4],
                                          const uint64_t (&b)[4], uint8_t* ring, int u, const uint64_t (&x)[4],
                                          uint64_t (&y)[4]) {
  uint64_t q[4];
  if constexpr (ROT != kQkAdjacent) {
    float f[8];
    qk_halves<T, ROT>(p, sub, lane, ring, u, f);
    qk_pair(f, q);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = x[j ^ 1];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = fmul2(x[j], a[j]);
  if (p.rot == p.dim) {
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = ffma2(q[j], b[j], y[j]);
  } else {
    float yf[8], zf[8];
    uint64_t z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = ffma2(q[j], b[j], y[j]);
    qk_unpair(y, yf);
    qk_unpair(z, zf);
#pragma unroll
    for (int i = 0; i < 8; ++i) yf[i] = 8 * sub + i < p.rot ? zf[i] : yf[i];
    qk_pair(yf, y);
  }
}

// The same on single values.
template <typename T, int ROT>
__device__ __forceinline__ void qk_rotate(const QkNormParams& p, int sub, int lane, const float (&c)[8],
                                          const float (&s)[8], uint8_t* ring, int u, float (&x)[8]) {
  float q[8];
  if constexpr (ROT != kQkAdjacent) {
    qk_halves<T, ROT>(p, sub, lane, ring, u, q);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = x[i ^ 1];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = fmaf(q[i], s[i], x[i] * c[i]);
    x[i] = p.rot == p.dim || 8 * sub + i < p.rot ? y : x[i];
  }
}

// Values e of a head weight, 1 without one.
template <typename T>
__device__ __forceinline__ float qk_weight1(const QkNormParams& p, int t, int e) {
  return p.w_f32 ? __ldg(static_cast<const float*>(p.w[t]) + e) : qk_widen<T>(static_cast<const T*>(p.w[t])[e]);
}

template <typename T>
__device__ __forceinline__ void qk_weight(const QkNormParams& p, int t, int sub, bool in, float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (p.w[t] == nullptr || !in) return;
  if (!p.w_f32 && p.w_vec) {
    Qk8<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(&r)[i] =
          __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.w[t]) + 8 * sub) + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = qk_widen<T>(r.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = qk_weight1<T>(p, t, 8 * sub + i);
  }
}

// The weights of the partners of a lane's values.
template <typename T, int ROT>
__device__ __forceinline__ void qk_partner_weight(const QkNormParams& p, int t, int sub, bool in, const float (&w)[8],
                                                  float (&wp)[8]) {
  const int half = p.rot / 2, e0 = 8 * sub;
  if constexpr (ROT == kQkHalves) {
    qk_weight<T>(p, t, sub + (e0 < half ? half / 8 : e0 < p.rot ? -(half / 8) : 0), in, wp);
  } else if constexpr (ROT == kQkHalvesOff) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = e0 + i, to = e < half ? e + half : e < p.rot ? e - half : e;
      wp[i] = p.w[t] != nullptr && in ? qk_weight1<T>(p, t, to) : 1.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) wp[i] = w[i ^ 1];
  }
}

// One warp per (token, tensor, chunk of heads).
template <typename T, int G, int ROT, bool VEC>
__global__ void __launch_bounds__(kQkThreads, kQkFwdPerSm) qk_norm_rope_kernel(const __grid_constant__ QkNormParams p) {
  constexpr int kGroups = 32 / G;
  extern __shared__ __align__(16) uint8_t qk_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = qk_smem + warp * kQkRing;
  pdl_wait();
  uint32_t item = blockIdx.x * kQkWarps + warp;
  const uint32_t q_items = p.tokens * p.chunks[0];
  const int t = item >= q_items;
  if (t) item -= q_items;
  if (t && item >= p.tokens * p.chunks[1]) return;
  const QkItem it = qk_item(p, item, p.chunks[t], kGroups * p.rows);
  const int sub = lane % G, group = lane / G;
  const bool in = 8 * sub < p.dim;
  const int end = min(it.first + kGroups * p.rows, p.heads[t]);
  const int mine = (end - it.first - group + kGroups - 1) / kGroups;  // this lane group's rows
  {
    const int64_t at = it.b * p.xs[t][0] + it.l * p.xs[t][1] + (it.first + group) * p.xs[t][2] + 8 * sub;
    if (!in) qk_blank<T>(ring, lane);
    else qk_fetch_rows<T, VEC>(ring, lane, p.x[t], at, p.xs[t][2] * kGroups, mine);
  }
  // y = r (x a + x_partner b):  a = w c,  b = w_partner s
  uint64_t a[4], b[4];
  {
    float w[8];
    qk_weight<T>(p, t, sub, in, w);
    if constexpr (ROT != kQkNoTurn) {
      float c[8], s[8], wp[8];
      qk_angles<ROT, 1>(p, it, sub, c, s);
      qk_partner_weight<T, ROT>(p, t, sub, in, w, wp);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] *= c[i];
        s[i] *= wp[i];
      }
      qk_pair(s, b);
    }
    qk_pair(w, a);
  }
  cp_async_wait_all();
  __syncwarp();
  const int64_t step = p.os[t][2] * kGroups;
  T* out = reinterpret_cast<T*>(p.out[t]) + it.b * p.os[t][0] + it.l * p.os[t][1] + (it.first + group) * p.os[t][2] + 8 * sub;
  const int n = (end - it.first + kGroups - 1) / kGroups;
  for (int u0 = 0; u0 < n; u0 += 2, out += 2 * step) {
    uint64_t x[2][4];
    float r[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      qk_pairs_of<T>(qk_take<T>(ring, u0 + u, lane), x[u]);
      uint64_t ss = fmul2(x[u][0], x[u][0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) ss = ffma2(x[u][j], x[u][j], ss);
      r[u] = qk_total(ss);
    }
    if (p.norm) {
#pragma unroll
      for (int u = 0; u < 2; ++u) r[u] = rsqrtf(fmaf(qk_group_sum<G>(r[u]), p.inv_dim, p.eps));
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint64_t y[4];
      if constexpr (ROT != kQkNoTurn) {
        qk_rotate<T, ROT>(p, sub, lane, a, b, ring, u0 + u, x[u], y);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = fmul2(x[u][j], a[j]);
      }
      if (p.norm) {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = fmul2(y[j], pk2(r[u], r[u]));
      }
      float yf[8];
      qk_unpair(y, yf);
      if (in && u0 + u < mine) qk_store<T, VEC>(out + u * step, yf);
    }
  }
}

__device__ __forceinline__ void qk_store_weight_grad(void* out, int dtype, int e, float v) {
  if (out == nullptr) return;
  if (dtype == DGXM_DTYPE_F32) static_cast<float*>(out)[e] = v;
  else if (dtype == DGXM_DTYPE_F16) static_cast<__half*>(out)[e] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(v);
}

// Gradients.  The blocks stride over q's items, then over k's; each lane adds
// g n of its eight columns over all the rows it meets, the block sums its
// warps in a fixed order, and the blocks' sums are added in order by
// qk_weight_grad_kernel, or, in a call small enough for one cluster, by the
// cluster itself: no atomics, so the same call gives the same bits.
template <typename T, int G, int ROT, bool VEC>
__global__ void __launch_bounds__(kQkThreads, kQkBwdPerSm) qk_norm_rope_bwd_kernel(const __grid_constant__ QkNormParams p) {
  constexpr int kGroups = 32 / G;
  extern __shared__ __align__(16) uint8_t qk_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = qk_smem + warp * (2 * kQkRing);
  uint8_t* xring = ring + kQkRing;
  pdl_wait();
  const int sub = lane % G, group = lane / G;
  const bool in = 8 * sub < p.dim;
  const uint32_t warps = gridDim.x * kQkWarps;
  uint32_t skip = 0;  // q's items taken: k's go on with the next warp
  float total[2][256 / kQkThreads];  // this thread's columns of the block's sums
#pragma unroll
  for (int j = 0; j < 256 / kQkThreads; ++j) total[0][j] = total[1][j] = 0.f;
  for (int t = 0; t < 2; ++t) {
    if (!in) {
      qk_blank<T>(ring, lane);
      qk_blank<T>(xring, lane);
    }
    float dw[8], w[8];
    qk_weight<T>(p, t, sub, in, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[i] = 0.f;
    const uint32_t items = p.tokens * p.chunks[t];
    const int64_t step = p.os[t][2] * kGroups;
    for (uint32_t item = (blockIdx.x * kQkWarps + warp + warps - skip) % warps; item < items; item += warps) {
      const QkItem it = qk_item(p, item, p.chunks[t], kGroups * p.rows);
      const int end = min(it.first + kGroups * p.rows, p.heads[t]);
      const int mine = (end - it.first - group + kGroups - 1) / kGroups;
      if (in) {
        const int h = it.first + group;
        qk_fetch_rows<T, VEC>(ring, lane, p.dy[t], it.b * p.ds[t][0] + it.l * p.ds[t][1] + h * p.ds[t][2] + 8 * sub,
                              p.ds[t][2] * kGroups, mine);
        if (p.norm)
          qk_fetch_rows<T, VEC>(xring, lane, p.x[t], it.b * p.xs[t][0] + it.l * p.xs[t][1] + h * p.xs[t][2] + 8 * sub,
                                p.xs[t][2] * kGroups, mine);
        // rows that the other groups of the warp have and this one has not: nothing for dw
        for (int u = mine; u < p.rows; ++u) {
          qk_blank_row<T>(ring, u, lane);
          qk_blank_row<T>(xring, u, lane);
        }
      }
      float c[8], s[8];
      if constexpr (ROT != kQkNoTurn) qk_angles<ROT, -1>(p, it, sub, c, s);
      cp_async_wait_all();
      __syncwarp();
      T* out = reinterpret_cast<T*>(p.out[t]) + it.b * p.os[t][0] + it.l * p.os[t][1] + (it.first + group) * p.os[t][2] + 8 * sub;
      const int n = (end - it.first + kGroups - 1) / kGroups;
      for (int u = 0; u < n; ++u, out += step) {
        const Qk8<T> raw = qk_take<T>(ring, u, lane);
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = qk_widen<T>(raw.v[i]);
        if constexpr (ROT != kQkNoTurn) qk_rotate<T, ROT>(p, sub, lane, c, s, ring, u, g);
        if (p.norm) {
          const Qk8<T> xraw = qk_take<T>(xring, u, lane);
          float x[8], xx = 0.f, gx = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = qk_widen<T>(xraw.v[i]);
            xx = fmaf(x[i], x[i], xx);
            gx = fmaf(g[i] * w[i], x[i], gx);
          }
          xx = qk_group_sum<G>(xx);
          gx = qk_group_sum<G>(gx);
          // (a row that this group has not is blank: without an eps its r would be infinite, and dw NaN)
          const float r = u < mine ? rsqrtf(fmaf(xx, p.inv_dim, p.eps)) : 0.f;
          const float m = -gx * r * p.inv_dim;  // -mean(g w n); n and m stay in range however small x is
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float n1 = x[i] * r;
            dw[i] = fmaf(g[i], n1, dw[i]);
            g[i] = r * fmaf(n1, m, g[i] * w[i]);
          }
        }
        if (in && u < mine) qk_store<T, VEC>(out, g);
      }
      __syncwarp();  // every lane has read its values and partners: the next item's may come
    }
    skip = items % warps;
    if (p.partial == nullptr && p.cluster == 0) continue;  // uniform over the grid
    __syncthreads();
    float* sums = reinterpret_cast<float*>(qk_smem);  // (warps, 256)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = dw[i];
#pragma unroll
      for (int o = G; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (group == 0 && in) sums[warp * 256 + 8 * sub + i] = v;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 256 / kQkThreads; ++j) {
      const int e = threadIdx.x + j * kQkThreads;
      if (e >= p.dim) break;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kQkWarps; ++k) v += sums[k * 256 + e];
      if (t == 0) total[0][j] = v;
      else total[1][j] = v;
      if (p.cluster == 0) p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + t) * p.dim + e] = v;
    }
    __syncthreads();
  }
  if (p.cluster == 0) return;  // uniform over the grid
  // The blocks' sums in rank order, each block a share of the columns.
  float* mine = reinterpret_cast<float*>(qk_smem);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < 256 / kQkThreads; ++j)
      if (threadIdx.x + j * kQkThreads < p.dim) mine[t * 256 + threadIdx.x + j * kQkThreads] = total[t][j];
  cluster_sync();
  for (int i = blockIdx.x * kQkThreads + threadIdx.x; i < 2 * p.dim; i += p.cluster * kQkThreads) {
    const int t = i >= p.dim, e = i - t * p.dim;
    float v = 0.f;
    for (int r = 0; r < p.cluster; ++r) {
      float other;
      asm volatile("ld.shared::cluster.f32 %0, [%1];"
                   : "=f"(other)
                   : "r"(mapa_shared(smem_u32(mine + t * 256 + e), r))
                   : "memory");
      v += other;
    }
    qk_store_weight_grad(p.gw[t], p.gw_dtype, e, v);
  }
  cluster_sync();  // no block leaves while another reads its sums
}

struct QkWeightGradParams {
  const float* partial;
  void* out[2];
  int blocks, dim, dtype;
};

// Sum of the blocks' partial sums: 32 columns a block, 32 warps over the rows, then the warps in order.
__global__ void __launch_bounds__(1024) qk_weight_grad_kernel(const __grid_constant__ QkWeightGradParams p) {
  __shared__ float part[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * 32 + lane;  // over q | k
  float v = 0.f;
  pdl_wait();
  if (col < 2 * p.dim) {
#pragma unroll 8
    for (int b = warp; b < p.blocks; b += 32) v += p.partial[static_cast<int64_t>(b) * 2 * p.dim + col];
  }
  part[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || col >= 2 * p.dim) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < 32; ++k) v += part[k][lane];
  const int t = col >= p.dim, e = col - t * p.dim;
  qk_store_weight_grad(p.out[t], p.dtype, e, v);
}

// How a call is cut into warps: chunks of as many rows as a warp has under
// way, of equal length, unless that gives fewer than twelve warps for every
// SM partition; then shorter ones.
struct QkCut {
  int group, rows, chunks[2], blocks;
  int64_t warps;
};

// Lanes for one row.  Tensors off 16 bytes take 32 whatever their head_dim
// (one kernel for a rare case).
static int qk_group(int dim, bool vec) { return !vec || dim > 128 ? 32 : dim > 64 ? 16 : 8; }

static QkCut qk_cut(const dgxm_qk_norm_desc* d, bool back, bool vec) {
  QkCut c;
  c.group = qk_group(d->head_dim, vec);
  const int groups = 32 / c.group, most = d->dtype == DGXM_DTYPE_F32 ? kQkRows<float> : kQkRows<__half>;
  const int64_t tokens = static_cast<int64_t>(d->batch) * d->seq;
  const int longest = (std::max(d->q_heads, d->k_heads) + groups - 1) / groups;  // rows of the longer tensor
  c.rows = c.chunks[0] = c.chunks[1] = c.blocks = 0;
  c.warps = tokens;
  if (longest == 0 || tokens == 0 || tokens > (int64_t(1) << 31) - 1) return c;  // nothing to do, or too much
  for (int parts = (longest + most - 1) / most;; ++parts) {
    c.rows = (longest + parts - 1) / parts;
    c.chunks[0] = (d->q_heads + groups * c.rows - 1) / (groups * c.rows);
    c.chunks[1] = (d->k_heads + groups * c.rows - 1) / (groups * c.rows);
    c.warps = tokens * (c.chunks[0] + c.chunks[1]);
    if (c.rows <= 1 || c.warps >= 148 * 4 * 12) break;
  }
  const int64_t blocks = std::min<int64_t>((c.warps + kQkWarps - 1) / kQkWarps, int64_t(1) << 30);
  c.blocks = static_cast<int>(back ? std::min<int64_t>(blocks, kQkBwdBlocks) : blocks);
  return c;
}

static int qk_check(const dgxm_qk_norm_desc* d) {
  if (d == nullptr) return fail(DGXM_ERR_INVALID, "NULL Q/K norm descriptor");
  if (d->batch < 0 || d->seq < 0 || d->q_heads < 0 || d->k_heads < 0)
    return fail(DGXM_ERR_INVALID, "negative extents: batch %d, rows %d, heads %d / %d", d->batch, d->seq, d->q_heads,
                d->k_heads);
  if (d->q_heads > (1 << 20) || d->k_heads > (1 << 20))
    return fail(DGXM_ERR_UNSUPPORTED, "%d / %d heads (up to 2^20)", d->q_heads, d->k_heads);
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
                     void* const (&out)[2], const void* const (&w)[2], const float* rope, QkNormParams* p,
                     QkCut* cut, bool* vec) {
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
  *cut = qk_cut(d, back, *vec);
  if (cut->warps > (int64_t(1) << 31) - 1)
    return fail(DGXM_ERR_UNSUPPORTED, "%lld head groups in one call (up to 2^31 - 1)", (long long)cut->warps);
  p->rows = cut->rows;
  p->chunks[0] = cut->chunks[0];
  p->chunks[1] = cut->chunks[1];
  p->seq = static_cast<uint32_t>(d->seq);
  p->tokens = static_cast<uint32_t>(static_cast<int64_t>(d->batch) * d->seq);
  p->dim = d->head_dim;
  p->rot = p->rope != nullptr ? d->rot_dim : 0;
  p->halves = d->rope_halves != 0;
  p->norm = d->norm_mode == DGXM_NORM_HEAD;
  p->w_f32 = d->weight_dtype == DGXM_DTYPE_F32;
  p->w_vec = (reinterpret_cast<uintptr_t>(w[0]) | reinterpret_cast<uintptr_t>(w[1])) % 16 == 0;
  p->eps = d->eps;
  p->inv_dim = 1.f / d->head_dim;
  return DGXM_OK;
}

using QkKernel = void (*)(QkNormParams);

template <bool BACK, typename T, int G, bool VEC>
static QkKernel qk_pick_turn(int rot) {
  if constexpr (BACK)
    return rot == kQkNoTurn ? qk_norm_rope_bwd_kernel<T, G, kQkNoTurn, VEC>
           : rot == kQkAdjacent ? qk_norm_rope_bwd_kernel<T, G, kQkAdjacent, VEC>
           : rot == kQkHalves   ? qk_norm_rope_bwd_kernel<T, G, kQkHalves, VEC>
                                : qk_norm_rope_bwd_kernel<T, G, kQkHalvesOff, VEC>;
  else
    return rot == kQkNoTurn ? qk_norm_rope_kernel<T, G, kQkNoTurn, VEC>
           : rot == kQkAdjacent ? qk_norm_rope_kernel<T, G, kQkAdjacent, VEC>
           : rot == kQkHalves   ? qk_norm_rope_kernel<T, G, kQkHalves, VEC>
                                : qk_norm_rope_kernel<T, G, kQkHalvesOff, VEC>;
}

template <bool BACK, typename T>
static QkKernel qk_pick_group(int group, int rot, bool vec) {
  if (!vec) return qk_pick_turn<BACK, T, 32, false>(rot);
  return group == 8    ? qk_pick_turn<BACK, T, 8, true>(rot)
         : group == 16 ? qk_pick_turn<BACK, T, 16, true>(rot)
                       : qk_pick_turn<BACK, T, 32, true>(rot);
}

template <bool BACK>
static QkKernel qk_pick(int dtype, int group, const QkNormParams& p, bool vec) {
  const int rot = p.rope == nullptr ? kQkNoTurn : !p.halves ? kQkAdjacent : p.rot % 16 ? kQkHalvesOff : kQkHalves;
  if (dtype == DGXM_DTYPE_BF16) return qk_pick_group<BACK, __nv_bfloat16>(group, rot, vec);
  if (dtype == DGXM_DTYPE_F16) return qk_pick_group<BACK, __half>(group, rot, vec);
  return qk_pick_group<BACK, float>(group, rot, vec);
}

}  // namespace dgxm

extern "C" int dgxm_qk_norm_rope(const dgxm_qk_norm_desc* d, const void* q, const void* k, const void* norm_q_w,
                                 const void* norm_k_w, const float* rope, void* q_out, void* k_out, void* stream) {
  using namespace dgxm;
  if (int rc = qk_check(d)) return rc;
  if (d->batch == 0 || d->seq == 0 || d->q_heads + d->k_heads == 0) return DGXM_OK;
  QkNormParams p;
  QkCut cut;
  bool vec = false;
  if (int rc = qk_params(d, {q, k}, {nullptr, nullptr}, {q_out, k_out}, {norm_q_w, norm_k_w}, rope, &p, &cut, &vec))
    return rc;
  DGXM_CUDA_TRY(launch_overlapped(qk_pick<false>(d->dtype, cut.group, p, vec), cut.blocks, kQkThreads, kQkWarps * kQkRing,
                                  static_cast<cudaStream_t>(stream), p));
  return DGXM_OK;
}

extern "C" int64_t dgxm_qk_norm_rope_backward_workspace(const dgxm_qk_norm_desc* d) {
  using namespace dgxm;
  if (qk_check(d)) return -1;
  // Whether the call is small enough for a cluster depends on the tensors' alignment too: both ways.
  int64_t need = 0;
  for (bool vec : {false, true}) {
    const QkCut cut = qk_cut(d, true, vec);
    if (cut.warps > kQkClusterWarps) need = std::max<int64_t>(need, int64_t(cut.blocks) * 2 * d->head_dim * 4);
  }
  return need;
}

extern "C" int dgxm_qk_norm_rope_backward(const dgxm_qk_norm_desc* d, const void* dq, const void* dk, const void* q,
                                          const void* k, const void* norm_q_w, const void* norm_k_w,
                                          const float* rope, void* gq, void* gk, void* g_norm_q_w, void* g_norm_k_w,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dgxm;
  if (int rc = qk_check(d)) return rc;
  const bool weights = d->norm_mode == DGXM_NORM_HEAD && (g_norm_q_w != nullptr || g_norm_k_w != nullptr);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  QkNormParams p;
  memset(&p, 0, sizeof(p));
  int blocks = 0;
  if (d->batch > 0 && d->seq > 0 && d->q_heads + d->k_heads > 0) {
    bool vec = false;
    if ((d->q_heads > 0 && dq == nullptr) || (d->k_heads > 0 && dk == nullptr))
      return fail(DGXM_ERR_INVALID, "NULL upstream gradient");
    QkCut cut;
    if (int rc = qk_params(d, {q, k}, {dq, dk}, {gq, gk}, {norm_q_w, norm_k_w}, rope, &p, &cut, &vec)) return rc;
    blocks = cut.blocks;
    if (weights && cut.warps <= kQkClusterWarps) {
      p.cluster = blocks <= 1 ? 1 : blocks <= 2 ? 2 : blocks <= 4 ? 4 : 8;
      blocks = p.cluster;
      p.gw[0] = g_norm_q_w;
      p.gw[1] = g_norm_k_w;
      p.gw_dtype = d->weight_dtype;
    } else if (weights) {
      const int64_t need = int64_t(blocks) * 2 * d->head_dim * 4;
      if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 4 || workspace_bytes < need)
        return fail(DGXM_ERR_INVALID, "workspace of %lld bytes (%lld needed)", (long long)workspace_bytes, (long long)need);
      p.partial = static_cast<float*>(workspace);
    }
    DGXM_CUDA_TRY(launch_overlapped(qk_pick<true>(d->dtype, cut.group, p, vec), blocks, kQkThreads, kQkWarps * 2 * kQkRing,
                                    st, p, p.cluster > 0 ? p.cluster : 1));
  }
  if (p.cluster > 0) return DGXM_OK;
  if (!weights) return DGXM_OK;
  QkWeightGradParams wp;
  wp.partial = p.partial;
  wp.out[0] = g_norm_q_w;
  wp.out[1] = g_norm_k_w;
  wp.blocks = blocks;
  wp.dim = d->head_dim;
  wp.dtype = d->weight_dtype;
  DGXM_CUDA_TRY(launch_overlapped(qk_weight_grad_kernel, (2 * d->head_dim + 31) / 32, 1024, 0, st, wp));
  return DGXM_OK;
}
