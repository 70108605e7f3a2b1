// Microscaled 4-bit floating point: a matrix to e2m1 codes with block scales
// (nvfp4, mxfp4) and back.
//
//   nvfp4  g = the tensor's scale (given, or amax / 2688), per block of 16
//          s = e4m3(amax / (6 g)),  code = e2m1(x / (s g))
//   mxfp4  per block of 32  s = 2^(floor(log2 amax) - 2),  code = e2m1(x / s)
// each to the nearest value, ties to the even code, saturating.  A block with
// a NaN or an infinity gets a NaN scale; an empty scale gives zero codes.
//
// The roundings are those of the real quotients x / (s g), not of a rounded
// division, and a kernel that DRAM is to bound has few instructions for it
// (2 bytes in and 0.56 out for a bf16 value):
//
// - Away from the borders between codes a product with an fp32 reciprocal,
//   good to 2^-21, rounds like the quotient.
// - A 16-bit x comes near a border b s g only if b s g itself lies near a
//   value of x's type.  The seven borders have four significands and s has
//   eight, so 32 products a warp show for which they do, within 2^-16.  Each such border
//   has one value X beside it, and the sign of fma(b s, g, -X) says on which
//   side (b s has 7 bits: the one rounding of the fma cannot change the sign).
//   If all agree, a reciprocal moved by 2^-18 to that side decides them right,
//   and no value near no border can notice.  With g = amax / 2688 a quarter
//   of all blocks are of this kind: s = 1.75 meets the border 0.75 where
//   21 divides out, and misses it by the rounding of g alone.
// - Where they disagree or X lies on the border, or x is fp32, two products
//   bound the quotient from below and above.  Where they round alike that
//   code is right; where not, one border lies between, and the sign of
//   fma(b s, g, -|x|) decides.
// - A g of at most 16 significant bits (a power of two, a scale that came as
//   bf16 or fp16) makes b s g and ties with it exact numbers, so that many
//   blocks would take that way.  There the residual x - q s g, exact in an
//   fma, corrects the product q: a tie becomes its border exactly, and nothing
//   else can reach one, since b s g and x are at least 2^-23 apart.
//
// g is brought near 1 by a power of two first (with x, exactly), so that no
// product leaves fp32's range.
#include <type_traits>

#include "common.h"
#include "fp4.cuh"

namespace dgxm {

constexpr int kFp4Threads = 256;
constexpr int kFp4Cols = 32;  // columns of an item: a block of mxfp4, two of nvfp4
// Up to here one launch of a cluster finds the amax and quantises; beyond, a
// pass of its own does (us at 160, 1280 and 2560 items: 3.5, 4.5, 5.6 against
// 4.4, 4.7, 4.7, and one launch less of host time).
constexpr uint32_t kFp4ClusterItems = 8 * 256;
constexpr int kFp4Partials = 148 * 4;  // blocks of the amax pass, one partial maximum each

struct Fp4Params {
  const char* x;       // (rows, cols), row stride in elements; dequantise: the output
  int64_t row_stride;
  uint8_t* values;
  uint8_t* scales;
  const void* scale;   // the given scale, or NULL
  float* scale_out;    // the fp32 scale of the tensor
  uint32_t* partials;  // bit patterns of the blocks' amax
  int64_t pitch, groups;
  uint32_t items, per_row;  // an item is 32 columns of one row (16 where values are read back), padded to whole scale words
  int cols, n_partials, scale_dtype, wide;
  int cluster;         // blocks that find the amax by themselves (the whole grid, a cluster), or 0
  float scale_value;   // the given scale where `scale` is NULL
};

// One block's values as they lie in memory.
template <typename T, int N>
struct __align__(32) Fp4Raw {
  T v[N];
};

// 32 bytes at once (32-byte aligned): a whole sector a thread.
__device__ __forceinline__ void ld_global_32(const void* p, uint32_t* r) {
  asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}

__device__ __forceinline__ void st_global_32(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// The n <= N values at p (the rest zero).  VEC: p is 16-byte aligned, wide:
// 32-byte.  Otherwise, and for a row's last values, p's 16-byte words are
// loaded -- those that hold one of the values, none else -- and shifted.
template <typename T, int N, bool VEC>
__device__ __forceinline__ Fp4Raw<T, N> fp4_load(const T* p, int n, bool wide) {
  Fp4Raw<T, N> r;
  uint32_t* out = reinterpret_cast<uint32_t*>(&r);
  constexpr int kWords = static_cast<int>(sizeof(r)) / 4;
  if (VEC && n >= N && wide) {
#pragma unroll
    for (int i = 0; i < kWords / 8; ++i) ld_global_32(p + i * (32 / sizeof(T)), out + 8 * i);
    return r;
  }
  if (VEC && n >= N) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4*>(out)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    return r;
  }
  const uint32_t off = reinterpret_cast<uintptr_t>(p) & 15u;  // bytes of the first word before p
  const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - off);
  const int bytes = n > 0 ? min(n, N) * static_cast<int>(sizeof(T)) : 0;
  uint32_t w[kWords + 4];
#pragma unroll
  for (int i = 0; i < kWords / 4 + 1; ++i) {
    const bool in = bytes > 0 && 16 * i < static_cast<int>(off) + bytes;
    const uint4 v = in ? __ldg(from + i) : make_uint4(0u, 0u, 0u, 0u);
    w[4 * i] = v.x;
    w[4 * i + 1] = v.y;
    w[4 * i + 2] = v.z;
    w[4 * i + 3] = v.w;
  }
#pragma unroll
  for (int i = 0; i < kWords + 2; ++i) w[i] = (off & 8u) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < kWords + 1; ++i) w[i] = (off & 4u) ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const uint32_t v = __funnelshift_r(w[i], w[i + 1], 8 * (off & 3u));
    const int left = bytes - 4 * i;  // bytes of this word that are values
    out[i] = left >= 4 ? v : left == 2 ? v & 0xFFFFu : 0u;
  }
  return r;
}

// Bits of the largest magnitude.  As integers magnitudes order like their
// values, infinity above all numbers and NaN above infinity.
template <typename T, int N>
__device__ __forceinline__ uint32_t fp4_amax_bits(const T* v) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
  uint32_t m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
    return m;
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    return max(m & 0xFFFFu, m >> 16);
  }
}

template <typename T>
__device__ __forceinline__ float fp4_widen_bits(uint32_t bits);
template <>
__device__ __forceinline__ float fp4_widen_bits<float>(uint32_t bits) { return __uint_as_float(bits); }
template <>
__device__ __forceinline__ float fp4_widen_bits<__nv_bfloat16>(uint32_t bits) { return __uint_as_float(bits << 16); }
template <>
__device__ __forceinline__ float fp4_widen_bits<__half>(uint32_t bits) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

template <typename T>
__device__ __forceinline__ float fp4_widen(T v);
template <>
__device__ __forceinline__ float fp4_widen(float v) { return v; }
template <>
__device__ __forceinline__ float fp4_widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float fp4_widen(__half v) { return __half2float(v); }

// Largest magnitude of what this block sees of the matrix, as float bits, in every thread.
template <typename T, bool VEC>
__device__ __forceinline__ uint32_t fp4_block_amax(const Fp4Params& p) {
  constexpr int kUnroll = 2;
  __shared__ uint32_t red[kFp4Threads / 32];
  uint32_t m = 0;
  const uint32_t step = gridDim.x * kFp4Threads;
  for (uint64_t i0 = blockIdx.x * kFp4Threads + threadIdx.x; i0 < p.items; i0 += uint64_t(step) * kUnroll) {
    Fp4Raw<T, kFp4Cols> raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t item = i0 + uint64_t(u) * step;
      const uint32_t row = static_cast<uint32_t>(item) / p.per_row, b = static_cast<uint32_t>(item) - row * p.per_row;
      const int n = item < p.items ? p.cols - static_cast<int>(b) * kFp4Cols : 0;
      raw[u] = fp4_load<T, kFp4Cols, VEC>(
          reinterpret_cast<const T*>(p.x) + (n > 0 ? row * p.row_stride + int64_t(b) * kFp4Cols : 0), n, p.wide);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) m = max(m, fp4_amax_bits<T, kFp4Cols>(raw[u].v));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kFp4Threads / 32; ++i) m = max(m, red[i]);
  return __float_as_uint(fp4_widen_bits<T>(m));
}

// One partial a block.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kFp4Threads) fp4_amax_kernel(const __grid_constant__ Fp4Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t m = fp4_block_amax<T, VEC>(p);
  if (threadIdx.x == 0) p.partials[blockIdx.x] = m;
}

// The nearest e4m3 code of amax / (6 g), and the decision at a border.
__device__ __forceinline__ uint32_t fp4_e4m3_scale(float amax, float g, float inv6g) {
  constexpr float kBelow = 1.f - 0x1p-21f, kAbove = 1.f + 0x1p-21f;
  const float t = amax * inv6g;
  const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(t * kBelow, t * kAbove), __NV_SATFINITE, __NV_E4M3);
  const uint32_t lo = two & 0xFFu, hi = (two >> 8) & 0xFFu;
  if (lo == hi) return lo;
  const float mid = 0.5f * (fp4_scale_value<DGXM_FP4_NVFP4>(lo) + fp4_scale_value<DGXM_FP4_NVFP4>(hi));
  const float d = fmaf(6.f * mid, g, -amax);
  return d > 0.f ? lo : d < 0.f ? hi : (lo & 1u) ? hi : lo;
}

// What the borders' four significands times s g, u when rounded, have beside them: 0 no value
// of T within 2^-16, 1 or -1 one or more, all above or all below their
// borders, 2 both kinds, or one on its border.
template <typename T>
__device__ __forceinline__ int fp4_beside(float s, float g, float u) {
  // The bits of u past T's significand are all zeros or ones but for the last seven.
  constexpr uint32_t kPast = std::is_same<T, __nv_bfloat16>::value ? 0xFFFFu : 0x1FFFu;
  const float w[4] = {u, 1.25f * u, 1.5f * u, 1.75f * u};
  uint32_t past[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) past[i] = (__float_as_uint(w[i]) + 128u) & kPast;
  if (min(min(past[0], past[1]), min(past[2], past[3])) > 256u) return 0;
  bool above = false, below = false, on = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (past[i] > 256u) continue;
    const float x = __uint_as_float((__float_as_uint(w[i]) + 128u) & ~kPast);  // the value of T
    const float d = fmaf((1.f + 0.25f * i) * s, g, -x);
    above |= d < 0.f;
    below |= d > 0.f;
    on |= d == 0.f;
  }
  return on || (above && below) ? 2 : above ? 1 : -1;
}

// 1 / v to 2^-23.
__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Eight codes of nvfp4 values under s g (g > 0 and near 1 after `up`), by the
// ways that the head of this file gives.
template <typename T>
__device__ __forceinline__ uint32_t fp4_codes_quick(const T* x, float r) {
  const uint64_t rr = pk2(r, r);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) upk2(fmul2(pk2(fp4_widen<T>(x[i]), fp4_widen<T>(x[i + 1])), rr), q[i], q[i + 1]);
  return fp4_encode8(q);
}

template <typename T>
__device__ __forceinline__ uint32_t fp4_codes_residual(const T* x, float up, float u, float r) {
  const uint64_t nr = pk2(-r, -r), uu = pk2(u, u), nup = pk2(-up, -up);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t nv = fmul2(pk2(fp4_widen<T>(x[i]), fp4_widen<T>(x[i + 1])), nup);  // -x
    const uint64_t a = fmul2(nv, nr);
    upk2(ffma2(ffma2(a, uu, nv), nr, a), q[i], q[i + 1]);  // a - (a u - x) r; in these signs -0 stays -0
  }
  return fp4_encode8(q);
}

template <typename T>
__device__ __forceinline__ uint32_t fp4_codes_decided(const T* x, float up, float s, float g, float r) {
  constexpr float kBelow = 1.f - 0x1p-21f, kAbove = 1.f + 0x1p-21f;
  const float r0 = r * kBelow, r1 = r * kAbove;
  float v[8], lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = fp4_widen<T>(x[i]) * up;
    lo[i] = v[i] * r0;
    hi[i] = v[i] * r1;
  }
  uint32_t c = fp4_encode8(lo);
  const uint32_t d = c ^ fp4_encode8(hi);
  if (d != 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (((d >> (4 * i)) & 15u) == 0) continue;
      const int k = (c >> (4 * i)) & 7;  // the border lies between codes k and k + 1
      const float border = k < 4 ? 0.5f * k + 0.25f : k == 6 ? 5.f : k - 1.5f;
      const float e = fmaf(border * s, g, -fabsf(v[i]));
      if (e < 0.f || (e == 0.f && (k & 1))) c += 1u << (4 * i);
    }
  }
  return c;
}

template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(kFp4Threads) fp4_quantize_kernel(const __grid_constant__ Fp4Params p) {
  constexpr int B = fp4_block(FORMAT);
  pdl_launch_dependents();
  pdl_wait();
  float g = 1.f, up = 1.f, inv6g = 1.f;
  bool bad = false, few_bits = false;
  uint32_t side_up = 0, side_down = 0, undecided = 0xFFu;  // fp4_beside by the significand of s
  if constexpr (FORMAT == DGXM_FP4_NVFP4) {
    if (p.cluster > 0) {
      __shared__ uint32_t mine;
      uint32_t m = fp4_block_amax<T, VEC>(p);
      if (threadIdx.x == 0) mine = m;
      cluster_sync();
      for (int r = 0; r < p.cluster; ++r) {
        uint32_t other;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(other) : "r"(mapa_shared(smem_u32(&mine), r)) : "memory");
        m = max(m, other);
      }
      g = __fdiv_rn(__uint_as_float(m), 2688.f);
    } else if (p.partials != nullptr) {
      __shared__ uint32_t red[kFp4Threads / 32];
      uint32_t m = 0;
      for (int i = threadIdx.x; i < p.n_partials; i += kFp4Threads) m = max(m, p.partials[i]);
      m = __reduce_max_sync(0xffffffffu, m);
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kFp4Threads / 32; ++i) m = max(m, red[i]);
      g = __fdiv_rn(__uint_as_float(m), 2688.f);
    } else {
      g = p.scale != nullptr ? fp4_read_scale(p.scale, p.scale_dtype) : p.scale_value;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.scale_out = g;
    bad = !(g >= 0.f && g < INFINITY);  // NaN, negative or infinite; -0 is a zero
    up = g < 0x1p-64f ? 0x1p64f : g > 0x1p64f ? 0x1p-64f : 1.f;
    g *= up;
    inv6g = g > 0.f ? __frcp_rn(6.f * g) : 0.f;
    few_bits = (__float_as_uint(g) & 0xFFu) == 0;  // at most 16 significant bits
    if constexpr (sizeof(T) == 2) {  // lane i: the block scales of significand 1 + i / 8
      const float s = 1.f + 0.125f * (threadIdx.x & 7u);
      const int side = up != 1.f ? 2 : fp4_beside<T>(s, g, s * g);
      side_up = __ballot_sync(0xffffffffu, side == 1);
      side_down = __ballot_sync(0xffffffffu, side == -1);
      undecided = __ballot_sync(0xffffffffu, side == 2);
    }
  }
  // From the last item to the first: behind an amax pass the end of the
  // matrix is what L2 still holds.
  const int64_t items = p.items, step = int64_t(gridDim.x) * kFp4Threads;
  for (int64_t i0 = (items + step - 1) / step * step - step + blockIdx.x * kFp4Threads + (threadIdx.x & ~31u); i0 >= 0;
       i0 -= step) {
    if (i0 >= items) continue;  // only the first round is not full
    const uint32_t item = static_cast<uint32_t>(i0) + (threadIdx.x & 31u);
    const bool live = item < p.items;  // a scale word's items are live together
    const uint32_t row = item / p.per_row, c32 = item - row * p.per_row;
    const int n = live ? p.cols - static_cast<int>(c32) * kFp4Cols : 0;  // <= 0: padding
    const Fp4Raw<T, kFp4Cols> raw = fp4_load<T, kFp4Cols, VEC>(
        reinterpret_cast<const T*>(p.x) + (n > 0 ? row * p.row_stride + int64_t(c32) * kFp4Cols : 0), n, p.wide);
    uint32_t codes[kFp4Cols / 8];
    uint32_t word = 0;  // this item's scale bytes
#pragma unroll
    for (int k = 0; k < kFp4Cols / B; ++k) {
      const T* x = raw.v + k * B;
      uint32_t* c = codes + k * (B / 8);
      const float amax = fp4_widen_bits<T>(fp4_amax_bits<T, B>(x));
      uint32_t byte;
      if constexpr (FORMAT == DGXM_FP4_NVFP4) {
        byte = bad || __float_as_uint(amax) >= 0x7F800000u ? 0x7Fu : inv6g == 0.f ? 0u : fp4_e4m3_scale(amax * up, g, inv6g);
        const float s = fp4_scale_value<FORMAT>(byte);
        const bool on = s > 0.f;  // false for zero and NaN
        const float u = s * g, r = on ? rcp_approx(u) : 0.f;
        if (few_bits && amax * up * r < 0x1p100f) {  // (a residual of quotients beyond fp32's range is none)
#pragma unroll
          for (int j = 0; j < B / 8; ++j) c[j] = fp4_codes_residual<T>(x + 8 * j, up, u, r);
        } else {
          const uint32_t bit = 1u << ((__float_as_uint(s) >> 20) & 7u);
          if (undecided & bit) {
#pragma unroll
            for (int j = 0; j < B / 8; ++j) c[j] = fp4_codes_decided<T>(x + 8 * j, up, s, g, r);
          } else {
            const float moved = fmaf(r, (side_up & bit) ? 0x1p-18f : (side_down & bit) ? -0x1p-18f : 0.f, r);
#pragma unroll
            for (int j = 0; j < B / 8; ++j) c[j] = fp4_codes_quick<T>(x + 8 * j, moved);
          }
        }
#pragma unroll
        for (int j = 0; j < B / 8; ++j) c[j] = on ? c[j] : 0u;
      } else {
        const uint32_t ab = __float_as_uint(amax);
        const int e = static_cast<int>(ab >> 23) - 2;  // floor(log2 amax) - 2 + 127; the scale is exact, and so is x / s
        byte = ab >= 0x7F800000u ? 0xFFu : static_cast<uint32_t>(e < 0 ? 0 : e);
        const bool on = byte != 0xFFu;
        const float r = on ? __uint_as_float((254u - byte) << 23) : 0.f;
#pragma unroll
        for (int j = 0; j < B / 8; ++j) {
          c[j] = fp4_codes_quick<T>(x + 8 * j, r);
          c[j] = on ? c[j] : 0u;
        }
      }
      if (n > k * B) word |= byte << (8 * k);  // zero past the last column
    }
    // The neighbouring items' bytes complete the word of the tile.
    constexpr int kBytes = kFp4Cols / B, kItems = 4 / kBytes;
    const uint32_t at = threadIdx.x % kItems;
    word <<= 8 * kBytes * at;
#pragma unroll
    for (int o = 1; o < kItems; o *= 2) word |= __shfl_xor_sync(0xffffffffu, word, o);
    if (live && at == 0) *reinterpret_cast<uint32_t*>(p.scales + fp4_scale_at(row, c32 * kBytes, p.groups)) = word;
    if (live && int64_t(c32) * 16 < p.pitch)
      *reinterpret_cast<uint4*>(p.values + row * p.pitch + int64_t(c32) * 16) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
  }
  if (FORMAT == DGXM_FP4_NVFP4 && p.cluster > 0) cluster_sync();  // no block leaves while another reads its amax
}

// The values that a packed tensor stands for: (code s) is exact in fp32, the
// product with the tensor's scale is rounded once, and once more to a 16-bit
// type.  One thread a run of 16 values.
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(kFp4Threads) fp4_dequantize_kernel(const __grid_constant__ Fp4Params p) {
  constexpr int B = fp4_block(FORMAT);
  pdl_launch_dependents();
  pdl_wait();
  const float g = FORMAT == DGXM_FP4_NVFP4 ? *static_cast<const float*>(p.scale) : 1.f;
  const uint64_t gg = pk2(g, g);
  const int lane = threadIdx.x & 31;
  const uint32_t step = gridDim.x * kFp4Threads;
  for (uint64_t i0 = blockIdx.x * kFp4Threads + threadIdx.x - lane; i0 < p.items; i0 += step) {
    const uint32_t item = static_cast<uint32_t>(i0) + lane;
    const bool live = item < p.items;
    const uint32_t row = item / p.per_row, c16 = item - row * p.per_row;
    uint2 code = make_uint2(0u, 0u);
    uint32_t byte = 0;
    if (live) {
      code = __ldg(reinterpret_cast<const uint2*>(p.values + row * p.pitch) + c16);
      byte = __ldg(p.scales + fp4_scale_at(row, c16 * 16 / B, p.groups));
    }
    __half2 h[2][4];
    fp4_decode8(code.x, h[0]);
    fp4_decode8(code.y, h[1]);
    Fp4Raw<T, 16> out;
    if constexpr (FORMAT == DGXM_FP4_NVFP4) {
      // 6 significant bits between 2^-10 and 2688: exact in fp16 already.
      const __half2 s = __half2half2(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i / 4][i % 4] = __hmul2(h[i / 4][i % 4], s);
    }
    const uint64_t ss = FORMAT == DGXM_FP4_NVFP4 ? gg : pk2(fp4_scale_value<FORMAT>(byte), fp4_scale_value<FORMAT>(byte));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __half22float2(h[i / 4][i % 4]);
      float a, b;
      upk2(fmul2(pk2(f.x, f.y), ss), a, b);
      out.v[2 * i] = static_cast<T>(a);
      out.v[2 * i + 1] = static_cast<T>(b);
    }
    const int n = live ? p.cols - static_cast<int>(c16) * 16 : 0;
    T* dst = reinterpret_cast<T*>(const_cast<char*>(p.x)) + row * p.row_stride + int64_t(c16) * 16;
    if (VEC && n >= 16 && p.wide) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(out) / 32); ++i)
        st_global_32(dst + i * (32 / sizeof(T)), reinterpret_cast<const uint32_t*>(&out) + 8 * i);
    } else if (VEC && n >= 16) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(out) / 16); ++i)
        reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(&out)[i];
    } else if (VEC) {  // a row's last values
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < n) dst[i] = out.v[i];
    } else {
      // Rows off 16 bytes: the warp's runs pass through shared memory, and
      // neighbouring lanes store neighbouring values.
      constexpr int kPitch = 16 * sizeof(T) + 16;  // 16 bytes on: neighbouring runs lie in other banks
      __shared__ __align__(16) uint8_t runs[kFp4Threads * kPitch];
      uint8_t* warp_runs = runs + (threadIdx.x - lane) * kPitch;
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(out) / 16); ++i)
        reinterpret_cast<uint4*>(warp_runs + lane * kPitch)[i] = reinterpret_cast<const uint4*>(&out)[i];
      __syncwarp();
#pragma unroll 4
      for (int k = 0; k < 16; ++k) {
        const int run = 2 * k + lane / 16, e = lane % 16;
        T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), run));
        const int many = __shfl_sync(0xffffffffu, n, run);
        if (e < many) to[e] = reinterpret_cast<const T*>(warp_runs + run * kPitch)[e];
      }
      __syncwarp();
    }
  }
}

static int fp4_check(const dgxm_fp4_desc* d) {
  if (d == nullptr) return fail(DGXM_ERR_INVALID, "NULL 4-bit descriptor");
  if (d->format != DGXM_FP4_NVFP4 && d->format != DGXM_FP4_MXFP4)
    return fail(DGXM_ERR_UNSUPPORTED, "4-bit format %d (nvfp4 or mxfp4)", d->format);
  if (d->rows < 0 || d->cols <= 0 || d->cols > (1 << 30))
    return fail(DGXM_ERR_INVALID, "%lld x %lld matrix", (long long)d->rows, (long long)d->cols);
  if (d->dtype != DGXM_DTYPE_BF16 && d->dtype != DGXM_DTYPE_F16 && d->dtype != DGXM_DTYPE_F32)
    return fail(DGXM_ERR_UNSUPPORTED, "dtype %d (bf16, f16 or f32)", d->dtype);
  if (d->rows > 1 && d->row_stride < d->cols)
    return fail(DGXM_ERR_INVALID, "row stride %lld below %lld columns", (long long)d->row_stride, (long long)d->cols);
  if (d->scale_dtype != DGXM_DTYPE_BF16 && d->scale_dtype != DGXM_DTYPE_F16 && d->scale_dtype != DGXM_DTYPE_F32)
    return fail(DGXM_ERR_UNSUPPORTED, "scale dtype %d (bf16, f16 or f32)", d->scale_dtype);
  return DGXM_OK;
}

static int fp4_params(const dgxm_fp4_desc* d, const void* x, const void* values, const void* scales, int64_t per_row,
                      Fp4Params* p, bool* vec) {
  memset(p, 0, sizeof(*p));
  const int elt = d->dtype == DGXM_DTYPE_F32 ? 4 : 2;
  if (d->rows > 0 && (x == nullptr || values == nullptr || scales == nullptr))
    return fail(DGXM_ERR_INVALID, "NULL matrix, values or scales");
  if ((reinterpret_cast<uintptr_t>(values) | reinterpret_cast<uintptr_t>(scales)) % 16)
    return fail(DGXM_ERR_INVALID, "values and scales must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(x) % elt) return fail(DGXM_ERR_INVALID, "the matrix is not aligned to its elements");
  if (d->rows > (int64_t(1) << 31) || d->rows * per_row > (int64_t(1) << 31) - 1)
    return fail(DGXM_ERR_UNSUPPORTED, "%lld x %lld is more than 2^31 - 1 blocks", (long long)d->rows, (long long)d->cols);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(d->rows == 1 ? 0 : d->row_stride * elt);
  *vec = bits % 16 == 0;
  p->wide = bits % 32 == 0;
  p->x = static_cast<const char*>(x);
  p->row_stride = d->row_stride;
  p->values = static_cast<uint8_t*>(const_cast<void*>(values));
  p->scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  p->pitch = fp4_pitch(d->cols);
  p->groups = fp4_groups(d->cols, d->format);
  p->items = static_cast<uint32_t>(d->rows * per_row);
  p->per_row = static_cast<uint32_t>(per_row);
  p->cols = static_cast<int>(d->cols);
  p->scale_dtype = d->scale_dtype;
  p->scale_value = d->scale_value;
  return DGXM_OK;
}

static unsigned fp4_grid(uint32_t items, int per_sm) {
  const unsigned want = (items + kFp4Threads - 1) / kFp4Threads, most = 148u * per_sm;
  return want < 1 ? 1u : want < most ? want : most;
}

template <typename T, int FORMAT, bool VEC>
static cudaError_t fp4_launch_quantize(Fp4Params& p, bool amax, cudaStream_t st) {
  if (amax && p.items <= kFp4ClusterItems) {  // a small matrix: one launch, its blocks a cluster
    p.cluster = p.items <= kFp4Threads ? 1 : p.items <= 2 * kFp4Threads ? 2 : p.items <= 4 * kFp4Threads ? 4 : 8;
    return launch_overlapped(fp4_quantize_kernel<T, FORMAT, VEC>, p.cluster, kFp4Threads, 0, st, p, p.cluster);
  }
  if (amax) {
    const unsigned grid = std::min<unsigned>(fp4_grid(p.items, 8), kFp4Partials);
    p.n_partials = static_cast<int>(grid);
    const cudaError_t e = launch_overlapped(fp4_amax_kernel<T, VEC>, grid, kFp4Threads, 0, st, p);
    if (e != cudaSuccess) return e;
  }
  return launch_overlapped(fp4_quantize_kernel<T, FORMAT, VEC>, fp4_grid(p.items, 8), kFp4Threads, 0, st, p);
}

template <typename T>
static cudaError_t fp4_quantize_typed(Fp4Params& p, int format, bool vec, bool amax, cudaStream_t st) {
  if (format == DGXM_FP4_NVFP4)
    return vec ? fp4_launch_quantize<T, DGXM_FP4_NVFP4, true>(p, amax, st)
               : fp4_launch_quantize<T, DGXM_FP4_NVFP4, false>(p, amax, st);
  return vec ? fp4_launch_quantize<T, DGXM_FP4_MXFP4, true>(p, false, st)
             : fp4_launch_quantize<T, DGXM_FP4_MXFP4, false>(p, false, st);
}

template <typename T>
static cudaError_t fp4_dequantize_typed(const Fp4Params& p, int format, bool vec, cudaStream_t st) {
  const auto kernel = format == DGXM_FP4_NVFP4
                          ? (vec ? fp4_dequantize_kernel<T, DGXM_FP4_NVFP4, true> : fp4_dequantize_kernel<T, DGXM_FP4_NVFP4, false>)
                          : (vec ? fp4_dequantize_kernel<T, DGXM_FP4_MXFP4, true> : fp4_dequantize_kernel<T, DGXM_FP4_MXFP4, false>);
  return launch_overlapped(kernel, fp4_grid(p.items, 8), kFp4Threads, 0, st, p);
}

}  // namespace dgxm

extern "C" int64_t dgxm_fp4_values_bytes(int64_t rows, int64_t cols) {
  return rows < 0 || cols <= 0 || rows > (int64_t(1) << 31) || cols > (1 << 30) ? -1 : rows * dgxm::fp4_pitch(cols);
}

extern "C" int64_t dgxm_fp4_scales_bytes(int64_t rows, int64_t cols, int32_t format) {
  if (rows < 0 || cols <= 0 || rows > (int64_t(1) << 31) || cols > (1 << 30) || (format != DGXM_FP4_NVFP4 && format != DGXM_FP4_MXFP4)) return -1;
  return (rows + 127) / 128 * dgxm::fp4_groups(cols, format) * 512;
}

extern "C" int64_t dgxm_quantize_fp4_workspace(void) { return dgxm::kFp4Partials * 4; }

extern "C" int dgxm_quantize_fp4(const dgxm_fp4_desc* d, const void* x, const void* scale, void* values, void* scales,
                                 float* scale_out, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dgxm;
  if (int rc = fp4_check(d)) return rc;
  const bool nv = d->format == DGXM_FP4_NVFP4;
  const bool amax = nv && scale == nullptr && d->scale_value == 0.f;
  if (nv && (scale_out == nullptr || reinterpret_cast<uintptr_t>(scale_out) % 4))
    return fail(DGXM_ERR_INVALID, "nvfp4 needs scale_out for the tensor's fp32 scale");
  if (!nv && (scale != nullptr || d->scale_value != 0.f))
    return fail(DGXM_ERR_INVALID, "mxfp4 has no scale for the tensor");
  if (reinterpret_cast<uintptr_t>(scale) % (d->scale_dtype == DGXM_DTYPE_F32 ? 4 : 2))
    return fail(DGXM_ERR_INVALID, "the given scale is not aligned to its type");
  if (!(d->scale_value >= 0.f) || d->scale_value > 3.4e38f)
    return fail(DGXM_ERR_INVALID, "the given scale must be finite and not negative");
  if (amax && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 4 ||
               workspace_bytes < dgxm_quantize_fp4_workspace()))
    return fail(DGXM_ERR_INVALID, "workspace of %lld bytes (%lld needed)", (long long)workspace_bytes,
                (long long)dgxm_quantize_fp4_workspace());
  if (d->rows == 0 && !nv) return DGXM_OK;  // nvfp4: the launch below still writes the scale (0 where none is given)
  Fp4Params p;
  bool vec = false;
  if (int rc = fp4_params(d, x, values, scales, fp4_groups(d->cols, d->format) * 4 * fp4_block(d->format) / kFp4Cols, &p, &vec)) return rc;
  p.scale = scale;
  p.scale_out = scale_out;
  p.partials = amax ? static_cast<uint32_t*>(workspace) : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  DGXM_CUDA_TRY(d->dtype == DGXM_DTYPE_BF16  ? fp4_quantize_typed<__nv_bfloat16>(p, d->format, vec, amax, st)
                : d->dtype == DGXM_DTYPE_F16 ? fp4_quantize_typed<__half>(p, d->format, vec, amax, st)
                                             : fp4_quantize_typed<float>(p, d->format, vec, amax, st));
  return DGXM_OK;
}

extern "C" int dgxm_dequantize_fp4(const dgxm_fp4_desc* d, const void* values, const void* scales, const float* scale,
                                   void* out, void* stream) {
  using namespace dgxm;
  if (int rc = fp4_check(d)) return rc;
  if ((d->format == DGXM_FP4_NVFP4) != (scale != nullptr) || reinterpret_cast<uintptr_t>(scale) % 4)
    return fail(DGXM_ERR_INVALID, "nvfp4 takes the tensor's fp32 scale, mxfp4 none");
  if (d->rows == 0) return DGXM_OK;
  Fp4Params p;
  bool vec = false;
  if (int rc = fp4_params(d, out, values, scales, (d->cols + 15) / 16, &p, &vec)) return rc;
  p.scale = scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  DGXM_CUDA_TRY(d->dtype == DGXM_DTYPE_BF16  ? fp4_dequantize_typed<__nv_bfloat16>(p, d->format, vec, st)
                : d->dtype == DGXM_DTYPE_F16 ? fp4_dequantize_typed<__half>(p, d->format, vec, st)
                                             : fp4_dequantize_typed<float>(p, d->format, vec, st));
  return DGXM_OK;
}
