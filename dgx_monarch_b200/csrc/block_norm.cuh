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
// Every value is moved once and takes a few operations, so DRAM bounds both as
// long as no warp waits for another's sums.  So the warps of a block share the
// work out by kind, a ring of rows in shared memory between them:
//   one fetches, a bulk copy a row and tensor, so that rows under way cost
//     neither registers nor instructions of the others;
//   three to eight take the rows' statistics, a row each at a time;
//   the rest make the outputs.  A thread of theirs holds the same columns of
//     every row, so the modulation of a sample and the weights stay in its
//     registers, and so do the sums over rows, which a second kernel adds in
//     the order of the blocks.
// Means and variances are fp32, gathered a chunk at a time from deviations
// (never as a difference of squares); every output is rounded once.
//
// Calls on B200: 9450 x 5120 bf16 with branch, gate and modulation 76 us (5.1
// TB/s), its gradient 118; 2 x 2640 x 2048 with fp32 values for each token 44;
// one row 10 us, which is the call.  With sums that all warps of a block wait
// for, the first two took 82 and 173 us.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "device_error.cuh"
#include "gemm_tile.cuh"
#include "ptx.cuh"

namespace dgxm {

constexpr int kBnMaxWidth = 8192;  // six fp32 rows fit the shared memory of a block
constexpr int kBnMaxIn = 6;
constexpr int kBnMaxSlots = 16;
// Streams of rows that a block reads: forward (x, branch, gate, scale, shift),
// backward (dy, dr, r, branch, gate, scale); the modulations where each token
// has its own.
enum { kBnX = 0, kBnBranch = 1, kBnGate = 2, kBnScale = 3, kBnShift = 4 };
enum { kBnDy = 0, kBnDr = 1, kBnR = 2, kBnBranchB = 3, kBnGateB = 4, kBnScaleB = 5 };

struct BlockNormParams {
  const char* in[kBnMaxIn];  // streams, NULL: absent
  int64_t in_sb[kBnMaxIn], in_sr[kBnMaxIn];  // bytes between samples, rows
  int in_elt[kBnMaxIn];      // bytes of a value: 4 for a modulation of fp32 beside 16-bit tensors
  int in_off[kBnMaxIn];      // bytes into the stage
  int in_pitch[kBnMaxIn];    // bytes of a row in the stage, a multiple of 16
  int n_in, slot_bytes, slots, param_bytes, stage_bytes;  // the ring, behind the statistics' copies, before the warps' staging
  // Values of a column that serve every row of a sample (gate, scale, shift), or all rows; NULL: absent
  const char *gate, *scale, *shift, *norm_w, *norm_b, *branch_w;
  int64_t gate_sb, scale_sb, shift_sb;  // bytes between samples
  int mod_f32, w_f32;
  char *out, *x_out;         // forward: y and r; backward: dbranch and dx
  int64_t out_sb, out_sr, x_out_sb, x_out_sr;  // bytes
  char *g_gate, *g_scale, *g_shift;  // backward, a row each token: contiguous
  float* partial;            // backward: (block + sample, 3, width)
  int want;                  // which of the three sums are wanted, a bit each
  int batch, seq, width, mode, branch_norm, factor;  // factor: backward, dn = e a with other than ones
  int64_t rows, rows_each;
  int rows_more;
  float eps, inv_width;
};

// A thread works on pairs of fp32 (sm_100 f32x2 arithmetic); a chunk, the 16
// bytes of the tensors' type that it takes at a time, is kPairs of them.
template <typename T>
constexpr int kBnChunk = 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ __forceinline__ uint64_t bn_widen2(uint32_t w);
template <>
__device__ __forceinline__ uint64_t bn_widen2<__nv_bfloat16>(uint32_t w) {
  return pk2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ uint64_t bn_widen2<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pk2(f.x, f.y);
}

__device__ __forceinline__ uint64_t bn_both(float v) { return pk2(v, v); }

__device__ __forceinline__ float bn_total(uint64_t v) {
  float lo, hi;
  upk2(v, lo, hi);
  return lo + hi;
}

// 16 bytes global -> this CTA's shared memory and on, `bytes` a multiple of
// 16, both ends aligned; completion counted on `bar`.
__device__ __forceinline__ void bn_bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// N pairs of chunk q (2 N values of T) of a staged row.  Rows off 16 bytes
// (!VEC) lie in the stage as they do in memory: `off` bytes behind a 16-byte
// border; values past the row's end read as zeros.
template <typename T, bool VEC, int N>
__device__ __forceinline__ void bn_read(const uint8_t* row, int off, int q, int width, uint64_t (&v)[N]) {
  constexpr int kWords = 2 * N / kBnChunk<T>;
  const uint4* p = reinterpret_cast<const uint4*>(row) + q * kWords;
#pragma unroll
  for (int k = 0; k < kWords; ++k) {
    uint4 w = p[k];
    if (!VEC && off) w = fp4_bytes_from(w, p[k + 1], off);
    if constexpr (sizeof(T) == 4) {
      v[2 * k] = pk2(__uint_as_float(w.x), __uint_as_float(w.y));
      v[2 * k + 1] = pk2(__uint_as_float(w.z), __uint_as_float(w.w));
    } else {
      v[4 * k] = bn_widen2<T>(w.x);
      v[4 * k + 1] = bn_widen2<T>(w.y);
      v[4 * k + 2] = bn_widen2<T>(w.z);
      v[4 * k + 3] = bn_widen2<T>(w.w);
    }
  }
  if (!VEC && (q + 1) * 2 * N > width) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float lo, hi;
      upk2(v[i], lo, hi);
      v[i] = pk2(q * 2 * N + 2 * i < width ? lo : 0.f, q * 2 * N + 2 * i + 1 < width ? hi : 0.f);
    }
  }
}

// One value of a column vector of T or fp32.
template <typename T>
__device__ __forceinline__ float bn_value(const char* base, int f32, int col) {
  return f32 ? reinterpret_cast<const float*>(base)[col] : static_cast<float>(reinterpret_cast<const T*>(base)[col]);
}

// 2 N values from column `col` on, `fill` without a vector or past its end, in
// whole 16-byte words; value by value only at the ends of a vector off 16 bytes.
template <typename V, int N>
__device__ __forceinline__ void bn_vector_of(const char* base, int col, int width, float fill, uint64_t (&v)[N]) {
  constexpr int kElt = static_cast<int>(sizeof(V)), kWords = 2 * N * kElt / 16 > 0 ? 2 * N * kElt / 16 : 1;
  const char* at = base + static_cast<int64_t>(col) * kElt;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
  const bool whole = 2 * N * kElt % 16 == 0 && col + 2 * N <= width;
  if (whole && (off == 0 || (col * kElt >= off && (col + 2 * N) * kElt + 16 - off <= width * kElt))) {
    const uint4* p = reinterpret_cast<const uint4*>(at - off);
    uint4 w[kWords + 1];
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = __ldg(p + k);
    if (off) {
      w[kWords] = __ldg(p + kWords);
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = fp4_bytes_from(w[k], w[k + 1], off);
    }
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
      if constexpr (kElt == 4) {
        v[2 * k] = pk2(__uint_as_float(u[0]), __uint_as_float(u[1]));
        if (N > 1) v[2 * k + 1] = pk2(__uint_as_float(u[2]), __uint_as_float(u[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4 && 4 * k + i < N; ++i) v[4 * k + i] = bn_widen2<V>(u[i]);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    v[i] = pk2(col + 2 * i < width ? bn_value<V>(base, 0, col + 2 * i) : fill,
               col + 2 * i + 1 < width ? bn_value<V>(base, 0, col + 2 * i + 1) : fill);
}

template <typename T, int N>
__device__ __forceinline__ void bn_vector(const char* base, int f32, int col, int width, float fill, uint64_t (&v)[N]) {
  if (base == nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = bn_both(fill);
  } else if (f32) {
    bn_vector_of<float>(base, col, width, fill, v);
  } else {
    bn_vector_of<T>(base, col, width, fill, v);
  }
}

// Bytes of a warp's staging for rows off 16 bytes: its chunks, and 16 more.
constexpr int kBnStage = 33 * 16;

// Store N pairs of a row from column `col` on.  Off 16 bytes (!VEC) the warp's
// chunks, neighbours in the row, pass through its staging: a lane stores an
// aligned word out of two of them, and the few values before the first word
// and behind the last go one by one.  (With the values of every chunk behind
// conditions of their own a row took 8000 cycles instead of 2000.)
template <typename T, bool VEC, int N>
__device__ __forceinline__ void bn_store(char* row, int col, int width, const uint64_t (&v)[N], uint8_t* stage) {
  float f[2 * N];
#pragma unroll
  for (int i = 0; i < N; ++i) upk2(v[i], f[2 * i], f[2 * i + 1]);
  constexpr int CH = 2 * N, kElt = static_cast<int>(sizeof(T)), kWords = CH * kElt / 16;
  uint4 w[kWords];
#pragma unroll
  for (int k = 0; k < kWords; ++k) {
    const float* g = f + k * (16 / kElt);
    if constexpr (kElt == 4) {
      w[k] = make_uint4(__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3]));
    } else {
      constexpr bool kHalf = std::is_same<T, __half>::value;
      w[k] = make_uint4(pack16<kHalf>(g[0], g[1]), pack16<kHalf>(g[2], g[3]), pack16<kHalf>(g[4], g[5]), pack16<kHalf>(g[6], g[7]));
    }
  }
  if constexpr (VEC) {
    uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<T*>(row) + col);
#pragma unroll
    for (int k = 0; k < kWords; ++k) to[k] = w[k];
  } else {
    using Elt = typename std::conditional<kElt == 4, uint32_t, uint16_t>::type;
    const int lane = threadIdx.x & 31, first = col - lane * CH;
    // The lanes with a chunk of the row are the first ones of the warp.
    const int lanes = min(32, (width - first + CH - 1) / CH);
    const uint32_t mask = lanes == 32 ? 0xffffffffu : (1u << lanes) - 1u;
#pragma unroll
    for (int k = 0; k < kWords; ++k) {  // (chunks of 32 bytes: first halves, then second ones)
      char* const to = row + static_cast<int64_t>(first) * kElt;
      if constexpr (kWords == 1) {
        reinterpret_cast<uint4*>(stage)[lane] = w[0];
        __syncwarp(mask);
        const int bytes = min(lanes * CH, width - first) * kElt;
        const int head = min(static_cast<int>(-reinterpret_cast<uintptr_t>(to) & 15u), bytes);
        const int words = (bytes - head) / 16, end = head + 16 * words;
        if (lane < words) {
          const uint4 a = reinterpret_cast<const uint4*>(stage)[lane];
          *reinterpret_cast<uint4*>(to + head + 16 * lane) =
              head ? fp4_bytes_from(a, reinterpret_cast<const uint4*>(stage)[lane + 1], head) : a;
        }
        for (int at = lane * kElt; at < head; at += lanes * kElt)
          *reinterpret_cast<Elt*>(to + at) = *reinterpret_cast<const Elt*>(stage + at);
        for (int at = end + lane * kElt; at < bytes; at += lanes * kElt)
          *reinterpret_cast<Elt*>(to + at) = *reinterpret_cast<const Elt*>(stage + at);
        __syncwarp(mask);
      } else {
        const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + 4 * k + i < width) reinterpret_cast<uint32_t*>(row)[col + 4 * k + i] = u[i];
      }
    }
  }
}

template <typename T, bool VEC, int N>
__device__ __forceinline__ void bn_store_mod(char* base, int64_t row, int f32, int col, int width, const uint64_t (&v)[N],
                                             uint8_t* stage) {
  if (f32) bn_store<float, VEC>(base + row * width * 4, col, width, v, stage);
  else bn_store<T, VEC>(base + row * width * static_cast<int>(sizeof(T)), col, width, v, stage);
}

// A block's rows: contiguous, one after the other.
struct BnWalk {
  int64_t row, last;
  int b, l, seq;
  int slot = 0, parity = 0, slots;
  __device__ __forceinline__ BnWalk(const BlockNormParams& p) : seq(p.seq), slots(p.slots) {
    // the first `rows_more` blocks have a row more than the others
    const int more = min(static_cast<int>(blockIdx.x), p.rows_more);
    row = static_cast<int64_t>(blockIdx.x) * p.rows_each + more;
    last = row + p.rows_each + (static_cast<int>(blockIdx.x) < p.rows_more);
    b = static_cast<int>(last <= 0xffffffffLL ? static_cast<uint32_t>(row) / static_cast<uint32_t>(seq) : row / seq);
    l = static_cast<int>(row - static_cast<int64_t>(b) * seq);
  }
  __device__ __forceinline__ bool more() const { return row < last; }
  __device__ __forceinline__ void next() {
    ++row;
    if (++l == seq) {
      l = 0;
      ++b;
    }
    if (++slot == slots) {
      slot = 0;
      parity ^= 1;
    }
  }
};

// A row's statistics.  n = (r - mean) root.
struct __align__(16) BnStats {
  float mean, root, root2, m1, m2, m3, spare[2];
};

struct BnShared {
  uint64_t full[kBnMaxSlots], ready[kBnMaxSlots], empty[kBnMaxSlots];
  BnStats stats[kBnMaxSlots];
};

// Every wait is bounded; after one that ran out, a warp waits no more.
__device__ __forceinline__ void bn_wait(uint64_t* bar, int parity, bool& dead) {
  if (!dead) dead = !mbar_wait(smem_u32(bar), parity, nullptr);
}

__device__ __forceinline__ void bn_start(const BlockNormParams& p, BnShared& sh, int out_warps) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.slots; ++s) {
      mbar_init(smem_u32(&sh.full[s]), 1);
      mbar_init(smem_u32(&sh.ready[s]), 1);
      mbar_init(smem_u32(&sh.empty[s]), out_warps);
    }
    mbar_fence_init();
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
}

// The fetching warp: lane i takes stream i.
template <bool VEC>
__device__ __forceinline__ void bn_fetch(const BlockNormParams& p, uint8_t* ring, BnShared& sh) {
  const int lane = threadIdx.x & 31;
  const bool mine = lane < p.n_in && p.in[lane < kBnMaxIn ? lane : 0] != nullptr;
  bool dead = false;
  BnWalk w(p);
  for (; w.more(); w.next()) {
    bn_wait(&sh.empty[w.slot], w.parity ^ 1, dead);
    if ((dead = __any_sync(0xffffffffu, dead))) break;  // nothing more is loaded over what may still be read
    const uint32_t full = smem_u32(&sh.full[w.slot]);
    uint8_t* to = ring + w.slot * p.slot_bytes;
    const char* from = nullptr;
    uint32_t bytes = 0;
    if (mine) {
      to += p.in_off[lane];
      from = p.in[lane] + w.b * p.in_sb[lane] + w.l * p.in_sr[lane];
      bytes = p.width * p.in_elt[lane];
    }
    if constexpr (!VEC) {
      // Whole 16-byte words by the bulk copy; the ends value by value, lanes 0 .. 7
      // the first and 8 .. 15 the last of the first half of the streams, the others the second's.
      constexpr int kHalf = kBnMaxIn / 2;
      const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from)) & 15u;
      const uint32_t head = min((16u - off) & 15u, bytes), tail = (bytes - head) & 15u;
      uint16_t end[kHalf];
      uint32_t at[kHalf];
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        const int s = i + (lane >= 16 ? kHalf : 0);
        const uint64_t f = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(from), s);
        const uint32_t n = __shfl_sync(0xffffffffu, bytes, s), h = __shfl_sync(0xffffffffu, head, s);
        const uint32_t e = __shfl_sync(0xffffffffu, tail, s), unit = 2 * (lane & 7);
        at[i] = (lane & 8) == 0 ? (unit < h ? unit : ~0u) : (unit < e ? n - e + unit : ~0u);
        if (at[i] != ~0u) end[i] = *reinterpret_cast<const uint16_t*>(f + at[i]);
      }
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        const int s = i + (lane >= 16 ? kHalf : 0);
        const uint32_t dst = __shfl_sync(0xffffffffu, smem_u32(to) + off, s);
        if (at[i] != ~0u) asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + at[i]), "h"(end[i]) : "memory");
      }
      // Rows of a slot lie at different offsets: this row's words cover bytes that an earlier row's ends were stored to.
      tma_store_fence();
      to += off + head;
      from += head;
      bytes -= head + tail;
    }
    const uint32_t sum = __reduce_add_sync(0xffffffffu, bytes);
    __syncwarp();  // the ends' stores come before lane 0's arrival
    if (lane == 0) {
      if (sum > 0) mbar_expect_tx(full, sum);
      else mbar_arrive(full);
    }
    __syncwarp();
    if (bytes > 0) bn_bulk_load(smem_u32(to), from, bytes, full);
  }
  if (dead) report_device_error(kErrProducerTimeout);
  // Every load lands before the block can exit, also where its readers have given up waiting.  (Slots before the walk's are
  // a round ahead of the others; of one never used the round before its first counts as over.)
  for (int s = 0; s < p.slots; ++s) mbar_wait(smem_u32(&sh.full[s]), s < w.slot ? w.parity : w.parity ^ 1, nullptr);
}

// Bytes that a row of stream s lies behind a 16-byte border.
template <bool VEC>
__device__ __forceinline__ int bn_offset(const BlockNormParams& p, int s, const BnWalk& w) {
  if (VEC) return 0;
  return static_cast<int>(reinterpret_cast<uintptr_t>(p.in[s] + w.b * p.in_sb[s] + w.l * p.in_sr[s]) & 15);
}

// Chunk q of stream s of the row in `slot`: the tensors, and the modulations of each token.
template <typename T, bool VEC, int N>
__device__ __forceinline__ void bn_get(const BlockNormParams& p, const uint8_t* slot, int s, const BnWalk& w, int q,
                                       uint64_t (&v)[N]) {
  bn_read<T, VEC>(slot + p.in_off[s], bn_offset<VEC>(p, s, w), q, p.width, v);
}

template <typename T, bool VEC, int N>
__device__ __forceinline__ void bn_get_mod(const BlockNormParams& p, const uint8_t* slot, int s, const BnWalk& w, int q,
                                           uint64_t (&v)[N]) {
  if (p.mod_f32) bn_get<float, VEC>(p, slot, s, w, q, v);
  else bn_get<T, VEC>(p, slot, s, w, q, v);
}

// ------------------------------------------------------------ the statistics' warps
// A row is one warp's: its sums are shuffles, and several rows' latencies overlap.
template <int N>
__device__ __forceinline__ void bn_warp_sum(float (&v)[N]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}

// Count, mean and sum of squared deviations of a set, and of two sets
// together: every term of the sum is positive, so nothing cancels.
struct BnMoments {
  float n = 0.f, mean = 0.f, m2 = 0.f;
  __device__ __forceinline__ void add(float on, float omean, float om2) {
    const float all = n + on, share = all > 0.f ? __fdividef(on, all) : 0.f, delta = omean - mean;
    mean = fmaf(delta, share, mean);
    m2 += fmaf(delta * delta, n * share, om2);
    n = all;
  }
};

// The moments of a chunk's first `count` values (the rest are zeros).
template <int N>
__device__ __forceinline__ void bn_add_chunk(BnMoments& all, uint64_t (&v)[N], int count) {
  uint64_t s = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) s = fadd2(s, v[i]);
  const float mean = bn_total(s) * (count == 2 * N ? 1.f / (2 * N) : 1.f / count);
  uint64_t ss = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint64_t d = fadd2(v[i], bn_both(-mean));
    if (count < 2 * N) {
      float lo, hi;
      upk2(d, lo, hi);
      d = pk2(2 * i < count ? lo : 0.f, 2 * i + 1 < count ? hi : 0.f);
    }
    ss = ffma2(d, d, ss);
  }
  all.add(static_cast<float>(count), mean, bn_total(ss));
}

// Mean and mean squared deviation over the warp.
__device__ __forceinline__ float2 bn_warp_moments(BnMoments v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float n = __shfl_down_sync(0xffffffffu, v.n, o), mean = __shfl_down_sync(0xffffffffu, v.mean, o);
    const float m2 = __shfl_down_sync(0xffffffffu, v.m2, o);
    v.add(n, mean, m2);
  }
  return make_float2(__shfl_sync(0xffffffffu, v.mean, 0), __shfl_sync(0xffffffffu, __fdividef(v.m2, v.n), 0));
}

// The statistics' copy of column vectors of the row's sample, `each` values
// one: loaded when the sample changes, which every one of their warps sees at
// the same row.
template <int WARPS, typename Make>
__device__ __forceinline__ void bn_param(const BlockNormParams& p, float* param, int t, int each, Make&& make) {
  if (p.param_bytes == 0) return;
  named_barrier_sync(1, WARPS * 32);
  for (int which = 0; which * each < p.param_bytes / 4; ++which)
#pragma unroll 8
    for (int c = t; c < each; c += WARPS * 32) param[which * each + c] = c < p.width ? make(c, which) : 0.f;
  named_barrier_sync(1, WARPS * 32);
}

template <int N>
__device__ __forceinline__ void bn_param_get(const float* param, int q, uint64_t (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float4 f = *reinterpret_cast<const float4*>(param + q * 2 * N + 2 * i);
    v[i] = pk2(f.x, f.y);
    v[i + 1] = pk2(f.z, f.w);
  }
}

// What a row's values are made of, for its mean and squares: one stream
// (kBnAlone); x plus a branch as it is, times a vector of the statistics' copy,
// or times a gate of each token; or (kBnAny) whatever the parameters say.  Each
// has a loop of its own: ways not taken between the few instructions of one
// cost more than the instructions (250 cycles a chunk instead of 100).
enum { kBnAlone, kBnPlain, kBnScaled, kBnToken, kBnAny };

// Sum (of deviations from the mean, in LAYER) of squares, and the mean, over a row: one warp's.
template <typename T, bool VEC, bool FULL, bool LAYER, int SRC>
__device__ __forceinline__ float2 bn_row_sums(const BlockNormParams& p, const uint8_t* slot, int s, const BnWalk& w,
                                              const float* param, float root2) {
  constexpr int CH = kBnChunk<T>, N = CH / 2;
  const int lane = threadIdx.x & 31;
  BnMoments moments;
  uint64_t ss = 0;
#pragma unroll 2
  for (int q = lane; q * CH < p.width; q += 32) {
    uint64_t r[N];
    bn_get<T, VEC>(p, slot, s, w, q, r);
    if constexpr (SRC != kBnAlone) {
      uint64_t m[N], g[N];
      bn_get<T, VEC>(p, slot, kBnBranch, w, q, m);
      if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < N; ++i) m[i] = fmul2(m[i], bn_both(root2));
      }
      if constexpr (SRC == kBnToken || SRC == kBnAny) {
        if (SRC == kBnToken || p.in[kBnGate] != nullptr) {
          bn_get_mod<T, VEC>(p, slot, kBnGate, w, q, g);
#pragma unroll
          for (int i = 0; i < N; ++i) m[i] = fmul2(m[i], g[i]);
        }
      }
      if constexpr (SRC == kBnAny) {
        bn_vector<T>(p.gate ? p.gate + w.b * p.gate_sb : nullptr, p.mod_f32, q * CH, p.width, 1.f, g);
#pragma unroll
        for (int i = 0; i < N; ++i) m[i] = fmul2(m[i], g[i]);
        bn_vector<T>(p.branch_w, p.w_f32, q * CH, p.width, 1.f, g);
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = ffma2(g[i], m[i], r[i]);
      } else if (SRC == kBnScaled || (SRC == kBnToken && p.param_bytes > 0)) {
        bn_param_get(param, q, g);
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = ffma2(g[i], m[i], r[i]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = fadd2(r[i], m[i]);
      }
    }
    if constexpr (LAYER) {
      bn_add_chunk(moments, r, VEC ? CH : min(CH, p.width - q * CH));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) ss = ffma2(r[i], r[i], ss);
    }
  }
  if constexpr (LAYER) {
    return bn_warp_moments(moments);
  } else {
    float sum[1] = {bn_total(ss)};
    bn_warp_sum(sum);
    return make_float2(0.f, sum[0] * p.inv_width);
  }
}

template <typename T, bool VEC, bool FULL, int SRC>
__device__ __forceinline__ float2 bn_row_stats(const BlockNormParams& p, const uint8_t* slot, int s, const BnWalk& w,
                                               const float* param, float root2) {
  return p.mode == DGXM_BLOCK_NORM_LAYER ? bn_row_sums<T, VEC, FULL, true, SRC>(p, slot, s, w, param, root2)
                                         : bn_row_sums<T, VEC, FULL, false, SRC>(p, slot, s, w, param, root2);
}

template <typename T, bool VEC, bool FULL, int STAT>
__device__ __forceinline__ void bn_forward_stats(const BlockNormParams& p, float* param, const uint8_t* ring, BnShared& sh,
                                                 int t) {
  const int lane = t & 31;
  // Rows in turn, by no more warps than there are slots, whose number is a
  // multiple: all rows of a slot are one warp's, so that none waits for a phase
  // of a slot whose last one may still be open (rows land in any order).
  const int warps = min(STAT, p.slots);
  int turn = t >> 5 < warps ? t >> 5 : 0x7fffffff;  // rows until this warp's next
  const bool wanted = p.gate != nullptr || p.branch_w != nullptr;
  const int src = p.in[kBnBranch] == nullptr          ? kBnAlone
                  : wanted && p.param_bytes == 0      ? kBnAny
                  : FULL && p.in[kBnGate] != nullptr  ? kBnToken
                  : wanted                            ? kBnScaled
                                                      : kBnPlain;
  int sample = -1;
  bool dead = false;
  for (BnWalk w(p); w.more(); w.next()) {
    if (w.b != sample) {
      sample = w.b;
      bn_param<STAT>(p, param, t, p.param_bytes / 4, [&](int c, int) {
        const float g = p.gate ? bn_value<T>(p.gate + sample * p.gate_sb, p.mod_f32, c) : 1.f;
        return FULL && p.branch_w ? g * bn_value<T>(p.branch_w, p.w_f32, c) : g;
      });
    }
    if (turn-- > 0) continue;
    turn = warps - 1;
    bn_wait(&sh.full[w.slot], w.parity, dead);
    const uint8_t* slot = ring + w.slot * p.slot_bytes;
    float root2 = 1.f;
    if (FULL && p.branch_norm)
      root2 = rsqrtf(bn_row_sums<T, VEC, FULL, false, kBnAlone>(p, slot, kBnBranch, w, param, 1.f).y + p.eps);
    float2 v = make_float2(0.f, 0.f);
    if (p.mode != DGXM_BLOCK_NORM_NONE) {
      if (src == kBnScaled) v = bn_row_stats<T, VEC, FULL, kBnScaled>(p, slot, kBnX, w, param, root2);
      else if (src == kBnAlone) v = bn_row_stats<T, VEC, FULL, kBnAlone>(p, slot, kBnX, w, param, root2);
      else if (src == kBnPlain) v = bn_row_stats<T, VEC, FULL, kBnPlain>(p, slot, kBnX, w, param, root2);
      else if (FULL && src == kBnToken) v = bn_row_stats<T, VEC, FULL, FULL ? kBnToken : kBnAlone>(p, slot, kBnX, w, param, root2);
      else v = bn_row_stats<T, VEC, FULL, kBnAny>(p, slot, kBnX, w, param, root2);
    }
    if (lane == 0) {
      sh.stats[w.slot].mean = v.x;
      sh.stats[w.slot].root = rsqrtf(v.y + p.eps);
      sh.stats[w.slot].root2 = root2;
      mbar_arrive(smem_u32(&sh.ready[w.slot]));
    }
  }
  if (dead) report_device_error(kErrSoftmaxTimeout);
}

// ------------------------------------------------------------ the kernels
// The warps that make the outputs hold E values a thread, chunks of 16 bytes
// t, t + threads, ... of each row.  FULL: with a branch norm, or modulations
// of each token.
template <typename T, int E, bool VEC, bool FULL, int MAXT, int STAT, int PER_SM>
__global__ void __launch_bounds__(MAXT + 32 * STAT + 32, PER_SM) block_norm_kernel(const __grid_constant__ BlockNormParams p) {
  constexpr int CH = kBnChunk<T>, NV = E / CH, N = CH / 2;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ BnShared sh;
  const int threads = blockDim.x - 32 * STAT - 32, t = threadIdx.x;
  uint8_t* ring = smem + p.param_bytes;
  bn_start(p, sh, threads >> 5);
  if (t >= threads + 32 * STAT) {
    bn_fetch<VEC>(p, ring, sh);
    return;
  }
  if (t >= threads) {
    bn_forward_stats<T, VEC, FULL, STAT>(p, reinterpret_cast<float*>(smem), ring, sh, t - threads);
    return;
  }
  const bool branch = p.in[kBnBranch] != nullptr, norm = p.mode != DGXM_BLOCK_NORM_NONE;
  uint64_t g[NV][N], a[NV][N], c[NV][N];
  uint8_t* const stage = ring + p.slots * p.slot_bytes + (t >> 5) * kBnStage;  // (where !VEC)
  int sample = -1;
  bool dead = false;
  for (BnWalk w(p); w.more(); w.next()) {
    if (w.b != sample) {
      sample = w.b;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (t + k * threads) * CH;
        uint64_t wt[N], bias[N];
        bn_vector<T>(p.gate ? p.gate + sample * p.gate_sb : nullptr, p.mod_f32, col, p.width, 1.f, g[k]);
        bn_vector<T>(p.scale ? p.scale + sample * p.scale_sb : nullptr, p.mod_f32, col, p.width, 0.f, a[k]);
        bn_vector<T>(p.shift ? p.shift + sample * p.shift_sb : nullptr, p.mod_f32, col, p.width, 0.f, c[k]);
        if constexpr (FULL) {  // r = x + g m, with the branch's weight in g
          if (p.branch_w != nullptr) {
            bn_vector<T>(p.branch_w, p.w_f32, col, p.width, 1.f, wt);
#pragma unroll
            for (int i = 0; i < N; ++i) g[k][i] = fmul2(g[k][i], wt[i]);
          }
        }
        bn_vector<T>(p.norm_w, p.w_f32, col, p.width, 1.f, wt);
        bn_vector<T>(p.norm_b, p.w_f32, col, p.width, 0.f, bias);
#pragma unroll
        for (int i = 0; i < N; ++i) {  // y = n a + c
          a[k][i] = fadd2(a[k][i], bn_both(1.f));
          c[k][i] = ffma2(bias[i], a[k][i], c[k][i]);
          a[k][i] = fmul2(a[k][i], wt[i]);
        }
      }
    }
    bn_wait(&sh.full[w.slot], w.parity, dead);
    bn_wait(&sh.ready[w.slot], w.parity, dead);
    const uint8_t* slot = ring + w.slot * p.slot_bytes;
    const BnStats st = sh.stats[w.slot];
    char* const to_r = p.x_out + w.b * p.x_out_sb + w.l * p.x_out_sr;
    char* const to_y = p.out + w.b * p.out_sb + w.l * p.out_sr;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = t + k * threads, col = q * CH;
      if (col >= p.width) continue;
      uint64_t r[N];
      bn_get<T, VEC>(p, slot, kBnX, w, q, r);
      if (branch) {
        uint64_t m[N];
        bn_get<T, VEC>(p, slot, kBnBranch, w, q, m);
        if constexpr (FULL) {
#pragma unroll
          for (int i = 0; i < N; ++i) m[i] = fmul2(m[i], bn_both(st.root2));
          if (p.in[kBnGate] != nullptr) {
            uint64_t of[N];
            bn_get_mod<T, VEC>(p, slot, kBnGate, w, q, of);
#pragma unroll
            for (int i = 0; i < N; ++i) m[i] = fmul2(m[i], of[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = ffma2(g[k][i], m[i], r[i]);
        bn_store<T, VEC>(to_r, col, p.width, r, stage);
      }
      if (!norm) continue;
#pragma unroll
      for (int i = 0; i < N; ++i)
        r[i] = ffma2(fmul2(fadd2(r[i], bn_both(-st.mean)), bn_both(st.root)), a[k][i], c[k][i]);
      if constexpr (FULL) {
        uint64_t s[N];
        if (p.in[kBnScale] != nullptr) {
          bn_get_mod<T, VEC>(p, slot, kBnScale, w, q, s);
#pragma unroll
          for (int i = 0; i < N; ++i) r[i] = ffma2(r[i], s[i], r[i]);
        }
        if (p.in[kBnShift] != nullptr) {
          bn_get_mod<T, VEC>(p, slot, kBnShift, w, q, s);
#pragma unroll
          for (int i = 0; i < N; ++i) r[i] = fadd2(r[i], s[i]);
        }
      }
      bn_store<T, VEC>(to_y, col, p.width, r, stage);
    }
    __syncwarp();
    if ((t & 31) == 0) mbar_arrive(smem_u32(&sh.empty[w.slot]));
  }
  if (dead) report_device_error(kErrEpilogueTimeout);
}

// The gradient's row of one chunk: e = dy, under a scale of each token dh, and n.
template <typename T, bool VEC, int N>
__device__ __forceinline__ void bn_normed(const BlockNormParams& p, const uint8_t* slot, const BnWalk& w, const BnStats& st,
                                          int q, uint64_t (&e)[N], uint64_t (&n)[N]) {
  bn_get<T, VEC>(p, slot, kBnDy, w, q, e);
  bn_get<T, VEC>(p, slot, kBnR, w, q, n);
#pragma unroll
  for (int i = 0; i < N; ++i) n[i] = fmul2(fadd2(n[i], bn_both(-st.mean)), bn_both(st.root));
  if (!VEC && (q + 1) * 2 * N > p.width) {  // zeros past the row's end
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float lo, hi;
      upk2(n[i], lo, hi);
      n[i] = pk2(q * 2 * N + 2 * i < p.width ? lo : 0.f, q * 2 * N + 2 * i + 1 < p.width ? hi : 0.f);
    }
  }
}

template <typename T, bool VEC, bool FULL, int N>
__device__ __forceinline__ void bn_modulate(const BlockNormParams& p, const uint8_t* slot, const BnWalk& w, int q,
                                            uint64_t (&e)[N]) {
  if (!FULL || p.in[kBnScaleB] == nullptr) return;
  uint64_t s[N];
  bn_get_mod<T, VEC>(p, slot, kBnScaleB, w, q, s);
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = ffma2(e[i], s[i], e[i]);
}

// R, the stream's gradient; dn = e a.
template <typename T, bool VEC, int N>
__device__ __forceinline__ void bn_stream_grad(const BlockNormParams& p, const uint8_t* slot, const BnWalk& w,
                                               const BnStats& st, int q, const uint64_t (&e)[N], const uint64_t (&n)[N],
                                               const uint64_t (&a)[N], uint64_t (&big)[N]) {
  if (p.in[kBnDr] != nullptr) {
    bn_get<T, VEC>(p, slot, kBnDr, w, q, big);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) big[i] = 0;
  }
  if (p.mode == DGXM_BLOCK_NORM_NONE) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint64_t inner = ffma2(e[i], a[i], ffma2(n[i], bn_both(-st.m2), bn_both(-st.m1)));
    big[i] = ffma2(bn_both(st.root), inner, big[i]);
  }
}

// The factor a of dn = e a: ones, the statistics' copy, or (kBnAny) from memory.
template <typename T, int SRC, int N>
__device__ __forceinline__ void bn_factor(const BlockNormParams& p, const float* param, const BnWalk& w, int q, uint64_t (&a)[N]) {
  if constexpr (SRC == kBnScaled) {
    bn_param_get(param, q, a);
  } else if constexpr (SRC == kBnPlain) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = bn_both(1.f);
  } else {
    uint64_t wt[N];
    bn_vector<T>(p.scale ? p.scale + w.b * p.scale_sb : nullptr, p.mod_f32, q * 2 * N, p.width, 0.f, a);
    bn_vector<T>(p.norm_w, p.w_f32, q * 2 * N, p.width, 1.f, wt);
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = fmul2(fadd2(a[i], bn_both(1.f)), wt[i]);
  }
}

// Sums of dn and dn n over a row.
template <typename T, bool VEC, bool FULL, int SRC>
__device__ __forceinline__ float2 bn_row_dn(const BlockNormParams& p, const uint8_t* slot, const BnWalk& w, const BnStats& st,
                                            const float* param) {
  constexpr int CH = kBnChunk<T>, N = CH / 2;
  uint64_t s1[N] = {}, s2[N] = {};
#pragma unroll 2
  for (int q = threadIdx.x & 31; q * CH < p.width; q += 32) {
    uint64_t e[N], n[N], a[N];
    bn_normed<T, VEC>(p, slot, w, st, q, e, n);
    bn_modulate<T, VEC, FULL>(p, slot, w, q, e);
    bn_factor<T, SRC>(p, param, w, q, a);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint64_t dn = fmul2(e[i], a[i]);
      s1[i] = fadd2(s1[i], dn);
      s2[i] = ffma2(dn, n[i], s2[i]);
    }
  }
#pragma unroll
  for (int i = 1; i < N; ++i) {
    s1[0] = fadd2(s1[0], s1[i]);
    s2[0] = fadd2(s2[0], s2[i]);
  }
  float sums[2] = {bn_total(s1[0]), bn_total(s2[0])};
  bn_warp_sum(sums);
  return make_float2(sums[0], sums[1]);
}

// The sum of dn2 n2 over a row.  The second vector of the statistics' copy is
// what R is multiplied by to dn2, without a gate of each token.
template <typename T, bool VEC, int SRC>
__device__ __forceinline__ float bn_row_dn2(const BlockNormParams& p, const uint8_t* slot, const BnWalk& w, const BnStats& st,
                                            const float* param) {
  constexpr int CH = kBnChunk<T>, N = CH / 2;
  uint64_t part[N] = {};
  for (int q = threadIdx.x & 31; q * CH < p.width; q += 32) {
    uint64_t e[N], n[N], a[N], big[N];
    if (p.mode != DGXM_BLOCK_NORM_NONE) {
      bn_normed<T, VEC>(p, slot, w, st, q, e, n);
      bn_modulate<T, VEC, true>(p, slot, w, q, e);
      if (SRC == kBnScaled && p.factor == 0) bn_factor<T, kBnPlain>(p, param, w, q, a);
      else bn_factor<T, SRC>(p, param, w, q, a);
    }
    bn_stream_grad<T, VEC>(p, slot, w, st, q, e, n, a, big);
    bn_get<T, VEC>(p, slot, kBnBranchB, w, q, n);
    if (p.in[kBnGateB] != nullptr) {
      bn_get_mod<T, VEC>(p, slot, kBnGateB, w, q, a);
#pragma unroll
      for (int i = 0; i < N; ++i) big[i] = fmul2(big[i], a[i]);
    }
    if constexpr (SRC == kBnScaled) {
      bn_param_get(param + p.param_bytes / 8, q, a);
    } else {
      bn_vector<T>(p.gate ? p.gate + w.b * p.gate_sb : nullptr, p.mod_f32, q * CH, p.width, 1.f, a);
      bn_vector<T>(p.branch_w, p.w_f32, q * CH, p.width, 1.f, e);
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] = fmul2(a[i], e[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = ffma2(fmul2(big[i], a[i]), n[i], part[i]);
  }
#pragma unroll
  for (int i = 1; i < N; ++i) part[0] = fadd2(part[0], part[i]);
  float sum[1] = {bn_total(part[0])};
  bn_warp_sum(sum);
  return sum[0] * st.root2;
}

template <typename T, bool VEC, bool FULL, int STAT>
__device__ __forceinline__ void bn_backward_stats(const BlockNormParams& p, float* param, const uint8_t* ring, BnShared& sh,
                                                  int t) {
  const int lane = t & 31;
  // Rows in turn, by no more warps than there are slots, whose number is a
  // multiple: all rows of a slot are one warp's, so that none waits for a phase
  // of a slot whose last one may still be open (rows land in any order).
  const int warps = min(STAT, p.slots);
  int turn = t >> 5 < warps ? t >> 5 : 0x7fffffff;  // rows until this warp's next
  const bool norm = p.mode != DGXM_BLOCK_NORM_NONE, layer = p.mode == DGXM_BLOCK_NORM_LAYER;
  const bool post = FULL && p.branch_norm;
  int sample = -1;
  bool dead = false;
  for (BnWalk w(p); w.more(); w.next()) {
    if (w.b != sample) {
      sample = w.b;
      const char* const scale = p.scale ? p.scale + sample * p.scale_sb : nullptr;
      const int each = post ? p.param_bytes / 8 : p.param_bytes / 4;  // values of a vector
      bn_param<STAT>(p, param, t, each, [&](int c, int which) {
        if (which == 0) {
          const float up = scale ? 1.f + bn_value<T>(scale, p.mod_f32, c) : 1.f;
          return p.norm_w ? up * bn_value<T>(p.norm_w, p.w_f32, c) : up;
        }
        const float g = p.gate ? bn_value<T>(p.gate + sample * p.gate_sb, p.mod_f32, c) : 1.f;
        return p.branch_w ? g * bn_value<T>(p.branch_w, p.w_f32, c) : g;
      });
    }
    if (turn-- > 0) continue;
    turn = warps - 1;
    bn_wait(&sh.full[w.slot], w.parity, dead);
    const uint8_t* slot = ring + w.slot * p.slot_bytes;
    BnStats st;
    st.mean = st.root = st.m1 = st.m2 = st.m3 = 0.f;
    st.root2 = 1.f;
    if (norm) {
      float2 v = bn_row_stats<T, VEC, FULL, kBnAlone>(p, slot, kBnR, w, param, 1.f);
      st.mean = v.x;
      st.root = rsqrtf(v.y + p.eps);
      if (p.factor == 0) v = bn_row_dn<T, VEC, FULL, kBnPlain>(p, slot, w, st, param);
      else if (p.param_bytes > 0) v = bn_row_dn<T, VEC, FULL, kBnScaled>(p, slot, w, st, param);
      else v = bn_row_dn<T, VEC, FULL, kBnAny>(p, slot, w, st, param);
      st.m1 = layer ? v.x * p.inv_width : 0.f;
      st.m2 = v.y * p.inv_width;
    }
    if constexpr (FULL) {
      if (post) {
        st.root2 = rsqrtf(bn_row_sums<T, VEC, FULL, false, kBnAlone>(p, slot, kBnBranchB, w, param, 1.f).y + p.eps);
        const float sum = p.param_bytes > 0 ? bn_row_dn2<T, VEC, kBnScaled>(p, slot, w, st, param)
                                            : bn_row_dn2<T, VEC, kBnAny>(p, slot, w, st, param);
        st.m3 = sum * p.inv_width;
      }
    }
    if (lane == 0) {
      sh.stats[w.slot] = st;
      mbar_arrive(smem_u32(&sh.ready[w.slot]));
    }
  }
  if (dead) report_device_error(kErrSoftmaxTimeout);
}

// The gradient.  The sums over rows that a thread keeps for its columns are
//   0: sum e,  1: sum e n,  2: sum f n2
// with e = dy and f = R where the modulation serves a sample, so that the
// gradients of weights and modulations both follow from them, and e = dh,
// f = dm where each token has its own (n2 = branch without a branch norm).
template <typename T, int E, bool VEC, bool FULL, int MAXT, int STAT, int PER_SM>
__global__ void __launch_bounds__(MAXT + 32 * STAT + 32, PER_SM) block_norm_backward_kernel(const __grid_constant__ BlockNormParams p) {
  constexpr int CH = kBnChunk<T>, NV = E / CH, N = CH / 2;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ BnShared sh;
  const int threads = blockDim.x - 32 * STAT - 32, t = threadIdx.x;
  uint8_t* ring = smem + p.param_bytes;
  bn_start(p, sh, threads >> 5);
  if (t >= threads + 32 * STAT) {
    bn_fetch<VEC>(p, ring, sh);
    return;
  }
  if (t >= threads) {
    bn_backward_stats<T, VEC, FULL, STAT>(p, reinterpret_cast<float*>(smem), ring, sh, t - threads);
    return;
  }
  const bool branch = p.in[kBnBranchB] != nullptr, norm = p.mode != DGXM_BLOCK_NORM_NONE;
  uint64_t g[NV][N], a[NV][N], acc[3][NV][N];
  uint8_t* const stage = ring + p.slots * p.slot_bytes + (t >> 5) * kBnStage;  // (where !VEC)
  int sample = -1;
  bool dead = false;
  auto flush = [&]() {
    if (sample < 0 || p.partial == nullptr) return;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      if (!(p.want >> j & 1)) continue;
      char* to = reinterpret_cast<char*>(p.partial + ((blockIdx.x + static_cast<int64_t>(sample)) * 3 + j) * p.width);
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (const int col = (t + k * threads) * CH; col < p.width) bn_store<float, VEC>(to, col, p.width, acc[j][k], stage);
    }
  };
  for (BnWalk w(p); w.more(); w.next()) {
    if (w.b != sample) {
      flush();
      sample = w.b;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (t + k * threads) * CH;
        uint64_t wt[N];
        bn_vector<T>(p.gate ? p.gate + sample * p.gate_sb : nullptr, p.mod_f32, col, p.width, 1.f, g[k]);
        bn_vector<T>(p.scale ? p.scale + sample * p.scale_sb : nullptr, p.mod_f32, col, p.width, 0.f, a[k]);
        if constexpr (FULL) {  // dn2 = R g, with the branch's weight in g
          if (p.branch_w != nullptr) {
            bn_vector<T>(p.branch_w, p.w_f32, col, p.width, 1.f, wt);
#pragma unroll
            for (int i = 0; i < N; ++i) g[k][i] = fmul2(g[k][i], wt[i]);
          }
        }
        bn_vector<T>(p.norm_w, p.w_f32, col, p.width, 1.f, wt);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          a[k][i] = fmul2(fadd2(a[k][i], bn_both(1.f)), wt[i]);
          acc[0][k][i] = acc[1][k][i] = acc[2][k][i] = 0;
        }
      }
    }
    bn_wait(&sh.full[w.slot], w.parity, dead);
    bn_wait(&sh.ready[w.slot], w.parity, dead);
    const uint8_t* slot = ring + w.slot * p.slot_bytes;
    const BnStats st = sh.stats[w.slot];
    char* const to_x = p.x_out + w.b * p.x_out_sb + w.l * p.x_out_sr;
    char* const to_m = p.out + w.b * p.out_sb + w.l * p.out_sr;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int q = t + k * threads, col = q * CH;
      if (col >= p.width) continue;
      uint64_t e[N], n[N], big[N];
      if (norm) {
        bn_normed<T, VEC>(p, slot, w, st, q, e, n);
        if constexpr (FULL) {
          if (p.g_scale != nullptr) {  // a token's own: dy h
            uint64_t h[N], bias[N];
            bn_vector<T>(p.norm_w, p.w_f32, col, p.width, 1.f, h);
            bn_vector<T>(p.norm_b, p.w_f32, col, p.width, 0.f, bias);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = fmul2(e[i], ffma2(n[i], h[i], bias[i]));
            bn_store_mod<T, VEC>(p.g_scale, w.row, p.mod_f32, col, p.width, h, stage);
          }
          if (p.g_shift != nullptr) bn_store_mod<T, VEC>(p.g_shift, w.row, p.mod_f32, col, p.width, e, stage);
        }
        bn_modulate<T, VEC, FULL>(p, slot, w, q, e);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          acc[0][k][i] = fadd2(acc[0][k][i], e[i]);
          acc[1][k][i] = ffma2(e[i], n[i], acc[1][k][i]);
        }
      }
      bn_stream_grad<T, VEC>(p, slot, w, st, q, e, n, a[k], big);
      if (p.x_out != nullptr) bn_store<T, VEC>(to_x, col, p.width, big, stage);
      if (!branch) continue;
      uint64_t m[N];
      bn_get<T, VEC>(p, slot, kBnBranchB, w, q, m);
      if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < N; ++i) m[i] = fmul2(m[i], bn_both(st.root2));
        if (p.in[kBnGateB] != nullptr) {
          uint64_t of[N];
          if (p.g_gate != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) of[i] = fmul2(fmul2(big[i], m[i]), g[k][i]);
            bn_store_mod<T, VEC>(p.g_gate, w.row, p.mod_f32, col, p.width, of, stage);
          }
          bn_get_mod<T, VEC>(p, slot, kBnGateB, w, q, of);
#pragma unroll
          for (int i = 0; i < N; ++i) big[i] = fmul2(big[i], of[i]);  // f = dm
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        acc[2][k][i] = ffma2(big[i], m[i], acc[2][k][i]);
        big[i] = fmul2(big[i], g[k][i]);
      }
      if (p.out == nullptr) continue;
      if (FULL && p.branch_norm) {
#pragma unroll
        for (int i = 0; i < N; ++i) big[i] = fmul2(bn_both(st.root2), ffma2(m[i], bn_both(-st.m3), big[i]));
      }
      bn_store<T, VEC>(to_m, col, p.width, big, stage);
    }
    __syncwarp();
    if ((t & 31) == 0) mbar_arrive(smem_u32(&sh.empty[w.slot]));
  }
  flush();
  if (dead) report_device_error(kErrEpilogueTimeout);
}

inline int64_t bn_rows(const dgxm_block_norm_desc* d) { return static_cast<int64_t>(d->batch) * d->seq; }

// How a call is cut: sixteen values a thread that makes outputs; for narrow
// (0), middle (1) and wide (2) rows, how many of those a block has at the most
// and how many warps for the statistics.
constexpr int kBnEach = 16;

template <bool BACK, int SIZE>
struct BnKind {
  static constexpr int kThreads = SIZE == 0 ? 128 : SIZE == 1 ? 320 : 512;
  static constexpr int kStat = SIZE == 1 ? (BACK ? 5 : 8) : 3;
  static constexpr int kMost = kThreads + 32 * kStat + 32;
  // blocks of an SM of the most threads by the registers of its warps, which come in fours
  static constexpr int kPerSm = SIZE == 0 ? (BACK ? 2 : 3) : 1;
};

struct BnCut {
  int threads, blocks, per_sm;
};

inline int bn_size(const dgxm_block_norm_desc* d) { return d->width <= 2048 ? 0 : d->width <= 5120 ? 1 : 2; }

template <bool BACK, int SIZE>
static BnCut bn_cut_of(const dgxm_block_norm_desc* d) {
  using K = BnKind<BACK, SIZE>;
  BnCut cut;
  cut.threads = ((d->width + kBnEach - 1) / kBnEach + 31) / 32 * 32;
  // by their registers: rows below the kind's widest have smaller blocks (9450 x 512, forward and gradient: 19.7 and 47 us
  // with 3 and 2 blocks an SM, 17.7 and 35 with 4 and 3)
  cut.per_sm = K::kPerSm * K::kMost / (cut.threads + 32 * K::kStat + 32);
  cut.blocks = static_cast<int>(std::min<int64_t>(bn_rows(d), 148 * cut.per_sm));
  return cut;
}

template <bool BACK>
static BnCut bn_cut(const dgxm_block_norm_desc* d) {
  const int size = bn_size(d);
  return size == 0 ? bn_cut_of<BACK, 0>(d) : size == 1 ? bn_cut_of<BACK, 1>(d) : bn_cut_of<BACK, 2>(d);
}

inline int bn_elt(int dtype) { return dtype == DGXM_DTYPE_F32 ? 4 : 2; }

// Place the streams of a row in a slot of the ring, and as many slots as the
// block's share of the shared memory holds.  `slack`: 16 bytes each for rows
// off 16 bytes.  `stat`: warps that take statistics; `vectors`: column vectors that the statistics want a copy of.
inline void bn_layout(const dgxm_block_norm_desc* d, const BnCut& cut, BlockNormParams* p, int stat, int vectors, bool slack) {
  const int ch = d->dtype == DGXM_DTYPE_F32 ? 4 : 8;
  const int padded = (d->width + ch - 1) / ch * ch;
  int room = (224 / cut.per_sm - 4) * 1024;  // beside the static part
  p->stage_bytes = slack ? cut.threads / 32 * kBnStage : 0;
  room -= p->stage_bytes;
  int at = 0;
  for (int s = 0; s < p->n_in; ++s) {
    p->in_off[s] = at;
    if (p->in[s] == nullptr) continue;
    p->in_pitch[s] = padded * p->in_elt[s] + (slack ? 16 : 0);
    at += p->in_pitch[s];
  }
  p->slot_bytes = at;
  // copies only where they leave three slots (their readers can do without)
  p->param_bytes = 3 * at + vectors * padded * 4 <= room ? vectors * padded * 4 : 0;
  p->slots = std::max(1, std::min(kBnMaxSlots, (room - p->param_bytes) / at));
  if (p->slots > stat) p->slots -= p->slots % stat;
}

// Every row of every stream and output on 16 bytes.
inline bool bn_vec(const dgxm_block_norm_desc* d, const BlockNormParams& p) {
  uint64_t bits = 0;
  for (int s = 0; s < p.n_in; ++s)
    if (p.in[s] != nullptr) bits |= reinterpret_cast<uintptr_t>(p.in[s]) | p.in_sb[s] | p.in_sr[s];
  bits |= reinterpret_cast<uintptr_t>(p.out) | p.out_sb | p.out_sr;
  if (p.x_out != nullptr) bits |= reinterpret_cast<uintptr_t>(p.x_out) | p.x_out_sb | p.x_out_sr;
  for (char* q : {p.g_gate, p.g_scale, p.g_shift}) bits |= reinterpret_cast<uintptr_t>(q);
  bits |= reinterpret_cast<uintptr_t>(p.partial);
  return bits % 16 == 0 && d->width % (d->dtype == DGXM_DTYPE_F32 ? 4 : 8) == 0;
}

template <bool BACK, typename T, int SIZE, bool VEC, bool FULL>
static int bn_launch_as(const dgxm_block_norm_desc* d, BlockNormParams& p, cudaStream_t st) {
  using K = BnKind<BACK, SIZE>;
  static std::atomic<uint64_t> done{0};
  void (*kernel)(BlockNormParams);
  if constexpr (BACK) kernel = block_norm_backward_kernel<T, kBnEach, VEC, FULL, K::kThreads, K::kStat, K::kPerSm>;
  else kernel = block_norm_kernel<T, kBnEach, VEC, FULL, K::kThreads, K::kStat, K::kPerSm>;
  const BnCut cut = bn_cut<BACK>(d);
  p.rows_each = p.rows / cut.blocks;
  p.rows_more = static_cast<int>(p.rows % cut.blocks);
  const bool forward_copy = p.gate != nullptr || p.branch_w != nullptr;
  p.factor = BACK && (p.scale != nullptr || p.norm_w != nullptr);
  bn_layout(d, cut, &p, K::kStat, BACK ? (p.branch_norm ? 2 : p.factor) : forward_copy, !VEC);
  DGXM_CUDA_TRY(set_smem_limit_once(kernel, 220 * 1024, done));
  DGXM_CUDA_TRY(launch_overlapped(kernel, cut.blocks, cut.threads + 32 * K::kStat + 32,
                                  p.param_bytes + p.slots * p.slot_bytes + p.stage_bytes, st, p));
  return DGXM_OK;
}

template <bool BACK, typename T, int SIZE>
static int bn_launch_size(const dgxm_block_norm_desc* d, BlockNormParams& p, cudaStream_t st) {
  const bool full = p.branch_norm || d->gate_form == DGXM_MOD_TOKEN || d->mod_form == DGXM_MOD_TOKEN;
  if (bn_vec(d, p))
    return full ? bn_launch_as<BACK, T, SIZE, true, true>(d, p, st) : bn_launch_as<BACK, T, SIZE, true, false>(d, p, st);
  return bn_launch_as<BACK, T, SIZE, false, true>(d, p, st);
}

// Compiled a type at a time, in units of their own.
template <bool BACK, typename T>
int bn_launch(const dgxm_block_norm_desc* d, BlockNormParams& p, cudaStream_t st) {
  const int size = bn_size(d);
  return size == 0   ? bn_launch_size<BACK, T, 0>(d, p, st)
         : size == 1 ? bn_launch_size<BACK, T, 1>(d, p, st)
                     : bn_launch_size<BACK, T, 2>(d, p, st);
}

}  // namespace dgxm
