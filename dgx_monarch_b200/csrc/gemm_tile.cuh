// What the 4-bit product and the 16-bit Linear share: the block's shape, the
// elected instructions of the loading and MMA warps, the order of tiles, and
// the way finished rows leave through staging rows of 128 bytes.
#pragma once

#include <type_traits>

#include "common.h"
#include "ptx.cuh"

namespace dgxm {

constexpr int kGemmThreads = 10 * 32;
constexpr int kGemmSmemMax = 227 * 1024;
constexpr int kGemmCtrlBytes = 512;
constexpr int kGemmStageRows = 32 * 128;  // a warp's staging: 32 rows of 128 bytes of output

// The MMA warp runs its loop as one, every lane with the same values, and each
// instruction is predicated by an elect.sync of its own: its operands stay in
// uniform registers.  A branch on the lane around them, or a predicate made
// from the lane number, has each operand moved there before each instruction
// (9450 x 13824 x 5120 nvfp4: 495 and 357 us, against 275).
#define DGXM_ELECT "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\t"

// Arrive on `bar` (PAIR: in both CTAs) when what the warp issued has completed.
template <bool PAIR>
__device__ __forceinline__ void fp4_commit(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(DGXM_ELECT
                 "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], "
                 "%1;\n\t}\n" ::"r"(bar), "h"(static_cast<uint16_t>(0x3))
                 : "memory");
  else
    asm volatile(DGXM_ELECT "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar)
                 : "memory");
}

// Load a tile and report its bytes on `bar`: this CTA's barrier, or (PAIR)
// the shared::cluster address of the even CTA's.
template <bool PAIR>
__device__ __forceinline__ void fp4_tma(uint32_t dst, const void* map, uint32_t bar, int c0, int c1, int c2) {
  if constexpr (PAIR) tma_load_4d_pair(dst, map, bar, c0, c1, c2, 0);
  else tma_load_4d(dst, map, bar, c0, c1, c2, 0);
}

// 16 bytes into the shared memory of a CTA of the cluster.
__device__ __forceinline__ void st_shared_cluster(uint32_t addr, const uint32_t* v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}

// 16-byte piece i of a lane's row in words: four fp32, or eight of a 16-bit type.
template <int ELT, typename P>
__device__ __forceinline__ uint4 fp4_piece(const P& p, const float* f) {
  if constexpr (ELT == 4)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else if (p.out_dtype == DGXM_DTYPE_BF16)
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  else
    return make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7]));
}

// 16 bytes of the 32 in a and b from byte n on, n even and below 16.
__device__ __forceinline__ uint4 fp4_bytes_from(uint4 a, uint4 b, uint32_t n) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = (n & 8u) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = (n & 4u) ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (n & 3u));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Whether a chunk of kCols columns goes out as one bulk store.
template <int kCols, int ELT, typename P>
__device__ __forceinline__ bool fp4_by_bulk(const P& p, int q0) {
  // a row that ends inside 16 bytes would have the rest of them written too
  return kCols == 128 / ELT && p.vec && (q0 + kCols <= p.q_rows || p.q_rows % (16 / ELT) == 0);
}

// Store a warp's 32 rows x kCols columns from staging rows of 128 bytes,
// 16-byte piece i of row r at piece i ^ (r & 7): the 128-byte swizzle, so that
// a whole chunk goes out as one bulk store (rows on 16 bytes), which leaves
// the warp to its arithmetic (9450 x 5120 x 256: 47 us with stores of the
// lanes, 23 us), or, otherwise, neighbouring lanes store neighbouring words or
// elements.  ELT: bytes of an output element.
template <int kCols, int ELT, typename P>
__device__ __forceinline__ void fp4_flush_rows(const P& p, uint8_t* stage, int pr0, int q0, int lane) {
  constexpr int kEach = 16 / ELT;  // elements of a piece
  constexpr int kPieces = kCols / kEach;
  using Elt = typename std::conditional<ELT == 4, uint32_t, uint16_t>::type;
  const bool bulk = fp4_by_bulk<kCols, ELT>(p, q0);
  if (bulk) {
    tma_store_fence();
    __syncwarp();
    if (lane == 0) {
      if (pr0 < p.p_rows) tma_store_4d(&p.tmap_out, smem_u32(stage), q0, 0, pr0, 0);
      tma_store_commit();
    }
    return;
  }
  __syncwarp();
  if (p.vec && q0 + kCols <= p.q_rows) {
    char* out = static_cast<char*>(p.out);
    const int i = lane % kPieces;
#pragma unroll
    for (int r = lane / kPieces; r < 32; r += 32 / kPieces)
      if (pr0 + r < p.p_rows)
        *reinterpret_cast<uint4*>(out + ((pr0 + r) * p.ld_out + q0 + i * kEach) * ELT) =
            *reinterpret_cast<const uint4*>(stage + r * 128 + ((i ^ (r & 7)) << 4));
  } else if (kPieces >= 4) {
    // Rows off 16 bytes, or ending here: whole aligned words, each from two
    // neighbouring pieces, and by elements the bytes before the first word
    // and behind the last (9450 x 5121 x 256: 102 us by elements alone, 55;
    // 100000 x 100 x 512, half a chunk at the end: 31, 23).
    auto store = [&](auto whole, int bytes) {
      constexpr bool kWhole = decltype(whole)::value;
      const int i = lane % kPieces;
#pragma unroll 4
      for (int r = lane / kPieces; r < min(32, p.p_rows - pr0); r += 32 / kPieces) {
        auto piece = [&](int k) { return stage + r * 128 + ((k ^ (r & 7)) << 4); };
        char* row = static_cast<char*>(p.out) + ((pr0 + r) * p.ld_out + q0) * ELT;
        const int head = static_cast<int>(-reinterpret_cast<uintptr_t>(row) & 15u);
        const int words = kWhole ? kPieces - (head > 0) : max(bytes - head, 0) / 16;
        if (i < words)
          *reinterpret_cast<uint4*>(row + head + 16 * i) =
              fp4_bytes_from(*reinterpret_cast<const uint4*>(piece(i)),
                             *reinterpret_cast<const uint4*>(piece(min(i + 1, kPieces - 1))), head);
        auto element = [&](int at) {
          *reinterpret_cast<Elt*>(row + at) = *reinterpret_cast<const Elt*>(piece(at / 16) + at % 16);
        };
#pragma unroll
        for (int e = i; e < kEach; e += kPieces) {
          if (kWhole) {  // the bytes before and behind are none, or as many as a piece has
            if (head > 0) element(e * ELT < head ? e * ELT : 16 * (kPieces - 1) + e * ELT);
          } else {
            if (e * ELT < min(head, bytes)) element(e * ELT);
            if (head + 16 * words + e * ELT < bytes) element(head + 16 * words + e * ELT);
          }
        }
      }
    };
    if (q0 + kCols <= p.q_rows) store(std::true_type{}, kCols * ELT);
    else store(std::false_type{}, (p.q_rows - q0) * ELT);
  } else {
    const int cols = min(kCols, p.q_rows - q0), rows = min(32, p.p_rows - pr0);
    Elt* to = reinterpret_cast<Elt*>(p.out) + pr0 * p.ld_out + q0;
#pragma unroll
    for (int e = lane; e < kCols; e += 32) {
      if (e >= cols) break;
#pragma unroll 8
      for (int r = 0; r < 32; ++r)
        if (r < rows)
          to[r * p.ld_out + e] =
              *reinterpret_cast<const Elt*>(stage + r * 128 + (((e / kEach) ^ (r & 7)) << 4) + (e % kEach) * ELT);
    }
  }
  __syncwarp();
}

// Tiles run in groups of eight P tiles, Q outermost within a group, so that
// the CTAs resident at one time share a few panels of both operands.
template <typename P>
__device__ __forceinline__ void fp4_tile_coords(const P& p, int tile, int& pt, int& qt) {
  const int per_group = 8 * p.q_tiles;
  const int g = tile / per_group, r = tile - g * per_group;
  const int rows = min(8, p.p_tiles - g * 8);
  pt = g * 8 + r % rows;
  qt = r / rows;
}

}  // namespace dgxm
