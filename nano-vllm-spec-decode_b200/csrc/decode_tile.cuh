// Row-tile helpers of the paged decode kernels, which put a KV tile's 128 tokens on the TMEM lanes and a kv head's query
// rows on the UMMA N columns and reduce over tokens across lanes.  Both (paged_decode.cu, paged_decode_fp8.cu) use the
// constants, warp_columns and mma_width; the choice of a row width and merge_pieces are the bf16 kernel's alone.
#pragma once
#include <cstdint>
#include <type_traits>

#include "nva_kernels.h"
#include "nva_ptx.cuh"

namespace nva {

namespace {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr uint32_t kFull = 0xffffffffu;
constexpr int kMergePieces = 16;   // pieces of a cut segment merged through the shared weight table
constexpr int kTicketStride = 4;   // merge tickets per CTA: one per softmax warpgroup (at most 3)

// Transposed butterfly over the 32 lanes of a warp for NR (power of two <= 32) columns held by every lane: each
// stage sends half of the remaining columns to the partner lane and keeps the other half, so the whole reduction
// costs NR - 1 + (5 - log2 NR) shuffles with the shuffles of a stage independent of each other.  On return lane l
// holds the reduction of column l / (32 / NR) in v[0]; lanes with l % (32 / NR) == 0 store it to dst[column].
template <int N, int O, bool kMax>
__device__ __forceinline__ void column_stage(float* v, int lane) {
  if constexpr (O > 0) {
    if constexpr (N > 1) {
      constexpr int H = N / 2;
      const bool upper = (lane & O) != 0;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float send = upper ? v[i] : v[i + H];
        const float keep = upper ? v[i + H] : v[i];
        const float recv = __shfl_xor_sync(kFull, send, O);
        v[i] = kMax ? fmaxf(keep, recv) : keep + recv;
      }
      column_stage<H, O / 2, kMax>(v, lane);
    } else {
      const float recv = __shfl_xor_sync(kFull, v[0], O);
      v[0] = kMax ? fmaxf(v[0], recv) : v[0] + recv;
      column_stage<1, O / 2, kMax>(v, lane);
    }
  }
}

template <int NR, bool kMax>
__device__ __forceinline__ void column_reduce(float* v, float* dst, int lane) {
  column_stage<NR, 16, kMax>(v, lane);
  constexpr int kRep = 32 / NR;
  if ((lane & (kRep - 1)) == 0) dst[lane / kRep] = v[0];
}

// Column reduction of NR (8, 16, 24, 32 or 48) values per thread within one warp into dst[0..NR).
template <int NR, bool kMax>
__device__ __forceinline__ void warp_columns(const float* x, float* dst, int lane) {
  float v[32];
  if constexpr (NR <= 16) {
#pragma unroll
    for (int i = 0; i < NR; ++i) v[i] = x[i];
    column_reduce<NR, kMax>(v, dst, lane);
  } else if constexpr (NR == 24) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = x[i];
    column_reduce<16, kMax>(v, dst, lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[16 + i];
    column_reduce<8, kMax>(v, dst + 16, lane);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = x[i];
    column_reduce<32, kMax>(v, dst, lane);
    if constexpr (NR == 48) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = x[32 + i];
      column_reduce<16, kMax>(v, dst + 32, lane);
    }
  }
}

// Rows a segment carries through the softmax: its real rows rounded up to 8, 16, 32 or 48 (never above NP).
__device__ __forceinline__ int rows_width(int R) { return R <= 8 ? 8 : R <= 16 ? 16 : R <= 32 ? 32 : 48; }
// UMMA N for a segment (M = 128 needs N to be a multiple of 16).
__device__ __forceinline__ int mma_width(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : 48; }

// Calls f(integral_constant<NR>) for the row width nr, limited to the kernel's NP.
template <int NP, class F>
__device__ __forceinline__ void with_rows(int nr, F&& f) {
  if (nr <= 8) {
    f(std::integral_constant<int, 8>{});
  } else if (nr <= 16 || NP == 16) {
    f(std::integral_constant<int, 16>{});
  } else if (nr <= 32 || NP == 32) {
    f(std::integral_constant<int, (NP >= 32 ? 32 : 16)>{});
  } else {
    f(std::integral_constant<int, NP>{});
  }
}

// Rows each of `wg_count` softmax warpgroups carries for an NR-wide tile: all NR with one group; otherwise NR split
// into equal shares rounded up to whole 8-row P^T vectors (8, 16 or 24 rows); groups past NR hold padding only.
__host__ __device__ constexpr int group_rows_rt(int wg_count, int nr) {
  return wg_count == 1 ? nr : nr <= 8 ? 8 : ((nr + wg_count - 1) / wg_count + 7) / 8 * 8;
}

// HR consecutive TMEM columns (8, 16 or 24) of this warp's lanes, one wait.
template <int HR>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, float* v) {
  if constexpr (HR == 8) {
    tmem_ld8(taddr, v);
  } else if constexpr (HR == 16) {
    tmem_ld16(taddr, v);
  } else {
    static_assert(HR == 24, "row group width");
    tmem_ld24(taddr, v);
  }
}

// Merge the pieces of a cut segment (CTAs c0..c1) into its output rows [r0, r1), from one 128-thread group (all of
// its threads call this; named barrier bar_id).  Each piece is weighted by 2^(lse - max lse) / sum.  The partials were
// written by other CTAs, so they are read past L1 (ld.global.cg).  Two pieces: (row, 4 dims) items six at a time
// with all their loads in one round.  Up to kMergePieces pieces: one thread per row puts the row's weights in the
// group's table `wsm`, then items four at a time (two memory rounds).  More pieces: a plain loop.
template <int NP, class Params>
__device__ __forceinline__ void merge_pieces(const Params& p, int c0, int c1, int r0, int r1, int G,
                                             int64_t out_base, int ct, float* wsm, uint32_t bar_id) {
  const int pieces = c1 - c0 + 1;
  auto slot_of = [&](int pi) { return pi == 0 ? 2 * c0 + 1 : 2 * (c0 + pi); };
  auto store = [&](int idx, float4 a, float inv) {
    const int r = r0 + (idx >> 5), l4 = idx & 31;
    const int i = r / G, h = r - i * G;
    uint2 packed;
    packed.x = pack_bf16x2(a.x * inv, a.y * inv);
    packed.y = pack_bf16x2(a.z * inv, a.w * inv);
    *reinterpret_cast<uint2*>(p.out + out_base + (int64_t)i * p.out_row_stride + h * kHeadDim + l4 * 4) = packed;
  };
  if (pieces == 2) {
    // a segment cut once (the usual case): every load of a round of six items issued together
    const int s0 = 2 * c0 + 1, s1 = 2 * c0 + 2;
    const int nitems = (r1 - r0) * 32;
    constexpr int kRound = 2;
    for (int base = ct; base < nitems; base += kRound * 128) {
      float4 a0[kRound], a1[kRound];
      float e0[kRound], e1[kRound];
#pragma unroll
      for (int u = 0; u < kRound; ++u) {
        const int idx = base + u * 128;
        if (idx < nitems) {
          const int r = r0 + (idx >> 5), l4 = idx & 31;
          e0[u] = __ldcg(p.part_lse + s0 * NP + r);
          e1[u] = __ldcg(p.part_lse + s1 * NP + r);
          a0[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + ((int64_t)s0 * NP + r) * kHeadDim) + l4);
          a1[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + ((int64_t)s1 * NP + r) * kHeadDim) + l4);
        }
      }
#pragma unroll
      for (int u = 0; u < kRound; ++u) {
        const int idx = base + u * 128;
        if (idx < nitems) {
          const float mx = fmaxf(e0[u], e1[u]);
          const float w0 = (mx == kNegInf || e0[u] == kNegInf) ? 0.f : fast_exp2(e0[u] - mx);
          const float w1 = (mx == kNegInf || e1[u] == kNegInf) ? 0.f : fast_exp2(e1[u] - mx);
          const float den = w0 + w1;
          const float4 acc = make_float4(w0 * a0[u].x + w1 * a1[u].x, w0 * a0[u].y + w1 * a1[u].y,
                                         w0 * a0[u].z + w1 * a1[u].z, w0 * a0[u].w + w1 * a1[u].w);
          store(idx, acc, den > 0.f ? 1.f / den : 0.f);
        }
      }
    }
    return;
  }
  if (pieces <= kMergePieces) {
    for (int r = r0 + ct; r < r1; r += 128) {
      float* w = wsm + (r - r0) * kMergePieces;
      float mx = kNegInf;
      for (int pi = 0; pi < pieces; ++pi) {
        const float v = __ldcg(p.part_lse + slot_of(pi) * NP + r);
        w[pi] = v;
        mx = fmaxf(mx, v);
      }
      float den = 0.f;
      for (int pi = 0; pi < pieces; ++pi) {
        const float e = (mx == kNegInf || w[pi] == kNegInf) ? 0.f : fast_exp2(w[pi] - mx);
        w[pi] = e;
        den += e;
      }
      const float inv = den > 0.f ? 1.f / den : 0.f;
      for (int pi = 0; pi < pieces; ++pi) w[pi] *= inv;
    }
    named_bar_sync(bar_id, 128);
    const int nitems = (r1 - r0) * 32;
    for (int base = ct; base < nitems; base += 4 * 128) {
      float4 acc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int idx = base + u * 128;
        if (idx < nitems) {
          const int r = r0 + (idx >> 5), l4 = idx & 31;
          const float* w = wsm + (r - r0) * kMergePieces;
          for (int pi = 0; pi < pieces; ++pi) {
            const float4 v =
                __ldcg(reinterpret_cast<const float4*>(p.part_o + ((int64_t)slot_of(pi) * NP + r) * kHeadDim) + l4);
            const float wp = w[pi];
            acc[u].x += wp * v.x;
            acc[u].y += wp * v.y;
            acc[u].z += wp * v.z;
            acc[u].w += wp * v.w;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int idx = base + u * 128;
        if (idx < nitems) store(idx, acc[u], 1.f);
      }
    }
    return;
  }
  for (int idx = ct; idx < (r1 - r0) * 32; idx += 128) {
    const int r = r0 + (idx >> 5), l4 = idx & 31;
    float mx = kNegInf;
    for (int pi = 0; pi < pieces; ++pi) mx = fmaxf(mx, __ldcg(p.part_lse + slot_of(pi) * NP + r));
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
    if (mx != kNegInf) {
#pragma unroll 4
      for (int pi = 0; pi < pieces; ++pi) {
        const float lse = __ldcg(p.part_lse + slot_of(pi) * NP + r);
        const float4 v =
            __ldcg(reinterpret_cast<const float4*>(p.part_o + ((int64_t)slot_of(pi) * NP + r) * kHeadDim) + l4);
        const float w = lse == kNegInf ? 0.f : fast_exp2(lse - mx);
        acc.x += w * v.x;
        acc.y += w * v.y;
        acc.z += w * v.z;
        acc.w += w * v.w;
        den += w;
      }
    }
    store(idx, acc, den > 0.f ? 1.f / den : 0.f);
  }
}

}  // namespace

}  // namespace nva
