// KV scatter into an 8-bit paged cache: e4m3 values with one float32 scale, a power of two, for each block of G
// consecutive slots and kv head (k and v apart).
//
// For a scale block b that this call writes, and a kv head:
//     amax   = largest |x| over the rows written to b          (finite values only)
//     e      = least whole number with amax <= 448 * 2^e, kept in [-40, 40]   (448: the largest e4m3 value)
//     scale' = 2^e if a row is written to b's first slot (the block starts afresh), else max(scale, 2^e)
//     rows the block already held: rn_e4m3(c * scale / scale') when the scale grew, else as they are
//     rows written:                rn_e4m3(clamp(x / scale', -448, 448)); NaN and infinities become NaN
// Powers of two make x / scale' and c * scale / scale' exact, so a value is rounded once when it is written and again
// only where the larger scale pushes it below e4m3's normal range; they cost at most one binade of that range.
//
// What it has to move: 2 bytes read and 1 byte written per value and nothing else worth counting (8192 tokens of 8 kv
// heads: 50 MB, 7.7 us at the measured copy rate).  No value may be rounded before the largest one of its block is
// known, and nothing tells the host which rows share a block, so the grouping happens on the chip: each CTA takes a run
// of the call's tokens, reads the whole slot list (4 bytes per token against 4 KB of rows, out of L2) through a bitmap
// of its own tokens' blocks, and keeps the blocks whose first token in the call is its own, with a table of the last
// token written to each of their slots.  One warp then owns one (block, head, k or v): no atomics on global memory, no
// second launch, no workspace, and a result that depends on nothing but the arguments (a slot named twice keeps its
// last token).  The rows of a block of 16 stay in registers between the two passes over them.
#include <algorithm>
#include <climits>
#include <type_traits>
#include <cuda_fp8.h>

#include "../../include/nvattn.h"
#include "nva_ptx.cuh"
#include "nva_kernels.h"

namespace nva {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxChunk = 64;          // tokens of the call per CTA
constexpr int kBitmapWords = 128;      // 4096 bits over block ids
constexpr int kHeld = 8;               // row pairs of a block in registers at a time
constexpr int kExpMin = -40, kExpMax = 40;

struct StoreFp8Params {
  const __nv_bfloat16* src[2];
  int64_t src_stride[2];
  uint8_t* cache[2];
  float* scale[2];
  const int32_t* slots;
  int64_t num_slots;
  int32_t num_tokens;
  int32_t kv_heads;
  int32_t chunk;
  int32_t lg_block;    // log2 of the slots per scale block
  int32_t page_blocks;  // scale blocks per page
};

// Largest |x| of eight bf16 values with `m`'s, as their 15 bits (ordered like the magnitudes), two to a word.
__device__ __forceinline__ uint32_t amax8(uint32_t m, uint4 v) {
  m = __vmaxu2(m, __vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu));
  return __vmaxu2(m, __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
}
// The same over finite values only.
__device__ __forceinline__ uint32_t amax8_finite(uint32_t m, uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = w[i] & 0x7FFF7FFFu;
    m = __vmaxu2(m, a & __vcmpltu2(a, 0x7F807F80u));
  }
  return m;
}

// Scale for a largest magnitude given as bf16 bits: amax = 1.m * 2^(E - 127) <= 448 * 2^e = 1.75 * 2^(8 + e).
__device__ __forceinline__ float scale_of(uint32_t bits) {
  const int E = static_cast<int>(bits >> 7);
  int e = E - 127 - 8 + ((bits & 0x7Fu) > 0x60u ? 1 : 0);   // 1.m > 1.75
  e = bits == 0 ? kExpMin : min(max(e, kExpMin), kExpMax);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Two bf16 values times inv, rounded to e4m3 (nearest even, saturating; NaN and, with kAny, infinities to NaN).
template <bool kAny>
__device__ __forceinline__ uint32_t quant2(uint32_t w, float inv) {
  float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  if constexpr (kAny) {   // x * 0 is NaN for NaN and infinities, 0 otherwise
    f.x = fmaf(f.x, inv, f.x * 0.f);
    f.y = fmaf(f.y, inv, f.y * 0.f);
  } else {
    f.x *= inv;
    f.y *= inv;
  }
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3));
}
template <bool kAny>
__device__ __forceinline__ uint2 quant8(uint4 v, float inv) {
  return make_uint2(quant2<kAny>(v.x, inv) | (quant2<kAny>(v.y, inv) << 16),
                    quant2<kAny>(v.z, inv) | (quant2<kAny>(v.w, inv) << 16));
}

// Four e4m3 values times f (a power of two at most 1), rounded to e4m3.
__device__ __forceinline__ uint32_t requant4(uint32_t c, float f) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c >> (16 * i)), __NV_E4M3);
    float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
    x.x *= f;
    x.y *= f;
    out |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3)) << (16 * i);
  }
  return out;
}

__device__ __forceinline__ uint32_t hash_block(int32_t b) { return (static_cast<uint32_t>(b) * 0x9E3779B1u) >> 20; }

__global__ void __launch_bounds__(kThreads, 2) store_fp8_kernel(const StoreFp8Params p) {
  extern __shared__ int32_t winner[];          // [entries][G]: 1 + the last token of the call written to the slot
  __shared__ int32_t blk[kMaxChunk];           // distinct blocks of this CTA's tokens
  __shared__ int32_t own_blk[kMaxChunk];       // block of each of its tokens (-1: none)
  __shared__ int32_t earlier[kMaxChunk];       // an earlier token of the call writes the block: another CTA owns it
  __shared__ uint32_t bitmap[kBitmapWords];
  __shared__ int32_t entries_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = 1 << p.lg_block;
  const int i0 = blockIdx.x * p.chunk;
  const int i1 = min(p.num_tokens, i0 + p.chunk);
  const int cnt = i1 - i0;

  if (tid < kBitmapWords) bitmap[tid] = 0u;
  if (tid < cnt) {
    const int64_t slot = __ldg(p.slots + i0 + tid);
    if (slot >= p.num_slots || slot < -1) atomicOr(&g_error_word, kErrSlotRange);
    own_blk[tid] = slot >= 0 && slot < p.num_slots ? static_cast<int32_t>(slot >> p.lg_block) : -1;
    earlier[tid] = 0;
  }
  for (int i = tid; i < cnt * G; i += kThreads) winner[i] = 0;
  __syncthreads();
  // distinct blocks, in the order of their first token (two warps' worth of tokens at most)
  if (warp == 0) {
    int entries = 0;
    for (int base = 0; base < cnt; base += 32) {
      const int t = base + lane;
      const int32_t b = t < cnt ? own_blk[t] : -1;
      bool first = b >= 0;
      for (int u = 0; u < min(t, cnt); ++u) first = first && own_blk[u] != b;
      const uint32_t vote = __ballot_sync(0xffffffffu, first);
      if (first) {
        blk[entries + __popc(vote & ((1u << lane) - 1u))] = b;
        const uint32_t h = hash_block(b);
        atomicOr(&bitmap[h >> 5], 1u << (h & 31));
      }
      entries += __popc(vote);
    }
    if (lane == 0) entries_s = entries;
  }
  __syncthreads();
  const int entries = entries_s;
  if (entries == 0) return;

  // the whole call's slots: who else writes these blocks
  int32_t lo_slot = INT_MAX, hi_slot = -1;
  for (int e = lane; e < entries; e += 32) {
    lo_slot = min(lo_slot, blk[e]);
    hi_slot = max(hi_slot, blk[e]);
  }
  lo_slot = __reduce_min_sync(0xffffffffu, lo_slot) << p.lg_block;
  hi_slot = (__reduce_max_sync(0xffffffffu, hi_slot) << p.lg_block) + (G - 1);
  auto visit = [&](int i, int32_t slot) {
    if (slot < lo_slot || slot > hi_slot) return;   // (most of a call: other sequences' pages)
    const int32_t b = slot >> p.lg_block;
    const uint32_t h = hash_block(b);
    if (!((bitmap[h >> 5] >> (h & 31)) & 1u)) return;
    for (int e = 0; e < entries; ++e)
      if (blk[e] == b) {
        if (i < i0) earlier[e] = 1;
        atomicMax(&winner[e * G + (slot & (G - 1))], i + 1);
        return;
      }
  };
  if ((reinterpret_cast<uintptr_t>(p.slots) & 15u) == 0) {
    const int nv = p.num_tokens >> 2;
    constexpr int kAhead = 4;
    for (int v0 = tid; v0 < nv; v0 += kAhead * kThreads) {
      int4 s[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        s[i] = v0 + i * kThreads < nv ? __ldg(reinterpret_cast<const int4*>(p.slots) + v0 + i * kThreads)
                                      : make_int4(-1, -1, -1, -1);
#pragma unroll 1
      for (int i = 0; i < kAhead; ++i) {
        const int v = v0 + i * kThreads;
        const int4 t = i == 0 ? s[0] : i == 1 ? s[1] : i == 2 ? s[2] : s[3];
        visit(4 * v, t.x);
        visit(4 * v + 1, t.y);
        visit(4 * v + 2, t.z);
        visit(4 * v + 3, t.w);
      }
    }
    for (int i = 4 * nv + tid; i < p.num_tokens; i += kThreads) visit(i, __ldg(p.slots + i));
  } else {
    for (int i = tid; i < p.num_tokens; i += kThreads) visit(i, __ldg(p.slots + i));
  }
  __syncthreads();

  // one warp per (block, head, k or v), neighbouring warps on neighbouring heads: half a warp reads a row (16 bytes a
  // lane), so that the 16 rows of a block are eight loads in flight
  const int tasks = entries * p.kv_heads * 2;
  const int half = lane >> 4, col = (lane & 15) * 8;
  const int64_t row = static_cast<int64_t>(p.kv_heads) * kHeadDim;
  for (int task = warp; task < tasks; task += kWarps) {
    const int head = task % p.kv_heads;
    const int kv = (task / p.kv_heads) & 1;
    const int e = task / (2 * p.kv_heads);
    if (earlier[e]) continue;
    const int32_t b = blk[e];
    const int32_t* win = winner + e * G;
    const int page = b / p.page_blocks;
    float* scale = p.scale[kv] + (static_cast<int64_t>(page) * p.kv_heads + head) * p.page_blocks +
                   (b - page * p.page_blocks);
    const float old = *scale;
    const __nv_bfloat16* src = p.src[kv] + head * kHeadDim + col;
    const int64_t stride = p.src_stride[kv];
    uint8_t* dst = p.cache[kv] + ((static_cast<int64_t>(b) << p.lg_block) * p.kv_heads + head) * kHeadDim + col;
    const bool fresh = win[0] != 0;
    uint4 held[kHeld];
    auto fetch = [&](int base) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int s = base + 2 * i + half;
        const int w = s < G ? win[s] : 0;
        held[i] = make_uint4(0u, 0u, 0u, 0u);
        if (w != 0) held[i] = __ldg(reinterpret_cast<const uint4*>(src + (w - 1) * stride));
      }
    };
    // pass 1: the largest magnitude
    auto largest = [&](auto finite) {
      uint32_t m = 0;
      for (int base = 0; base < G; base += 2 * kHeld) {
        if (G > 2 * kHeld || !decltype(finite)::value) fetch(base);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) m = decltype(finite)::value ? amax8_finite(m, held[i]) : amax8(m, held[i]);
      }
      return __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16));
    };
    uint32_t m = largest(std::false_type{});
    const bool any = m >= 0x7F80u;   // NaN or infinities among them: they have no say in the scale
    if (any) m = largest(std::true_type{});
    const float now = fresh ? scale_of(m) : fmaxf(old, scale_of(m));
    const float inv = 1.0f / now;
    // pass 2: write the rows (blocks of more than 16 slots read theirs again, out of L1 / L2)
    for (int base = 0; base < G; base += 2 * kHeld) {
      if (G > 2 * kHeld) fetch(base);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int s = base + 2 * i + half;
        if (s < G && win[s] != 0)
          *reinterpret_cast<uint2*>(dst + s * row) = any ? quant8<true>(held[i], inv) : quant8<false>(held[i], inv);
      }
    }
    if (!fresh && now > old) {
      // the scale grew: what the block holds besides is rounded to it
      const float factor = old * inv;
#pragma unroll 4
      for (int s = half; s < G; s += 2)
        if (win[s] == 0) {
          uint2* at = reinterpret_cast<uint2*>(dst + s * row);
          const uint2 c = *at;
          *at = make_uint2(requant4(c.x, factor), requant4(c.y, factor));
        }
    }
    if (lane == 0) *scale = now;
  }
}

}  // namespace

}  // namespace nva

extern "C" NVA_API int nva_store_kvcache_fp8(const void* key, int64_t key_row_stride, const void* value,
                                             int64_t value_row_stride, void* k_cache, void* v_cache, float* k_scale,
                                             float* v_scale, int32_t num_blocks, int32_t block_size,
                                             int32_t scale_block, const int32_t* slot_mapping, int32_t num_tokens,
                                             int32_t num_kv_heads, int32_t head_dim, void* stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks < 0 || block_size <= 0 || scale_block <= 0)
    return NVA_ERR_INVALID_ARGUMENT;
  if (head_dim != nva::kHeadDim) return NVA_ERR_UNSUPPORTED;
  if ((scale_block & (scale_block - 1)) != 0 || scale_block < NVA_MIN_SCALE_BLOCK ||
      scale_block > NVA_MAX_SCALE_BLOCK || block_size % scale_block != 0)
    return NVA_ERR_UNSUPPORTED;
  const int64_t num_slots = static_cast<int64_t>(num_blocks) * block_size;
  if (num_slots >= (int64_t(1) << 31)) return NVA_ERR_UNSUPPORTED;
  if (num_tokens == 0) return NVA_OK;
  if (key == nullptr || value == nullptr || k_cache == nullptr || v_cache == nullptr || k_scale == nullptr ||
      v_scale == nullptr || slot_mapping == nullptr)
    return NVA_ERR_INVALID_ARGUMENT;
  const int64_t row_elems = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (key_row_stride < row_elems || value_row_stride < row_elems) return NVA_ERR_INVALID_ARGUMENT;
  // 16-byte vectors of the rows, 8-byte vectors of the cache
  auto misaligned = [](const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) != 0; };
  if (misaligned(key, 16) || misaligned(value, 16) || key_row_stride % 8 != 0 || value_row_stride % 8 != 0 ||
      misaligned(k_cache, 8) || misaligned(v_cache, 8) || misaligned(k_scale, 4) || misaligned(v_scale, 4) ||
      misaligned(slot_mapping, 4))
    return NVA_ERR_ALIGNMENT;
  const int sms = nva::sm_count();
  if (sms == 0) return nva::cuda_fail(cudaGetLastError());
  nva::StoreFp8Params p{};
  p.src[0] = static_cast<const __nv_bfloat16*>(key);
  p.src[1] = static_cast<const __nv_bfloat16*>(value);
  p.src_stride[0] = key_row_stride;
  p.src_stride[1] = value_row_stride;
  p.cache[0] = static_cast<uint8_t*>(k_cache);
  p.cache[1] = static_cast<uint8_t*>(v_cache);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.slots = slot_mapping;
  p.num_slots = num_slots;
  p.num_tokens = num_tokens;
  p.kv_heads = num_kv_heads;
  p.lg_block = __builtin_ctz(static_cast<unsigned>(scale_block));
  p.page_blocks = block_size / scale_block;
  // tokens per CTA: about two CTAs per SM over the call (8192 tokens: 28, 21 us; one or three per SM 27 and 29 us), and
  // a winner table of at most 32 KB
  const int64_t want = (static_cast<int64_t>(num_tokens) + 2 * sms - 1) / (2 * sms);
  const int most = std::min(nva::kMaxChunk, 32768 / 4 / scale_block);
  p.chunk = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(want, most)));
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(num_tokens) + p.chunk - 1) / p.chunk);
  const size_t smem = static_cast<size_t>(p.chunk) * scale_block * sizeof(int32_t);
  nva::store_fp8_kernel<<<grid, nva::kThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? NVA_OK : nva::cuda_fail(e);
}
