// Paged GQA attention over an 8-bit KV cache for sm_100a: decode, speculative verify and varlen (prefill chunks, mixed
// batches), the 8-bit counterpart of flash_attn_with_kvcache (nanovllm/layers/attention.py:75-77) and of the paged
// flash_attn_varlen_func (:67-70).
//
// The cache holds e4m3 values c with a float32 scale per (block of tokens, kv head): k = kc * ks, v = vc * vs.
//     x[r, t]  = (q[r] . kc[t]) * ks[t] * softmax_scale * log2(e)         score in log2 units
//     y[r, t]  = x[r, t] + log2 vs[t]                                     the scale of v moved into the exponent
//     w[r, t]  = 2^(y - m[r] + 8)         m: running row maximum of y
//     out[r]   = sum_t w[r, t] vc[t] / sum_t w[r, t] / vs[t]
// so neither k nor v is ever multiplied out: both products read the cache's own bytes on the 8-bit tensor pipe, and one
// pass over K and V serves every q head of the group and every query row.  The other operand of each product is split
// into two 8-bit parts that accumulate into the same TMEM columns, which keeps the 16-bit kernels' accuracy:
//   q  = (hi + lo) * 2^e, both e4m3, e from the row's largest value: four significant bits each, together all eight of a
//        bf16 value (exact for values down to 2^-10 of the row's largest, off by at most 2^-18 of that below);
//   w  = hi + lo, hi rounded to e5m2 (three bits, range to 2^-16), lo the rest in e4m3: off by at most 2^-7 of w
//        (0.12% rms, bf16's rounding is 0.16%) and never below 2^-17 where the row's largest is 2^8 to 2^11, so tokens
//        down to 2^-25 of the largest weight still count.  Sums of weights stay in float32, unrounded.
//
// Bound: HBM, one byte per cached value (decode of 64 sequences, contexts 512 to 4096: 303 MB, 46 us at the measured
// copy rate).  A 128-token tile then takes 0.74 us of an SM's share of the bandwidth, half of the bf16 cache's, which is
// less than one tile's chain S -> weights -> PV takes; so two CTAs share an SM and their chains overlap.
//
// Orientation, roles and the merge of split segments are those of paged_decode.cu: tokens on the TMEM lanes (UMMA M),
// query rows on N; warp 0 = K producer, 1 = TMEM + UMMA issuer, 2 = Q loader, 3 = V producer, 4.. = softmax groups.
// K tile: K-major, 128-byte swizzle, 128 dims = one swizzle row.  V tile: the same bytes read MN-major.  P^T: MN-major
// without swizzle, 16 rows of a token per 16 bytes.
//
// Work split: every CTA owns an equal share of cost positions (tiles + 3 per segment) in (sequence, piece, kv head,
// tile) order, where a piece is a run of at most max_n queries of a sequence: a prefill chunk is walked piece by piece,
// each over the keys its last query sees.  A CTA finds its start with one scan over the lengths and walks on from there,
// so there is no table of sequences on the chip and no bound on their number.
#include <algorithm>
#include <cuda_fp8.h>

#include "../../include/nvattn.h"
#include "decode_tile.cuh"
#include "nva_kernels.h"
#include "nva_ptx.cuh"

namespace nva {

namespace {

constexpr int kTile = 128 * 128;        // one K or V tile: 128 tokens x 128 bytes
constexpr int kConsumerBase = 128;
constexpr int kInfoRing = 8;            // tile descriptors; the producer is at most 6 tiles ahead of the softmax warps
constexpr int kQScaleRing = 8;          // row scales by segment; the Q loader is at most 4 segments ahead
constexpr int kSegCost = 3;             // a segment's start and end, in tiles
constexpr float kBase = 8.0f;           // the largest weight of a row is 2^kBase when its maximum is exact ...
constexpr float kSlack = 3.0f;          // ... and may pass it by this much (log2) before the maximum moves
constexpr float kWeightMax = 2048.0f;   // 2^(kBase + kSlack): lo <= 2^-3 w stays inside e4m3's range

template <int NP>
struct Cfg8 {
  static constexpr int kWG = NP >= 32 ? 2 : 1;        // softmax groups of 128 threads, each with a share of the rows
  static constexpr int kThreads = kConsumerBase + 128 * kWG;
  static constexpr int kRows = NP / kWG;
  // Rings that let two CTAs fit an SM (113 KB each): 3 + 2 tiles at 16 rows, 2 + 2 with the wider Q and P buffers
  static constexpr int kKStages = NP == 16 ? 3 : 2;
  static constexpr int kVStages = 2;
  static constexpr int kQBuf = NP == 48 ? 1 : 2;
  static constexpr int kPBuf = 2;
  static constexpr int kOperand = 2 * NP * 128;       // hi and lo of Q or P^T
  static constexpr int kTmemCols = NP == 16 ? 64 : NP == 32 ? 128 : 256;   // S, O double buffered: 4 NP, a power of two
  static constexpr int kK = 0;
  static constexpr int kV = kK + kKStages * kTile;
  static constexpr int kQ = kV + kVStages * kTile;
  static constexpr int kP = kQ + kQBuf * kOperand;
  static constexpr int kBarCount = 32;
  static constexpr int kBars = kP + kPBuf * kOperand;
  static constexpr int kInfo = kBars + kBarCount * 8;               // [kInfoRing][3] int4
  static constexpr int kQScale = kInfo + kInfoRing * 48;            // [kQScaleRing][NP]
  static constexpr int kRed = kQScale + kQScaleRing * NP * 4;       // [4][NP]
  static constexpr int kM = kRed + 4 * NP * 4;                      // [NP] running maxima
  static constexpr int kNegM = kM + NP * 4;                         // [NP] kBase - maximum
  static constexpr int kAlpha = kNegM + NP * 4;                     // [NP]
  static constexpr int kLred = kAlpha + NP * 4;                     // [4][NP]
  static constexpr int kRowOut = kLred + 4 * NP * 4;                // [NP] int64
  static constexpr int kRowInv = kRowOut + NP * 8;                  // [NP]
  static constexpr int kMergeW = kRowInv + NP * 4;                  // [NP][kMergePieces] (a group's rows at its own)
  static constexpr int kStart = (kMergeW + NP * kMergePieces * 4 + 15) / 16 * 16;   // Start
  static constexpr int kScan = kStart + 64;                         // [16] int64
  static constexpr int kTmem = kScan + 16 * 8;
  static constexpr int kAbort = kTmem + 4;
  static constexpr int kEnd = kAbort + 4;
  static constexpr int kBytes = kEnd + 1024;                        // + slack for 1024-byte alignment
};
static_assert(Cfg8<16>::kBytes <= 115712 && Cfg8<32>::kBytes <= 115712 && Cfg8<48>::kBytes <= 115712,
              "two CTAs per SM");

enum {
  B_KFULL = 0, B_KEMPTY = 3, B_VFULL = 6, B_VEMPTY = 8, B_SFULL = 10, B_SEMPTY = 12, B_PFULL = 14, B_OFULL = 16,
  B_QFULL = 18, B_QEMPTY = 20, B_INFO = 22, B_KSTART = 30
};

// The f8f6f4 instruction descriptor: float32 accumulator, A e4m3, B e4m3 or e5m2.
__host__ __device__ constexpr uint32_t idesc_f8(int N, bool b_e5m2, bool mn_major) {
  return (1u << 4) | (0u << 7) | (static_cast<uint32_t>(b_e5m2) << 10) | (static_cast<uint32_t>(mn_major) << 15) |
         (static_cast<uint32_t>(mn_major) << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void umma_f8_ss(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// Two floats to two packed 8-bit values, the first in the low byte (nearest even, saturating).
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t pack_e5m2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E5M2);
}
__device__ __forceinline__ float2 unpack_e4m3(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xFFFFu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

struct Shape8 {
  int n, L, q0;
};

__device__ __forceinline__ Shape8 shape_of(const Fp8DecodeParams& p, int b) {
  Shape8 s;
  if (p.cu_q != nullptr) {
    const int a = __ldg(p.cu_q + b);
    s.n = max(__ldg(p.cu_q + b + 1) - a, 0);
    s.q0 = a;
    s.L = max(__ldg(p.cu_k + b + 1) - __ldg(p.cu_k + b), 0);
  } else {
    s.n = p.n_fixed;
    s.q0 = b * p.n_fixed;   // (num_seqs * n_fixed < 2^31, checked on the host)
    s.L = max(__ldg(p.ctx_lens + b), 0);
  }
  return s;
}

// Tiles of piece i of a sequence: the keys its last query sees.
__device__ __forceinline__ int piece_keys(int n, int L, int i, int max_n) {
  return max(L - n + min(n, (i + 1) * max_n), 0);
}
__device__ __forceinline__ int tiles_of(int keys) { return (keys + 127) >> 7; }

// Cost of a sequence per kv head, in tiles.
__device__ __forceinline__ long long seq_cost(int n, int L, int max_n) {
  long long c = 0;
  for (int i = 0; i * max_n < n; ++i) {
    const int nt = tiles_of(piece_keys(n, L, i, max_n));
    c += nt > 0 ? nt + kSegCost : 0;
  }
  return c;
}

// Where a CTA starts.
struct Start {
  long long segpos;   // cost position of its first segment
  long long x0, x1;   // its share of positions
  long long per;
  int b, piece, g, j;
  int any;
};
static_assert(sizeof(Start) <= 64, "Start");

// The tiles of one CTA in order.  Every lane of the warp holds the same state.
struct Walk {
  long long segpos, x1;
  int b, piece, g, j;
  int n, L, q0;       // the sequence
  int np, Lp, nt;     // the piece: queries, keys its last query sees, tiles
  bool valid;

  __device__ __forceinline__ void load_seq(const Fp8DecodeParams& p) {
    const Shape8 s = shape_of(p, b);
    n = s.n;
    L = s.L;
    q0 = s.q0;
  }
  __device__ __forceinline__ void set_piece(const Fp8DecodeParams& p) {
    np = min(p.max_n, n - piece * p.max_n);
    Lp = piece_keys(n, L, piece, p.max_n);
    nt = tiles_of(Lp);
  }
  __device__ __forceinline__ void begin(const Fp8DecodeParams& p, const Start& s) {
    segpos = s.segpos;
    x1 = s.x1;
    b = s.b;
    piece = s.piece;
    g = s.g;
    j = s.j;
    valid = s.any != 0;
    if (valid) {
      load_seq(p);
      set_piece(p);
    }
  }
  __device__ __forceinline__ void next_segment(const Fp8DecodeParams& p) {
    segpos += nt + kSegCost;
    j = 0;
    if (++g == p.num_kv_heads) {
      g = 0;
      do {
        ++piece;
        while (piece * p.max_n >= n) {
          piece = 0;
          if (++b >= p.num_seqs) {
            valid = false;
            return;
          }
          load_seq(p);
        }
        set_piece(p);
      } while (nt == 0);
    }
    valid = segpos + kSegCost < x1;
  }
  __device__ __forceinline__ void next_tile(const Fp8DecodeParams& p) {
    if (++j < nt) {
      valid = segpos + kSegCost + j < x1;
    } else {
      next_segment(p);
    }
  }
};

template <int NP, int NR>
__device__ __forceinline__ constexpr int group_rows8() {
  return group_rows_rt(Cfg8<NP>::kWG, NR);
}

template <int NP>
__global__ void __launch_bounds__(Cfg8<NP>::kThreads, 2)
paged_decode_fp8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const Fp8DecodeParams p) {
  using C = Cfg8<NP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  int4* info = reinterpret_cast<int4*>(smem + C::kInfo);
  float* qscale = reinterpret_cast<float*>(smem + C::kQScale);
  float* red = reinterpret_cast<float*>(smem + C::kRed);
  float* m_s = reinterpret_cast<float*>(smem + C::kM);
  float* negm_s = reinterpret_cast<float*>(smem + C::kNegM);
  float* alpha_s = reinterpret_cast<float*>(smem + C::kAlpha);
  float* lred = reinterpret_cast<float*>(smem + C::kLred);
  int64_t* row_out = reinterpret_cast<int64_t*>(smem + C::kRowOut);
  float* row_inv = reinterpret_cast<float*>(smem + C::kRowInv);
  float* merge_w = reinterpret_cast<float*>(smem + C::kMergeW);
  Start* start = reinterpret_cast<Start*>(smem + C::kStart);
  long long* scan = reinterpret_cast<long long*>(smem + C::kScan);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kTmem);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + C::kAbort);

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int KVH = p.num_kv_heads;
  const int G = p.group;

  if (tid == 0) {
    for (int s = 0; s < C::kKStages; ++s) {
      mbar_init(&bars[B_KFULL + s], 1);
      mbar_init(&bars[B_KEMPTY + s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[B_VFULL + s], 1);
      mbar_init(&bars[B_VEMPTY + s], 1);
      mbar_init(&bars[B_SFULL + s], 1);
      mbar_init(&bars[B_SEMPTY + s], 128 * C::kWG);
      mbar_init(&bars[B_PFULL + s], 128 * C::kWG);
      mbar_init(&bars[B_OFULL + s], 1);
      mbar_init(&bars[B_QFULL + s], 32);
      mbar_init(&bars[B_QEMPTY + s], 1);
    }
    for (int i = 0; i < kInfoRing; ++i) mbar_init(&bars[B_INFO + i], 1);
    mbar_init(&bars[B_KSTART], 1);
    *abort = 0;
    start->any = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // ------------------------------------------------------------ the work split
  // Two scans over the sequences' costs: the total (hence each CTA's share), then the sequence that holds this CTA's
  // first position.  Batches of up to kThreads sequences keep the first scan's values in registers.
  {
    constexpr int T = C::kThreads, W = T / 32;
    long long mine = 0, excl = 0, total = 0;
    int n = 0, L = 0;
    auto scan_chunk = [&](int base) {   // -> mine, excl (relative to the chunk); returns the chunk's sum
      const int b = base + tid;
      n = 0;
      L = 0;
      mine = 0;
      if (b < p.num_seqs) {
        const Shape8 s = shape_of(p, b);
        n = s.n;
        L = s.L;
        mine = KVH * seq_cost(n, L, p.max_n);
      }
      long long x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(kFull, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) scan[warp] = x;
      __syncthreads();
      long long before = 0, sum = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const long long v = scan[w];
        before += w < warp ? v : 0;
        sum += v;
      }
      excl = before + x - mine;
      __syncthreads();
      return sum;
    };
    for (int base = 0; base < p.num_seqs; base += T) total += scan_chunk(base);
    const long long per = total > 0 ? (total + gridDim.x - 1) / gridDim.x : 1;
    const long long x0 = per * blockIdx.x, x1 = x0 + per;
    auto find = [&](int base, long long before) {   // the thread whose sequence holds position x0
      const long long lo = before + excl;
      if (mine > 0 && x0 >= lo && x0 < lo + mine) {
        long long rem = x0 - lo;
        int i = 0, nt = 0;
        for (;; ++i) {
          nt = tiles_of(piece_keys(n, L, i, p.max_n));
          const long long pc = nt > 0 ? static_cast<long long>(KVH) * (nt + kSegCost) : 0;
          if (rem < pc) break;
          rem -= pc;
        }
        const int g = static_cast<int>(rem / (nt + kSegCost));
        const int o = static_cast<int>(rem - static_cast<long long>(g) * (nt + kSegCost));
        start->segpos = x0 - o;
        start->b = base + tid;
        start->piece = i;
        start->g = g;
        start->j = max(0, o - kSegCost);
        start->any = x0 - o + kSegCost + start->j < x1 ? 1 : 0;
      }
    };
    if (tid == 0) {
      start->x0 = x0;
      start->x1 = x1;
      start->per = per;
    }
    if (p.num_seqs <= T) {
      find(0, 0);
    } else {
      long long before = 0;
      for (int base = 0; base < p.num_seqs; base += T) {
        const long long sum = scan_chunk(base);
        find(base, before);
        before += sum;
      }
    }
    __syncthreads();
  }
  // query rows in pieces without a key (batch padding) belong to no tile: zero, written by CTA b % grid
  for (int b = blockIdx.x; b < p.num_seqs; b += gridDim.x) {
    const Shape8 ss = shape_of(p, b);
    const int rows = ss.L >= ss.n ? 0 : ss.L <= 0 ? ss.n : (ss.n - ss.L) / p.max_n * p.max_n;
    const int per_row = p.num_heads * kHeadDim / 8;
    for (int64_t idx = tid; idx < static_cast<int64_t>(rows) * per_row; idx += C::kThreads) {
      const int64_t i = idx / per_row;
      reinterpret_cast<uint4*>(p.out + (ss.q0 + i) * p.out_row_stride)[idx - i * per_row] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const Start st0 = *start;
  if (!st0.any) return;   // nothing for this CTA: no TMEM, no pipeline

  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------ K (warp 0) and V (warp 3) producers
    // They leave when their tiles are issued; the other warps wait for every tile, so the block outlives the copies.
    const bool is_k = warp == 0;
    const CUtensorMap* tm = is_k ? &tm_k : &tm_v;
    uint8_t* ring = smem + (is_k ? C::kK : C::kV);
    uint64_t* full = bars + (is_k ? B_KFULL : B_VFULL);
    uint64_t* empty = bars + (is_k ? B_KEMPTY : B_VEMPTY);
    const int stages = is_k ? C::kKStages : C::kVStages;
    Walk w;
    w.begin(p, st0);
    bool stop = !is_k && !mbar_wait_warp(&bars[B_KSTART], 0, abort);
    bool first_of_cta = true;
    for (int jj = 0; w.valid && !stop;) {
      // descriptors of the next tiles, one per lane (their block-table reads overlap); a short first round, so that
      // the first copies start early
      const int round = jj == 0 ? 4 : 32;
      int g = 0, j = 0, flags = 0, np = 0, Lp = 0, qrow = 0, nt = 0, b = 0, cnt = 0;
      long long segpos = 0;
      for (; cnt < round && w.valid; ++cnt) {
        const bool first = first_of_cta || w.j == 0;
        const bool seg_end = w.j == w.nt - 1;
        if (lane == cnt) {
          g = w.g;
          j = w.j;
          np = w.np;
          Lp = w.Lp;
          nt = w.nt;
          b = w.b;
          qrow = w.q0 + w.piece * p.max_n;
          segpos = w.segpos;
        }
        first_of_cta = false;
        w.next_tile(p);
        if (lane == cnt) flags = (first ? 1 : 0) | (seg_end || !w.valid ? 2 : 0) | (!w.valid ? 4 : 0);
      }
      int page = -1, off = 0;
      if (lane < cnt) {
        const int col = (j * 128) / p.block_size;
        off = j * 128 - col * p.block_size;
        if (col < p.bt_width) page = __ldg(p.block_tables + static_cast<int64_t>(b) * p.bt_stride + col);
        if (page < 0 || page >= p.num_blocks) {
          if (is_k) atomicOr(&g_error_word, kErrBlockRange);
          page = -1;   // TMA fills out-of-range rows with zeros; nothing outside the pool is read
        }
      }
      for (int i = 0; i < cnt; ++i, ++jj) {
        const int st = jj % stages;
        const int gi = __shfl_sync(kFull, g, i), pi = __shfl_sync(kFull, page, i), oi = __shfl_sync(kFull, off, i);
        int ji = 0, fi = 0, ni = 0, Li = 0, qi = 0, ti = 0;
        long long si = 0;
        if (is_k) {
          ji = __shfl_sync(kFull, j, i);
          fi = __shfl_sync(kFull, flags, i);
          ni = __shfl_sync(kFull, np, i);
          Li = __shfl_sync(kFull, Lp, i);
          qi = __shfl_sync(kFull, qrow, i);
          ti = __shfl_sync(kFull, nt, i);
          si = __shfl_sync(kFull, segpos, i);
        }
        if (!mbar_wait_warp(&empty[st], ((jj / stages) & 1) ^ 1, abort)) {
          stop = true;
          break;
        }
        if (elect_one()) {
          if (is_k) {
            const int e = jj % kInfoRing;
            info[3 * e] = make_int4(ji * 128, pi, oi, gi);
            info[3 * e + 1] = make_int4(ni, Li, qi, ti);
            info[3 * e + 2] = make_int4(fi, 0, static_cast<int>(si), static_cast<int>(si >> 32));
            mbar_arrive(&bars[B_INFO + e]);
          }
          mbar_arrive_expect_tx(&full[st], kTile);
          tma_load_3d(ring + st * kTile, tm, 0, gi, pi < 0 ? -kTileTokens : pi * p.block_size + oi, &full[st]);
          if (is_k && jj == 0) mbar_arrive(&bars[B_KSTART]);
        }
        __syncwarp();
      }
    }
    return;
  }
  // ------------------------------------------------------------ the other warps: TMEM, then their roles
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  named_bar_sync(3, C::kThreads - 64);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 1) {
    // ------------------------------------------------------------ UMMA issuer (the warp waits, an elected lane issues)
    const uint64_t q_desc0 = umma_desc_sw128(smem_u32(smem + C::kQ), 16, 1024);
    const uint64_t k_desc0 = umma_desc_sw128(smem_u32(smem + C::kK), 16, 1024);
    const uint64_t v_desc0 = umma_desc_sw128(smem_u32(smem + C::kV), kTile, 1024);
    const uint64_t p_desc0 = umma_desc_noswz(smem_u32(smem + C::kP), 128, 2048);
    int qk = 0, pv = 0, qseg = 0, oseg = 0;
    bool ok = true, qk_done = false;
    // order: QK(0), QK(1), then PV(j), QK(j + 2), ...
    auto issue_qk = [&]() {
      if (!ok || qk_done) return;
      const int st = qk % C::kKStages;
      const int e = qk % kInfoRing;
      if (!mbar_wait_warp(&bars[B_INFO + e], (qk / kInfoRing) & 1, abort) ||
          !mbar_wait_warp(&bars[B_KFULL + st], (qk / C::kKStages) & 1, abort)) { ok = false; return; }
      const int flags = info[3 * e + 2].x;
      const uint32_t idesc = idesc_f8(min(NP, mma_width(info[3 * e + 1].x * G)), false, false);
      const int qb = qseg % C::kQBuf;
      if ((flags & 1) && !mbar_wait_warp(&bars[B_QFULL + qb], (qseg / C::kQBuf) & 1, abort)) { ok = false; return; }
      const int buf = qk & 1;
      if (!mbar_wait_warp(&bars[B_SEMPTY + buf], ((qk >> 1) & 1) ^ 1, abort)) { ok = false; return; }
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = k_desc0 + ((st * kTile) >> 4);
        const uint64_t b = q_desc0 + ((qb * C::kOperand) >> 4);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int k = 0; k < 4; ++k)   // 32 dims a step: +32 bytes inside the 128-byte rows
            umma_f8_ss(tmem + buf * NP, a + 2 * k, b + ((part * NP * 128) >> 4) + 2 * k, idesc, part + k > 0);
        umma_commit(&bars[B_SFULL + buf]);
        umma_commit(&bars[B_KEMPTY + st]);
        if (flags & 2) umma_commit(&bars[B_QEMPTY + qb]);
      }
      __syncwarp();
      if (flags & 2) ++qseg;
      if (flags & 4) qk_done = true;
      ++qk;
    };
    issue_qk();
    issue_qk();
    while (ok) {
      const int st = pv % C::kVStages;
      const int pb = pv & 1;
      if (!mbar_wait_warp(&bars[B_PFULL + pb], (pv >> 1) & 1, abort)) break;
      if (!mbar_wait_warp(&bars[B_VFULL + st], (pv / C::kVStages) & 1, abort)) break;
      const int e = pv % kInfoRing;
      const int flags = info[3 * e + 2].x;
      if ((flags & 1) && pv > 0) oseg ^= 1;
      const int width = min(NP, mma_width(info[3 * e + 1].x * G));
      const uint32_t idesc_hi = idesc_f8(width, true, true), idesc_lo = idesc_f8(width, false, true);
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = v_desc0 + ((st * kTile) >> 4);
        const uint64_t b = p_desc0 + ((pb * C::kOperand) >> 4);
        const uint32_t d = tmem + (2 + oseg) * NP;
        const uint32_t fresh = (flags & 1) ? 0u : 1u;
#pragma unroll
        for (int k = 0; k < 4; ++k)   // 32 tokens a step: four groups of 8 (V: 1024 bytes each, P^T: 128)
          umma_f8_ss(d, a + 256 * k, b + 32 * k, idesc_hi, k > 0 ? 1u : fresh);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f8_ss(d, a + 256 * k, b + ((NP * 128) >> 4) + 32 * k, idesc_lo, 1u);
        umma_commit(&bars[B_OFULL + pb]);
        umma_commit(&bars[B_VEMPTY + st]);
      }
      __syncwarp();
      ++pv;
      if (flags & 4) break;
      issue_qk();
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ Q loader: bf16 rows -> two e4m3 parts + row scale
    Walk w;
    w.begin(p, st0);
    for (int qi = 0; w.valid; ++qi) {
      const int qb = qi % C::kQBuf;
      if (!mbar_wait_warp(&bars[B_QEMPTY + qb], ((qi / C::kQBuf) & 1) ^ 1, abort)) break;
      const int R = w.np * G;
      const int rows = min(NP, mma_width(R));   // the rows the S product reads; those past R are zero
      uint8_t* qs = smem + C::kQ + qb * C::kOperand;
      float* sc = qscale + (qi % kQScaleRing) * NP;
      const int64_t base = static_cast<int64_t>(w.q0 + w.piece * p.max_n);
      constexpr int kBatch = 8;
      for (int r0 = 0; r0 < rows; r0 += kBatch) {
        uint2 x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int r = r0 + u;
          x[u] = make_uint2(0u, 0u);
          if (r < R) {
            const int i = r / G, h = r - i * G;
            x[u] = __ldg(reinterpret_cast<const uint2*>(p.q + (base + i) * p.q_row_stride +
                                                        static_cast<int64_t>(w.g * G + h) * kHeadDim + lane * 4));
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int r = r0 + u;
          uint32_t mx = max(max(x[u].x & 0x7FFFu, (x[u].x >> 16) & 0x7FFFu),
                            max(x[u].y & 0x7FFFu, (x[u].y >> 16) & 0x7FFFu));
          mx = __reduce_max_sync(kFull, mx);
          // the row's largest value to [2^7, 2^8): times 2^(134 - E); NaN or infinity anywhere makes the row NaN
          const int E = max(static_cast<int>(mx >> 7), 8);
          const float f = __uint_as_float(static_cast<uint32_t>(261 - min(E, 254)) << 23);
          const float back = E == 255 ? __uint_as_float(0x7FC00000u)
                                      : __uint_as_float(static_cast<uint32_t>(E - 7) << 23);
          const float2 a01 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[u].x));
          const float2 a23 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[u].y));
          const float v0 = a01.x * f, v1 = a01.y * f, v2 = a23.x * f, v3 = a23.y * f;
          const uint32_t h01 = pack_e4m3(v0, v1), h23 = pack_e4m3(v2, v3);
          const float2 u01 = unpack_e4m3(h01), u23 = unpack_e4m3(h23);
          const uint32_t l01 = pack_e4m3(v0 - u01.x, v1 - u01.y), l23 = pack_e4m3(v2 - u23.x, v3 - u23.y);
          uint8_t* at = qs + sw128_offset(r, lane >> 2) + (lane & 3) * 4;
          *reinterpret_cast<uint32_t*>(at) = h01 | (h23 << 16);
          *reinterpret_cast<uint32_t*>(at + NP * 128) = l01 | (l23 << 16);
          if (lane == 0) sc[r] = back;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive(&bars[B_QFULL + qb]);
      w.next_segment(p);
    }
  } else {
    // ------------------------------------------------------------ softmax
    // Group wg owns rows [rb, rb + hr) of the segment's nr-wide tile.  Every wait is warp-uniform and every named
    // barrier that can end the loop ORs "gave up" over the group's warps, so they leave together.
    const int cidx = tid - kConsumerBase;
    const int ct = cidx & 127;                // TMEM lane: token ct of S^T, dim ct of O^T
    const int wg = cidx >> 7;
    const int wq = ct >> 5;
    const uint32_t bar_id = 1 + wg;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    constexpr int NPH = C::kRows;
    float l[NPH], s[NPH];
    int R = 0, nr = 8, n = 0, L = 0, q0 = 0, seg_g = 0, seg_nt = 0, ob = 0, seg = -1;
    long long segpos = 0;
    bool alive = true;
    float ks_next = 0.f, vs_next = 1.f;

    auto arrive_and_merge = [&](int c0, int c1, int rb_, int hr_) {
      named_bar_sync(bar_id, 128);
      bool last_arrival = false;
      if (ct == 0) {
        int32_t* ticket = p.counters + kTicketStride * c0 + wg;
        __threadfence();   // release: the group's partial rows before the ticket
        last_arrival = atomicAdd(ticket, 1) == c1 - c0;
        if (last_arrival) {
          __threadfence();   // acquire: the other pieces' rows
          *ticket = 0;
        }
      }
      if (named_bar_any(bar_id, 128, last_arrival))
        merge_pieces<NP>(p, c0, c1, rb_, min(rb_ + hr_, R), G,
                         (int64_t)q0 * p.out_row_stride + (int64_t)seg_g * G * kHeadDim, ct,
                         merge_w + rb_ * kMergePieces, bar_id);
    };
    // This token's scales of tile e's descriptor.  Tokens past the keys and pages outside the pool read nothing.
    auto load_scales = [&](const int4 a, const int4 b) {
      ks_next = 0.f;
      vs_next = 1.f;
      if (a.y >= 0 && a.x + ct < b.y) {
        const int64_t at = (static_cast<int64_t>(a.y) * KVH + a.w) * p.page_blocks + ((a.z + ct) >> p.lg_block);
        ks_next = __ldg(p.k_scale + at);
        vs_next = __ldg(p.v_scale + at);
      }
    };

    alive = mbar_wait_warp(&bars[B_INFO], 0, abort);
    if (alive) load_scales(info[0], info[1]);
    for (int jj = 0;; ++jj) {
      const int st = jj % C::kVStages;
      const int buf = jj & 1;
      const int e = jj % kInfoRing;
      alive = alive && mbar_wait_warp(&bars[B_INFO + e], (jj / kInfoRing) & 1, abort);
      int4 ia = make_int4(0, 0, 0, 0), ib = ia, ic = make_int4(7, 0, 0, 0);
      if (alive) {
        ia = info[3 * e];
        ib = info[3 * e + 1];
        ic = info[3 * e + 2];
      }
      const bool first = ic.x & 1, last = ic.x & 2, last_tile = ic.x & 4;
      if (first) {
        if (jj > 0) ob ^= 1;
        ++seg;
        n = ib.x;
        L = ib.y;
        q0 = ib.z;
        seg_nt = ib.w;
        seg_g = ia.w;
        segpos = (static_cast<long long>(ic.w) << 32) | static_cast<uint32_t>(ic.z);
        R = n * G;
        nr = min(NP, rows_width(R));
#pragma unroll
        for (int r = 0; r < NPH; ++r) l[r] = 0.f;
      }
      const int hr = group_rows_rt(C::kWG, nr);
      const int rb = wg * hr;
      const int tok0 = ia.x;
      const int tok = tok0 + ct;
      // this token's factors; the next tile's scales are on their way while this tile is worked on
      const bool live = tok < L;
      const float vs = fminf(fmaxf(vs_next, 9.094947e-13f), 1.0995116e12f);   // 2^-40 .. 2^40
      const float a = live ? ks_next * p.scale_log2 : 0.f;
      const float lv = __log2f(vs);
      const float ivs = live ? __frcp_rn(vs) : 0.f;
      if (alive && !last_tile) {
        const int e1 = (jj + 1) % kInfoRing;
        alive = mbar_wait_warp(&bars[B_INFO + e1], ((jj + 1) / kInfoRing) & 1, abort);
        if (alive) load_scales(info[3 * e1], info[3 * e1 + 1]);
      }
      if (C::kWG > 1 && rb >= R) {
        // every row of this group is padding: keep the S and P phases paced as the working group does
        alive = alive && mbar_wait_warp(&bars[B_SFULL + buf], (jj >> 1) & 1, abort);
        if (alive) mbar_arrive(&bars[B_SEMPTY + buf]);
        if (jj >= 2) alive = alive && mbar_wait_warp(&bars[B_OFULL + buf], ((jj - 2) >> 1) & 1, abort);
        if (alive) mbar_arrive(&bars[B_PFULL + buf]);
        // mirrors the working path's two votes on the way out, so that warps of one group that disagree about the
        // segment after a wait gave up still meet and leave together
        if (named_bar_any(bar_id, 128, !alive)) {
          named_bar_any(bar_id, 128, true);
          break;
        }
        if (last_tile) break;
        continue;
      }
      alive = alive && mbar_wait_warp(&bars[B_SFULL + buf], (jj >> 1) & 1, abort);
      bool need = first;
      const bool open_tile = tok0 + 127 <= L - n;   // every row sees every token
      const int d = tok - (L - n);                  // row r = i * G + h sees the token iff r >= G * d
      const int rmin = !live ? NP : d > 0 ? d * G : 0;
      const float* qs = qscale + (seg % kQScaleRing) * NP + rb;
      // s <- y (offset `add` apart): score, scale of q, scale of k, log2 of v's scale; -inf where masked
      auto scores = [&](auto hr_c, const float* add) {
        constexpr int HR = decltype(hr_c)::value;
        tmem_ld_cols<HR>(t_lane + buf * NP + rb, s);
        const float2 a2 = make_float2(a, a), lv2 = make_float2(lv, lv);
#pragma unroll
        for (int r = 0; r < HR; r += 2) {
          const float2 q2 = *reinterpret_cast<const float2*>(qs + r);
          const float2 o2 = add != nullptr ? fadd2(*reinterpret_cast<const float2*>(add + r), lv2) : lv2;
          const float2 y = ffma2(fmul2(make_float2(s[r], s[r + 1]), a2), q2, o2);
          s[r] = y.x;
          s[r + 1] = y.y;
        }
        if (!open_tile) {
#pragma unroll
          for (int i = 0; i < HR; ++i) {
            const int r = rb + i;
            s[i] = (r >= rmin && r < R) ? s[i] : kNegInf;
          }
        }
      };
      if (alive) {
        tc_fence_after();
        with_rows<NP>(nr, [&](auto nr_c) {
          constexpr int HR = group_rows8<NP, decltype(nr_c)::value>();
          if (!first) {
            scores(std::integral_constant<int, HR>{}, negm_s + rb);
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < HR; ++i) {
              s[i] = fast_exp2(s[i]);
              top = fmaxf(top, s[i]);
            }
            need = top > kWeightMax;
          }
        });
      }
      // one vote per tile; a warp that gave up votes too and is caught by the second vote below
      const bool rescale = named_bar_any(bar_id, 128, need || !alive);
      if (rescale) {
        if (named_bar_any(bar_id, 128, !alive)) break;
        with_rows<NP>(nr, [&](auto nr_c) {
          constexpr int HR = group_rows8<NP, decltype(nr_c)::value>();
          scores(std::integral_constant<int, HR>{}, nullptr);
          warp_columns<HR, true>(s, red + wq * NP + rb, lane);
        });
        named_bar_sync(bar_id, 128);
        if (ct < hr) {
          const int row = rb + ct;
          float mn = 0.f, neg = kNegInf, alpha = 1.f;   // rows past R: no weight
          if (row < R) {
            const float tm = fmaxf(fmaxf(red[row], red[NP + row]), fmaxf(red[2 * NP + row], red[3 * NP + row]));
            const float mo = first ? kNegInf : m_s[row];
            mn = (first || tm > mo + kSlack) ? fmaxf(mo, tm) : mo;
            neg = mn == kNegInf ? 0.f : kBase - mn;   // a row that has seen no key yet: its scores are -inf
            alpha = (mo == kNegInf || mn == mo) ? 1.f : fast_exp2(mo - mn);
          }
          m_s[row] = mn;
          negm_s[row] = neg;
          alpha_s[row] = alpha;
        }
        named_bar_sync(bar_id, 128);
      }
      with_rows<NP>(nr, [&](auto nr_c) {
        constexpr int HR = group_rows8<NP, decltype(nr_c)::value>();
        if (rescale) {
          const float* nm = negm_s + rb;
          const float* al = alpha_s + rb;
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            s[r] = fast_exp2(s[r] + nm[r]);
            l[r] *= al[r];
          }
        }
#pragma unroll
        for (int r = 0; r < HR; r += 2) {
          const float2 l2 = ffma2(make_float2(s[r], s[r + 1]), make_float2(ivs, ivs), make_float2(l[r], l[r + 1]));
          l[r] = l2.x;
          l[r + 1] = l2.y;
        }
        // S(jj) is no longer read: its buffer may take S(jj + 2)
        tc_fence_before();
        mbar_arrive(&bars[B_SEMPTY + buf]);
        // some row maxima moved: the group's O rows scale once PV(jj - 1) has added onto them
        if (rescale && !first && alive) {
          alive = mbar_wait_warp(&bars[B_OFULL + (buf ^ 1)], ((jj - 1) >> 1) & 1, abort);
          if (alive) {
            tc_fence_after();
            const float* al = alpha_s + rb;
#pragma unroll
            for (int c = 0; c < HR; c += 8) {
              float ot[8];
              tmem_ld8(t_lane + (2 + ob) * NP + rb + c, ot);
#pragma unroll
              for (int i = 0; i < 8; ++i) ot[i] *= al[c + i];
              tmem_st8(t_lane + (2 + ob) * NP + rb + c, ot);
            }
            tc_fence_before();
          }
        }
        // P(jj) goes where PV(jj - 2) read
        if (jj >= 2 && alive) alive = mbar_wait_warp(&bars[B_OFULL + buf], ((jj - 2) >> 1) & 1, abort);
        // rows past the piece's keys may hold anything, NaN too: zero V there, so that no weight of 0 meets it
        if (alive && wg == 0 && L - tok0 < kTileTokens) {
          alive = mbar_wait_warp(&bars[B_VFULL + st], (jj / C::kVStages) & 1, abort);
          if (alive && !live) {
            uint4* vrow = reinterpret_cast<uint4*>(smem + C::kV + st * kTile + ct * 128);
#pragma unroll
            for (int c = 0; c < 8; ++c) vrow[c] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        if (alive) {
          // P^T: hi rounded to three significant bits (half up), lo = w - hi exactly; 8 rows of token ct are 8 bytes
          uint8_t* pb = smem + C::kP + buf * C::kOperand + ct * 16;
#pragma unroll
          for (int m = 0; m < HR / 8; ++m) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float t[4], u[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float w = s[8 * m + 4 * h + i];
                t[i] = __uint_as_float((__float_as_uint(w) + 0x00100000u) & 0xFFE00000u);
                u[i] = w - t[i];
              }
              hi[h] = pack_e5m2(t[0], t[1]) | (pack_e5m2(t[2], t[3]) << 16);
              lo[h] = pack_e4m3(u[0], u[1]) | (pack_e4m3(u[2], u[3]) << 16);
            }
            const int row = rb + 8 * m;
            uint8_t* at = pb + (row >> 4) * 2048 + (row & 8);
            *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(at + NP * 128) = make_uint2(lo[0], lo[1]);
          }
          fence_proxy_async_smem();
          mbar_arrive(&bars[B_PFULL + buf]);
        }
        if (last && alive) {
          alive = mbar_wait_warp(&bars[B_OFULL + buf], (jj >> 1) & 1, abort);
          if (alive) {
            tc_fence_after();
            warp_columns<HR, false>(l, lred + wq * NP + rb, lane);
            tmem_ld_cols<HR>(t_lane + (2 + ob) * NP + rb, s);   // the segment's accumulated O
            tc_fence_before();
          }
        }
      });
      if (named_bar_any(bar_id, 128, !alive)) break;
      if (last) {
        const long long per = st0.per;
        const int c0 = static_cast<int>((segpos + kSegCost) / per);
        const int c1 = static_cast<int>((segpos + kSegCost + seg_nt - 1) / per);
        const bool complete = c0 == c1;
        const int slot = 2 * blockIdx.x + (segpos + kSegCost < st0.x0 ? 0 : 1);
        if (ct < hr) {
          const int r = rb + ct;
          if (r < R) {
            const float lt = lred[r] + lred[NP + r] + lred[2 * NP + r] + lred[3 * NP + r];
            row_inv[r] = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);   // a NaN sum stays NaN
            if (complete) {
              const int qi = r / G, h = r - qi * G;
              row_out[r] = (int64_t)(q0 + qi) * p.out_row_stride + (int64_t)(seg_g * G + h) * kHeadDim;
            } else {
              row_out[r] = ((int64_t)slot * NP + r) * kHeadDim;
              p.part_lse[slot * NP + r] = lt == 0.f ? kNegInf : m_s[r] + __log2f(lt);
            }
          }
        }
        named_bar_sync(bar_id, 128);
        with_rows<NP>(nr, [&](auto nr_c) {
          constexpr int HR = group_rows8<NP, decltype(nr_c)::value>();
#pragma unroll
          for (int i = 0; i < HR; ++i) {
            const int r = rb + i;
            if (r < R) {
              const float val = s[i] * row_inv[r];
              if (complete) {
                p.out[row_out[r] + ct] = __float2bfloat16_rn(val);
              } else {
                p.part_o[row_out[r] + ct] = val;
              }
            }
          }
        });
        if (!complete) arrive_and_merge(c0, c1, rb, hr);
      }
      if (last_tile) break;
    }
  }

  named_bar_sync(3, C::kThreads - 64);
  if (*abort) {
    // a wait gave up: let any copy or MMA still in flight land before the shared memory and TMEM go away
    if (tid == kConsumerBase) atomicOr(&g_error_word, kErrTimeout);
    for (int i = 0; i < 1000; ++i) sleep_ns(1000);
    named_bar_sync(3, C::kThreads - 64);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

template <int NP>
cudaError_t launch8(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const Fp8DecodeParams& p, int grid,
                    cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(paged_decode_fp8_kernel<NP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg8<NP>::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(paged_decode_fp8_kernel<NP>, dim3(grid), dim3(Cfg8<NP>::kThreads), Cfg8<NP>::kBytes, stream,
                       false, tm_k, tm_v, p);
}

// 8-bit view {128 bytes, heads, rows} of a cache, 128 x 1 x 128 boxes, 128-byte swizzle.
int encode_rows8(CUtensorMap* tm, const void* base, int64_t heads, int64_t rows) {
  cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {128, static_cast<cuuint64_t>(heads) * 128};
  cuuint32_t box[3] = {128, 1, 128};
  return encode_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box);
}

// Rows of a tile for runs of up to `rows` packed query rows.
int tile_rows(int rows) { return rows <= 8 ? 16 : rows <= 32 ? 32 : rows <= 48 ? 48 : 0; }

size_t workspace8(int sms, int np) {
  return decode_ticket_bytes(sms) + static_cast<size_t>(2) * (2 * sms) * np * (kHeadDim + 1) * sizeof(float);
}

// The part of both calls after their own checks.
int run_attention(Fp8DecodeParams p, const void* k_cache, const void* v_cache, const float* k_scale,
                  const float* v_scale, int32_t scale_block, int np, void* workspace, size_t workspace_bytes,
                  void* stream) {
  const int64_t rows = static_cast<int64_t>(p.num_blocks) * p.block_size;
  const int sms = sm_count();
  if (sms == 0) return cuda_fail(cudaGetLastError());
  if (workspace == nullptr || workspace_bytes < workspace8(sms, np) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
    return NVA_ERR_WORKSPACE;
  CUtensorMap tm_k, tm_v;
  int rc;
  if ((rc = encode_rows8(&tm_k, k_cache, p.num_kv_heads, rows)) != NVA_OK) return rc;
  if ((rc = encode_rows8(&tm_v, v_cache, p.num_kv_heads, rows)) != NVA_OK) return rc;
  const int grid = 2 * sms;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.page_blocks = p.block_size / scale_block;
  p.lg_block = __builtin_ctz(static_cast<unsigned>(scale_block));
  p.max_n = np / p.group;
  p.counters = static_cast<int32_t*>(workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + decode_ticket_bytes(sms));
  p.part_lse = p.part_o + static_cast<size_t>(2) * grid * np * kHeadDim;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = np == 16   ? launch8<16>(tm_k, tm_v, p, grid, s)
                        : np == 32 ? launch8<32>(tm_k, tm_v, p, grid, s)
                                   : launch8<48>(tm_k, tm_v, p, grid, s);
  return e == cudaSuccess ? NVA_OK : cuda_fail(e);
}

int check_common(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache, const float* k_scale,
                 const float* v_scale, int32_t num_blocks, int32_t block_size, int32_t scale_block,
                 const int32_t* block_tables, int32_t bt_row_stride, int32_t bt_width, int32_t num_heads,
                 int32_t num_kv_heads, int32_t head_dim, const void* out, int64_t out_row_stride) {
  if (k_cache == nullptr || v_cache == nullptr || k_scale == nullptr || v_scale == nullptr || num_blocks <= 0 ||
      block_size <= 0 || scale_block <= 0 || q == nullptr || out == nullptr || block_tables == nullptr ||
      bt_width < 1 || bt_row_stride < bt_width)
    return NVA_ERR_INVALID_ARGUMENT;
  if (block_size % kTileTokens != 0 || (scale_block & (scale_block - 1)) != 0 || scale_block < NVA_MIN_SCALE_BLOCK ||
      scale_block > NVA_MAX_SCALE_BLOCK || block_size % scale_block != 0 ||
      static_cast<int64_t>(num_blocks) * block_size >= (int64_t(1) << 31))
    return NVA_ERR_UNSUPPORTED;
  const int64_t row = static_cast<int64_t>(num_heads) * head_dim;
  if (q_row_stride < row || out_row_stride < row) return NVA_ERR_INVALID_ARGUMENT;
  auto misaligned = [](const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) != 0; };
  if (misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(q, 16) || q_row_stride % 8 != 0 ||
      misaligned(out, 16) || out_row_stride % 8 != 0 || misaligned(k_scale, 4) || misaligned(v_scale, 4))
    return NVA_ERR_ALIGNMENT;
  return NVA_OK;
}

bool positive_finite(float s) { return s > 0.f && s < 3.0e38f; }

}  // namespace

}  // namespace nva

extern "C" {

NVA_API size_t nva_paged_decode_fp8_workspace_bytes(int32_t q_per_seq, int32_t num_heads, int32_t num_kv_heads,
                                                    int32_t head_dim) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || q_per_seq < 1 ||
      head_dim != nva::kHeadDim)
    return 0;
  const int64_t rows = static_cast<int64_t>(q_per_seq) * (num_heads / num_kv_heads);
  const int np = rows <= nva::kMaxDecodeRows ? nva::tile_rows(static_cast<int>(rows)) : 0;
  const int sms = nva::sm_count();
  return np == 0 || sms == 0 ? 0 : nva::workspace8(sms, np);
}

NVA_API size_t nva_varlen_fp8_workspace_bytes(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim != nva::kHeadDim ||
      num_heads / num_kv_heads > nva::kMaxDecodeRows)
    return 0;
  const int sms = nva::sm_count();
  return sms == 0 ? 0 : nva::workspace8(sms, 48);
}

NVA_API int nva_paged_decode_fp8(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                 const float* k_scale, const float* v_scale, int32_t num_blocks, int32_t block_size,
                                 int32_t scale_block, const int32_t* context_lens, const int32_t* block_tables,
                                 int32_t bt_row_stride, int32_t bt_width, int32_t num_seqs, int32_t q_per_seq,
                                 int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float softmax_scale,
                                 void* out, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (num_seqs < 0 || q_per_seq < 1 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      !nva::positive_finite(softmax_scale))
    return NVA_ERR_INVALID_ARGUMENT;
  if (head_dim != nva::kHeadDim) return NVA_ERR_UNSUPPORTED;
  if (num_seqs == 0) return NVA_OK;
  int rc = nva::check_common(q, q_row_stride, k_cache, v_cache, k_scale, v_scale, num_blocks, block_size, scale_block,
                             block_tables, bt_row_stride, bt_width, num_heads, num_kv_heads, head_dim, out,
                             out_row_stride);
  if (rc != NVA_OK) return rc;
  if (context_lens == nullptr) return NVA_ERR_INVALID_ARGUMENT;
  const int64_t rows = static_cast<int64_t>(q_per_seq) * (num_heads / num_kv_heads);
  const int np = rows <= nva::kMaxDecodeRows ? nva::tile_rows(static_cast<int>(rows)) : 0;
  if (np == 0 || static_cast<int64_t>(num_seqs) * q_per_seq >= (int64_t(1) << 31)) return NVA_ERR_UNSUPPORTED;
  nva::Fp8DecodeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_row_stride = q_row_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_row_stride = out_row_stride;
  p.ctx_lens = context_lens;
  p.block_tables = block_tables;
  p.bt_stride = bt_row_stride;
  p.bt_width = bt_width;
  p.num_seqs = num_seqs;
  p.n_fixed = q_per_seq;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = num_heads / num_kv_heads;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  return nva::run_attention(p, k_cache, v_cache, k_scale, v_scale, scale_block, np, workspace, workspace_bytes, stream);
}

NVA_API int nva_varlen_attention_fp8(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                     const float* k_scale, const float* v_scale, int32_t num_blocks,
                                     int32_t block_size, int32_t scale_block, const int32_t* cu_seqlens_q,
                                     const int32_t* cu_seqlens_k, int32_t num_seqs, int32_t total_q,
                                     const int32_t* block_tables, int32_t bt_row_stride, int32_t bt_width,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float softmax_scale,
                                     void* out, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (num_seqs < 0 || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      !nva::positive_finite(softmax_scale))
    return NVA_ERR_INVALID_ARGUMENT;
  if (head_dim != nva::kHeadDim || num_heads / num_kv_heads > nva::kMaxDecodeRows) return NVA_ERR_UNSUPPORTED;
  if (num_seqs == 0 || total_q == 0) return NVA_OK;
  int rc = nva::check_common(q, q_row_stride, k_cache, v_cache, k_scale, v_scale, num_blocks, block_size, scale_block,
                             block_tables, bt_row_stride, bt_width, num_heads, num_kv_heads, head_dim, out,
                             out_row_stride);
  if (rc != NVA_OK) return rc;
  if (cu_seqlens_q == nullptr || cu_seqlens_k == nullptr) return NVA_ERR_INVALID_ARGUMENT;
  nva::Fp8DecodeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_row_stride = q_row_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_row_stride = out_row_stride;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.block_tables = block_tables;
  p.bt_stride = bt_row_stride;
  p.bt_width = bt_width;
  p.num_seqs = num_seqs;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = num_heads / num_kv_heads;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  return nva::run_attention(p, k_cache, v_cache, k_scale, v_scale, scale_block, 48, workspace, workspace_bytes, stream);
}

}  // extern "C"
