// Paged GQA attention over an 8-bit KV cache for sm_100a: decode, speculative verify and varlen (prefill chunks, mixed
// batches), the 8-bit counterpart of flash_attn_with_kvcache (nanovllm/layers/attention.py:75-77) and of the paged
// flash_attn_varlen_func (:67-70).
//
// The cache holds e4m3 values c with a float32 scale per (block of tokens, kv head): k = kc * ks, v = vc * vs.
//     x[r, t]  = (q[r] . kc[t]) * ks[t] * softmax_scale * log2(e)         score in log2 units
//     y[r, t]  = x[r, t] + log2 vs[t]                                     the scale of v moved into the exponent
//     w[r, t]  = 2^(y - m[r] + 12)        m: running row maximum of y
//     out[r]   = sum_t w[r, t] vc[t] / sum_t w[r, t] / vs[t]
// so neither k nor v is ever multiplied out: both products read the cache's own bytes on the 8-bit tensor pipe, and one
// pass over K and V serves every q head of the group and every query row.  The other operand of each product is split
// into 8-bit parts that accumulate into the same TMEM columns, which keeps the 16-bit kernels' accuracy:
//   q  = (hi + lo) * 2^e, both e4m3, e from the row's largest value: four significant bits each, together all eight of a
//        bf16 value (exact for values down to 2^-10 of the row's largest, off by at most 2^-18 of that below);
//   w  rounded to float16, whose eleven bits are the sum of three e5m2 parts of three bits and their signs (the upper
//        byte of a float16 is an e5m2 value, so that splitting takes integer operations on pairs): off by at most 2^-11
//        of w (bf16's rounding: 2^-8) and by 2^-17, the parts' smallest step, where the row's largest is 2^12 to 2^15.
//        So weights keep seven bits down to 2^-22 of the largest, and the 2^-17 of every one of 100,000 tokens that are
//        all rounded the same way come to 2^-12 of it.  Two parts, e5m2 and a rest in e4m3, had no more than three bits
//        below 2^-15 of the largest: a long flat tail behind one heavy token was off by up to a tenth of itself.  Sums of
//        weights stay in float32, unrounded.
//
// Bound: HBM, one byte per cached value (decode of 64 sequences, contexts 512 to 4096: 303 MB, 46 us at the copy rate).  A
// 128-token tile then takes 0.74 us of an SM's share of the bandwidth, half of the bf16 cache's, which is less than one
// tile's chain S -> weights -> PV takes; so two CTAs share an SM and their chains overlap.
//
// Orientation, roles and the merge of split segments are those of paged_decode.cu: tokens on the TMEM lanes (UMMA M),
// query rows on N; warp 0 = K producer, 1 = TMEM + UMMA issuer, 2 = Q loader, 3 = V producer, 4.. = softmax groups.
// K tile: K-major, 128-byte swizzle, 128 dims = one swizzle row.  V tile: the same bytes read MN-major.  P^T: MN-major
// without swizzle, 16 rows of a token per 16 bytes.
//
// Work split: heads go in sets of 8 (or 4, 2, 1) that as many CTAs walk side by side, tile for tile, so that the rows of
// a token, 128 bytes a head, are fetched as the 1 KB that lies together (contexts of 50,000 of 8 sequences: 196 us a head
// alone, 135 in sets; short ones 28.0 and 28.8).  Every set owns an equal share of cost positions (tiles + 3 per segment)
// in (sequence, piece, set, tile) order, where a piece is a run of at most max_n queries of a sequence: a longer run is
// walked piece by piece, each over the keys its last query sees, up to where the prefill kernel takes it (kMinPrefillRun).
// A set finds its start with one scan over the lengths and walks on from there, so there is no table of sequences on the
// chip and no bound on their number.
//
// Measured (32 q heads over 8, copy rate 6.57 TB/s): decode of 64 sequences of 512 to 4096 60 to 65 us (71 to 77%), of 8192
// 167 us (97%), 8 of 40,000 to 65,536 141 us (93%); verify of 32 sequences of 256 to 2048, k = 4, 41 to 43 us (7 to 10 tiles
// a CTA); 4 sequences of 37 to 1000 18 us, of which the start takes 6, the tiles 5 and the ends 5; 256 single queries with
// three prefill chunks 247 us: three kernels, each launched so that its blocks start where the last one's leave.
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
constexpr int kMaxRows8 = 40;           // packed query rows (queries x group) of a tile
constexpr int kSegCost = 3;             // a segment's start and end, in tiles
constexpr float kBase = 12.0f;          // the largest weight of a row is 2^kBase when its maximum is exact ...
constexpr float kSlack = 3.0f;          // ... and may pass it by this much (log2) before the maximum moves
constexpr float kWeightMax = 32768.0f;  // 2^(kBase + kSlack): inside float16's range

// NR: the most query rows a softmax thread carries.  One softmax group of 128 threads at 128 registers each: at 40 rows
// (weights and sums of 40 rows, 80 registers) a few words spill; with more rows they spill past an L1 that two CTAs' shared
// memory leaves next to nothing, and a tile takes four times as long.
template <int NR>
struct Cfg8 {
  static constexpr int kThreads = kConsumerBase + 128;
  static constexpr int NP = (NR + 15) / 16 * 16;      // UMMA N
  // Rings that let two CTAs fit an SM (113 KB each): 3 + 2 tiles at 16 rows, 2 + 2 with the wider Q and P buffers
  static constexpr int kKStages = NP == 16 ? 3 : 2;
  static constexpr int kVStages = 2;
  static constexpr int kQBuf = 2;
  static constexpr int kPBuf = NP == 48 ? 1 : 2;
  // The three parts of P^T, in chunks of 16 rows: up to 16 rows side by side in one product (8 rows: two parts to a chunk),
  // whose columns are added up at the segment's end; a product of few columns takes as long as reading V for it, so that
  // three of them onto the same columns cost more (8 rows, 8 sequences of 40,000 to 65,536: 156 us, one product 141; 16
  // rows, 64 sequences of 4000: 108 and 106).  With more rows three are as fast (20 rows, 4000 tokens: 131, one product
  // 133; 32 sequences of 256 to 2048: 43.4 and 42.9), and at 40 TMEM has no room for one.
  static constexpr int kOParts = NP == 16 ? 3 : 1;
  static constexpr int kOStep = NR == 8 ? 8 : NP;      // from a part's columns of O to the next one's
  static constexpr int kOCols = NR == 8 ? 32 : kOParts * NP;
  // hi and lo of Q: NR rows (a UMMA wider than that reads the bytes behind them into columns nobody looks at)
  static constexpr int kQHalf = (NR < 16 ? 16 : NR) * 128, kQBytes = 2 * kQHalf;
  static constexpr int kPPart = NP * 128, kPBytes = NR == 8 ? kOCols * 128 : 3 * kPPart;
  // S, O double buffered, in all a power of two
  static constexpr int kTmemCols = 2 * (NP + kOCols) <= 64 ? 64 : 2 * (NP + kOCols) <= 128 ? 128 : 256;
  static constexpr int kK = 0;
  static constexpr int kV = kK + kKStages * kTile;
  static constexpr int kQ = kV + kVStages * kTile;
  static constexpr int kP = kQ + kQBuf * kQBytes;
  static constexpr int kBarCount = 32;
  static constexpr int kBars = kP + kPBuf * kPBytes;
  static constexpr int kInfo = kBars + kBarCount * 8;               // [kInfoRing][3] int4
  static constexpr int kQScale = kInfo + kInfoRing * 48;            // [kQScaleRing][NR]
  static constexpr int kRed = kQScale + kQScaleRing * NR * 4;       // [4][NP]: row maxima by warp, or sums at the end
  static constexpr int kM = kRed + 4 * NP * 4;                      // [NP] running maxima
  static constexpr int kNegM = kM + NP * 4;                         // [NP] kBase - maximum
  static constexpr int kAlpha = kNegM + NP * 4;                     // [NP]
  static constexpr int kRowInv = kAlpha + NP * 4;                   // [NP] 1 / sum
  static constexpr int kStart = (kRowInv + NP * 4 + 15) / 16 * 16;  // Start
  static constexpr int kPending = kStart + 64;                      // [2] Pending
  static constexpr int kScan = kPending + 2 * 24;                   // [8] int64
  static constexpr int kTmem = kScan + 8 * 8;
  static constexpr int kAbort = kTmem + 4;
  static constexpr int kEnd = kAbort + 4;
  static constexpr int kBytes = kEnd + 1024;                        // + slack for 1024-byte alignment
};
static_assert(Cfg8<16>::kBytes <= 115712 && Cfg8<32>::kBytes <= 115712 && Cfg8<40>::kBytes <= 115712,
              "two CTAs per SM");

enum {
  B_KFULL = 0, B_KEMPTY = 3, B_VFULL = 6, B_VEMPTY = 8, B_SFULL = 10, B_SEMPTY = 12, B_PFULL = 14, B_OFULL = 16,
  B_QFULL = 18, B_QEMPTY = 20, B_INFO = 22, B_KSTART = 30
};

// The f8f6f4 instruction descriptor: float32 accumulator, A e4m3, B e4m3 (q) or e5m2 (weights).
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

// Two floats to two packed e4m3 values, the first in the low byte (nearest even, saturating).
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 unpack_e4m3(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xFFFFu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// A pair of float16 numbers to the nearest ones of three significant bits (half up in magnitude; subnormal ones to
// multiples of 2^-16): their upper bytes as e5m2.  No carry leaves a number: magnitudes are at most 2^15.
__device__ __forceinline__ uint32_t round_e5m2(uint32_t h2) { return (h2 + 0x00800080u) & 0xFF00FF00u; }
__device__ __forceinline__ uint32_t sub_h2(uint32_t a, uint32_t b) {
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}

struct Shape8 {
  int n, L, q0;
};

__device__ __forceinline__ Shape8 shape_of(const Fp8DecodeParams& p, int b) {
  Shape8 s;
  if (p.cu_q != nullptr) {
    const int a = __ldg(p.cu_q + b);
    s.n = max(__ldg(p.cu_q + b + 1) - a, 0);
    if (s.n > p.longest || s.n < p.shortest) s.n = 0;   // (another kernel's)
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

// Calls f(first piece, count, tiles) for the runs of pieces of equal tile count of a sequence, in order, until it returns
// true.  (By tiles, not by pieces: a prompt of 16,384 has 2048 pieces but 128 tile counts.)
template <class F>
__device__ __forceinline__ void piece_runs(const Fp8DecodeParams& p, int n, int L, F&& f) {
  const int m = p.max_n, full = n / m, before = L - n;   // piece i < full ends at key before + (i + 1) m
  int i = before + m >= 1 ? 1 : -before / m + 1;         // (1-based) the first with a key
#pragma unroll 1
  while (i <= full) {
    const int t = (before + m * i + 127) >> 7;
    const int last = min(full, (128 * t - before) / m);
    if (f(i - 1, last - i + 1, t)) return;
    i = last + 1;
  }
  const int rest = n - full * m;
  if (rest > 0 && L > 0) f(full, 1, tiles_of(L));
}

// Where a CTA starts.
struct Start {
  long long segpos;   // cost position of the first segment
  long long x0, x1;   // the CTA's share of positions
  long long per;
  int b, piece, g, j; // (g: the head set)
  int any, unused[3];
};
static_assert(sizeof(Start) == 64, "Start");

// The tiles of one CTA in order.  Every lane of the warp holds the same state.  Tile j of a segment at segpos sits at
// position segpos + kSegCost + j; a CTA owns the tiles whose positions are in [x0, x1).  Positions are kept
// relative to x0.
struct Walk {
  int rel, span;      // segpos - x0, x1 - x0
  int b, piece, g, j;
  int n, L, q0;       // the sequence
  int np, Lp, nt;     // the piece: queries, keys its last query sees, tiles
  bool fresh;         // the first tile of this CTA's share
  bool valid;
  int ahead, ahead_n, ahead_L, ahead_q0;   // sequences ahead .. ahead + 31, one per lane

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
    ahead = -64;
    valid = s.any != 0;
    if (valid) {
      rel = static_cast<int>(s.segpos - s.x0);
      span = static_cast<int>(s.x1 - s.x0);
      b = s.b;
      piece = s.piece;
      g = s.g;
      j = s.j;
      load_seq(p);
      set_piece(p);
      valid = rel + kSegCost + j < span;
    }
    fresh = valid;
  }
  // Whether a sequence has a piece with keys.
  __device__ __forceinline__ bool has_piece(const Fp8DecodeParams& p, int n_, int L_) const {
    const int full = n_ / p.max_n;
    return (full > 0 && L_ - n_ + full * p.max_n > 0) || (n_ > full * p.max_n && L_ > 0);
  }
  // The next segment (all lanes of the warp together).
  __device__ __forceinline__ void advance(const Fp8DecodeParams& p) {
    rel += nt + kSegCost;
    j = 0;
    valid = rel + kSegCost < span;
    if (!valid || ++g < p.num_kv_heads / p.head_set) return;
    g = 0;
    do {
      ++piece;
      if (piece * p.max_n >= n) {
        // the next sequence that has one: 32 at a time, read once
        const int lane = threadIdx.x & 31;
        uint32_t vote = 0;
        int from = b + 1;
        while (true) {
          if (from < ahead || from >= ahead + 32) {
            ahead = from;
            ahead_n = ahead_L = ahead_q0 = 0;
            if (from + lane < p.num_seqs) {
              const Shape8 s = shape_of(p, from + lane);
              ahead_n = s.n;
              ahead_L = s.L;
              ahead_q0 = s.q0;
            }
          }
          vote = __ballot_sync(kFull, ahead + lane >= from && has_piece(p, ahead_n, ahead_L));
          if (vote != 0 || ahead + 32 >= p.num_seqs) break;
          from = ahead + 32;
        }
        if (vote == 0) {
          valid = false;
          return;
        }
        const int src = __ffs(vote) - 1;
        b = ahead + src;
        n = __shfl_sync(kFull, ahead_n, src);
        L = __shfl_sync(kFull, ahead_L, src);
        q0 = __shfl_sync(kFull, ahead_q0, src);
        piece = 0;
      }
      set_piece(p);
    } while (nt == 0);
  }
  __device__ __forceinline__ void next_segment(const Fp8DecodeParams& p) {
    fresh = false;
    advance(p);
  }
  __device__ __forceinline__ void next_tile(const Fp8DecodeParams& p) {
    fresh = false;
    if (++j < nt) {
      valid = rel + kSegCost + j < span;
    } else {
      advance(p);
    }
  }
};

// A cut segment that this CTA has to merge (c1 < 0: none).
struct Pending {
  int c0, c1, rows;
  int64_t out_base;
};

// One row of q (four bf16 values per lane) as its two e4m3 parts in the swizzled operand at qs, and its scale.
__device__ __forceinline__ void put_q_row(uint2 x, uint8_t* qs, int half_bytes, float* scales, int r, int lane) {
  uint32_t mx = max(max(x.x & 0x7FFFu, (x.x >> 16) & 0x7FFFu), max(x.y & 0x7FFFu, (x.y >> 16) & 0x7FFFu));
  mx = __reduce_max_sync(kFull, mx);
  // the row's largest value to [2^7, 2^8): times 2^(134 - E); NaN or infinity anywhere makes the row NaN
  const int E = max(static_cast<int>(mx >> 7), 8);
  const float f = __uint_as_float(static_cast<uint32_t>(261 - min(E, 254)) << 23);
  const float back = E == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float(static_cast<uint32_t>(E - 7) << 23);
  const float2 a01 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x.x));
  const float2 a23 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x.y));
  const float v0 = a01.x * f, v1 = a01.y * f, v2 = a23.x * f, v3 = a23.y * f;
  const uint32_t h01 = pack_e4m3(v0, v1), h23 = pack_e4m3(v2, v3);
  const float2 u01 = unpack_e4m3(h01), u23 = unpack_e4m3(h23);
  const uint32_t l01 = pack_e4m3(v0 - u01.x, v1 - u01.y), l23 = pack_e4m3(v2 - u23.x, v3 - u23.y);
  uint8_t* at = qs + sw128_offset(r, lane >> 2) + (lane & 3) * 4;
  *reinterpret_cast<uint32_t*>(at) = h01 | (h23 << 16);
  *reinterpret_cast<uint32_t*>(at + half_bytes) = l01 | (l23 << 16);
  if (lane == 0) scales[r] = back;
}

template <int HR>
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, float* v) {
  if constexpr (HR == 8) {
    tmem_ld8(taddr, v);
  } else {
    static_assert(HR == 16, "rows per TMEM load");
    tmem_ld16(taddr, v);
  }
}

// Column reduction of HR values per thread within one warp into dst[0..HR), sixteen columns at a time (the butterfly
// works on a copy: few registers next to the rows).
template <int HR, bool kMax>
__device__ __forceinline__ void warp_rows(const float* x, float* dst, int lane) {
#pragma unroll
  for (int c = 0; c + 16 <= HR; c += 16) warp_columns<16, kMax>(x + c, dst + c, lane);
  if constexpr (HR % 16 != 0) warp_columns<8, kMax>(x + HR / 16 * 16, dst + HR / 16 * 16, lane);
}

template <int NR>
__global__ void __launch_bounds__(Cfg8<NR>::kThreads, 2)
paged_decode_fp8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const Fp8DecodeParams p) {
  using C = Cfg8<NR>;
  constexpr int NP = C::NP;
  extern __shared__ uint8_t smem_raw[];
  // aligned by an offset, not through an integer: the compiler keeps knowing that these are shared-memory addresses
  // (32-bit, LDS / STS) instead of generic ones
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBars);
  int4* info = reinterpret_cast<int4*>(smem + C::kInfo);
  float* qscale = reinterpret_cast<float*>(smem + C::kQScale);
  float* red = reinterpret_cast<float*>(smem + C::kRed);
  float* m_s = reinterpret_cast<float*>(smem + C::kM);
  float* negm_s = reinterpret_cast<float*>(smem + C::kNegM);
  float* alpha_s = reinterpret_cast<float*>(smem + C::kAlpha);
  float* row_inv = reinterpret_cast<float*>(smem + C::kRowInv);
  Start* start = reinterpret_cast<Start*>(smem + C::kStart);
  Pending* pending = reinterpret_cast<Pending*>(smem + C::kPending);
  long long* scan = reinterpret_cast<long long*>(smem + C::kScan);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kTmem);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + C::kAbort);

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int KVH = p.num_kv_heads;
  const int G = p.group;
  const int sets = KVH / p.head_set;                            // the walk's head sets
  const int teams = static_cast<int>(gridDim.x) / p.head_set;   // CTAs that share the work of one head of each set
  const int member = blockIdx.x % p.head_set, team = blockIdx.x / p.head_set;
  const int vcta = member * teams + team;   // the pieces of a cut segment are consecutive in this numbering

  if (tid == 0) {
    for (int s = 0; s < C::kKStages; ++s) {
      mbar_init(&bars[B_KFULL + s], 1);
      mbar_init(&bars[B_KEMPTY + s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars[B_VFULL + s], 1);
      mbar_init(&bars[B_VEMPTY + s], 1);
      mbar_init(&bars[B_SFULL + s], 1);
      mbar_init(&bars[B_SEMPTY + s], 128);
      mbar_init(&bars[B_PFULL + s], 128);
      mbar_init(&bars[B_OFULL + s], 1);
      mbar_init(&bars[B_QFULL + s], 1);
      mbar_init(&bars[B_QEMPTY + s], 1);
    }
    for (int i = 0; i < kInfoRing; ++i) mbar_init(&bars[B_INFO + i], 1);
    mbar_init(&bars[B_KSTART], 1);
    *abort = 0;
    start->any = 0;
    for (int i = 0; i < 2; ++i) pending[i].c1 = -1;
    fence_barrier_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // With a programmatic dependency on the prefill plan: wait for it (and what came before it).  Then let the call's next
  // kernel start its blocks where this grid's leave.
  if (p.wait_primary) griddep_wait();
  if (tid == 0) griddep_launch_dependents();
  // ------------------------------------------------------------ the work split
  // Two scans over the sequences' costs: the total (hence each CTA's share), then the sequence that holds this CTA's
  // first position.  Batches of up to kThreads sequences keep the first scan's values in registers.
  {
    constexpr int T = C::kThreads, W = T / 32;
    long long total = 0, x0 = 0, per = 0, before = 0, mine = 0, excl = 0, sum = 0;
    int n = 0, L = 0;
    const bool single = p.num_seqs <= T;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
      for (int base = 0; base < p.num_seqs; base += T) {
        if (pass == 0 || !single) {
          n = L = 0;
          if (base + tid < p.num_seqs) {
            const Shape8 s = shape_of(p, base + tid);
            n = s.n;
            L = s.L;
          }
          mine = 0;
          piece_runs(p, n, L, [&](int, int count, int nt) {
            mine += static_cast<long long>(sets) * count * (nt + kSegCost);
            return false;
          });
          long long x = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(kFull, x, o);
            if (lane >= o) x += y;
          }
          if (lane == 31) scan[warp] = x;
          excl = x - mine;
          __syncthreads();
          sum = 0;
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const long long v = scan[w];
            excl += w < warp ? v : 0;
            sum += v;
          }
          __syncthreads();
        }
        if (pass == 0) {
          total += sum;
          continue;
        }
        // the thread whose sequence holds position x0
        const long long lo = before + excl;
        before += sum;
        if (mine > 0 && x0 >= lo && x0 < lo + mine) {
          long long rem = x0 - lo;
          piece_runs(p, n, L, [&](int first, int count, int nt) {
            const int seg = nt + kSegCost;
            const long long run = static_cast<long long>(sets) * count * seg;
            if (rem >= run) {
              rem -= run;
              return false;
            }
            const int i = static_cast<int>(rem / (sets * seg));
            const int r = static_cast<int>(rem) - i * sets * seg, g = r / seg, o = r - g * seg;
            start->segpos = x0 - o;
            start->b = base + tid;
            start->piece = first + i;
            start->g = g;
            start->j = max(0, o - kSegCost);
            start->any = 1;
            return true;
          });
        }
      }
      if (pass == 0) {
        per = total > 0 ? (total + teams - 1) / teams : 1;
        x0 = per * team;
        if (tid == 0) {
          start->x0 = x0;
          start->x1 = min(x0 + per, total);
          start->per = per;
        }
      }
    }
    __syncthreads();
  }
  // query rows in pieces without a key (batch padding) belong to no tile: zero, written by CTA b % grid
  for (int b = blockIdx.x; b < p.num_seqs; b += gridDim.x) {
    const Shape8 ss = shape_of(p, b);
    const int rows = ss.L >= ss.n ? 0 : ss.L <= 0 ? ss.n : (ss.n - ss.L) / p.max_n * p.max_n;
#pragma unroll 1
    for (int i = 0; i < rows; ++i)
#pragma unroll 1
      for (int c = tid; c < p.num_heads * (kHeadDim / 8); c += C::kThreads)
        reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(ss.q0 + i) * p.out_row_stride)[c] =
            make_uint4(0u, 0u, 0u, 0u);
  }
  Walk w;
  w.begin(p, *start);
  // A grid that did not wait for the one before it must not complete first: one block waits at its end.
  const bool holds = p.pdl && !p.wait_primary && blockIdx.x == 0;
  if (!w.valid) {         // nothing for this CTA: no TMEM, no pipeline
    if (holds) griddep_wait();
    return;
  }
  if (warp < 4) {
  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------ K (warp 0) and V (warp 3) producers
    // They leave when their tiles are issued; the other warps wait for every tile, so the block outlives the copies.
    const bool is_k = warp == 0;
    const CUtensorMap* tm = is_k ? &tm_k : &tm_v;
    uint8_t* ring = smem + (is_k ? C::kK : C::kV);
    uint64_t* full = bars + (is_k ? B_KFULL : B_VFULL);
    uint64_t* empty = bars + (is_k ? B_KEMPTY : B_VEMPTY);
    const int stages = is_k ? C::kKStages : C::kVStages;
    bool stop = !is_k && !mbar_wait_warp(&bars[B_KSTART], 0, abort);
    for (int jj = 0; w.valid && !stop;) {
      // descriptors of the next tiles, one per lane (their block-table reads overlap); a short first round, so that
      // the first copies start early
      const int round = jj == 0 ? 4 : 32;
      int g = 0, j = 0, flags = 0, np = 0, Lp = 0, qrow = 0, nt = 0, b = 0, rel = 0, cnt = 0;
      for (; cnt < round && w.valid; ++cnt) {
        const bool first = w.fresh || w.j == 0;
        const bool seg_end = w.j == w.nt - 1;
        if (lane == cnt) {
          g = w.g * p.head_set + member;
          j = w.j;
          np = w.np;
          Lp = w.Lp;
          nt = w.nt;
          b = w.b;
          qrow = w.q0 + w.piece * p.max_n;
          rel = w.rel;
        }
        w.next_tile(p);
        // 1: first, 2: last tile of this CTA's part of a segment, 4: of the CTA
        if (lane == cnt) flags = (first ? 1 : 0) | (seg_end || !w.valid || w.fresh ? 2 : 0) | (!w.valid ? 4 : 0);
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
        int ji = 0, fi = 0, ni = 0, Li = 0, qi = 0, ti = 0, ri = 0;
        if (is_k) {
          ji = __shfl_sync(kFull, j, i);
          fi = __shfl_sync(kFull, flags, i);
          ni = __shfl_sync(kFull, np, i);
          Li = __shfl_sync(kFull, Lp, i);
          qi = __shfl_sync(kFull, qrow, i);
          ti = __shfl_sync(kFull, nt, i);
          ri = __shfl_sync(kFull, rel, i);
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
            info[3 * e + 2] = make_int4(fi, ri, 0, 0);
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
  // the other warps meet on named barrier 3 once TMEM is there, and again at the end
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  named_bar_sync(3, C::kThreads - 64);
  if (warp == 1) {
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // ------------------------------------------------------------ UMMA issuer (the warp waits, an elected lane issues)
    const uint64_t q_desc0 = umma_desc_sw128(smem_u32(smem + C::kQ), 16, 1024);
    const uint64_t k_desc0 = umma_desc_sw128(smem_u32(smem + C::kK), 16, 1024);
    const uint64_t v_desc0 = umma_desc_sw128(smem_u32(smem + C::kV), kTile, 1024);
    const uint64_t p_desc0 = umma_desc_noswz(smem_u32(smem + C::kP), 128, 2048);
    int qseg = 0, oseg = 0;
    bool qk_done = false;
    // order: QK(0), QK(1), PV(0), QK(2), PV(1), ...
#pragma unroll 1
    for (int it = 0;; ++it) {
      if (!qk_done) {
        const int st = it % C::kKStages, e = it % kInfoRing, buf = it & 1;
        if (!mbar_wait_warp(&bars[B_INFO + e], (it / kInfoRing) & 1, abort)) break;
        const int flags = info[3 * e + 2].x;
        const uint32_t idesc = idesc_f8(min(NP, mma_width(info[3 * e + 1].x * G)), false, false);
        const int qb = qseg % C::kQBuf;
        if ((flags & 1) && !mbar_wait_warp(&bars[B_QFULL + qb], (qseg / C::kQBuf) & 1, abort)) break;
        if (!mbar_wait_warp(&bars[B_KFULL + st], (it / C::kKStages) & 1, abort)) break;
        if (!mbar_wait_warp(&bars[B_SEMPTY + buf], ((it >> 1) & 1) ^ 1, abort)) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a = k_desc0 + ((st * kTile) >> 4);
          const uint64_t b = q_desc0 + ((qb * C::kQBytes) >> 4);
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < 4; ++k)   // 32 dims a step: +32 bytes inside the 128-byte rows
              umma_f8_ss(tmem + buf * NP, a + 2 * k, b + ((part * C::kQHalf) >> 4) + 2 * k, idesc, part + k > 0);
          umma_commit(&bars[B_SFULL + buf]);
          umma_commit(&bars[B_KEMPTY + st]);
          if (flags & 2) umma_commit(&bars[B_QEMPTY + qb]);
        }
        __syncwarp();
        if (flags & 2) ++qseg;
        qk_done = flags & 4;
      }
      if (it == 0) continue;
      const int pv = it - 1;
      const int st = pv % C::kVStages, pb = pv & 1, e = pv % kInfoRing;
      if (!mbar_wait_warp(&bars[B_PFULL + pb], (pv >> 1) & 1, abort)) break;
      if (!mbar_wait_warp(&bars[B_VFULL + st], (pv / C::kVStages) & 1, abort)) break;
      const int flags = info[3 * e + 2].x;
      if ((flags & 1) && pv > 0) oseg ^= 1;
      const int width = min(NP, mma_width(info[3 * e + 1].x * G));
      const uint32_t idesc = idesc_f8(C::kOParts == 3 ? C::kOCols : width, true, true);
      tc_fence_after();
      if (elect_one()) {
        const uint64_t a = v_desc0 + ((st * kTile) >> 4);
        const uint64_t b = p_desc0 + ((pv % C::kPBuf * C::kPBytes) >> 4);
        const uint32_t d = tmem + 2 * NP + oseg * C::kOCols;
        const uint32_t fresh = (flags & 1) ? 0u : 1u;
#pragma unroll
        for (int part = 0; part < (C::kOParts == 3 ? 1 : 3); ++part)
#pragma unroll
          for (int k = 0; k < 4; ++k)   // 32 tokens a step: four groups of 8 (V: 1024 bytes each, P^T: 128)
            umma_f8_ss(d, a + 256 * k, b + ((part * C::kPPart) >> 4) + 32 * k, idesc, part + k > 0 ? 1u : fresh);
        umma_commit(&bars[B_OFULL + pb]);
        umma_commit(&bars[B_VEMPTY + st]);
      }
      __syncwarp();
      if (flags & 4) break;
    }
  } else {
    // ------------------------------------------------------------ Q loader: bf16 rows -> two e4m3 parts + row scale
    // (the softmax warps, idle until the first scores, put the first segment's rows)
    w.next_segment(p);
    for (int qi = 1; w.valid; ++qi) {
      const int qb = qi % C::kQBuf;
      if (!mbar_wait_warp(&bars[B_QEMPTY + qb], ((qi / C::kQBuf) & 1) ^ 1, abort)) break;
      const int R = w.np * G;
      uint8_t* qs = smem + C::kQ + qb * C::kQBytes;
      float* sc = qscale + (qi % kQScaleRing) * NR;
      const __nv_bfloat16* base = p.q + static_cast<int64_t>(w.q0 + w.piece * p.max_n) * p.q_row_stride +
                                  static_cast<int64_t>(w.g * p.head_set + member) * G * kHeadDim + lane * 4;
      // a few rows at a time, the next ones' loads in flight.  Rows past R stay as they are: whatever the products make
      // of them ends in columns that nobody reads.
      constexpr int kBatch = NR <= 16 ? 4 : 8;
      uint2 next[kBatch];
      int fi = 0, fh = 0;   // query and head of the next row to fetch
      auto fetch = [&](int r0) {
#pragma unroll
        for (int v = 0; v < kBatch; ++v) {
          next[v] = make_uint2(0u, 0u);
          if (r0 + v < R)
            next[v] = __ldg(reinterpret_cast<const uint2*>(base + fi * p.q_row_stride + fh * kHeadDim));
          if (++fh == G) {
            fh = 0;
            ++fi;
          }
        }
      };
      fetch(0);
#pragma unroll 1
      for (int r0 = 0; r0 < R; r0 += kBatch) {
        uint2 x[kBatch];
#pragma unroll
        for (int v = 0; v < kBatch; ++v) x[v] = next[v];
        fetch(r0 + kBatch);
#pragma unroll
        for (int v = 0; v < kBatch; ++v) {
          const int r = r0 + v;
          put_q_row(x[v], qs, C::kQHalf, sc, r, lane);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[B_QFULL + qb]);
      w.next_segment(p);
    }
  }
  } else {
    named_bar_sync(3, C::kThreads - 64);
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // ------------------------------------------------------------ softmax
    // Every wait is warp-uniform and every named barrier that can end the loop ORs "gave up" over the group's warps, so
    // they leave together.
    const int ct = tid - kConsumerBase;       // TMEM lane: token ct of S^T, dim ct of O^T
    const int wq = ct >> 5;
    constexpr uint32_t bar_id = 1;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    bool alive = true, done = false;
    float ks_next = 0.f, vs_next = 1.f;   // the next tile's scales of this thread's token

    // A piece of a cut segment is done (its rows written): take a ticket.  The CTA that brings
    // it to the number of pieces puts the counter back to zero and merges them all; a CTA has at most two cut segments,
    // so it notes them and merges after its last tile, out of the loop's registers.
    constexpr int kSlots = 2;   // pieces a CTA may leave
    auto arrive_piece = [&](int p_first, int p_last, int R, int64_t out_base) {
      named_bar_sync(bar_id, 128);
      if (ct == 0) {
        // the CTAs of the segment's first and last tile
        const Start& st = *start;
        const int c0 = member * teams + static_cast<int>((st.x0 + p_first) / st.per);
        const int c1 = member * teams + static_cast<int>((st.x0 + p_last) / st.per);
        int32_t* ticket = p.counters + kTicketStride * c0;
        __threadfence();   // release: the group's partial rows before the ticket
        if (atomicAdd(ticket, 1) == c1 - c0) {
          *ticket = 0;
          Pending* d = pending;
          while (d->c1 >= 0) ++d;   // (at most one for each of the CTA's cut segments)
          d->c0 = c0;
          d->c1 = c1;
          d->rows = R;
          d->out_base = out_base;
        }
      }
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

    {
      // the first segment's q, the four warps' rows apart: the Q loader alone took 3 us longer on 20 rows
      const int rows = w.np * G;
      const __nv_bfloat16* base = p.q + static_cast<int64_t>(w.q0 + w.piece * p.max_n) * p.q_row_stride +
                                  static_cast<int64_t>(w.g * p.head_set + member) * G * kHeadDim + lane * 4;
      constexpr int kOwn = NR / 4;
      uint2 x[kOwn];
#pragma unroll
      for (int v = 0; v < kOwn; ++v) {
        const int r = wq + 4 * v, i = r / G;
        x[v] = make_uint2(0u, 0u);
        if (r < rows) x[v] = __ldg(reinterpret_cast<const uint2*>(base + i * p.q_row_stride + (r - i * G) * kHeadDim));
      }
#pragma unroll
      for (int v = 0; v < kOwn; ++v)
        if (wq + 4 * v < rows) put_q_row(x[v], smem + C::kQ, C::kQHalf, qscale, wq + 4 * v, lane);
      fence_proxy_async_smem();
      named_bar_sync(bar_id, 128);
      if (ct == 0) mbar_arrive(&bars[B_QFULL]);
    }
    alive = mbar_wait_warp(&bars[B_INFO], 0, abort);
    if (alive) load_scales(info[0], info[1]);
    int jj = 0;   // tile of this CTA
    for (int seg = 0; !done; ++seg) {
      // one segment
      const uint32_t t_o = t_lane + 2 * NP + (seg & 1) * C::kOCols;   // O accumulator, by segment parity
      const float* qs = qscale + (seg % kQScaleRing) * NR;
      [&] {
        constexpr int HR = NR;
        constexpr int kChunk = HR % 16 == 0 ? 16 : 8;   // rows per TMEM load
        float l[HR], s[HR];
#pragma unroll
        for (int r = 0; r < HR; ++r) l[r] = 0.f;
        for (;; ++jj) {
          const int st = jj % C::kVStages;
          const int buf = jj & 1;
          const int e = jj % kInfoRing;
          alive = alive && mbar_wait_warp(&bars[B_INFO + e], (jj / kInfoRing) & 1, abort);
          int tok0 = 0, n = 0, L = 0, flags = 7;
          if (alive) {
            tok0 = info[3 * e].x;
            const int2 nl = *reinterpret_cast<const int2*>(&info[3 * e + 1]);
            n = nl.x;
            L = nl.y;
            flags = info[3 * e + 2].x;
          }
          const bool first = flags & 1, last = flags & 2;
          const int R = n * G;
          const int tok = tok0 + ct;
          // this token's factors; the next tile's scales are on their way while this tile is worked on
          const bool live = tok < L;
          const float vs = fminf(fmaxf(vs_next, 9.094947e-13f), 1.0995116e12f);   // 2^-40 .. 2^40
          const float a = live ? ks_next * p.scale_log2 : 0.f;
          const float lv = __log2f(vs);
          const float ivs = live ? __frcp_rn(vs) : 0.f;
          if (alive && !(flags & 4)) {
            const int e1 = (jj + 1) % kInfoRing;
            alive = mbar_wait_warp(&bars[B_INFO + e1], ((jj + 1) / kInfoRing) & 1, abort);
            if (alive) load_scales(info[3 * e1], info[3 * e1 + 1]);
          }
          alive = alive && mbar_wait_warp(&bars[B_SFULL + buf], (jj >> 1) & 1, abort);
          const bool open_tile = tok0 + 127 <= L - n;   // every row sees every token
          // s <- score * scale of q * scale of k + log2 of v's scale (+ add[row]); -inf where masked: row r = i * G + h
          // sees the token iff r >= G * (token - (L - n))
          // (a few rows at a time, so that the rows' factors in shared memory are not all fetched ahead)
          const int rmin = open_tile ? 0 : !live ? NP : max(tok - (L - n), 0) * G;
          auto scores = [&](const float* add) {
#pragma unroll
            for (int c = 0; c < HR; c += kChunk) {
              tmem_ld_rows<kChunk>(t_lane + buf * NP + c, s + c);
              const float2 a2 = make_float2(a, a), lv2 = make_float2(lv, lv);
#pragma unroll
              for (int r = c; r < c + kChunk; r += 2) {
                const float2 q2 = *reinterpret_cast<const float2*>(qs + r);
                const float2 o2 = add != nullptr ? fadd2(*reinterpret_cast<const float2*>(add + r), lv2) : lv2;
                const float2 y = ffma2(fmul2(make_float2(s[r], s[r + 1]), a2), q2, o2);
                s[r] = y.x;
                s[r + 1] = y.y;
              }
              if (!open_tile) {
#pragma unroll
                for (int r = c; r < c + kChunk; ++r) s[r] = (r >= rmin && r < R) ? s[r] : kNegInf;
              }
            }
          };
          bool need = first;
          if (alive) tc_fence_after();
          if (alive && !first) {
            scores(negm_s);
            float top = 0.f;
#pragma unroll
            for (int r = 0; r < HR; ++r) {
              s[r] = fast_exp2(s[r]);
              top = fmaxf(top, s[r]);
            }
            need = top > kWeightMax;
          }
          // one vote per tile; a warp that gave up votes too and is caught by the second vote
          const bool rescale = named_bar_any(bar_id, 128, need || !alive);
          if (rescale) {
            if (named_bar_any(bar_id, 128, !alive)) {
              done = true;
              return;
            }
            scores(nullptr);
            warp_rows<HR, true>(s, red + wq * NP, lane);
            named_bar_sync(bar_id, 128);
            if (ct < HR) {
              float mn = 0.f, neg = kNegInf, alpha = 1.f;   // rows past R: no weight
              if (ct < R) {
                const float tm = fmaxf(fmaxf(red[ct], red[NP + ct]), fmaxf(red[2 * NP + ct], red[3 * NP + ct]));
                const float mo = first ? kNegInf : m_s[ct];
                mn = (first || tm > mo + kSlack) ? fmaxf(mo, tm) : mo;
                neg = mn == kNegInf ? 0.f : kBase - mn;   // a row that has seen no key yet: its scores are -inf
                alpha = (mo == kNegInf || mn == mo) ? 1.f : fast_exp2(mo - mn);
              }
              m_s[ct] = mn;
              negm_s[ct] = neg;
              alpha_s[ct] = alpha;
            }
            named_bar_sync(bar_id, 128);
#pragma unroll
            for (int c = 0; c < HR; c += 8) {
              asm volatile("" ::: "memory");   // (eight rows' factors at a time)
#pragma unroll
              for (int r = c; r < c + 8; ++r) {
                s[r] = fast_exp2(s[r] + negm_s[r]);
                l[r] *= alpha_s[r];
              }
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
          // some row maxima moved: the O rows scale once PV(jj - 1) has added onto them
          if (rescale && !first) {
            alive = alive && mbar_wait_warp(&bars[B_OFULL + (buf ^ 1)], ((jj - 1) >> 1) & 1, abort);
            if (alive) {
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < C::kOParts * C::kOStep; k += C::kOStep)
                for (int c = 0; c < R; c += 8) {
                  float ot[8];
                  tmem_ld8(t_o + k + c, ot);
#pragma unroll
                  for (int i = 0; i < 8; ++i) ot[i] *= alpha_s[c + i];
                  tmem_st8(t_o + k + c, ot);
                }
              tc_fence_before();
            }
          }
          // P(jj) goes where PV(jj - kPBuf) read
          if (jj >= C::kPBuf)
            alive = alive && mbar_wait_warp(&bars[B_OFULL + ((jj - C::kPBuf) & 1)], ((jj - C::kPBuf) >> 1) & 1, abort);
          // rows past the piece's keys may hold anything, NaN too: zero V there, so that no weight of 0 meets it
          if (L - tok0 < kTileTokens) {
            alive = alive && mbar_wait_warp(&bars[B_VFULL + st], (jj / C::kVStages) & 1, abort);
            if (alive && !live) {
              uint4* vrow = reinterpret_cast<uint4*>(smem + C::kV + st * kTile + ct * 128);
#pragma unroll
              for (int c = 0; c < 8; ++c) vrow[c] = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          if (alive) {
            // P^T: the three parts of the weights in float16; 8 rows of token ct are 8 bytes
            uint8_t* pb = smem + C::kP + jj % C::kPBuf * C::kPBytes + ct * 16;
#pragma unroll
            for (int m = 0; m < HR / 8; ++m) {
              uint32_t part[3][2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t x[2], y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const int r = 8 * m + 4 * h + 2 * i;
                  const __half2 w = __floats2half2_rn(s[r], s[r + 1]);
                  x[i] = *reinterpret_cast<const uint32_t*>(&w);
                }
#pragma unroll
                for (int k = 0; k < 3; ++k) {
#pragma unroll
                  for (int i = 0; i < 2; ++i) y[i] = k < 2 ? round_e5m2(x[i]) : x[i] + 0x00800080u;
                  part[k][h] = __byte_perm(y[0], y[1], 0x7531);   // the upper bytes
#pragma unroll
                  for (int i = 0; i < 2; ++i) x[i] = sub_h2(x[i], y[i]);   // (exact; the last one is not used)
                }
              }
              uint8_t* at = pb + (m >> 1) * 2048 + (m & 1) * 8;
#pragma unroll
              for (int k = 0; k < 3; ++k)
                *reinterpret_cast<uint2*>(at + (NR == 8 ? (k >> 1) * 2048 + (k & 1) * 8 : k * C::kPPart)) =
                    make_uint2(part[k][0], part[k][1]);
            }
            fence_proxy_async_smem();
            mbar_arrive(&bars[B_PFULL + buf]);
          }
          if (last) break;   // (a warp that gave up in the middle of a segment is caught by the next tile's vote)
        }
        warp_rows<HR, false>(l, red + wq * NP, lane);
      }();
      if (done) break;
      // ---- the segment's end (tile jj): 1 / sum, and the rows of this CTA's part
      const int e = jj % kInfoRing;
      alive = alive && mbar_wait_warp(&bars[B_OFULL + (jj & 1)], (jj >> 1) & 1, abort);
      if (named_bar_any(bar_id, 128, !alive)) break;
      const int4 ib = info[3 * e + 1], ic = info[3 * e + 2];
      const int seg_g = info[3 * e].w;
      const int R = ib.x * G;
      // positions of the segment's first and last tile relative to this CTA's share: a segment inside it is finished
      // here, one that is cut leaves a piece
      const int span = static_cast<int>(start->x1 - start->x0);
      const int p_first = ic.y + kSegCost, p_last = p_first + ib.w - 1;
      const bool complete = p_first >= 0 && p_last < span;
      const int slot = kSlots * vcta + (p_first < 0 ? 0 : 1);   // (of a piece)
      const int64_t out_base = ib.z * p.out_row_stride + static_cast<int64_t>(seg_g) * G * kHeadDim;
      if (ct < R) {
        const float lt = red[ct] + red[NP + ct] + red[2 * NP + ct] + red[3 * NP + ct];
        row_inv[ct] = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);   // a NaN sum stays NaN
        if (!complete) p.part_lse[slot * NP + ct] = lt == 0.f ? kNegInf : m_s[ct] + __log2f(lt);
      }
      named_bar_sync(bar_id, 128);
      tc_fence_after();
      // the accumulated O, eight rows at a time; lane = dim
      __nv_bfloat16* o = p.out + out_base + ct;
      float* part = p.part_o + static_cast<int64_t>(slot) * NP * kHeadDim + ct;
      int h = 0;
#pragma unroll 1
      for (int c = 0; c < R; c += 8) {
        float ot[8];
        tmem_ld8(t_o + c, ot);
#pragma unroll
        for (int k = 1; k < C::kOParts; ++k) {
          float more[8];
          tmem_ld8(t_o + k * C::kOStep + c, more);
#pragma unroll
          for (int i = 0; i < 8; ++i) ot[i] += more[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 inv = *reinterpret_cast<const float4*>(row_inv + c + i);
          ot[i] *= inv.x;
          ot[i + 1] *= inv.y;
          ot[i + 2] *= inv.z;
          ot[i + 3] *= inv.w;
        }
        if (complete) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (c + i < R) *o = __float2bfloat16_rn(ot[i]);
            if (++h == G) {
              h = 0;
              o += p.out_row_stride - (G - 1) * kHeadDim;
            } else {
              o += kHeadDim;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < R) part[(c + i) * kHeadDim] = ot[i];
        }
      }
      tc_fence_before();
      if (!complete) arrive_piece(p_first, p_last, R, out_base);
      done = ic.x & 4;
      ++jj;
    }
    // the pieces this group was the last to finish
    const bool gave_up = named_bar_any(bar_id, 128, !alive);
    __threadfence();   // acquire: the other pieces' rows
#pragma unroll 1
    for (int i = 0; i < kSlots && !gave_up; ++i) {
      const Pending d = pending[i];
      if (d.c1 < 0) continue;
      // the piece of CTA c lies in its second slot where the segment begins (c0), in its first slot behind that
      const int pieces = d.c1 - d.c0 + 1;
      float* table = reinterpret_cast<float*>(smem + C::kK);   // [rows][pieces] weights; the rings are idle
      auto piece_row = [&](int c, int r) {
        return static_cast<int64_t>(kSlots * (d.c0 + c) + (c == 0 ? 1 : 0)) * NP + r;
      };
      // weights 2^(lse - max) / sum of pieces that saw a key; partials come from other CTAs: past L1
      if (pieces <= 16) {   // (a thread per row)
        if (ct < d.rows) {
          float mx = kNegInf, den = 0.f;
#pragma unroll 8
          for (int c = 0; c < pieces; ++c) {
            const float v = __ldcg(p.part_lse + piece_row(c, ct));
            table[ct * pieces + c] = v;
            mx = fmaxf(mx, v);
          }
#pragma unroll 1
          for (int c = 0; c < pieces; ++c) {
            const float v = table[ct * pieces + c];
            const float e = v == kNegInf ? 0.f : fast_exp2(v - mx);
            table[ct * pieces + c] = e;
            den += e;
          }
          const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll 1
          for (int c = 0; c < pieces; ++c) table[ct * pieces + c] *= inv;
        }
      } else {              // (a warp per row)
#pragma unroll 1
        for (int r = wq; r < d.rows; r += 4) {
          float mx = kNegInf, den = 0.f;
#pragma unroll 1
          for (int c = lane; c < pieces; c += 32) {
            const float v = __ldcg(p.part_lse + piece_row(c, r));
            table[r * pieces + c] = v;
            mx = fmaxf(mx, v);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
#pragma unroll 1
          for (int c = lane; c < pieces; c += 32) {
            const float v = table[r * pieces + c];
            const float e = v == kNegInf ? 0.f : fast_exp2(v - mx);
            table[r * pieces + c] = e;
            den += e;
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(kFull, den, o);
          const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll 1
          for (int c = lane; c < pieces; c += 32) table[r * pieces + c] *= inv;
        }
      }
      named_bar_sync(bar_id, 128);
      // four rows of four dims a thread, their loads together
#pragma unroll 1
      for (int r0 = wq; r0 < d.rows; r0 += 16) {
        float4 acc[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int c = 0; c < pieces; ++c) {
          const float4* src = reinterpret_cast<const float4*>(p.part_o) + piece_row(c, r0) * 32 + lane;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (r0 + 4 * k < d.rows) {
              const float4 v = __ldcg(src + 4 * k * 32);
              const float wgt = table[(r0 + 4 * k) * pieces + c];
              acc[k].x = fmaf(wgt, v.x, acc[k].x);
              acc[k].y = fmaf(wgt, v.y, acc[k].y);
              acc[k].z = fmaf(wgt, v.z, acc[k].z);
              acc[k].w = fmaf(wgt, v.w, acc[k].w);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = r0 + 4 * k;
          if (r < d.rows) {
            const int q = r / G, h = r - q * G;
            *reinterpret_cast<uint2*>(p.out + d.out_base + q * p.out_row_stride + h * kHeadDim + lane * 4) =
                make_uint2(pack_bf16x2(acc[k].x, acc[k].y), pack_bf16x2(acc[k].z, acc[k].w));
          }
        }
      }
      named_bar_sync(bar_id, 128);
    }
  }

  named_bar_sync(3, C::kThreads - 64);
  if (*abort) {
    // a wait gave up: let any copy or MMA still in flight land before the shared memory and TMEM go away
    if (tid == kConsumerBase) atomicOr(&g_error_word, kErrTimeout);
#pragma unroll 1
    for (int i = 0; i < 1000; ++i) sleep_ns(1000);
    named_bar_sync(3, C::kThreads - 64);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, C::kTmemCols);
    if (holds) griddep_wait();
  }
}

template <int NR>
cudaError_t launch8(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const Fp8DecodeParams& p, int grid,
                    cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(paged_decode_fp8_kernel<NR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg8<NR>::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(paged_decode_fp8_kernel<NR>, dim3(grid), dim3(Cfg8<NR>::kThreads), Cfg8<NR>::kBytes, stream,
                       p.pdl != 0, tm_k, tm_v, p);
}

// 8-bit view {128 bytes, heads, rows} of a cache, 128 x 1 x 128 boxes, 128-byte swizzle.
int encode_rows8(CUtensorMap* tm, const void* base, int64_t heads, int64_t rows) {
  cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {128, static_cast<cuuint64_t>(heads) * 128};
  cuuint32_t box[3] = {128, 1, 128};
  return encode_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box);
}

// Softmax rows of the kernel for runs of up to `rows` packed query rows: longer ones are walked in pieces of 40 rows.
int tile_rows(int64_t rows) {
  return rows <= 8 ? 8 : rows >= kMaxRows8 ? kMaxRows8 : static_cast<int>((rows + 7) / 8 * 8);
}

// The kernel for runs of up to max_q queries: one at least (a bound of 0 says nothing about the runs there are), so that a
// tile holds a query's whole group.
int rows_for(int32_t max_q, int group) { return tile_rows(static_cast<int64_t>(std::max(max_q, 1)) * group); }

// Query runs of at least this many tokens take the prefill kernel, which gives each q head 128 rows of its own and costs
// the same for 33 queries as for 128, while here every 40 packed rows are walked anew.  us here and there, with 1, 4 and 8
// q heads per kv head (8 kv heads):
//                                runs of 48                   runs of 64                   runs of 96
//   4 runs over 1000 keys    29/37   42/39   55/57       29/38   47/39   66/58       34/39   56/40   90/60
//   32 runs over 1000 keys   71/60  165/155 311/287      73/61  219/156 406/289     102/62  319/159 618/293
//   8 runs over 8000 keys    96/150 198/278 364/533      98/150 262/279 466/534     133/153 368/284 707/543
// So the bound suits many runs and short contexts; few runs over long contexts would do better here up to 70 tokens (4 q
// heads a kv head) or 96 (one).
constexpr int kMinPrefillRun = 64;

// Queries of the runs that a split call leaves to the kernel of the fewest rows.
int short_run(int group) { return std::max(1, 8 / group); }

// Whether a varlen call runs twice, short runs (up to 8 packed rows, or one query) and the others each in a kernel of
// their own rows: one kernel gives every run the rows of the longest.  Two have two starts, so it pays where short runs
// outnumber the long ones' pieces, as the totals tell if all long runs are alike (runs for the prefill kernel count as
// none).  Single queries + long runs over 2000 keys, 32 q heads over 8, one kernel and two: 32 + 2 x 60 79 and 77 us, 64 +
// 2 x 60 121 and 100, 256 + 16 x 20 371 and 245, 128 + 16 x 9 200 and 140, 256 + 2 x 5 236 and 195, 64 + 32 x 5 109 and 105,
// 64 + 8 x 5 83 and 84.
bool two_kernels(int nr, int group, int64_t total_q, int64_t num_seqs, int64_t longest, bool prefill) {
  if (nr <= tile_rows(static_cast<int64_t>(short_run(group)) * group)) return false;
  if (prefill) return true;
  const int64_t runs = std::max<int64_t>((total_q - num_seqs + longest - 2) / (longest - 1), 0);
  const int64_t pieces = runs * ((longest * group + nr - 1) / nr);
  return num_seqs - runs >= 2 * pieces;
}

// Two pieces of a kernel's rows per CTA of two per SM.
size_t parts_bytes(int sms, int nr) {
  return (2 * static_cast<size_t>(sms)) * 2 * ((nr + 15) / 16 * 16) * (kHeadDim + 1) * sizeof(float);
}

// Tickets, the pieces of the two kernels of a split call, then the prefill kernel's plan.
size_t pieces_bytes(int sms, int nr, int group) {
  const int first = tile_rows(static_cast<int64_t>(short_run(group)) * group);
  return (decode_ticket_bytes(sms) + parts_bytes(sms, nr) + (nr > first ? parts_bytes(sms, first) : 0) + 255) & ~size_t(255);
}

size_t workspace8(int sms, int nr, int group) {
  return pieces_bytes(sms, nr, group) + sizeof(int32_t) * (2 + static_cast<size_t>(kMaxPrefillTiles));
}

// The part of both calls after their own checks: runs of shortest to longest queries in the kernel for nr rows.  `second`:
// behind the kernel of the short runs, beside whose last blocks its own may run (other tickets, other pieces).
int run_attention(Fp8DecodeParams p, const void* k_cache, const void* v_cache, const float* k_scale,
                  const float* v_scale, int32_t scale_block, int nr, bool second, void* workspace,
                  size_t workspace_bytes, void* stream) {
  const int64_t rows = static_cast<int64_t>(p.num_blocks) * p.block_size;
  const int sms = sm_count();
  if (sms == 0) return cuda_fail(cudaGetLastError());
  if (workspace == nullptr || workspace_bytes < workspace8(sms, nr, p.group) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
    return NVA_ERR_WORKSPACE;
  CUtensorMap tm_k, tm_v;
  int rc;
  if ((rc = encode_rows8(&tm_k, k_cache, p.num_kv_heads, rows)) != NVA_OK) return rc;
  if ((rc = encode_rows8(&tm_v, v_cache, p.num_kv_heads, rows)) != NVA_OK) return rc;
  const int grid = 2 * sms;
  // (merge weights of a segment cut into as many pieces as there are CTAs fit the idle K and V rings)
  if (static_cast<size_t>(nr) * grid * sizeof(float) > 4 * kTile) return NVA_ERR_UNSUPPORTED;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.page_blocks = p.block_size / scale_block;
  p.lg_block = __builtin_ctz(static_cast<unsigned>(scale_block));
  // heads that walk side by side (the work split, above)
  p.head_set = 1;
  for (int h = 8; h > 1; h /= 2)
    if (p.num_kv_heads % h == 0 && grid % h == 0) {
      p.head_set = h;
      break;
    }
  p.max_n = nr / p.group;
  p.counters = static_cast<int32_t*>(workspace) + (second ? 1 : 0);
  const size_t first = parts_bytes(sms, tile_rows(static_cast<int64_t>(short_run(p.group)) * p.group));
  p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + decode_ticket_bytes(sms) + (second ? first : 0));
  p.part_lse = p.part_o + static_cast<size_t>(grid) * 2 * ((nr + 15) / 16 * 16) * kHeadDim;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (nr) {
    case 8: e = launch8<8>(tm_k, tm_v, p, grid, s); break;
    case 16: e = launch8<16>(tm_k, tm_v, p, grid, s); break;
    case 24: e = launch8<24>(tm_k, tm_v, p, grid, s); break;
    case 32: e = launch8<32>(tm_k, tm_v, p, grid, s); break;
    default: e = launch8<40>(tm_k, tm_v, p, grid, s);
  }
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

NVA_API size_t nva_paged_attention_fp8_workspace_bytes(int32_t max_q, int32_t num_heads, int32_t num_kv_heads,
                                                       int32_t head_dim) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || max_q < 0 ||
      head_dim != nva::kHeadDim || num_heads / num_kv_heads > nva::kMaxRows8)
    return 0;
  const int sms = nva::sm_count();
  const int group = num_heads / num_kv_heads;
  return sms == 0 ? 0 : nva::workspace8(sms, nva::rows_for(max_q, group), group);
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
  if (head_dim != nva::kHeadDim || num_heads / num_kv_heads > nva::kMaxRows8) return NVA_ERR_UNSUPPORTED;
  if (num_seqs == 0) return NVA_OK;
  int rc = nva::check_common(q, q_row_stride, k_cache, v_cache, k_scale, v_scale, num_blocks, block_size, scale_block,
                             block_tables, bt_row_stride, bt_width, num_heads, num_kv_heads, head_dim, out,
                             out_row_stride);
  if (rc != NVA_OK) return rc;
  if (context_lens == nullptr) return NVA_ERR_INVALID_ARGUMENT;
  if (static_cast<int64_t>(num_seqs) * q_per_seq >= (int64_t(1) << 31)) return NVA_ERR_UNSUPPORTED;
  const int nr = nva::rows_for(q_per_seq, num_heads / num_kv_heads);
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
  return nva::run_attention(p, k_cache, v_cache, k_scale, v_scale, scale_block, nr, false, workspace, workspace_bytes,
                            stream);
}

NVA_API int nva_varlen_attention_fp8(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                     const float* k_scale, const float* v_scale, int32_t num_blocks,
                                     int32_t block_size, int32_t scale_block, const int32_t* cu_seqlens_q,
                                     const int32_t* cu_seqlens_k, int32_t num_seqs, int32_t total_q,
                                     int32_t max_seqlen_q, const int32_t* block_tables, int32_t bt_row_stride,
                                     int32_t bt_width,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float softmax_scale,
                                     void* out, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (num_seqs < 0 || total_q < 0 || max_seqlen_q < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      !nva::positive_finite(softmax_scale))
    return NVA_ERR_INVALID_ARGUMENT;
  if (head_dim != nva::kHeadDim || num_heads / num_kv_heads > nva::kMaxRows8) return NVA_ERR_UNSUPPORTED;
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
  const int nr = nva::rows_for(max_seqlen_q, p.group);
  // Long runs: the prefill kernel, as far as its plan holds the call (1024 sequences, 4096 query tiles).
  const int64_t tiles = static_cast<int64_t>(total_q) / 128 + num_seqs + 1;
  const bool prefill = max_seqlen_q >= nva::kMinPrefillRun && num_seqs <= nva::kMaxDecodeSeqs &&
                       tiles <= nva::kMaxPrefillTiles;
  // The decode kernel's part: all runs up to the prefill kernel's at once, or the short ones and the others.
  const bool two = nva::two_kernels(nr, p.group, total_q, num_seqs, max_seqlen_q, prefill);
  auto decode = [&]() -> int {
    p.shortest = 0;
    p.longest = prefill ? nva::kMinPrefillRun - 1 : 0x7FFFFFFF;
    p.pdl = p.wait_primary = prefill ? 1 : 0;
    if (two) {
      const int64_t longest = p.longest;
      p.longest = nva::short_run(p.group);
      const int first = nva::tile_rows(static_cast<int64_t>(p.longest) * p.group);
      const int e = nva::run_attention(p, k_cache, v_cache, k_scale, v_scale, scale_block, first, false, workspace,
                                       workspace_bytes, stream);
      if (e != NVA_OK) return e;
      p.shortest = p.longest + 1;
      p.longest = static_cast<int32_t>(longest);
      p.pdl = 1;
      p.wait_primary = 0;
    }
    return nva::run_attention(p, k_cache, v_cache, k_scale, v_scale, scale_block, nr, two, workspace, workspace_bytes,
                              stream);
  };
  if (prefill) {
    const int sms = nva::sm_count();
    if (sms == 0) return nva::cuda_fail(cudaGetLastError());
    if (workspace == nullptr || workspace_bytes < nva::workspace8(sms, nr, p.group) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
      return NVA_ERR_WORKSPACE;
    CUtensorMap tm_q, tm_k, tm_v, tm_o;
    const int64_t rows = static_cast<int64_t>(num_blocks) * block_size;
    if ((rc = nva::encode_rows8(&tm_k, k_cache, num_kv_heads, rows)) != NVA_OK) return rc;
    if ((rc = nva::encode_rows8(&tm_v, v_cache, num_kv_heads, rows)) != NVA_OK) return rc;
    if ((rc = nva::encode_rows(&tm_q, q, num_heads, total_q, q_row_stride * 2)) != NVA_OK) return rc;
    if ((rc = nva::encode_rows(&tm_o, out, num_heads, total_q, out_row_stride * 2)) != NVA_OK) return rc;
    nva::PrefillParams pp{};
    pp.q = p.q;
    pp.q_row_stride = q_row_stride;
    pp.out = p.out;
    pp.out_row_stride = out_row_stride;
    pp.cu_q = cu_seqlens_q;
    pp.cu_k = cu_seqlens_k;
    pp.block_tables = block_tables;
    pp.bt_stride = bt_row_stride;
    pp.bt_width = bt_width;
    pp.num_seqs = num_seqs;
    pp.num_heads = num_heads;
    pp.num_kv_heads = num_kv_heads;
    pp.group = p.group;
    pp.min_q = nva::kMinPrefillRun;
    pp.block_size = block_size;
    pp.num_blocks = num_blocks;
    pp.q_tiles_bound = static_cast<int32_t>(tiles);
    pp.tiles_per_item = 1;
    pp.o_tma = 1;
    pp.wait_primary = 0;
    pp.scale_log2 = p.scale_log2;
    pp.k_scale = k_scale;
    pp.v_scale = v_scale;
    pp.page_blocks = block_size / scale_block;
    pp.lg_block = __builtin_ctz(static_cast<unsigned>(scale_block));
    pp.plan = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + nva::pieces_bytes(sms, nr, p.group));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int grid = static_cast<int>(std::min<int64_t>(sms, tiles * num_heads));
    // plan, short runs, long runs: the prefill kernel's blocks take their items from a counter as SMs come free
    cudaError_t e = nva::launch_prefill_plan(pp, s);
    if (e != cudaSuccess) return nva::cuda_fail(e);
    if ((rc = decode()) != NVA_OK) return rc;
    e = nva::launch_prefill(tm_q, tm_k, tm_v, tm_o, pp, grid, s);
    return e == cudaSuccess ? NVA_OK : nva::cuda_fail(e);
  }
  return decode();
}

}  // extern "C"
