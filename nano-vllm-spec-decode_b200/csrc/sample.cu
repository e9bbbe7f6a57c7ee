// Sampling from rows of logits, and speculative sampling of fixed drafts (the random branches of Sampler.forward,
// nanovllm/layers/sampler.py:7-16, and verify_drafts, :68-78 and 83-102), from given uniform numbers.
//
// For a row l[0..V) with temperature T > 0, m = max l:
//     w_i = exp((l_i - m) / T)                      (1 where l_i == m, whatever m is)
//     min-p:  tokens with w_i < min_p go
//     top-k:  the k largest stay (equal logits: lowest indices first)
//     top-p:  of what is left, in falling order (same rule for equals), a token stays while the weight before it is less
//             than top_p times the weight of what is left
//     draw:   the first index i with  sum_{j <= i, kept} w_j > u * sum_kept w_j
// and T <= 0 takes the argmax (lowest index; NaN above everything).  NaN counts as -inf for T > 0.  A draft d of a row
// is accepted when u' * sum_kept w < w_d (0 when d is not kept); the token behind the last accepted draft is drawn from
// its row without the draft that was turned down there.
//
// A token id is a whole number: two programs agree on it only if the running sums they compare agree far below the gap
// between neighbouring sums, and a vocabulary has 150,000 of those.  So weights are fixed-point integers, w * 2^44
// rounded from a double-precision exponential (a table of 2^(j/16) and five terms of the exponential series, off by
// 1.5e-13 at most), and sums are exact 64-bit integer sums: no order of additions, atomics included, can change a result.
// Weights below 2^-45 are 0.
//
// Three ways, by the settings of a row (the arguments that are given, and their values on the device):
//   * none of top-k, top-p and min-p given: no threshold, so no row has to stay on the chip.  One kernel gives a warp each
//     a segment of 4 KB, straight from registers (its maximum, then its weights' sum against that), a second one brings a
//     row's segments to one maximum, draws a segment and walks it.  510 rows of 151,936 in bf16: 71 us, a third of the
//     copy bandwidth (140 us with the row in shared memory); the issue slots of the exponentials bound it.
//   * else a cluster of CTAs keeps a row in its shared memory (V = 151,936 in bf16: four CTAs of 78 KB) -- one pass over
//     HBM.  Where top-k or min-p leaves few tokens, the CTAs list what passes a bound, and the first of them sorts the
//     lists and finishes alone: one row 14 us (20 with the histograms), of which loads take 1.5, the list 2.5, an
//     exchange across the cluster 2.5, the sort and the draw 5: latency.
//   * other rows: thresholds from histograms (counts, or fixed-point weights) over 1024 bins, first of equal width in l
//     (so that neighbouring logits rarely meet in one bin), then of the crossing bin's keys until one key is left; at
//     that key the first m equal tokens stay, in index order.  CTAs exchange maxima, histograms and sums through
//     distributed shared memory.  For the draw every thread owns a run of consecutive tokens, a prefix sum over threads
//     and CTAs names the run that holds u * W, and one warp walks it.  One row with top-p 0.9 takes 35 us (the histogram
//     of weights 7, exchanges 5, the crossing bin 9, the run sums 6), 64 of them 79.
// A batch of 64 rows in fp32 with all kinds of settings takes 53 us: its rows do not fit the chip at once, and rows that
// start second wait for shared memory.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "../../include/nvattn.h"
#include "nva_kernels.h"
#include "nva_ptx.cuh"

namespace nva {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kTable = 16;            // 128 bytes: whatever entries a warp's lanes ask for, no two meet in a bank
constexpr int kList = 1024;            // tokens of a crossing bin kept aside per CTA
constexpr int kRowsPerThread = 4;      // rows that the order by work goes up to, per thread
constexpr int kShort = 2048;           // tokens that rank 0 sorts and finishes by itself
constexpr int kMaxCluster = 8;
constexpr float kReach = 31.5f;        // exp(-31.5) < 2^-45: weight 0
constexpr uint32_t kAll = 0xffffffffu;
constexpr uint32_t kNone = 0xffffffffu;
using u64 = unsigned long long;

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  int32_t rows, vocab;
  int32_t run_words;                   // 32-bit words of a row per thread (odd: neighbouring threads, other banks)
  int32_t group;                       // rows that share one set of settings: 1, or k + 1 (verify)
  int32_t by_work;                     // 1: rows start in the order of their work
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const void* uniform;                 // per set of settings
  int32_t uniform_bytes;
  int64_t* ids;                        // sample: [rows]
  // verify
  const void* drafts;
  int64_t draft_stride;
  const void* num_drafts;
  int32_t id_bytes;
  const void* accept_uniform;          // [sets, k] at accept_stride
  int64_t accept_stride;
  int2* row_result;                    // [rows] (token, accepted)
};

// What a cluster agrees on; every CTA holds a copy.
struct Control {
  u64 before;                          // count or weight above the crossing bin
  double target;                       // where the running count or weight has to get
  uint32_t bin;                        // the crossing bin (kNone: everything stays)
  uint32_t last;                       // this CTA's tokens in the last bin
  u64 draft_weight;
  u64 sum;                             // this CTA's kept weight (equals of the threshold apart) ...
  uint32_t ties;                       // ... and number of tokens at the threshold
  float top;                           // its largest logit
  uint32_t first;                      // its first index of the row's largest logit
};

// Rows are held as they come, two bf16 or one float to a word; NaN as -inf (unless greedy), padding as NaN, which fails
// every comparison.  Keys are whole numbers in the logits' order, -0 equal to +0.
template <typename T>
struct Row;
template <>
struct Row<__nv_bfloat16> {
  static constexpr int kPerWord = 2;
  static constexpr uint32_t kPad = 0xFFFFu;
  static __device__ __forceinline__ uint32_t both(float l) {   // in every place of a word, rounded to the type
    const __nv_bfloat162 v = __float2bfloat162_rn(l);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {   // the number where one is NaN
    const __nv_bfloat162 v =
        __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  template <class F>
  static __device__ __forceinline__ void each(uint32_t w, F&& f) {
    f(__uint_as_float(w << 16), 0);
    f(__uint_as_float(w & 0xFFFF0000u), 1);
  }
  static __device__ __forceinline__ uint32_t key(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return ((b & 0x80000000u) ? ~b : (b | 0x80000000u)) >> 16;
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(((k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu)) << 16);
  }
};
template <>
struct Row<float> {
  static constexpr int kPerWord = 1;
  static constexpr uint32_t kPad = 0xFFFFFFFFu;
  static __device__ __forceinline__ uint32_t both(float l) { return __float_as_uint(l); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  template <class F>
  static __device__ __forceinline__ void each(uint32_t w, F&& f) { f(__uint_as_float(w), 0); }
  static __device__ __forceinline__ uint32_t key(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
};

__device__ __forceinline__ double read_uniform(const void* u, int64_t at, int bytes) {
  const double v = bytes == 8 ? static_cast<const double*>(u)[at] : static_cast<const float*>(u)[at];
  return v > 0.0 ? fmin(v, 0.99999999999999988) : 0.0;   // (NaN and negative numbers: 0)
}
__device__ __forceinline__ int64_t read_id(const void* p, int64_t at, int bytes) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[at] : static_cast<const int32_t*>(p)[at];
}

// Whether a row of a verify call lies behind its sequence's last draft's, where nothing is drawn.
template <bool kVerify>
__device__ __forceinline__ bool behind_drafts(const SampleParams& p, int row) {
  if constexpr (!kVerify) return false;
  const int set = row / p.group, j = row - set * p.group;
  return j > 0 && j > read_id(p.num_drafts, set, p.id_bytes);
}

// w * 2^44 of a logit within reach of the maximum: 2^(u / 16) with u = 16 log2(e) (l - m) / T = 16 e + j + r, |r| <= 1/2,
// from a table of 2^(j / 16 + 44), e added to its exponent, and five terms of the exponential series in r ln 2 / 16 (the
// sixth is below 1.5e-13: a running sum is off by as little, against gaps of 1e-6 between a vocabulary's sums).
struct Weight {
  double m, c;           // row maximum, 16 log2(e) / T
  float low;             // logits above it have a weight
  const double* table;
  __device__ __forceinline__ double2 factors(float l) const {   // their product is the weight (only for l > low)
    const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double d = static_cast<double>(l) - m;
    const double n = fma(d, c, magic);
    const double r = fma(d, c, magic - n);
    const int k = __double2loint(n);
    double s = fma(r, 1.271587195055813e-09, 1.467610032291943e-07);   // (ln 2 / 16)^5 / 120, ^4 / 24
    s = fma(s, r, 1.3550807779497455e-05);                            // ^3 / 6
    s = fma(s, r, 0.0009383847928089871);                             // ^2 / 2
    s = fma(s, r, 0.04332169878499658);                              // ln 2 / 16
    s = fma(s, r, 1.0);
    const double t = table[k & 15];
    return make_double2(s, __hiloint2double(__double2hiint(t) + ((k & ~15) << 16), __double2loint(t)));   // + e << 20
  }
  // as a double, and as the whole number in the low 52 bits of one in [2^52, 2^53)
  __device__ __forceinline__ double value(float l) const {
    const double2 f = factors(l);
    return f.x * f.y;
  }
  __device__ __forceinline__ u64 bits(float l) const {
    const double2 f = factors(l);
    return __double_as_longlong(fma(f.x, f.y, 4503599627370496.0));
  }
  static constexpr u64 kZero = 0x4330000000000000ull;   // the bits of 2^52
  __device__ __forceinline__ u64 operator()(float l) const { return l > low ? bits(l) - kZero : 0ull; }
};

// Weights of logits up to `top` > -inf, finite, at temperature `temp`.
__device__ __forceinline__ Weight make_weight(float top, float temp, const double* table) {
  Weight w;
  w.m = top;
  w.c = 23.083120654223414 / static_cast<double>(temp);   // 16 log2(e)
  // (below the maximum however large that is; at an infinite temperature everything but -inf)
  w.low = fminf(fmaxf(top - kReach * temp, -FLT_MAX), nextafterf(top, -__int_as_float(0x7F800000)));
  w.table = table;
  return w;
}

// Exclusive prefix sums of a weight and a count over a block of kCount warps; `tot` receives the block's sums.
template <int kCount>
__device__ __forceinline__ void block_scan(u64& mass, uint32_t& count, u64* wm, uint32_t* wc, u64* tot_m,
                                           uint32_t* tot_c, int lane, int warp) {
  u64 x = mass;
  uint32_t c = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(kAll, x, o);
    const uint32_t z = __shfl_up_sync(kAll, c, o);
    if (lane >= o) {
      x += y;
      c += z;
    }
  }
  if (lane == 31) {
    wm[warp] = x;
    wc[warp] = c;
  }
  __syncthreads();
  u64 bm = 0, tm = 0;
  uint32_t bc = 0, tc = 0;
#pragma unroll
  for (int w = 0; w < kCount; ++w) {
    if (w < warp) {
      bm += wm[w];
      bc += wc[w];
    }
    tm += wm[w];
    tc += wc[w];
  }
  mass = bm + x - mass;
  count = bc + c - count;
  *tot_m = tm;
  *tot_c = tc;
  __syncthreads();
}

template <typename T, bool kVerify>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  using R = Row<T>;
  constexpr int kPer = R::kPerWord;
  const float kInf = __int_as_float(0x7F800000);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int row = blockIdx.x / ranks;

  extern __shared__ __align__(16) uint8_t smem[];
  const int words = p.run_words * kThreads;
  uint32_t* data = reinterpret_cast<uint32_t*>(smem);
  // histograms (counts, or weights: low and high words); rank 0's sorted tokens of a short list
  __shared__ __align__(16) union {
    uint32_t hist[2][kBins];
    u64 sorted[kShort];
  } bins;
  auto& hist = bins.hist;
  __shared__ double table[kTable];
  __shared__ __align__(16) union {
    uint32_t keys[kList];
    u64 tokens[kShort];
  } lists;
  auto& list = lists.keys;
  __shared__ uint32_t list_count;
  __shared__ u64 scan_m[kWarps];
  __shared__ uint32_t scan_c[kWarps];
  __shared__ Control ctrl;
  __shared__ int found_thread;
  __shared__ u64 found_rest;
  __shared__ uint32_t found_ties;

  if (p.by_work) {
    // Rows that no small list finishes (30 to 45 us, the others 15) first, so that none of them starts last (160 rows of
    // verify in bf16: 77 us in their own order, 72 in this).
    uint32_t mine = 0, long_rows;
    u64 none = 0, none_t;
    const int first = tid * kRowsPerThread;
    auto is_long = [&](int r) {
      const int s = r / p.group;
      const int k = p.top_k != nullptr ? __ldg(p.top_k + s) : 0;
      return __ldg(p.temperature + s) > 0.f && !behind_drafts<kVerify>(p, r) && !(k > 0 && k <= kThreads / 2) &&
             !(p.min_p != nullptr && __ldg(p.min_p + s) > 0.f);
    };
    bool is[kRowsPerThread];
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      is[i] = first + i < p.rows && is_long(first + i);
      mine += is[i] ? 1 : 0;
    }
    block_scan<kWarps>(none, mine, scan_m, scan_c, &none_t, &long_rows, lane, warp);
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      const int place = is[i] ? static_cast<int>(mine) : static_cast<int>(long_rows) + first + i - static_cast<int>(mine);
      if (first + i < p.rows && place == row) found_thread = first + i;
      mine += is[i] ? 1 : 0;
    }
    __syncthreads();
    row = found_thread;
    __syncthreads();
  }
  if (behind_drafts<kVerify>(p, row)) return;
  const int set = row / p.group;
  const float temp = __ldg(p.temperature + set);
  const bool greedy = !(temp > 0.f);
  int k = p.top_k != nullptr ? __ldg(p.top_k + set) : 0;
  if (k >= p.vocab) k = 0;
  const float bin_scale = (kBins / 32.0f) / temp;

  // ---------------------------------------------------------------- the row
  const int e0 = rank * words * kPer;          // first token of this CTA
  const int n = max(0, min(p.vocab - e0, words * kPer));
  float top = -kInf, cta_top, own_top = -kInf;  // the largest logit of the row, the CTA and this thread's loads
  {
    const T* src = static_cast<const T*>(p.logits) + row * p.row_stride + e0;
    const uint32_t* src32 = reinterpret_cast<const uint32_t*>(src);
    bool nan = false;
    const uint32_t low = kPer == 2 ? 0xFF80FF80u : 0xFF800000u;   // -inf
    uint32_t best = low;
    auto keep = [&](uint32_t w) -> uint32_t {
      const uint32_t x = R::larger(w, low);
      best = R::larger(best, x);
      if (!greedy) return x;
      R::each(w, [&](float l, int) { nan |= l != l; });
      return w;
    };
    int done = 0;   // words in place
    if ((reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
      const int nv = n / (4 * kPer);
      constexpr int kUnroll = 8;
      for (int v0 = tid; v0 < nv; v0 += kUnroll * kThreads) {
        uint4 raw[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
          if (v0 + i * kThreads < nv) raw[i] = __ldg(reinterpret_cast<const uint4*>(src32) + v0 + i * kThreads);
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
          if (v0 + i * kThreads < nv)
            reinterpret_cast<uint4*>(data)[v0 + i * kThreads] =
                make_uint4(keep(raw[i].x), keep(raw[i].y), keep(raw[i].z), keep(raw[i].w));
      }
      done = nv * 4;
    }
    for (int w = done + tid; w < words; w += kThreads) {
      // (the row's end) padding takes no part in the maximum
      uint32_t x = low, pad = 0;
#pragma unroll
      for (int h = 0; h < kPer; ++h) {
        const int e = w * kPer + h;
        const uint32_t mask = (kPer == 2 ? 0xFFFFu : 0xFFFFFFFFu) << (16 * h);
        if (e < n) {
          const uint32_t v = kPer == 2 ? static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(src) + e))
                                       : __ldg(src32 + e);
          x = (x & ~mask) | (v << (16 * h));
        } else {
          pad |= (R::kPad << (16 * h)) & mask;
        }
      }
      data[w] = keep(x) | pad;   // (-inf's bits are among the padding's NaN's)
    }
    if (tid < kTable) table[tid] = exp2(static_cast<double>(tid) / kTable + 44.0);
    R::each(best, [&](float l, int) { own_top = fmaxf(own_top, l); });
    top = own_top;
    // as a key (NaN, which only a greedy row looks for, above +inf)
    uint32_t k = __float_as_uint(top + 0.f);
    k = nan ? kNone : (k & 0x80000000u) ? ~k : (k | 0x80000000u);
    k = __reduce_max_sync(kAll, k);
    if (lane == 0) scan_c[warp] = k;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) k = max(k, scan_c[w]);
    if (tid == 0) ctrl.first = k;
    cta_top = __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
  // Appends the CTA's tokens above a logit to its list (key complemented and index: ascending from the largest).
  auto list_above = [&](float above) {
    for (int v = tid; v < words / 4; v += kThreads) {   // (whole warps: words are a multiple of 512)
      const uint4 x = reinterpret_cast<const uint4*>(data)[v];
      bool any = false;
      R::each(R::larger(R::larger(x.x, x.y), R::larger(x.z, x.w)), [&](float l, int) { any |= l > above; });
      if (__ballot_sync(kAll, any) == 0) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        R::each(i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w, [&](float l, int h) {
          const bool in = l > above;
          const uint32_t vote = __ballot_sync(kAll, in);
          if (vote == 0) return;
          uint32_t at = 0;
          if (lane == 0) at = atomicAdd(&list_count, static_cast<uint32_t>(__popc(vote)));
          at = __shfl_sync(kAll, at, 0) + __popc(vote & ((1u << lane) - 1u));
          if (in && at < kShort)
            lists.tokens[at] = static_cast<u64>(~R::key(l)) << 32 | static_cast<uint32_t>(e0 + (v * 4 + i) * kPer + h);
        });
    }
  };
  // a little below every logit that lies in bins up to `bin` of a maximum
  auto below_bin = [&](float max, int bin) {
    return nextafterf(nextafterf(max - (static_cast<float>(bin) + 1.01f) / bin_scale, -kInf), -kInf);
  };
  // A small top-k: every CTA lists its own k largest, and whatever its bound lets through, before it knows the others'
  // (one exchange in all instead of three).  The bound: the k-th largest of its threads' maxima, to a bin, so that 512
  // numbers are counted and not its share of the row; about k + k^2 / 1024 tokens pass it.  Beyond 256 tokens in all
  // the longer sort costs more than the exchanges (64 rows of four CTAs in bf16, this and one bound for the row: k = 50
  // 22.7 and 22.7 us, 128 28.9 and 24.8, 256 43 and 28; one row of eight, k = 128: 24.8 and 18.5).
  bool listed = !greedy && k > 0 && k <= kThreads / 2 && k * ranks <= kThreads / 2;
  if (listed) {
    for (int i = tid; i < kBins; i += kThreads) hist[0][i] = 0;
    if (tid == 0) list_count = 0;
    __syncthreads();
    if (cta_top - cta_top == 0.f) {
      if (own_top > -kInf) atomicAdd(&hist[0][min(kBins - 1, __float2int_rz((cta_top - own_top) * bin_scale))], 1u);
      __syncthreads();
      const uint2 c = reinterpret_cast<const uint2*>(&hist[0][0])[tid];
      u64 none = 0, none_t;
      uint32_t pre = c.x + c.y, tot;
      if (tid == 0) found_ties = kBins - 1;      // (fewer maxima than k: no bound)
      block_scan<kWarps>(none, pre, scan_m, scan_c, &none_t, &tot, lane, warp);
      const uint32_t want = static_cast<uint32_t>(k);
      if (pre < want && pre + c.x >= want) found_ties = 2 * tid;
      if (pre + c.x < want && pre + c.x + c.y >= want) found_ties = 2 * tid + 1;
      __syncthreads();
      const int bin = static_cast<int>(found_ties);
      list_above(bin < kBins - 1 ? below_bin(cta_top, bin) : -kInf);
    }
  }
  cluster.sync();
  {
    // (lane r reads CTA r's: one trip, not one per CTA)
    const uint32_t k = __reduce_max_sync(kAll, lane < ranks ? cluster.map_shared_rank(&ctrl, lane)->first : 0u);
    top = __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
  const int run0 = tid * p.run_words;          // this thread's run of words

  int draft = -1;
  if constexpr (kVerify) {
    const int k = p.group - 1, j = row - set * p.group;
    if (j < k && j < read_id(p.num_drafts, set, p.id_bytes)) {
      const int64_t d = read_id(p.drafts, set * p.draft_stride + j, p.id_bytes);
      draft = d >= 0 && d < p.vocab ? static_cast<int>(d) : p.vocab;   // (p.vocab: no such token, never accepted)
    }
  }

  if (greedy) {
    // ---------------------------------------------------------------- argmax: the first index of the largest logit
    cluster.sync();   // (ctrl.first is read; below it is written again)
    const bool nan = top != top;
    uint32_t first = kNone;
    for (int w = run0; w < run0 + p.run_words && first == kNone; ++w)
      R::each(data[w], [&](float l, int h) {
        const int e = w * kPer + h;
        if (first == kNone && e < n && (nan ? l != l : l == top)) first = static_cast<uint32_t>(e0 + e);
      });
    first = __reduce_min_sync(kAll, first);
    if (lane == 0) scan_c[warp] = first;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) first = min(first, scan_c[w]);
      ctrl.first = first;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int r = 1; r < ranks; ++r) first = min(first, cluster.map_shared_rank(&ctrl, r)->first);
      if constexpr (kVerify) {
        p.row_result[row] = make_int2(static_cast<int>(first), draft == static_cast<int>(first) ? 1 : 0);
      } else {
        p.ids[row] = static_cast<int64_t>(first);
      }
    }
    cluster.sync();
    return;
  }

  if (top - top != 0.f) {
    // an infinite maximum: its equals weigh 1, all others nothing
    for (int w = tid; w < words; w += kThreads) {
      uint32_t x = 0;
      R::each(data[w], [&](float l, int h) {
        const uint32_t v = l != l ? R::kPad : l == top ? 0u : (kPer == 2 ? 0xFF80u : 0xFF800000u);
        x |= v << (16 * h);
      });
      data[w] = x;
    }
    own_top = own_top == top ? 0.f : -kInf;
    top = 0.f;
    listed = false;
    __syncthreads();
  }

  // ---------------------------------------------------------------- thresholds
  const Weight weight = make_weight(top, temp, table);
  // kept: logits above `cut`, and the first `cut_ties` tokens at it
  float cut = -kInf;
  uint32_t cut_ties = 0;
  if (p.min_p != nullptr) {
    const double mp = fmin(static_cast<double>(__ldg(p.min_p + set)), 1.0);
    if (mp > 0.0) {
      const double at = weight.m + static_cast<double>(temp) * log(mp);   // l >= at
      float f = static_cast<float>(at);
      if (static_cast<double>(f) < at) f = nextafterf(f, kInf);
      if (f == f) cut = nextafterf(f, -kInf);
    }
  }
  auto linear_bin = [&](float l) {             // rises as the logit falls; bins of T / 32, the last takes the rest
    return min(kBins - 1, __float2int_rz((top - l) * bin_scale));
  };
  // Ascending, n different numbers in v: every warp sorts 32 in its registers, then runs are merged in pairs into the
  // other buffer, each number's place from a binary search of the other run (180 numbers: 1.5 us; a bitonic network in
  // shared memory: 5).  Returns the buffer they end in.
  auto sort = [&](u64* v, u64* other, int n) -> u64* {
    for (int at = tid; at - lane < n; at += kThreads) {   // (whole warps)
      u64 own = at < n ? v[at] : ~0ull;
#pragma unroll
      for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int j = size >> 1; j > 0; j >>= 1) {
          const u64 y = __shfl_xor_sync(kAll, own, j);
          const bool keep_less = ((lane & j) == 0) == ((lane & size) == 0);
          if ((y < own) == keep_less) own = y;
        }
      if (at < n) v[at] = own;
    }
    __syncthreads();
    for (int run = 32; run < n; run <<= 1) {
      for (int at = tid; at < n; at += kThreads) {
        const u64 own = v[at];
        const int start = (at & -run) ^ run, length = min(run, n - start);
        int less = 0;
        if (length > 0) {
          for (int step = run; step > 0; step >>= 1) {
            const int to = less + step;
            const u64 x = v[start + min(to, length) - 1];
            less = to <= length && x < own ? to : less;
          }
        }
        other[(at & -(2 * run)) + (at & (run - 1)) + less] = own;
      }
      u64* const t = v;
      v = other;
      other = t;
      __syncthreads();
    }
    return v;
  };
  auto clear = [&]() {
    for (int i = tid; i < 2 * kBins; i += kThreads) (&hist[0][0])[i] = 0;
    if (tid == 0) list_count = 0;
    __syncthreads();
  };
  // (rank 0) the CTAs' bins together, two per thread: the first at which the target is reached, to everyone
  auto cross = [&](auto by_weight, u64 before, bool linear, uint32_t k, double share) {
    constexpr bool kMass = decltype(by_weight)::value;
    if (rank == 0) {
      u64 v[2] = {0, 0};
      constexpr int kAtOnce = kMass ? 4 : kMaxCluster;   // CTAs' bins on their way at once
#pragma unroll 1
      for (int r0 = 0; r0 < ranks; r0 += kAtOnce) {
        uint2 low[kAtOnce], high[kAtOnce];
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r) {
          low[r] = high[r] = make_uint2(0u, 0u);
          if (r0 + r < ranks) {
            const uint2* h = reinterpret_cast<const uint2*>(cluster.map_shared_rank(&hist[0][0], r0 + r));
            low[r] = h[tid];
            if constexpr (kMass) high[r] = h[kBins / 2 + tid];
          }
        }
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r) {
          v[0] += low[r].x + (static_cast<u64>(high[r].x) << 32);
          v[1] += low[r].y + (static_cast<u64>(high[r].y) << 32);
        }
      }
      uint32_t last = 0;
      if (!kMass && linear && warp == 0)
        last = __reduce_add_sync(kAll, lane < ranks ? cluster.map_shared_rank(&ctrl, lane)->last : 0u);
      u64 pre = v[0] + v[1], tot;
      uint32_t none = 0, none_t;
      block_scan<kWarps>(pre, none, scan_m, scan_c, &tot, &none_t, lane, warp);
      // (the first token always stays: a target of 0 would find no crossing)
      const double target = !linear ? ctrl.target : kMass ? fmax(share * static_cast<double>(tot), 1.0) : k;
      auto tell = [&](uint32_t bin, u64 above) {
        for (int r = 0; r < ranks; ++r) {
          Control* c = cluster.map_shared_rank(&ctrl, r);
          c->bin = bin;
          c->before = above;
          c->target = target;
        }
      };
      pre += before;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (v[i] != 0 && static_cast<double>(pre) < target && static_cast<double>(pre + v[i]) >= target)
          tell(static_cast<uint32_t>(2 * tid + i), pre);
        pre += v[i];
      }
      if (!kMass && linear && tid == 0 && tot < k)   // not within the bins counted
        tell(tot + last > k ? static_cast<uint32_t>(kBins - 1) : kNone, tot);
    }
    cluster.sync();
  };
  uint32_t kept_tokens = 0x7FFFFFFFu;          // an upper bound on the tokens kept
  // Sets the threshold to the logit at which the running count from the top reaches `k`, or the running weight `share`
  // of the whole, with the number of its equals that still belong; leaves it where everything stays.
  auto select = [&](auto by_weight, uint32_t k, double share) {
    constexpr bool kMass = decltype(by_weight)::value;
    const float floor = cut;                   // tokens eligible: above it, and (weights) cut_ties at it
    const u64 w_floor = kMass && cut_ties > 0 ? cut_ties * weight(floor) : 0ull;
    auto add_mass = [&](int b, u64 v) {
      const uint32_t x = static_cast<uint32_t>(v);
      const uint32_t old = atomicAdd(&hist[0][b], x);
      const uint32_t up = static_cast<uint32_t>(v >> 32) + (old + x < old ? 1u : 0u);
      if (up != 0) atomicAdd(&hist[1][b], up);
    };
    clear();
    uint32_t lo = R::key(floor), hi = R::key(top);   // (the threshold itself may be no bf16 number: a bound)
    u64 before = 0;
    // weights of no more tokens than a CTA has threads (what a top-k left): no need of bins
    const bool direct = kMass && lo < hi && kept_tokens + 2 <= kThreads;
    if (!direct) {
      uint32_t last = 0;
      for (int w = tid; w < words; w += kThreads)
        R::each(data[w], [&](float l, int) {
          if (!(l > (kMass ? fmaxf(floor, weight.low) : floor))) return;
          const int b = linear_bin(l);
          if constexpr (kMass) {
            add_mass(b, weight.bits(l) - Weight::kZero);
          } else if (b < kBins - 1) {
            atomicAdd(&hist[0][b], 1u);
          } else {
            ++last;   // (most of a vocabulary at a low temperature: not through one counter)
          }
        });
      if constexpr (kMass) {
        if (rank == 0 && tid == 0 && w_floor != 0) add_mass(linear_bin(floor), w_floor);
      } else {
        last = __reduce_add_sync(kAll, last);
        if (lane == 0) scan_c[warp] = last;
        __syncthreads();
        if (tid == 0) {
          for (int w = 1; w < kWarps; ++w) last += scan_c[w];
          ctrl.last = last;
        }
      }
      cluster.sync();
      cross(by_weight, 0, true, k, share);
      if (ctrl.bin == kNone) return;
      // the crossing bin's keys: from the least with linear_bin <= bin to the last before linear_bin < bin, by 32-way
      // searches
      {
        auto search = [&](auto pred, uint32_t a, uint32_t b) {   // least key in [a, b] with pred, which holds at b
          while (a < b) {
            const uint32_t step = (b - a) / 32 + 1;
            const u64 far = a + static_cast<u64>(step) * lane;
            const uint32_t x = far < b ? static_cast<uint32_t>(far) : b;
            const uint32_t yes = __ballot_sync(kAll, x == b || pred(R::value(x)));
            const int f = yes != 0 ? __ffs(yes) - 1 : 32;   // points below f: no, point f: yes
            const uint32_t below = __shfl_sync(kAll, x, f > 0 ? f - 1 : 0);
            const uint32_t at = __shfl_sync(kAll, x, f < 32 ? f : 0);
            if (f > 0) a = below + 1;
            b = f == 0 ? a : f < 32 ? at : b;
          }
          return b;
        };
        const int ib = static_cast<int>(ctrl.bin);
        lo = search([&](float l) { return linear_bin(l) <= ib; }, lo, hi);
        if (ib > 0) hi = max(lo, search([&](float l) { return linear_bin(l) < ib; }, lo, hi) - 1);
      }
      before = ctrl.before;
    }
    if (lo < hi) {
      // its tokens, kept aside when they are few: the levels below read those instead of the row
      const float flo = R::value(lo), fhi = R::value(hi);
      for (int w = tid; w < words; w += kThreads)
        R::each(data[w], [&](float l, int) {
          if (l > floor && l >= flo && l <= fhi) {
            const uint32_t at = atomicAdd(&list_count, 1u);
            if (at < kList) list[at] = R::key(l);
          }
        });
    }
    if (lo < hi) {
      // Few tokens in all: rank 0 takes everyone's, sorts them and runs along them to the target.
      cluster.sync();
      const uint32_t mine = lane < ranks ? *cluster.map_shared_rank(&list_count, lane) : 0u;
      const uint32_t all = __reduce_add_sync(kAll, mine);
      const uint32_t longest = __reduce_max_sync(kAll, mine);
      if (all + 1 <= kShort && longest <= kList) {
        if (rank == 0) {
          int count = static_cast<int>(all);
          for (int i = tid; i - lane < count; i += kThreads) {   // (bins.sorted: the histogram has been read)
            int from = -1, place = 0;         // the CTA whose list holds token i, and where
            uint32_t first = 0;
            for (int r = 0; r < ranks; ++r) {
              const uint32_t c = __shfl_sync(kAll, mine, r);
              if (static_cast<uint32_t>(i) >= first && static_cast<uint32_t>(i) < first + c) {
                from = r;
                place = i - static_cast<int>(first);
              }
              first += c;
            }
            if (from >= 0)
              bins.sorted[i] = static_cast<u64>(~cluster.map_shared_rank(&list[0], from)[place]) << 32 |
                               static_cast<uint32_t>(i);
          }
          if (kMass && w_floor != 0 && R::key(floor) >= lo && R::key(floor) <= hi) {   // the equals of the floor, as one
            if (tid == 0) bins.sorted[count] = static_cast<u64>(~R::key(floor)) << 32 | kNone;
            ++count;
          }
          if (tid == 0) found_thread = -1;
          __syncthreads();
          const u64* a = sort(bins.sorted, lists.tokens, count);
          const int per_thread = (count + kThreads - 1) / kThreads;
          const int begin = min(tid * per_thread, count), end = min(begin + per_thread, count);
          auto mass = [&](u64 x) -> u64 {
            if constexpr (!kMass) return 1ull;
            return static_cast<uint32_t>(x) == kNone ? w_floor : weight(R::value(static_cast<uint32_t>(~(x >> 32))));
          };
          u64 sum = 0, tot;
          for (int i = begin; i < end; ++i) sum += mass(a[i]);
          u64 above = sum;
          uint32_t none = 0, none_t;
          block_scan<kWarps>(above, none, scan_m, scan_c, &tot, &none_t, lane, warp);
          above += before;
          const double target = direct ? fmax(share * static_cast<double>(tot), 1.0) : ctrl.target;
          u64 run = above;
          for (int i = begin; i < end; ++i) {
            const u64 to = run + mass(a[i]);
            if (static_cast<double>(run) < target && static_cast<double>(to) >= target) found_thread = i;
            run = to;
          }
          __syncthreads();
          if (found_thread >= 0) {
            const uint32_t key = static_cast<uint32_t>(a[found_thread] >> 32);   // (complemented)
            run = above;
            for (int i = begin; i < end; ++i) {
              if (static_cast<uint32_t>(a[i] >> 32) == key && (i == 0 || static_cast<uint32_t>(a[i - 1] >> 32) != key))
                for (int r = 0; r < ranks; ++r) {   // the first of the equals: what lies above them
                  Control* c = cluster.map_shared_rank(&ctrl, r);
                  c->bin = ~key;
                  c->before = run;
                  c->target = target;
                }
              run += mass(a[i]);
            }
          }
        }
        cluster.sync();
        lo = hi = ctrl.bin;
        before = ctrl.before;
      }
    }
    while (lo < hi) {
      __syncthreads();
      const uint32_t listed = list_count;
      for (int i = tid; i < 2 * kBins; i += kThreads) (&hist[0][0])[i] = 0;
      __syncthreads();
      const int shift = max(0, 32 - __clz(hi - lo) - 10);
      auto add = [&](uint32_t key) {
        if (key < lo || key > hi) return;
        const int b = static_cast<int>((hi - key) >> shift);
        if constexpr (kMass) {
          const u64 v = weight(R::value(key));
          if (v != 0) add_mass(b, v);
        } else {
          atomicAdd(&hist[0][b], 1u);
        }
      };
      if (listed <= kList) {
        for (uint32_t i = tid; i < listed; i += kThreads) add(list[i]);
      } else {
        for (int w = tid; w < words; w += kThreads)
          R::each(data[w], [&](float l, int) {
            if (l > floor) add(R::key(l));
          });
      }
      if (kMass && rank == 0 && tid == 0 && w_floor != 0 && R::key(floor) >= lo && R::key(floor) <= hi)
        add_mass(static_cast<int>((hi - R::key(floor)) >> shift), w_floor);
      cluster.sync();
      cross(by_weight, before, false, k, share);
      const uint32_t bin = ctrl.bin;
      before = ctrl.before;
      const uint32_t nhi = hi - (bin << shift);
      lo = (nhi - lo) >> shift == 0 ? lo : nhi - ((1u << shift) - 1u);
      hi = nhi;
    }
    // equals of the threshold that still belong
    cut = R::value(lo);
    if constexpr (kMass) {
      const double w = static_cast<double>(weight(cut));
      const double want = fmax(ceil((ctrl.target - static_cast<double>(before)) / w), 1.0);
      const uint32_t limit = cut == floor ? cut_ties : kNone;
      cut_ties = min(limit, static_cast<uint32_t>(fmin(want, 4.0e9)));
    } else {
      cut_ties = k - static_cast<uint32_t>(before);
      kept_tokens = k;
    }
    __syncthreads();   // (ctrl is read)
  };

  const float share = p.top_p != nullptr ? __ldg(p.top_p + set) : 1.f;

  // (rank 0) the rest for the `count` tokens of a short list, in bins.sorted: sorts them, applies top-k and top-p, draws.
  // Nothing is held in registers from one loop to the next: next to rows that fill the shared memory there is no L1 to
  // spill to.
  auto finish = [&](int count) {
    u64* const weights = reinterpret_cast<u64*>(data);   // (this CTA's share of the row has been searched)
    u64* a = sort(bins.sorted, lists.tokens, count);
    const int kept_k = k > 0 ? min(k, count) : count;
    const int per_thread = (count + kThreads - 1) / kThreads;   // positions of a thread, side by side
    const int first = min(tid * per_thread, count), last = min(first + per_thread, count);
    u64 sum = 0, total, none64;
    uint32_t none = 0, none_t;
    for (int at = first; at < last; ++at) {
      const float l = R::value(static_cast<uint32_t>(~(a[at] >> 32)));
      const u64 w = at < kept_k && l > cut ? weight(l) : 0ull;
      weights[at] = w;
      sum += w;
    }
    u64 before = sum;
    block_scan<kWarps>(before, none, scan_m, scan_c, &total, &none_t, lane, warp);
    int kept = kept_k;
    if (share < 1.f) {
      const double target = fmax(static_cast<double>(fmaxf(share, 0.f)) * static_cast<double>(total), 1.0);
      uint32_t n = 0;
      sum = 0;
      for (int at = first; at < last; ++at) {
        if (at >= kept_k || !(static_cast<double>(before) < target)) break;
        before += weights[at];
        sum += weights[at];
        ++n;
      }
      block_scan<kWarps>(sum, n, scan_m, scan_c, &total, &none_t, lane, warp);
      kept = static_cast<int>(none_t);
    }
    // the kept ones in the order of their indices
    if (tid == 0) found_rest = 0;
    __syncthreads();
    for (int at = tid; at < kept; at += kThreads) {
      const uint32_t token = static_cast<uint32_t>(a[at]);
      a[at] = static_cast<u64>(token) << 32 | static_cast<uint32_t>(at);
      if (kVerify && static_cast<int>(token) == draft) found_rest = weights[at];
    }
    __syncthreads();
    bool accepted = false;
    if constexpr (kVerify) {
      const u64 draft_w = found_rest;
      if (draft >= 0) {
        const double ua = read_uniform(p.accept_uniform, set * p.accept_stride + (row - set * p.group), p.uniform_bytes);
        accepted = ua * static_cast<double>(total) < static_cast<double>(draft_w);
      }
      total -= draft_w;
    }
    a = sort(a, a == bins.sorted ? lists.tokens : bins.sorted, kept);
    auto weight_at = [&](int at) {
      const u64 x = a[at];
      return kVerify && static_cast<int>(x >> 32) == draft ? 0ull : weights[x & 0xFFFFFFFFull];
    };
    const int begin = min(first, kept), end = min(last, kept);
    sum = 0;
    for (int at = begin; at < end; ++at) sum += weight_at(at);
    u64 run = sum;
    block_scan<kWarps>(run, none, scan_m, scan_c, &none64, &none_t, lane, warp);
    const double un = read_uniform(p.uniform, set, p.uniform_bytes);
    u64 want = static_cast<u64>(un * static_cast<double>(total));
    if (total > 0 && want >= total) want = total - 1;
    if (want >= run && want - run < sum) {
      int at = begin;
      for (u64 rest = want - run; at < end - 1; ++at) {
        const u64 w = weight_at(at);
        if (rest < w) break;
        rest -= w;
      }
      const int token = static_cast<int>(a[at] >> 32);
      if constexpr (kVerify) {
        p.row_result[row] = make_int2(token, accepted ? 1 : 0);
      } else {
        p.ids[row] = token;
      }
    }
    if (kVerify && total == 0 && tid == 0)   // nothing but the (then accepted) draft
      p.row_result[row] = make_int2(draft, accepted ? 1 : 0);
  };

  // Few tokens left by min-p or a top-k: rank 0 takes them all, sorts them (by logit, then index) and finishes alone.  A
  // bound that a larger top-k keeps: as above, over all the CTAs' threads.  (64 rows of 151,936 in fp32, mixed settings:
  // 76 us with the histograms below for every row, 60 with the lists.)
  if ((k > 0 && k <= kShort) || cut > -kInf) {
    for (;;) {
      if (!listed) {
        float above = cut;
        clear();
        if (k > 0 && k <= kShort) {
          if (own_top > cut) atomicAdd(&hist[0][linear_bin(own_top)], 1u);
          if (tid == 0) ctrl.last = 0;
          cluster.sync();
          cross(std::false_type{}, 0, true, static_cast<uint32_t>(k), 0.0);
          const uint32_t bin = ctrl.bin;
          if (bin < kBins - 1) above = fmaxf(cut, below_bin(top, static_cast<int>(bin)));   // (else too few maxima)
        }
        list_above(above);
        cluster.sync();
      }
      const uint32_t mine = lane < ranks ? *cluster.map_shared_rank(&list_count, lane) : 0u;
      const uint32_t count = __reduce_add_sync(kAll, mine);
      const uint32_t longest = __reduce_max_sync(kAll, mine);
      if (longest <= kShort && count <= kShort) {
        if (rank == 0) {
          for (int i = tid; i - lane < static_cast<int>(count); i += kThreads) {
            int from = -1, place = 0;
            uint32_t first = 0;
            for (int r = 0; r < ranks; ++r) {
              const uint32_t c = __shfl_sync(kAll, mine, r);
              if (static_cast<uint32_t>(i) >= first && static_cast<uint32_t>(i) < first + c) {
                from = r;
                place = i - static_cast<int>(first);
              }
              first += c;
            }
            if (from >= 0) bins.sorted[i] = cluster.map_shared_rank(&lists.tokens[0], from)[place];
          }
        }
        cluster.sync();   // the lists are read: the other CTAs are done
        if (rank == 0) finish(static_cast<int>(count));
        return;
      }
      cluster.sync();     // (list_count is read)
      if (!listed) break;
      listed = false;     // too many tokens near a CTA's k-th: once more with a bound from all of them
    }
  }

  if (k > 0) select(std::false_type{}, static_cast<uint32_t>(k), 0.0);
  if (share < 1.f) select(std::true_type{}, 0, static_cast<double>(fmaxf(share, 0.f)));

  // ---------------------------------------------------------------- the draw
  // kept weight of this thread's run, of the runs and CTAs before it, and of all
  const u64 w_cut = cut_ties > 0 ? weight(cut) : 0ull;
  u64 mine = 0;
  uint32_t ties = 0;
  {
    const float dust = top - 1.3f * (top - weight.low);   // about 41 T below: 2^-59
    // (from 2^23 T on the logits' steps grow past T: there `dust` lies too near or beyond the exponential's range)
    if (cut <= weight.low && top - dust > 36.f * temp && top - dust < 60.f * temp && dust > -FLT_MAX) {
      // Nothing cut off: (nearly) every token has a weight.  All are taken, those without (and padding) as dust; the run's
      // sum is one double, rounded to a whole number at its end (the order inside a run is fixed).
      double sum = 0.0;
#pragma unroll 4
      for (int w = run0; w < run0 + p.run_words; ++w)
        R::each(data[w], [&](float l, int) { sum += weight.value(fmaxf(l, dust)); });
      mine = static_cast<u64>(__double2ll_rn(sum));
    } else {
      for (int w = run0; w < run0 + p.run_words; ++w)
        R::each(data[w], [&](float l, int) {
          if (l > cut) mine += weight(l);
        });
    }
    if (cut_ties > 0)
      for (int w = run0; w < run0 + p.run_words; ++w)
        R::each(data[w], [&](float l, int) { ties += l == cut ? 1u : 0u; });
  }
  u64 pre_m = mine, total = 0;
  uint32_t pre_c = ties, total_c = 0;
  {
    u64 tm;
    uint32_t tc;
    block_scan<kWarps>(pre_m, pre_c, scan_m, scan_c, &tm, &tc, lane, warp);
    if (tid == 0) {
      ctrl.sum = tm;
      ctrl.ties = tc;
      ctrl.draft_weight = 0;
    }
    cluster.sync();
    u64 s = 0;
    uint32_t t = 0;
    if (lane < ranks) {
      const Control* c = cluster.map_shared_rank(&ctrl, lane);
      s = c->sum;
      t = c->ties;
    }
    u64 before = lane < rank ? s : 0ull;
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
      before += __shfl_xor_sync(kAll, before, o);
      s += __shfl_xor_sync(kAll, s, o);
    }
    pre_m += __shfl_sync(kAll, before, 0);
    total = __shfl_sync(kAll, s, 0);
    pre_c += __reduce_add_sync(kAll, lane < rank ? t : 0u);
    total_c = __reduce_add_sync(kAll, t);
    total += w_cut * min(cut_ties, total_c);
  }
  const uint32_t own_ties = min(cut_ties, pre_c + ties) - min(cut_ties, pre_c);   // of this run, kept
  u64 kept = mine + w_cut * own_ties;
  u64 at = pre_m + w_cut * min(cut_ties, pre_c);   // kept weight before this run
  bool accepted = false;
  if constexpr (kVerify) {
    // the draft's own weight, from the thread whose run holds it, to everyone
    const int dw = draft >= 0 && draft < p.vocab ? draft / kPer - e0 / kPer : -1;   // its word in this CTA
    if (dw >= run0 && dw < run0 + p.run_words) {
      uint32_t seen = pre_c;
      float l = 0.f;
      for (int w = run0; w <= dw; ++w)
        R::each(data[w], [&](float x, int h) {
          if (w == dw && h == draft % kPer) l = x;
          if (w < dw || h < draft % kPer) seen += x == cut ? 1u : 0u;
        });
      const u64 v = l > cut ? weight(l) : (l == cut && seen < cut_ties) ? w_cut : 0ull;
      for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(&ctrl, r)->draft_weight = v;
    }
    cluster.sync();
    const u64 draft_w = ctrl.draft_weight;
    if (draft >= 0) {
      const double ua = read_uniform(p.accept_uniform, set * p.accept_stride + (row - set * p.group), p.uniform_bytes);
      accepted = ua * static_cast<double>(total) < static_cast<double>(draft_w);
    }
    // without the draft: its run has less, the runs behind it begin earlier
    total -= draft_w;
    if (draft_w != 0) {
      const int draft_word = draft / kPer, my_word = e0 / kPer + run0;
      if (draft_word < my_word) {
        at -= draft_w;
      } else if (draft_word < my_word + p.run_words) {
        kept -= draft_w;
      }
    }
  }
  const double un = read_uniform(p.uniform, set, p.uniform_bytes);
  u64 want = static_cast<u64>(un * static_cast<double>(total));
  if (total > 0 && want >= total) want = total - 1;
  if (tid == 0) found_thread = -1;
  __syncthreads();
  if (kept > 0 && want >= at && want < at + kept) {
    found_thread = tid;
    found_rest = want - at;
    found_ties = pre_c;
  }
  if (kVerify && total == 0 && rank == 0 && tid == 0)   // nothing but the (then accepted) draft
    p.row_result[row] = make_int2(draft, accepted ? 1 : 0);
  __syncthreads();
  if (found_thread >= 0 && warp == 0) {   // one warp walks the run
    const int first_word = found_thread * p.run_words;
    const int count = p.run_words * kPer;
    u64 rest = found_rest;
    uint32_t seen = found_ties;
    int last = -1;         // the last token with a weight: the tokens' rounded weights may end just short of the run's sum
    uint32_t best = 0;     // (a run of parts below 2^-44 each: its largest)
    int best_token = 0;
    for (int base = 0; base < count; base += 32) {
      const int e = base + lane;
      float l = __int_as_float(0x7FFFFFFF);
      if (e < count)
        R::each(data[first_word + e / kPer], [&](float x, int h) { l = h == e % kPer ? x : l; });
      const bool tie = l == cut;
      const uint32_t tie_vote = __ballot_sync(kAll, tie);
      const bool tie_kept = tie && seen + __popc(tie_vote & ((1u << lane) - 1u)) < cut_ties;
      u64 v = l > cut ? weight(l) : tie_kept ? w_cut : 0ull;
      const int token = e0 + first_word * kPer + e;
      if (kVerify && token == draft) v = 0;
      const uint32_t key = l > -kInf && !(kVerify && token == draft) ? R::key(l) : 0u;
      const uint32_t most = __reduce_max_sync(kAll, key);
      if (most > best) {
        best = most;
        best_token = __shfl_sync(kAll, token, __ffs(__ballot_sync(kAll, key == most)) - 1);
      }
      u64 x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(kAll, x, o);
        if (lane >= o) x += y;
      }
      const uint32_t some = __ballot_sync(kAll, v != 0), hit = __ballot_sync(kAll, x > rest);
      if (some != 0) last = __shfl_sync(kAll, token, 31 - __clz(hit != 0 ? hit & -hit : some));
      if (hit != 0) break;
      rest -= __shfl_sync(kAll, x, 31);
      seen += __popc(tie_vote);
    }
    if (last < 0) last = best != 0 ? best_token : draft;
    if (lane == 0) {
      if constexpr (kVerify) {
        p.row_result[row] = make_int2(last, accepted ? 1 : 0);
      } else {
        p.ids[row] = last;
      }
    }
  }
  cluster.sync();   // nobody's shared memory goes while another CTA reads it
}

// ------------------------------------------------------------------------------------------------ temperature alone
constexpr int kVectors = 8;            // 16-byte vectors of a segment per lane
template <typename T>
constexpr int kSegment = 32 * kVectors * 4 * Row<T>::kPerWord;   // tokens

struct Segment {
  double sum;                          // weights against `top` (equals of an infinite one count 1)
  float top;
  uint32_t first;                      // greedy: first index of the segment's largest logit (or of its first NaN)
};
static_assert(sizeof(Segment) == 16, "Segment");

// The same weights, two at a time, for sums that start at a segment's maximum: the argument 16 log2(e) l / T is reduced in
// single precision with its rounding error carried along (u = n + q, |q| <= 1/2, from the constant's two parts), the
// maximum's own q taken off, so that its weight is 1.  Rounding q and the series leaves 2e-9 of a token's weight, either
// way and different from token to token; the products with the table, and the sums, are in double precision.
// Needs |16 log2(e) l / T| < 2^20.  One double-precision multiply-add and one sum per token instead of eleven operations
// (the segments of 510 rows of 151,936: 86 -> 63 us).
struct PairWeight {
  float c, lo, q0, zero;
  double one;                    // 1 / the maximum's weight as `sum` has it
  const double* table;           // 2^(j / 16), less j << 16 in its high word
  static constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: the sum's low bits are the nearest whole number
  __device__ __forceinline__ PairWeight(float top, const Weight& w, const double* shifted) {
    c = static_cast<float>(w.c);
    lo = static_cast<float>(w.c - static_cast<double>(c));
    const float n = fmaf(top, c, kMagic) - kMagic;
    const float n16 = floorf(n * 0.0625f) * 16.f;      // taken off n, the rest of it stays in the table's index
    zero = kMagic - n16;
    q0 = fmaf(top, lo, fmaf(top, c, -n));
    table = shifted;
    one = 1.0 / w.table[static_cast<int>(n - n16) & 15];
  }
  __device__ __forceinline__ double scaled(float s, int n) const {   // n = 16 e + j: e << 20 with j << 16 below it
    const double t = table[n & 15];
    const double e = __hiloint2double(__double2hiint(t) + (n << 16), __double2loint(t));
    return fma(static_cast<double>(s), e, e);
  }
  __device__ __forceinline__ double sum(float2 l) const {
    const float2 y = ffma2(l, make_float2(c, c), make_float2(zero, zero));
    const float2 n = fsub2(make_float2(zero, zero), y);
    float2 r = ffma2(l, make_float2(lo, lo), ffma2(l, make_float2(c, c), n));
    r = fsub2(r, make_float2(q0, q0));
    float2 s = ffma2(r, make_float2(1.271587195055813e-09f, 1.271587195055813e-09f),
                     make_float2(1.467610032291943e-07f, 1.467610032291943e-07f));
    s = ffma2(s, r, make_float2(1.3550807779497455e-05f, 1.3550807779497455e-05f));
    s = ffma2(s, r, make_float2(0.0009383847928089871f, 0.0009383847928089871f));
    s = ffma2(s, r, make_float2(0.04332169878499658f, 0.04332169878499658f));
    s = fmul2(s, r);
    return scaled(s.x, __float_as_int(y.x)) + scaled(s.y, __float_as_int(y.y));
  }
};

// This lane's words of kCount vectors from token e0 of the row: vector v, lane l are the tokens from
// e0 + ((v * 32 + l) * 4) * kPer.  Tokens past the row are -inf.
template <typename T, int kCount>
__device__ __forceinline__ void load_vectors(const T* row, int vocab, int e0, int lane, uint4 (&x)[kCount]) {
  constexpr int kPer = Row<T>::kPerWord;
  const uint32_t low = kPer == 2 ? 0xFF80FF80u : 0xFF800000u;
  const T* src = row + e0;
  if ((reinterpret_cast<uintptr_t>(src) & 15u) == 0 && e0 + kCount * 128 * kPer <= vocab) {
#pragma unroll
    for (int v = 0; v < kCount; ++v) x[v] = __ldg(reinterpret_cast<const uint4*>(src) + v * 32 + lane);
    return;
  }
#pragma unroll
  for (int v = 0; v < kCount; ++v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = low;
#pragma unroll
      for (int h = 0; h < kPer; ++h) {
        const int e = ((v * 32 + lane) * 4 + i) * kPer + h;
        if (e0 + e < vocab) {
          const uint32_t b = kPer == 2 ? static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(src) + e))
                                       : __ldg(reinterpret_cast<const uint32_t*>(src) + e);
          w[i] = kPer == 2 ? (w[i] & ~(0xFFFFu << (16 * h))) | (b << (16 * h)) : b;
        }
      }
    }
    x[v] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

template <typename T, bool kVerify>
__global__ void __launch_bounds__(256, 4) segment_kernel(const SampleParams p, Segment* __restrict__ segments,
                                                         int per_row) {
  using R = Row<T>;
  constexpr int kPer = R::kPerWord;
  const float kInf = __int_as_float(0x7F800000);
  __shared__ double table[kTable], shifted[kTable];
  if (threadIdx.x < kTable) {
    const double t = exp2(static_cast<double>(threadIdx.x) / kTable);
    table[threadIdx.x] = t;
    shifted[threadIdx.x] = __hiloint2double(__double2hiint(t) - static_cast<int>(threadIdx.x << 16), __double2loint(t));
  }
  const int lane = threadIdx.x & 31;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int row = static_cast<int>(id / per_row), seg = static_cast<int>(id - static_cast<int64_t>(row) * per_row);
  const bool any = row < p.rows && !behind_drafts<kVerify>(p, row);
  uint4 x[kVectors];
  float temp = 0.f;
  const int e0 = seg * kSegment<T>;
  if (any) {
    temp = __ldg(p.temperature + row / p.group);
    load_vectors<T>(static_cast<const T*>(p.logits) + row * p.row_stride, p.vocab, e0, lane, x);
  }
  __syncthreads();
  if (!any) return;
  const bool greedy = !(temp > 0.f);
  const uint32_t low = kPer == 2 ? 0xFF80FF80u : 0xFF800000u;   // -inf
  uint32_t best = low;    // (never NaN)
  bool nan = false;
#pragma unroll
  for (int v = 0; v < kVectors; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i) best = R::larger(best, word_of(x[v], i));
  if (greedy) {
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) R::each(word_of(x[v], i), [&](float l, int) { nan |= l != l; });
  }
  float top = -kInf;
  R::each(best, [&](float l, int) { top = fmaxf(top, l); });
  uint32_t k = __float_as_uint(top + 0.f);
  k = __reduce_max_sync(kAll, (k & 0x80000000u) ? ~k : (k | 0x80000000u));
  top = __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  Segment out;
  out.top = top;
  out.first = 0;
  out.sum = 0.0;
  if (greedy) {
    nan = __any_sync(kAll, nan);
    uint32_t first = kNone;
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        R::each(word_of(x[v], i), [&](float l, int h) {
          const int e = e0 + ((v * 32 + lane) * 4 + i) * kPer + h;
          if (first == kNone && e < p.vocab && (nan ? l != l : l == top)) first = static_cast<uint32_t>(e);
        });
    out.first = __reduce_min_sync(kAll, first);
    if (nan) out.top = __int_as_float(0x7FFFFFFF);
  } else {
    double sum = 0.0;
    if (top - top != 0.f) {
      // an infinite maximum: its equals weigh 1 (segments of nothing but -inf count where the whole row is so)
      int count = 0;
#pragma unroll
      for (int v = 0; v < kVectors; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          R::each(word_of(x[v], i), [&](float l, int h) {
            count += fmaxf(l, -kInf) == top && e0 + ((v * 32 + lane) * 4 + i) * kPer + h < p.vocab ? 1 : 0;
          });
      sum = count;
    } else {
      const Weight weight = make_weight(top, temp, table);
      // about 41 T below, 2^-59; (nearly) every token has a weight, and those that have not (padding and NaN too) count
      // as dust
      const uint32_t dusts = R::both(top - 1.3f * (top - weight.low));
      float dust = 0.f;
      R::each(dusts, [&](float l, int) { dust = l; });
      const PairWeight pair(top, weight, shifted);
      if (top - dust > 36.f * temp && top - dust < 60.f * temp && dust > -FLT_MAX &&
          fmaxf(fabsf(top), fabsf(dust)) * pair.c < 1048576.f) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
          float l[4 * kPer];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            R::each(R::larger(word_of(x[v], i), dusts), [&](float y, int h) { l[i * kPer + h] = y; });
#pragma unroll
          for (int i = 0; i < 4 * kPer; i += 2) sum += pair.sum(make_float2(l[i], l[i + 1]));
        }
        sum *= pair.one;
      } else {
        for (int v = 0; v < kVectors; ++v) {
          const uint4 w = v == 0 ? x[0] : v == 1 ? x[1] : v == 2 ? x[2] : v == 3 ? x[3] : v == 4 ? x[4]
                          : v == 5 ? x[5] : v == 6 ? x[6] : x[7];
          for (int i = 0; i < 4; ++i)
            R::each(word_of(w, i), [&](float l, int) {
              if (l > weight.low) sum += weight.value(l);
            });
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
    out.sum = sum;
  }
  if (lane == 0) segments[id] = out;
}

// One block per row; a thread holds up to four neighbouring segments (blocks of one segment a thread, 512 threads, took one
// SM each: 30 us for 510 rows instead of 9).
constexpr int kDrawThreads = 128;
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr int kDrawSegments = 4;

template <typename T, bool kVerify>
__global__ void __launch_bounds__(kDrawThreads, 4) draw_kernel(const SampleParams p, const Segment* __restrict__ segments,
                                                            int per_row) {
  using R = Row<T>;
  constexpr int kPer = R::kPerWord;
  const float kInf = __int_as_float(0x7F800000);
  static_assert(NVA_MAX_SAMPLE_VOCAB <= kDrawThreads * kDrawSegments * kSegment<float>, "segments of a row");
  __shared__ double table[kTable];
  __shared__ u64 scan_m[kDrawWarps];
  __shared__ uint32_t scan_c[kDrawWarps];
  __shared__ u64 draft_part;             // the draft's weight, as far as its segment's sum has it
  __shared__ u64 found_rest;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x;
  if (behind_drafts<kVerify>(p, row)) return;
  const int set = row / p.group;
  const float temp = __ldg(p.temperature + set);
  const T* src = static_cast<const T*>(p.logits) + row * p.row_stride;
  if (tid < kTable) table[tid] = exp2(static_cast<double>(tid) / kTable + 44.0);
  if (tid == 0) {
    found = 0;
    found_rest = 0;
    draft_part = 0;
  }
  int draft = -1;
  if constexpr (kVerify) {
    const int k = p.group - 1, j = row - set * p.group;
    if (j < k && j < read_id(p.num_drafts, set, p.id_bytes)) {
      const int64_t d = read_id(p.drafts, set * p.draft_stride + j, p.id_bytes);
      draft = d >= 0 && d < p.vocab ? static_cast<int>(d) : p.vocab;
    }
  }
  const int s0 = tid * kDrawSegments;
  Segment seg[kDrawSegments];
#pragma unroll
  for (int i = 0; i < kDrawSegments; ++i) {
    seg[i].top = -kInf;
    seg[i].sum = 0.0;
    seg[i].first = kNone;
    if (s0 + i < per_row) seg[i] = segments[static_cast<int64_t>(row) * per_row + s0 + i];
  }
  auto tell = [&](int token, bool accepted) {
    if constexpr (kVerify) {
      p.row_result[row] = make_int2(token, accepted ? 1 : 0);
    } else {
      p.ids[row] = token;
    }
  };
  // the row's maximum
  auto key = [](float l) {
    const uint32_t k = __float_as_uint(l + 0.f);
    return l != l ? kNone : (k & 0x80000000u) ? ~k : (k | 0x80000000u);
  };
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kDrawSegments; ++i) most = max(most, key(seg[i].top));
  most = __reduce_max_sync(kAll, most);
  if (lane == 0) scan_c[warp] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kDrawWarps; ++w) most = max(most, scan_c[w]);
  __syncthreads();
  if (!(temp > 0.f)) {   // argmax: the first segment with the row's largest holds it
    uint32_t first = kNone;
#pragma unroll
    for (int i = 0; i < kDrawSegments; ++i)
      if (key(seg[i].top) == most) first = min(first, seg[i].first);
    first = __reduce_min_sync(kAll, first);
    if (lane == 0) scan_c[warp] = first;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kDrawWarps; ++w) first = min(first, scan_c[w]);
      tell(static_cast<int>(first), draft == static_cast<int>(first));
    }
    return;
  }
  const float top = __uint_as_float((most & 0x80000000u) ? (most & 0x7FFFFFFFu) : ~most);
  const bool flat = top - top != 0.f;      // infinite: its equals weigh 1
  const Weight weight = make_weight(flat ? 0.f : top, temp, table);
  auto weigh = [&](float l) -> u64 { return flat ? (l == top ? 1ull << 44 : 0ull) : weight(l); };
  u64 draft_w = 0;
  if (kVerify && draft >= 0 && draft < p.vocab) {
    // the draft's weight (every thread: one address)
    const uint32_t b = kPer == 2 ? static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(src) + draft)) << 16
                                 : __ldg(reinterpret_cast<const uint32_t*>(src) + draft);
    const float l = __uint_as_float(b);
    draft_w = weigh(l != l ? -kInf : l);
  }
  // segments against the row's maximum, as whole numbers
  u64 kept[kDrawSegments];
  u64 mine = 0;
#pragma unroll
  for (int i = 0; i < kDrawSegments; ++i) {
    double f = seg[i].top == top ? 1.0 : 0.0;
    if (!flat && seg[i].top != top && seg[i].top > -kInf)
      f = exp((static_cast<double>(seg[i].top) - static_cast<double>(top)) / static_cast<double>(temp));
    kept[i] = static_cast<u64>(__double2ll_rn(seg[i].sum * f * 17592186044416.0));   // 2^44
    if (kVerify && draft >= 0 && s0 + i == draft / kSegment<T>) draft_part = min(draft_w, kept[i]);
    mine += kept[i];
  }
  u64 at = mine, total;
  uint32_t none = 0, none_t;
  block_scan<kDrawWarps>(at, none, scan_m, scan_c, &total, &none_t, lane, warp);
  bool accepted = false;
  if constexpr (kVerify) {
    if (draft >= 0) {
      const double ua = read_uniform(p.accept_uniform, set * p.accept_stride + (row - set * p.group), p.uniform_bytes);
      accepted = ua * static_cast<double>(total) < static_cast<double>(draft_w);
      // without the draft
      const int there = draft / kSegment<T>;
      const u64 less = draft_part;
#pragma unroll
      for (int i = 0; i < kDrawSegments; ++i)
        if (s0 + i == there) kept[i] -= less;
      if (s0 > there) at -= less;
      total -= less;
    }
  }
  const double un = read_uniform(p.uniform, set, p.uniform_bytes);
  u64 want = static_cast<u64>(un * static_cast<double>(total));
  if (total > 0 && want >= total) want = total - 1;
#pragma unroll
  for (int i = 0; i < kDrawSegments; ++i) {
    if (want >= at && want - at < kept[i]) {
      found = s0 + i;
      found_rest = want - at;
    }
    at += kept[i];
  }
  __syncthreads();
  if (total == 0) {         // nothing but the (then accepted) draft
    if (tid == 0) tell(draft, accepted);
    return;
  }
  // the block walks the segment: a share of its vectors each warp, in index order
  constexpr int kShare = kVectors / kDrawWarps;
  const int e0 = found * kSegment<T>, e1 = e0 + warp * kShare * 128 * kPer;
  u64 rest = found_rest;
  u64 w[kShare][4 * kPer], sum[kShare], up_to[kShare], share = 0;
  {
    uint4 x[kShare];
    load_vectors<T>(src, p.vocab, e1, lane, x);
#pragma unroll
    for (int v = 0; v < kShare; ++v) {
      sum[v] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        R::each(word_of(x[v], i), [&](float l, int h) {
          const int e = e1 + ((v * 32 + lane) * 4 + i) * kPer + h;
          u64 y = e < p.vocab ? weigh(l != l ? -kInf : l) : 0ull;
          if (kVerify && e == draft) y = 0;
          w[v][i * kPer + h] = y;
          sum[v] += y;
        });
      up_to[v] = sum[v];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(kAll, up_to[v], o);
        if (lane >= o) up_to[v] += y;
      }
      up_to[v] += share;
      share = __shfl_sync(kAll, up_to[v], 31);
    }
  }
  if (lane == 0) scan_m[warp] = share;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kDrawWarps; ++i) {
    if (i < warp) before += scan_m[i];
    all += scan_m[i];
  }
  if (all != 0) {
    // (the segment's own sum is rounded differently: a number past the last weight draws the last token with one)
    rest = min(rest, all - 1);
#pragma unroll
    for (int v = 0; v < kShare; ++v) {
      u64 run = before + up_to[v] - sum[v];
      if (rest < run || rest - run >= sum[v]) continue;
      int token = -1;
#pragma unroll
      for (int i = 0; i < 4 * kPer; ++i) {
        run += w[v][i];
        if (token < 0 && run > rest) token = e1 + (v * 32 + lane) * 4 * kPer + i;
      }
      tell(token, accepted);
    }
    return;
  }
  // a sum of parts below 2^-44 each: its largest
  if (warp != 0) return;
  uint4 x[kVectors];
  load_vectors<T>(src, p.vocab, e0, lane, x);
  int last;
  {
    uint32_t best = 0;
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        R::each(word_of(x[v], i), [&](float l, int h) {
          const int e = e0 + ((v * 32 + lane) * 4 + i) * kPer + h;
          if (l > -kInf && !(kVerify && e == draft)) best = max(best, key(l));
        });
    best = __reduce_max_sync(kAll, best);
    uint32_t first = kNone;
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        R::each(word_of(x[v], i), [&](float l, int h) {
          const int e = e0 + ((v * 32 + lane) * 4 + i) * kPer + h;
          if (l > -kInf && !(kVerify && e == draft) && key(l) == best) first = min(first, static_cast<uint32_t>(e));
        });
    first = __reduce_min_sync(kAll, first);
    last = first != kNone ? static_cast<int>(first) : draft;
  }
  if (lane == 0) tell(last, accepted);
}

// Accepted drafts of each sequence and the token behind them.
template <typename I>
__global__ void __launch_bounds__(128) verify_merge_kernel(const int2* __restrict__ rows, int32_t sets, int32_t k,
                                                           const I* __restrict__ num_drafts, I* __restrict__ accepted,
                                                           I* __restrict__ next) {
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s >= sets) return;
  const int64_t nd = static_cast<int64_t>(num_drafts[s]);
  int a = 0;
  int2 r = rows[static_cast<int64_t>(s) * (k + 1)];
  while (a < k && a < nd && r.y != 0) r = rows[static_cast<int64_t>(s) * (k + 1) + ++a];
  accepted[s] = static_cast<I>(a);
  next[s] = static_cast<I>(r.x);
}

constexpr int kShareWords = 38 * kThreads;   // of a row per CTA, while more CTAs can be had

// Words per thread of a CTA that holds `words` of a row.
constexpr int run_words(int words) { return ((words + kThreads - 1) / kThreads) | 1; }
constexpr int share_bytes(int words) {
  return std::max(run_words(words) * kThreads * 4, kShort * static_cast<int>(sizeof(u64)));
}
// The most that a call of the type needs: an eighth of the largest vocabulary, or a CTA's share.
template <typename T>
constexpr int kMostBytes = share_bytes(
    std::max(kShareWords, (NVA_MAX_SAMPLE_VOCAB / Row<T>::kPerWord + kMaxCluster - 1) / kMaxCluster));

template <typename T, bool kVerify>
cudaError_t launch_rows(SampleParams p, int sms, cudaStream_t stream) {
  constexpr int kPer = Row<T>::kPerWord;
  const int words = (p.vocab + kPer - 1) / kPer;
  // CTAs per row: a share of at most 78 KB, so that two CTAs fit an SM and one row's exchange runs beside another's
  // loads; more of them (at least 4 KB each) while no SM has to take two, which from two CTAs for three SMs on happens, as
  // a cluster's lie in one part of the chip.  151,936 in bf16, 4 and 8 CTAs a row: top-p 12 rows 50 and 35 us, 16 rows 50
  // and 49; top-k 12 rows 17.7 and 16.6, 16 rows 17.2 and 20.7.
  int cluster = 1;
  while (cluster < kMaxCluster && (words > cluster * kShareWords ||
                                   (3 * static_cast<int64_t>(p.rows) * cluster <= sms && words >= cluster * 2048)))
    cluster *= 2;
  const int per_cta = (words + cluster - 1) / cluster;
  p.run_words = run_words(per_cta);
  p.by_work = static_cast<int64_t>(p.rows) * cluster > 2 * sms && p.rows <= kRowsPerThread * kThreads ? 1 : 0;
  auto kernel = sample_kernel<T, kVerify>;
  // (the same for every call: the limit is the function's, and another thread's smaller call may come before the launch)
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostBytes<T>);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(share_bytes(per_cta));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, bool kVerify>
cudaError_t launch_plain(const SampleParams& p, Segment* segments, cudaStream_t stream) {
  const int per_row = (p.vocab + kSegment<T> - 1) / kSegment<T>;
  const int64_t blocks = (static_cast<int64_t>(p.rows) * per_row + 7) / 8;
  segment_kernel<T, kVerify><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p, segments, per_row);
  draw_kernel<T, kVerify><<<static_cast<unsigned>(p.rows), kDrawThreads, 0, stream>>>(p, segments, per_row);
  return cudaGetLastError();
}

size_t segments_bytes(int64_t rows, int32_t vocab, int32_t elem_bytes) {
  const int tokens = elem_bytes == 2 ? kSegment<__nv_bfloat16> : kSegment<float>;
  return static_cast<size_t>(rows) * static_cast<size_t>((vocab + tokens - 1) / tokens) * sizeof(Segment);
}

// `scratch`: segments_bytes, used without any of top-k, top-p and min-p.
template <bool kVerify>
int launch_sample(const SampleParams& p, int elem_bytes, void* scratch, cudaStream_t stream) {
  cudaError_t e;
  if (p.top_k == nullptr && p.top_p == nullptr && p.min_p == nullptr) {
    Segment* segments = static_cast<Segment*>(scratch);
    e = elem_bytes == 2 ? launch_plain<__nv_bfloat16, kVerify>(p, segments, stream)
                        : launch_plain<float, kVerify>(p, segments, stream);
  } else {
    const int sms = sm_count();
    if (sms == 0) return cuda_fail(cudaGetLastError());
    e = elem_bytes == 2 ? launch_rows<__nv_bfloat16, kVerify>(p, sms, stream)
                        : launch_rows<float, kVerify>(p, sms, stream);
  }
  return e == cudaSuccess ? NVA_OK : cuda_fail(e);
}

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

}  // namespace

}  // namespace nva

extern "C" {

NVA_API int nva_sample_tokens(const void* logits, int64_t row_stride, int32_t rows, int32_t vocab, int32_t elem_bytes,
                              const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                              const void* uniform, int32_t uniform_bytes, int64_t* ids, void* workspace,
                              size_t workspace_bytes, void* stream) {
  if (rows < 0 || vocab < 0) return NVA_ERR_INVALID_ARGUMENT;
  if ((elem_bytes != 2 && elem_bytes != 4) || (uniform_bytes != 4 && uniform_bytes != 8)) return NVA_ERR_UNSUPPORTED;
  if (rows == 0) return NVA_OK;
  if (vocab == 0 || logits == nullptr || row_stride < vocab || temperature == nullptr || uniform == nullptr ||
      ids == nullptr)
    return NVA_ERR_INVALID_ARGUMENT;
  if (vocab > NVA_MAX_SAMPLE_VOCAB || rows > NVA_MAX_SAMPLE_ROWS) return NVA_ERR_UNSUPPORTED;
  if (nva::misaligned(logits, static_cast<uintptr_t>(elem_bytes)) ||
      nva::misaligned(uniform, static_cast<uintptr_t>(uniform_bytes)) || nva::misaligned(ids, 8))
    return NVA_ERR_ALIGNMENT;
  if (top_k == nullptr && top_p == nullptr && min_p == nullptr &&
      (workspace == nullptr || workspace_bytes < nva_sample_workspace_bytes(rows, vocab, elem_bytes) ||
       nva::misaligned(workspace, 16)))
    return NVA_ERR_WORKSPACE;
  nva::SampleParams p{};
  p.logits = logits;
  p.row_stride = row_stride;
  p.rows = rows;
  p.vocab = vocab;
  p.group = 1;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.uniform = uniform;
  p.uniform_bytes = uniform_bytes;
  p.ids = ids;
  return nva::launch_sample<false>(p, elem_bytes, workspace, static_cast<cudaStream_t>(stream));
}

NVA_API size_t nva_sample_workspace_bytes(int32_t rows, int32_t vocab, int32_t elem_bytes) {
  if (rows < 0 || vocab < 0 || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  return static_cast<size_t>(rows) * sizeof(int4) + nva::segments_bytes(rows, vocab, elem_bytes);
}

NVA_API int nva_verify_sampled(const void* logits, int64_t row_stride, int32_t num_seqs, int32_t k, int32_t vocab,
                               int32_t elem_bytes, const void* draft_ids, int64_t draft_row_stride,
                               const void* num_drafts, int32_t id_bytes, const float* temperature,
                               const int32_t* top_k, const float* top_p, const float* min_p,
                               const void* accept_uniform, int64_t accept_row_stride, const void* uniform,
                               int32_t uniform_bytes, void* num_accepted, void* next_tokens, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (num_seqs < 0 || k < 0 || vocab < 0) return NVA_ERR_INVALID_ARGUMENT;
  if ((elem_bytes != 2 && elem_bytes != 4) || (uniform_bytes != 4 && uniform_bytes != 8) ||
      (id_bytes != 4 && id_bytes != 8))
    return NVA_ERR_UNSUPPORTED;
  if (num_seqs == 0) return NVA_OK;
  if (vocab == 0 || logits == nullptr || row_stride < vocab || num_drafts == nullptr || temperature == nullptr ||
      uniform == nullptr || num_accepted == nullptr || next_tokens == nullptr)
    return NVA_ERR_INVALID_ARGUMENT;
  if (k > 0 && (draft_ids == nullptr || draft_row_stride < k || accept_uniform == nullptr || accept_row_stride < k))
    return NVA_ERR_INVALID_ARGUMENT;
  const int64_t rows = static_cast<int64_t>(num_seqs) * (static_cast<int64_t>(k) + 1);
  if (vocab > NVA_MAX_SAMPLE_VOCAB || rows > NVA_MAX_SAMPLE_ROWS) return NVA_ERR_UNSUPPORTED;
  const uintptr_t ub = static_cast<uintptr_t>(uniform_bytes), ib = static_cast<uintptr_t>(id_bytes);
  if (nva::misaligned(logits, static_cast<uintptr_t>(elem_bytes)) || nva::misaligned(uniform, ub) ||
      (k > 0 && (nva::misaligned(accept_uniform, ub) || nva::misaligned(draft_ids, ib))) ||
      nva::misaligned(num_drafts, ib) || nva::misaligned(num_accepted, ib) || nva::misaligned(next_tokens, ib))
    return NVA_ERR_ALIGNMENT;
  if (workspace == nullptr || workspace_bytes < (top_k != nullptr || top_p != nullptr || min_p != nullptr
                             ? static_cast<size_t>(rows) * sizeof(int4)
                             : nva_sample_workspace_bytes(static_cast<int32_t>(rows), vocab, elem_bytes)) ||
      nva::misaligned(workspace, 16))
    return NVA_ERR_WORKSPACE;
  nva::SampleParams p{};
  p.logits = logits;
  p.row_stride = row_stride;
  p.rows = static_cast<int32_t>(rows);
  p.vocab = vocab;
  p.group = k + 1;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.uniform = uniform;
  p.uniform_bytes = uniform_bytes;
  p.drafts = draft_ids;
  p.draft_stride = draft_row_stride;
  p.num_drafts = num_drafts;
  p.id_bytes = id_bytes;
  p.accept_uniform = accept_uniform;
  p.accept_stride = accept_row_stride;
  // the rows' results, then the segments (16 bytes a row: the segments stay aligned)
  p.row_result = static_cast<int2*>(workspace);
  void* scratch = static_cast<uint8_t*>(workspace) + static_cast<size_t>(rows) * sizeof(int4);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = nva::launch_sample<true>(p, elem_bytes, scratch, s);
  if (rc != NVA_OK) return rc;
  const unsigned blocks = static_cast<unsigned>((num_seqs + 127) / 128);
  if (id_bytes == 4)
    nva::verify_merge_kernel<int32_t><<<blocks, 128, 0, s>>>(
        p.row_result, num_seqs, k, static_cast<const int32_t*>(num_drafts), static_cast<int32_t*>(num_accepted),
        static_cast<int32_t*>(next_tokens));
  else
    nva::verify_merge_kernel<int64_t><<<blocks, 128, 0, s>>>(
        p.row_result, num_seqs, k, static_cast<const int64_t*>(num_drafts), static_cast<int64_t*>(num_accepted),
        static_cast<int64_t*>(next_tokens));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? NVA_OK : nva::cuda_fail(e);
}

}  // extern "C"
