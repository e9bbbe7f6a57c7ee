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
// rounded from a double-precision exponential (relative error 1e-16: a table of 2^(j/256) and four terms of the
// exponential series), and every sum is an exact 64-bit integer sum: no order of additions, atomics included, can change
// a result.  Weights below 2^-45 are 0.
//
// One pass over HBM: a cluster of CTAs keeps a row in its shared memory (V = 151,936 in bf16: four CTAs of 76 KB) as
// order-preserving integer keys.  Thresholds of top-k and top-p come from histograms (counts, or fixed-point weights)
// over 1024 bins, first of equal width in l (so that neighbouring logits rarely meet in one bin), then of the crossing
// bin's keys until one key is left; at that key the first m equal tokens stay, in index order.  CTAs exchange maxima,
// histograms and sums through distributed shared memory.  For the draw every thread owns a run of consecutive tokens, a
// prefix sum over threads and CTAs names the run that holds u * W, and one warp walks it.
// Bound: the double-precision exponentials, one per token that no threshold removes (a row with top-k only takes them
// for the k kept ones), next to the one read of the logits.
#include <cooperative_groups.h>

#include <algorithm>
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
constexpr int kTable = 256;
constexpr int kMaxCluster = 8;
constexpr float kReach = 31.5f;        // exp(-31.5) < 2^-45: weight 0
constexpr uint32_t kAll = 0xffffffffu;
using u64 = unsigned long long;

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  int32_t rows, vocab;
  int32_t run_words;                   // 32-bit words of a row per thread (odd: neighbouring threads, other banks)
  int32_t group;                       // rows that share one set of settings: 1, or k + 1 (verify)
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
  u64 before;                          // count or weight above the current key range
  uint32_t lo, hi;                     // its keys
  uint32_t bin;
  u64 draft_weight;
  u64 sum;                             // this CTA's kept weight (equals of the threshold key apart) ...
  uint32_t ties;                       // ... and number of tokens at that key
  uint32_t top;                        // its largest key
  uint32_t first;                      // its first index of the row's largest key
};

template <typename T>
struct KeyOf;
// Order-preserving keys; 0 is padding.  -0 equals +0.  NaN: above everything when greedy, else -inf.
template <>
struct KeyOf<__nv_bfloat16> {
  static constexpr int kPerWord = 2;
  static __device__ __forceinline__ uint32_t one(uint32_t b, bool greedy) {
    if ((b & 0x7FFFu) > 0x7F80u) b = greedy ? 0x7FFFu : 0xFF80u;
    if (b == 0x8000u) b = 0u;
    return (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
  }
  static __device__ __forceinline__ uint32_t word(uint32_t w, bool greedy) {
    return one(w & 0xFFFFu, greedy) | (one(w >> 16, greedy) << 16);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(((k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu)) << 16);
  }
};
template <>
struct KeyOf<float> {
  static constexpr int kPerWord = 1;
  static __device__ __forceinline__ uint32_t one(uint32_t b, bool greedy) {
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) b = greedy ? 0x7FFFFFFFu : 0xFF800000u;
    if (b == 0x80000000u) b = 0u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  }
  static __device__ __forceinline__ uint32_t word(uint32_t w, bool greedy) { return one(w, greedy); }
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

// w * 2^44 of one logit, rounded: 2^(u / 256) with u = 256 log2(e) (l - m) / T = 256 e + j + r, |r| <= 1/2.
struct Weight {
  double m, c;           // row maximum, 256 log2(e) / T
  float mf, reach;       // row maximum, kReach * T
  const double* table;   // 2^(j / 256)
  __device__ __forceinline__ u64 operator()(float l) const {
    if (l == mf) return 1ull << 44;
    if (!(mf - l <= reach)) return 0ull;
    const double u = (static_cast<double>(l) - m) * c;
    const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are rint(u)
    const double n = u + magic;
    const double r = u - (n - magic);
    const int k = __double2loint(n);           // >= -256 * 45.5
    // 2^(r / 256), four terms in a = r ln 2 / 256 (|a| <= 0.00136: the fifth is below 4e-17)
    const double a = r * 0.0027076061740622863;
    double s = fma(a, 0.041666666666666664, 0.16666666666666666);
    s = fma(a, s, 0.5);
    s = fma(a, s, 1.0);
    s = fma(a, s, 1.0);
    // times 2^(j / 256) * 2^(e + 44), rounded to a whole number by adding 2^52
    const double scale = __hiloint2double(((k >> 8) + 44 + 1023) << 20, 0);
    const double y = fma(s * table[k & 255], scale, 4503599627370496.0);
    return __double_as_longlong(y) & 0xFFFFFFFFFFFFFull;
  }
};

// Block-wide exclusive prefix sums of a weight and a count; `tot` receives the block's sums.
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
  for (int w = 0; w < kWarps; ++w) {
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
  using K = KeyOf<T>;
  constexpr int kPer = K::kPerWord;
  constexpr uint32_t kKeyMask = kPer == 2 ? 0xFFFFu : 0xFFFFFFFFu;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / ranks;

  extern __shared__ __align__(16) uint8_t smem[];
  const int words = p.run_words * kThreads;
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  __shared__ uint32_t hist[3][kBins];          // counts; weights, low and high words
  __shared__ double table[kTable];
  __shared__ u64 scan_m[kWarps];
  __shared__ uint32_t scan_c[kWarps];
  __shared__ Control ctrl;
  __shared__ int found_thread;
  __shared__ u64 found_rest;
  __shared__ uint32_t found_ties;

  const int set = row / p.group;
  const float temp = __ldg(p.temperature + set);
  const bool greedy = !(temp > 0.f);

  // ---------------------------------------------------------------- the row, as keys
  const int e0 = rank * words * kPer;          // first token of this CTA
  const int n = max(0, min(p.vocab - e0, words * kPer));
  uint32_t top = 0;
  {
    const T* src = static_cast<const T*>(p.logits) + row * p.row_stride + e0;
    const uint32_t* src32 = reinterpret_cast<const uint32_t*>(src);
    auto best = [&](uint32_t w) {
      top = kPer == 2 ? __vmaxu2(top, w) : max(top, w);
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
          if (v0 + i * kThreads < nv) {
            uint4 k;
            k.x = K::word(raw[i].x, greedy);
            k.y = K::word(raw[i].y, greedy);
            k.z = K::word(raw[i].z, greedy);
            k.w = K::word(raw[i].w, greedy);
            best(k.x);
            best(k.y);
            best(k.z);
            best(k.w);
            reinterpret_cast<uint4*>(keys)[v0 + i * kThreads] = k;
          }
      }
      done = nv * 4;
    }
    for (int w = done + tid; w < words; w += kThreads) {
      uint32_t k = 0;
#pragma unroll
      for (int h = 0; h < kPer; ++h) {
        const int e = w * kPer + h;
        if (e < n) {
          const uint32_t b = kPer == 2 ? static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(src) + e))
                                       : __ldg(src32 + e);
          k |= K::one(b, greedy) << (16 * h);
        }
      }
      best(k);
      keys[w] = k;
    }
    if (tid < kTable) table[tid] = exp2(static_cast<double>(tid) / kTable);
    if (kPer == 2) top = max(top & 0xFFFFu, top >> 16);
    top = __reduce_max_sync(kAll, top);
    if (lane == 0) scan_c[warp] = top;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) top = max(top, scan_c[w]);
      ctrl.top = top;
    }
  }
  cluster.sync();
  top = 0;
  for (int r = 0; r < ranks; ++r) top = max(top, cluster.map_shared_rank(&ctrl, r)->top);

  // this CTA's tokens of one word
  auto each = [&](uint32_t w, auto&& f) {
    f(w & kKeyMask, 0);
    if constexpr (kPer == 2) f(w >> 16, 1);
  };
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
    // ---------------------------------------------------------------- argmax: the first index of the largest key
    uint32_t first = 0xFFFFFFFFu;
    for (int w = run0; w < run0 + p.run_words && first == 0xFFFFFFFFu; ++w)
      each(keys[w], [&](uint32_t k, int h) {
        if (k == top && first == 0xFFFFFFFFu) first = static_cast<uint32_t>(e0 + w * kPer + h);
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

  // ---------------------------------------------------------------- thresholds
  Weight weight;
  weight.mf = K::value(top);
  weight.m = weight.mf;
  weight.c = 369.3299304675746 / static_cast<double>(temp);   // 256 log2(e)
  weight.reach = fminf(kReach * temp, 3.0e38f);   // (-inf stays out at an infinite temperature)
  weight.table = table;
  // tokens below it are gone (the keys under -inf's are no numbers)
  const uint32_t least = K::one(kPer == 2 ? 0xFF80u : 0xFF800000u, false);
  uint32_t floor_key = least;
  if (p.min_p != nullptr) {
    const double mp = fmin(static_cast<double>(__ldg(p.min_p + set)), 1.0);
    if (mp > 0.0) {
      const double at = weight.m + static_cast<double>(temp) * log(mp);   // l >= at
      float f = static_cast<float>(at);
      if (static_cast<double>(f) < at) f = nextafterf(f, __int_as_float(0x7F800000));
      if (f == f) {
        if constexpr (kPer == 2) {
          // the least bf16 at or above f: round its bits up (away from zero when positive, towards it when negative)
          uint32_t b = __float_as_uint(f);
          b = (b & 0x80000000u) ? (b >> 16) : ((b + 0xFFFFu) >> 16);
          floor_key = max(least, K::one(b, false));
        } else {
          floor_key = max(least, K::one(__float_as_uint(f), false));
        }
      }
    }
  }
  uint32_t cut = floor_key - 1;                // kept: keys above it, and the first `cut_ties` tokens at it
  uint32_t cut_ties = 0;
  const float bin_scale = (kBins / 32.0f) / temp;
  auto linear_bin = [&](uint32_t k) {          // rises as the key falls
    return min(kBins - 1, __float2int_rz((weight.mf - K::value(k)) * bin_scale));
  };
  // The key at which the running count (or weight) from the top reaches `target`, and what lies above it.  Tokens
  // eligible: keys above `cut`, and `cut_ties` tokens at it.
  auto select = [&](auto by_weight, double target, u64& before) -> uint32_t {
    constexpr bool kMass = decltype(by_weight)::value;
    uint32_t lo = cut_ties > 0 ? cut : cut + 1, hi = top;
    before = 0;
    bool linear = true;
    while (true) {
      const int shift = linear ? 0 : max(0, 32 - __clz(hi - lo) - 10);
      for (int i = tid; i < kBins; i += kThreads) {
        hist[0][i] = 0;
        if constexpr (kMass) hist[1][i] = hist[2][i] = 0;
      }
      __syncthreads();
      auto bin_of = [&](uint32_t k) { return linear ? linear_bin(k) : static_cast<int>((hi - k) >> shift); };
      auto add_mass = [&](int b, u64 v) {
        const uint32_t x = static_cast<uint32_t>(v);
        const uint32_t old = atomicAdd(&hist[1][b], x);
        const uint32_t up = static_cast<uint32_t>(v >> 32) + (old + x < old ? 1u : 0u);
        if (up != 0) atomicAdd(&hist[2][b], up);
      };
      for (int w = tid; w < words; w += kThreads)
        each(keys[w], [&](uint32_t k, int) {
          if (k < lo || k > hi || (kMass && k == cut)) return;
          if constexpr (kMass) {
            const u64 v = weight(K::value(k));
            if (v != 0) add_mass(bin_of(k), v);
          } else {
            atomicAdd(&hist[0][bin_of(k)], 1u);
          }
        });
      if (kMass && rank == 0 && tid == 0 && cut_ties > 0 && lo <= cut && cut <= hi)
        add_mass(bin_of(cut), cut_ties * weight(K::value(cut)));
      cluster.sync();
      if (rank == 0) {   // merge the CTAs' bins, two per thread, and find the crossing
        u64 v[2] = {0, 0};
        for (int r = 0; r < ranks; ++r) {
          const uint32_t* h = cluster.map_shared_rank(&hist[0][0], r);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int b = 2 * tid + i;
            v[i] += kMass ? h[kBins + b] + (static_cast<u64>(h[2 * kBins + b]) << 32) : static_cast<u64>(h[b]);
          }
        }
        u64 pre = v[0] + v[1], tot;
        uint32_t none = 0, none_t;
        block_scan(pre, none, scan_m, scan_c, &tot, &none_t, lane, warp);
        pre += before;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (v[i] != 0 && static_cast<double>(pre) < target && static_cast<double>(pre + v[i]) >= target)
            for (int r = 0; r < ranks; ++r) {
              Control* c = cluster.map_shared_rank(&ctrl, r);
              c->bin = static_cast<uint32_t>(2 * tid + i);
              c->before = pre;
            }
          pre += v[i];
        }
      }
      cluster.sync();
      const uint32_t bin = ctrl.bin;
      before = ctrl.before;
      if (linear) {
        // the keys of the crossing bin: [least with linear_bin <= bin, largest with linear_bin >= bin], each by a
        // 32-way search
        auto search = [&](auto pred, uint32_t a, uint32_t b) {   // least key in [a, b] with pred, which holds at b
          while (a < b) {
            const uint32_t step = (b - a) / 32 + 1;
            const u64 far = a + static_cast<u64>(step) * lane;
            const uint32_t x = far < b ? static_cast<uint32_t>(far) : b;
            const uint32_t yes = __ballot_sync(kAll, x == b || pred(x));
            const int f = yes != 0 ? __ffs(yes) - 1 : 32;   // points below f: no, point f: yes
            const uint32_t below = __shfl_sync(kAll, x, f > 0 ? f - 1 : 0);
            const uint32_t at = __shfl_sync(kAll, x, f < 32 ? f : 0);
            if (f > 0) a = below + 1;
            b = f == 0 ? a : f < 32 ? at : b;
          }
          return b;
        };
        const int ib = static_cast<int>(bin);
        const uint32_t nlo = search([&](uint32_t k) { return linear_bin(k) <= ib; }, lo, hi);
        const uint32_t past = ib == 0 ? hi + 1 : search([&](uint32_t k) { return linear_bin(k) < ib; }, nlo, hi);
        lo = nlo;
        hi = ib == 0 ? hi : max(nlo, past - 1);
        linear = false;
      } else {
        const uint32_t nhi = hi - (bin << shift);
        lo = (nhi - lo) >> shift == 0 ? lo : nhi - ((1u << shift) - 1u);
        hi = nhi;
      }
      if (lo == hi) return lo;
    }
  };

  if (p.top_k != nullptr) {
    const int k = __ldg(p.top_k + set);
    if (k > 0 && k < p.vocab) {
      // fewer than k tokens may have passed min-p: count them first
      uint32_t c = 0;
      if (floor_key > least) {
        for (int w = tid; w < words; w += kThreads)
          each(keys[w], [&](uint32_t key, int) { c += key > cut ? 1u : 0u; });
        u64 none = 0, tm;
        uint32_t tc;
        block_scan(none, c, scan_m, scan_c, &tm, &tc, lane, warp);
        if (tid == 0) ctrl.ties = tc;
        cluster.sync();
        c = 0;
        for (int r = 0; r < ranks; ++r) c += cluster.map_shared_rank(&ctrl, r)->ties;
        cluster.sync();
      } else {
        c = static_cast<uint32_t>(p.vocab);
      }
      if (c > static_cast<uint32_t>(k)) {
        u64 above;
        cut = select(std::false_type{}, static_cast<double>(k), above);
        cut_ties = static_cast<uint32_t>(k - static_cast<int>(above));
      }
    }
  }
  // kept weight of this thread's run and of the runs and CTAs before it
  u64 mine, total, pre_m;
  uint32_t ties, pre_c, total_c;
  auto sums = [&](u64 w_cut) {
    mine = 0;
    ties = 0;
    for (int w = run0; w < run0 + p.run_words; ++w)
      each(keys[w], [&](uint32_t k, int) {
        if (k > cut) mine += weight(K::value(k));
        ties += k == cut ? 1u : 0u;
      });
    pre_m = mine;
    pre_c = ties;
    u64 tm;
    uint32_t tc;
    block_scan(pre_m, pre_c, scan_m, scan_c, &tm, &tc, lane, warp);
    if (tid == 0) {
      ctrl.sum = tm;
      ctrl.ties = tc;
    }
    cluster.sync();
    total = 0;
    total_c = 0;
    for (int r = 0; r < ranks; ++r) {
      const Control* c = cluster.map_shared_rank(&ctrl, r);
      const u64 s = c->sum;
      const uint32_t t = c->ties;
      if (r < rank) {
        pre_m += s;
        pre_c += t;
      }
      total += s;
      total_c += t;
    }
    // the first cut_ties tokens at the cut, in index order
    total += w_cut * min(cut_ties, total_c);
  };
  auto cut_weight = [&]() { return cut_ties > 0 ? weight(K::value(cut)) : 0ull; };

  if (p.top_p != nullptr) {
    const double tp = __ldg(p.top_p + set);
    if (tp < 1.0) {
      sums(cut_weight());
      cluster.sync();   // (the controls are read; select writes them)
      u64 above;
      const double target = fmax(tp, 0.0) * static_cast<double>(total);
      // (the first token always stays: a target of 0 would find no crossing)
      const uint32_t key = select(std::true_type{}, fmax(target, 1.0), above);
      const double w = static_cast<double>(weight(K::value(key)));
      const double want = ceil((fmax(target, 1.0) - static_cast<double>(above)) / w);
      const uint32_t limit = key == cut ? cut_ties : 0xFFFFFFFFu;
      cut = key;
      cut_ties = min(limit, static_cast<uint32_t>(fmin(fmax(want, 1.0), 4.0e9)));
    }
  }

  // ---------------------------------------------------------------- the draw
  const u64 w_cut = cut_weight();
  sums(w_cut);
  const uint32_t own_ties = min(cut_ties, pre_c + ties) - min(cut_ties, pre_c);   // of this run, kept
  u64 kept = mine + w_cut * own_ties;
  u64 at = pre_m + w_cut * min(cut_ties, pre_c);   // kept weight before this run
  u64 draft_w = 0;
  bool accepted = false;
  if constexpr (kVerify) {
    // the draft's own weight, from the thread whose run holds it, to everyone
    const int dw = draft >= 0 && draft < p.vocab ? draft / kPer - e0 / kPer : -1;   // its word in this CTA
    if (tid == 0) ctrl.draft_weight = 0;
    cluster.sync();
    if (dw >= run0 && dw < run0 + p.run_words) {
      uint32_t seen = pre_c, key = 0;
      for (int w = run0; w <= dw; ++w)
        each(keys[w], [&](uint32_t k, int h) {
          if (w == dw && h == draft % kPer) key = k;
          if (w < dw || h < draft % kPer) seen += k == cut ? 1u : 0u;
        });
      const u64 v = key > cut ? weight(K::value(key)) : (key == cut && seen < cut_ties) ? w_cut : 0ull;
      for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(&ctrl, r)->draft_weight = v;
    }
    cluster.sync();
    draft_w = ctrl.draft_weight;
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
    for (int base = 0; base < count; base += 32) {
      const int e = base + lane;
      uint32_t k = 0;
      if (e < count) {
        const uint32_t w = keys[first_word + e / kPer];
        k = kPer == 2 ? ((e & 1) ? w >> 16 : w & 0xFFFFu) : w;
      }
      const bool tie = k == cut;
      const uint32_t tie_vote = __ballot_sync(kAll, tie);
      const bool tie_kept = tie && seen + __popc(tie_vote & ((1u << lane) - 1u)) < cut_ties;
      u64 v = k > cut ? weight(K::value(k)) : tie_kept ? w_cut : 0ull;
      const int token = e0 + first_word * kPer + e;
      if (kVerify && token == draft) v = 0;
      u64 x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(kAll, x, o);
        if (lane >= o) x += y;
      }
      const uint32_t hit = __ballot_sync(kAll, x > rest);
      if (hit != 0) {
        if (lane == __ffs(hit) - 1) {
          if constexpr (kVerify) {
            p.row_result[row] = make_int2(token, accepted ? 1 : 0);
          } else {
            p.ids[row] = token;
          }
        }
        break;
      }
      rest -= __shfl_sync(kAll, x, 31);
      seen += __popc(tie_vote);
    }
  }
  cluster.sync();   // nobody's shared memory goes while another CTA reads it
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

template <typename T, bool kVerify>
cudaError_t launch_rows(SampleParams p, int sms, cudaStream_t stream) {
  constexpr int kPer = KeyOf<T>::kPerWord;
  const int words = (p.vocab + kPer - 1) / kPer;
  // CTAs per row: a share of at most 80 KB, so that two CTAs fit an SM and one row's exchange runs beside another's
  // loads; more of them when there are few rows (but at least 4 KB each)
  int cluster = 1;
  while (cluster < kMaxCluster &&
         (words > cluster * 20480 || (static_cast<int64_t>(p.rows) * cluster * 2 <= 2 * sms && words >= cluster * 2048)))
    cluster *= 2;
  const int per_cta = (words + cluster - 1) / cluster;
  p.run_words = ((per_cta + kThreads - 1) / kThreads) | 1;
  const size_t smem = static_cast<size_t>(p.run_words) * kThreads * 4;
  auto kernel = sample_kernel<T, kVerify>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <bool kVerify>
int launch_sample(const SampleParams& p, int elem_bytes, cudaStream_t stream) {
  const int sms = sm_count();
  if (sms == 0) return cuda_fail(cudaGetLastError());
  const cudaError_t e = elem_bytes == 2 ? launch_rows<__nv_bfloat16, kVerify>(p, sms, stream)
                                        : launch_rows<float, kVerify>(p, sms, stream);
  return e == cudaSuccess ? NVA_OK : cuda_fail(e);
}

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

}  // namespace

}  // namespace nva

extern "C" {

NVA_API int nva_sample_tokens(const void* logits, int64_t row_stride, int32_t rows, int32_t vocab, int32_t elem_bytes,
                              const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                              const void* uniform, int32_t uniform_bytes, int64_t* ids, void* stream) {
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
  return nva::launch_sample<false>(p, elem_bytes, static_cast<cudaStream_t>(stream));
}

NVA_API size_t nva_verify_sampled_workspace_bytes(int32_t num_seqs, int32_t k) {
  return num_seqs < 0 || k < 0 ? 0 : static_cast<size_t>(num_seqs) * (static_cast<size_t>(k) + 1) * sizeof(int2);
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
  if (workspace == nullptr || workspace_bytes < nva_verify_sampled_workspace_bytes(num_seqs, k) ||
      nva::misaligned(workspace, 8))
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
  p.row_result = static_cast<int2*>(workspace);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = nva::launch_sample<true>(p, elem_bytes, s);
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
