// sample_rows.cu -- temperature / top-k / top-p / min-p sampling of rows of
// logits from given uniform numbers (sm_100a).
//
// A token's place in the order (logit descending, index ascending) is one
// 64-bit number, (order key of the logit) << 32 | ~index, so that ties need no
// care: every filter keeps the tokens at or above some number.  Weights
// w = exp((l - largest) / T) are integers of 2^-45 (f64 arithmetic), whose
// sums do not depend on their order.
//
// A row of at most kList logits is a list in one CTA's shared memory.  A longer
// row lies in the shared memory of a cluster of CTAs, its logits read from HBM
// once, and is cut down to a list:
//   small top-k: the least of the CTAs' own (k / CTAs)-th largest thread
//     maxima has k logits above it and few more; those are the list;
//   otherwise a histogram over (largest - l) / T of counts (top-k) or weights
//     (top-p) gives the bin in which the last kept token lies, and that bin's
//     tokens are the list.
// In a list the token at which the running count or weight reaches a target is
// found by histograms over the range that still holds it, until one warp can
// put the rest in order.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "engine.h"
#include "kv8.h"

namespace cg = cooperative_groups;

namespace qtts {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kFix = 45;     // fraction bits of a weight: 2^18 weights of 1 stay below 2^63
constexpr int kList = 2048;  // tokens of a list
constexpr int kBins = 1024;
typedef unsigned long long u64;

struct SampleRowsDesc {
  const void* logits = nullptr;
  long ld = 0;
  int V = 0, per = 0;  // columns, columns of a CTA
  const float* temperature = nullptr;
  const int* top_k = nullptr;
  const float *top_p = nullptr, *min_p = nullptr, *u = nullptr;
  int *token = nullptr, *kept = nullptr;
  float* logprob = nullptr;
};

// Order keys: larger for a larger logit, equal for the two zeros, 0 for what is
// never drawn (NaN, -inf).  A 16-bit logit has a 16-bit key.
template <typename T>
struct Key {  // f16, bf16
  using Stored = uint16_t;
  static __device__ __forceinline__ float f32(uint32_t bits) {
    const uint16_t b = (uint16_t)bits;
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(b));
    else return __uint_as_float((uint32_t)b << 16);
  }
  static __device__ __forceinline__ uint32_t of(uint32_t bits) {
    constexpr uint32_t inf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    const uint32_t mag = bits & 0x7fffu;
    const uint32_t k = bits & 0x8000u ? 0x8000u - mag : 0x8000u + mag;
    return mag > inf || bits == (0x8000u | inf) ? 0u : k;
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return f32(k >= 0x8000u ? k - 0x8000u : 0x8000u | (0x8000u - k));
  }
};
template <>
struct Key<float> {
  using Stored = uint32_t;
  static __device__ __forceinline__ uint32_t of(uint32_t bits) {
    const float l = __uint_as_float(bits);
    return l > -INFINITY ? f32_order_key(l) : 0u;
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  }
};
__device__ __forceinline__ u64 place_of(uint32_t key, int index) { return ((u64)key << 32) | (uint32_t)~index; }
__device__ __forceinline__ uint32_t key_in(u64 place) { return (uint32_t)(place >> 32); }

struct Weigh {
  float top;  // the largest logit
  float inv_tf;
  double inv_t;
  const double* exp2_32;  // 2^(i / 32)
  __device__ __forceinline__ double z(float l) const {
    const double x = ((double)l - (double)top) * inv_t;
    return l == top ? 0.0 : x <= 0.0 ? x : -INFINITY;  // an infinite top over an infinite temperature is no number
  }
  // false: the weight is surely 0 (z < -34 whatever the f32 roundings)
  __device__ __forceinline__ bool counts(float l) const { return !((top - l) * inv_tf > 34.0f); }
  // exp(z) 2^45 to the nearest integer: z = n ln2/32 + r, exp(r) by its series
  // to r^5 (|r| < 0.011: 2e-15), 2^(n/32) by table and exponent.  Below -33
  // (a weight of less than 1/8 of 2^-45) it is 0.
  __device__ __forceinline__ u64 of_z(double x) const {
    const bool some = x > -33.0;
    x = some ? x : -33.0;
    const double shift = 0x1.8p52;
    const double nd = __fma_rn(x, 46.166241308446828, shift);  // 32 / ln 2
    const int n = __double2loint(nd);
    const double r = __fma_rn(nd - shift, -0.021660849392498290, x);  // ln 2 / 32
    double p = __fma_rn(r, 1.0 / 120.0, 1.0 / 24.0);
    p = __fma_rn(p, r, 1.0 / 6.0);
    p = __fma_rn(p, r, 0.5);
    p = __fma_rn(p, r, 1.0);
    p = __fma_rn(p, r, 1.0);
    const double t = exp2_32[n & 31];
    const double s = __hiloint2double(__double2hiint(t) + (((n >> 5) + kFix) << 20), __double2loint(t));
    const double w = __fma_rn(s, p, 0x1p52);  // the sum's mantissa is the integer
    return some ? (u64)(__double_as_longlong(w) - __double_as_longlong(0x1p52)) : 0;
  }
  __device__ __forceinline__ u64 operator()(float l) const { return of_z(z(l)); }
};

// Histogram bins: counts, and weights as three words of 15 bits, whose sums of
// up to 2^17 tokens stay in 32 bits (64-bit shared atomics are retry loops).
struct Bins {
  unsigned count[kBins];
  unsigned w[3][kBins];
  __device__ __forceinline__ void add(int b, u64 weight) {
    const unsigned lo = (unsigned)weight & 0x7fffu, mid = (unsigned)(weight >> 15) & 0x7fffu, hi = (unsigned)(weight >> 30);
    if (lo) atomicAdd(&w[0][b], lo);
    if (mid) atomicAdd(&w[1][b], mid);
    if (hi) atomicAdd(&w[2][b], hi);
  }
  __device__ __forceinline__ u64 weight(int b) const { return (u64)w[0][b] + ((u64)w[1][b] << 15) + ((u64)w[2][b] << 30); }
};

constexpr int kFew = 32;  // tokens that one warp puts in order
struct Shared {
  Bins bins;
  union {
    u64 list[kList];
    struct {  // cluster: this CTA's share of the merged bins, read before any list is made
      u64 weight[kBins];
      unsigned count[kBins];
    } merged;
  };
  u64 weight[kList];  // of the list; before it is made, this CTA's part of the list
  u64 few[kFew], few_weight[kFew];
  double exp2_32[32];
  u64 scan[33];
  u64 word[4];            // what this CTA tells the cluster
  unsigned part[32];      // tokens in this CTA's part of the list, by warp
  unsigned offset[8 * 32];
  u64 found_before;
  unsigned found_bin, found_n, n;
};

enum Mode { COUNT, WEIGHT };

template <int TH>
struct Block {
  static constexpr int kWarps = TH / 32;
  Shared& sh;
  const int tid = threadIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __device__ explicit Block(Shared& s) : sh(s) {}

  template <typename Op>
  __device__ __forceinline__ u64 reduce(u64 v, Op op) {  // every thread gets the result
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(kFull, v, o));
    __syncthreads();
    if (lane == 0) sh.scan[warp] = v;
    __syncthreads();
    v = sh.scan[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v = op(v, sh.scan[w]);
    return v;
  }
  __device__ __forceinline__ u64 sum(u64 v) {
    return reduce(v, [](u64 a, u64 b) { return a + b; });
  }
  __device__ __forceinline__ u64 most(u64 v) {
    return reduce(v, [](u64 a, u64 b) { return a > b ? a : b; });
  }
  __device__ __forceinline__ u64 least(u64 v) {
    return reduce(v, [](u64 a, u64 b) { return a < b ? a : b; });
  }
  // exclusive prefix over the threads, and the total
  __device__ __forceinline__ u64 prefix(u64 v, u64* total) {
    u64 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(kFull, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh.scan[warp] = x;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const u64 s = sh.scan[w];
      if (w < warp) before += s;
      all += s;
    }
    *total = all;
    return before + x - v;
  }
  __device__ __forceinline__ void clear(Mode mode) {
    for (int i = tid; i < kBins; i += TH) {
      sh.bins.count[i] = 0;
      if (mode == WEIGHT) sh.bins.w[0][i] = sh.bins.w[1][i] = sh.bins.w[2][i] = 0;
    }
    __syncthreads();
  }
  // Of kBins values (value(b), bin 0 first) the bin in which the running sum
  // reaches target(total) (clamped to the total): found_bin, found_n,
  // found_before.  Returns the target.
  template <typename Target, typename Value, typename Count>
  __device__ __forceinline__ u64 find(Target target_of, Value value, Count count) {
    constexpr int N = kBins / TH;
    u64 v[N], own = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[j] = value(tid * N + j);
      own += v[j];
    }
    u64 total;
    u64 run = prefix(own, &total);
    const u64 want = target_of(total), target = want > total ? total : want;
    if (run < target && target <= run + own) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (run < target && target <= run + v[j]) {
          sh.found_bin = tid * N + j;
          sh.found_n = count(tid * N + j);
          sh.found_before = run;
        }
        run += v[j];
      }
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    return target;
  }
  // The entry of the list (all in [lo, hi], or 0: not taking part), from the
  // largest down, at which the running count or weight reaches `target` (at
  // least 1).  Histograms narrow the range until a warp can order what is left.
  __device__ u64 select(Mode mode, int n, u64 lo, u64 hi, u64 target) {
    for (;;) {
      const u64 span = hi - lo;
      const int s = span < kBins ? 0 : 64 - __clzll(span) - 10;
      clear(mode);
      for (int i = tid; i < n; i += TH) {
        const u64 c = sh.list[i];
        if (c < lo || c > hi || c == 0) continue;
        const int b = (int)((hi - c) >> s);
        atomicAdd(&sh.bins.count[b], 1u);
        if (mode == WEIGHT) sh.bins.add(b, sh.weight[i]);
      }
      __syncthreads();
      target = find([&](u64) { return target; },
                    [&](int b) { return mode == COUNT ? (u64)sh.bins.count[b] : sh.bins.weight(b); },
                    [&](int b) { return sh.bins.count[b]; });
      target -= sh.found_before;
      hi -= (u64)sh.found_bin << s;
      const u64 width = (1ull << s) - 1;
      if (hi - lo > width) lo = hi - width;
      if (sh.found_n > kFew) continue;
      for (int i = tid; i < n; i += TH) {
        const u64 c = sh.list[i];
        if (c >= lo && c <= hi && c) {
          const unsigned at = atomicAdd(&sh.n, 1u);
          sh.few[at] = c;
          sh.few_weight[at] = mode == COUNT ? 1 : sh.weight[i];
        }
      }
      __syncthreads();
      // every warp for itself: the weight at or above this lane's entry
      const bool have = lane < (int)sh.n;
      const u64 c = have ? sh.few[lane] : 0, w = have ? sh.few_weight[lane] : 0;
      u64 incl = 0;
      for (int i = 0; i < (int)sh.n; ++i) {
        const u64 ci = sh.few[i], wi = sh.few_weight[i];
        if (ci >= c) incl += wi;
      }
      const bool at = have && incl >= target && incl - w < target;
      return __shfl_sync(kFull, c, __ffs(__ballot_sync(kFull, at)) - 1);
    }
  }
};

// Weight at which top-p is reached, of `total`.
__device__ __forceinline__ u64 nucleus(float p, u64 total) {
  const double want = (double)p * (double)total;
  return want > 1.0 ? (u64)ceil(want) : 1;  // at least the first token
}
// Weight that the drawn token's running sum passes: the floor of u * total.
__device__ __forceinline__ u64 goal_of(float u, u64 total) {
  const u64 goal = u > 0.0f ? (u64)(fmin((double)u, 1.0) * (double)total) : 0;
  return goal >= total ? total - 1 : goal;
}

struct Filters {
  int k;  // 0: off
  float p;
  bool use_p;
  double zmin;
  float u;
};

__device__ __forceinline__ void answer(const SampleRowsDesc& d, int row, int token, int kept, double logw, u64 total) {
  d.token[row] = token;
  if (d.kept) d.kept[row] = kept;
  if (d.logprob) d.logprob[row] = token < 0 ? -INFINITY : (float)(logw - log((double)total * (1.0 / (1ull << kFix))));
}

// All filters and the draw on a list that holds every token they can keep, in
// the order of the indices; its places lie in [lo, hi], or are 0.
template <typename T, int TH>
__device__ void draw_from_list(Block<TH>& bk, const SampleRowsDesc& d, const Weigh& weigh, const Filters& f, int row,
                               int n, u64 lo, u64 hi) {
  constexpr int N = kList / TH;  // entries of a thread: they stay in registers, next to each other in the list
  Shared& sh = bk.sh;
  u64 last = 1;
  if (f.k > 0 && f.k < n) last = bk.select(COUNT, n, lo, hi, f.k);
  const int each = (n + TH - 1) / TH, i0 = min(n, (int)threadIdx.x * each), i1 = min(n, i0 + each);
  u64 c[N], w[N], total = 0;
  double z[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    c[j] = i0 + j < i1 ? sh.list[i0 + j] : 0;
    if (c[j] < last) c[j] = 0;
    z[j] = c[j] ? weigh.z(Key<T>::value(key_in(c[j]))) : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    w[j] = 0;
    if (j < each) w[j] = weigh.of_z(z[j]);
    total += w[j];
  }
  if (f.use_p) {
    total = bk.sum(total);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i0 + j < i1) {
        sh.list[i0 + j] = c[j];
        sh.weight[i0 + j] = w[j];
      }
    last = bk.select(WEIGHT, n, lo, hi, nucleus(f.p, total));
  }
  u64 own = 0;
  unsigned cnt = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const bool keep = c[j] >= last && c[j] && z[j] >= f.zmin;
    if (!keep) w[j] = 0;
    cnt += keep;
    own += w[j];
  }
  u64 sum;
  u64 run = bk.prefix(own, &sum);
  cnt = (unsigned)bk.sum(cnt);
  const u64 goal = goal_of(f.u, sum);
  if (run <= goal && goal < run + own) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (run <= goal && goal < run + w[j])
        answer(d, row, (int)~(uint32_t)c[j], (int)cnt, z[j], sum);
      run += w[j];
    }
  }
}

// Words that each CTA of a cluster tells the others: sums, and the sum of lower ranks.
__device__ __forceinline__ void cluster_sum(cg::cluster_group& cl, Shared& sh, u64 a, u64 b, u64* ta, u64* tb, u64* before_a) {
  if (threadIdx.x == 0) {
    sh.word[0] = a;
    sh.word[1] = b;
  }
  cl.sync();
  u64 sa = 0, sb = 0, before = 0;
  for (unsigned r = 0; r < cl.num_blocks(); ++r) {
    const u64* w = cl.map_shared_rank(sh.word, r);
    const u64 x = w[0];
    if (r < cl.block_rank()) before += x;
    sa += x;
    sb += w[1];
  }
  *ta = sa;
  *tb = sb;
  *before_a = before;
  cl.sync();
}

// One CTA's columns [0, n) of the row, the keys in shared memory.
template <typename T, int TH>
struct Slice {
  const typename Key<T>::Stored* keys;
  int n, base;  // base: the first one's index
  // f(i, key, place) of every column, kUnroll at a time
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += TH) {
      const uint32_t k = keys[i];
      f(i, k, place_of(k, base + i));
    }
  }
  // f(i, key, weight) of columns [first, last) step `step` whose place is at
  // least `floor`: four independent chains of f64 arithmetic
  template <typename F>
  __device__ __forceinline__ void weighed(int first, int last, int step, u64 floor, const Weigh& weigh, F f) const {
    for (int i0 = first; i0 < last; i0 += 4 * step) {
      uint32_t k[4];
      float l[4];
      bool on[4], any = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * step;
        k[j] = i < last ? keys[i] : 0u;
        on[j] = k[j] != 0 && place_of(k[j], base + i) >= floor;
        l[j] = Key<T>::value(on[j] ? k[j] : 1u);
        any |= on[j] && weigh.counts(l[j]);
      }
      if (any) {
        u64 w[4];
        double z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = weigh.z(l[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = weigh.of_z(z[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (on[j]) f(i0 + j * step, k[j], z[j], w[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (on[j]) f(i0 + j * step, k[j], weigh.z(l[j]), 0ull);
      }
    }
  }
};

// The whole cluster's search for the place at which the running count or weight
// of the tokens at or above `lo` reaches target(total).
template <typename T, int TH, typename Target>
__device__ u64 cluster_select(cg::cluster_group& cl, Block<TH>& bk, const Slice<T, TH>& sl, Mode mode, Target target_of,
                              u64 lo, u64 hi, const Weigh& weigh, float bins_per_unit) {
  Shared& sh = bk.sh;
  const int tid = threadIdx.x;
  const unsigned ranks = cl.num_blocks(), rank = cl.block_rank();
  // level 0: bins of (top - l) / T; then, where a bin holds more than a list,
  // bins of the places [lo, hi]
  auto first_bin = [&](uint32_t k) {
    const float l = Key<T>::value(k), x = (weigh.top - l) * bins_per_unit;
    return l == weigh.top ? 0 : x < (float)(kBins - 1) ? (int)x : kBins - 1;
  };
  int s = -1;
  u64 target = 0;
  for (;;) {
    bk.clear(mode);
    auto bin_of = [&](uint32_t k, u64 c) { return s < 0 ? first_bin(k) : (int)((hi - c) >> s); };
    if (mode == COUNT) {
      sl.each([&](int, uint32_t k, u64 c) {
        if (k != 0 && c >= lo && c <= hi) atomicAdd(&sh.bins.count[bin_of(k, c)], 1u);
      });
    } else {
      sl.weighed(tid, sl.n, TH, lo, weigh, [&](int i, uint32_t k, double, u64 w) {
        const u64 c = place_of(k, sl.base + i);
        if (c > hi) return;
        const int b = bin_of(k, c);
        atomicAdd(&sh.bins.count[b], 1u);
        sh.bins.add(b, w);
      });
    }
    cl.sync();
    const int share = kBins / ranks, b0 = rank * share;  // ranks: a power of two
    for (int b = b0 + tid; b < b0 + share; b += TH) {
      unsigned c = 0;
      u64 w = 0;
      for (unsigned r = 0; r < ranks; ++r) {
        const Bins* o = cl.map_shared_rank(&sh.bins, r);
        c += o->count[b];
        if (mode == WEIGHT) w += o->weight(b);
      }
      sh.merged.count[b] = c;
      sh.merged.weight[b] = mode == COUNT ? c : w;
    }
    cl.sync();
    target = bk.find([&](u64 total) { return s < 0 ? target_of(total) : target; },
                     [&](int b) { return cl.map_shared_rank(sh.merged.weight, b / share)[b]; },
                     [&](int b) { return cl.map_shared_rank(sh.merged.count, b / share)[b]; });
    const int bin0 = sh.found_bin;
    const unsigned count = sh.found_n;
    target -= sh.found_before;
    if (s >= 0) {
      hi -= (u64)bin0 << s;
      const u64 width = (1ull << s) - 1;
      if (hi - lo > width) lo = hi - width;
    }
    auto inside = [&](uint32_t k, u64 c) { return k != 0 && c >= lo && c <= hi && (s >= 0 || first_bin(k) == bin0); };
    if (count <= kList) {
      // every CTA gathers the bin's tokens from all, each from its own part
      u64 a = ~0ull, z = 0;
      sl.each([&](int, uint32_t k, u64 c) {
        if (inside(k, c)) sh.weight[atomicAdd(&sh.n, 1u)] = c;  // (the weights are filled in below)
      });
      cl.sync();
      unsigned at = 0;
      for (unsigned r = 0; r < ranks; ++r) {
        const unsigned m = *cl.map_shared_rank(&sh.n, r);
        const u64* from = cl.map_shared_rank(sh.weight, r);
        for (unsigned i = tid; i < m; i += TH) {
          const u64 c = from[i];
          sh.list[at + i] = c;
          a = c < a ? c : a;
          z = c > z ? c : z;
        }
        at += m;
      }
      a = bk.least(a);
      z = bk.most(z);
      cl.sync();
      if (mode == WEIGHT)
        for (unsigned i = tid; i < at; i += TH) sh.weight[i] = weigh(Key<T>::value(key_in(sh.list[i])));
      return bk.select(mode, (int)at, a, z, target);
    }
    // the range of the bin's places
    u64 a = ~0ull, z = 0;
    sl.each([&](int, uint32_t k, u64 c) {
      if (inside(k, c)) {
        a = c < a ? c : a;
        z = c > z ? c : z;
      }
    });
    a = bk.least(a);
    z = bk.most(z);
    if (tid == 0) {
      sh.word[0] = a;
      sh.word[1] = z;
    }
    cl.sync();
    for (unsigned r = 0; r < ranks; ++r) {
      const u64* w = cl.map_shared_rank(sh.word, r);
      a = w[0] < a ? w[0] : a;
      z = w[1] > z ? w[1] : z;
    }
    cl.sync();
    lo = a;
    hi = z;
    const u64 span = hi - lo;
    s = span < kBins ? 0 : 64 - __clzll(span) - 10;
  }
}

// Reads columns [0, n) at src; put(i, key) for each.  16 bytes a load where the
// row starts on that boundary.
template <typename T, int TH, typename Put>
__device__ __forceinline__ void read_columns(const T* src, int n, Put put) {
  constexpr int E = 16 / sizeof(T);
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const uint4* v = reinterpret_cast<const uint4*>(src);
    const int nv = n / E;
#pragma unroll 4
    for (int i = threadIdx.x; i < nv; i += TH) {
      const uint4 u = __ldcs(v + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (E == 4) {
          put(i * E + j, Key<T>::of(w[j]));
        } else {
          put(i * E + 2 * j, Key<T>::of(w[j] & 0xffffu));
          put(i * E + 2 * j + 1, Key<T>::of(w[j] >> 16));
        }
      }
    }
    done = nv * E;
  }
#pragma unroll 8
  for (int i = done + threadIdx.x; i < n; i += TH) {
    if constexpr (E == 4) put(i, Key<T>::of(reinterpret_cast<const uint32_t*>(src)[i]));
    else put(i, Key<T>::of(reinterpret_cast<const uint16_t*>(src)[i]));
  }
}

template <typename T, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) sample_rows_kernel(const __grid_constant__ SampleRowsDesc d) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  auto* keys = reinterpret_cast<typename Key<T>::Stored*>(smem + sizeof(Shared));
  if (threadIdx.x < 32) sh.exp2_32[threadIdx.x] = exp2(threadIdx.x * (1.0 / 32.0));
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group cl = cg::this_cluster();
  constexpr int kWarps = TH / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x;
  const unsigned rank = cl.block_rank(), ranks = cl.num_blocks();
  const int base = (int)rank * d.per, n = max(0, min(d.per, d.V - base));
  const T* src = static_cast<const T*>(d.logits) + (size_t)row * d.ld + base;
  const bool short_row = d.V <= kList;  // the row is the list
  Block<TH> bk(sh);
  Filters f;
  const float temp = d.temperature ? d.temperature[row] : 1.0f;
  f.k = d.top_k ? d.top_k[row] : 0;
  f.p = d.top_p ? d.top_p[row] : 1.0f;
  const float mp = d.min_p ? d.min_p[row] : 0.0f;
  f.u = d.u[row];
  f.use_p = f.p < 1.0f;
  if (f.k < 0 || f.k >= d.V) f.k = 0;

  // ---- the row, and the first token of the order ---------------------------------
  uint32_t my_key = 0;
  int my_at = 0;
  read_columns<T, TH>(src, n, [&](int i, uint32_t k) {
    if (short_row) sh.list[i] = k ? place_of(k, i) : 0ull;
    else keys[i] = (typename Key<T>::Stored)k;
    if (k > my_key || (k == my_key && i < my_at)) {
      my_key = k;
      my_at = i;
    }
  });
  u64 best = bk.most(my_key ? place_of(my_key, base + my_at) : 0ull);
  if (!short_row) {
    if (tid == 0) sh.word[2] = best;
    cl.sync();
    for (unsigned r = 0; r < ranks; ++r) {
      const u64 x = cl.map_shared_rank(sh.word, r)[2];
      best = best > x ? best : x;
    }
  }
  if (best == 0 || !(temp > 0.0f)) {
    if (rank == 0 && tid == 0) answer(d, row, best == 0 ? -1 : (int)~(uint32_t)best, best != 0, 0.0, 1ull << kFix);
    if (!short_row) cl.sync();  // no CTA leaves while its word is read
    return;
  }
  Weigh weigh;
  weigh.top = Key<T>::value(key_in(best));
  weigh.inv_tf = 1.0f / temp;
  weigh.inv_t = 1.0 / (double)temp;
  weigh.exp2_32 = sh.exp2_32;
  f.zmin = mp > 0.0f ? log((double)fminf(mp, 1.0f)) : -INFINITY;
  const u64 lowest = 1ull << 32;  // the least place that can be drawn
  if (short_row) {
    draw_from_list<T>(bk, d, weigh, f, row, n, lowest, best);
    return;
  }
  const Slice<T, TH> sl{keys, n, base};
  const int seg = (d.per + kWarps - 1) / kWarps, s0 = min(n, warp * seg), s1 = min(n, s0 + seg);  // a warp's columns

  // ---- small top-k: the list of what lies above a bound ---------------------------
  if (f.k > 0 && f.k <= kList / 2 && f.k * 4 <= (int)ranks * TH) {
    constexpr int kPart = kList / kWarps;  // tokens of a warp's part
    sh.list[tid] = my_key ? place_of(my_key, tid) : 0ull;
    __syncthreads();
    const int each = (f.k + ranks - 1) / ranks;
    uint32_t bound = 1;
    if (bk.sum(my_key != 0) >= (u64)each) bound = key_in(bk.select(COUNT, TH, lowest, ~0ull, each));
    if (tid == 0) sh.word[0] = bound;
    cl.sync();
    for (unsigned r = 0; r < ranks; ++r) bound = min(bound, (uint32_t)cl.map_shared_rank(sh.word, r)[0]);
    unsigned mine = 0;
    for (int i0 = s0; i0 < s1; i0 += 128) {  // in the order of the columns
      uint32_t k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * 32 + lane;
        k[j] = i < s1 ? keys[i] : 0u;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned hits = __ballot_sync(kFull, k[j] >= bound);
        const unsigned at = mine + __popc(hits & ((1u << lane) - 1));
        if (k[j] >= bound && at < kPart) sh.weight[warp * kPart + at] = place_of(k[j], base + i0 + j * 32 + lane);
        mine += __popc(hits);
      }
    }
    if (lane == 0) sh.part[warp] = mine;
    cl.sync();
    const int parts = (int)ranks * kWarps;  // at most 8 * 16
    const unsigned m = tid < parts ? cl.map_shared_rank(sh.part, tid / kWarps)[tid % kWarps] : 0u;
    u64 total;
    const u64 at = bk.prefix(m, &total);
    const bool fits = total <= kList && __syncthreads_and(m <= (unsigned)kPart);
    if (fits) {
      if (rank == 0) {
        if (tid < parts) sh.offset[tid] = ((unsigned)at << 12) | m;
        __syncthreads();
        for (int p = warp; p < parts; p += kWarps) {
          const unsigned o = sh.offset[p] >> 12, c = sh.offset[p] & 4095u;
          const u64* from = cl.map_shared_rank(sh.weight, p / kWarps) + (p % kWarps) * kPart;
          for (unsigned i = lane; i < c; i += 32) sh.list[o + i] = from[i];
        }
      }
      cl.sync();
      if (rank == 0) draw_from_list<T>(bk, d, weigh, f, row, (int)total, place_of(bound, 0x7fffffff), best);
      return;
    }
    cl.sync();
  }

  // ---- otherwise: the last kept place by histograms over the cluster ----------------
  const float bins_per_unit = 32.0f / temp;
  u64 last = lowest;
  if (f.k > 0)
    last = cluster_select(cl, bk, sl, COUNT, [&](u64) { return (u64)f.k; }, last, best, weigh, bins_per_unit);
  if (f.use_p)
    last = cluster_select(cl, bk, sl, WEIGHT, [&](u64 total) { return nucleus(f.p, total); }, last, best, weigh,
                          bins_per_unit);

  // ---- the draw: a warp's columns, then the threads of the CTA over that warp's ----
  u64 sum = 0, cnt = 0;
  sl.weighed(s0 + lane, s1, 32, last, weigh, [&](int, uint32_t, double z, u64 w) {
    const bool keep = z >= f.zmin;
    sum += keep ? w : 0;
    cnt += keep;
  });
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
  cnt = bk.sum(cnt);
  __syncthreads();
  if (lane == 0) sh.scan[warp] = sum;
  __syncthreads();
  u64 mine = 0;
  for (int w = 0; w < kWarps; ++w) mine += sh.scan[w];
  u64 total, count, run;
  cluster_sum(cl, sh, mine, cnt, &total, &count, &run);
  const u64 goal = goal_of(f.u, total);
  if (goal < run || goal >= run + mine) return;  // another CTA's
  int w = 0;
  while (goal >= run + sh.scan[w]) run += sh.scan[w++];
  const int t0 = min(n, w * seg), t1 = min(n, t0 + seg), each = (t1 - t0 + TH - 1) / TH;
  const int a0 = min(t1, t0 + tid * each), a1 = min(t1, a0 + each);
  u64 own = 0, all;
  sl.weighed(a0, a1, 1, last, weigh, [&](int, uint32_t, double z, u64 w) { own += z >= f.zmin ? w : 0; });
  u64 at = run + bk.prefix(own, &all);
  if (goal < at || goal >= at + own) return;
  sl.weighed(a0, a1, 1, last, weigh, [&](int i, uint32_t, double z, u64 w) {
    if (!(z >= f.zmin)) return;
    if (at <= goal && goal < at + w) answer(d, row, base + i, (int)count, z, total);
    at += w;
  });
}

template <typename T, int TH>
cudaError_t launch_t(const SampleRowsDesc& d, int n_rows, int ranks, cudaStream_t st) {
  constexpr size_t key = sizeof(typename Key<T>::Stored);
  const size_t smem = sizeof(Shared) + (d.V <= kList ? 0 : (size_t)d.per * key);
  static std::atomic<int> ready[kMaxDevices];
  const cudaError_t e = once_per_device(ready, [] {
    return cudaFuncSetAttribute(sample_rows_kernel<T, TH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)(sizeof(Shared) + QTTS_SAMPLE_ROWS_MAX_V / 8 * key));
  });
  if (e != cudaSuccess) return e;
  return launch_k(sample_rows_kernel<T, TH>, dim3(n_rows, ranks), dim3(TH), smem, st,
                  LaunchOpts{true, (unsigned)ranks}, d);
}
template <typename T>
cudaError_t launch(SampleRowsDesc d, int n_rows, int sms, cudaStream_t st) {
  // A cluster's CTAs hold at most 32768 logits each; rows that do not fill the
  // device are spread over more, down to 4096 logits a CTA.
  int ranks = 1;
  while (ranks < 8 && (d.V > ranks * 32768 || (d.V > ranks * 4096 && (long)n_rows * ranks < 2l * sms))) ranks *= 2;
  d.per = ((d.V + ranks - 1) / ranks + 31) / 32 * 32;
  return d.V <= kList ? launch_t<T, 256>(d, n_rows, 1, st) : launch_t<T, 512>(d, n_rows, ranks, st);
}

}  // namespace
}  // namespace qtts

using namespace qtts;

extern "C" int qtts_sample_rows_dev(const void* logits, int64_t ld, int dtype, int n_rows, int V,
                                    const float* temperature, const int32_t* top_k, const float* top_p,
                                    const float* min_p, const float* u, int32_t* token, int32_t* kept, float* logprob,
                                    void* stream) try {
  if (dtype != QTTS_F32 && dtype != QTTS_F16 && dtype != QTTS_BF16)
    return fail(QTTS_ERR_BADARG, "sample rows: unknown dtype");
  if (n_rows < 0 || V <= 0 || ld < V) return fail(QTTS_ERR_BADARG, "sample rows: bad sizes");
  if (V > QTTS_SAMPLE_ROWS_MAX_V) return fail(QTTS_ERR_RANGE, "sample rows: more than 262144 logits in a row");
  if (n_rows == 0) return QTTS_OK;
  if (!logits || !u || !token) return fail(QTTS_ERR_BADARG, "sample rows: a null pointer");
  if (reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dtype))
    return fail(QTTS_ERR_BADARG, "sample rows: misaligned logits");
  OnDeviceOf on(logits);
  if (on.err) return fail(on.code, std::string("sample rows, the logits: ") + on.err);
  SampleRowsDesc d;
  d.logits = logits;
  d.ld = ld;
  d.V = V;
  d.temperature = temperature;
  d.top_k = top_k;
  d.top_p = top_p;
  d.min_p = min_p;
  d.u = u;
  d.token = token;
  d.kept = kept;
  d.logprob = logprob;
  cudaError_t e;
  switch (dtype) {
    case QTTS_F16: e = launch<__half>(d, n_rows, on.sm_count, (cudaStream_t)stream); break;
    case QTTS_BF16: e = launch<__nv_bfloat16>(d, n_rows, on.sm_count, (cudaStream_t)stream); break;
    default: e = launch<float>(d, n_rows, on.sm_count, (cudaStream_t)stream);
  }
  if (e == cudaSuccess) return QTTS_OK;
  cudaGetLastError();
  return fail(QTTS_ERR_CUDA, cudaGetErrorString(e));
} catch (...) {
  return QTTS_ERR_OOM;
}
