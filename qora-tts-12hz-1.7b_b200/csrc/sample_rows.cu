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
// found by histograms over the range that still holds it.  The same search
// along the indices draws the token.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>

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

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// order key: larger for a larger logit; 0 for what is never drawn (NaN, -inf)
__device__ __forceinline__ uint32_t key_of(float l) { return l > -INFINITY ? f32_order_key(l) : 0u; }
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 place_of(uint32_t key, int index) { return ((u64)key << 32) | (uint32_t)~index; }

struct Weigh {
  float top;              // the largest logit
  double inv_t;
  const double* exp2_32;  // 2^(i / 32)
  __device__ __forceinline__ double z(float l) const {
    const double x = ((double)l - (double)top) * inv_t;
    return l == top ? 0.0 : x <= 0.0 ? x : -INFINITY;  // an infinite top over an infinite temperature is no number
  }
  // exp(z) 2^45 to the nearest integer: z = n ln2/32 + r, exp(r) by its series
  // to r^5 (|r| < 0.011: 2e-15), 2^(n/32) by table and exponent.  Below -33
  // (a weight of less than 1/8 of 2^-45) it is 0.
  __device__ __forceinline__ u64 operator()(float l) const {
    const double x = z(l);
    if (!(x > -33.0)) return 0;
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
    return (u64)(__double_as_longlong(w) - __double_as_longlong(0x1p52));
  }
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

struct Shared {
  Bins bins;
  u64 list[kList];
  u64 weight[kList];
  u64 merged[kBins];       // cluster: this CTA's share of the merged bins
  unsigned merged_n[kBins];
  double exp2_32[32];
  u64 scan[33];
  u64 word[4];             // what this CTA tells the cluster
  u64 found_at, found_before;
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
  // reaches `target` (clamped to the total): found_bin, found_n, found_before.
  template <typename Value, typename Count>
  __device__ __forceinline__ void find(u64 target, Value value, Count count) {
    constexpr int N = kBins / TH;
    u64 v[N], own = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[j] = value(tid * N + j);
      own += v[j];
    }
    u64 total;
    u64 run = prefix(own, &total);
    if (target > total) target = total;
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
    __syncthreads();
  }
  // The list's entry, from the largest down, at which the running count or
  // weight reaches `target` (at least 1); entries of 0 do not take part.
  __device__ u64 select(Mode mode, int n, u64 target) {
    u64 lo = ~0ull, hi = 0;
    for (int i = tid; i < n; i += TH) {
      const u64 c = sh.list[i];
      if (c) {
        lo = c < lo ? c : lo;
        hi = c > hi ? c : hi;
      }
    }
    lo = least(lo);
    hi = most(hi);
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
      find(target, [&](int b) { return mode == COUNT ? (u64)sh.bins.count[b] : sh.bins.weight(b); },
           [&](int b) { return sh.bins.count[b]; });
      const u64 b = sh.found_bin;
      target -= sh.found_before;
      hi -= b << s;
      const u64 width = (1ull << s) - 1;
      if (hi - lo > width) lo = hi - width;
      if (sh.found_n == 1 || lo == hi) {
        for (int i = tid; i < n; i += TH) {
          const u64 c = sh.list[i];
          if (c >= lo && c <= hi) sh.found_at = c;
        }
        __syncthreads();
        return sh.found_at;
      }
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

// All filters and the draw on a list that holds every token they can keep.
template <typename T, int TH>
__device__ void draw_from_list(Block<TH>& bk, const SampleRowsDesc& d, const Weigh& weigh, const Filters& f, int row, int n) {
  Shared& sh = bk.sh;
  const int tid = threadIdx.x;
  if (f.k > 0 && f.k < n) {
    const u64 last = bk.select(COUNT, n, f.k);
    for (int i = tid; i < n; i += TH)
      if (sh.list[i] < last) sh.list[i] = 0;
    __syncthreads();
  }
  u64 total = 0;
  for (int i = tid; i < n; i += TH) {
    const u64 c = sh.list[i], w = c ? weigh(value_of((uint32_t)(c >> 32))) : 0;
    sh.weight[i] = w;
    total += w;
  }
  u64 last = 1;
  if (f.use_p) {
    total = bk.sum(total);
    last = bk.select(WEIGHT, n, nucleus(f.p, total));
  }
  // what is kept, from here on in the order of the indices
  u64 sum = 0, cnt = 0;
  for (int i = tid; i < n; i += TH) {
    const u64 c = sh.list[i];
    const bool keep = c >= last && weigh.z(value_of((uint32_t)(c >> 32))) >= f.zmin;
    sh.list[i] = keep ? (u64)(uint32_t)c : 0;  // ~index, never 0
    if (keep) {
      sum += sh.weight[i];
      ++cnt;
    }
  }
  sum = bk.sum(sum);
  cnt = bk.sum(cnt);
  const u64 at = bk.select(WEIGHT, n, goal_of(f.u, sum) + 1);
  if (tid == 0) {
    const int token = (int)~(uint32_t)at;
    const float l = to_f32(static_cast<const T*>(d.logits)[(size_t)row * d.ld + token]);
    answer(d, row, token, (int)cnt, weigh.z(l), sum);
  }
}

// Words that each CTA of a cluster tells the others: sum and the sum of lower ranks.
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

// The whole cluster's search for the place at which the running count or weight
// of the tokens at or above `floor_place` reaches `target`.
template <int TH>
__device__ u64 cluster_select(cg::cluster_group& cl, Block<TH>& bk, const uint32_t* keys, int n, int base, Mode mode,
                              u64 target, u64 floor_place, const Weigh& weigh, float bins_per_unit) {
  Shared& sh = bk.sh;
  const int tid = threadIdx.x;
  const unsigned ranks = cl.num_blocks(), rank = cl.block_rank();
  // level 0: bins of (top - l) / T; then, where a bin holds more than a list,
  // bins of the places [lo, hi]
  auto first_bin = [&](uint32_t k) {
    const float l = value_of(k), x = (weigh.top - l) * bins_per_unit;
    return l == weigh.top ? 0 : x < (float)(kBins - 1) ? (int)x : kBins - 1;
  };
  u64 lo = floor_place, hi = ~0ull;
  int s = -1, bin0 = 0;
  for (;;) {
    bk.clear(mode);
    for (int i = tid; i < n; i += TH) {
      const uint32_t k = keys[i];
      const u64 c = place_of(k, base + i);
      if (k == 0 || c < lo || c > hi) continue;
      const int b = s < 0 ? first_bin(k) : (int)((hi - c) >> s);
      atomicAdd(&sh.bins.count[b], 1u);
      if (mode == WEIGHT) sh.bins.add(b, weigh(value_of(k)));
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
      sh.merged_n[b] = c;
      sh.merged[b] = mode == COUNT ? c : w;
    }
    cl.sync();
    bk.find(target, [&](int b) { return cl.map_shared_rank(sh.merged, b / share)[b]; },
            [&](int b) { return cl.map_shared_rank(sh.merged_n, b / share)[b]; });
    const int b = sh.found_bin;
    const unsigned count = sh.found_n;
    target -= sh.found_before;
    if (s >= 0) {
      hi -= (u64)b << s;
      const u64 width = (1ull << s) - 1;
      if (hi - lo > width) lo = hi - width;
    }
    bin0 = b;
    auto inside = [&](uint32_t k, u64 c) { return k != 0 && c >= lo && c <= hi && (s >= 0 || first_bin(k) == bin0); };
    if (count <= kList) {
      // every CTA gathers the bin's tokens from all, each from its own list
      if (tid == 0) sh.n = 0;
      __syncthreads();
      for (int i = tid; i < n; i += TH) {
        const uint32_t k = keys[i];
        const u64 c = place_of(k, base + i);
        if (inside(k, c)) sh.weight[atomicAdd(&sh.n, 1u)] = c;  // (the weights are filled in below)
      }
      cl.sync();
      unsigned at = 0;
      for (unsigned r = 0; r < ranks; ++r) {
        const unsigned m = *cl.map_shared_rank(&sh.n, r);
        const u64* from = cl.map_shared_rank(sh.weight, r);
        for (unsigned i = tid; i < m; i += TH) sh.list[at + i] = from[i];
        at += m;
      }
      cl.sync();
      if (mode == WEIGHT)
        for (unsigned i = tid; i < at; i += TH) sh.weight[i] = weigh(value_of((uint32_t)(sh.list[i] >> 32)));
      __syncthreads();
      return bk.select(mode, (int)at, target);
    }
    // the range of the bin's places
    u64 a = ~0ull, z = 0;
    for (int i = tid; i < n; i += TH) {
      const uint32_t k = keys[i];
      const u64 c = place_of(k, base + i);
      if (inside(k, c)) {
        a = c < a ? c : a;
        z = c > z ? c : z;
      }
    }
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

template <typename T, int TH>
__global__ void __launch_bounds__(TH) sample_rows_kernel(const __grid_constant__ SampleRowsDesc d) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem + sizeof(Shared));
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, row = blockIdx.x;
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
  if (tid < 32) sh.exp2_32[tid] = exp2(tid * (1.0 / 32.0));

  // ---- the row, and the first token of the order ---------------------------------
  u64 best = 0;
  uint32_t my_key = 0;
  if (short_row) {
    for (int i = tid; i < n; i += TH) {
      const uint32_t k = key_of(to_f32(src[i]));
      const u64 c = k ? place_of(k, i) : 0ull;
      sh.list[i] = c;
      best = best > c ? best : c;
    }
    best = bk.most(best);
  } else {
    for (int i = tid; i < n; i += TH) {
      const uint32_t k = key_of(to_f32(src[i]));
      keys[i] = k;
      const u64 c = k ? place_of(k, base + i) : 0ull;
      best = best > c ? best : c;
    }
    my_key = (uint32_t)(best >> 32);
    best = bk.most(best);
    if (tid == 0) sh.word[2] = best;
    cl.sync();
    for (unsigned r = 0; r < ranks; ++r) {
      const u64 x = cl.map_shared_rank(sh.word, r)[2];
      best = best > x ? best : x;
    }
    cl.sync();
  }
  if (best == 0 || !(temp > 0.0f)) {
    if (rank == 0 && tid == 0) answer(d, row, best == 0 ? -1 : (int)~(uint32_t)best, best != 0, 0.0, 1ull << kFix);
    return;
  }
  Weigh weigh;
  weigh.top = value_of((uint32_t)(best >> 32));
  weigh.inv_t = 1.0 / (double)temp;
  weigh.exp2_32 = sh.exp2_32;
  f.zmin = mp > 0.0f ? log((double)fminf(mp, 1.0f)) : -INFINITY;
  if (short_row) {
    draw_from_list<T>(bk, d, weigh, f, row, n);
    return;
  }

  // ---- small top-k: the list of what lies above a bound ---------------------------
  if (f.k > 0 && f.k <= kList / 2 && f.k * 4 <= (int)ranks * TH) {
    sh.list[tid] = my_key ? place_of(my_key, tid) : 0ull;
    __syncthreads();
    const int each = (f.k + ranks - 1) / ranks;
    const u64 some = bk.sum(my_key != 0);
    uint32_t bound = 1;
    if (some >= (u64)each) bound = (uint32_t)(bk.select(COUNT, TH, each) >> 32);
    if (tid == 0) {
      sh.word[0] = bound;
      sh.n = 0;
    }
    cl.sync();
    for (unsigned r = 0; r < ranks; ++r) bound = min(bound, (uint32_t)cl.map_shared_rank(sh.word, r)[0]);
    for (int i = tid; i < n; i += TH) {
      const uint32_t k = keys[i];
      if (k >= bound) {
        const unsigned at = atomicAdd(&sh.n, 1u);
        if (at < kList) sh.weight[at] = place_of(k, base + i);
      }
    }
    cl.sync();
    unsigned total = 0;
    for (unsigned r = 0; r < ranks; ++r) total += *cl.map_shared_rank(&sh.n, r);
    if (total <= kList) {
      if (rank == 0) {
        unsigned at = 0;
        for (unsigned r = 0; r < ranks; ++r) {
          const unsigned m = *cl.map_shared_rank(&sh.n, r);
          const u64* from = cl.map_shared_rank(sh.weight, r);
          for (unsigned i = tid; i < m; i += TH) sh.list[at + i] = from[i];
          at += m;
        }
      }
      cl.sync();
      if (rank == 0) draw_from_list<T>(bk, d, weigh, f, row, (int)total);
      return;
    }
    cl.sync();
  }

  // ---- otherwise: the last kept place by histograms over the cluster ----------------
  const float bins_per_unit = 32.0f / temp;
  u64 last = 1ull << 32;  // every token that can be drawn
  u64 unused;
  if (f.k > 0) last = cluster_select(cl, bk, keys, n, base, COUNT, (u64)f.k, last, weigh, bins_per_unit);
  if (f.use_p) {
    u64 total = 0, other;
    for (int i = tid; i < n; i += TH) {
      const uint32_t k = keys[i];
      if (k && place_of(k, base + i) >= last) total += weigh(value_of(k));
    }
    total = bk.sum(total);
    cluster_sum(cl, sh, total, 0, &total, &other, &unused);
    last = cluster_select(cl, bk, keys, n, base, WEIGHT, nucleus(f.p, total), last, weigh, bins_per_unit);
  }

  // ---- the draw: a warp's columns, then the threads of the CTA over that warp's ----
  constexpr int kWarps = TH / 32;
  const int warp = tid >> 5, lane = tid & 31;
  const int seg = (d.per + kWarps - 1) / kWarps, s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
  auto kept_weight = [&](int i, u64* count) -> u64 {
    const uint32_t k = keys[i];
    if (k == 0 || place_of(k, base + i) < last) return 0;
    const float l = value_of(k);
    if (!(weigh.z(l) >= f.zmin)) return 0;
    ++*count;
    return weigh(l);
  };
  u64 sum = 0, cnt = 0;
  for (int i = s0 + lane; i < s1; i += 32) sum += kept_weight(i, &cnt);
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
  u64 own = 0, dummy = 0, all;
  for (int i = a0; i < a1; ++i) own += kept_weight(i, &dummy);
  u64 at = run + bk.prefix(own, &all);
  if (goal < at || goal >= at + own) return;
  for (int i = a0; i < a1; ++i) {
    at += kept_weight(i, &dummy);
    if (at > goal) {
      answer(d, row, base + i, (int)count, weigh.z(value_of(keys[i])), total);
      break;
    }
  }
}

template <typename T, int TH>
cudaError_t launch_t(const SampleRowsDesc& d, int n_rows, int ranks, cudaStream_t st) {
  const size_t smem = sizeof(Shared) + (d.V <= kList ? 0 : (size_t)d.per * 4);
  static std::atomic<int> ready[kMaxDevices];
  const cudaError_t e = once_per_device(ready, [] {
    return cudaFuncSetAttribute(sample_rows_kernel<T, TH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)(sizeof(Shared) + QTTS_SAMPLE_ROWS_MAX_V / 8 * 4));
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
