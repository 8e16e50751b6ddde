// sample_rows.cu -- temperature / top-k / top-p / min-p sampling of rows of
// logits from given uniform numbers (sm_100a).
//
// A token's place in the order (logit descending, index ascending) is one
// 64-bit number, (order key of the logit) << 32 | ~index, so that ties need no
// care: every filter keeps the tokens at or above some number.  Weights
// w = exp((l - largest) / T) are integers of 2^-45 (f64 arithmetic), whose
// sums do not depend on their order.
//
// A row is cut down to a list of at most kList tokens in one CTA's shared memory:
//   a short row is one;
//   small top-k: a key that (k / CTAs) of each CTA's thread maxima reach has k
//     logits above it and few more; those are the list;
//   otherwise a histogram over (largest - l) / T of counts (top-k) or weights
//     (top-p) gives the bin in which the last kept token lies, and that bin's
//     tokens are the list.
// In a list the token at which the running count or weight reaches a target is
// found by histograms over the range that still holds it, until there is a
// thread for each token.  A long row is shared by a cluster of CTAs, which keep
// their columns in shared memory where they fit, and otherwise read them again
// from the L2 cache.
//
// A row's bytes would take HBM a fraction of this; what bounds it:
//   256 rows of 2048 f32 logits, top-k 50: 7.8 us (0.27 TB/s), a dozen block-wide
//     steps one after the other;
//   one row of 151936 f32, top-p: 29 us on 16 SMs, the same and the f64
//     exponentials (a quarter of it); 55 us between other kernels, which put its
//     code out of the instruction caches;
//   128 rows of 151936 bf16, top-k 1000, top-p, min-p: 40 us, 39 MB at 1.0 TB/s,
//     half of it the two passes over the row;
//   the same rows with top-p alone: 146 us, of which the weights' histogram takes
//     55 (about 90 issue slots a logit, the f64 series the most of it).
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
// Tokens of a list, and logits of a row that is one.  Rows past that go through
// the larger kernel (256 rows, f32, top-k 50: 2048 logits 8.0 us, 2049 9.6, 4096
// 9.8).
constexpr int kList = 2048;
constexpr int kBins = 1024;
constexpr int kShortThreads = 256;  // of a CTA that has a row of at most kList logits; 512 otherwise
typedef unsigned long long u64;

struct SampleRowsDesc {
  const void* logits = nullptr;
  long ld = 0;
  int V = 0, per = 0;  // columns, columns of a CTA
  bool keep = false;   // a CTA's columns stay in shared memory
  const float* temperature = nullptr;
  const int* top_k = nullptr;
  const float *top_p = nullptr, *min_p = nullptr, *u = nullptr;
  int *token = nullptr, *kept = nullptr;
  float* logprob = nullptr;
};

// Order keys: larger for a larger logit, equal for the two zeros.  Those of NaN
// lie above kInf or (sign bit set) below kNone, that of -inf is kNone: a row
// with a key above kInf is read again with such keys set to 0, and what is at
// most kNone is never drawn.  A 16-bit logit has a 16-bit key.
template <typename T>
struct Key {  // f16, bf16
  static constexpr uint32_t kInfBits = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  static constexpr uint32_t kInf = 0x8000u + kInfBits, kNone = 0x8000u - kInfBits;
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint32_t bits = k >= 0x8000u ? k - 0x8000u : 0x8000u | (0x8000u - k);
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((uint16_t)bits));
    else return __uint_as_float(bits << 16);
  }
  static __device__ __forceinline__ uint32_t near(float l) {  // the key of the nearest T
    uint32_t bits;
    if constexpr (std::is_same<T, __half>::value) bits = __half_as_ushort(__float2half_rn(l));
    else bits = __bfloat16_as_ushort(__float2bfloat16_rn(l));
    return of_word(bits) & 0xffffu;
  }
  // two logits' keys: 0x8000 + magnitude, or 0x8000 - magnitude
  static __device__ __forceinline__ uint32_t of_word(uint32_t w) {
    const uint32_t sign = (w >> 15) & 0x00010001u;
    return (w ^ (sign * 0x7fffu) ^ 0x80008000u) + sign;
  }
  static __device__ __forceinline__ uint32_t without_nan(uint32_t k) {
    if ((k & 0xffffu) > kInf) k &= 0xffff0000u;
    if ((k >> 16) > kInf) k &= 0xffffu;
    return k;
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ uint32_t largest(uint32_t w) { return max(w & 0xffffu, w >> 16); }
};
template <>
struct Key<float> {
  static constexpr uint32_t kInf = 0xff800000u, kNone = 0x00800000u;
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k >= 0x80000000u ? k - 0x80000000u : 0x80000000u | (0x80000000u - k));
  }
  static __device__ __forceinline__ uint32_t near(float l) { return of_word(__float_as_uint(l)); }
  static __device__ __forceinline__ uint32_t of_word(uint32_t w) {  // 2^31 + magnitude, or 2^31 - magnitude
    const int sign = (int)w >> 31;
    return (uint32_t)(((int)(w & 0x7fffffffu) ^ sign) - sign) + 0x80000000u;
  }
  static __device__ __forceinline__ uint32_t without_nan(uint32_t k) { return k > kInf ? 0u : k; }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ uint32_t largest(uint32_t w) { return w; }
};
__device__ __forceinline__ u64 place_of(uint32_t key, int index) { return ((u64)key << 32) | (uint32_t)~index; }
__device__ __forceinline__ uint32_t key_in(u64 place) { return (uint32_t)(place >> 32); }

struct Weigh {
  static constexpr double kStepsPerUnit = 46.166241308446828;  // 32 / ln 2
  float top;              // the largest logit
  float light;            // about top - 36 T: what lies below weighs nothing
  double top_d, inv_t;
  bool infinite;          // top is: the infinite logits share, whatever the temperature
  const uint32_t* exp2_32;  // the low words of 2^(i / 32), then the high ones: no two of them share a bank
  __device__ __forceinline__ Weigh(float t, float temp, const uint32_t* table) : top(t), exp2_32(table) {
    light = top - 36.0f * temp;
    top_d = top;
    inv_t = 1.0 / (double)temp;
    infinite = isinf(top);
  }
  __device__ __forceinline__ double z(float l) const {
    if (infinite) return l == top ? 0.0 : -INFINITY;
    return ((double)l - top_d) * inv_t;
  }
  // exp(z) 2^45 to the nearest integer, for a finite top and z of -500 to 0:
  // z = n ln2/32 + r, exp(r) by its series to r^5 (|r| < 0.011: 2e-15),
  // 2^(n/32) by table and exponent
  __device__ __forceinline__ u64 finite(float l) const {
    int n;
    return finite(l, n);
  }
  // n of such a z: it never falls as l grows
  __device__ __forceinline__ int steps(float l) const {
    return __double2loint(__fma_rn(((double)l - top_d) * inv_t, kStepsPerUnit, 0x1.8p52));
  }
  __device__ __forceinline__ u64 finite(float l, int& n) const {
    const double x = ((double)l - top_d) * inv_t;
    const double shift = 0x1.8p52;
    const double nd = __fma_rn(x, kStepsPerUnit, shift);
    n = __double2loint(nd);
    const double r = __fma_rn(nd - shift, -0.021660849392498290, x);  // ln 2 / 32
    double p = __fma_rn(r, 1.0 / 120.0, 1.0 / 24.0);
    p = __fma_rn(p, r, 1.0 / 6.0);
    p = __fma_rn(p, r, 0.5);
    p = __fma_rn(p, r, 1.0);
    p = __fma_rn(p, r, 1.0);
    const uint32_t* t = exp2_32 + (n & 31);
    const double s = __hiloint2double((int)t[32] + (((n >> 5) + kFix) << 20), (int)t[0]);
    const double w = __fma_rn(s, p, 0x1p52);  // the sum's mantissa is the integer
    return (u64)(__double_as_longlong(w) - __double_as_longlong(0x1p52));
  }
  __device__ __forceinline__ u64 operator()(float l) const {
    if (infinite) return l == top ? 1ull << kFix : 0;
    return z(l) > -36.0 ? finite(l) : 0;
  }
};

// Histogram bins: counts, and weights as three words of 15 bits (64-bit shared
// atomics are retry loops).  The high word of a weight of 1 is 2^15, so a sum of
// fewer than 2^17 tokens stays in 32 bits; kMaxSlice sees to it.
constexpr int kMaxSlice = 98304;  // columns of a CTA
static_assert(((u64)kMaxSlice << (kFix - 30)) <= 0xffffffffull && kFix <= 45, "a bin's words hold a slice's weights");
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

constexpr int kFew = 128;     // tokens that a search leaves to a thread each
constexpr int kSmall = 64;    // tokens whose filters and draw one warp does alone
struct alignas(16) Shared {
  Bins bins;
  union {
    u64 list[kList];
    u64 merged[kBins];  // cluster: this CTA's share of the bins, read before any list is made
  };
  u64 weight[kList];  // of the list; before it is made, this CTA's part of the list
  u64 few[kFew], few_weight[kFew];
  uint32_t exp2_32[64];
  u64 scan[32];
  unsigned scan32[32];
  u64 word[2];            // what this CTA tells the cluster
  unsigned key_word[2];
  unsigned part[32];      // tokens in this CTA's part of the list, by warp
  unsigned offset[16 * 16];
  u64 found_before, found_at;
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
    v = sh.scan[lane & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) v = op(v, __shfl_xor_sync(kFull, v, o));
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
  __device__ __forceinline__ unsigned sum32(unsigned v) {
    v = __reduce_add_sync(kFull, v);
    __syncthreads();
    if (lane == 0) sh.scan32[warp] = v;
    __syncthreads();
    return __reduce_add_sync(kFull, lane < kWarps ? sh.scan32[lane] : 0u);
  }
  __device__ __forceinline__ unsigned most32(unsigned v) {
    v = __reduce_max_sync(kFull, v);
    __syncthreads();
    if (lane == 0) sh.scan32[warp] = v;
    __syncthreads();
    return __reduce_max_sync(kFull, lane < kWarps ? sh.scan32[lane] : 0u);
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
    u64 s = lane < kWarps ? sh.scan[lane] : 0;
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const u64 y = __shfl_up_sync(kFull, s, o);
      if (lane >= o) s += y;
    }
    *total = __shfl_sync(kFull, s, kWarps - 1);
    const u64 before = __shfl_sync(kFull, s, max(0, warp - 1));
    return (warp ? before : 0) + x - v;
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
  // The entry of the list (0: not taking part), from the largest down, at which
  // the running count or weight reaches `target` (at least 1).  The first
  // histogram goes by first_bin(place), the next ones by the places of the bin
  // that holds the target, until one warp can order what is left.
  template <typename FirstBin>
  __device__ u64 select(Mode mode, int n, u64 target, FirstBin first_bin) {
    u64 lo = 1, hi = ~0ull;
    int s = -1, bin = 0;
    for (;;) {
      clear(mode);
      for (int i = tid; i < n; i += TH) {
        const u64 c = sh.list[i];
        if (c < lo || c > hi) continue;
        const int b = s < 0 ? first_bin(c) : (int)((hi - c) >> s);
        atomicAdd(&sh.bins.count[b], 1u);
        if (mode == WEIGHT) sh.bins.add(b, sh.weight[i]);
      }
      __syncthreads();
      target = find([&](u64) { return target; },
                    [&](int b) { return mode == COUNT ? (u64)sh.bins.count[b] : sh.bins.weight(b); },
                    [&](int b) { return sh.bins.count[b]; });
      target -= sh.found_before;
      bin = sh.found_bin;
      if (s >= 0) {
        hi -= (u64)bin << s;
        const u64 width = (1ull << s) - 1;
        if (hi - lo > width) lo = hi - width;
      }
      auto inside = [&](u64 c) { return c >= lo && c <= hi && (s >= 0 || first_bin(c) == bin); };
      if (sh.found_n <= kFew) {
        for (int i = tid; i < n; i += TH) {
          const u64 c = sh.list[i];
          if (inside(c)) {
            const unsigned at = atomicAdd(&sh.n, 1u);
            sh.few[at] = c;
            sh.few_weight[at] = mode == COUNT ? 1 : sh.weight[i];
          }
        }
        __syncthreads();
        if (const int m = sh.n; tid < m) {  // the weight at or above each thread's entry
          const u64 c = sh.few[tid], w = sh.few_weight[tid];
          u64 incl = 0;
#pragma unroll 4
          for (int i = 0; i < m; ++i) incl += sh.few[i] >= c ? sh.few_weight[i] : 0;
          if (incl >= target && incl - w < target) sh.found_at = c;
        }
        __syncthreads();
        return sh.found_at;
      }
      u64 a = ~0ull, z = 0;
      for (int i = tid; i < n; i += TH) {
        const u64 c = sh.list[i];
        if (inside(c)) {
          a = c < a ? c : a;
          z = c > z ? c : z;
        }
      }
      lo = least(a);
      hi = most(z);
      const u64 span = hi - lo;
      s = span < kBins ? 0 : 64 - __clzll(span) - 10;
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
  u64 min_place;  // min-p: the least place that it keeps
  float u;
  float bins_per_unit;
};

__device__ __forceinline__ void answer(const SampleRowsDesc& d, int row, int token, int kept, double logw, u64 total) {
  d.token[row] = token;
  if (d.kept) d.kept[row] = kept;
  if (d.logprob) d.logprob[row] = token < 0 ? -INFINITY : (float)(logw - log((double)total * (1.0 / (1ull << kFix))));
}

// The bin of a logit in the histogram over (top - l) / T, 32 bins a unit.
template <typename T>
struct FirstBin {
  float top, per_unit;
  __device__ __forceinline__ int logit(float l) const {
    const float x = (top - l) * per_unit;
    return l == top ? 0 : x < (float)(kBins - 1) ? (int)x : kBins - 1;
  }
  __device__ __forceinline__ int operator()(u64 place) const { return logit(Key<T>::value(key_in(place))); }
};

// All filters and the draw on a list of at most kSmall tokens that holds every
// one they can keep, in the order of the indices: one warp, each lane's two
// tokens against all of them.
template <typename T>
__device__ void draw_small(Shared& sh, const SampleRowsDesc& d, const Weigh& weigh, const Filters& f, int row, int n) {
  const int lane = threadIdx.x & 31;
  u64 c[2], w[2], sum = 0;
  double z[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane * 2 + j;
    c[j] = i < n ? sh.list[i] : 0;
    const float l = Key<T>::value(key_in(c[j]));
    z[j] = weigh.z(l);
    w[j] = c[j] ? weigh(l) : 0;
    if (i < kSmall) sh.weight[i] = w[j];
  }
  __syncwarp();
  u64 above[2] = {0, 0};
  int rank[2] = {0, 0};
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const u64 ci = sh.list[i], wi = sh.weight[i];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool before = ci > c[j];
      rank[j] += before && ci;
      above[j] += before ? wi : 0;
    }
  }
  bool keep[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    keep[j] = c[j] != 0 && (f.k == 0 || rank[j] < f.k);
    sum += keep[j] ? w[j] : 0;
  }
  if (f.use_p) {  // a token whose weight before it reaches the target is not kept
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    const u64 target = nucleus(f.p, sum);
#pragma unroll
    for (int j = 0; j < 2; ++j) keep[j] = keep[j] && above[j] < target;
  }
  u64 own = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    keep[j] = keep[j] && c[j] >= f.min_place;
    if (!keep[j]) w[j] = 0;
    own += w[j];
  }
  const unsigned cnt = __reduce_add_sync(kFull, (unsigned)keep[0] + (unsigned)keep[1]);
  u64 incl = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(kFull, incl, o);
    if (lane >= o) incl += y;
  }
  const u64 total = __shfl_sync(kFull, incl, 31), goal = goal_of(f.u, total);
  u64 run = incl - own;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (run <= goal && goal < run + w[j]) answer(d, row, (int)~(uint32_t)c[j], (int)cnt, z[j], total);
    run += w[j];
  }
}

// The same on a longer list.
template <typename T, int TH>
__device__ void draw_from_list(Block<TH>& bk, const SampleRowsDesc& d, const Weigh& weigh, const Filters& f, int row, int n) {
  constexpr int N = kList / TH;  // entries of a thread: they stay in registers, next to each other in the list
  Shared& sh = bk.sh;
  const FirstBin<T> first_bin{weigh.top, f.bins_per_unit};
  u64 last = 1;
  if (f.k > 0 && f.k < n) last = bk.select(COUNT, n, f.k, first_bin);
  const int each = (n + TH - 1) / TH, i0 = min(n, (int)threadIdx.x * each), i1 = min(n, i0 + each);
  u64 c[N], w[N], total = 0;
  double z[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    c[j] = i0 + j < i1 ? sh.list[i0 + j] : 0;
    if (c[j] < last) c[j] = 0;
    const float l = Key<T>::value(key_in(c[j]));
    z[j] = weigh.z(l);
    w[j] = 0;
    if (c[j]) w[j] = weigh(l);
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
    last = bk.select(WEIGHT, n, nucleus(f.p, total), first_bin);
  }
  last = last > f.min_place ? last : f.min_place;
  u64 own = 0;
  unsigned cnt = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const bool keep = c[j] >= last;
    if (!keep) w[j] = 0;
    cnt += keep;
    own += w[j];
  }
  u64 sum;
  u64 run = bk.prefix(own, &sum);
  cnt = bk.sum32(cnt);
  const u64 goal = goal_of(f.u, sum);
  if (run <= goal && goal < run + own) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (run <= goal && goal < run + w[j]) answer(d, row, (int)~(uint32_t)c[j], (int)cnt, z[j], sum);
      run += w[j];
    }
  }
}

// Over the lanes of a warp; every lane gets the result.
template <typename Op>
__device__ __forceinline__ u64 over_lanes(u64 v, Op op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
__device__ __forceinline__ u64 lanes_sum(u64 v) {
  return over_lanes(v, [](u64 a, u64 b) { return a + b; });
}
// What the CTAs of a cluster (at most 16) tell each other is read by a lane a
// CTA, as one read of another SM's shared memory takes hundreds of cycles.
template <typename V>
__device__ __forceinline__ V of_lane_rank(cg::cluster_group& cl, V* word, V none) {
  const unsigned r = threadIdx.x & 31;
  return r < cl.num_blocks() ? *cl.map_shared_rank(word, r) : none;
}
// Sums of all CTAs, and of the CTAs of lower ranks.
__device__ __forceinline__ void cluster_sum(cg::cluster_group& cl, Shared& sh, u64 a, u64 b, u64* ta, u64* tb, u64* before_a) {
  if (threadIdx.x == 0) {
    sh.word[0] = a;
    sh.word[1] = b;
  }
  cl.sync();
  const u64 x = of_lane_rank<u64>(cl, &sh.word[0], 0), y = of_lane_rank<u64>(cl, &sh.word[1], 0);
  *ta = lanes_sum(x);
  *tb = lanes_sum(y);
  *before_a = lanes_sum((threadIdx.x & 31) < cl.block_rank() ? x : 0);
  cl.sync();
}

// One CTA's columns [0, n) of the row, as vectors of E columns: 16 bytes a load
// where the row starts on that boundary.  Those of a short slice are kept.
template <typename T, int TH>
struct Slice {
  using K = Key<T>;
  static constexpr int E = 16 / sizeof(T);
  const T* src;
  int n, nv, base;  // columns, vectors, the first column's index
  bool aligned, nan;
  uint4* kept;      // the vectors in shared memory, or null

  __device__ __forceinline__ uint4 raw(int v) const {
    if (aligned && (v + 1) * E <= n) return reinterpret_cast<const uint4*>(src)[v];
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (E == 4) {
        w[j] = v * E + j < n ? reinterpret_cast<const uint32_t*>(src)[v * E + j] : 0xff800000u;
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
        const uint32_t none = 0x8000u | K::kInfBits;  // -inf behind the last column
        const int i = v * E + 2 * j;
        w[j] = (i < n ? h[i] : none) | ((i + 1 < n ? h[i + 1] : none) << 16);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ uint4 to_keys(uint4 u) const {
    u = make_uint4(K::of_word(u.x), K::of_word(u.y), K::of_word(u.z), K::of_word(u.w));
    if (nan) u = make_uint4(K::without_nan(u.x), K::without_nan(u.y), K::without_nan(u.z), K::without_nan(u.w));
    return u;
  }
  // the first pass: the thread's largest key in each place of a vector (E == 8:
  // two in a word)
  __device__ __forceinline__ void largest(uint32_t (&most)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) most[j] = 0;
    for (int v0 = threadIdx.x; v0 < nv; v0 += 4 * TH) {
      uint4 u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + j * TH < nv) u[j] = raw(v0 + j * TH);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + j * TH < nv) {
          if (kept) kept[v0 + j * TH] = u[j];
          u[j] = to_keys(u[j]);
          most[0] = K::larger(most[0], u[j].x);
          most[1] = K::larger(most[1], u[j].y);
          most[2] = K::larger(most[2], u[j].z);
          most[3] = K::larger(most[3], u[j].w);
        }
    }
  }
  // later passes: a vector, and its keys in words
  __device__ __forceinline__ uint4 again(int v) const { return kept ? kept[v] : raw(v); }
  __device__ __forceinline__ uint4 words(int v) const { return to_keys(again(v)); }
  static __device__ __forceinline__ uint32_t largest_of(uint4 u) {
    return K::largest(K::larger(K::larger(u.x, u.y), K::larger(u.z, u.w)));
  }
  static __device__ __forceinline__ uint32_t pick(uint4 u, int j) {  // the j-th key
    const int i = j * 4 / E;
    const uint32_t w = i & 2 ? (i & 1 ? u.w : u.z) : (i & 1 ? u.y : u.x);
    return E == 4 ? w : (w >> (16 * (j & 1))) & 0xffffu;
  }
  static __device__ __forceinline__ void apart(uint4 u, uint32_t (&k)[E]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (E == 4) {
        k[j] = w[j];
      } else {
        k[2 * j] = w[j] & 0xffffu;
        k[2 * j + 1] = w[j] >> 16;
      }
    }
  }
  // The logits of a vector as they are: NaN compares like what is never drawn.
  static __device__ __forceinline__ void logits(uint4 u, float (&l)[E]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (E == 4) {
        l[j] = __uint_as_float(w[j]);
      } else if constexpr (std::is_same<T, __half>::value) {
        l[2 * j] = __half2float(__ushort_as_half((uint16_t)(w[j] & 0xffffu)));
        l[2 * j + 1] = __half2float(__ushort_as_half((uint16_t)(w[j] >> 16)));
      } else {
        l[2 * j] = __uint_as_float(w[j] << 16);
        l[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  }
  // f(logit, place) of the columns whose places lie in [lo, hi] (lo above
  // kNone), as long as go(); the loads of four vectors are on their way at once
  template <typename F, typename Go>
  __device__ __forceinline__ void between(u64 lo, u64 hi, F f, Go go) const {
    const float from = K::value(key_in(lo)), to = K::value(key_in(hi));
#pragma unroll 1
    for (int v0 = threadIdx.x; v0 < nv && go(); v0 += 4 * TH) {
      uint4 u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + j * TH < nv) u[j] = again(v0 + j * TH);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (v0 + j * TH >= nv) break;
        float l[E];
        logits(u[j], l);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (l[e] >= from && l[e] <= to) {
            const u64 c = place_of(K::near(l[e]), base + (v0 + j * TH) * E + e);
            if (c >= lo && c <= hi) f(l[e], c);
          }
      }
    }
  }
  template <typename F>
  __device__ __forceinline__ void between(u64 lo, u64 hi, F f) const {
    between(lo, hi, f, [] { return true; });
  }
  // A floor (a place) in terms of logits and columns of this slice
  struct Floor {
    float l, heavy;  // what lies below heavy weighs nothing
    int last;        // the last column that reaches the floor with a logit of l
    __device__ __forceinline__ bool operator()(float x, int i) const { return x > l || (x == l && i <= last); }
  };
  __device__ __forceinline__ Floor floor_of(u64 floor, const Weigh& weigh) const {
    const long last = (long)(uint32_t)~(uint32_t)floor - base;
    // Keys below that of `light` have z < -35; keys from it on z > -73, as a T
    // so near to the largest that 36 T is less than half a step gives its key.
    return Floor{K::value(key_in(floor)), K::value(max(K::near(weigh.light), K::kNone + 1)),
                 (int)max(-1l, min(last, (long)n))};
  }
  // f(i, logit, weight, steps) of the columns of vectors [first, last) step
  // `step` that reach the floor: four independent chains of f64 arithmetic
  template <typename F>
  __device__ __forceinline__ void weighed(int first, int last, int step, const Floor& floor, const Weigh& weigh, F f) const {
#pragma unroll 1
    for (int v = first; v < last; v += step) {
      float l[E];
      logits(again(v), l);
#pragma unroll
      for (int h = 0; h < E; h += 4) {
        const float* x = l + h;
        u64 w[4] = {0, 0, 0, 0};
        int steps[4] = {0, 0, 0, 0};
        if (weigh.infinite) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = x[j] == weigh.top ? 1ull << kFix : 0;
        } else if (fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= floor.heavy) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool on = x[j] >= floor.heavy;  // (not NaN, not far below the range of `finite`)
            const u64 y = weigh.finite(on ? x[j] : weigh.top, steps[j]);
            w[j] = on ? y : 0;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = v * E + h + j;
          if (floor(x[j], i)) f(i, x[j], w[j], steps[j]);
        }
      }
    }
  }
  // Weight and number of the columns of a warp's vectors [first, last) that
  // reach a floor that few do: each lane puts theirs in a column of shared
  // memory (TH x 16 floats), and the weights are worked out a row at a time.
  __device__ __forceinline__ void gathered(int first, int last, const Floor& floor, const Weigh& weigh, float* column,
                                           u64& sum, unsigned& count) const {
    constexpr int kDeep = 16;
    const int lane = threadIdx.x & 31;
    float* own = column + threadIdx.x;
    int have = 0;
    auto work_out = [&] {
      const int rows = __reduce_max_sync(kFull, have);
#pragma unroll 1
      for (int r = 0; r < rows; r += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float l = r + j < have ? own[(r + j) * TH] : weigh.top;
          const bool on = r + j < have && (weigh.infinite ? l == weigh.top : l >= floor.heavy);
          const u64 y = weigh.infinite ? 1ull << kFix : weigh.finite(on ? l : weigh.top);
          sum += on ? y : 0;
        }
      }
      have = 0;
    };
#pragma unroll 2
    for (int v0 = first; v0 < last; v0 += 32) {
      if (__any_sync(kFull, have > kDeep - E)) work_out();
      const int v = v0 + lane;
      if (v < last) {
        float l[E];
        logits(again(v), l);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (floor(l[j], v * E + j)) {
            own[have * TH] = l[j];
            ++have;
            ++count;
          }
      }
    }
    work_out();
  }
};

// The lowest of the keys (kNone, top] for which keeps() holds, which it does for
// `top` and for every key above one; mostly within two keys of `guess`.
template <typename T, typename Keeps>
__device__ __forceinline__ uint32_t lowest_key(uint32_t top, float guess, Keeps keeps) {
  uint32_t lo = Key<T>::kNone, hi = top;
  const uint32_t k = min(max(Key<T>::near(guess), lo), hi);
  if (k > lo + 2 && !keeps(k - 2)) lo = k - 2;
  if (k + 2 < hi && keeps(k + 2)) hi = k + 2;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (keeps(mid)) hi = mid;
    else lo = mid;
  }
  return hi;
}

// The whole cluster's search for the place at which the running count or weight
// of the tokens at or above `lo` reaches target(total).
template <typename T, int TH, typename Target>
__device__ u64 cluster_select(cg::cluster_group& cl, Block<TH>& bk, const Slice<T, TH>& sl, Mode mode, Target target_of,
                              u64 lo, uint32_t top, const Weigh& weigh, float bins_per_unit) {
  using K = Key<T>;
  Shared& sh = bk.sh;
  const int tid = threadIdx.x;
  const unsigned ranks = cl.num_blocks(), rank = cl.block_rank();
  const FirstBin<T> first_bin{weigh.top, bins_per_unit};
  const auto floor = sl.floor_of(lo, weigh);
  // the first histogram's bin of a key: over (top - l) / T for counts; for
  // weights the steps of ln2 / 32 that their arithmetic has at hand
  auto bin_of_steps = [&](int steps) { return min(-steps, kBins - 1); };
  auto bin_of_key = [&](uint32_t k) {
    const float l = K::value(k);
    if (mode == COUNT) return first_bin.logit(l);
    if (weigh.infinite) return l == weigh.top ? 0 : kBins - 1;
    return l >= floor.heavy ? bin_of_steps(weigh.steps(l)) : kBins - 1;
  };
  u64 hi = ((u64)top << 32) | 0xffffffffu;
  int s = -1;
  u64 target = 0;
  for (;;) {
    bk.clear(mode);
    if (mode == COUNT) {
      sl.between(lo, hi, [&](float l, u64 c) { atomicAdd(&sh.bins.count[s < 0 ? first_bin.logit(l) : (int)((hi - c) >> s)], 1u); });
    } else {
      sl.weighed(tid, sl.nv, TH, floor, weigh, [&](int i, float l, u64 w, int steps) {
        int b = bin_of_steps(steps);
        if (s >= 0) {
          const u64 c = place_of(K::near(l), sl.base + i);
          if (c < lo || c > hi) return;
          b = (int)((hi - c) >> s);
        }
        sh.bins.add(b, w);
      });
    }
    cl.sync();
    // each CTA adds up its share of the bins, a thread a CTA's bin
    const int share = kBins / ranks, b0 = rank * share;  // ranks: a power of two
#pragma unroll
    for (int j = 0; j < kBins / TH; ++j) {
      const int i = tid + j * TH, b = b0 + i % share;
      const Bins* o = cl.map_shared_rank(&sh.bins, i / share);
      sh.weight[i] = mode == COUNT ? o->count[b] : o->weight(b);
    }
    __syncthreads();
    for (int i = tid; i < share; i += TH) {
      u64 w = 0;
#pragma unroll 4
      for (unsigned r = 0; r < ranks; ++r) w += sh.weight[r * share + i];
      sh.merged[b0 + i] = w;
    }
    cl.sync();
    target = bk.find([&](u64 total) { return s < 0 ? target_of(total) : target; },
                     [&](int b) { return cl.map_shared_rank(sh.merged, b / share)[b]; }, [](int) { return 0u; });
    const int bin = sh.found_bin;
    target -= sh.found_before;
    if (s >= 0) {
      hi -= (u64)bin << s;
      const u64 width = (1ull << s) - 1;
      if (hi - lo > width) lo = hi - width;
    } else {
      // the bin's keys: two warps look for its ends
      if (tid < 64) {
        const int most = tid < 32 ? bin : bin - 1;
        const float unit = mode == COUNT ? (bin + (tid < 32)) / bins_per_unit
                                         : (float)((bin + (tid < 32 ? 0.5 : -0.5)) / (Weigh::kStepsPerUnit * weigh.inv_t));
        const uint32_t k = most < 0 ? top + 1 : lowest_key<T>(top, weigh.top - unit, [&](uint32_t x) { return bin_of_key(x) <= most; });
        if ((tid & 31) == 0) sh.key_word[tid >> 5] = k;
      }
      __syncthreads();
      const u64 k0 = (u64)sh.key_word[0] << 32, k1 = ((u64)sh.key_word[1] << 32) - 1;
      lo = k0 > lo ? k0 : lo;
      hi = k1 < hi ? k1 : hi;
    }
    // every CTA gathers the bin's tokens from all, each from its own part
    volatile unsigned* count = &sh.n;
    sl.between(lo, hi, [&](float, u64 c) {
      const unsigned at = atomicAdd(&sh.n, 1u);
      if (at < kList) sh.weight[at] = c;  // (the weights are filled in below)
    }, [&] { return *count <= kList; });
    cl.sync();
    const unsigned m = of_lane_rank<unsigned>(cl, &sh.n, 0u), all = __reduce_add_sync(kFull, m);
    if (all <= kList) {
      // warp w takes part w / ranks of the tokens of CTA w % ranks
      const unsigned r = bk.warp % ranks, mine = __shfl_sync(kFull, m, r);
      const unsigned before = __reduce_add_sync(kFull, bk.lane < (int)r ? m : 0u);
      const u64* from = cl.map_shared_rank(sh.weight, r);
      u64 a = ~0ull, z = 0;
#pragma unroll 4
      for (unsigned i = bk.warp / ranks * 32 + bk.lane; i < mine; i += TH / ranks) {
        const u64 c = from[i];
        sh.list[before + i] = c;
        a = c < a ? c : a;
        z = c > z ? c : z;
      }
      a = bk.least(a);
      z = bk.most(z);
      cl.sync();
      if (mode == WEIGHT)
        for (unsigned i = tid; i < all; i += TH) sh.weight[i] = weigh(K::value(key_in(sh.list[i])));
      // the bin's places spread evenly over the first histogram
      const u64 span = z - a;
      const int shift = span < kBins ? 0 : 64 - __clzll(span) - 10;
      return bk.select(mode, (int)all, target, [&](u64 c) { return (int)((z - c) >> shift); });
    }
    // the range of the bin's places
    u64 a = ~0ull, z = 0;
    sl.between(lo, hi, [&](float, u64 c) {
      a = c < a ? c : a;
      z = c > z ? c : z;
    });
    a = bk.least(a);
    z = bk.most(z);
    if (tid == 0) {
      sh.word[0] = a;
      sh.word[1] = z;
    }
    cl.sync();
    a = over_lanes(of_lane_rank<u64>(cl, &sh.word[0], ~0ull), [](u64 x, u64 y) { return x < y ? x : y; });
    z = over_lanes(of_lane_rank<u64>(cl, &sh.word[1], 0), [](u64 x, u64 y) { return x > y ? x : y; });
    cl.sync();
    lo = a;
    hi = z;
    const u64 span = hi - lo;
    s = span < kBins ? 0 : 64 - __clzll(span) - 10;
  }
}

// A key that at least `each` of the CTA's keys v (N a thread, `top` the largest)
// reach, and not many more; 1 above kNone if there are fewer.  Histograms over
// the range of keys that holds the each-th, until its bin has few.  (Two bits
// of the key a step, by counts: 11000 cycles a row for k = 1000, and 4000 so.)
template <typename T, int TH, int N>
__device__ __forceinline__ uint32_t bound_of(Block<TH>& bk, const uint32_t (&v)[N], unsigned each, uint32_t top) {
  Shared& sh = bk.sh;
  uint32_t lo = ~0u, hi = top;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (v[j] > Key<T>::kNone) lo = min(lo, v[j]);
  lo = ~bk.most32(~lo);
  if (lo == ~0u) return Key<T>::kNone + 1;
  unsigned want = each;
  for (;;) {
    const uint32_t span = hi - lo;
    const int s = span < kBins ? 0 : 32 - __clz(span) - 10;
    bk.clear(COUNT);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (v[j] >= lo && v[j] <= hi) atomicAdd(&sh.bins.count[(hi - v[j]) >> s], 1u);
    __syncthreads();
    auto count = [&](int b) { return sh.bins.count[b]; };
    if (bk.find([&](u64) { return (u64)want; }, [&](int b) { return (u64)count(b); }, count) < want) return Key<T>::kNone + 1;
    want -= (unsigned)sh.found_before;
    hi -= sh.found_bin << s;
    if (hi - lo >= (1u << s)) lo = hi - ((1u << s) - 1);
    if (s == 0 || sh.found_n <= 32 || sh.found_n * 4 <= each) return lo;
  }
}

// The same by one warp, without barriers, for its keys alone, but for low bits
// of a 32-bit key left at 0: two bits a step.
template <typename T, int N>
__device__ __forceinline__ uint32_t warp_bound_of(const uint32_t (&v)[N], unsigned each) {
  constexpr int kTop = sizeof(T) == 4 ? 30 : 14, kLow = sizeof(T) == 4 ? 12 : 0;
  uint32_t bound = 0;
#pragma unroll 1
  for (int b = kTop; b >= kLow; b -= 2) {
    unsigned c[3] = {0, 0, 0};
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int q = 0; q < 3; ++q) c[q] += v[j] >= (bound | ((uint32_t)(q + 1) << b));
    const unsigned two = __reduce_add_sync(kFull, c[0] | c[1] << 16), three = __reduce_add_sync(kFull, c[2]);
    const uint32_t q = three >= each ? 3 : (two >> 16) >= each ? 2 : (two & 0xffffu) >= each ? 1 : 0;
    bound |= q << b;
  }
  return max(bound, Key<T>::kNone + 1);
}

// The least key that min-p keeps: the lowest with z >= log(min_p).
template <typename T>
__device__ __forceinline__ uint32_t min_p_key(float min_p, uint32_t top, float temp, const Weigh& weigh) {
  const double zmin = log((double)fminf(min_p, 1.0f));
  if (weigh.infinite) return top;
  return lowest_key<T>(top, (float)(weigh.top_d + zmin * (double)temp),
                       [&](uint32_t k) { return weigh.z(Key<T>::value(k)) >= zmin; });
}

template <typename T, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) sample_rows_kernel(const __grid_constant__ SampleRowsDesc d) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  if (threadIdx.x < 32) {
    const double e = exp2(threadIdx.x * (1.0 / 32.0));
    sh.exp2_32[threadIdx.x] = __double2loint(e);
    sh.exp2_32[threadIdx.x + 32] = __double2hiint(e);
  }
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group cl = cg::this_cluster();
  constexpr int kWarps = TH / 32, kPart = kList / kWarps;  // tokens of a warp's part of the list
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x;
  constexpr bool kShort = TH == kShortThreads;  // a row of at most kList logits, one CTA
  const unsigned rank = kShort ? 0 : cl.block_rank(), ranks = kShort ? 1 : cl.num_blocks();
  const int base = (int)rank * d.per, n = max(0, min(d.per, d.V - base));
  constexpr int E = Slice<T, TH>::E;
  Slice<T, TH> sl;
  sl.src = static_cast<const T*>(d.logits) + (size_t)row * d.ld + base;
  sl.n = n;
  sl.nv = (n + E - 1) / E;
  sl.base = base;
  sl.aligned = (reinterpret_cast<uintptr_t>(sl.src) & 15) == 0;
  sl.kept = d.keep ? reinterpret_cast<uint4*>(smem + sizeof(Shared)) : nullptr;
  Block<TH> bk(sh);
  Filters f;
  const float temp = d.temperature ? d.temperature[row] : 1.0f;
  f.k = d.top_k ? d.top_k[row] : 0;
  f.p = d.top_p ? d.top_p[row] : 1.0f;
  const float mp = d.min_p ? d.min_p[row] : 0.0f;
  f.u = d.u[row];
  f.use_p = f.p < 1.0f;
  if (f.k < 0 || f.k >= d.V) f.k = 0;
  f.bins_per_unit = 32.0f / temp;
  const bool greedy = !(temp > 0.0f);
  // small top-k: the list is what lies above a bound
  const bool bounded = !greedy && f.k > 0 && f.k <= kList / 2 && f.k * 4 <= (int)ranks * TH * E;
  const unsigned each = bounded ? (f.k + ranks - 1) / ranks : 0;
  // 256 rows of 2048, k = 50: 8.0 us with one warp and a maximum a thread, 10.5
  // us with the whole CTA and all maxima, which a larger k needs
  const bool by_warp = f.k * 4 <= (int)ranks * TH;

  // ---- the row, its largest key and the bound ----------------------------------------
  uint32_t top = 0, bound = 0;
  sl.nan = false;
  for (;;) {
    uint32_t most[4], maxima[E];
    sl.largest(most);
    sl.apart(make_uint4(most[0], most[1], most[2], most[3]), maxima);
    const uint32_t own_top = sl.largest_of(make_uint4(most[0], most[1], most[2], most[3]));
    top = bk.most32(own_top);
    if (bounded && by_warp) {
      unsigned* own = reinterpret_cast<unsigned*>(sh.weight);
      own[tid] = own_top;
      __syncthreads();
      if (warp == 0) {
        uint32_t v[kWarps];
#pragma unroll
        for (int j = 0; j < kWarps; ++j) v[j] = own[j * 32 + lane];
        bound = warp_bound_of<T>(v, each);
      }
      if (ranks == 1) {
        if (tid == 0) sh.key_word[1] = bound;
        __syncthreads();
        bound = sh.key_word[1];
      }
    } else if (bounded) {
      bound = bound_of<T, TH>(bk, maxima, each, top);
    }
    if (ranks > 1) {
      if (tid == 0) {
        sh.key_word[0] = top;
        sh.key_word[1] = bound;
      }
      cl.sync();
      top = __reduce_max_sync(kFull, of_lane_rank<unsigned>(cl, &sh.key_word[0], 0u));
      bound = __reduce_min_sync(kFull, of_lane_rank<unsigned>(cl, &sh.key_word[1], ~0u));
    }
    if (top <= Key<T>::kInf || sl.nan) break;
    sl.nan = true;  // the same again without them
    if (ranks > 1) cl.sync();
  }
  if (top <= Key<T>::kNone || greedy) {
    // the first column with the largest key
    unsigned at = 0xffffffffu;
    if (top > Key<T>::kNone)
      sl.between((u64)top << 32, ((u64)top << 32) | 0xffffffffu, [&](float, u64 c) { at = min(at, ~(uint32_t)c); });
    at = ~bk.most32(~at);
    if (ranks > 1) {
      if (tid == 0) sh.word[0] = at;
      cl.sync();
      at = __reduce_min_sync(kFull, (unsigned)of_lane_rank<u64>(cl, &sh.word[0], ~0ull));
      cl.sync();  // no CTA leaves while its word is read
    }
    if (rank == 0 && tid == 0) answer(d, row, (int)at, at != 0xffffffffu, 0.0, 1ull << kFix);
    return;
  }
  const Weigh weigh(Key<T>::value(top), temp, sh.exp2_32);
  f.min_place = (u64)(mp > 0.0f ? min_p_key<T>(mp, top, temp, weigh) : Key<T>::kNone + 1) << 32;
  const int seg = (sl.nv + kWarps - 1) / kWarps, v0 = min(sl.nv, warp * seg), v1 = min(sl.nv, v0 + seg);  // a warp's vectors

  // ---- a list: what lies above the bound, or a short row ---------------------------
  if (bounded) {
    unsigned mine = 0;
    for (int w0 = v0; w0 < v1; w0 += 64) {  // in the order of the columns
      uint4 u[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int v = w0 + q * 32 + lane;
        u[q] = make_uint4(0, 0, 0, 0);
        if (v < v1) u[q] = sl.words(v);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (w0 + q * 32 >= v1) break;
        const unsigned lanes = __ballot_sync(kFull, sl.largest_of(u[q]) >= bound);
        if (!lanes) continue;
        uint32_t k[E];
        sl.apart(u[q], k);
        unsigned hits = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) hits |= k[j] >= bound ? 1u << j : 0u;
        // the hits of lower lanes: mostly one a lane
        const unsigned own = __popc(hits);
        unsigned at = __popc(lanes & ((1u << lane) - 1)), all = __popc(lanes);
        if (__any_sync(kFull, own > 1)) {
          at = own;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(kFull, at, o);
            if (lane >= o) at += y;
          }
          all = __shfl_sync(kFull, at, 31);
          at -= own;
        }
        at += mine;
        for (; hits; hits &= hits - 1, ++at) {
          const int j = __ffs(hits) - 1;
          if (at < kPart) sh.weight[warp * kPart + at] = place_of(sl.pick(u[q], j), base + (w0 + q * 32 + lane) * E + j);
        }
        mine += all;
      }
    }
    if (lane == 0) sh.part[warp] = mine;
    if (ranks > 1) cl.sync();
    else __syncthreads();
    const int parts = (int)ranks * kWarps;  // at most 16 * 16
    unsigned m = 0;
    if (tid < parts) m = ranks > 1 ? cl.map_shared_rank(sh.part, tid / kWarps)[tid % kWarps] : sh.part[tid];
    u64 total;
    const u64 at = bk.prefix(m, &total);
    const bool fits = __syncthreads_and(total <= kList && m <= (unsigned)kPart);
    if (fits) {
      if (rank == 0) {
        if (tid < parts) sh.offset[tid] = ((unsigned)at << 12) | m;
        __syncthreads();
        const int g = TH / parts, p = tid / g;  // threads of a part (powers of two)
        const unsigned o = sh.offset[p] >> 12, c = sh.offset[p] & 4095u;
        const u64* from = (ranks > 1 ? cl.map_shared_rank(sh.weight, p / kWarps) : sh.weight) + (p % kWarps) * kPart;
#pragma unroll 4
        for (unsigned i = tid % g; i < c; i += g) sh.list[o + i] = from[i];
      }
      if (ranks > 1) cl.sync();
      else __syncthreads();
      if (rank != 0) return;
      if (total <= kSmall) {
        if (warp == 0) draw_small<T>(sh, d, weigh, f, row, (int)total);
      } else {
        draw_from_list<T>(bk, d, weigh, f, row, (int)total);
      }
      return;
    }
    if (ranks > 1) cl.sync();
  }
  if constexpr (kShort) {
    for (int v = tid; v < sl.nv; v += TH) {
      uint32_t k[E];
      sl.apart(sl.words(v), k);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (v * E + j < n) sh.list[v * E + j] = k[j] > Key<T>::kNone ? place_of(k[j], v * E + j) : 0ull;
    }
    __syncthreads();
    draw_from_list<T>(bk, d, weigh, f, row, n);
  } else {
    // ---- otherwise: the last kept place by histograms over the cluster ----------------
    u64 last = (u64)(Key<T>::kNone + 1) << 32;
    if (f.k > 0)
      last = cluster_select(cl, bk, sl, COUNT, [&](u64) { return (u64)f.k; }, last, top, weigh, f.bins_per_unit);
    if (f.use_p)
      last = cluster_select(cl, bk, sl, WEIGHT, [&](u64 total) { return nucleus(f.p, total); }, last, top, weigh,
                            f.bins_per_unit);

    // ---- the draw: a warp's vectors, then the threads of the CTA over that warp's ----
    last = last > f.min_place ? last : f.min_place;
    const auto floor = sl.floor_of(last, weigh);
    u64 sum = 0;
    unsigned cnt = 0;
    static_assert(sizeof(sh.list) + sizeof(sh.weight) >= TH * 16 * sizeof(float), "a column of 16 a thread");
    if (key_in(last) > Key<T>::kNone + 1) {
      __syncthreads();
      sl.gathered(v0, v1, floor, weigh, reinterpret_cast<float*>(sh.list), sum, cnt);
    } else {
      sl.weighed(v0 + lane, v1, 32, floor, weigh, [&](int, float, u64 w, int) {
        sum += w;
        ++cnt;
      });
    }
    sum = lanes_sum(sum);
    cnt = bk.sum32(cnt);
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
    const int t0 = min(sl.nv, w * seg), t1 = min(sl.nv, t0 + seg), more = (t1 - t0 + TH - 1) / TH;
    const int a0 = min(t1, t0 + tid * more), a1 = min(t1, a0 + more);
    u64 own = 0, all;
    sl.weighed(a0, a1, 1, floor, weigh, [&](int, float, u64 w, int) { own += w; });
    u64 at = run + bk.prefix(own, &all);
    if (goal < at || goal >= at + own) return;
    sl.weighed(a0, a1, 1, floor, weigh, [&](int i, float l, u64 w, int) {
      if (at <= goal && goal < at + w) answer(d, row, base + i, (int)count, weigh.z(l), total);
      at += w;
    });
  }
}

// Bytes of a CTA's columns up to which they stay in shared memory: two CTAs an
// SM fit.  (One row of 151936 f32 logits, 38 KB a CTA, top-p: 30.3 us, and 31.4
// us read through the L2 cache pass by pass.)
constexpr int kKeep = 48 * 1024;
template <typename T, int TH>
cudaError_t launch_t(const SampleRowsDesc& d, int n_rows, int ranks, cudaStream_t st) {
  const size_t smem = sizeof(Shared) + (d.keep ? d.per * sizeof(T) : 0);
  static std::atomic<int> ready[kMaxDevices];
  const cudaError_t set = once_per_device(ready, [] {
    const cudaError_t e = cudaFuncSetAttribute(sample_rows_kernel<T, TH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)sizeof(Shared) + kKeep);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(sample_rows_kernel<T, TH>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (set != cudaSuccess) return set;
  return launch_k(sample_rows_kernel<T, TH>, dim3(n_rows, ranks), dim3(TH), smem, st,
                  LaunchOpts{true, (unsigned)ranks}, d);
}
template <typename T>
cudaError_t launch(SampleRowsDesc d, int n_rows, int sms, cudaStream_t st) {
  // Rows that do not fill the device (two CTAs an SM) are spread over more
  // CTAs, down to 4096 logits each.
  int ranks = 1;
  while (ranks < 16 && (d.V > ranks * kMaxSlice || (d.V > ranks * 4096 && (long)n_rows * ranks <= sms))) ranks *= 2;
  d.per = ((d.V + ranks - 1) / ranks + 31) / 32 * 32;
  d.keep = d.per * sizeof(T) <= kKeep;
  return d.V <= kList ? launch_t<T, kShortThreads>(d, n_rows, 1, st) : launch_t<T, 512>(d, n_rows, ranks, st);
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
  if (!words_aligned({temperature, top_k, top_p, min_p, u, token, kept, logprob}))
    return fail(QTTS_ERR_BADARG, "sample rows: a misaligned array of a value a row");
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
