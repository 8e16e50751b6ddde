// sample_rows.cu -- temperature / top-k / top-p / min-p sampling of rows of
// logits from given uniform numbers (sm_100a).
//
// A cluster of CTAs holds one row in shared memory (order keys of its f32
// logits), so that the logits are read from HBM once whatever the filters.
// Weights w = exp((l - largest) / T) become integers of 2^-45 (f64 exp), whose
// sums do not depend on their order.  The last kept token of the top-k and
// top-p filters is found by a radix selection over the keys, counts and
// weights per digit; ties at it are kept in index order.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "engine.h"
#include "kv8.h"

namespace cg = cooperative_groups;

namespace qtts {

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr unsigned kFull = 0xffffffffu;
constexpr int kFix = 45;  // fraction bits of a weight: 2^18 weights of 1 stay below 2^63
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

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

struct Weigh {
  float top;    // the largest logit
  double inv_t;
  __device__ __forceinline__ double z(float l) const {
    const double x = ((double)l - (double)top) * inv_t;
    return l == top ? 0.0 : x <= 0.0 ? x : -INFINITY;  // an infinite top over an infinite temperature is no number
  }
  __device__ __forceinline__ u64 operator()(float l) const {
    const double x = z(l);
    return x < -33.0 ? 0ull : __double2ull_rn(exp(x) * (double)(1ull << kFix));
  }
};

struct Shared {
  u64 mass[256];
  unsigned count[256];
  u64 scan[kWarps + 1];
  u64 part[4];  // this CTA's word for the cluster
  u64 best;
  u64 sel_mass;
  unsigned sel_count, sel_digit;
  int found;
};

// sum of one value per CTA over the cluster, and the sum over lower ranks
__device__ __forceinline__ void cluster_sum(cg::cluster_group& cl, Shared& sh, u64 v, u64* total, u64* before) {
  if (threadIdx.x == 0) sh.part[0] = v;
  cl.sync();
  u64 t = 0, b = 0;
  for (unsigned r = 0; r < cl.num_blocks(); ++r) {
    const u64 x = cl.map_shared_rank(sh.part, r)[0];
    if (r < cl.block_rank()) b += x;
    t += x;
  }
  *total = t;
  *before = b;
  cl.sync();
}
// sum of one value per warp over the CTA; *before: over lower warps
__device__ __forceinline__ u64 block_sum(Shared& sh, u64 warp_value, u64* before) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) sh.scan[warp] = warp_value;
  __syncthreads();
  u64 t = 0, b = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) b += sh.scan[w];
    t += sh.scan[w];
  }
  *before = b;
  return t;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_rows_kernel(const __grid_constant__ SampleRowsDesc d) {
  extern __shared__ uint32_t keys[];
  __shared__ Shared sh;
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x;
  const unsigned rank = cl.block_rank(), ranks = cl.num_blocks();
  const int base = (int)rank * d.per, n = max(0, min(d.per, d.V - base));
  const T* src = static_cast<const T*>(d.logits) + (size_t)row * d.ld + base;

  // ---- the row's keys, and the first token of the order -----------------------
  u64 best = 0;
  for (int i = tid; i < n; i += kThreads) {
    const uint32_t k = key_of(to_f32(src[i]));
    keys[i] = k;
    const u64 b = k ? ((u64)k << 32) | (uint32_t)~(base + i) : 0ull;
    best = best > b ? best : b;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const u64 x = __shfl_xor_sync(kFull, best, o);
    best = best > x ? best : x;
  }
  if (lane == 0) sh.scan[warp] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 0; w < kWarps; ++w) best = best > sh.scan[w] ? best : sh.scan[w];
    sh.best = best;
  }
  cl.sync();
  best = 0;
  for (unsigned r = 0; r < ranks; ++r) {
    const u64 x = *cl.map_shared_rank(&sh.best, r);
    best = best > x ? best : x;
  }
  const float temp = d.temperature ? d.temperature[row] : 1.0f;
  if (best == 0 || !(temp > 0.0f)) {
    if (rank == 0 && tid == 0) {
      d.token[row] = best == 0 ? -1 : (int)~(uint32_t)best;
      if (d.kept) d.kept[row] = best == 0 ? 0 : 1;
      if (d.logprob) d.logprob[row] = best == 0 ? -INFINITY : 0.0f;
    }
    cl.sync();  // no CTA leaves while its word is read
    return;
  }
  Weigh weigh;
  weigh.top = value_of((uint32_t)(best >> 32));
  weigh.inv_t = 1.0 / (double)temp;

  // ---- last kept key of top-k, then of top-p ------------------------------------
  const int k = d.top_k ? d.top_k[row] : 0;
  const float pf = d.top_p ? d.top_p[row] : 1.0f;
  const bool use_k = k > 0 && k < d.V, use_p = pf < 1.0f;
  uint32_t tau = 1;           // keys above tau are kept, and the first `ties` of those equal to it
  u64 ties = ~0ull;
  for (int pass = 0; pass < 2; ++pass) {
    if (!(pass ? use_p : use_k)) continue;
    u64 target = (u64)k;  // the entry at which the running count (weight) reaches this is the last kept
    if (pass == 1) {
      u64 s = 0, unused;
      if (use_k) {  // weight of the top-k set
        for (int i = tid; i < n; i += kThreads)
          if (keys[i] > tau) s += weigh(value_of(keys[i]));
      } else {
        for (int i = tid; i < n; i += kThreads)
          if (keys[i]) s += weigh(value_of(keys[i]));
      }
      s = block_sum(sh, warp_sum(s), &unused);
      u64 total;
      cluster_sum(cl, sh, s, &total, &unused);
      if (use_k) total += (ties == ~0ull ? 0 : ties) * weigh(value_of(tau));
      const double want = (double)pf * (double)total;
      target = want > 1.0 ? (u64)ceil(want) : 1;  // at least the first token
    }
    // digits from the top: `above` counts (weighs) the keys above the prefix
    uint32_t prefix = 0;
    u64 above = 0;
    unsigned equal = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) {
        sh.mass[i] = 0;
        sh.count[i] = 0;
      }
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const uint32_t x = keys[i];
        if (x < tau || x == 0) continue;  // outside the top-k set
        if (shift < 24 && (x >> (shift + 8)) != (prefix >> (shift + 8))) continue;
        const int b = (x >> shift) & 255;
        atomicAdd(&sh.count[b], 1u);
        if (pass) atomicAdd(&sh.mass[b], weigh(value_of(x)));
      }
      cl.sync();
      if (warp == 0) {  // eight digits a lane, from the top one down
        u64 w[8], own = 0;
        unsigned c[8];
        for (int j = 0; j < 8; ++j) {
          const int b = 255 - (lane * 8 + j);
          w[j] = 0;
          c[j] = 0;
          for (unsigned r = 0; r < ranks; ++r) {
            c[j] += cl.map_shared_rank(sh.count, r)[b];
            w[j] += cl.map_shared_rank(sh.mass, r)[b];
          }
          if (pass == 0) w[j] = c[j];
          own += w[j];
        }
        u64 incl = own;
        for (int o = 1; o < 32; o <<= 1) {
          const u64 x = __shfl_up_sync(kFull, incl, o);
          if (lane >= o) incl += x;
        }
        u64 run = above + incl - own;
        // the lane whose digits hold the target; the last one with anything if none does
        const bool hit = run < target && run + own >= target;
        const unsigned hits = __ballot_sync(kFull, hit), some = __ballot_sync(kFull, own > 0);
        const int who = hits ? __ffs(hits) - 1 : 31 - __clz(some | 1u);
        if (lane == who) {
          int j = 0, last = 0;
          u64 at = run;
          for (; j < 8; ++j) {
            if (w[j] == 0) continue;
            last = j;
            at = run;
            if (run + w[j] >= target) break;
            run += w[j];
          }
          sh.sel_digit = 255 - (lane * 8 + last);
          sh.sel_mass = at;
          sh.sel_count = c[last];
        }
      }
      __syncthreads();
      prefix |= sh.sel_digit << shift;
      above = sh.sel_mass;
      equal = sh.sel_count;
      cl.sync();
    }
    // `equal` tokens have the key; how many of them, in index order, are kept
    const u64 each = pass == 0 ? 1 : weigh(value_of(prefix));
    u64 t = each ? (target - above + each - 1) / each : equal;
    if (pass == 1 && prefix == tau && t > ties) t = ties;
    if (t > equal) t = equal;
    tau = prefix;
    ties = t;
  }

  // ---- ties in index order, min-p, and the draw ------------------------------------
  const float mp = d.min_p ? d.min_p[row] : 0.0f;
  const double zmin = mp > 0.0f ? log((double)fminf(mp, 1.0f)) : -INFINITY;
  const int seg = (d.per + kWarps - 1) / kWarps, s0 = min(n, warp * seg), s1 = min(n, s0 + seg);  // a warp's columns
  u64 tie_before = 0;
  if (ties != ~0ull) {
    u64 e = 0, wb, total, cb;
    for (int i = s0 + lane; i < s1; i += 32) e += keys[i] == tau;
    e = warp_sum(e);
    const u64 mine = block_sum(sh, e, &wb);
    cluster_sum(cl, sh, mine, &total, &cb);
    tie_before = wb + cb;
  }
  u64 sum = 0, cnt = 0, tb = tie_before;
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t x = i < s1 ? keys[i] : 0u;
    const unsigned eq = __ballot_sync(kFull, i < s1 && x == tau);
    bool keep = x != 0 && (x > tau || (x == tau && tb + __popc(eq & ((1u << lane) - 1)) < ties));
    tb += __popc(eq);
    if (keep) {
      const float l = value_of(x);
      if (weigh.z(l) >= zmin) {
        sum += weigh(l);
        ++cnt;
      }
    }
  }
  sum = warp_sum(sum);
  cnt = warp_sum(cnt);
  u64 wb, wc, total, before, count, cb;
  const u64 mine = block_sum(sh, sum, &wb);
  cluster_sum(cl, sh, mine, &total, &before);
  const u64 mine_c = block_sum(sh, cnt, &wc);
  cluster_sum(cl, sh, mine_c, &count, &cb);
  const float uf = d.u[row];
  const double want = uf > 0.0f ? fmin((double)uf, 1.0) * (double)total : 0.0;
  u64 goal = (u64)want;  // the running sum passes u * total: it is above its floor
  if (goal >= total) goal = total - 1;
  u64 run = before + wb;
  if (run <= goal && goal < run + sum) {  // this warp holds the drawn token
    tb = tie_before;
    for (int i0 = s0; i0 < s1; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t x = i < s1 ? keys[i] : 0u;
      const unsigned eq = __ballot_sync(kFull, i < s1 && x == tau);
      bool keep = x != 0 && (x > tau || (x == tau && tb + __popc(eq & ((1u << lane) - 1)) < ties));
      tb += __popc(eq);
      u64 w = 0;
      if (keep) {
        const float l = value_of(x);
        if (weigh.z(l) >= zmin) w = weigh(l);
      }
      u64 incl = w;
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += y;
      }
      const unsigned past = __ballot_sync(kFull, run + incl > goal);
      if (past) {
        if (lane == __ffs(past) - 1) {
          d.token[row] = base + i;
          if (d.kept) d.kept[row] = (int)count;
          if (d.logprob) d.logprob[row] = (float)(weigh.z(value_of(x)) - log((double)total * (1.0 / (1ull << kFix))));
        }
        break;
      }
      run += __shfl_sync(kFull, incl, 31);
    }
  }
}

template <typename T>
cudaError_t launch_t(SampleRowsDesc d, int n_rows, int ranks, cudaStream_t st) {
  const size_t smem = (size_t)d.per * 4;
  const cudaError_t e =
      cudaFuncSetAttribute(sample_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  return launch_k(sample_rows_kernel<T>, dim3(n_rows, ranks), dim3(kThreads), smem, st, LaunchOpts{true, (unsigned)ranks},
                  d);
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
  int ranks = 1;
  while (ranks < 8 && (V > ranks * 16384 || (V > ranks * 4096 && n_rows * ranks < on.sm_count))) ranks *= 2;
  d.per = ((V + ranks - 1) / ranks + 31) / 32 * 32;
  cudaError_t e;
  switch (dtype) {
    case QTTS_F16: e = launch_t<__half>(d, n_rows, ranks, (cudaStream_t)stream); break;
    case QTTS_BF16: e = launch_t<__nv_bfloat16>(d, n_rows, ranks, (cudaStream_t)stream); break;
    default: e = launch_t<float>(d, n_rows, ranks, (cudaStream_t)stream);
  }
  if (e == cudaSuccess) return QTTS_OK;
  cudaGetLastError();
  return fail(QTTS_ERR_CUDA, cudaGetErrorString(e));
} catch (...) {
  return QTTS_ERR_OOM;
}
