// kv8.cu -- the paged K/V cache held in 8 bits (sm_100a): appending to it with
// QK-norm and position rotation on the way, and attention over it.
//
// A page holds 16 positions of every K/V head: codes int8
// [page][K|V][kv_head][16][head_dim], one f32 scale per [page][K|V][kv_head];
// an element's value is code * scale.
#include <cooperative_groups.h>
#include <float.h>

#include <algorithm>

#include "common.cuh"
#include "engine.h"
#include "kv8.cuh"

namespace cg = cooperative_groups;

namespace qtts {

namespace {

// ---- append --------------------------------------------------------------------
// A head's row of HD values lies on HD / 4 lanes, four consecutive values each,
// so that loads and the 4-byte code stores are whole lines and the rotation's
// partner (half a head away) is one lane shuffle away.

// RMS norm over the head (the formula of the q/k/v epilogue): the mean of
// squares is summed in f64 (order-free to f32, so that a code does not depend
// on the reduction tree), everything after it is one f32 rounding per step.
//
// N heads (or tokens) at a time: their sums of squares are reduced together (at
// each step half of the lanes keep one half of the values), after which lane j
// of a head's lanes holds the sum of value j % N; the square root and the
// division, a few dozen instructions, are done once for all of them.
template <int HD, int N>
__device__ __forceinline__ void head_norm(float4 (&x)[N], float4 g) {
  constexpr int L = HD / 4;  // lanes of a head
  static_assert((N & (N - 1)) == 0 && N <= L, "values are halved between lanes");
  const int lane = threadIdx.x & 31;
  double ss[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    ss[i] = (double)x[i].x * x[i].x + (double)x[i].y * x[i].y + (double)x[i].z * x[i].z + (double)x[i].w * x[i].w;
#pragma unroll
  for (int n = N / 2; n; n >>= 1) {  // lane bit n: which half of the values this lane keeps
    const bool up = lane & n;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const double give = up ? ss[i] : ss[i + n], keep = up ? ss[i + n] : ss[i];
      ss[i] = keep + __shfl_xor_sync(kFull, give, n);
    }
  }
#pragma unroll
  for (int o = N; o < L; o <<= 1) ss[0] += __shfl_xor_sync(kFull, ss[0], o);
  const float own = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn((float)(ss[0] / HD), 1e-6f)));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float inv = __shfl_sync(kFull, own, (lane & ~(N - 1)) | i);
    x[i] = make_float4(__fmul_rn(__fmul_rn(x[i].x, inv), g.x), __fmul_rn(__fmul_rn(x[i].y, inv), g.y),
                       __fmul_rn(__fmul_rn(x[i].z, inv), g.z), __fmul_rn(__fmul_rn(x[i].w, inv), g.w));
  }
}
// (a, b) -> (a cos - b sin, b cos + a sin) of the two halves, products and sum
// rounded one by one (no contraction); s is -sin on the lanes of the first half
// (a product's sign change is exact).
template <int HD>
__device__ __forceinline__ float4 rotate(float4 x, float4 c, float4 s) {
  const float4 y = make_float4(__shfl_xor_sync(kFull, x.x, HD / 8), __shfl_xor_sync(kFull, x.y, HD / 8),
                               __shfl_xor_sync(kFull, x.z, HD / 8), __shfl_xor_sync(kFull, x.w, HD / 8));
  return make_float4(__fadd_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, s.x)),
                     __fadd_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, s.y)),
                     __fadd_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, s.z)),
                     __fadd_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, s.w)));
}
__device__ __forceinline__ float4 signed_sin(float4 s, bool upper) {
  return upper ? s : make_float4(-s.x, -s.y, -s.z, -s.w);
}
__device__ __forceinline__ float4 norm_weight(const __half* w, int d0) {
  return w ? load4(w + d0) : make_float4(1.f, 1.f, 1.f, 1.f);
}

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= FLT_MAX ? a : 0.0f;  // NaN and infinities set no scale
}
// nearest code, ties to even; NaN -> 0, infinities -> +-127
__device__ __forceinline__ uint32_t code_of(float v, float inv) {
  const int q = __float2int_rn(__fmul_rn(v, inv));
  return (uint32_t)max(-127, min(127, q)) & 0xffu;
}
__device__ __forceinline__ uint32_t codes4(float4 v, float inv) {
  return code_of(v.x, inv) | (code_of(v.y, inv) << 8) | (code_of(v.z, inv) << 16) | (code_of(v.w, inv) << 24);
}
// The same for finite values of at most 127 steps: the sum with 1.5 * 2^23
// rounds to the nearest, ties to even, and its low byte is the code.
__device__ __forceinline__ uint32_t small_codes4(float4 v, float inv) {
  const float b = 12582912.0f;
  const uint32_t x = __float_as_uint(__fadd_rn(__fmul_rn(v.x, inv), b)), y = __float_as_uint(__fadd_rn(__fmul_rn(v.y, inv), b)),
                 z = __float_as_uint(__fadd_rn(__fmul_rn(v.z, inv), b)), w = __float_as_uint(__fadd_rn(__fmul_rn(v.w, inv), b));
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t abs_bits4(float4 v) {
  return max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
}
__device__ __forceinline__ uint32_t requant4(uint32_t w, float ratio) {
  const float4 v = make_float4((float)(int8_t)(w & 0xff), (float)(int8_t)((w >> 8) & 0xff),
                               (float)(int8_t)((w >> 16) & 0xff), (float)(int8_t)(w >> 24));
  return codes4(v, ratio);
}

// four elements as they lie in memory
template <typename T>
struct alignas(4 * sizeof(T)) Raw4 {
  uint32_t w[sizeof(T)];
};

// Tokens of a block that registers hold in a chunk of a prompt.  16 chunks of
// 611 rows: 66 us with 4; 122, 78 and 73 us with 16, 8 and 2 (fewer need more
// passes, more leave fewer warps an SM to hide the loads).
constexpr int kAppendKeep = 4;
// Rows [chunk * d.chunk, + d.chunk): every block (run of rows of one sequence,
// consecutive positions, one page) that starts there, for one K or V head.
// KEEP tokens are worked out at a time; between the maximum and the codes those
// of a longer block lie in `kept`, this lane's part of shared memory.
template <typename T, int HD, int KEEP>
__device__ void append_blocks(const Kv8AppendDesc& d, int chunk, int which, int h, float4* kept) {
  constexpr int LPT = HD / 4, TPW = 32 / LPT, STEPS = KEEP / TPW;  // lanes per token, tokens per step
  const int lane = threadIdx.x & 31, sub = lane / LPT, d0 = (lane % LPT) * 4;
  const bool upper = (lane % LPT) >= LPT / 2;
  const qtts_kv8_cache& c = d.c;
  // lane i holds row first + i; a block that starts in the chunk ends before lane 32
  const int first = chunk * d.chunk - 1, row = first + lane;
  int seq = -1, pos = -1, rope = -1;
  if (row >= 0 && row < d.n_rows) {
    seq = d.seq[row];
    pos = d.pos[row];
    rope = d.rope_pos ? d.rope_pos[row] : pos;
  }
  const bool turn = which == 0 && d.rope_cos != nullptr;
  const bool ok = seq >= 0 && seq < c.n_seqs && pos >= 0 && pos < c.pages_per_seq * kKv8Page;
  if (seq >= 0 && !ok && lane >= 1 && lane <= d.chunk) raise(d.flags, QTTS_KV8_BAD_ROW);
  const int pseq = __shfl_up_sync(kFull, seq, 1), ppos = __shfl_up_sync(kFull, pos, 1);
  const bool cont = ok && lane > 0 && pseq == seq && ppos == pos - 1 && pos % kKv8Page != 0;
  const unsigned conts = __ballot_sync(kFull, cont);
  unsigned starts = __ballot_sync(kFull, ok && !cont && lane >= 1 && lane <= d.chunk);
  const T* src = static_cast<const T*>(which ? d.v : d.k);
  const long ld = which ? d.ldv : d.ldk;
  const float4 g = norm_weight(which ? nullptr : d.k_norm, d0);
  while (starts) {
    const int i = __ffs(starts) - 1;
    starts &= starts - 1;
    const int n = i == 31 ? 1 : __ffs(~(conts >> (i + 1)));  // 1 + the rows that continue it
    const int bseq = __shfl_sync(kFull, seq, i), bpos = __shfl_sync(kFull, pos, i);
    const int slot0 = bpos % kKv8Page;
    const int page = c.page_table[(size_t)bseq * c.pages_per_seq + bpos / kKv8Page];
    if (page < 0 || page >= c.n_pages) {
      if (lane == 0) raise(d.flags, QTTS_KV8_BAD_PAGE);
      continue;
    }
    float* sp = block_scale(c, page, which, h);
    int8_t* codes = block_codes(c, page, which, h);
    const float had = slot0 ? *sp : 0.0f;
    float4 x[STEPS];
    uint32_t most = 0;  // the largest |value|'s bits, above those of FLT_MAX if one is not finite
    // the angles of a step's token; false: there are none (a rotation by 1 and 0
    // would not do, as 0 times an infinity half a head away is NaN)
    auto angles = [&](int t, float4& cs, float4& sn) {
      const int rp = __shfl_sync(kFull, rope, min(31, i + t));
      cs = sn = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t >= n) return false;
      if (rp < 0 || rp >= d.rope_rows) {
        raise(d.flags, QTTS_KV8_ROPE_RANGE);
        return false;
      }
      cs = load4(d.rope_cos + (size_t)rp * (HD / 2) + d0 % (HD / 2));
      sn = signed_sin(load4(d.rope_sin + (size_t)rp * (HD / 2) + d0 % (HD / 2)), upper);
      return true;
    };
    Raw4<T> raw[STEPS];  // the next tokens, on their way while the ones before are worked on
    const T* from = src + (size_t)(first + i + sub) * ld + (size_t)h * HD + d0;
    auto read = [&](int t0) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        raw[s] = Raw4<T>{};
        if (t0 + s * TPW + sub < n) raw[s] = *reinterpret_cast<const Raw4<T>*>(from + (size_t)(t0 + s * TPW) * ld);
      }
    };
    // x = tokens t0 .. t0 + KEEP of the block, normed and rotated; their largest
    auto tokens = [&](int t0) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) x[s] = load4(reinterpret_cast<const T*>(&raw[s]));
      if (t0 + KEEP < n) read(t0 + KEEP);
      float4 cs, sn;
      bool has = turn && angles(t0 + sub, cs, sn);  // (of each step while the one before is worked on)
      if (which == 0 && d.k_norm) {
        if (STEPS > 1 && n - t0 <= TPW) {  // one step
          float4 one[1] = {x[0]};
          head_norm<HD, 1>(one, g);
          x[0] = one[0];
        } else {
          head_norm<HD, STEPS>(x, g);
        }
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (t0 + s * TPW >= n) break;
        if (turn) {
          const float4 c0 = cs, s0 = sn;
          const bool now = has;
          if (s + 1 < STEPS && t0 + (s + 1) * TPW < n) has = angles(t0 + (s + 1) * TPW + sub, cs, sn);
          const float4 y = rotate<HD>(x[s], c0, s0);
          if (now) x[s] = y;
        }
        if (t0 + s * TPW + sub < n) most = max(most, abs_bits4(x[s]));
        if (n > KEEP) kept[(t0 / TPW + s) * 32] = x[s];
      }
    };
    auto each = [&](auto f) {  // f(x, token) for what this lane holds
#pragma unroll 1
      for (int t0 = 0; t0 < n; t0 += KEEP)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const int t = t0 + s * TPW + sub;
          if (t < n) f(n > KEEP ? kept[(t0 / TPW + s) * 32] : x[s], t);
        }
    };
    read(0);
#pragma unroll 1
    for (int t0 = 0; t0 < n; t0 += KEEP) tokens(t0);
    most = __reduce_max_sync(kFull, most);
    float big = __uint_as_float(most);
    const bool finite = most <= 0x7f7fffffu;
    if (!finite) {
      big = 0.0f;
      each([&](float4 v, int) {
        big = fmaxf(big, fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w))));
      });
#pragma unroll
      for (int o = 16; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(kFull, big, o));
    }
    // 127 steps to the largest value; the floor keeps 1 / scale finite
    const float need = big > 0.0f ? fmaxf(__fmul_rn(big, (float)(1.0 / 127.0)), FLT_MIN) : 0.0f;
    float scale = need;
    if (slot0) {
      // A block that grows does so by a quarter at least: its earlier codes
      // are rounded again, and with steps of 1.25 those roundings add up to
      // at most 1/2 (1 + 1/1.25 + ...) = 2.5 of the final steps.
      scale = need <= had ? had : fmaxf(need, __fmul_rn(1.25f, had));
      if (scale != had) {
        const float ratio = scale > 0.0f ? __fdiv_rn(had, scale) : 0.0f;
        for (int t = sub; t < slot0; t += TPW) {
          uint32_t* w = reinterpret_cast<uint32_t*>(codes + t * HD + d0);
          *w = requant4(*w, ratio);
        }
      }
    }
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    auto put = [&](int t, uint32_t w) { *reinterpret_cast<uint32_t*>(codes + (slot0 + t) * HD + d0) = w; };
    if (finite) each([&](float4 v, int t) { put(t, small_codes4(v, inv)); });
    else each([&](float4 v, int t) { put(t, codes4(v, inv)); });
    if (lane == 0) *sp = scale;
  }
}

constexpr int kQHeads = 4;  // query heads of a warp
// Rows of a warp of query heads: one where most rows are single tokens, which are
// few, and 2 of a prompt, whose loads hide each other.  (16 chunks of 611 rows:
// 55.2, 50.9, 51.9 and 56.2 us with 1, 2, 3 and 4.)
template <int KEEP>
constexpr int kQRows = KEEP == kAppendKeep ? 2 : 1;

// kQHeads query heads of rows [row, row + ROWS), from h0 on: the loads of all
// rows are on their way before the first is worked on.
template <typename T, int HD, int ROWS>
__device__ void rotate_queries(const Kv8AppendDesc& d, int row, int h0) {
  constexpr int LPT = HD / 4, TPW = 32 / LPT, N = kQHeads / TPW;
  const int lane = threadIdx.x & 31, sub = lane / LPT, d0 = (lane % LPT) * 4;
  const bool upper = (lane % LPT) >= LPT / 2;
  Raw4<T> raw[ROWS][N];
  int rp[ROWS];
  bool ok[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int at = min(row + r, d.n_rows - 1);
    const int seq = d.seq[at], pos = d.pos[at];
    rp[r] = d.rope_pos ? d.rope_pos[at] : pos;
    // (what is out of range is flagged with K and V)
    ok[r] = row + r < d.n_rows && seq >= 0 && seq < d.c.n_seqs && pos >= 0 && pos < d.c.pages_per_seq * kKv8Page;
    const T* src = static_cast<const T*>(d.q) + (size_t)at * d.ldq;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int h = h0 + i * TPW + sub;
      raw[r][i] = Raw4<T>{};
      if (h < d.heads) raw[r][i] = *reinterpret_cast<const Raw4<T>*>(src + (size_t)h * HD + d0);
    }
  }
  float4 cs[ROWS], sn[ROWS];
  bool turn[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    turn[r] = ok[r] && d.rope_cos != nullptr;
    if (turn[r]) {
      turn[r] = rp[r] >= 0 && rp[r] < d.rope_rows;
      if (turn[r]) {
        cs[r] = load4(d.rope_cos + (size_t)rp[r] * (HD / 2) + d0 % (HD / 2));
        sn[r] = load4(d.rope_sin + (size_t)rp[r] * (HD / 2) + d0 % (HD / 2));
      } else {
        raise(d.flags, QTTS_KV8_ROPE_RANGE);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (!ok[r]) continue;
    float4 x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = load4(reinterpret_cast<const T*>(&raw[r][i]));
    if (d.q_norm) head_norm<HD, N>(x, norm_weight(d.q_norm, d0));
    T* dst = static_cast<T*>(d.q_out) + (size_t)(row + r) * d.ldqo;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int h = h0 + i * TPW + sub;
      if (turn[r]) x[i] = rotate<HD>(x[i], cs[r], signed_sin(sn[r], upper));
      if (h < d.heads) store4(dst + (size_t)h * HD + d0, x[i]);
    }
  }
}

// A warp takes the blocks that start in a chunk of rows, for one K or V head
// (they are its alone: the block's scale needs all of its new tokens), or
// kQHeads query heads of one row.  Every input is read from HBM once, every
// output written once, and a block that grows has its earlier codes read and
// written again.  16 chunks of 611 bf16 rows (16 query, 8 K/V heads of 128):
// 51 us, 109 MB at 2.1 TB/s: 32 million warp instructions (norm, rotation and
// codes with each rounding of its own), issued in 57% of the cycles by 19 warps
// an SM, which wait for loads in between.  512 single f32 tokens: 8.2 us, 22 MB at
// 2.7 TB/s, which is 2.9 rounds of one warp's chain of loads and reductions; one
// token: 3.1 us.
template <typename T, int HD, int KEEP>
__global__ void __launch_bounds__(128, 6) kv8_append_kernel(const __grid_constant__ Kv8AppendDesc d) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kSteps = kKv8Page * HD / 128;  // float4 of a lane for a block's tokens
  __shared__ float4 s_kept[4][kSteps][32];
  const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w < d.kv_warps) {
    const int per = 2 * d.c.kv_heads, j = (int)(w % per);
    append_blocks<T, HD, KEEP>(d, (int)(w / per), j & 1, j >> 1, &s_kept[threadIdx.x >> 5][0][threadIdx.x & 31]);
  } else {
    const int per = (d.heads + kQHeads - 1) / kQHeads;
    const long i = w - d.kv_warps;
    const long row = per > 0 ? i / per * kQRows<KEEP> : d.n_rows;
    if (row < d.n_rows) rotate_queries<T, HD, kQRows<KEEP>>(d, (int)row, (int)(i % per) * kQHeads);
  }
}

// ---- attention -------------------------------------------------------------------
// Single tokens and few rows: a slot is a query head of a row, and a unit is up
// to 8 slots that share a K/V head and its pages; a warp takes every n-th page
// and keeps the running maximum and sum of each slot, and the output's sums.
// Scores: a query, scaled, is an integer of at most 127 * 2^16 in three signed
// bytes, and the products with the 8-bit codes on the integer matrix
// units are exact (f16 hi + lo took 13% longer).  A product of 16 rows takes
// two of the bytes of 8 slots.  Output: a weight times the V scale is split
// into f16 hi + lo, lo scaled by 2^11, about 22 bits, and V's codes are exact
// in f16: hi in row s and lo in row s + 8 of the 16-row operand, so the split
// costs nothing, and hi + lo of a slot meet in one thread; sums in f32.
//
// 256 sequences of up to 4099 positions (16 heads, 8 K/V heads of 128), one bf16
// row each: 288 - 312 us, 1.61 GB at 5.2 - 5.6 TB/s: HBM bounds it.  With fewer
// pages a warp, about 500 instructions a page and the start do (rows, then the
// table, then the pages: three trips to HBM; at the end the warps' sums): 64
// sequences of up to 530, f32: 21 us, 53 MB at 2.5 TB/s; one of 32003 in
// clusters of 10 CTAs of 12 warps: 29 us, 49 MB at 1.7 TB/s, as clusters of a
// K/V head each leave 68 SMs idle; one of 265: 7.0 us.

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void imma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Integer sums start at the bits of 1.5 * 2^23, so that a sum of less than
// 2^22 is read as a float by one subtraction.
constexpr int kIntBias = 0x4B400000;
constexpr float kFloatBias = 12582912.0f;
// Four numbers of at most 127 * 2^16 as three signed bytes each (x = 65536 l0 +
// 256 l1 + l2): the words of their l0, l1 and l2.
__device__ __forceinline__ void limbs4(float4 v, float up, uint32_t& w0, uint32_t& w1, uint32_t& w2) {
  const float x[4] = {v.x, v.y, v.z, v.w};
  w0 = w1 = w2 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int y = __float2int_rn(x[i] * up);
    w2 |= (uint32_t)(y & 255) << (8 * i);
    y = (y - (int)(int8_t)(y & 255)) >> 8;
    w1 |= (uint32_t)(y & 255) << (8 * i);
    y = (y - (int)(int8_t)(y & 255)) >> 8;
    w0 |= (uint32_t)(y & 255) << (8 * i);
  }
}
constexpr int kSlots = 8;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory of the single-token kernel.  Each warp has a ring of kStages
// pages; a page's K and V block is copied 16 bytes a lane, and the 16-byte
// chunks of a row change places so that the fragment reads below (8 lanes of
// 16 bytes at a time: K two rows x four chunks, V four rows x two chunks) hit
// every bank once.
constexpr int kStages = 4, kStep = 2;
template <int HD>
struct Ring {
  static constexpr int kBlock = kKv8Page * HD;  // bytes of one K or V block
  static constexpr int kPer = kBlock / 512;     // copies of a lane per block
  static constexpr int kWarp = kStages * 2 * kBlock;
  static __device__ __forceinline__ int k_at(int row, int byte) {
    return HD == 128 ? row * 128 + (byte ^ ((row & 1) << 6)) : row * 64 + byte;
  }
  static __device__ __forceinline__ int v_at(int row, int byte) {
    if (HD == 128) return row * 128 + (byte ^ ((row & 6) << 4));
    const int line = row >> 1;
    return line * 128 + ((((row & 1) << 6) | byte) ^ ((line & 3) << 5));
  }
};

template <typename T, int HD, int NW>
__global__ void __launch_bounds__(NW * 32, 12 / NW) kv8_attn_kernel(const __grid_constant__ Kv8AttnDesc d) {
  constexpr int NT = HD / 8;   // dims a thread's V chunk holds, and n-tiles of the output
  constexpr int KJ = HD / 64;  // 64-dim halves of a row
  using R = Ring<HD>;
  extern __shared__ __align__(128) uint8_t ring[];
  float(*s_o)[kSlots][HD] = reinterpret_cast<float(*)[kSlots][HD]>(ring);  // after the pages: each warp's sums
  static_assert(R::kWarp >= kSlots * HD * 4, "the warps' sums lie over the ring");
  __shared__ float s_scale[NW][kStages][2];
  __shared__ float s_m[NW][kSlots], s_l[NW][kSlots];
  __shared__ float s_po[kSlots][HD];
  __shared__ float s_pm[kSlots], s_pl[kSlots];
  pdl_launch_dependents();
  pdl_wait();
  const qtts_kv8_cache& c = d.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int nsplit = gridDim.y, split = blockIdx.y;
  const int per = c.kv_heads * d.head_chunks;
  const int unit = blockIdx.x / per, rest = blockIdx.x % per;
  const int kvh = rest / d.head_chunks, hc = rest % d.head_chunks;
  const int group = d.heads / c.kv_heads;
  const int h0 = kvh * group + hc * d.unit_heads;               // first query head of the unit
  const int nh = min(d.unit_heads, group - hc * d.unit_heads);  // its heads
  const int cap = c.pages_per_seq * kKv8Page;
  cg::cluster_group cluster = cg::this_cluster();
  uint8_t* my_ring = ring + warp * R::kWarp;
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(my_ring);
  const uint32_t scale_s = (uint32_t)__cvta_generic_to_shared(&s_scale[warp][0][0]);

  // lane i: row i of the unit
  const int unit_row0 = unit * d.group_rows, unit_rows = min(d.group_rows, d.n_rows - unit_row0);
  int rseq = -1, rpos = -1;
  if (lane < unit_rows) {
    rseq = d.seq[unit_row0 + lane];
    rpos = d.pos[unit_row0 + lane];
    if (rseq >= 0 && (rseq >= c.n_seqs || rpos >= cap)) {
      if (warp == 0) raise(d.flags, QTTS_KV8_BAD_ROW);
      if (rseq >= c.n_seqs) rseq = -1;
      rpos = min(rpos, cap - 1);
    }
  }
  for (int i0 = 0; i0 < unit_rows;) {
    // the next run of rows of one sequence: rows [i0, i0 + rows) of the unit
    const int seq = __shfl_sync(kFull, rseq, i0);
    const unsigned other = __ballot_sync(kFull, rseq != seq || lane >= unit_rows) & (kFull << i0);
    const int rows = (other ? __ffs(other) - 1 : 32) - i0;
    const bool mine = lane >= i0 && lane < i0 + rows && rpos >= 0;
    const int hi = __reduce_max_sync(kFull, mine ? rpos + 1 : 0);
    const int lo = __reduce_min_sync(kFull, mine ? (d.window > 0 ? max(0, rpos + 1 - d.window) : 0) : 0x7fffffff);
    const int row0 = unit_row0 + i0;
    const int slot_row = i0 + min(g / nh, rows - 1);
    const int slot_pos = __shfl_sync(kFull, rpos, slot_row);
    i0 += rows;
    if (seq < 0) continue;  // padding
    const int nslots = rows * nh;
    const bool on = g < nslots;

    // the slot's query is on its way before the pages, which would hold it up
    Raw4<T> raw[KJ][4];
    {
      const T* qp = static_cast<const T*>(d.q) + (size_t)(unit_row0 + slot_row) * d.ldq +
                    (size_t)(h0 + (on ? g % nh : 0)) * HD;
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          raw[j][i] = Raw4<T>{};
          if (on) raw[j][i] = *reinterpret_cast<const Raw4<T>*>(qp + 16 * (t + 4 * j) + 4 * i);
        }
    }

    // this split's pages [pb, pe); the warp takes every NW-th of them
    const int p0 = hi > 0 ? lo / kKv8Page : 0, p1 = (hi + kKv8Page - 1) / kKv8Page;
    const int share = (p1 - p0 + nsplit - 1) / nsplit;
    const int pb = p0 + split * share + warp, pe = min(p1, p0 + (split + 1) * share);
    const int np = pb < pe ? (pe - pb + NW - 1) / NW : 0;
    const int* table = c.page_table + (size_t)seq * c.pages_per_seq;
    int entries = -1;        // lane i: the page of the 32 * k + i-th of them
    unsigned skip = 0;       // bit s: stage s holds no page
    auto issue_page = [&](int i) {
      const int s = i % kStages;
      skip |= 1u << s;
      if (i < np) {
        if ((i & 31) == 0) {
          const int pg = pb + (i + lane) * NW;
          entries = pg < pe ? table[pg] : -1;
          if (pg < pe && (entries < 0 || entries >= c.n_pages)) {
            raise(d.flags, QTTS_KV8_BAD_PAGE);
            entries = -1;
          }
        }
        const int page = __shfl_sync(kFull, entries, i & 31);
        if (page >= 0) {
          skip &= ~(1u << s);
          const int8_t* kb = block_codes(c, page, 0, kvh) + lane * 16;
          const int8_t* vb = block_codes(c, page, 1, kvh) + lane * 16;
          const uint32_t dst = ring_s + s * 2 * R::kBlock;
#pragma unroll
          for (int j = 0; j < R::kPer; ++j) {
            const int row = (lane * 16 + j * 512) / HD, byte = lane * 16 % HD;
            cp_async16(dst + R::k_at(row, byte), kb + j * 512);
            cp_async16(dst + R::kBlock + R::v_at(row, byte), vb + j * 512);
          }
          if (lane < 2) cp_async4(scale_s + (s * 2 + lane) * 4, block_scale(c, page, lane, kvh));
        }
      }
    };
    auto issue = [&](int i) {
#pragma unroll
      for (int k = 0; k < kStep; ++k) issue_page(i + k);
      cp_async_commit();  // one group a step, empty or not
    };
#pragma unroll
    for (int i = 0; i < kStages; i += kStep) issue(i);

    // this thread's slot: query limbs, scale, and the positions it sees
    uint32_t q0[KJ * 4], q1[KJ * 4], q2[KJ * 4];
    float qscale;
    int see_lo = 0, see_hi = 0;
    {
      float4 x[KJ][4];
      float big = 0.0f;
      bool finite = true;
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[j][i] = load4(reinterpret_cast<const T*>(&raw[j][i]));
          const float4 v = make_float4(fabsf(x[j][i].x), fabsf(x[j][i].y), fabsf(x[j][i].z), fabsf(x[j][i].w));
          finite &= v.x <= FLT_MAX && v.y <= FLT_MAX && v.z <= FLT_MAX && v.w <= FLT_MAX;
          big = fmaxf(big, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
        }
      big = fmaxf(big, __shfl_xor_sync(kFull, big, 1));
      big = fmaxf(big, __shfl_xor_sync(kFull, big, 2));
      finite = ((__ballot_sync(kFull, finite) >> (lane & 28)) & 15u) == 15u;
      constexpr float kMost = 127.0f * 65536.0f;  // what the largest becomes: three signed bytes hold it
      const float top = fmaxf(big, 0x1p-100f), up = __fdiv_rn(kMost, top);
      qscale = finite ? d.scale * 1.4426950408889634f * (top * (1.0f / kMost)) : NAN;  // scores in units of log 2
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) limbs4(x[j][i], up, q0[j * 4 + i], q1[j * 4 + i], q2[j * 4 + i]);
      if (on) {
        see_hi = slot_pos + 1;
        see_lo = d.window > 0 ? max(0, see_hi - d.window) : 0;
      }
    }
    // The matrix units' sums are cut off, not rounded, which adds up over a long
    // cache (26177 positions, 4 warps: 1.3e-5).  With f32 rows they hold one step,
    // and `sum` all of them, rounded (2.7e-6, and 8e-7 with l's roundings made up
    // for); 16-bit results do not show the difference.
    constexpr bool kRounded = sizeof(T) == 4;
    float o[NT][4], sum[kRounded ? NT : 1][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
      if constexpr (kRounded) sum[i][0] = sum[i][1] = 0.0f;
    }
    float m = -INFINITY, mo = -INFINITY, l = 0.0f, lost = 0.0f;  // lost: what roundings added to l

    // kStep pages at a time: independent chains of products and one running
    // maximum for all of them
    for (int i = 0; i < np; i += kStep) {
      cp_async_wait<kStages / kStep - 1>();
      __syncwarp();  // every lane's copies of these pages are there
      const int st = i % kStages;
      const uint8_t* base = my_ring + st * 2 * R::kBlock;
      const int at0 = (pb + i * NW) * kKv8Page + 2 * t;
      // scores of positions 8n + 2t, + 1 of slot g: l0, l1 in hi, l2 in lo
      int hi_[kStep][2][4], lo_[kStep][2][4];
#pragma unroll
      for (int k = 0; k < kStep; ++k)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) hi_[k][n][e] = lo_[k][n][e] = kIntBias;
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int k = 0; k < kStep; ++k)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint4 w = *reinterpret_cast<const uint4*>(base + k * 2 * R::kBlock + R::k_at(n * 8 + g, 16 * (t + 4 * j)));
            imma16832(hi_[k][n], q0[j * 4], q1[j * 4], q0[j * 4 + 1], q1[j * 4 + 1], w.x, w.y);
            imma16832(lo_[k][n], q2[j * 4], 0, q2[j * 4 + 1], 0, w.x, w.y);
            imma16832(hi_[k][n], q0[j * 4 + 2], q1[j * 4 + 2], q0[j * 4 + 3], q1[j * 4 + 3], w.z, w.w);
            imma16832(lo_[k][n], q2[j * 4 + 2], 0, q2[j * 4 + 3], 0, w.z, w.w);
          }
      float s[kStep][2][2], pm[kStep], ev[kStep], fr[kStep];
#pragma unroll
      for (int k = 0; k < kStep; ++k) {
        const bool there = !((skip >> (st + k)) & 1);
        const float f = qscale * s_scale[warp][st + k][0], sv = there ? s_scale[warp][st + k][1] : 0.0f;
        pm[k] = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at = at0 + k * NW * kKv8Page + n * 8 + e;
            s[k][n][e] = there && at >= see_lo && at < see_hi
                             ? f * fmaf(__int_as_float(hi_[k][n][e]) - kFloatBias, 65536.0f,
                                        fmaf(__int_as_float(hi_[k][n][e + 2]) - kFloatBias, 256.0f,
                                             __int_as_float(lo_[k][n][e]) - kFloatBias))
                             : -INFINITY;
            pm[k] = fmaxf(pm[k], s[k][n][e]);
          }
        // sv = fr * 2^ev; the output's running exponent follows score + ev, so
        // that the weights times sv stay within f16 whatever the scales are
        split_scale(sv, ev[k], fr[k]);
      }
#pragma unroll
      for (int k = 0; k < kStep; ++k) pm[k] = fmaxf(pm[k], __shfl_xor_sync(kFull, pm[k], 1));
#pragma unroll
      for (int k = 0; k < kStep; ++k) pm[k] = fmaxf(pm[k], __shfl_xor_sync(kFull, pm[k], 2));
      float mn = m, mon = mo;
#pragma unroll
      for (int k = 0; k < kStep; ++k) {
        mn = fmaxf(mn, pm[k]);
        mon = fmaxf(mon, pm[k] + ev[k]);
      }
      const float mz = mn == -INFINITY ? 0.0f : mn;
      const float alpha = ex2(m - mz);
      float part = 0.0f;  // of l
      const float beta = mo == mon ? 1.0f : ex2(mo - mon);
      if (kRounded || __any_sync(kFull, beta != 1.0f)) {
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[k][e] = kRounded ? 0.0f : o[k][e] * beta;
      }
      m = mn;
      mo = mon;
#pragma unroll
      for (int k = 0; k < kStep; ++k) {
        // (a page that the slot does not see has no say, even with an infinite or NaN scale)
        const float fac = pm[k] == -INFINITY ? 0.0f : ex2(fminf(mz - mon + ev[k], 120.0f)) * fr[k];
        uint32_t pa[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float a = ex2(s[k][n][0] - mz), b = ex2(s[k][n][1] - mz);
          part += a + b;
          split_pair(a * fac, b * fac, pa[n * 2], pa[n * 2 + 1]);
        }
        const uint8_t* vb = base + k * 2 * R::kBlock + R::kBlock;
        uint32_t vw[4][NT / 4];  // positions 2t, 2t + 1, 2t + 8, 2t + 9, dims NT * g ...
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint8_t* src = vb + R::v_at(2 * t + (e & 1) + (e >> 1) * 8, NT * g);
          if (NT == 16) {
            const uint4 u = *reinterpret_cast<const uint4*>(src);
            vw[e][0] = u.x;
            vw[e][1] = u.y;
            vw[e][NT / 4 - 2] = u.z;
            vw[e][NT / 4 - 1] = u.w;
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(src);
            vw[e][0] = u.x;
            vw[e][1] = u.y;
          }
        }
#pragma unroll
        for (int q = 0; q < NT / 4; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = vw[e][q] ^ 0x80808080u;
          const uint32_t a01 = __byte_perm(w[0], w[1], 0x5140), a23 = __byte_perm(w[0], w[1], 0x7362);
          const uint32_t b01 = __byte_perm(w[2], w[3], 0x5140), b23 = __byte_perm(w[2], w[3], 0x7362);
          mma16816(o[q * 4 + 0], pa, half2_of(a01, 0x4140), half2_of(b01, 0x4140));
          mma16816(o[q * 4 + 1], pa, half2_of(a01, 0x4342), half2_of(b01, 0x4342));
          mma16816(o[q * 4 + 2], pa, half2_of(a23, 0x4140), half2_of(b23, 0x4140));
          mma16816(o[q * 4 + 3], pa, half2_of(a23, 0x4342), half2_of(b23, 0x4342));
        }
      }
      {
        const float add = fmaf(lost, -alpha, part), before = l * alpha;
        l = before + add;
        lost = (l - before) - add;
      }
      __syncwarp();  // every lane has read these pages
      issue(i + kStages);
      if constexpr (kRounded) {
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) sum[k][e] = fmaf(sum[k][e], beta, fmaf(o[k][e + 2], 1.0f / kSplitLoScale, o[k][e]));
      }
    }
    // join the warps, then the splits of the cluster, in their order
    l += __shfl_xor_sync(kFull, l, 1);
    l += __shfl_xor_sync(kFull, l, 2);
    if (l != l) m = INFINITY;  // a NaN score: the joins below then give NaN
    const float back = m == -INFINITY || mo == -INFINITY ? 0.0f : ex2(mo - m);
    cp_async_wait<0>();
    __syncthreads();
    if (on) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < NT; k += 4) {
          auto all = [&](int i) {
            if constexpr (kRounded) return sum[i][e] * back;
            else return (o[i][e] + o[i][e + 2] * (1.0f / kSplitLoScale)) * back;
          };
          const float4 v = make_float4(all(k), all(k + 1), all(k + 2), all(k + 3));
          *reinterpret_cast<float4*>(&s_o[warp][g][NT * (2 * t + e) + k]) = v;
        }
      if (t == 0) {
        s_m[warp][g] = m;
        s_l[warp][g] = l;
      }
    }
    __syncthreads();
    auto write = [&](int s, int e, float mx, float ll, float sum) {
      const size_t orow = row0 + s / nh;
      const int head = h0 + s % nh;
      const float v = mx == -INFINITY ? 0.0f : __fdiv_rn(sum, ll);
      T* op = static_cast<T*>(d.out) + orow * d.ldo + (size_t)head * HD + e;
      if constexpr (sizeof(T) == 4) *op = v;
      else *op = T(v);
      if (e == 0 && d.lse)
        d.lse[orow * d.heads + head] = mx == -INFINITY ? -INFINITY : (mx + log2f(ll)) * 0.6931471805599453f;
    };
    for (int i = tid; i < nslots * HD; i += NW * 32) {
      const int s = i / HD, e = i % HD;
      float mx = s_m[0][s];
#pragma unroll
      for (int w = 1; w < NW; ++w) mx = fmaxf(mx, s_m[w][s]);
      float sum = 0.0f, ll = 0.0f;
      if (mx > -INFINITY) {
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float k = ex2(s_m[w][s] - mx);
          sum += s_o[w][s][e] * k;
          ll += s_l[w][s] * k;
        }
      }
      if (nsplit == 1) {
        write(s, e, mx, ll, sum);
      } else {
        s_po[s][e] = sum;
        if (e == 0) {
          s_pm[s] = mx;
          s_pl[s] = ll;
        }
      }
    }
    if (nsplit == 1) {
      __syncthreads();
      continue;
    }
    cluster.sync();
    for (int i = tid + split * NW * 32; i < nslots * HD; i += nsplit * NW * 32) {
      const int s = i / HD, e = i % HD;
      float mx = -INFINITY, sum = 0.0f, ll = 0.0f;
      for (int r = 0; r < nsplit; ++r) {
        // one pass: the sums so far are scaled down when a larger maximum comes
        const float rm = *cluster.map_shared_rank(&s_pm[s], r), ro = *cluster.map_shared_rank(&s_po[s][e], r),
                    rl = *cluster.map_shared_rank(&s_pl[s], r);
        const float mn = fmaxf(mx, rm);
        if (mn == -INFINITY) continue;
        const float a = ex2(mx - mn), b = ex2(rm - mn);
        sum = sum * a + ro * b;
        ll = ll * a + rl * b;
        mx = mn;
      }
      write(s, e, mx, ll, sum);
    }
    cluster.sync();  // no CTA goes on while its sums are read
  }
}

template <typename T, int HD>
cudaError_t launch_append_t(const Kv8AppendDesc& d, bool single, cudaStream_t st) {
  const int rows = single ? 1 : kQRows<kAppendKeep>;
  const long warps = d.kv_warps + (d.q ? ((long)d.n_rows + rows - 1) / rows * ((d.heads + kQHeads - 1) / kQHeads) : 0);
  const auto kernel = single ? kv8_append_kernel<T, HD, 128 / HD> : kv8_append_kernel<T, HD, kAppendKeep>;
  return launch_k(kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, st, LaunchOpts{true, 1}, d);
}
// NW warps a CTA, a unit's pages split over clusters of ns CTAs (more than 8
// need an opt-in).
template <typename T, int HD, int NW>
cudaError_t launch_attn_w(const Kv8AttnDesc& d, long units, unsigned ns, cudaStream_t st) {
  constexpr int smem = NW * Ring<HD>::kWarp;
  static std::atomic<int> ready[kMaxDevices];
  const cudaError_t set = once_per_device(ready, [] {
    const cudaError_t e =
        cudaFuncSetAttribute(kv8_attn_kernel<T, HD, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(kv8_attn_kernel<T, HD, NW>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (set != cudaSuccess) return set;
  return launch_k(kv8_attn_kernel<T, HD, NW>, dim3((unsigned)units, ns), dim3(NW * 32), smem, st, LaunchOpts{true, ns},
                  d);
}
template <typename T, int HD>
cudaError_t launch_attn_by(const Kv8AttnDesc& d, long units, int warps, unsigned ns, cudaStream_t st) {
  switch (warps) {
    case 12: return launch_attn_w<T, HD, 12>(d, units, ns, st);
    case 4: return launch_attn_w<T, HD, 4>(d, units, ns, st);
    case 3: return launch_attn_w<T, HD, 3>(d, units, ns, st);
    default: return launch_attn_w<T, HD, 2>(d, units, ns, st);
  }
}
// clusters of such a launch that fit the device at once
template <typename T, int HD>
long attn_clusters(const Kv8AttnDesc& d, long units, int warps, unsigned ns, cudaStream_t st) {
  g_occ_query = true;
  g_occ_clusters = 0;
  const cudaError_t e = launch_attn_by<T, HD>(d, units, warps, ns, st);
  g_occ_query = false;
  return e == cudaSuccess ? g_occ_clusters : 0;
}
template <typename T, int HD>
cudaError_t launch_attn_t(const Kv8AttnDesc& d, long units, int pages, int sms, cudaStream_t st) {
  // CTAs that fit the device at once (12 warps an SM), of the fewest steps a
  // warp, a cluster of n counting like 0.4 + 0.1 n steps and a warp like 0.05:
  // 512 units of 19 pages take 15.0 us with 3 warps, 17.4 with 2, 20.1 with 4
  // (two waves); 128 units of 63 pages 16.5 us with 12 warps, 21.2 as 6 x 2; 256
  // of 63 pages 21.6 us as 2 x 3, 23.6 with 4; 8 of 2001 pages 29 us as 10 x 12.
  // Clusters of more than 8 have to fit the GPU's processing clusters (16 x 12
  // warps: two waves, 42 us).
  int best_w = 0;
  unsigned best_n = 1;
  double best = 1e30;
  for (const int w : {12, 4, 3, 2})
    for (unsigned n = 1; n <= 16 && units * n <= (long)(12 / w) * sms && (n == 1 || (int)n * w <= pages); ++n) {
      const int each = (pages + (int)n * w - 1) / ((int)n * w);
      const double t = (each + kStep - 1) / kStep + (n > 1 ? 0.4 + 0.1 * n : 0.0) + 0.05 * w;
      if (t >= best || (n > 8 && attn_clusters<T, HD>(d, units, w, n, st) < units)) continue;
      best = t;
      best_w = w;
      best_n = n;
    }
  // More units than that: small CTAs where a unit is short (2048 units of 19
  // pages: 48 us with 2 warps, 58 with 4; of 192 pages: 326 and 296).
  if (best_w == 0) best_w = pages <= 32 ? 2 : 4;
  return launch_attn_by<T, HD>(d, units, best_w, best_n, st);
}

}  // namespace

cudaError_t launch_kv8_append(Kv8AppendDesc d, int dtype, int sms, cudaStream_t st) {
  // A warp per row, head and K / V up to 64 warps an SM, of which 24 are there at
  // once; above that a warp looks at 2 to 16 rows, which hold one block of a long
  // prompt or as many of single tokens.  Each side as measured, f32, in us with a
  // border of 24, 64 and 200 warps: 1024 tokens 15.2, 13.6, 15.8; 2048 32.0, 26.6,
  // 28.7; 4096 58.4, 48.2, 50.3; a chunk of 1000 rows 15.4, 16.7, 18.6.
  d.chunk = 1;
  auto kv_warps = [&] { return ((long)d.n_rows + d.chunk - 1) / d.chunk * 2 * d.c.kv_heads; };
  while (d.chunk < kKv8Page && kv_warps() > (long)sms * 64) d.chunk *= 2;
  d.kv_warps = kv_warps();
  // Single tokens or chunks?  The host sees neither seq nor pos, and takes fewer
  // rows than twice the cache's sequences for single tokens.  Right: 512 tokens f32
  // 8.1 us, 10.9 in the kernel of chunks; 16 chunks of 611 bf16 rows 60 us, 72 in
  // that of single tokens (tables of random angles).  Where the guess is wrong,
  // both kernels are right and one is slower by such a share: a chunk of 1000 bf16
  // rows in a cache of 512 sequences 14.8 us (13.5), 2 rows each of 2500
  // sequences, f32, 62 us (49).
  const bool single = d.n_rows < 2l * d.c.n_seqs;
  const bool w = d.c.head_dim == 128;
  switch (dtype) {
    case DT_F16: return w ? launch_append_t<__half, 128>(d, single, st) : launch_append_t<__half, 64>(d, single, st);
    case DT_BF16:
      return w ? launch_append_t<__nv_bfloat16, 128>(d, single, st) : launch_append_t<__nv_bfloat16, 64>(d, single, st);
    default: return w ? launch_append_t<float, 128>(d, single, st) : launch_append_t<float, 64>(d, single, st);
  }
}

cudaError_t launch_kv8_attention(Kv8AttnDesc d, int dtype, int max_rows, int max_len, int sms, cudaStream_t st) {
  const int group = d.heads / d.c.kv_heads;
  d.unit_heads = std::min(group, kSlots);
  d.head_chunks = (group + d.unit_heads - 1) / d.unit_heads;
  d.group_rows = std::max(1, std::min(max_rows, kSlots / d.unit_heads));
  const long units = ((long)d.n_rows + d.group_rows - 1) / d.group_rows * d.c.kv_heads * d.head_chunks;
  // what a unit of `rows` rows sees: the mean of a causal chunk, or its window
  auto seen = [&](int rows) {
    const long mean = std::max(1l, (long)max_len - max_rows / 2);
    return d.window > 0 ? std::min(mean, (long)d.window + rows - 1) : mean;
  };
  // Units of 8 slots here, or tiles of 128 (kv8_tile.cu)?  Both as measured, in
  // us: a unit costs 0.0085 and 0.0009 a page (of 128 dims) over 7; a CTA of
  // tiles 10 and 2.2 a tile over 4 (10 with splits), one an SM at a time.  Here and
  // in tiles, bf16 (f32), 16 heads, 8 K/V heads of 128: one sequence's 100 rows over
  // 100 positions 10.4 and 15.0 (10.6 and 16.5); 8 such 25.7 and 15.5 (26 and 17);
  // 2 of 300 over 300 30 and 22 (31 and 26); 4 of 64 rows over 4000 104 and 45
  // (112 and 58); 200 rows over 8000 147 and 64 (163 and 92); 16 of 4 over 2000 22
  // and 51 (23 and 74); 64 of 8 over 500 46 and 75 (49 and 94); 16 rows over 1000
  // 11.6 and 17.6 (11.2 and 20.4); 500 rows of 16 heads of 64, window 72: 14.9 and
  // 15.7 (14.8 and 17.6).
  if (max_rows > 1) {
    const double here = 7.0 + units * (0.0085 + 0.0009 * d.c.head_dim / 128 * ((seen(d.group_rows) + kKv8Page - 1) / kKv8Page));
    Kv8AttnDesc t = d;
    const TilePlan plan = plan_kv8_tile(t, dtype, max_rows, max_len, sms);
    const long tiles = (seen(t.group_rows) + 127) / 128, waves = (plan.units * plan.splits + sms - 1) / sms;
    if ((plan.splits > 1 ? 10.0 : 4.0) + waves * (10.0 + 2.2 * t.halves * ((tiles + plan.splits - 1) / plan.splits)) < here)
      return launch_kv8_tile(t, plan, dtype, st);
  }
  const int pages = (max_len + kKv8Page - 1) / kKv8Page;
  const bool w = d.c.head_dim == 128;
  switch (dtype) {
    case DT_F16:
      return w ? launch_attn_t<__half, 128>(d, units, pages, sms, st) : launch_attn_t<__half, 64>(d, units, pages, sms, st);
    case DT_BF16:
      return w ? launch_attn_t<__nv_bfloat16, 128>(d, units, pages, sms, st)
               : launch_attn_t<__nv_bfloat16, 64>(d, units, pages, sms, st);
    default:
      return w ? launch_attn_t<float, 128>(d, units, pages, sms, st) : launch_attn_t<float, 64>(d, units, pages, sms, st);
  }
}

// ---- host side of the entry points ----------------------------------------------

namespace {
thread_local unsigned g_wait_ns = kKv8WaitNs;
}

OnDeviceOf::OnDeviceOf(const void* p) {
  cudaPointerAttributes a;
  cudaError_t e = cudaPointerGetAttributes(&a, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    code = e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver ? QTTS_ERR_NODEV : QTTS_ERR_CUDA;
    err = cudaGetErrorString(e);
    return;
  }
  if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
    code = QTTS_ERR_BADARG;
    err = "not a device pointer";
    return;
  }
  int cur = -1;
  if (cudaGetDevice(&cur) != cudaSuccess || (cur != a.device && cudaSetDevice(a.device) != cudaSuccess)) {
    cudaGetLastError();
    code = QTTS_ERR_CUDA;
    err = "the device of the buffers cannot be made current";
    return;
  }
  if (cur != a.device) prev_ = cur;
  static std::atomic<int> sms[kMaxDevices];
  int n = a.device >= 0 && a.device < kMaxDevices ? sms[a.device].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, a.device) != cudaSuccess || n <= 0) n = 148;
    if (a.device >= 0 && a.device < kMaxDevices) sms[a.device].store(n, std::memory_order_relaxed);
  }
  sm_count = n;
}
OnDeviceOf::~OnDeviceOf() {
  if (prev_ >= 0) cudaSetDevice(prev_);
}

namespace {

// nullptr, or what is wrong with the cache description
const char* cache_fault(const qtts_kv8_cache* c) {
  if (!c || !c->codes || !c->scales || !c->page_table) return "the cache has a null pointer";
  if (c->head_dim != 64 && c->head_dim != 128) return "the cache's head_dim is not 64 or 128";
  if (c->kv_heads <= 0 || c->kv_heads > 1024) return "the cache's kv_heads is not 1..1024";
  if (c->n_pages <= 0 || c->n_seqs <= 0 || c->pages_per_seq <= 0) return "the cache has no pages or sequences";
  if (c->pages_per_seq > INT32_MAX / kKv8Page) return "a sequence's positions pass 2^31";
  if (c->page_stride < 2ll * c->kv_heads * kKv8Page * c->head_dim || c->page_stride % 16)
    return "page_stride is less than a page or not a multiple of 16";
  if (c->scale_stride < 2ll * c->kv_heads) return "scale_stride is less than a page's scales";
  if (!aligned(c->codes, 16) || !aligned(c->scales, 4) || !aligned(c->page_table, 4)) return "the cache is misaligned";
  return nullptr;
}
// rows of `cols` elements: four-element loads
const char* rows_fault(const void* p, int64_t ld, int64_t cols, int dtype) {
  if (!p) return "a null pointer";
  if (ld < cols || ld % 4) return "a row stride that is less than a row or not a multiple of 4";
  if (!aligned(p, 4 * dtype_bytes(dtype))) return "a misaligned pointer";
  return nullptr;
}
int refuse(const char* what, const char* why) { return fail(QTTS_ERR_BADARG, std::string(what) + ": " + why); }
int launched(cudaError_t e) {
  if (e == cudaSuccess) return QTTS_OK;
  cudaGetLastError();
  return fail(QTTS_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace
}  // namespace qtts

using namespace qtts;

extern "C" {

int qtts_kv8_append_dev(const qtts_kv8_cache* cache, const void* k, int64_t ldk, const void* v, int64_t ldv,
                        const void* q, int64_t ldq, void* q_out, int64_t ldqo, int heads, int dtype,
                        const uint16_t* q_norm, const uint16_t* k_norm, const float* rope_cos, const float* rope_sin,
                        int rope_rows, const int32_t* seq, const int32_t* pos, const int32_t* rope_pos, int n_rows,
                        int32_t* flags, void* stream) try {
  const char* f = cache_fault(cache);
  if (f) return refuse("kv8 append", f);
  if (dtype != QTTS_F32 && dtype != QTTS_F16 && dtype != QTTS_BF16) return refuse("kv8 append", "unknown dtype");
  if (n_rows < 0 || (n_rows > 0 && (!seq || !pos))) return refuse("kv8 append", "bad rows");
  const int64_t kv_cols = (int64_t)cache->kv_heads * cache->head_dim;
  if (n_rows > 0) {
    if ((f = rows_fault(k, ldk, kv_cols, dtype)) || (f = rows_fault(v, ldv, kv_cols, dtype))) return refuse("kv8 append, k or v", f);
    if (!q != !q_out) return refuse("kv8 append", "q and q_out go together");
    if (q) {
      if (heads <= 0 || heads > 16384) return refuse("kv8 append", "bad heads");
      const int64_t cols = (int64_t)heads * cache->head_dim;
      if ((f = rows_fault(q, ldq, cols, dtype)) || (f = rows_fault(q_out, ldqo, cols, dtype))) return refuse("kv8 append, q", f);
    }
  }
  if (!rope_cos != !rope_sin || (rope_cos && rope_rows <= 0)) return refuse("kv8 append", "bad rotation tables");
  if (!words_aligned({seq, pos, rope_pos, flags})) return refuse("kv8 append", "misaligned seq, pos, rope_pos or flags");
  if (!aligned(rope_cos, 16) || !aligned(rope_sin, 16) || !aligned(q_norm, 8) || !aligned(k_norm, 8))
    return refuse("kv8 append", "misaligned rotation tables or norm weights");
  if (n_rows == 0) return QTTS_OK;
  OnDeviceOf on(cache->codes);
  if (on.err) return fail(on.code, std::string("kv8 append, the cache: ") + on.err);
  Kv8AppendDesc d;
  d.c = *cache;
  d.q = q;
  d.k = k;
  d.v = v;
  d.q_out = q_out;
  d.ldq = ldq;
  d.ldk = ldk;
  d.ldv = ldv;
  d.ldqo = ldqo;
  d.heads = q ? heads : 0;
  d.q_norm = reinterpret_cast<const __half*>(q_norm);
  d.k_norm = reinterpret_cast<const __half*>(k_norm);
  d.rope_cos = rope_cos;
  d.rope_sin = rope_sin;
  d.rope_rows = rope_rows;
  d.seq = seq;
  d.pos = pos;
  d.rope_pos = rope_pos;
  d.n_rows = n_rows;
  d.flags = flags;
  return launched(launch_kv8_append(d, dtype, on.sm_count, (cudaStream_t)stream));
} catch (...) {
  return QTTS_ERR_OOM;
}

int qtts_kv8_attention_dev(const qtts_kv8_cache* cache, const void* q, int64_t ldq, int heads, int dtype, float scale,
                           int window, const int32_t* seq, const int32_t* pos, int n_rows, int max_rows, int max_len,
                           void* out, int64_t ldo, float* lse, int32_t* flags, void* stream) try {
  const char* f = cache_fault(cache);
  if (f) return refuse("kv8 attention", f);
  if (dtype != QTTS_F32 && dtype != QTTS_F16 && dtype != QTTS_BF16) return refuse("kv8 attention", "unknown dtype");
  if (heads <= 0 || heads % cache->kv_heads || heads > 16384)
    return refuse("kv8 attention", "heads is not a multiple of the cache's kv_heads (up to 16384)");
  if (window < 0 || max_rows < 0 || max_len < 0) return refuse("kv8 attention", "negative window, max_rows or max_len");
  if (n_rows < 0 || (n_rows > 0 && (!seq || !pos))) return refuse("kv8 attention", "bad rows");
  if (!words_aligned({seq, pos, lse, flags})) return refuse("kv8 attention", "misaligned seq, pos, lse or flags");
  if (n_rows == 0) return QTTS_OK;
  const int64_t cols = (int64_t)heads * cache->head_dim;
  if ((f = rows_fault(q, ldq, cols, dtype)) || (f = rows_fault(out, ldo, cols, dtype))) return refuse("kv8 attention, q or out", f);
  if ((int64_t)n_rows * heads > INT32_MAX) return fail(QTTS_ERR_RANGE, "kv8 attention: n_rows * heads passes 2^31");
  OnDeviceOf on(cache->codes);
  if (on.err) return fail(on.code, std::string("kv8 attention, the cache: ") + on.err);
  Kv8AttnDesc d;
  d.c = *cache;
  d.q = q;
  d.out = out;
  d.lse = lse;
  d.ldq = ldq;
  d.ldo = ldo;
  d.heads = heads;
  d.scale = scale;
  d.window = window;
  d.seq = seq;
  d.pos = pos;
  d.n_rows = n_rows;
  d.flags = flags;
  d.wait_ns = g_wait_ns;
  const int cap = cache->pages_per_seq * kKv8Page;
  int len = max_len == 0 ? cap : std::min(max_len, cap);
  max_rows = std::max(1, std::min(max_rows, n_rows));
  if (window > 0) len = (int)std::min<int64_t>(len, (int64_t)window + max_rows - 1);
  return launched(launch_kv8_attention(d, dtype, max_rows, len, on.sm_count, (cudaStream_t)stream));
} catch (...) {
  return QTTS_ERR_OOM;
}

int qtts_kv8_wait_limit(int64_t ns) {
  if (ns < 0 || ns > 2000000000ll) return refuse("kv8 wait limit", "not 0 .. 2e9 ns");
  g_wait_ns = (unsigned)ns;
  return QTTS_OK;
}

}  // extern "C"
