// kv8_tile.cu -- attention of many rows over the 8-bit paged cache (sm_100a):
// chunks of a prompt, or every frame of an utterance.
//
// A CTA takes one or two halves of 128 slots (query heads of consecutive rows
// that share a K/V head) and walks over the cache in tiles of 128 positions:
//   S = Q K^T     tcgen05.mma, Q and K in shared memory, S (f32) in TMEM
//   P = softmax   a thread per slot reads its row of S, keeps the running
//                 maximum and sum, and writes P as f16 over S
//   O += P V      tcgen05.mma, P from TMEM, V in shared memory, O in TMEM
// Four warps a half do the softmax, four turn codes into f16 operands (exact: a
// code has 8 bits), two tiles ahead at most, and one issues the products in an
// order that keeps the halves half a tile apart: those of one run while the
// other is in its softmax.  (A warp a half let them fall into step: 183 instead
// of 161 us for four chunks of 1000 rows.)  The next codes to convert are on their way to shared memory
// meanwhile (asynchronous copies; held in registers instead, they were spilled,
// and a tile took 8000 cycles, of which the conversion waited 4500 for them).
//
// Queries are scaled by a power of two that puts the largest element of a head
// between 1 and 2.  f16 then holds those of 16-bit types but for what lies far
// below it: below 2^-14 they are rounded to steps of 2^-24, so that none is off
// by more than 2^-25.  f32 queries are split into f16 hi + lo, and so is P then
// (rounding to 2^-25 of the largest), two products each; the two operands of a
// split query take the room of two halves, so that f32 has one half.
//
// P of 16-bit rows is f16 without a lo part: each weight is off by up to 2^-11,
// and the sum l that divides them is of the unrounded ones.  Measured against 64
// bits (2-norms; "rounded" are the exact values rounded once to the type): four
// chunks of 1000 bf16 rows over up to 3001 1.662e-3, rounded 1.659e-3; f16
// 2.32e-4, rounded 2.08e-4; f16 with a window of 100 2.91e-4.  A lo part would
// take its place in S's columns, but costs the softmax, which bounds the kernel,
// five more instructions for two weights and the products twice the time.
// The V scales are folded into P, relative to a running exponent of their own,
// so that P stays within f16 whatever the scales are; O is rescaled only when
// that exponent has grown by 6 (P then reaches 2^13).
//
// Four chunks of 1000 bf16 rows over up to 3001 positions (16 heads, 8 K/V heads
// of 128): 157 us, 49 GFLOP at 314 TFLOP/s.  A half's chain bounds it: a tile
// takes 6000 cycles, 3700 for the softmax and the rest for the products before
// and after it, while the exponentials' pipe is 27% and the tensor pipe 24% busy.
// f32 has twice the products and one half (four chunks of 64 rows over 4000: 44
// us in bf16, 56 in f32; the four chunks of 1000 rows: 295 us).
//
// A tile of rows may span sequences: its segments (runs of rows of one
// sequence) are taken one after the other, with the other slots masked.
#include <cooperative_groups.h>
#include <float.h>

#include <algorithm>

#include "common.cuh"
#include "engine.h"
#include "kv8.cuh"
#include "kv8_order.h"

namespace cg = cooperative_groups;

namespace qtts {

namespace {

constexpr int kTileM = 128, kTilePos = 128, kTilePages = kTilePos / kKv8Page;
constexpr int kSoft = 256, kConvert = 128;  // threads of the softmax (two halves) and of the conversion
constexpr int kTileThreads = kSoft + kConvert + 32;  // and a warp that issues the products
// Half h: S and P at 256 h, O at 256 h + 128.  With f32 rows, which have one
// half: O of tile n at 128 + 256 (n & 1), the sums of all tiles at kSums.
constexpr uint32_t kTmemCols = 512, kSums = 256;
constexpr float kNoPage = 4.0f;  // no fraction of a scale (split_scale)
constexpr int kScales = 4;  // tiles of scales kept: a half may be two tiles behind the conversion

struct TileSegment {
  int row0, rows, seq, lo, hi;  // rows of the unit, and the positions [lo, hi) that any of them sees
};
struct TileShared {
  uint64_t k_full[2], k_free[2], v_full[2], v_free[2];  // by buffer
  uint64_t s_full[2], p_full[2];                        // by half
  uint64_t o_full[2];  // by half; f32: by O's buffer (kv8_order.h)
  uint64_t o_free[2];  // f32: by O's buffer
  uint64_t summed;     // f32: once a segment
  uint64_t q_full, fin;
  uint32_t tmem;
  int over;  // a wait of the CTA has run out: nobody waits any longer
  int row0, rows, h0, nh;  // the unit, for mark_rows
  int n_segments;
  int seq[2 * kTileM], pos[2 * kTileM];
  TileSegment segment[2 * kTileM];
  // K scale, exponent and fraction of the V scale (kNoPage: none), and log2 of the
  // V scale; NaN keeps a page from the short way (Softmax::tile_short)
  float4 scale[kScales][kTilePages];
  float m[2 * kTileM], l[2 * kTileM];
  float mo[4][kTileM];  // f32: the exponent of O of the last tiles
};

template <typename T, int HD>
struct TileCfg {
  static constexpr bool kSplit = sizeof(T) == 4;
  static constexpr int kHalf = kTileM * HD * 2;  // bytes of a 128-row f16 operand
  // Q (two halves, or hi and lo), two of K and V, and the raw codes of one
  static constexpr int kQ = 0, kK = 2 * kHalf, kV = kK + 2 * kHalf, kRaw = kV + 2 * kHalf, kOps = kRaw + kHalf / 2;
  static_assert(kTileM * HD * 4 * (kSplit ? 1 : 2) <= 4 * kHalf, "the halves' sums lie over K and V");
  static constexpr int kUsed = kOps + (int)sizeof(TileShared);
  // One CTA an SM, as it takes all of TMEM (a second would wait for it, and its
  // cluster for the second).
  static constexpr int kSmem = kUsed > 120 * 1024 ? kUsed : 120 * 1024;
};

// Operands have no swizzle, 16-byte core-matrix rows.  Q and K (K-major): row r,
// 8-dim chunk c at (r/8) * 16 HD + c * 128 + (r%8) * 16.  V (MN-major): position
// p, 8-dim group g at g * 2048 + (p/8) * 128 + (p%8) * 16.  In both the leading
// offset is 128 bytes and a 16-deep step advances the start by 256.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t stride) {
  return ((addr >> 4) & 0x3FFFu) | ((uint64_t)(128u >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) | (1ull << 46);
}
// kind::f16, D f32, A and B f16, A K-major
__host__ __device__ constexpr uint32_t instruction(int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void commit_to(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_of(bar))
               : "memory");
}
__device__ __forceinline__ void bar_init(uint64_t* bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_of(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_of(bar)) : "memory");
}
// Waits for the phase, at most `ns` (less than the 4.3 s of the clock's low word)
// or until another thread has given up.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, unsigned parity, int* over, unsigned ns) {
  const uint32_t a = smem_of(bar);
  unsigned t0 = 0;
  for (unsigned it = 0;; ++it) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return true;
    if ((it & 255u) == 255u) {
      if (*reinterpret_cast<volatile int*>(over)) return false;
      unsigned t;
      asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
      if (it == 255u) t0 = t;
      else if (t - t0 > ns) {
        *reinterpret_cast<volatile int*>(over) = 1;
        return false;
      }
    }
  }
}
// 32 columns on their way into r, which may be read after tmem_wait(r).
__device__ __forceinline__ void tmem_start(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&q)[32], float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(q[0]), "+r"(q[1]), "+r"(q[2]), "+r"(q[3]), "+r"(q[4]), "+r"(q[5]), "+r"(q[6]), "+r"(q[7]),
                 "+r"(q[8]), "+r"(q[9]), "+r"(q[10]), "+r"(q[11]), "+r"(q[12]), "+r"(q[13]), "+r"(q[14]), "+r"(q[15]),
                 "+r"(q[16]), "+r"(q[17]), "+r"(q[18]), "+r"(q[19]), "+r"(q[20]), "+r"(q[21]), "+r"(q[22]), "+r"(q[23]),
                 "+r"(q[24]), "+r"(q[25]), "+r"(q[26]), "+r"(q[27]), "+r"(q[28]), "+r"(q[29]), "+r"(q[30]), "+r"(q[31])
               :
               : "memory");
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(q[j]);
}
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  tmem_start(addr, r);
  tmem_wait(r, v);
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void smem_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void store16(uint8_t* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  *reinterpret_cast<uint4*>(p) = make_uint4(a, b, c, d);
}
// plain f16 hi + lo (lo unscaled: the values are at most 128)
__device__ __forceinline__ uint32_t pack_half(float a, float b) { return half2_bits(__floats2half2_rn(a, b)); }
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_half(a - h.x, b - h.y);
}

// What the parts of a CTA share: its place in the work and its operands.
template <typename T, int HD>
struct TileJob {
  using C = TileCfg<T, HD>;
  const Kv8AttnDesc& d;
  TileShared& sh;
  uint8_t* ops;
  int row0, rows, kvh, h0, nh, nsplit, split, halves;
  uint32_t tmem;

  __device__ __forceinline__ void tiles(const TileSegment& g, int& p0, int& p1, int& t0, int& t1) const {
    p0 = g.lo / kKv8Page;
    p1 = (g.hi + kKv8Page - 1) / kKv8Page;
    const int nt = g.hi > 0 && g.seq >= 0 ? (p1 - p0 + kTilePages - 1) / kTilePages : 0;
    const int share = (nt + nsplit - 1) / nsplit;
    t0 = min(nt, split * share);
    t1 = min(nt, t0 + share);
  }
  // for a warp as one, so that it stays together
  __device__ __forceinline__ bool wait(uint64_t* bar, unsigned parity) const {
    return __all_sync(kFull, bar_wait(bar, parity, &sh.over, d.wait_ns));
  }
  // whether half h holds rows of the segment
  __device__ __forceinline__ bool takes(const TileSegment& g, int h) const {
    return h < halves && g.row0 * nh < (h + 1) * kTileM && (g.row0 + g.rows) * nh > h * kTileM;
  }
};

// ---- codes to operands -----------------------------------------------------------
template <typename T, int HD>
struct Converter {
  using J = TileJob<T, HD>;
  static constexpr int N = HD / 16;  // 16-byte pieces of a thread, per operand
  const J& job;
  const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  uint4* raw;  // this thread's pieces at raw[i * kConvert]
  float sk = 0.0f, sv = 0.0f;

  __device__ explicit Converter(const J& j)
      : job(j), raw(reinterpret_cast<uint4*>(j.ops + J::C::kRaw) + (threadIdx.x & (kConvert - 1))) {}
  // piece i: positions 8 at a time, dims 16 at a time
  __device__ __forceinline__ int block_of(int i) const { return HD == 128 ? warp + 4 * (i >> 1) : warp + 4 * i; }
  __device__ __forceinline__ int chunk_of(int i) const { return HD == 128 ? (lane >> 3) + 4 * (i & 1) : lane >> 3; }

  __device__ __forceinline__ int pages(const int* table, int p0, int p1, int tile) {
    const qtts_kv8_cache& c = job.d.c;
    const int pg = p0 + tile * kTilePages + lane;
    int id = -1;
    if (lane < kTilePages && pg < p1) {
      id = table[pg];
      if (id < 0 || id >= c.n_pages) {
        raise(job.d.flags, QTTS_KV8_BAD_PAGE);
        id = -1;
      }
    }
    return id;
  }
  // starts the copies of K or V of the tile whose pages lanes 0..7 hold in `ids`
  // (zeros for a missing one); the pieces there have been read
  __device__ __forceinline__ void fetch(int which, int ids) const {
    const qtts_kv8_cache& c = job.d.c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int b = block_of(i), page = __shfl_sync(kFull, ids, b >> 1);
      const int8_t* src = block_codes(c, max(page, 0), which, job.kvh) + ((b & 1) * 8 + (lane & 7)) * HD + chunk_of(i) * 16;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_of(raw + i * kConvert)),
                   "l"(src), "r"(page >= 0 ? 16 : 0)
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void fetch_scales(int ids) {
    sk = sv = 0.0f;
    if (ids >= 0) {
      sk = *block_scale(job.d.c, ids, 0, job.kvh);
      sv = *block_scale(job.d.c, ids, 1, job.kvh);
    }
  }
  __device__ __forceinline__ void put(uint8_t* p, int next, uint4 u) const {  // 16 dims: two core-matrix rows
    const uint2 a = halves_of(u.x), b = halves_of(u.y), c = halves_of(u.z), d = halves_of(u.w);
    store16(p, a.x, a.y, b.x, b.y);
    store16(p + next, c.x, c.y, d.x, d.y);
  }
  __device__ __forceinline__ void put_k(int b) const {
    uint8_t* base = job.ops + J::C::kK + b * J::C::kHalf;
#pragma unroll
    for (int i = 0; i < N; ++i)
      put(base + block_of(i) * (16 * HD) + chunk_of(i) * 256 + (lane & 7) * 16, 128, raw[i * kConvert]);
  }
  __device__ __forceinline__ void put_v(int b) const {
    uint8_t* base = job.ops + J::C::kV + b * J::C::kHalf;
#pragma unroll
    for (int i = 0; i < N; ++i)
      put(base + chunk_of(i) * 4096 + block_of(i) * 128 + (lane & 7) * 16, 2048, raw[i * kConvert]);
  }
  // One segment; `it` counts the CTA's tiles.
  __device__ bool run(const TileSegment& g, int& it) {
    TileShared& sh = job.sh;
    int p0, p1, t0, t1;
    job.tiles(g, p0, p1, t0, t1);
    if (t0 == t1) return true;
    const int* table = job.d.c.page_table + (size_t)g.seq * job.d.c.pages_per_seq;
    int ids = pages(table, p0, p1, t0), next = pages(table, p0, p1, t0 + 1);
    fetch(0, ids);
    fetch_scales(ids);
    for (int t = t0; t < t1; ++t, ++it) {
      const int b = it & 1;
      const unsigned before = (unsigned)((it >> 1) - 1) & 1u;  // the buffers' last use
      const int after = pages(table, p0, p1, t + 2);
      if (it > 1 && !job.wait(&sh.k_free[b], before)) return false;
      if (warp == 0 && lane < kTilePages) {
        float ev, fr;
        split_scale(sv, ev, fr);
        const bool plain = ids >= 0 && sk >= 0.0f && sv >= FLT_MIN && sv <= FLT_MAX;
        sh.scale[it % kScales][lane] = make_float4(sk, ev, ids >= 0 ? fr : kNoPage, plain ? log2f(sv) : NAN);
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");  // this thread's own copies
      put_k(b);
      smem_to_async();
      bar_arrive(&sh.k_full[b]);
      fetch(1, ids);
      fetch_scales(next);
      if (it > 1 && !job.wait(&sh.v_free[b], before)) return false;
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      put_v(b);
      smem_to_async();
      bar_arrive(&sh.v_full[b]);
      if (t + 1 < t1) fetch(0, next);
      ids = next;
      next = after;
    }
    return true;
  }
};

// ---- the products ------------------------------------------------------------------
template <typename T, int HD>
struct Products {
  using J = TileJob<T, HD>;
  using C = TileCfg<T, HD>;
  const J& job;
  const int lane = threadIdx.x & 31;
  int done[2] = {0, 0};  // tiles of each half

  __device__ explicit Products(const J& j) : job(j) {}
  __device__ __forceinline__ bool wait_for(uint64_t (&bars)[2], TileTurn at) const {
    return job.wait(&bars[at.bar], at.parity);
  }
  // S = Q K^T of half h with K of buffer b; last: no other half reads this K
  __device__ __forceinline__ bool score(int h, int b, bool last) const {
    TileShared& sh = job.sh;
    constexpr uint32_t idesc = instruction(kTilePos, false);
    // P of the half's tile before lies where S goes
    if (done[h] > 0 && !wait_for(sh.o_full, o_full_turn(C::kSplit, h, done[h] - 1))) return false;
    if (lane == 0) {
      const uint32_t q = smem_of(job.ops + C::kQ) + h * C::kHalf, k = smem_of(job.ops + C::kK) + b * C::kHalf;
      const uint32_t s = job.tmem + 256 * h;
      tc_fence_after();
      // lo first: each product's sum is cut off, which is less while it is small
      // (f32 rows over 2714 positions: 1.46e-6 of the result with lo last or
      // between, 6.3e-7 so)
      if (C::kSplit) {
#pragma unroll
        for (int e = 0; e < HD / 16; ++e)
          mma_ss(s, operand(q + C::kHalf + e * 256, 16 * HD), operand(k + e * 256, 16 * HD), idesc, e > 0);
      }
#pragma unroll
      for (int e = 0; e < HD / 16; ++e)
        mma_ss(s, operand(q + e * 256, 16 * HD), operand(k + e * 256, 16 * HD), idesc, C::kSplit || e > 0);
      commit_to(&sh.s_full[h]);
      if (last) commit_to(&sh.k_free[b]);
      // a plain arrival besides the products' own: it passes on what the
      // converters wrote (the scales) to who waits for S
      bar_arrive(&sh.s_full[h]);
    }
    __syncwarp();
    return true;
  }
  // O += P V of half h with V of buffer b; last: no other half reads this V
  __device__ __forceinline__ bool weigh(int h, int b, bool first, bool last) {
    TileShared& sh = job.sh;
    constexpr uint32_t idesc = instruction(HD, true);
    if (!job.wait(&sh.p_full[h], done[h] & 1)) return false;
    const int n = done[h]++;
    // the buffer's tile before has been added up
    if (C::kSplit && n > 1 && !wait_for(sh.o_free, o_free_turn(n - 2))) return false;
    if (lane == 0) {
      const uint32_t v = smem_of(job.ops + C::kV) + b * C::kHalf, s = job.tmem + 256 * h;
      const uint32_t o = s + kTilePos + (C::kSplit ? 256 * (n & 1) : 0);
      uint64_t* full = &sh.o_full[o_full_turn(C::kSplit, h, n).bar];
      tc_fence_after();
      auto columns = [&](int e) { return s + 32 * (e >> 1) + 8 * (e & 1); };
      if (C::kSplit) {
#pragma unroll
        for (int e = 0; e < kTilePos / 16; ++e) mma_ts(o, columns(e) + 16, operand(v + e * 256, 2048), idesc, e > 0);
      }
#pragma unroll
      for (int e = 0; e < kTilePos / 16; ++e)
        mma_ts(o, columns(e), operand(v + e * 256, 2048), idesc, C::kSplit || !first || e > 0);
      commit_to(full);
      if (C::kSplit) bar_arrive(full);  // (passes on sh.mo, as above)
      if (last) commit_to(&sh.v_free[b]);
    }
    __syncwarp();
    return true;
  }
  __device__ bool run(const TileSegment& g, int& it) {
    TileShared& sh = job.sh;
    int p0, p1, t0, t1;
    job.tiles(g, p0, p1, t0, t1);
    const bool one = job.takes(g, 0), two = job.takes(g, 1);
    for (int t = t0; t < t1; ++t, ++it) {
      const int b = it & 1;
      const unsigned use = (unsigned)(it >> 1) & 1u;
      if (!job.wait(&sh.k_full[b], use)) return false;
      if (one && !score(0, b, !two)) return false;
      if (two && t > t0 && !weigh(1, b ^ 1, t - 1 == t0, true)) return false;
      if (two && !score(1, b, true)) return false;
      if (!job.wait(&sh.v_full[b], use)) return false;
      if (one && !weigh(0, b, t == t0, !two)) return false;
    }
    return !two || t0 == t1 || weigh(1, (it - 1) & 1, t1 - 1 == t0, true);
  }
};

// ---- softmax -----------------------------------------------------------------------
// P starts at up to 2^kAbove: the lo of a pair is rounded to 2^-25, which a
// typical weight of a long row, 2^-6 of the largest, would show (f32 rows over
// 2714 positions: 1.58e-6 of the result with P up to 1, 1.46e-6 so).
constexpr float kAbove = 6.0f;
struct Running {
  float m, mo, l;  // largest score, exponent of O, sum of exp2(score - m)
  float lost;      // f32: what roundings added to l
};
// A tile's weights come to l, scaled by alpha.  With f32 rows the rounding of
// each sum is made up for in the next (30000 positions, 235 tiles: the worst row is
// off by 1.5e-6 so, and was by 2.8e-6 with plain sums page by page and by 9e-6
// position by position).
template <bool SPLIT>
__device__ __forceinline__ void add_weights(float alpha, float part, float& l, float& lost) {
  if constexpr (SPLIT) {
    const float add = fmaf(lost, -alpha, part), before = l * alpha;
    l = before + add;
    lost = (l - before) - add;
  } else {
    l = fmaf(l, alpha, part);
  }
}

// The running exponent of O follows max(score + exponent of the V scale); O is
// rescaled when it has grown by 6.  (mo of -inf: nothing is in O yet.)
template <int HD, bool SPLIT>
__device__ __forceinline__ void grow_to(float mon, float& mo, uint32_t o) {
  const bool grow = mon > mo + 2 * kAbove, rescale = grow && mo > -INFINITY;
  if (!SPLIT && __any_sync(kFull, rescale)) {
    const float beta = rescale ? ex2(mo - (mon - kAbove)) : 1.0f;
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
      float x[32];
      tmem_load(o + 32 * c, x);
      uint32_t r[16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(x[16 * h + e] * beta);
        tmem_store16(o + 32 * c + 16 * h, r);
      }
    }
  }
  if (grow || mo == -INFINITY) mo = mon - kAbove;
}

// Any tile: S at columns s (this warp's lanes), of which this slot sees positions
// from .. from + width relative to its first.
template <int HD, bool SPLIT>
__device__ __noinline__ Running tile_long(Running r, uint32_t s, unsigned from, unsigned width, float qs,
                                          const float4* sc) {
  float mn = r.m, mon = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float x[32];
    tmem_load(s + 32 * c, x);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 k = sc[2 * c + q];
      const float f = qs * k.x;
      float pm = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (from + 32 * c + 16 * q + e < width) pm = fmaxf(pm, x[16 * q + e] * f);
      if (k.z != kNoPage) {
        mn = fmaxf(mn, pm);
        mon = fmaxf(mon, pm + k.y);
      }
    }
  }
  grow_to<HD, SPLIT>(mon, r.mo, s + kTilePos);
  const float mz = mn == -INFINITY ? 0.0f : mn;
  const float alpha = ex2(r.m - mz);
  r.m = mn;
  float part = 0.0f;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float x[32];
    tmem_load(s + 32 * c, x);
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 k = sc[2 * c + q];
      const float f = qs * k.x;
      const float fac = r.mo == -INFINITY ? 0.0f : ex2(fminf(mz - r.mo + k.y, 120.0f)) * k.z;
      const unsigned at = k.z != kNoPage ? from + 32 * c + 16 * q : 0x80000000u;  // (no width reaches it)
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float p[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool seen = at + e + j < width;
          const float w = seen ? ex2(fmaf(x[16 * q + e + j], f, -mz)) : 0.0f;
          sum[j] += w;
          p[j] = seen ? w * fac : 0.0f;  // (fac may be infinite or NaN)
        }
        hi[8 * q + e / 2] = pack_half(p[0], p[1]);
        if (SPLIT) lo[8 * q + e / 2] = pack_rest(p[0], p[1], hi[8 * q + e / 2]);
      }
      part += sum[0] + sum[1];
    }
    tmem_store16(s + 32 * c, hi);
    if (SPLIT) tmem_store16(s + 32 * c + 16, lo);
  }
  add_weights<SPLIT>(alpha, part, r.l, r.lost);
  return r;
}

template <typename T, int HD>
struct Softmax {
  using J = TileJob<T, HD>;
  using C = TileCfg<T, HD>;
  const J& job;
  const int half = threadIdx.x >> 7, slot = threadIdx.x, row, head;
  float qs = 0.0f;
  float m, mo, l, lost;
  int see_lo, see_hi;
  int done = 0;  // tiles of this half
  int segments = 0;  // of at least one tile

  __device__ explicit Softmax(const J& j) : job(j), row((int)threadIdx.x / j.nh), head((int)threadIdx.x % j.nh) {}
  __device__ __forceinline__ uint32_t columns() const {
    return job.tmem + 256 * half + ((threadIdx.x & 96u) << 16);
  }

  // The slot's query as the operand's row, scaled by a power of two.
  __device__ void put_query() {
    const bool on = row < job.rows && job.sh.seq[row] >= 0;
    const T* src = static_cast<const T*>(job.d.q) + (size_t)(job.row0 + (on ? row : 0)) * job.d.ldq +
                   (size_t)(job.h0 + head) * HD;
    float big = 0.0f;
    bool finite = true;
    if (on) {
#pragma unroll 16
      for (int c = 0; c < HD / 4; ++c) {
        const float4 x = load4(src + 4 * c);
        const float a = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
        finite &= fabsf(x.x) <= FLT_MAX && fabsf(x.y) <= FLT_MAX && fabsf(x.z) <= FLT_MAX && fabsf(x.w) <= FLT_MAX;
        big = fmaxf(big, a);
      }
    }
    const bool use = on && finite;
    const int ex = min(126, max(-120, ((__float_as_int(big) >> 23) & 255) - 127));
    const float dn = ldexpf(1.0f, -ex);
    qs = finite ? ldexpf(job.d.scale * 1.4426950408889634f, ex) : NAN;  // scores in units of log 2
    uint8_t* dst = job.ops + C::kQ + half * C::kHalf + ((slot & 127) >> 3) * (16 * HD) + (slot & 7) * 16;
#pragma unroll 4
    for (int c = 0; c < HD / 8; ++c) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (use) {
        a = load4(src + 8 * c);
        b = load4(src + 8 * c + 4);
      }
      a = make_float4(a.x * dn, a.y * dn, a.z * dn, a.w * dn);
      b = make_float4(b.x * dn, b.y * dn, b.z * dn, b.w * dn);
      const uint32_t h0 = pack_half(a.x, a.y), h1 = pack_half(a.z, a.w), h2 = pack_half(b.x, b.y), h3 = pack_half(b.z, b.w);
      store16(dst + c * 128, h0, h1, h2, h3);
      if (C::kSplit)
        store16(dst + C::kHalf + c * 128, pack_rest(a.x, a.y, h0), pack_rest(a.z, a.w, h1), pack_rest(b.x, b.y, h2),
                pack_rest(b.z, b.w, h3));
    }
  }

  // One tile that every slot of the warp sees in whole, of pages with ordinary
  // scales: the weights times the V scale come straight from the exponential,
  // exp2(score + log2 sv - mo), and the sum l from their sum per page.  False if
  // the exponents are too far apart for that (nothing is done then).
  __device__ __forceinline__ bool tile_short(const float4* sc) {
    // (each load of 32 columns is on its way while the one before is worked on)
    const uint32_t s = columns();
    uint32_t r[2][32];
    float pm[kTilePages], f[kTilePages], log_v[kTilePages];
    tmem_start(s, r[0]);
#pragma unroll
    for (int k = 0; k < kTilePages; ++k) {
      const float4 z = sc[k];
      f[k] = qs * z.x;
      log_v[k] = z.w;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float x[32];
      tmem_wait(r[c & 1], x);
      tmem_start(s + 32 * ((c + 1) & 3), r[(c + 1) & 1]);  // (after the last, the first again)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float a = fmaxf(x[16 * k], x[16 * k + 1]), b = fmaxf(x[16 * k + 2], x[16 * k + 3]);
#pragma unroll
        for (int e = 4; e < 16; e += 4) {
          a = fmaxf(fmaxf(a, x[16 * k + e]), x[16 * k + e + 1]);
          b = fmaxf(fmaxf(b, x[16 * k + e + 2]), x[16 * k + e + 3]);
        }
        pm[2 * c + k] = fmaxf(a, b) * f[2 * c + k];
      }
    }
    float mn = m, mon = -INFINITY;
    bool near = qs >= 0.0f;  // (a negative or NaN scale goes the long way)
#pragma unroll
    for (int k = 0; k < kTilePages; ++k) {
      mn = fmaxf(mn, pm[k]);
      mon = fmaxf(mon, pm[k] + log_v[k]);
    }
    const float mo_new = mon > mo + 2 * kAbove || mo == -INFINITY ? mon - kAbove : mo;
#pragma unroll
    for (int k = 0; k < kTilePages; ++k) near &= fabsf(mn + log_v[k] - mo_new) < 40.0f;  // (false for NaN)
    if (!__all_sync(kFull, near)) {
      float x[32];
      tmem_wait(r[0], x);  // the load on its way
      return false;
    }
    grow_to<HD, C::kSplit>(mon, mo, s + kTilePos);
    const float alpha = ex2(m - mn);
    float part = 0.0f;
    m = mn;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float x[32];
      tmem_wait(r[c & 1], x);
      if (c < 3) tmem_start(s + 32 * (c + 1), r[(c + 1) & 1]);
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = 2 * c + q;
        const float off = log_v[k] - mo;
        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = ex2(fmaf(x[16 * q + e], f[k], off)), p1 = ex2(fmaf(x[16 * q + e + 1], f[k], off));
          sum0 += p0;
          sum1 += p1;
          hi[8 * q + e / 2] = pack_half(p0, p1);
          if (C::kSplit) lo[8 * q + e / 2] = pack_rest(p0, p1, hi[8 * q + e / 2]);
        }
        part = fmaf(sum0 + sum1, ex2(-off - m), part);
      }
      tmem_store16(s + 32 * c, hi);
      if (C::kSplit) tmem_store16(s + 32 * c + 16, lo);
    }
    add_weights<C::kSplit>(alpha, part, l, lost);
    return true;
  }

  __device__ bool run(const TileSegment& g, int& it) {
    TileShared& sh = job.sh;
    int p0, p1, t0, t1;
    job.tiles(g, p0, p1, t0, t1);
    const bool mine = row >= g.row0 && row < g.row0 + g.rows;
    see_hi = mine ? max(0, sh.pos[row] + 1) : 0;
    see_lo = mine && job.d.window > 0 ? max(0, see_hi - job.d.window) : 0;
    m = mo = -INFINITY;
    l = lost = 0.0f;
    if (!job.takes(g, half)) {
      it += t1 - t0;
      return true;
    }
    for (int t = t0; t < t1; ++t, ++it, ++done) {
      const int at = (p0 + t * kTilePages) * kKv8Page;
      if (!job.wait(&sh.s_full[half], done & 1)) return false;
      tc_fence_after();
      const float4* sc = sh.scale[it % kScales];
      // a slot of another segment has no say: its row is never read
      const bool all = !mine || (see_lo <= at && see_hi >= at + kTilePos);
      if (!__all_sync(kFull, all) || !tile_short(sc)) {
        const Running r = tile_long<HD, C::kSplit>(Running{m, mo, l, lost}, columns(), (unsigned)(at - see_lo),
                                                   (unsigned)(see_hi - see_lo), qs, sc);
        m = r.m;
        mo = r.mo;
        l = r.l;
        lost = r.lost;
      }
      if (C::kSplit) sh.mo[done & 3][slot] = mo;
      tmem_store_wait();
      tc_fence_before();
      bar_arrive(&sh.p_full[half]);
    }
    if (t1 > t0) {
      const TileTurn at = o_full_turn(false, half, done - 1);
      if (!(C::kSplit ? job.wait(&sh.summed, summed_parity(segments))
                      : job.wait(&sh.o_full[at.bar], at.parity)))
        return false;
      ++segments;
      tc_fence_after();
    }
    return true;
  }

  // O of the finished segment, relative to the maximum m: f(first dim, 32 values)
  template <typename F>
  __device__ __forceinline__ void output(bool any, F f) const {
    const float back = m == -INFINITY || mo == -INFINITY ? 0.0f : ex2(mo - m);
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
      float x[32];
      if (any) {
        tmem_load(columns() + (C::kSplit ? kSums : kTilePos) + 32 * c, x);
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] *= back;
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = 0.0f;
      }
      f(32 * c, x);
    }
  }
};

// ---- sums of f32 rows --------------------------------------------------------------
// The matrix units' sums are cut off, not rounded, which adds up over many tiles
// (2700 positions: 7.6e-6 of the result).  With f32 rows O holds one tile, and
// the warps of the second half, which these rows leave free, add it up in f32.
template <typename T, int HD>
struct Sums {
  using J = TileJob<T, HD>;
  const J& job;
  const uint32_t columns;
  int done = 0;

  __device__ explicit Sums(const J& j) : job(j), columns(j.tmem + ((threadIdx.x & 96u) << 16)) {}
  __device__ bool run(const TileSegment& g) {
    TileShared& sh = job.sh;
    int p0, p1, t0, t1;
    job.tiles(g, p0, p1, t0, t1);
    float last = -INFINITY;
    for (int t = t0; t < t1; ++t, ++done) {
      const TileTurn full = o_full_turn(true, 0, done);
      if (!job.wait(&sh.o_full[full.bar], full.parity)) return false;
      tc_fence_after();
      const float mo = sh.mo[done & 3][threadIdx.x & (kTileM - 1)];
      const float beta = last == mo ? 1.0f : ex2(last - mo);  // (0 after -inf)
      last = mo;
      const uint32_t o = columns + kTilePos + 256 * (done & 1), sums = columns + kSums;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        float x[32], y[32];
        tmem_load(o + 32 * c, x);
        if (t > t0) {
          tmem_load(sums + 32 * c, y);
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = fmaf(y[e], beta, x[e]);
        }
        uint32_t r[16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(x[16 * h + e]);
          tmem_store16(sums + 32 * c + 16 * h, r);
        }
      }
      tmem_store_wait();
      tc_fence_before();
      bar_arrive(&sh.o_free[o_free_turn(done).bar]);
    }
    if (t1 > t0) bar_arrive(&sh.summed);
    return true;
  }
};

template <typename T>
__device__ __forceinline__ void store_row(T* p, const float (&x)[32], float mul) {
#pragma unroll
  for (int e = 0; e < 32; e += 4)
    store4(p + e, make_float4(x[e] * mul, x[e + 1] * mul, x[e + 2] * mul, x[e + 3] * mul));
}
// A split's sums: dim e of slot s, groups of four dims changing places by the
// slot, so that the slots of a warp write to eight places at once, not to one.
template <int HD>
__device__ __forceinline__ int sum_at(int s, int e) {
  return s * HD + (e ^ ((s & 7) << 2));
}

// A wait ran out: the unit's rows say so.  (A call of its own, so that its
// registers are not taken from the loops.)
template <typename T, int HD>
__device__ __noinline__ void mark_rows(const Kv8AttnDesc& d, const TileShared& sh) {
  for (int i = threadIdx.x; i < sh.rows * sh.nh * (HD / 4); i += kTileThreads) {
    const int s = i / (HD / 4), e = i % (HD / 4) * 4, row = s / sh.nh, head = sh.h0 + s % sh.nh;
    if (sh.seq[row] < 0) continue;
    const size_t at = sh.row0 + row;
    store4(static_cast<T*>(d.out) + at * d.ldo + (size_t)head * HD + e, make_float4(NAN, NAN, NAN, NAN));
    if (e == 0 && d.lse) d.lse[at * d.heads + head] = NAN;
  }
  if (threadIdx.x == 0) raise(d.flags, QTTS_KV8_TIMEOUT);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTileThreads, 1)
    kv8_tile_kernel(const __grid_constant__ Kv8AttnDesc d) {
  using C = TileCfg<T, HD>;
  extern __shared__ __align__(128) uint8_t smem[];
  TileShared& sh = *reinterpret_cast<TileShared*>(smem + C::kOps);
  pdl_wait();
  const qtts_kv8_cache& c = d.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  cg::cluster_group cluster = cg::this_cluster();
  // The last rows of a sequence see most of it and are taken first: of every
  // d.seq_units units (a sequence's, where the rows are a grid) the last, then
  // the last but one, ...  (Four chunks of 1000 rows: 161 us in unit order, 157 in this.)
  const int per = c.kv_heads * d.head_chunks, rest = blockIdx.x % per, order = blockIdx.x / per;
  const int columns = gridDim.x / per / d.seq_units;
  const int unit = order % columns * d.seq_units + d.seq_units - 1 - order / columns;
  if (unit * d.group_rows >= d.n_rows) return;
  const int group = d.heads / c.kv_heads, hc = rest % d.head_chunks;
  TileJob<T, HD> job{d, sh, smem};
  job.kvh = rest / d.head_chunks;
  job.h0 = job.kvh * group + hc * d.unit_heads;
  job.nh = min(d.unit_heads, group - hc * d.unit_heads);
  job.row0 = unit * d.group_rows;
  job.rows = min(d.group_rows, d.n_rows - job.row0);
  job.nsplit = gridDim.y;
  job.split = blockIdx.y;
  job.halves = d.halves;
  const int cap = c.pages_per_seq * kKv8Page;

  // ---- rows, segments, barriers, TMEM, queries ------------------------------------
  for (int i = tid; i < 2 * kTileM; i += kTileThreads) {
    int seq = -1, pos = -1;
    if (i < job.rows) {
      seq = d.seq[job.row0 + i];
      pos = d.pos[job.row0 + i];
      if (seq >= 0 && (seq >= c.n_seqs || pos >= cap)) {
        raise(d.flags, QTTS_KV8_BAD_ROW);
        if (seq >= c.n_seqs) seq = -1;
        pos = min(pos, cap - 1);
      }
    }
    sh.seq[i] = seq;
    sh.pos[i] = pos;
    sh.segment[i] = TileSegment{0, 0, -1, 0x7fffffff, 0};
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(&sh.k_full[i], kConvert);
      bar_init(&sh.v_full[i], kConvert);
      bar_init(&sh.k_free[i], 1);
      bar_init(&sh.v_free[i], 1);
      bar_init(&sh.s_full[i], 2);
      bar_init(&sh.p_full[i], kTileM);
      bar_init(&sh.o_full[i], C::kSplit ? 2 : 1);
      bar_init(&sh.o_free[i], kTileM);
    }
    bar_init(&sh.summed, kTileM);
    bar_init(&sh.q_full, kTileM * d.halves);
    bar_init(&sh.fin, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.over = 0;
    sh.row0 = job.row0;
    sh.rows = job.rows;
    sh.h0 = job.h0;
    sh.nh = job.nh;
  }
  constexpr int kLast = kTileThreads / 32 - 1;  // the warp of the products
  if (warp == kLast) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_of(&sh.tmem)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  __syncthreads();
  if (warp == kLast) {  // runs of rows of one sequence
    int n = 0;
    for (int r0 = 0; r0 < job.rows; r0 += 32) {
      const int r = r0 + lane;
      const bool in = r < job.rows;
      const bool start = in && (r == 0 || sh.seq[r] != sh.seq[r - 1]);
      const unsigned starts = __ballot_sync(kFull, start);
      const int g = n + __popc(starts & (kFull >> (31 - lane))) - 1;
      if (start) {
        sh.segment[g].row0 = r;
        sh.segment[g].seq = sh.seq[r];
      }
      __syncwarp();
      if (in) {
        atomicAdd(&sh.segment[g].rows, 1);
        const int p = sh.pos[r];
        if (p >= 0) {
          atomicMax(&sh.segment[g].hi, p + 1);
          atomicMin(&sh.segment[g].lo, d.window > 0 ? max(0, p + 1 - d.window) : 0);
        }
      }
      n += __popc(starts);
      __syncwarp();
    }
    if (lane == 0) sh.n_segments = n;
  }
  Softmax<T, HD> soft(job);
  const bool softmax = tid < kTileM * d.halves;  // (the second half's warps have nothing to do with one half)
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  job.tmem = sh.tmem;

  Converter<T, HD> conv(job);
  Products<T, HD> products(job);
  Sums<T, HD> sums_of(job);
  bool ok = true;
  int it = 0;
  if (softmax) {  // (while the first codes are on their way)
    soft.put_query();
    smem_to_async();
    if (d.wait_ns > 0) bar_arrive(&sh.q_full);  // (0: the wait for it is to run out)
  }
  if (warp == kLast) ok = job.wait(&sh.q_full, 0);
  for (int g = 0; g < sh.n_segments; ++g) {
    const TileSegment seg = sh.segment[g];
    if (seg.seq < 0) continue;  // padding
    if (ok) {
      if (softmax) ok = soft.run(seg, it);
      else if (warp == kLast) ok = products.run(seg, it);
      else if (tid >= kSoft) ok = conv.run(seg, it);
      else if (C::kSplit) ok = sums_of.run(seg);
    }
    const bool mine = softmax && soft.row >= seg.row0 && soft.row < seg.row0 + seg.rows;
    int p0, p1, t0, t1;
    job.tiles(seg, p0, p1, t0, t1);
    if (job.nsplit == 1) {
      if (softmax && ok && job.takes(seg, soft.half)) {
        const size_t row = job.row0 + soft.row;
        const int head = job.h0 + soft.head;
        const bool none = soft.m == -INFINITY && soft.l == soft.l;
        const float inv = none ? 0.0f : __fdiv_rn(1.0f, soft.l);
        T* out = static_cast<T*>(d.out) + row * d.ldo + (size_t)head * HD;
        soft.output(t1 > t0, [&](int e, const float(&x)[32]) {
          if (mine) store_row(out + e, x, inv);
        });
        if (mine && d.lse)
          d.lse[row * d.heads + head] = none ? -INFINITY : (soft.m + log2f(soft.l)) * 0.6931471805599453f;
        tc_fence_before();
      }
      continue;
    }
    // join the splits of the cluster, in their order: O over the K and V operands
    float* sums = reinterpret_cast<float*>(smem + C::kK);
    __syncthreads();
    if (softmax && job.takes(seg, soft.half)) {
      soft.output(t1 > t0 && ok, [&](int e0, const float(&x)[32]) {
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          store4(sums + sum_at<HD>(soft.slot, e0 + e), make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]));
      });
      sh.m[tid] = soft.l == soft.l ? soft.m : INFINITY;  // a NaN sum makes the join NaN
      sh.l[tid] = soft.l;
      tc_fence_before();
    }
    cluster.sync();
    const int first = seg.row0 * job.nh, n = seg.rows * job.nh * HD;
    for (int i = tid + job.split * kTileThreads; i < n; i += job.nsplit * kTileThreads) {
      const int s = first + i / HD, e = i % HD;
      float mx = -INFINITY, sum = 0.0f, ll = 0.0f;
      for (int r = 0; r < job.nsplit; ++r) {
        const float rm = *cluster.map_shared_rank(&sh.m[s], r), rl = *cluster.map_shared_rank(&sh.l[s], r),
                    ro = *cluster.map_shared_rank(&sums[sum_at<HD>(s, e)], r);
        const float mn = fmaxf(mx, rm);
        if (mn == -INFINITY) continue;
        const float a = ex2(mx - mn), b = ex2(rm - mn);
        sum = sum * a + ro * b;
        ll = ll * a + rl * b;
        mx = mn;
      }
      const size_t row = job.row0 + s / job.nh;
      const int head = job.h0 + s % job.nh;
      const float v = mx == -INFINITY ? 0.0f : __fdiv_rn(sum, ll);
      T* op = static_cast<T*>(d.out) + row * d.ldo + (size_t)head * HD + e;
      if constexpr (sizeof(T) == 4) *op = v;
      else *op = T(v);
      if (e == 0 && d.lse)
        d.lse[row * d.heads + head] = mx == -INFINITY ? -INFINITY : (mx + log2f(ll)) * 0.6931471805599453f;
    }
    cluster.sync();  // no CTA goes on while its sums are read
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // (none is left unless a wait ran out)
  // A dependent kernel may start now: it could take TMEM that a CTA of this one
  // still had to get, had it started before the allocation.
  pdl_launch_dependents();
  __syncthreads();
  if (sh.over) mark_rows<T, HD>(d, sh);  // (after what other CTAs of the cluster have written)
  // every product is done (a wait that ran out leaves some in flight) before TMEM goes
  if (tid == kLast * 32) commit_to(&sh.fin);
  if (warp == kLast) {
    int over = 0;  // (of this wait alone)
    bar_wait(&sh.fin, 0, &over, kKv8WaitNs);
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(job.tmem), "r"(kTmemCols));
  }
}

template <typename T, int HD>
cudaError_t launch_tile_t(const Kv8AttnDesc& d, const TilePlan& plan, cudaStream_t st) {
  using C = TileCfg<T, HD>;
  static std::atomic<int> ready[kMaxDevices];
  const cudaError_t set = once_per_device(ready, [] {
    return cudaFuncSetAttribute(kv8_tile_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (set != cudaSuccess) return set;
  return launch_k(kv8_tile_kernel<T, HD>, dim3((unsigned)plan.units, plan.splits), dim3(kTileThreads), (size_t)C::kSmem,
                  st, LaunchOpts{true, plan.splits}, d);
}

}  // namespace

TilePlan plan_kv8_tile(Kv8AttnDesc& d, int dtype, int max_rows, int max_len, int sms) {
  const int group = d.heads / d.c.kv_heads;
  d.unit_heads = std::min(group, kTileM);
  d.head_chunks = (group + d.unit_heads - 1) / d.unit_heads;
  // Rows of a unit: what its slots hold, or a sequence's rows in equal shares.
  // Two halves (16-bit rows) where the units still fill the device.
  TilePlan plan{0, 1};
  for (d.halves = dtype == DT_F32 ? 1 : 2;; d.halves = 1) {
    const int most = d.halves * kTileM / d.unit_heads, parts = (max_rows + most - 1) / most;
    d.group_rows = std::min(most, (max_rows + parts - 1) / parts);
    d.seq_units = (max_rows + d.group_rows - 1) / d.group_rows;
    const long all = ((long)d.n_rows + d.group_rows - 1) / d.group_rows;
    plan.units = (all + d.seq_units - 1) / d.seq_units * d.seq_units * d.c.kv_heads * d.head_chunks;
    if (d.halves == 1 || (plan.units >= sms && d.group_rows * d.unit_heads > kTileM)) break;
  }
  // the positions are split while the CTAs do not fill the device and keep two tiles
  const int seen = d.window > 0 ? (int)std::min<long>(max_len, (long)d.window + d.group_rows - 1) : max_len;
  const int tiles = (seen + kTilePos - 1) / kTilePos;
  while (plan.splits < 8 && plan.units * plan.splits * 2 <= sms && tiles >= (int)plan.splits * 4) plan.splits *= 2;
  return plan;
}

cudaError_t launch_kv8_tile(const Kv8AttnDesc& d, const TilePlan& plan, int dtype, cudaStream_t st) {
  const bool w = d.c.head_dim == 128;
  switch (dtype) {
    case DT_F16: return w ? launch_tile_t<__half, 128>(d, plan, st) : launch_tile_t<__half, 64>(d, plan, st);
    case DT_BF16:
      return w ? launch_tile_t<__nv_bfloat16, 128>(d, plan, st) : launch_tile_t<__nv_bfloat16, 64>(d, plan, st);
    default: return w ? launch_tile_t<float, 128>(d, plan, st) : launch_tile_t<float, 64>(d, plan, st);
  }
}

}  // namespace qtts
