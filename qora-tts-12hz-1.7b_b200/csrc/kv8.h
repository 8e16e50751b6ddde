// kv8.h -- the 8-bit paged K/V cache: descriptors and launchers of its append
// and attention kernels, and what the entry points on device pointers share.
#pragma once
#include <atomic>
#include <cstdint>
#include <initializer_list>

#include "../../include/qtts.h"
#include "kernels.h"

namespace qtts {

constexpr int kKv8Page = 16;  // positions per page, the block a scale belongs to
constexpr unsigned kKv8WaitNs = 1000000000u;  // limit of a device wait

enum DType : int { DT_F32 = QTTS_F32, DT_F16 = QTTS_F16, DT_BF16 = QTTS_BF16 };
inline int dtype_bytes(int t) { return t == DT_F32 ? 4 : 2; }

// what an entry point asks of a pointer before a kernel follows it
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool words_aligned(std::initializer_list<const void*> all) {  // of 4 bytes; null is
  for (const void* p : all)
    if (!aligned(p, 4)) return false;
  return true;
}

// Makes the device that holds `p` current while it lives, so that a caller's
// buffers may lie on another device than its current one.  `err` says why not
// (a host pointer, no device).
class OnDeviceOf {
 public:
  explicit OnDeviceOf(const void* p);
  ~OnDeviceOf();
  const char* err = nullptr;
  int code = 0;
  int sm_count = 148;

 private:
  int prev_ = -1;
};

// Runs `set` (function attributes, which belong to a device) the first time on
// each device; `state` is one word a device, kept by the caller.
constexpr int kMaxDevices = 64;
template <typename F>
cudaError_t once_per_device(std::atomic<int>* state, F set) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kMaxDevices && state[dev].load(std::memory_order_acquire)) return cudaSuccess;
  e = set();
  if (e == cudaSuccess && dev < kMaxDevices) state[dev].store(1, std::memory_order_release);
  return e;
}

struct Kv8AppendDesc {
  qtts_kv8_cache c;
  const void *q = nullptr, *k = nullptr, *v = nullptr;
  void* q_out = nullptr;
  long ldq = 0, ldk = 0, ldv = 0, ldqo = 0;
  int heads = 0;
  const __half *q_norm = nullptr, *k_norm = nullptr;
  const float *rope_cos = nullptr, *rope_sin = nullptr;
  int rope_rows = 0;
  const int *seq = nullptr, *pos = nullptr, *rope_pos = nullptr;
  int n_rows = 0;
  int* flags = nullptr;
  int chunk = 1;       // rows whose blocks one warp looks for (1, 2, 4, 8 or 16)
  long kv_warps = 0;   // warps of K / V blocks
};
cudaError_t launch_kv8_append(Kv8AppendDesc d, int dtype, int sms, cudaStream_t st);

struct Kv8AttnDesc {
  qtts_kv8_cache c;
  const void* q = nullptr;
  void* out = nullptr;
  float* lse = nullptr;
  long ldq = 0, ldo = 0;
  int heads = 0;
  float scale = 1.0f;
  int window = 0;
  const int *seq = nullptr, *pos = nullptr;
  int n_rows = 0;
  int* flags = nullptr;
  int group_rows = 1;   // rows of one unit
  int head_chunks = 1;  // units along the query heads of one K/V head
  int unit_heads = 1;   // query heads of a unit
  int halves = 1;       // tile kernel: halves of 128 slots of a unit
  int seq_units = 1;    // tile kernel: units of a sequence of max_rows rows
  unsigned wait_ns = kKv8WaitNs;  // tile kernel: limit of a wait; 0: one is made to run out
};
cudaError_t launch_kv8_attention(Kv8AttnDesc d, int dtype, int max_rows, int max_len, int sms, cudaStream_t st);
// The same for many rows: tiles of 128 slots on the tensor cores (kv8_tile.cu).
// The plan fills the descriptor's shape of a unit.
struct TilePlan {
  long units;
  unsigned splits;  // CTAs of a cluster that share a unit's positions
};
TilePlan plan_kv8_tile(Kv8AttnDesc& d, int dtype, int max_rows, int max_len, int sms);
cudaError_t launch_kv8_tile(const Kv8AttnDesc& d, const TilePlan& plan, int dtype, cudaStream_t st);

}  // namespace qtts
