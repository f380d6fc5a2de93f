// Copies of KV pages (fork and compaction of sequences) for gfx950.
//
// A move copies the first `slots` token slots of one physical page into
// another, in every cache (K and V of each layer): cache[c][dst][s] =
// cache[c][src][s] for s < slots; the destination's other slots keep their
// values. The slots of a page are contiguous ([16][kv_heads][128] bf16), so a
// (move, cache) pair is one contiguous copy of at most 32 KiB at 8 KV heads.
//
// The moves come from the host's page pool, so they travel in the launch's
// arguments (kMovesPerLaunch at a time): no list in device memory, nothing to
// keep alive after the call, and a captured graph holds its own. The callers
// refuse lists in which a destination occurs twice or is a source, so the
// workgroups of all launches of a call are independent.
#include "common.hpp"
#include "kernels.hpp"

namespace fh {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kMovesPerLaunch = 256;
constexpr uint32_t kCopyThreads = 256;

struct MoveList {
  uint32_t src[kMovesPerLaunch], dst[kMovesPerLaunch];
  uint8_t slots[kMovesPerLaunch];
};

// Workgroup (move, cache).
__global__ __launch_bounds__(kCopyThreads) void kv_copy_kernel(uint16_t* caches, uint64_t cache_stride, uint32_t kvh,
                                                               MoveList list) {
  const uint32_t i = blockIdx.x;
  const uint32_t chunks = list.slots[i] * kvh * 16;  // 16-byte chunks of the slots
  const uint64_t page = (uint64_t)16 * kvh * 128;
  uint16_t* cache = caches + blockIdx.y * cache_stride;
  const u32x4* src = reinterpret_cast<const u32x4*>(cache + list.src[i] * page);
  u32x4* dst = reinterpret_cast<u32x4*>(cache + list.dst[i] * page);
  for (uint32_t c = threadIdx.x; c < chunks; c += kCopyThreads) dst[c] = src[c];
}

}  // namespace

hipError_t launch_kv_copy(uint16_t* caches, uint32_t cache_count, uint64_t cache_stride, const uint32_t* src,
                          const uint32_t* dst, const uint32_t* slots, uint64_t step, uint32_t count, uint32_t kvh,
                          hipStream_t s) {
  for (uint32_t at = 0; at < count; at += kMovesPerLaunch) {
    const uint32_t n = count - at < kMovesPerLaunch ? count - at : kMovesPerLaunch;
    MoveList list;
    for (uint32_t i = 0; i < kMovesPerLaunch; ++i) {
      const uint64_t k = (uint64_t)(at + (i < n ? i : 0)) * step;
      list.src[i] = src[k];
      list.dst[i] = dst[k];
      list.slots[i] = (uint8_t)(i < n ? slots[k] : 0);
    }
    hipLaunchKernelGGL(kv_copy_kernel, dim3(n, cache_count), dim3(kCopyThreads), 0, s, caches, cache_stride, kvh, list);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace fh
