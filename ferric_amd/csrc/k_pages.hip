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
constexpr uint32_t kCopyThreads = 256, kCopyChunks = 8;
// Bytes from which a call streams past the caches (the last-level one holds 256 MB).
constexpr uint64_t kStreamBytes = 256ull << 20;

struct MoveList {
  uint32_t src[kMovesPerLaunch], dst[kMovesPerLaunch];
  uint8_t slots[kMovesPerLaunch];
};

// Workgroup (move, cache): kCopyChunks 16-byte loads per thread in flight (a
// whole page at 8 KV heads), then the stores. What bounds it is memory, both
// ways. STREAM: non-temporal, for calls that move more than the caches hold
// (1111 whole pages of 72 caches, 5.2 GB: 1018 us, 5.1 TB/s, against 1054 with
// ordinary accesses). Below that the copies are ordinary: a fork's source page
// is read once per fork out of the L2s and the next step reads the new pages
// (31 forks at 9 slots, 42 MB: 9.6 us against 10.1 with non-temporal stores and
// 17.9 with non-temporal loads). Other shapes measured (caches fastest in the
// grid, 128 to 1024 threads) were between 2 % faster and 45 % slower. One fork
// of Qwen3-0.6B, 0.6 MB: 4.6 us a launch in a row, which is the launch.
template <bool STREAM>
__global__ __launch_bounds__(kCopyThreads) void kv_copy_kernel(uint16_t* caches, uint64_t cache_stride, uint32_t kvh,
                                                               MoveList list) {
  const uint32_t i = blockIdx.x;
  const uint32_t chunks = list.slots[i] * kvh * 16;  // 16-byte chunks of the slots
  const uint64_t page = (uint64_t)16 * kvh * 128;
  uint16_t* cache = caches + blockIdx.y * cache_stride;
  const u32x4* src = reinterpret_cast<const u32x4*>(cache + list.src[i] * page);
  u32x4* dst = reinterpret_cast<u32x4*>(cache + list.dst[i] * page);
  for (uint32_t base = threadIdx.x; base < chunks; base += kCopyThreads * kCopyChunks) {
    u32x4 v[kCopyChunks];
#pragma unroll
    for (uint32_t u = 0; u < kCopyChunks; ++u) {
      const uint32_t c = base + u * kCopyThreads;
      if (c < chunks) v[u] = STREAM ? __builtin_nontemporal_load(src + c) : src[c];
    }
#pragma unroll
    for (uint32_t u = 0; u < kCopyChunks; ++u) {
      const uint32_t c = base + u * kCopyThreads;
      if (c >= chunks) continue;
      if constexpr (STREAM)
        __builtin_nontemporal_store(v[u], dst + c);
      else
        dst[c] = v[u];
    }
  }
}

}  // namespace

hipError_t launch_kv_copy(uint16_t* caches, uint32_t cache_count, uint64_t cache_stride, const uint32_t* src,
                          const uint32_t* dst, const uint32_t* slots, uint64_t step, uint32_t count, uint32_t kvh,
                          hipStream_t s) {
  uint64_t total = 0;
  for (uint32_t i = 0; i < count; ++i) total += slots[i * step];
  const bool stream = total * kvh * 256 * cache_count >= kStreamBytes;
  for (uint32_t at = 0; at < count; at += kMovesPerLaunch) {
    const uint32_t n = count - at < kMovesPerLaunch ? count - at : kMovesPerLaunch;
    MoveList list{};
    for (uint32_t i = 0; i < n; ++i) {
      const uint64_t k = (uint64_t)(at + i) * step;
      list.src[i] = src[k];
      list.dst[i] = dst[k];
      list.slots[i] = (uint8_t)slots[k];
    }
    if (stream)
      hipLaunchKernelGGL(kv_copy_kernel<true>, dim3(n, cache_count), dim3(kCopyThreads), 0, s, caches, cache_stride, kvh,
                         list);
    else
      hipLaunchKernelGGL(kv_copy_kernel<false>, dim3(n, cache_count), dim3(kCopyThreads), 0, s, caches, cache_stride,
                         kvh, list);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace fh
