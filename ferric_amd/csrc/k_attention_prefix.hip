// K4 for batches whose rows share a prefix (continuations of one prompt): the
// prefix's keys and values are read once for all rows of a group, each row's
// own ones once for the row.
//
// Contract of k_attention.hip: for a query row at position p, keys t = 0..p
// through the row's page table, score = (q . k_t) * f32(0x3db504f3), softmax,
// out = bf16(n / l). Attention over a union of key sets is the merge of the
// states over each: with (m_i, l_i, n_i) = (max s, sum e^(s - m_i), sum
// e^(s - m_i) v), M = max m_i, out = sum n_i e^(m_i - M) / sum l_i e^(m_i - M).
// A state covers a chunk of a prefix (for up to 128 query vectors of one KV head
// at once) or a part of a row's own keys. Two launches: the first leaves the
// chunks' states as FP32 records in the scratch; the second takes the own keys and
// joins them with the records.
//
// A wave owns 16 query vectors (vector j: row j / G, head j % G of the KV head)
// and walks keys 32 or 64 at a time:
//   S^T = K Q^T on v_mfma_f32_16x16x32_bf16, 16 keys a tile: lane l holds vector
//   l % 16 and keys 4 (l / 16) + e (e = 0..3), so a vector's maximum is two
//   exchanges between the four lane groups, and only when a tile's maximum
//   exceeds the running one by more than 8 in the exponent of 2 does it move (the
//   terms then reach at most 2^8: no precision is lost, and the accumulators are
//   rescaled rarely). Each lane sums its own keys' terms until the end.
//   O^T += V^T P^T on the same MFMA, 32 keys each: P is FP32 and enters as two
//   bf16 terms, hi = bf16(p) and lo = bf16(p - hi) (within 2^-17 p of p). The B
//   operand of two tiles is a lane's own eight terms, which fixes the order of the
//   32 keys inside the MFMA; the V^T operand follows it with transposing LDS reads
//   (ds_read_b64_tr_b16: 16 lanes read 4 keys x 16 dims, each lane gets one dim's
//   4 keys).
// LDS rows are 256 bytes (one token) with their 16-byte chunks permuted so that
// the reads spread over the banks: K chunk c of key t at c ^ (t % 16), V chunk c
// at c ^ 2 (t % 8). Slots that are no keys of the state are outside the loads'
// buffer bounds and arrive as zeros, so what they hold never meets an MFMA.
//
// Forms. Wide (prefix chunks of more than 16 vectors): the 8 waves share 64-key
// tiles of K and V, fetched global -> LDS directly, double-buffered: all 8 with
// vectors of their own (128 a workgroup), or 4 pairs of waves (64 vectors) of which
// each takes half of a tile's keys, which halves the time from a tile's arrival to
// the next fetch. Narrow (own keys, and prefix chunks of up to 16 vectors): the waves
// take 32 keys each, K straight into the A operand's registers (a token's 64-byte
// pieces), V through 8 KiB of LDS of the wave's own; their states meet in LDS at the
// end. All forms keep to 128 registers a thread, and to 68.6 KB of LDS for a prefix's
// chunks and 76.9 KB (in workgroups of 4 waves 38.5) for own keys, so that two
// workgroups (four) can share a CU. Own keys are cut for that many. A long prefix is cut
// into about as many chunks as there are CUs (kChunkWgs), so there a CU has one
// workgroup, and its waves have only one another to wait with.
//
// What bounds it (kernel times, 32 rows, 8 KV heads of 4 query heads): behind 8192
// shared tokens the first launch takes 15 us (33.6 MB of keys and values, which the
// 256 MB cache keeps between steps, and 17 MB of records) and the second 12, a
// chain of latencies: position -> records -> page table -> keys -> join. Behind
// 32000 tokens the first takes 38: 131 MB from HBM at 3.5 TB/s, a tile of 32 KB a CU
// in flight while the one before is computed, which takes turns with the loads at a
// barrier each tile. Four tiles in flight were slower (18 us and 42), for a reason
// that was not found.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace fh {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kKeys = 64;             // keys per tile of the wide form
constexpr size_t kTileBytes = 16 * 2 * kKeys * 16;  // K or V, double-buffered
// Least tokens of a prefix chunk (256 instead: 4 rows behind 1488 tokens 1.1 us slower).
constexpr uint32_t kMinChunk = 128;
// Chunks are cut for about this many workgroups: more of them write and join more records, fewer
// leave CUs idle (32 rows behind 8192 tokens: 26.4 us with 256; 192 and 384 were slower in every case tried).
constexpr uint32_t kChunkWgs = 256;
// From this many bytes of prefix that one pass reads once each it streams past the caches (32 rows
// behind 32000 tokens, 131 MB: 61.7 us cached, 53.2 streamed; smaller ones, which the
// 256 MB cache still holds from the step before, are 3 to 10 % slower streamed).
constexpr uint64_t kStreamBytes = 96ull << 20;
// Least own keys of a part where a row has several. A step of 256 keys takes about 3.5 us and the
// meeting of the parts about 3: with few (row, KV head) pairs 256 (2 rows of 2000 own keys:
// 18.9 us, with 512 21.0, with 1024 29.4), with many, where parts only take turns, 512
// (29 rows of up to 900: 25.8 us with 256, 24.5 with 512).
constexpr uint32_t kPartKeysFew = 256, kPartKeysMany = 512, kManyPairs = 128;
// Own keys in workgroups of 4 waves, four on a CU, where there are this many (row, KV head) pairs and none can have
// more than kShortOwn own keys, by the caller's context_tokens: who passes the batch's longest length has this form,
// who passes a capacity (a decode step, which also has at most 32 rows) the other one (160 rows of 8 KV heads with up
// to 300: 42.6 us, with 8 waves 47.6; 64 rows with up to 60: 14.2, 15.3). A longest row sets the time else, and 8
// waves are through with it sooner (80 rows with up to 1500: 39.6 us, with 4 waves 44.5; 128 with 500 to 2000: 97.4,
// 102.6).
constexpr uint32_t kManyOwn = 512, kShortOwn = 512;
constexpr uint32_t kMaxParts = 32;
constexpr uint32_t kSlots = 512;      // workgroups that run at once: two on each CU
constexpr uint32_t kVectors = 16;     // of a wave
// f32(0x3db504f3) (1/sqrt(128), paged_decode.rs:31-35) times log2 e.
constexpr float kScoreScale = 0.08838834764831845f * 1.44269504088896341f;
constexpr uint32_t kRecord = 132;     // m, l, two unused, n[128]: 16-byte aligned

struct Group {
  uint32_t first_row, rows, prefix_tokens;
  uint32_t item0;  // its first prefix item: vector block + blocks * chunk
};
struct Groups {
  uint32_t count, chunk, block_rows, prefix_slots, stream;
  Group g[kPrefixMaxGroups];
};

// What every state needs.
struct Args {
  const uint16_t *q, *kc, *vc;
  uint32_t qh, kvh, pages;
  uint32_t* err;
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// Keeps a wave's LDS accesses before and after it in order.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Largest and sum over the four 16-lane groups that hold a vector's keys.
__device__ __forceinline__ float group_max(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  const float w = fmaxf(__builtin_bit_cast(float, (uint32_t)s[0]), __builtin_bit_cast(float, (uint32_t)s[1]));
  const uint32_t c = __builtin_bit_cast(uint32_t, w);
  const auto t = __builtin_amdgcn_permlane32_swap(c, c, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)t[0]), __builtin_bit_cast(float, (uint32_t)t[1]));
}
__device__ __forceinline__ float group_sum(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  const float w = __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
  const uint32_t c = __builtin_bit_cast(uint32_t, w);
  const auto t = __builtin_amdgcn_permlane32_swap(c, c, false, false);
  return __builtin_bit_cast(float, (uint32_t)t[0]) + __builtin_bit_cast(float, (uint32_t)t[1]);
}

// A wave's running state of its 16 vectors.
struct State {
  float m, l, s_abs;  // of vector lane % 16: maximum, the lane's part of the sum, largest |score|
  f32x4 acc[8];       // dims 16 d + 4 (lane / 16) + e

  __device__ __forceinline__ void clear() {
    m = -__builtin_inff();
    l = s_abs = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Takes in T tiles of 16 scores: keys first + 16 t + 4 (lane / 16) + e below `end`.
  // v_at(t, d, v): the V^T operands of tiles t, t + 1 (t even) for dims 16 d .. + 63.
  template <int T, class V>
  __device__ __forceinline__ void take(f32x4 (&s)[T], uint32_t first, uint32_t end, const V& v_at) {
    const float kNegInf = -__builtin_inff();
    const uint32_t at = first + 4 * ((threadIdx.x & 63) >> 4);
    if (first + 16 * T > end) {
      // Keys past the end: no term (and no part in the finiteness check).
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool ok = at + 16 * t + e < end;
          s_abs = fmaxf(s_abs, ok ? __builtin_fabsf(s[t][e]) : 0.f);
          s[t][e] = ok ? s[t][e] : kNegInf;
        }
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s_abs = fmaxf(s_abs, __builtin_fabsf(s[t][e]));
    }
    float top = kNegInf;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, s[t][e]);
    top = group_max(top);
    // (No key at all so far: m and top both -inf, their difference NaN, no move.)
    if (__builtin_amdgcn_ballot_w64((top - m) * kScoreScale > 8.f) != 0ull) {
      const float m_new = fmaxf(m, top);
      const float a = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * kScoreScale);
      m = m_new;
      l *= a;
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[d][e] *= a;
    }
    const float mc = m == kNegInf ? 0.f : m * kScoreScale;
    // 32 keys at a time; the V operands of four dim tiles are requested before the MFMAs of the four before them,
    // the first ones before the exponentials.
    bf16x8 va[2][4];
    v_at(0, 0, va[0]);
#pragma unroll
    for (int t = 0; t < T; t += 2) {
      float p[8];
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t + (e >> 2)][e & 3], kScoreScale, -mc));
        l += p[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ph[e] = pack_bf16x2(p[2 * e], p[2 * e + 1]);
        asm volatile("" : "+v"(ph[e]));  // its halves by shift and mask, not by rounding again
        pl[e] = pack_bf16x2(p[2 * e] - lo_bf16(ph[e]), p[2 * e + 1] - hi_bf16(ph[e]));
      }
      const bf16x8 bh = __builtin_bit_cast(bf16x8, u32x4{ph[0], ph[1], ph[2], ph[3]});
      const bf16x8 bl = __builtin_bit_cast(bf16x8, u32x4{pl[0], pl[1], pl[2], pl[3]});
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half == 0)
          v_at(t, 4, va[1]);
        else if (t + 2 < T)
          v_at(t + 2, 0, va[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < 4; ++d)
          acc[4 * half + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[half][d], bh, acc[4 * half + d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < 4; ++d)
          acc[4 * half + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[half][d], bl, acc[4 * half + d], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // The vector's sum in every lane group.
  __device__ __forceinline__ void finish() {
    l = group_sum(l);
    s_abs = group_max(s_abs);
  }
};

typedef __attribute__((address_space(3))) unsigned char* LdsBytes;

// Transposing reads of V^T from LDS rows of tokens (256 bytes each): keys 16 t + 4 (lane / 16) + 0..3 of tiles t and
// t + 1, dims 16 d .. + 63. lane_v: a lane's address part, v_lane(); the chunk permutation makes dims 16 d of it an
// exclusive or with 32 d.
__device__ __forceinline__ uint32_t v_lane(int lane) {
  const uint32_t j = lane & 15, key = 4 * (lane >> 4) + (j >> 2);
  return key * 256 + 32 * (key & 7) + 8 * (j & 3);
}
__device__ __forceinline__ void v_operands(LdsBytes rows, uint32_t lane_v, int t, int d, bf16x8 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u32x2 w[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      w[u] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (__attribute__((address_space(3))) s16x4*)(rows + (lane_v ^ (32 * (d + i))) +
                                                                                      (t + u) * 4096)));
    v[i] = __builtin_bit_cast(bf16x8, u32x4{w[0][0], w[0][1], w[1][0], w[1][1]});
  }
}
// K operand of one 16-key tile: keys lane % 16, dims 32 i + 8 (lane / 16) .. + 7, i = 0..3.
__device__ __forceinline__ uint32_t k_lane(int lane) {
  return (lane & 15) * 256 + 16 * ((lane >> 4) ^ (lane & 15));
}
__device__ __forceinline__ void k_operands(LdsBytes rows, uint32_t lane_k, bf16x8 (&k)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    k[i] = *(__attribute__((address_space(3))) bf16x8*)(rows + (lane_k ^ (64 * i)));
}

// Query operand: vector lane % 16 of the wave's 16 (vector `vec` of nrows rows), dims 32 i + 8 (lane / 16) .. + 7.
template <int G>
__device__ __forceinline__ void load_q(u32x4 (&qv)[4], const Args& a, uint32_t row0, uint32_t nrows, uint32_t vec,
                                       uint32_t h) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    qv[i] = vec < nrows * G ? *reinterpret_cast<const u32x4*>(
                                  a.q + ((uint64_t)(row0 + vec / G) * a.qh + h * G + vec % G) * 128 + 32 * i +
                                  8 * (lane >> 4))
                            : u32x4{0u, 0u, 0u, 0u};
}

// Record of (row, query head): m in the exponent of 2, l, n.
__device__ __forceinline__ void store_record(float* r, const State& st, uint32_t* err) {
  const int g16 = (threadIdx.x & 63) >> 4;
  if (g16 == 0) {
    r[0] = st.m * kScoreScale;
    r[1] = st.l;
  }
#pragma unroll
  for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(r + 4 + 16 * d + 4 * g16) = st.acc[d];
  if (!(st.l > 0.f) | !(st.s_abs < __builtin_inff())) raise_error(err, ERR_NONFINITE);
}

// A page of the table: its base for KV head h and the bytes of its first `valid` tokens (none where the page
// is outside the pool).
struct Page {
  uint64_t base;
  uint32_t bytes;
};
__device__ __forceinline__ Page page_of(const Args& a, uint32_t page, uint32_t valid, uint32_t h, uint32_t& bad) {
  if (page >= a.pages) {
    bad |= valid;
    page = valid = 0;
  }
  return Page{((uint64_t)page * 16 * a.kvh + h) * 128, valid * a.kvh * 256};
}

// The wide form: nrows rows from row0 on (sharing trow's pages), keys [key0, key1) of KV head h, key0 a
// multiple of 16. The waves share 64-key tiles, the next one in flight: 8 / WK waves own the vectors; with WK = 2 two
// waves share them and take half of a tile's keys each. rec: record of (row 0, head 0), row and head steps of `slots`
// records.
template <int G, int WK>
__device__ __forceinline__ void attend_wide(unsigned char* lds_raw, const Args& a, const uint32_t* __restrict__ trow,
                                            uint32_t row0, uint32_t nrows, uint32_t key0, uint32_t key1, uint32_t h,
                                            bool stream, float* rec, uint32_t slots) {
  constexpr int WQ = kWaves / WK, kTiles = kKeys / 16 / WK;  // 16-key tiles a wave takes of each 64
  auto& klds = *reinterpret_cast<u32x4(*)[2][kKeys][16]>(lds_raw);
  auto& vlds = *reinterpret_cast<u32x4(*)[2][kKeys][16]>(lds_raw + kTileBytes);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wq = wave % WQ, wk = wave / WQ;
  const uint32_t page0 = key0 / 16, npages = (key1 - key0 + 15) / 16, tiles = (key1 - key0 + kKeys - 1) / kKeys;
  // Page-table entries of 64 pages, one per lane, the next 64 requested ahead.
  auto table_chunk = [&](uint32_t first) { return first + lane < npages ? trow[page0 + first + lane] : 0u; };
  uint32_t tab = table_chunk(0), tab_next = table_chunk(64);
  // Waves 0..3 copy K of the tile's pages 0..3, waves 4..7 V: four tokens per load (lane: token 4 i + lane / 16, LDS
  // chunk lane % 16).
  const int my_page = wave & 3;
  const bool is_v = wave >= 4;
  uint32_t off[4], bad_page = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t token = 4 * i + (lane >> 4), swizzle = is_v ? 2 * (token & 7) : token;
    off[i] = token * a.kvh * 256 + (((lane & 15) ^ swizzle) & 15) * 16;
  }
  auto fetch = [&](uint32_t t) {
    const uint32_t pi = 4 * t + my_page;
    const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)tab, (int)(pi & 63u));
    const Page p = page_of(a, page, pi < npages ? min(16u, key1 - key0 - pi * 16) : 0u, h, bad_page);
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)((is_v ? a.vc : a.kc) + p.base), 0, p.bytes, 0x00020000);
    u32x4(*to)[16] = (is_v ? vlds : klds)[t & 1] + 16 * my_page;
#define FH_FETCH(AUX_)                                                                                             \
  _Pragma("unroll") for (int i = 0; i < 4; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(                          \
      rsrc, (__attribute__((address_space(3))) void*)&to[4 * i][0], 16, off[i], 0, 0, AUX_)
    if (stream)
      FH_FETCH(2);  // non-temporal
    else
      FH_FETCH(0);
#undef FH_FETCH
  };
  fetch(0);
  const uint32_t vec = kVectors * wq + (lane & 15);
  const bool live = (uint32_t)(kVectors * wq) < nrows * G;  // a wave with no vectors only fetches
  u32x4 qv[4];
  load_q<G>(qv, a, row0, nrows, vec, h);
  uint32_t lane_k = k_lane(lane), lane_v = v_lane(lane);
  State st;
  st.clear();
  for (uint32_t t = 0; t < tiles; ++t) {
    __builtin_amdgcn_s_waitcnt(0 | (7u << 4) | (15u << 8));  // this wave's share of tile t is in LDS
    __syncthreads();  // everyone's is, and everyone is done with tile t - 1
    if (t + 1 < tiles) {
      if ((t + 1) % 16 == 0) {
        tab = tab_next;
        tab_next = table_chunk(4 * (t + 1) + 64);
      }
      fetch(t + 1);
    }
    if (!live) continue;
    asm volatile("" : "+v"(lane_k), "+v"(lane_v));  // the reads' addresses are made here each time: kept, they spill
    const int mine = kTiles * wk;
    const LdsBytes kb = (LdsBytes)&klds[t & 1][16 * mine][0], vb = (LdsBytes)&vlds[t & 1][16 * mine][0];
    f32x4 s[kTiles];
#pragma unroll
    for (int u = 0; u < kTiles; u += 2) {
      bf16x8 k[2][4];
      k_operands(kb + u * 4096, lane_k, k[0]);
      k_operands(kb + (u + 1) * 4096, lane_k, k[1]);
      s[u] = s[u + 1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < 2; ++w)
          s[u + w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[w][i], __builtin_bit_cast(bf16x8, qv[i]), s[u + w], 0, 0, 0);
    }
    st.template take<kTiles>(s, key0 + t * kKeys + 16 * mine, key1,
                             [&](int u, int d, bf16x8(&v)[4]) { v_operands(vb, lane_v, u, d, v); });
  }
  st.finish();
  if constexpr (WK == 2) {
    // The waves of the tiles' second halves hand their state over through LDS.
    struct Hand {
      f32x4 acc[8][64];
      float m[64], l[64], s_abs[64];
    };
    static_assert(sizeof(Hand) * WQ <= 2 * kTileBytes, "one slot per wave handing over");
    Hand* hand = reinterpret_cast<Hand*>(lds_raw) + wq;
    __syncthreads();  // every wave is done with the tiles
    if (live && wk == 1) {
#pragma unroll
      for (int d = 0; d < 8; ++d) hand->acc[d][lane] = st.acc[d];
      hand->m[lane] = st.m;
      hand->l[lane] = st.l;
      hand->s_abs[lane] = st.s_abs;
    }
    __syncthreads();
    if (live && wk == 0) {
      const float kNegInf = -__builtin_inff();
      const float m_new = fmaxf(st.m, hand->m[lane]);
      const float fs = st.m == kNegInf ? 0.f : __builtin_amdgcn_exp2f((st.m - m_new) * kScoreScale);
      const float fo = hand->m[lane] == kNegInf ? 0.f : __builtin_amdgcn_exp2f((hand->m[lane] - m_new) * kScoreScale);
      st.m = m_new;
      st.l = st.l * fs + hand->l[lane] * fo;
      st.s_abs = fmaxf(st.s_abs, hand->s_abs[lane]);
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.acc[d][e] = st.acc[d][e] * fs + hand->acc[d][lane][e] * fo;
    }
  }
  if (live && wk == 0 && vec < nrows * G)
    store_record(rec + ((uint64_t)(vec / G) * a.qh + vec % G) * slots * kRecord, st, a.err);
  if (bad_page != 0 && lane == 0) raise_error(a.err, ERR_PAGE);
}

// A state over some keys: the vector's maximum (in the exponent of 2), its sum and four of its dims.
struct Part {
  float m, l;
  f32x4 n;
};
__device__ __forceinline__ Part no_part() { return Part{-__builtin_inff(), 0.f, f32x4{0.f, 0.f, 0.f, 0.f}}; }
// The union's state with N more: their maximum, then one sum. (One without keys has m = -inf and l = 0.)
template <int N>
__device__ __forceinline__ Part join_all(const Part& t, const Part (&x)[N]) {
  const float kNegInf = -__builtin_inff();
  float m = t.m;
#pragma unroll
  for (int u = 0; u < N; ++u) m = fmaxf(m, x[u].m);
  const float f = t.m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(t.m - m);
  Part o{m, t.l * f, t.n};
#pragma unroll
  for (int e = 0; e < 4; ++e) o.n[e] *= f;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const float w = x[u].m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(x[u].m - m);
    o.l = __builtin_fmaf(x[u].l, w, o.l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o.n[e] = __builtin_fmaf(x[u].n[e], w, o.n[e]);
  }
  return o;
}

// LDS of the narrow form: V of each wave's 32 keys, then the waves' states.
// (Rows of 528 bytes keep the accumulators' stores off each other's banks.)
template <int NW>
struct NarrowState {
  float acc[NW][kVectors][132];
};
static_assert(sizeof(NarrowState<kWaves>) >= 2 * kTileBytes, "and the wide form's tiles fit too");
static_assert(sizeof(NarrowState<1>) >= 32 * 256, "and a wave's V");
template <int NW>
struct NarrowSums {
  float m[NW][kVectors], l[NW][kVectors];  // m in the exponent of 2
};

// The narrow form: as above for nrows * G <= 16 vectors and NW waves; their states are left in LDS, behind a
// barrier.
template <int G, int NW>
__device__ __forceinline__ void attend_narrow(unsigned char* lds_raw, NarrowSums<NW>& sums, const Args& a,
                                              const uint32_t* __restrict__ trow, uint32_t row0, uint32_t nrows,
                                              uint32_t key0, uint32_t key1, uint32_t h) {
  constexpr uint32_t kStep = 32 * NW;  // keys of the waves at once
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  u32x4(*vlds)[16] = reinterpret_cast<u32x4(*)[16]>(lds_raw) + 32 * wave;
  const uint32_t page0 = key0 / 16, npages = (key1 - key0 + 15) / 16, steps = (key1 - key0 + kStep - 1) / kStep;
  // Table entries of this wave's two pages of 32 steps: lane 2 i + u holds page u of step i.
  auto table_chunk = [&](uint32_t step) {
    const uint32_t pi = (step + (lane >> 1)) * (kStep / 16) + 2 * wave + (lane & 1);
    return pi < npages ? trow[page0 + pi] : 0u;
  };
  uint32_t tab = table_chunk(0), bad_page = 0;
  u32x4 qv[4];
  load_q<G>(qv, a, row0, nrows, lane & 15, h);
  uint32_t koff, voff[4];
  koff = (lane & 15) * a.kvh * 256 + 16 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t token = 4 * i + (lane >> 4);
    voff[i] = token * a.kvh * 256 + (((lane & 15) ^ (2 * (token & 7))) & 15) * 16;
  }
  uint32_t lane_v = v_lane(lane);
  State st;
  st.clear();
#pragma unroll 1
  for (uint32_t step = 0; step < steps; ++step) {
    const uint32_t first = step * kStep + 32 * wave;  // key0-relative
    if (first >= key1 - key0) break;  // no more keys for this wave (no barrier in the loop)
    if (step != 0 && step % 32 == 0) tab = table_chunk(step);
    // V first: the wait for K, whose registers the compiler tracks, then covers both kinds of loads.
    u32x4 kr[2][4];
    Page pg[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t pi = first / 16 + u;
      const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)tab, (int)(2 * (step & 31u) + u));
      pg[u] = page_of(a, page, pi < npages ? min(16u, key1 - key0 - pi * 16) : 0u, h, bad_page);
      auto vrs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vc + pg[u].base), 0, pg[u].bytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vrs, (__attribute__((address_space(3))) void*)&vlds[16 * u + 4 * i][0],
                                                 16, voff[i], 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      auto krs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kc + pg[u].base), 0, pg[u].bytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        kr[u][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(krs, koff, 64 * i, 0));
    }
    __builtin_amdgcn_s_waitcnt(0 | (7u << 4) | (15u << 8));
    wave_fence();
    f32x4 s[2];
    s[0] = s[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[u][i]),
                                                       __builtin_bit_cast(bf16x8, qv[i]), s[u], 0, 0, 0);
    asm volatile("" : "+v"(lane_v));  // V's read addresses are made here, not kept beside K
    st.template take<2>(s, key0 + first, key1,
                        [&](int u, int d, bf16x8(&v)[4]) { v_operands((LdsBytes)vlds, lane_v, u, d, v); });
    // The next step's loads overwrite V: this step's reads of it are done.
    __builtin_amdgcn_s_waitcnt(15u | (3u << 14) | (7u << 4) | (0u << 8));
    wave_fence();
  }
  st.finish();
  __syncthreads();  // every wave is done with its V
  auto& all = *reinterpret_cast<NarrowState<NW>*>(lds_raw);
  const uint32_t vec = lane & 15;
  if (vec < nrows * G) {
#pragma unroll
    for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(&all.acc[wave][vec][16 * d + 4 * (lane >> 4)]) = st.acc[d];
    if (lane < 16) {
      sums.m[wave][vec] = st.m * kScoreScale;
      sums.l[wave][vec] = st.l;
    }
    if (st.l != st.l || !(st.s_abs < __builtin_inff())) raise_error(a.err, ERR_NONFINITE);
  }
  if (bad_page != 0 && lane == 0) raise_error(a.err, ERR_PAGE);
  __syncthreads();
}

// The waves' states of vector v, dims 4 c .. 4 c + 3, joined in wave order (the maximum first, then one sum).
template <int NW>
__device__ __forceinline__ Part narrow_part(unsigned char* lds_raw, const NarrowSums<NW>& sums, uint32_t v, uint32_t c) {
  auto& all = *reinterpret_cast<NarrowState<NW>*>(lds_raw);
  Part o = no_part();
#pragma unroll
  for (int w = 0; w < NW; ++w) o.m = fmaxf(o.m, sums.m[w][v]);
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float f = sums.m[w][v] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(sums.m[w][v] - o.m);
    const f32x4 x = *reinterpret_cast<const f32x4*>(&all.acc[w][v][4 * c]);
    o.l += sums.l[w][v] * f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.n[e] += x[e] * f;
  }
  return o;
}

__device__ __forceinline__ uint32_t prefix_of(const Groups& gs, uint32_t r) {
  for (uint32_t i = 0; i < gs.count; ++i)
    if (r - gs.g[i].first_row < gs.g[i].rows) return gs.g[i].prefix_tokens;
  return 0;
}

// First launch: a workgroup takes one chunk of a prefix for a block of rows and a KV
// head (FORM: 0 narrow, 1 and 2 the wide form's WK); its records wait in the
// scratch. The first workgroup clears the counters of the second launch.
template <int G, int FORM>
__global__ __launch_bounds__(kThreads, 4) void prefix_kernel(Args a, const uint32_t* __restrict__ table, uint32_t stride,
                                                             uint32_t items, float* rec, uint32_t* counters,
                                                             uint32_t ncounters, Groups gs) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[sizeof(NarrowState<kWaves>)];
  const uint32_t h = blockIdx.x % a.kvh, item = blockIdx.x / a.kvh;
  if (blockIdx.x == 0 && threadIdx.x < ncounters) counters[threadIdx.x] = 0u;
  if (item >= items) return;
  uint32_t gi = 0;
  while (gi + 1 < gs.count && item >= gs.g[gi + 1].item0) ++gi;
  const Group g = gs.g[gi];
  const uint32_t blocks = (g.rows + gs.block_rows - 1) / gs.block_rows;
  const uint32_t block = (item - g.item0) % blocks, chunk = (item - g.item0) / blocks;
  const uint32_t in = block * gs.block_rows, nrows = min(gs.block_rows, g.rows - in);
  const uint32_t key0 = chunk * gs.chunk, key1 = min(key0 + gs.chunk, g.prefix_tokens);
  const uint32_t row0 = g.first_row + in;
  const uint32_t* trow = table + (uint64_t)row0 * stride;
  rec += (((uint64_t)row0 * a.qh + h * G) * gs.prefix_slots + chunk) * kRecord;
  if constexpr (FORM == 0) {
    __shared__ NarrowSums<kWaves> sums;
    attend_narrow<G, kWaves>(lds_raw, sums, a, trow, row0, nrows, key0, key1, h);
    for (uint32_t idx = threadIdx.x; idx < nrows * G * 32; idx += kThreads) {
      const uint32_t v = idx >> 5, c = idx & 31;
      const Part o = narrow_part(lds_raw, sums, v, c);
      float* r = rec + ((uint64_t)(v / G) * a.qh + v % G) * gs.prefix_slots * kRecord;
      *reinterpret_cast<f32x4*>(r + 4 + 4 * c) = o.n;
      if (c == 0) *reinterpret_cast<float2*>(r) = make_float2(o.m, o.l);
    }
  } else {
    attend_wide<G, FORM>(lds_raw, a, trow, row0, nrows, key0, key1, h, gs.stream != 0, rec, gs.prefix_slots);
  }
  if (h == 0) {
    // The rows of the block list the same pages here as the group's first row.
    const uint32_t p0 = key0 / 16, np = (key1 - key0 + 15) / 16;
    const uint32_t* lead = table + (uint64_t)g.first_row * stride;
    bool differ = false;
    for (uint32_t i = threadIdx.x; i < nrows * np; i += kThreads)
      differ |= table[(uint64_t)(row0 + i / np) * stride + p0 + i % np] != lead[p0 + i % np];
    if (differ) raise_error(a.err, ERR_PAGE);
  }
}

// Second launch: (KV head, row, part) takes a part of the row's own keys, which are
// cut into at most max_parts equal ones of at least part_keys keys, and the first part
// the records of the prefix's chunks too. A row of one part ends here; the parts
// of longer ones leave records, and the last one to arrive (a counter per row and KV
// head, which the first launch cleared) joins them in key order. Records and counter
// go through agent-scope atomics: the XCDs' L2 caches are not coherent with one
// another. As in k_attention.hip this rests on gfx950's lowering of them (stores
// written through, a wait that covers their completion, loads that bypass the L2).
#if defined(__HIP_DEVICE_COMPILE__) && !defined(__gfx950__)
#error "k_attention_prefix.hip: the in-kernel merge is written for gfx950's memory-model lowering"
#endif
template <int G, int NW>
__global__ __launch_bounds__(64 * NW, 4) void own_kernel(Args a, const uint32_t* __restrict__ positions,
                                                          const uint32_t* __restrict__ table, uint32_t rows,
                                                          uint32_t stride, uint32_t context, uint32_t max_parts,
                                                          uint32_t part_keys,
                                                          const float* __restrict__ prefix_rec, float* part_rec,
                                                          uint32_t* counters, uint16_t* __restrict__ out,
                                                          uint32_t out_mtiles, Groups gs) {
  constexpr uint32_t kThreads = 64 * NW, kStep = 32 * NW;
  constexpr uint32_t kDims = G * 32;                // (vector, four dims) pairs
  constexpr uint32_t kTeams = kThreads / kDims;     // threads per pair, for the prefix's records
  constexpr int kInFlight = 4;
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[sizeof(NarrowState<NW>)];
  __shared__ NarrowSums<NW> sums;
  const uint32_t h = blockIdx.x % a.kvh, r = blockIdx.x / a.kvh % rows, part = blockIdx.x / a.kvh / rows;
  const uint32_t pos = uniform(positions[r]), prefix = prefix_of(gs, r);
  if (pos >= context || pos / 16 >= stride || pos + 1 < prefix) {
    if (part == 0 && h == 0 && threadIdx.x == 0) raise_error(a.err, ERR_POSITION);
    return;
  }
  const uint32_t own = pos + 1 - prefix;
  const uint32_t wanted = max(1u, min(max_parts, own / part_keys));
  const uint32_t keys = (own + wanted * kStep - 1) / (wanted * kStep) * kStep;  // of a part
  const uint32_t parts = own > keys ? (own + keys - 1) / keys : 1u;
  if (part >= parts) return;
  const uint32_t v = threadIdx.x % kDims / 32, c = threadIdx.x % 32, team = threadIdx.x / kDims;
  __shared__ f32x4 team_n[kThreads];
  __shared__ float2 team_ml[kTeams][G];
  const uint32_t chunks = part == 0 ? (prefix + gs.chunk - 1) / gs.chunk : 0u;
  if (chunks) {
    // The records of the prefix's chunks, every kTeams-th one, kInFlight at a time: their maximum, then one sum.
    const float* p = prefix_rec + ((uint64_t)r * a.qh + h * G + v) * gs.prefix_slots * kRecord;
    Part t = no_part();
    for (uint32_t i0 = team; i0 < chunks; i0 += kTeams * kInFlight) {
      Part x[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const float* s = p + (uint64_t)min(i0 + u * kTeams, chunks - 1) * kRecord;
        const float2 ml = *reinterpret_cast<const float2*>(s);
        x[u] = Part{ml.x, ml.y, *reinterpret_cast<const f32x4*>(s + 4 + 4 * c)};
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
        if (i0 + u * kTeams >= chunks) x[u].m = -__builtin_inff();
      t = join_all(t, x);
    }
    team_n[threadIdx.x] = t.n;
    if (c == 0) team_ml[team][v] = make_float2(t.m, t.l);
  }
  const uint32_t key0 = prefix + part * keys, key1 = min(key0 + keys, pos + 1);
  attend_narrow<G, NW>(lds_raw, sums, a, table + (uint64_t)r * stride, r, 1, key0, key1, h);
  const bool mine = threadIdx.x < kDims;
  Part o = no_part();
  if (mine) {
    o = narrow_part(lds_raw, sums, v, c);
    if (chunks) {
      Part x[kTeams];
#pragma unroll
      for (uint32_t t = 0; t < kTeams; ++t)
        x[t] = Part{team_ml[t][v].x, team_ml[t][v].y, team_n[t * kDims + threadIdx.x]};
      o = join_all(o, x);
    }
  }
  if (parts > 1) {
    __shared__ uint32_t last;
    float* to = part_rec + (((uint64_t)r * a.kvh + h) * max_parts * G + v) * kRecord;
    if (mine) {
      float* x = to + (uint64_t)part * G * kRecord;
      if (c == 0) {
        __hip_atomic_store(x, o.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(x + 1, o.l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        __hip_atomic_store(x + 4 + 4 * c + e, o.n[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(counters + (uint64_t)r * a.kvh + h, 1u) == parts - 1 ? 1u : 0u;
    __syncthreads();
    if (!last) return;
    if (mine) {
      o = no_part();
      for (uint32_t i = 0; i < parts; ++i) {
        const float* x = to + (uint64_t)i * G * kRecord;
        Part y[1];
        y[0].m = __hip_atomic_load(x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        y[0].l = __hip_atomic_load(x + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[0].n[e] = __hip_atomic_load(x + 4 + 4 * c + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        o = join_all(o, y);
      }
    }
  }
  if (!mine) return;
  const uint32_t w0 = pack_bf16x2(o.n[0] / o.l, o.n[1] / o.l), w1 = pack_bf16x2(o.n[2] / o.l, o.n[3] / o.l);
  const uint32_t col = (h * G + v) * 128 + 4 * c;
  uint16_t* dst = out_mtiles ? out + act_offset_m(r, col, out_mtiles) : out + (uint64_t)r * a.qh * 128 + col;
  *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
  auto inf = [](uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; };
  if (!(o.l > 0.f) || inf(w0) || inf(w1)) raise_error(a.err, ERR_NONFINITE);
}

// The launches' work split: a rule on the groups, heads and numbers of rows alone, so
// that the scratch's size and the launch agree.
struct PrefixPlan {
  Groups gs;
  uint32_t items, form, max_parts, part_keys, own_waves, counters;
  uint64_t prefix_floats, part_floats;  // of the records
};

// (context: an upper bound of the positions, for the own keys' form alone; the scratch does not depend on it.)
PrefixPlan prefix_plan(const fh_prefix_group* groups, uint32_t ngroups, uint32_t rows, uint32_t qh, uint32_t kvh,
                       uint32_t context) {
  PrefixPlan p{};
  const uint32_t g = qh / kvh;
  uint32_t most = 0, longest = 0, shortest = context, grouped = 0;
  for (uint32_t i = 0; i < ngroups; ++i) {
    if (groups[i].prefix_pages == 0) continue;
    Group& to = p.gs.g[p.gs.count++];
    to = Group{groups[i].first_row, groups[i].rows, groups[i].prefix_pages * 16, 0};
    if (to.rows > most) most = to.rows;
    if (to.prefix_tokens > longest) longest = to.prefix_tokens;
    if (to.prefix_tokens < shortest) shortest = to.prefix_tokens;
    grouped += to.rows;
  }
  if (grouped < rows) shortest = 0;
  const uint64_t vectors = (uint64_t)most * g;
  if (most == 0) most = 1;
  // Tokens times blocks times KV heads with blocks of `rows` rows.
  auto tokens_of = [&](uint32_t rows) {
    uint64_t tokens = 0;
    for (uint32_t i = 0; i < p.gs.count; ++i)
      tokens += (uint64_t)p.gs.g[i].prefix_tokens * ((p.gs.g[i].rows + rows - 1) / rows) * kvh;
    return tokens;
  };
  // Blocks of 64 vectors unless the prefixes are long: 32 rows of 4 heads behind 8192 tokens 26.4 us
  // (29.8 in blocks of 128, whose waves take whole tiles), but 160 rows behind 4096 tokens 49.7 us (47.5 in
  // blocks of 128, which read the keys half as often) and 32 behind 32000 69.4 (61.7).
  p.form = vectors > kVectors ? 2 : 0;
  if (vectors > 64 && tokens_of(128 / g) / kChunkWgs >= 512) p.form = 1;
  p.gs.block_rows = (p.form == 1 ? 128 : p.form == 2 ? 64 : kVectors) / g;
  p.gs.stream = most <= p.gs.block_rows && tokens_of(most) * 512 >= kStreamBytes;
  uint64_t chunk = (tokens_of(p.gs.block_rows) / kChunkWgs + 63) / 64 * 64;
  if (chunk > longest) chunk = (longest + 63) / 64 * 64;  // (many rows and heads: tokens_of may pass 2^40)
  if (chunk < kMinChunk) chunk = kMinChunk;
  p.gs.chunk = (uint32_t)chunk;
  for (uint32_t i = 0; i < p.gs.count; ++i) {
    Group& to = p.gs.g[i];
    const uint32_t chunks = (to.prefix_tokens + p.gs.chunk - 1) / p.gs.chunk;
    to.item0 = p.items;
    p.items += chunks * ((to.rows + p.gs.block_rows - 1) / p.gs.block_rows);
    if (chunks > p.gs.prefix_slots) p.gs.prefix_slots = chunks;
  }
  // Parts of the own keys: what fills the slots; one where the rows and heads do.
  const uint64_t pairs = (uint64_t)rows * kvh;
  p.max_parts = pairs >= kSlots ? 1 : (uint32_t)(kSlots / pairs) < kMaxParts ? (uint32_t)(kSlots / pairs) : kMaxParts;
  p.part_keys = pairs > kManyPairs ? kPartKeysMany : kPartKeysFew;
  p.own_waves = pairs >= kManyOwn && context - shortest <= kShortOwn ? 4 : 8;
  p.counters = p.max_parts > 1 ? (uint32_t)pairs : 0;
  p.prefix_floats = (uint64_t)rows * qh * p.gs.prefix_slots * kRecord;
  p.part_floats = p.max_parts > 1 ? (uint64_t)rows * qh * p.max_parts * kRecord : 0;
  return p;
}

}  // namespace

uint64_t prefix_scratch_bytes(const fh_prefix_group* groups, uint32_t ngroups, uint32_t rows, uint32_t qh, uint32_t kvh) {
  const PrefixPlan p = prefix_plan(groups, ngroups, rows, qh, kvh, 0);
  return (p.prefix_floats + p.part_floats + p.counters + 4) * 4;  // never nothing
}

hipError_t launch_prefix_attention(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                   const uint32_t* positions, const uint32_t* table, const fh_prefix_group* groups,
                                   uint32_t ngroups, uint16_t* out, uint32_t out_tiled, void* scratch, uint32_t rows,
                                   uint32_t qh, uint32_t kvh, uint32_t stride, uint32_t pages, uint32_t context,
                                   uint32_t* err, hipStream_t s) {
  const PrefixPlan p = prefix_plan(groups, ngroups, rows, qh, kvh, context);
  float* prefix_rec = reinterpret_cast<float*>(scratch);
  float* part_rec = prefix_rec + p.prefix_floats;
  uint32_t* counters = reinterpret_cast<uint32_t*>(part_rec + p.part_floats);
  const Args a{q, k_cache, v_cache, qh, kvh, pages, err};
  const uint32_t mt = out_tiled ? act_mtiles(rows) : 0u;
  const uint32_t prefix_wgs = p.items ? p.items * kvh : p.counters ? 1 : 0;
#define FH_PREFIX_FORM(G_, FORM_)                                                                                      \
  hipLaunchKernelGGL((prefix_kernel<G_, FORM_>), dim3(prefix_wgs), dim3(kThreads), 0, s, a, table, stride, p.items, \
                     prefix_rec, counters, p.counters, p.gs)
#define FH_PREFIX_OWN(G_, NW_)                                                                                      \
  hipLaunchKernelGGL((own_kernel<G_, NW_>), dim3(kvh * rows * p.max_parts), dim3(64 * NW_), 0, s, a, positions, table, \
                     rows, stride, context, p.max_parts, p.part_keys, prefix_rec, part_rec, counters, out, mt, p.gs)
#define FH_PREFIX(G_)                                                                                               \
  do {                                                                                                              \
    if (prefix_wgs) {                                                                                               \
      if (p.form == 1)                                                                                              \
        FH_PREFIX_FORM(G_, 1);                                                                                      \
      else if (p.form == 2)                                                                                         \
        FH_PREFIX_FORM(G_, 2);                                                                                      \
      else                                                                                                          \
        FH_PREFIX_FORM(G_, 0);                                                                                      \
    }                                                                                                               \
    if (p.own_waves == 4)                                                                                           \
      FH_PREFIX_OWN(G_, 4);                                                                                         \
    else                                                                                                            \
      FH_PREFIX_OWN(G_, 8);                                                                                         \
  } while (0)
  switch (qh / kvh) {
    case 1: FH_PREFIX(1); break;
    case 2: FH_PREFIX(2); break;
    case 4: FH_PREFIX(4); break;
    case 8: FH_PREFIX(8); break;
    default: return hipErrorInvalidValue;
  }
#undef FH_PREFIX
#undef FH_PREFIX_FORM
#undef FH_PREFIX_OWN
  return hipGetLastError();
}

}  // namespace fh
