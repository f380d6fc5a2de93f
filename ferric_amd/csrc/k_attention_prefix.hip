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
// at once) or a unit of a row's own keys; states are FP32 records in the
// scratch, merged in ascending key order by a second launch.
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
// Two forms share the launch. Wide (prefix chunks of more than 16 vectors): the 8
// waves share 64-key tiles of K and V, fetched global -> LDS directly, double-
// buffered; 8 waves of vectors, or 4 with two of them sharing the tile's keys.
// Narrow (own keys, and prefix chunks of up to 16 vectors): the waves take 32 keys
// each, K straight into the A operand's registers (a token's 64-byte pieces), V
// through 8 KiB of LDS of the wave's own; their states meet in LDS at the end.
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
constexpr int kStep = 32 * kWaves;    // keys of the narrow form's waves at once
constexpr size_t kTileBytes = 16 * 2 * kKeys * 16;  // K or V, double-buffered
constexpr uint32_t kMinChunk = 256;   // least tokens of a prefix chunk
constexpr uint32_t kOwnUnits = 256;   // own keys are cut into about this many units
constexpr uint32_t kOwnWgs = 256;     // workgroups that take them
// f32(0x3db504f3) (1/sqrt(128), paged_decode.rs:31-35) times log2 e.
constexpr float kScoreScale = 0.08838834764831845f * 1.44269504088896341f;
constexpr uint32_t kRecord = 132;     // m, l, two unused, n[128]: 16-byte aligned

struct Group {
  uint32_t first_row, rows, prefix_tokens;
  uint32_t item0;  // its first prefix item: vector block + blocks * chunk
};
struct Groups {
  uint32_t count, chunk, block_rows, prefix_slots;
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

  // Takes in T tiles of 16 scores: keys first + 16 t + 4 (lane / 16) + e below `end`. v_at(t, d): the V^T
  // operand of tiles t, t + 1 (t even) for dims 16 d .. + 15.
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
        pl[e] = pack_bf16x2(p[2 * e] - lo_bf16(ph[e]), p[2 * e + 1] - hi_bf16(ph[e]));
      }
      const bf16x8 bh = __builtin_bit_cast(bf16x8, u32x4{ph[0], ph[1], ph[2], ph[3]});
      const bf16x8 bl = __builtin_bit_cast(bf16x8, u32x4{pl[0], pl[1], pl[2], pl[3]});
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const bf16x8 va = v_at(t, d);
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, bh, acc[d], 0, 0, 0);
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, bl, acc[d], 0, 0, 0);
      }
    }
  }

  // The vector's sum in every lane group.
  __device__ __forceinline__ void finish() {
    l = group_sum(l);
    s_abs = group_max(s_abs);
  }
};

// Transposing reads of V^T from LDS rows of tokens (u32x4[16] each): keys 16 t + 4 (lane / 16) + 0..3 of
// tiles t and t + 1, dims 16 d .. + 15.
__device__ __forceinline__ bf16x8 v_operand(const u32x4 (*rows)[16], int t, int d) {
  const int lane = threadIdx.x & 63;
  const uint32_t j = lane & 15, key = 4 * (lane >> 4) + (j >> 2);
  u32x2 v[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const uint32_t k = 16 * (t + u) + key, c = (2 * d + ((j & 3) >> 1)) ^ (2 * (key & 7));
    auto* src = reinterpret_cast<u32x2*>(const_cast<u32x4*>(&rows[k][c])) + (j & 1);
    v[u] = __builtin_bit_cast(u32x2,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)src));
  }
  return __builtin_bit_cast(bf16x8, u32x4{v[0][0], v[0][1], v[1][0], v[1][1]});
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
// multiple of 16. WK waves share a tile's keys, 8 / WK own the vectors. rec: record of (row 0, head 0), row
// and head steps of `slots` records.
template <int G, int WK>
__device__ __forceinline__ void attend_wide(unsigned char* lds_raw, const Args& a, const uint32_t* __restrict__ trow,
                                            uint32_t row0, uint32_t nrows, uint32_t key0, uint32_t key1, uint32_t h,
                                            float* rec, uint32_t slots) {
  constexpr int WQ = kWaves / WK, kTiles = kKeys / 16 / WK;  // 16-key tiles a wave takes of each 64
  auto& klds = *reinterpret_cast<u32x4(*)[2][kKeys][16]>(lds_raw);
  auto& vlds = *reinterpret_cast<u32x4(*)[2][kKeys][16]>(lds_raw + kTileBytes);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wq = wave % WQ, wk = wave / WQ;
  const uint32_t page0 = key0 / 16, npages = (key1 - key0 + 15) / 16, tiles = (key1 - key0 + kKeys - 1) / kKeys;
  // Page-table entries of 64 pages, one per lane, the next 64 requested ahead.
  auto table_chunk = [&](uint32_t first) { return first + lane < npages ? trow[page0 + first + lane] : 0u; };
  uint32_t tab = table_chunk(0), tab_next = table_chunk(64);
  // Waves 0..3 copy K of the tile's pages 0..3, waves 4..7 V: four tokens per load (lane: token 4 i + lane /
  // 16, LDS chunk lane % 16).
  const int my_page = wave & 3;
  const bool is_v = wave >= 4;
  uint32_t off[4], bad_page = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t token = 4 * i + (lane >> 4), swizzle = is_v ? 2 * (token & 7) : token;
    off[i] = token * a.kvh * 256 + (((lane & 15) ^ swizzle) & 15) * 16;
  }
  auto fetch = [&](uint32_t t, int buf) {
    const uint32_t pi = 4 * t + my_page;
    const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)tab, (int)(pi & 63u));
    const Page p = page_of(a, page, pi < npages ? min(16u, key1 - key0 - pi * 16) : 0u, h, bad_page);
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)((is_v ? a.vc : a.kc) + p.base), 0, p.bytes, 0x00020000);
    u32x4(*to)[16] = is_v ? vlds[buf] : klds[buf];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)&to[16 * my_page + 4 * i][0], 16, off[i], 0, 0, 0);
  };
  fetch(0, 0);
  const uint32_t vec = 16 * wq + (lane & 15);
  const bool live = (uint32_t)(16 * wq) < nrows * G;  // a wave with no vectors only fetches
  u32x4 qv[4];
  load_q<G>(qv, a, row0, nrows, vec, h);
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
      fetch(t + 1, (t + 1) & 1);
    }
    if (!live) continue;
    const int buf = t & 1, mine = kTiles * wk;
    f32x4 s[kTiles];
#pragma unroll
    for (int u = 0; u < kTiles; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 ka = klds[buf][16 * (mine + u) + (lane & 15)][(4 * i + (lane >> 4)) ^ (lane & 15)];
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ka), __builtin_bit_cast(bf16x8, qv[i]),
                                                       s[u], 0, 0, 0);
      }
    }
    st.template take<kTiles>(s, key0 + t * kKeys + 16 * mine, key1,
                             [&](int u, int d) { return v_operand(&vlds[buf][16 * mine], u, d); });
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

// LDS of the narrow form: V of each wave's 32 keys, then the waves' states.
struct NarrowState {
  float acc[kWaves][16][128];
};
static_assert(sizeof(NarrowState) == 2 * kTileBytes, "the states of 8 waves fill the tiles' LDS");

// The narrow form: as above for nrows * G <= 16 vectors. The record of vector v is rec + (v / G) * row_step +
// (v % G) * head_step.
template <int G>
__device__ __forceinline__ void attend_narrow(unsigned char* lds_raw, const Args& a, const uint32_t* __restrict__ trow,
                                              uint32_t row0, uint32_t nrows, uint32_t key0, uint32_t key1, uint32_t h,
                                              float* rec, uint64_t row_step, uint64_t head_step) {
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
  State st;
  st.clear();
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
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[u][i]),
                                                       __builtin_bit_cast(bf16x8, qv[i]), s[u], 0, 0, 0);
    }
    st.template take<2>(s, key0 + first, key1, [&](int u, int d) { return v_operand(vlds, u, d); });
    // The next step's loads overwrite V: this step's reads of it are done.
    __builtin_amdgcn_s_waitcnt(15u | (3u << 14) | (7u << 4) | (0u << 8));
    wave_fence();
  }
  st.finish();
  // The waves' states meet in LDS, the waves in order (one without keys has l = 0 and m = -inf).
  __shared__ float wm[kWaves][16], wl[kWaves][16];
  __syncthreads();  // every wave is done with its V
  auto& all = *reinterpret_cast<NarrowState*>(lds_raw);
  const uint32_t vec = lane & 15, nvec = nrows * G;
  if (vec < nvec) {
#pragma unroll
    for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(&all.acc[wave][vec][16 * d + 4 * (lane >> 4)]) = st.acc[d];
    if (lane < 16) {
      wm[wave][vec] = st.m * kScoreScale;
      wl[wave][vec] = st.l;
    }
    if (st.l != st.l || !(st.s_abs < __builtin_inff())) raise_error(a.err, ERR_NONFINITE);
  }
  if (bad_page != 0 && lane == 0) raise_error(a.err, ERR_PAGE);
  __syncthreads();
  for (uint32_t idx = threadIdx.x; idx < nvec * 32; idx += kThreads) {
    const uint32_t v = idx >> 5, c = idx & 31;  // four dims
    float M = wm[0][v];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, wm[w][v]);
    f32x4 n = f32x4{0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = wl[w][v] > 0.f ? __builtin_amdgcn_exp2f(wm[w][v] - M) : 0.f;
      const f32x4 x = *reinterpret_cast<const f32x4*>(&all.acc[w][v][4 * c]);
      L += wl[w][v] * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) n[e] += x[e] * f;
    }
    float* r = rec + (v / G) * row_step + (v % G) * head_step;
    *reinterpret_cast<f32x4*>(r + 4 + 4 * c) = n;
    if (c == 0) {
      r[0] = M;
      r[1] = L;
    }
  }
}

__device__ __forceinline__ uint32_t prefix_of(const Groups& gs, uint32_t r) {
  for (uint32_t i = 0; i < gs.count; ++i)
    if (r - gs.g[i].first_row < gs.g[i].rows) return gs.g[i].prefix_tokens;
  return 0;
}

// Pages of row r's own keys; 0 where the row is not computed.
__device__ __forceinline__ uint32_t own_pages(const uint32_t* positions, const Groups& gs, uint32_t r, uint32_t context,
                                              uint32_t stride, bool& bad) {
  const uint32_t pos = positions[r], prefix = prefix_of(gs, r);
  if (pos >= context || pos / 16 >= stride || pos + 1 < prefix) {
    bad = true;
    return 0;
  }
  return (pos + 1 - prefix + 15) / 16;
}

// Workgroups [0, prefix_wgs): one chunk of a prefix for a block of rows and a
// KV head (FORM: 0 narrow, 1 and 2 the wide form's WK). The others share the
// rows' own keys, cut into units of a number of pages that is a rule on the
// positions' total: every workgroup counts them for itself, takes units own, own
// + own_wgs, ... of each KV head, and the first one writes each row's first unit
// to `first` for the merge.
template <int G, int FORM>
__global__ __launch_bounds__(kThreads, 4) void prefix_kernel(Args a, const uint32_t* __restrict__ positions,
                                                             const uint32_t* __restrict__ table, uint32_t rows,
                                                             uint32_t stride, uint32_t context, uint32_t prefix_wgs,
                                                             uint32_t own_wgs, float* prefix_rec, float* own_rec,
                                                             uint32_t* first, Groups gs) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[2 * kTileBytes];
  const uint32_t kvh = a.kvh;
  if (blockIdx.x < prefix_wgs) {
    const uint32_t h = blockIdx.x % kvh, item = blockIdx.x / kvh;
    uint32_t gi = 0;
    while (gi + 1 < gs.count && item >= gs.g[gi + 1].item0) ++gi;
    const Group g = gs.g[gi];
    const uint32_t blocks = (g.rows + gs.block_rows - 1) / gs.block_rows;
    const uint32_t block = (item - g.item0) % blocks, chunk = (item - g.item0) / blocks;
    const uint32_t in = block * gs.block_rows, nrows = min(gs.block_rows, g.rows - in);
    const uint32_t key0 = chunk * gs.chunk, key1 = min(key0 + gs.chunk, g.prefix_tokens);
    const uint32_t row0 = g.first_row + in;
    if (h == 0) {
      // The rows of the block list the same pages here as the group's first row.
      const uint32_t p0 = key0 / 16, np = (key1 - key0 + 15) / 16;
      const uint32_t* lead = table + (uint64_t)g.first_row * stride;
      bool differ = false;
      for (uint32_t i = threadIdx.x; i < nrows * np; i += kThreads)
        differ |= table[(uint64_t)(row0 + i / np) * stride + p0 + i % np] != lead[p0 + i % np];
      if (differ) raise_error(a.err, ERR_PAGE);
    }
    const uint32_t* trow = table + (uint64_t)row0 * stride;
    float* rec = prefix_rec + (((uint64_t)row0 * a.qh + h * G) * gs.prefix_slots + chunk) * kRecord;
    if constexpr (FORM == 0)
      attend_narrow<G>(lds_raw, a, trow, row0, nrows, key0, key1, h, rec, (uint64_t)a.qh * gs.prefix_slots * kRecord,
                       (uint64_t)gs.prefix_slots * kRecord);
    else
      attend_wide<G, FORM>(lds_raw, a, trow, row0, nrows, key0, key1, h, rec, gs.prefix_slots);
    return;
  }
  const uint32_t own = blockIdx.x - prefix_wgs;
  __shared__ uint32_t scan[kThreads];
  __shared__ uint32_t wave_total[2][kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t turn = 0;
  // Sum over the workgroup (every thread gets it) and the sum up to this thread.
  auto block_scan = [&](uint32_t v, uint32_t& total) {
    uint32_t sum = v;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const uint32_t up = __shfl_up(sum, off, 64);
      if (lane >= off) sum += up;
    }
    uint32_t* t = wave_total[turn ^= 1];  // the other one may still be read
    if (lane == 63) t[wave] = sum;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t x = t[w];
      if (w < wave) sum += x;
      total += x;
    }
    total = uniform(total);
    return sum;
  };
  uint64_t all = 0;
  bool bad = false;
  uint32_t pages0 = 0;  // of this thread's row below kThreads
  for (uint32_t r0 = 0; r0 < rows; r0 += kThreads) {
    const uint32_t r = r0 + threadIdx.x;
    const uint32_t n = r < rows ? own_pages(positions, gs, r, context, stride, bad) : 0u;
    if (r0 == 0) pages0 = n;
    uint32_t total;
    block_scan(n, total);
    all += total;
  }
  if (bad && own == 0) raise_error(a.err, ERR_POSITION);
  // (The cap is beyond any row: one unit each.)
  constexpr uint32_t kStepPages = kStep / 16;
  const uint32_t unit_pages = (uint32_t)min((all * kvh / kOwnUnits + kStepPages) / kStepPages * kStepPages, (uint64_t)1 << 24);
  uint32_t base = 0;    // units of the rows before r0
  uint32_t next = own;  // this workgroup's next (unit, head)
  for (uint32_t r0 = 0; r0 < rows; r0 += kThreads) {
    const uint32_t r = r0 + threadIdx.x;
    const uint32_t n = r0 == 0 ? pages0 : r < rows ? own_pages(positions, gs, r, context, stride, bad) : 0u;
    const uint32_t mine = (n + unit_pages - 1) / unit_pages;
    uint32_t total;
    const uint32_t upto = block_scan(mine, total);
    scan[threadIdx.x] = upto;
    if (own == 0 && r < rows) {
      first[r] = base + upto - mine;
      if (r == rows - 1) first[rows] = base + upto;
    }
    __syncthreads();
    for (; next < (base + total) * kvh; next += own_wgs) {
      const uint32_t unit = next / kvh - base, h = next % kvh;
      uint32_t lo = 0, hi = kThreads - 1;  // the first row whose units end after this one
      while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (scan[mid] > unit)
          hi = mid;
        else
          lo = mid + 1;
      }
      const uint32_t row = uniform(r0 + lo), before = lo ? scan[lo - 1] : 0u;
      const uint32_t prefix = prefix_of(gs, row), end = uniform(positions[row]) + 1;
      const uint32_t key0 = uniform(prefix + (unit - before) * unit_pages * 16), key1 = min(key0 + unit_pages * 16, end);
      attend_narrow<G>(lds_raw, a, table + (uint64_t)row * stride, row, 1, key0, key1, h,
                       own_rec + (uint64_t)next * G * kRecord, 0, kRecord);
      __syncthreads();
    }
    base += total;
    __syncthreads();
  }
}

// One wave per (row, query head): its records in ascending key order, the
// prefix's chunks and then its own units. Up to 64 records at a time: lane i
// holds record i's weight, then every lane its two dims of eight records at once.
__global__ __launch_bounds__(256) void prefix_merge_kernel(const float* __restrict__ prefix_rec,
                                                          const float* __restrict__ own_rec,
                                                          const uint32_t* __restrict__ first,
                                                          const uint32_t* __restrict__ positions,
                                                          uint16_t* __restrict__ out, uint32_t out_mtiles, uint32_t rows,
                                                          uint32_t qh, uint32_t kvh, uint32_t stride, uint32_t context,
                                                          uint32_t* err, Groups gs) {
  const int lane = threadIdx.x & 63;
  const uint32_t id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = id / qh, head = id % qh;
  if (r >= rows) return;
  const uint32_t pos = positions[r], prefix = prefix_of(gs, r);
  if (pos >= context || pos / 16 >= stride || pos + 1 < prefix) return;  // reported by the own keys' part
  const uint32_t u0 = first[r], np = (prefix + gs.chunk - 1) / gs.chunk, n = np + first[r + 1] - u0;
  const uint32_t g = qh / kvh;
  const float* pp = prefix_rec + (uint64_t)id * gs.prefix_slots * kRecord;
  const float* po = own_rec + (((uint64_t)u0 * kvh + head / g) * g + head % g) * kRecord;
  const uint64_t ostep = (uint64_t)kvh * g * kRecord;
  auto record = [&](uint32_t i) { return i < np ? pp + (uint64_t)i * kRecord : po + (i - np) * ostep; };
  float M = -__builtin_inff();
  for (uint32_t i = lane; i < n; i += 64) M = fmaxf(M, record(i)[0]);
  M = wave_max(M);
  float L = 0.f, n0 = 0.f, n1 = 0.f;
  for (uint32_t c0 = 0; c0 < n; c0 += 64) {
    const uint32_t mine = min(c0 + lane, n - 1);
    const float w = c0 + lane < n ? __builtin_amdgcn_exp2f(record(mine)[0] - M) : 0.f;
    const float lw = w * record(mine)[1];
    L += wave_sum(lw);
    const uint32_t cn = min(64u, n - c0);
    for (uint32_t s0 = 0; s0 < cn; s0 += 8) {
      float a0[8], a1[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float2 v = *reinterpret_cast<const float2*>(record(c0 + min(s0 + u, cn - 1)) + 4 + 2 * lane);
        a0[u] = v.x;
        a1[u] = v.y;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float f = s0 + u < cn ? lane_bcast(w, (int)(s0 + u)) : 0.f;
        n0 = __builtin_fmaf(a0[u], f, n0);
        n1 = __builtin_fmaf(a1[u], f, n1);
      }
    }
  }
  const uint32_t o0 = f32_to_bf16(n0 / L), o1 = f32_to_bf16(n1 / L);
  const uint32_t col = head * 128 + 2 * lane;
  uint16_t* dst = out_mtiles ? out + act_offset_m(r, col, out_mtiles) : out + (uint64_t)r * qh * 128 + col;
  *reinterpret_cast<uint32_t*>(dst) = o0 | (o1 << 16);
  if (!(L > 0.f) || ((o0 & 0x7f80u) == 0x7f80u) || ((o1 & 0x7f80u) == 0x7f80u)) raise_error(err, ERR_NONFINITE);
}

// The launch's work split: a rule on the groups, heads and lengths alone, so
// that the scratch's size and the launch agree.
struct PrefixPlan {
  Groups gs;
  uint32_t items, form, own_wgs;
  uint64_t prefix_floats, own_floats;  // of the records
};

PrefixPlan prefix_plan(const fh_prefix_group* groups, uint32_t ngroups, uint32_t rows, uint32_t qh, uint32_t kvh) {
  PrefixPlan p{};
  const uint32_t g = qh / kvh;
  uint32_t most = 0;
  for (uint32_t i = 0; i < ngroups; ++i) {
    if (groups[i].prefix_pages == 0) continue;
    Group& to = p.gs.g[p.gs.count++];
    to = Group{groups[i].first_row, groups[i].rows, groups[i].prefix_pages * 16, 0};
    if (to.rows > most) most = to.rows;
  }
  const uint64_t vectors = (uint64_t)most * g;
  p.form = vectors > 64 ? 1 : vectors > 16 ? 2 : 0;
  p.gs.block_rows = (p.form == 1 ? 128 : p.form == 2 ? 64 : 16) / g;
  // Two workgroups per CU over the prefixes, of at least kMinChunk tokens.
  uint64_t tokens = 0;
  for (uint32_t i = 0; i < p.gs.count; ++i)
    tokens += (uint64_t)p.gs.g[i].prefix_tokens * ((p.gs.g[i].rows + p.gs.block_rows - 1) / p.gs.block_rows) * kvh;
  uint64_t chunk = (tokens / 512 + kKeys - 1) / kKeys * kKeys;
  if (chunk < kMinChunk) chunk = kMinChunk;
  p.gs.chunk = (uint32_t)chunk;
  for (uint32_t i = 0; i < p.gs.count; ++i) {
    Group& to = p.gs.g[i];
    const uint32_t chunks = (to.prefix_tokens + p.gs.chunk - 1) / p.gs.chunk;
    to.item0 = p.items;
    p.items += chunks * ((to.rows + p.gs.block_rows - 1) / p.gs.block_rows);
    if (chunks > p.gs.prefix_slots) p.gs.prefix_slots = chunks;
  }
  p.own_wgs = kOwnWgs;
  p.prefix_floats = (uint64_t)rows * qh * p.gs.prefix_slots * kRecord;
  // Units: a row's last one may be short, the others hold at least all / kOwnUnits pages and heads.
  p.own_floats = ((uint64_t)kOwnUnits + kvh + (uint64_t)rows * kvh) * g * kRecord;
  return p;
}

}  // namespace

uint64_t prefix_scratch_bytes(const fh_prefix_group* groups, uint32_t ngroups, uint32_t rows, uint32_t qh, uint32_t kvh) {
  const PrefixPlan p = prefix_plan(groups, ngroups, rows, qh, kvh);
  return (p.prefix_floats + p.own_floats + rows + 1) * 4;
}

hipError_t launch_prefix_attention(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                   const uint32_t* positions, const uint32_t* table, const fh_prefix_group* groups,
                                   uint32_t ngroups, uint16_t* out, uint32_t out_tiled, void* scratch, uint32_t rows,
                                   uint32_t qh, uint32_t kvh, uint32_t stride, uint32_t pages, uint32_t context,
                                   uint32_t* err, hipStream_t s) {
  const PrefixPlan p = prefix_plan(groups, ngroups, rows, qh, kvh);
  float* prefix_rec = reinterpret_cast<float*>(scratch);
  float* own_rec = prefix_rec + p.prefix_floats;
  uint32_t* first = reinterpret_cast<uint32_t*>(own_rec + p.own_floats);
  const uint32_t prefix_wgs = p.items * kvh;
  const Args a{q, k_cache, v_cache, qh, kvh, pages, err};
#define FH_PREFIX_FORM(G_, FORM_)                                                                                 \
  hipLaunchKernelGGL((prefix_kernel<G_, FORM_>), dim3(prefix_wgs + p.own_wgs), dim3(kThreads), 0, s, a, positions, \
                     table, rows, stride, context, prefix_wgs, p.own_wgs, prefix_rec, own_rec, first, p.gs)
#define FH_PREFIX(G_)            \
  do {                           \
    if (p.form == 1)             \
      FH_PREFIX_FORM(G_, 1);     \
    else if (p.form == 2)        \
      FH_PREFIX_FORM(G_, 2);     \
    else                         \
      FH_PREFIX_FORM(G_, 0);     \
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
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint64_t waves = (uint64_t)rows * qh;
  hipLaunchKernelGGL(prefix_merge_kernel, dim3((waves + 3) / 4), dim3(256), 0, s, prefix_rec, own_rec, first, positions,
                     out, out_tiled ? act_mtiles(rows) : 0u, rows, qh, kvh, stride, context, err, p.gs);
  return hipGetLastError();
}

}  // namespace fh
