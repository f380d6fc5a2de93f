// K4 for batches whose rows share a prefix (continuations of one prompt): the
// prefix's keys and values are read once for all rows of a group, each row's
// own ones once for the row.
//
// Contract of k_attention.hip: for a query row at position p, keys t = 0..p
// through the row's page table, score = (q . k_t) * f32(0x3db504f3), softmax,
// out = bf16(n / l). Attention over a union of key sets is the merge of the
// states over each: with (m_i, l_i, n_i) = (max s, sum e^(s - m_i), sum
// e^(s - m_i) v), M = max m_i, out = sum n_i e^(m_i - M) / sum l_i e^(m_i - M).
// A state covers a chunk of the prefix (for 128 / G, 64 / G or 32 / G rows at
// once) or of a row's own keys; states are FP32 records in the scratch, merged
// in ascending key order by a second launch.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace fh {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kKeys = 64;                      // keys per tile of a prefix chunk
constexpr int kPages = kKeys / 16;             // pages per tile
constexpr size_t kTileBytes = 16 * 2 * kKeys * 16;  // K or V, double-buffered
constexpr uint32_t kOwnPages = 16;             // pages of a row's own keys the waves take at once
constexpr uint32_t kMinChunk = 256;            // least tokens of a prefix chunk
constexpr uint32_t kOwnUnits = 512;            // own keys are cut into about this many units
// f32(0x3db504f3) (1/sqrt(128), paged_decode.rs:31-35) times log2 e.
constexpr float kScoreScale = 0.08838834764831845f;
constexpr float kLog2e = 1.44269504088896341f;
constexpr uint32_t kRecord = 132;  // m, l, two unused, n[128]: 16-byte aligned

struct Group {
  uint32_t first_row, rows, prefix_tokens;
  uint32_t item0;  // its first prefix item: vector block + blocks * chunk
};
struct Groups {
  uint32_t count, chunk, block_rows, prefix_slots;
  Group g[kPrefixMaxGroups];
};

// One state of nrows rows (consecutive from row0, sharing row0's table) over
// keys [key0, key1), key0 a multiple of 16, for KV head h: the records of chunk
// `slot`. WQ waves along the vectors (32 each), WK along the keys.
template <int G, int WQ, int WK>
__device__ __forceinline__ void attend_prefix(unsigned char* lds_raw, const uint16_t* __restrict__ q,
                                              const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
                                              const uint32_t* __restrict__ trow, uint32_t row0, uint32_t nrows,
                                              uint32_t key0, uint32_t key1, uint32_t h, uint32_t qh, uint32_t kvh,
                                              uint32_t pages, float* rec, uint32_t slots, uint32_t slot, uint32_t* err) {
  constexpr int kGroups = kKeys / 32 / WK;       // 32-key groups per wave and tile
  constexpr int kFetch = kPages / kWaves;        // pages of a tile each wave fetches
  auto& klds = *reinterpret_cast<u32x4(*)[2][kKeys][16]>(lds_raw);
  auto& vlds = *reinterpret_cast<u32x4(*)[2][kKeys][16]>(lds_raw + kTileBytes);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wq = wave / WK, wk = wave % WK;
  const uint32_t page0 = key0 / 16, npages = (key1 - key0 + 15) / 16, tiles = (key1 - key0 + kKeys - 1) / kKeys;

  auto table_chunk = [&](uint32_t first) { return first + lane < npages ? trow[page0 + first + lane] : 0u; };
  uint32_t tab = table_chunk(0), tab_next = table_chunk(64);

  const uint32_t token_bytes = kvh * 256;
  uint32_t koff[4], voff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t row = (4 * i + (lane >> 4)) * token_bytes;
    koff[i] = row + (((lane & 15) ^ (4 * i + (lane >> 4))) & 15) * 16;
    voff[i] = row + (((lane & 15) ^ ((lane >> 4) << 2)) & 15) * 16;
  }
  uint32_t bad_page = 0;  // uniform
  auto fetch = [&](uint32_t t, int buf) {
#pragma unroll
    for (int f = 0; f < kFetch; ++f) {
      const uint32_t in_tile = wave + f * kWaves, pi = kPages * t + in_tile;
      uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)tab, (int)(pi & 63u));
      uint32_t valid = pi < npages ? min(16u, key1 - key0 - pi * 16) : 0u;  // keys of the page
      if (page >= pages) {
        bad_page |= valid;
        page = 0;
        valid = 0;
      }
      // Loads of tokens past the keys are out of bounds and return zeros.
      const uint32_t bytes = valid * token_bytes;
      const uint64_t base = ((uint64_t)page * 16 * kvh + h) * 128;
      auto krs = __builtin_amdgcn_make_buffer_rsrc((void*)(kc + base), 0, bytes, 0x00020000);
      auto vrs = __builtin_amdgcn_make_buffer_rsrc((void*)(vc + base), 0, bytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            krs, (__attribute__((address_space(3))) void*)&klds[buf][16 * in_tile + 4 * i][0], 16, koff[i], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            vrs, (__attribute__((address_space(3))) void*)&vlds[buf][16 * in_tile + 4 * i][0], 16, voff[i], 0, 0, 0);
    }
  };
  fetch(0, 0);

  // Query operand: lane l holds vector l % 32 of the wave (row j / G, head
  // j % G), dims 16 i + 8 (l / 32) .. + 7; vectors past the rows are zeros.
  const uint32_t c = lane & 31, hi = lane >> 5;
  const uint32_t rj = (32 * wq + c) / G, head = h * G + c % G;
  const bool live = wq < WQ && (uint32_t)(32 * wq / G) < nrows;  // a wave with no rows only fetches
  const bool qvalid = live && rj < nrows;
  u32x4 qv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    qv[i] = qvalid ? *reinterpret_cast<const u32x4*>(q + ((uint64_t)(row0 + rj) * qh + head) * 128 + 16 * i + 8 * hi)
                   : u32x4{0u, 0u, 0u, 0u};

  const float kNegInf = -__builtin_inff();
  const float cs = kScoreScale * kLog2e;
  float m_run = kNegInf, l_run = 0.f, s_abs = 0.f;
  f32x16 acc[4];  // output dims 32 d + 8 (e / 4) + 4 hi + e % 4 of vector c
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;

  const u32x4* kl = &klds[0][c][0];
  const uint32_t kx = c & 15;
  const uint32_t tj = lane & 15, tkey = 4 * hi + (tj >> 2);
  const uint32_t tchunk = ((lane >> 4) & 1) * 2 + ((tj & 3) >> 1), thalf = tj & 1;

  auto compute = [&](uint32_t t) {
    const int buf = t & 1;
    const int own = kGroups * wk;  // this wave's first 32-key group of the tile
    f32x16 s[kGroups];
#pragma unroll
    for (int kt = 0; kt < kGroups; ++kt) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kt][e] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const u32x4 ka = kl[(buf * kKeys + 32 * (own + kt)) * 16 + ((2 * i + hi) ^ kx)];
        s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ka),
                                                        __builtin_bit_cast(bf16x8, qv[i]), s[kt], 0, 0, 0);
      }
    }
    const uint32_t first = key0 + t * kKeys + 32 * own, at = first + 4 * hi;
    if (first + 32 * kGroups > key1) {
      // Keys past the chunk: no term (and no part in the finiteness check).
#pragma unroll
      for (int kt = 0; kt < kGroups; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool ok = at + 32 * kt + 8 * (e >> 2) + (e & 3) < key1;
          s_abs = fmaxf(s_abs, ok ? __builtin_fabsf(s[kt][e]) : 0.f);
          s[kt][e] = ok ? s[kt][e] : kNegInf;
        }
    } else {
#pragma unroll
      for (int kt = 0; kt < kGroups; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) s_abs = fmaxf(s_abs, __builtin_fabsf(s[kt][e]));
    }
    float mt = kNegInf;
#pragma unroll
    for (int kt = 0; kt < kGroups; ++kt)
#pragma unroll
      for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[kt][e]);
    {
      const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, mt), __builtin_bit_cast(uint32_t, mt),
                                                       false, false);
      mt = fmaxf(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1]));
    }
    // A wave along the keys may meet no key in a tile (m_run and mt both
    // -inf: their difference is NaN, no move).
    if (__builtin_amdgcn_ballot_w64((mt - m_run) * cs > 8.f) != 0ull) {
      const float m_new = fmaxf(m_run, mt);
      const float alpha = m_run == kNegInf ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * cs);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] *= alpha;
    }
    const float mc = m_run == kNegInf ? 0.f : m_run * cs;
    float ps = 0.f;
#pragma unroll
    for (int g = 0; g < 2 * kGroups; ++g) {
      float p[8];
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][8 * (g & 1) + e], cs, -mc));
        ps += p[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ph[e] = pack_bf16x2(p[2 * e], p[2 * e + 1]);
        pl[e] = pack_bf16x2(p[2 * e] - lo_bf16(ph[e]), p[2 * e + 1] - hi_bf16(ph[e]));
      }
      const bf16x8 bh = __builtin_bit_cast(bf16x8, u32x4{ph[0], ph[1], ph[2], ph[3]});
      const bf16x8 bl = __builtin_bit_cast(bf16x8, u32x4{pl[0], pl[1], pl[2], pl[3]});
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        u32x2 vq[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t key = 32 * own + 16 * g + 8 * u + tkey;
          const uint32_t chunk = (4 * d + tchunk) ^ ((tj >> 2) << 2);
          auto* src = reinterpret_cast<u32x2*>(&vlds[buf][key][chunk]) + thalf;
          vq[u] = __builtin_bit_cast(
              u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)src));
        }
        const bf16x8 va = __builtin_bit_cast(bf16x8, u32x4{vq[0][0], vq[0][1], vq[1][0], vq[1][1]});
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, bh, acc[d], 0, 0, 0);
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, bl, acc[d], 0, 0, 0);
      }
    }
    l_run += ps;
  };
  for (uint32_t t = 0; t < tiles; ++t) {
    __builtin_amdgcn_s_waitcnt(0 | (7u << 4) | (15u << 8));  // this wave's share of tile t is in LDS
    __syncthreads();  // everyone's is, and everyone is done with tile t - 1
    if (t + 1 < tiles) {
      if ((t + 1) % (64 / kPages) == 0) {
        tab = tab_next;
        tab_next = table_chunk(kPages * (t + 1) + 64);
      }
      fetch(t + 1, (t + 1) & 1);
    }
    if (live) compute(t);
  }

  float L = l_run;
  {
    const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, L), __builtin_bit_cast(uint32_t, L),
                                                     false, false);
    L = __builtin_bit_cast(float, (uint32_t)sw[0]) + __builtin_bit_cast(float, (uint32_t)sw[1]);
  }
  if constexpr (WK > 1) {
    // Waves wk > 0 hand their state over through the tiles' LDS.
    constexpr size_t kSlot = sizeof(f32x4) * 16 * 64 + sizeof(float) * 3 * 64;
    static_assert(kSlot * WQ * (WK - 1) <= 2 * kTileBytes, "one slot per wave handing over");
    auto slot_acc = [&](int k) { return reinterpret_cast<f32x4*>(lds_raw + kSlot * (wq * (WK - 1) + k - 1)); };
    __syncthreads();  // every wave is done with the tiles
    if (live && wk > 0) {
      f32x4* sa = slot_acc(wk);
      float* sm = reinterpret_cast<float*>(sa + 16 * 64);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4)
          sa[(4 * d + e4) * 64 + lane] =
              f32x4{acc[d][4 * e4], acc[d][4 * e4 + 1], acc[d][4 * e4 + 2], acc[d][4 * e4 + 3]};
      sm[lane] = m_run;
      sm[64 + lane] = L;
      sm[128 + lane] = s_abs;
    }
    __syncthreads();
    if (live && wk == 0) {
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        const f32x4* sa = slot_acc(k);
        const float* sm = reinterpret_cast<const float*>(sa + 16 * 64);
        const float mo = sm[lane], lo = sm[64 + lane];
        s_abs = fmaxf(s_abs, sm[128 + lane]);
        const float m_new = fmaxf(m_run, mo);
        const float fs = m_run == kNegInf ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * cs);
        const float fo = mo == kNegInf ? 0.f : __builtin_amdgcn_exp2f((mo - m_new) * cs);
        m_run = m_new;
        L = L * fs + lo * fo;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[d][e] = acc[d][e] * fs + sa[(4 * d + (e >> 2)) * 64 + lane][e & 3] * fo;
      }
    }
  }
  if (live && wk == 0 && qvalid) {
    float* r = rec + (((uint64_t)(row0 + rj) * qh + head) * slots + slot) * kRecord;
    if (hi == 0) {
      r[0] = m_run * cs;  // in the exponent of 2
      r[1] = L;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4)
        *reinterpret_cast<f32x4*>(r + 4 + 32 * d + 8 * e4 + 4 * hi) =
            f32x4{acc[d][4 * e4], acc[d][4 * e4 + 1], acc[d][4 * e4 + 2], acc[d][4 * e4 + 3]};
    if (!(L > 0.f) | !(s_abs < __builtin_inff())) raise_error(err, ERR_NONFINITE);
  }
  if (bad_page != 0 && lane == 0) raise_error(err, ERR_PAGE);
}

__device__ __forceinline__ uint32_t prefix_of(const Groups& gs, uint32_t r) {
  for (uint32_t i = 0; i < gs.count; ++i)
    if (r - gs.g[i].first_row < gs.g[i].rows) return gs.g[i].prefix_tokens;
  return 0;
}

// Orders a wave's LDS accesses of the steps before and after it.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// What a workgroup that takes own keys needs of LDS.
template <int G>
struct OwnLds {
  float sbuf[kWaves][64][G];  // scores, then probabilities: [token of the wave's four pages][head]
  float stat[kWaves][2][G];
  float acc[kWaves][G][128];
  u32x4 ktile[kWaves][16][17];  // 272-byte rows keep the column reads conflict-free
};

// The state of row r over its keys of pages [page0, page1) of its table (keys
// below ctx), for KV head h: G records at rec.
template <int G>
__device__ __forceinline__ void attend_own(unsigned char* lds_raw, const uint16_t* __restrict__ q,
                                           const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
                                           const uint32_t* __restrict__ trow, uint32_t r, uint32_t ctx, uint32_t page0,
                                           uint32_t page1, uint32_t h, uint32_t qh, uint32_t kvh, uint32_t pages,
                                           float* rec, uint32_t* err) {
  constexpr uint32_t kWavePages = kOwnPages / kWaves;
  auto& lds = *reinterpret_cast<OwnLds<G>*>(lds_raw);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t g16 = lane >> 4, r16 = lane & 15;
  const float kNegInf = -__builtin_inff();
  const float cs = kScoreScale * kLog2e;
  float* sw = &lds.sbuf[wave][0][0];
  bool bad = false;
  uint32_t bad_page = 0;

  // B operand: query head h G + r16 (zero for r16 >= G), dims 32 i + 8 g16 .. + 7.
  u32x4 qv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    qv[i] = r16 < G ? *reinterpret_cast<const u32x4*>(q + ((uint64_t)r * qh + h * G + r16) * 128 + 32 * i + 8 * g16)
                    : u32x4{0u, 0u, 0u, 0u};
  float m[G], l[G], acc[G][2];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = kNegInf;
    l[g] = acc[g][0] = acc[g][1] = 0.f;
  }
  for (uint32_t at = page0; at < page1; at += kOwnPages) {
    const uint32_t w0 = at + wave * kWavePages, np = w0 < page1 ? min(page1 - w0, kWavePages) : 0u;
    if (np == 0) break;  // this wave has no more pages (no barrier in the loop)
    uint32_t phys = lane < (int)np ? trow[w0 + lane] : 0u;
    if (phys >= pages) {
      bad_page = 1;
      phys = 0;
    }
    auto phys_of = [&](uint32_t j) { return (uint32_t)__builtin_amdgcn_readlane((int)phys, (int)j); };
    // Whole 256-byte token rows per load (lane: token 4 i + g16, dims 8 r16 .. + 7).
    u32x4 kr[kWavePages][4];
#pragma unroll
    for (uint32_t u = 0; u < kWavePages; ++u)
      if (u < np) {
        const uint16_t* kp = kc + (((uint64_t)phys_of(u) * 16 + g16) * kvh + h) * 128 + 8 * r16;
#pragma unroll
        for (int i = 0; i < 4; ++i) kr[u][i] = *reinterpret_cast<const u32x4*>(kp + (uint64_t)4 * i * kvh * 128);
      }
    uint32_t vd[kWavePages][16];
#pragma unroll
    for (uint32_t u = 0; u < kWavePages; ++u)
      if (u < np) {
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(vc + (((uint64_t)phys_of(u) * 16) * kvh + h) * 128) + lane;
#pragma unroll
        for (int e = 0; e < 16; ++e) vd[u][e] = vp[(uint64_t)e * kvh * 64];
      }
    // Scores: S^T = K Q^T a page at a time; lane: query r16, tokens 4 g16 + e.
    float pm = kNegInf;
#pragma unroll
    for (uint32_t u = 0; u < kWavePages; ++u)
      if (u < np) {
#pragma unroll
        for (int i = 0; i < 4; ++i) lds.ktile[wave][4 * i + g16][r16] = kr[u][i];
        wave_fence();
        f32x4 sacc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, lds.ktile[wave][r16][g16 + 4 * i]),
                                                        __builtin_bit_cast(bf16x8, qv[i]), sacc, 0, 0, 0);
        wave_fence();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool valid = (w0 + u) * 16 + 4 * g16 + e < ctx;
          const float sv = valid ? sacc[e] * cs : kNegInf;
          bad |= valid && !is_finite_f32(sv);
          pm = fmaxf(pm, sv);
          if (r16 < G) sw[(u * 16 + 4 * g16 + e) * G + r16] = sv;
        }
      }
    pm = fmaxf(pm, __shfl_xor(pm, 16, 64));
    pm = fmaxf(pm, __shfl_xor(pm, 32, 64));
    float scale[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float m_new = fmaxf(m[g], lane_bcast(pm, g));  // finite: a wave's pages hold a key
      scale[g] = __builtin_amdgcn_exp2f(m[g] - m_new);
      m[g] = m_new;
    }
    wave_fence();
    // Probabilities in place, one token a lane; their sums.
    if (lane < (int)(np * 16)) {
#pragma unroll
      for (int g = 0; g < G; ++g) sw[lane * G + g] = __builtin_amdgcn_exp2f(sw[lane * G + g] - m[g]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float ps = lane < (int)(np * 16) ? sw[lane * G + g] : 0.f;
      l[g] = l[g] * scale[g] + wave_sum(ps);
      acc[g][0] *= scale[g];
      acc[g][1] *= scale[g];
    }
    wave_fence();
    // n += p v: lane owns dims 2 lane, 2 lane + 1.
#pragma unroll
    for (uint32_t u = 0; u < kWavePages; ++u)
      if (u < np) {
        const uint32_t valid = min(16u, ctx - (w0 + u) * 16);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t v = (uint32_t)e < valid ? vd[u][e] : 0u;  // slots past the context may hold anything
          const float v0 = lo_bf16(v), v1 = hi_bf16(v);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const float p = sw[(u * 16 + e) * G + g];
            acc[g][0] = __builtin_fmaf(p, v0, acc[g][0]);
            acc[g][1] = __builtin_fmaf(p, v1, acc[g][1]);
          }
        }
      }
    wave_fence();
  }
  // The waves' states in wave order (a wave without pages has l = 0).
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (lane == 0) {
      lds.stat[wave][0][g] = m[g];
      lds.stat[wave][1][g] = l[g];
    }
    lds.acc[wave][g][2 * lane] = acc[g][0];
    lds.acc[wave][g][2 * lane + 1] = acc[g][1];
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < G * 128; idx += kThreads) {
    const int g = idx >> 7, c = idx & 127;
    float M = lds.stat[0][0][g];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, lds.stat[w][0][g]);
    float n = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float lw = lds.stat[w][1][g];
      if (lw > 0.f) {
        const float f = __builtin_amdgcn_exp2f(lds.stat[w][0][g] - M);
        n += lds.acc[w][g][c] * f;
        L += lw * f;
      }
    }
    rec[g * kRecord + 4 + c] = n;
    if (c == 0) {
      rec[g * kRecord] = M;
      rec[g * kRecord + 1] = L;
      bad |= !(L > 0.f);
    }
  }
  if (bad) raise_error(err, ERR_NONFINITE);
  if (bad_page) raise_error(err, ERR_PAGE);
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
// KV head. The others share the rows' own keys, cut into units of unit_pages
// pages (a rule on the positions' total): every workgroup counts them for
// itself, takes units own, own + own_wgs, ... of each KV head, and the first
// one writes each row's first unit to `first` for the merge.
template <int G, int WQ, int WK>
__global__ __launch_bounds__(kThreads, 2) void prefix_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
    const uint32_t* __restrict__ positions, const uint32_t* __restrict__ table, uint32_t rows, uint32_t qh, uint32_t kvh,
    uint32_t stride, uint32_t pages, uint32_t context, uint32_t prefix_wgs, uint32_t own_wgs, float* prefix_rec,
    float* own_rec, uint32_t* first, uint32_t* err, Groups gs) {
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[2 * kTileBytes];
  static_assert(sizeof(OwnLds<G>) <= sizeof(lds_raw), "the own keys' part fits the tiles'");
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
      if (differ) raise_error(err, ERR_PAGE);
    }
    attend_prefix<G, WQ, WK>(lds_raw, q, kc, vc, table + (uint64_t)row0 * stride, row0, nrows, key0, key1, h, qh, kvh,
                             pages, prefix_rec, gs.prefix_slots, chunk, err);
    return;
  }
  const uint32_t own = blockIdx.x - prefix_wgs;
  __shared__ uint32_t scan[kThreads];
  __shared__ uint32_t wave_total[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Sum over the workgroup (every thread gets it) and the sum up to this thread.
  auto block_scan = [&](uint32_t v, uint32_t& total) {
    uint32_t sum = v;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const uint32_t up = __shfl_up(sum, off, 64);
      if (lane >= off) sum += up;
    }
    __syncthreads();
    if (lane == 63) wave_total[wave] = sum;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) sum += wave_total[w];
      total += wave_total[w];
    }
    return sum;
  };
  uint64_t all = 0;
  bool bad = false;
  for (uint32_t r0 = 0; r0 < rows; r0 += kThreads) {
    const uint32_t r = r0 + threadIdx.x;
    uint32_t total;
    block_scan(r < rows ? own_pages(positions, gs, r, context, stride, bad) : 0u, total);
    all += total;
  }
  if (bad && own == 0) raise_error(err, ERR_POSITION);
  // (The cap is beyond any row: one unit each.)
  const uint32_t unit_pages =
      (uint32_t)min((all * kvh / kOwnUnits + kOwnPages) / kOwnPages * kOwnPages, (uint64_t)1 << 24);
  uint32_t base = 0;  // units of the rows before r0
  uint32_t next = own;  // this workgroup's next (unit, head)
  for (uint32_t r0 = 0; r0 < rows; r0 += kThreads) {
    const uint32_t r = r0 + threadIdx.x;
    const uint32_t mine = r < rows ? (own_pages(positions, gs, r, context, stride, bad) + unit_pages - 1) / unit_pages : 0u;
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
      const uint32_t row = __builtin_amdgcn_readfirstlane(r0 + lo);
      const uint32_t before = lo ? scan[lo - 1] : 0u;
      const uint32_t prefix = prefix_of(gs, row), ctx = __builtin_amdgcn_readfirstlane(positions[row]) + 1;
      const uint32_t page0 = __builtin_amdgcn_readfirstlane(prefix / 16 + (unit - before) * unit_pages);
      const uint32_t page1 = min(page0 + unit_pages, (ctx + 15) / 16);
      attend_own<G>(lds_raw, q, kc, vc, table + (uint64_t)row * stride, row, ctx, page0, page1, h, qh, kvh, pages,
                    own_rec + (uint64_t)next * G * kRecord, err);
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
  p.form = vectors > 64 ? 1 : vectors > 32 ? 2 : 4;
  p.gs.block_rows = 128 / p.form / g;
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
  p.own_wgs = (uint64_t)rows * kvh < 256 ? 256 : 512;
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
#define FH_PREFIX_FORM(G_, WQ_, WK_)                                                                               \
  hipLaunchKernelGGL((prefix_kernel<G_, WQ_, WK_>), dim3(prefix_wgs + p.own_wgs), dim3(kThreads), 0, s, q, k_cache, \
                     v_cache, positions, table, rows, qh, kvh, stride, pages, context, prefix_wgs, p.own_wgs,      \
                     prefix_rec, own_rec, first, err, p.gs)
#define FH_PREFIX(G_)              \
  do {                             \
    if (p.form == 1)               \
      FH_PREFIX_FORM(G_, 4, 1);    \
    else if (p.form == 2)          \
      FH_PREFIX_FORM(G_, 2, 2);    \
    else                           \
      FH_PREFIX_FORM(G_, 1, 2);    \
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
