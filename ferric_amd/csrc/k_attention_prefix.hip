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
// keys [key0, key1), key0 a multiple of 16, for KV head h.
template <int G, int WK>
__device__ void attend(const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
                       const uint32_t* __restrict__ trow, uint32_t row0, uint32_t nrows, uint32_t key0, uint32_t key1,
                       uint32_t h, uint32_t qh, uint32_t kvh, uint32_t pages, float* rec, uint32_t slots, uint32_t slot,
                       uint32_t* err) {
  constexpr int WQ = kWaves / WK;                // waves along the vectors
  constexpr int kKeys = WK == 4 ? 128 : 64;      // keys per tile
  constexpr int kGroups = kKeys / 32 / WK;       // 32-key groups per wave and tile
  constexpr int kPages = kKeys / 16;             // pages per tile
  constexpr int kFetch = kPages / kWaves;        // of which each wave fetches this many
  constexpr size_t kTileBytes = sizeof(u32x4) * 2 * kKeys * 16;
  __shared__ __attribute__((aligned(16))) unsigned char lds_raw[2 * kTileBytes];
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
  const bool live = (uint32_t)(32 * wq / G) < nrows;  // a wave with no rows only fetches
  const bool qvalid = rj < nrows;
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
    static_assert(kSlot * WQ * (WK - 1) <= sizeof(lds_raw), "one slot per wave handing over");
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

// Prefix items: (KV head, item).
template <int G, int WK>
__global__ __launch_bounds__(64 * kWaves, WK == 4 ? 1 : 2) void prefix_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
    const uint32_t* __restrict__ table, uint32_t qh, uint32_t kvh, uint32_t stride, uint32_t pages, float* rec,
    uint32_t slots, uint32_t* err, Groups gs) {
  const uint32_t h = blockIdx.x, item = blockIdx.y;
  uint32_t gi = 0;
  while (gi + 1 < gs.count && item >= gs.g[gi + 1].item0) ++gi;
  const Group g = gs.g[gi];
  const uint32_t blocks = (g.rows + gs.block_rows - 1) / gs.block_rows;
  const uint32_t block = (item - g.item0) % blocks, chunk = (item - g.item0) / blocks;
  const uint32_t first = block * gs.block_rows, nrows = min(gs.block_rows, g.rows - first);
  const uint32_t key0 = chunk * gs.chunk, key1 = min(key0 + gs.chunk, g.prefix_tokens);
  const uint32_t row0 = g.first_row + first;
  const uint32_t* trow = table + (uint64_t)row0 * stride;
  if (h == 0) {
    // The rows of the block list the same pages here as the group's first row.
    const uint32_t p0 = key0 / 16, np = (key1 - key0 + 15) / 16;
    const uint32_t* lead = table + (uint64_t)g.first_row * stride;
    bool differ = false;
    for (uint32_t i = threadIdx.x; i < nrows * np; i += 64 * kWaves)
      differ |= table[(uint64_t)(row0 + i / np) * stride + p0 + i % np] != lead[p0 + i % np];
    if (differ) raise_error(err, ERR_PAGE);
  }
  attend<G, WK>(q, kc, vc, trow, row0, nrows, key0, key1, h, qh, kvh, pages, rec, slots, chunk, err);
}

__device__ __forceinline__ uint32_t prefix_of(const Groups& gs, uint32_t r) {
  for (uint32_t i = 0; i < gs.count; ++i)
    if (r - gs.g[i].first_row < gs.g[i].rows) return gs.g[i].prefix_tokens;
  return 0;
}

// A row's own keys [prefix, position], own_chunk at a time: (split, KV head, row).
template <int G>
__global__ __launch_bounds__(64 * kWaves, 1) void own_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
    const uint32_t* __restrict__ positions, const uint32_t* __restrict__ table, uint32_t qh, uint32_t kvh,
    uint32_t stride, uint32_t pages, uint32_t context, uint32_t own_chunk, float* rec, uint32_t slots, uint32_t* err,
    Groups gs) {
  const uint32_t split = blockIdx.x, h = blockIdx.y, r = blockIdx.z;
  const uint32_t pos = (uint32_t)__builtin_amdgcn_readfirstlane((int)positions[r]);
  const uint32_t prefix = prefix_of(gs, r);
  if (pos >= context || pos / 16 >= stride || pos + 1 < prefix) {
    if (split == 0 && h == 0 && threadIdx.x == 0) raise_error(err, ERR_POSITION);
    return;
  }
  const uint32_t key0 = prefix + split * own_chunk, key1 = min(key0 + own_chunk, pos + 1);
  if (key0 >= key1) return;
  attend<G, 4>(q, kc, vc, table + (uint64_t)r * stride, r, 1, key0, key1, h, qh, kvh, pages, rec, slots,
               gs.prefix_slots + split, err);
}

// One wave per (row, query head): its records in ascending key order.
__global__ __launch_bounds__(256) void prefix_merge_kernel(const float* __restrict__ rec,
                                                          const uint32_t* __restrict__ positions,
                                                          uint16_t* __restrict__ out, uint32_t out_mtiles, uint32_t rows,
                                                          uint32_t qh, uint32_t stride, uint32_t context,
                                                          uint32_t own_chunk, uint32_t slots, uint32_t* err, Groups gs) {
  const int lane = threadIdx.x & 63;
  const uint32_t id = blockIdx.x * 4 + (threadIdx.x >> 6), r = id / qh, head = id % qh;
  if (r >= rows) return;
  const uint32_t pos = positions[r], prefix = prefix_of(gs, r);
  if (pos >= context || pos / 16 >= stride || pos + 1 < prefix) return;  // reported by the own keys' kernel
  const uint32_t np = (prefix + gs.chunk - 1) / gs.chunk, no = (pos + 1 - prefix + own_chunk - 1) / own_chunk;
  const float* p = rec + (uint64_t)id * slots * kRecord;
  float M = -__builtin_inff(), L = 0.f, n0 = 0.f, n1 = 0.f;
  for (uint32_t i = 0; i < np + no; ++i) {
    const float* s = p + (uint64_t)(i < np ? i : gs.prefix_slots + i - np) * kRecord;
    const float m = s[0], m_new = fmaxf(M, m);
    const float a = __builtin_amdgcn_exp2f(M - m_new), b = __builtin_amdgcn_exp2f(m - m_new);
    M = m_new;
    L = L * a + s[1] * b;
    n0 = n0 * a + s[4 + 2 * lane] * b;
    n1 = n1 * a + s[5 + 2 * lane] * b;
  }
  const uint32_t o0 = f32_to_bf16(n0 / L), o1 = f32_to_bf16(n1 / L);
  const uint32_t col = head * 128 + 2 * lane;
  uint16_t* dst = out_mtiles ? out + act_offset_m(r, col, out_mtiles) : out + (uint64_t)r * qh * 128 + col;
  *reinterpret_cast<uint32_t*>(dst) = o0 | (o1 << 16);
  if (!(L > 0.f) || ((o0 & 0x7f80u) == 0x7f80u) || ((o1 & 0x7f80u) == 0x7f80u)) raise_error(err, ERR_NONFINITE);
}

}  // namespace

namespace {

constexpr uint32_t kOwnChunk = 512;

// The launch's work split: a rule on the groups, heads and lengths alone, so
// that the scratch's size and the launch agree.
struct PrefixPlan {
  Groups gs;
  uint32_t items, form, own_splits, slots;
};

PrefixPlan prefix_plan(const fh_prefix_group* groups, uint32_t ngroups, uint32_t qh, uint32_t kvh, uint32_t context) {
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
  // About one workgroup per CU over the prefixes, at least two tiles each.
  uint64_t tokens = 0;
  for (uint32_t i = 0; i < p.gs.count; ++i)
    tokens += (uint64_t)p.gs.g[i].prefix_tokens * ((p.gs.g[i].rows + p.gs.block_rows - 1) / p.gs.block_rows) * kvh;
  const uint32_t tile = p.form == 4 ? 128 : 64;
  uint64_t chunk = (tokens / 256 + tile - 1) / tile * tile;
  if (chunk < 2 * tile) chunk = 2 * tile;
  p.gs.chunk = (uint32_t)chunk;
  uint32_t at = 0;
  for (uint32_t i = 0; i < p.gs.count; ++i) {
    Group& to = p.gs.g[i];
    const uint32_t chunks = (to.prefix_tokens + p.gs.chunk - 1) / p.gs.chunk;
    to.item0 = at;
    at += chunks * ((to.rows + p.gs.block_rows - 1) / p.gs.block_rows);
    if (chunks > p.gs.prefix_slots) p.gs.prefix_slots = chunks;
  }
  p.items = at;
  p.own_splits = (context + kOwnChunk - 1) / kOwnChunk;
  p.slots = p.gs.prefix_slots + p.own_splits;
  return p;
}

}  // namespace

uint64_t prefix_scratch_bytes(const fh_prefix_group* groups, uint32_t ngroups, uint32_t rows, uint32_t qh, uint32_t kvh,
                              uint32_t context) {
  const PrefixPlan p = prefix_plan(groups, ngroups, qh, kvh, context);
  return (uint64_t)rows * qh * p.slots * kRecord * 4;
}

hipError_t launch_prefix_attention(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                   const uint32_t* positions, const uint32_t* table, const fh_prefix_group* groups,
                                   uint32_t ngroups, uint16_t* out, uint32_t out_tiled, void* scratch, uint32_t rows,
                                   uint32_t qh, uint32_t kvh, uint32_t stride, uint32_t pages, uint32_t context,
                                   uint32_t* err, hipStream_t s) {
  const PrefixPlan p = prefix_plan(groups, ngroups, qh, kvh, context);
  float* rec = reinterpret_cast<float*>(scratch);
#define FH_PREFIX_WK(G_, WK_)                                                                                    \
  hipLaunchKernelGGL((prefix_kernel<G_, WK_>), dim3(kvh, p.items), dim3(64 * kWaves), 0, s, q, k_cache, v_cache, \
                     table, qh, kvh, stride, pages, rec, p.slots, err, p.gs)
#define FH_PREFIX(G_)                                                                                            \
  do {                                                                                                           \
    if (p.items) {                                                                                               \
      if (p.form == 1)                                                                                           \
        FH_PREFIX_WK(G_, 1);                                                                                     \
      else if (p.form == 2)                                                                                      \
        FH_PREFIX_WK(G_, 2);                                                                                     \
      else                                                                                                       \
        FH_PREFIX_WK(G_, 4);                                                                                     \
    }                                                                                                            \
    hipLaunchKernelGGL((own_kernel<G_>), dim3(p.own_splits, kvh, rows), dim3(64 * kWaves), 0, s, q, k_cache,     \
                       v_cache, positions, table, qh, kvh, stride, pages, context, kOwnChunk, rec, p.slots, err, \
                       p.gs);                                                                                    \
  } while (0)
  switch (qh / kvh) {
    case 1: FH_PREFIX(1); break;
    case 2: FH_PREFIX(2); break;
    case 4: FH_PREFIX(4); break;
    case 8: FH_PREFIX(8); break;
    default: return hipErrorInvalidValue;
  }
#undef FH_PREFIX
#undef FH_PREFIX_WK
  const uint64_t waves = (uint64_t)rows * qh;
  hipLaunchKernelGGL(prefix_merge_kernel, dim3((waves + 3) / 4), dim3(256), 0, s, rec, positions, out,
                     out_tiled ? act_mtiles(rows) : 0u, rows, qh, stride, context, kOwnChunk, p.slots, err, p.gs);
  return hipGetLastError();
}

}  // namespace fh
