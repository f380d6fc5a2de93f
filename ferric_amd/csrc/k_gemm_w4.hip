// K1 projections with 4-bit weights and group scales for decode batches
// (m <= 32 token rows) on gfx950 MFMA with FP32 accumulation.
//
//   y[m][n] = sum over groups g of s[n][g] * sum_{k in g} (q[n][k] - z[n][g]) x[m][k]
//
// with q in 0..15, groups of 32, 64 or 128 consecutive columns, bf16 scales s
// and zero points z (8 where none are given).
//
// A 4-bit weight enters the MFMA as the bf16 number 16 + q, which is exact, from
// a shift and an and-or for two weights: the nibble is the top of the mantissa of
// 0x4180. The 16 comes off in the accumulators, which start a group as the MFMA of
// its activations with a tile of -16 (of -24 where there are no zero points: the 8
// with it); that, -16 sum x in every column, serves the zero points too:
// sum (q - z) x = [sum (16 + q) x - 16 sum x] + z / 16 (-16 sum x). The weight tiles
// of a wave share it. What cancels is at most 31 / 4.6 of what is left (root mean
// squares), so a group's FP32 roundings count up to seven times: the error measured
// is 9e-8 of the result's norm, against 8e-7 with 128 + q (one shift less) in its place.
//
// Layout (fh_op_tile_weight_w4): a 16-row x 128-column tile is 1 KiB, one
// 16-byte load per lane; lane = row + 16 (column % 32 / 8), its four words are
// the four 32-column k-blocks, so word j is the B operand of k-block j's MFMA
// before unpacking: columns 2 i and 2 i + 1 of a word's eight at bits 4 i and
// 16 + 4 i, so that a shift and 0x00780078 take out a pair. Tiles run k-fastest. Scales
// and zero points: [n / 16][groups][16]; a tile's are one load each, a lane's being
// its row's and those of one group of the 128 columns. Activations in their tile
// order (common.hpp act_offset) are the A operand. Lanes of rows past m read the
// last row again (less to fetch; their output rows are not stored).
//
// What bounds it: the weights' bytes from HBM in 7 rows through 151936 x 4096 (60
// us, 345 MB at 5.7 TB/s; a large copy reaches 5.4, reads alone 6.0); a launch's start and end beside them
// in one row through 24576 x 4096 (11.9 us, 52 MB; 9.6 at that rate). From about 16
// rows on, and with few weight rows a workgroup, the activations, which every workgroup
// reads whole from the L2: 32 rows through 4096 x 12288 take 786 KB into each CU
// beside 115 KB of weights, 15.2 us, and 12.2 with one in six of those loads made.
#include "common.hpp"
#include "kernels.hpp"

namespace fh {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// Waves of a workgroup, which divide its k: 4 where there are kMany workgroups (one row through 24576 x 4096
// in 768 of them: 11.9 us, 13.1 with 16 waves, 14.7 with 8), else 16 (4 rows through 4096 x 4096 in 256: 4.7 us,
// 5.7 with 8, 8.6 with 4; 1024 x 2048 in 64: 2.9, 3.0, 3.6).
constexpr uint32_t kMany = 512;
constexpr int kWavesFew = 16, kWavesMany = 4;
// Weight tiles of a workgroup, which share its activations: 4 where enough workgroups are left (7 rows through
// 151936 x 4096 60 us, 67 with 2; 32 rows through 24576 x 4096 17.5, 18.8). One row asks for more of them: through
// 24576 x 4096 12.9, with 2 tiles 11.9.
constexpr uint32_t kQuadFrom = 1024, kQuadFromWide = 256, kPairFrom = 256;

__device__ __forceinline__ bf16x8 unpack_w4(uint32_t w, uint32_t mask, uint32_t base) {
  // Eight nibbles to bf16 16 + q.
  const u32x4 v = {((w << 3) & mask) | base, ((w >> 1) & mask) | base, ((w >> 5) & mask) | base,
                   ((w >> 9) & mask) | base};
  return __builtin_bit_cast(bf16x8, v);
}

// One workgroup: NT consecutive 16-row weight tiles and one split of k, whose
// 128-column blocks its waves divide; wave partials are added in wave order
// through LDS. GB: 32-column k-blocks per group. MT: 16-row activation tiles.
// A wave has one block in flight and leaves the rest to the other waves of its SIMD, up to 8:
// with two or three in flight, which take the registers of as many waves, nothing was
// faster (32 rows through 24576 x 4096: 20.3 us with two, 17.5 with one). But where few
// workgroups take more than 16 rows, each wave's turns are few and long, and the weights of
// kAhead blocks are requested before the activations of the first (32 rows through 4096 x
// 12288: 15.2 us, 16.4 without; through 4096 x 4096 6.5, 7.0; one row through 4096 x
// 12288 8.1 without, 8.5 with it).
template <int NT, int MT, int GB, bool ZP, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES == 4 && (NT == 4 || MT == 2) ? 3 : 4) void gemm_w4_kernel(
    const uint16_t* __restrict__ xt, const uint32_t* __restrict__ w, const uint16_t* __restrict__ scales,
    const uint8_t* __restrict__ zeros, uint32_t m, uint32_t kb_count, uint32_t kb_split, uint32_t epi,
    const uint16_t* residual, void* out, uint32_t ldo, uint32_t* err) {
  constexpr int GP = 4 / GB;  // groups per 128 columns
  constexpr int kAhead = WAVES == kWavesFew && MT == 2 ? (NT == 1 ? 3 : 2) : 1;
  __shared__ float red[WAVES][NT * MT * 256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tile0 = blockIdx.x * NT, split = blockIdx.y;
  const uint32_t s_lo = min(split * kb_split, kb_count), s_hi = min(s_lo + kb_split, kb_count), s_n = s_hi - s_lo;
  const uint32_t kb_lo = s_lo + (s_n * wave) / WAVES, kb_hi = s_lo + (s_n * (wave + 1)) / WAVES;
  const uint32_t r16 = lane & 15, g16 = lane >> 4;

  struct Weights {  // of 128 columns
    u32x4 w[NT];
    uint32_t s[NT];           // scale of row lane % 16, group lane / 16 % GP
    uint32_t z[ZP ? NT : 1];  // its zero point
  };
  // Buffers: uniform bases, one 32-bit offset a lane.
  const uint32_t wbytes = kb_count * 1024, sbytes = kb_count * 32 * GP, zbytes = kb_count * 16 * GP;
  auto buffer = [](const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000);
  };
  const auto wr = buffer(reinterpret_cast<const char*>(w) + (uint64_t)tile0 * wbytes, NT * wbytes);
  const auto sr = buffer(reinterpret_cast<const char*>(scales) + (uint64_t)tile0 * sbytes, NT * sbytes);
  const auto zr = buffer(reinterpret_cast<const char*>(zeros) + (uint64_t)tile0 * zbytes, NT * zbytes);
  const auto xr = buffer(xt, kb_count * 8192);
  uint32_t xoff[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) xoff[mt] = mt * 1024 + (min(16 * mt + r16, m - 1) & 15u) * 16 + g16 * 256;
  auto load_x = [&](u32x4 (&x)[4][MT], uint32_t kb) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        x[j][mt] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                 xr, xoff[mt] + (j & 1) * 2048, kb * 8192 + (j >> 1) * 4096, 0));
  };
  auto load_w = [&](Weights& b, uint32_t kb) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      b.w[nt] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, lane * 16, nt * wbytes + kb * 1024, 2));  // non-temporal
      const uint32_t sat = nt * sbytes + kb * 32 * GP;
      const uint32_t at = g16 % GP * 16 + r16;
      b.s[nt] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sr, at * 2, sat, 0);
      if constexpr (ZP) b.z[nt] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(zr, at, nt * zbytes + kb * 16 * GP, 0);
    }
  };
  // In registers, so that a mask and an or are one instruction.
  uint32_t mask = 0x00780078u, base = 0x41804180u;
  asm volatile("" : "+s"(mask));
  asm volatile("" : "+v"(base));

  f32x4 acc[NT][MT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  // bf16 -16 (with zero points) or -24.
  constexpr uint32_t kOff = ZP ? 0xc180c180u : 0xc1c0c1c0u;
  const bf16x8 offset = __builtin_bit_cast(bf16x8, u32x4{kOff, kOff, kOff, kOff});
  auto compute = [&](const Weights& b, const u32x4 (&x)[4][MT]) {
    // Scale (low half) and zero point of a group in all lanes of its row: the lanes' words, their 16-lane groups
    // exchanged.
    uint32_t sz[NT][GP];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t v = b.s[nt];
      if constexpr (ZP) v |= b.z[nt] << 16;
      if constexpr (GP == 1) {
        sz[nt][0] = v;
      } else if constexpr (GP == 2) {
        const auto t = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        sz[nt][0] = t[0];
        sz[nt][1] = t[1];
      } else {
        const auto u = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        const auto t0 = __builtin_amdgcn_permlane16_swap(u[0], u[0], false, false);
        const auto t1 = __builtin_amdgcn_permlane16_swap(u[1], u[1], false, false);
        sz[nt][0] = t0[0];
        sz[nt][1] = t0[1];
        sz[nt][2] = t1[0];
        sz[nt][3] = t1[1];
      }
    }
#pragma unroll
    for (int p = 0; p < GP; ++p) {
      f32x4 part[NT][MT], sx[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        sx[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < GB; ++i)
          sx[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[p * GB + i][mt]), offset,
                                                           sx[mt], 0, 0, 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) part[nt][mt] = sx[mt];
      }
#pragma unroll
      for (int i = 0; i < GB; ++i) {
        const int j = p * GB + i;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const bf16x8 q = unpack_w4(b.w[nt][j], mask, base);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            part[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[j][mt]), q,
                                                                  part[nt][mt], 0, 0, 0);
        }
      }
      // Lane: weight row r16, activation rows 4 g16 + e.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float s = lo_bf16(sz[nt][p]);
        // sx is -16 times the activations' sum.
        const float z = ZP ? 0.0625f * (float)((sz[nt][p] >> 16) & 0xffu) : 0.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = ZP ? __builtin_fmaf(z, sx[mt][e], part[nt][mt][e]) : part[nt][mt][e];
            acc[nt][mt][e] = __builtin_fmaf(s, v, acc[nt][mt][e]);
          }
      }
    }
  };
  for (uint32_t kb = kb_lo; kb < kb_hi; kb += kAhead) {
    Weights b[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (i == 0 || kb + i < kb_hi) load_w(b[i], kb + i);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i != 0 && kb + i >= kb_hi) break;
      u32x4 x[4][MT];
      load_x(x, kb + i);
      __builtin_amdgcn_sched_barrier(0);  // all loads are on their way before the first wait
      compute(b[i], x);
    }
  }

#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][(nt * MT + mt) * 256 + (4 * g16 + e) * 16 + r16] = acc[nt][mt][e];
  __syncthreads();
  auto total = [&](int i) {
    float v = red[0][i];
#pragma unroll
    for (int wv = 1; wv < WAVES; ++wv) v += red[wv][i];
    return v;
  };
  if (epi == FH_EPI_SWIGLU) {
    if constexpr (NT % 2 == 0) {
      bool bad = false;
      for (int idx = threadIdx.x; idx < (NT / 2) * MT * 256; idx += WAVES * 64) {
        const int pair = idx / (MT * 256), rem = idx % (MT * 256);
        const uint32_t row = 16 * (rem >> 8) + ((rem >> 4) & 15), col = (tile0 / 2 + pair) * 16 + (rem & 15);
        const float gate = total(2 * pair * MT * 256 + rem), up = total((2 * pair + 1) * MT * 256 + rem);
        if (row < m)
          reinterpret_cast<uint16_t*>(out)[act_offset(row, col)] =
              (uint16_t)swiglu_bf16(round_bf16(gate), round_bf16(up), bad);
      }
      if (bad) raise_error(err, ERR_NONFINITE);
    }
    return;
  }
  for (int idx = threadIdx.x; idx < NT * MT * 256; idx += WAVES * 64) {
    const int tm = idx >> 8;
    const uint32_t row = 16 * (tm % MT) + ((idx >> 4) & 15);
    if (row >= m) continue;
    const float v = total(idx);
    const uint64_t o = (uint64_t)row * ldo + (uint64_t)(tile0 + tm / MT) * 16 + (idx & 15);
    if (epi == FH_EPI_PARTIAL)
      reinterpret_cast<float*>(out)[(uint64_t)split * kMaxRows * ldo + o] = v;
    else if (epi == FH_EPI_F32)
      reinterpret_cast<float*>(out)[o] = v;
    else if (epi == FH_EPI_BF16)
      reinterpret_cast<uint16_t*>(out)[o] = (uint16_t)f32_to_bf16(v);
    else  // residual, as the bf16 projections round it
      reinterpret_cast<uint16_t*>(out)[o] = (uint16_t)f32_to_bf16((0.0f + v) + bf16_to_f32(residual[o]));
  }
}

// Eight columns a thread; the threads of a group are neighbours in the wave.
__global__ __launch_bounds__(256) void quantize_w4_kernel(const uint16_t* __restrict__ src,
                                                          uint32_t* __restrict__ packed,
                                                          uint16_t* __restrict__ scales, uint64_t words,
                                                          uint32_t group_words, uint32_t* err) {
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const bool live = i < words;  // whole groups: a group's threads are all live or none
  float v[8] = {};
  if (live) {
    const u32x4 d = reinterpret_cast<const u32x4*>(src)[i];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      v[2 * p] = lo_bf16(d[p]);
      v[2 * p + 1] = hi_bf16(d[p]);
    }
  }
  float top = 0.f;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    bad |= !is_finite_f32(v[e]);
    top = fmaxf(top, __builtin_fabsf(v[e]));
  }
  for (uint32_t off = 1; off < group_words; off *= 2) top = fmaxf(top, __shfl_xor(top, (int)off, 64));
  if (bad) raise_error(err, ERR_NONFINITE);
  if (!live) return;
  const uint32_t bits = f32_to_bf16(__fdiv_rn(top, 7.0f));
  const float s = bf16_to_f32(bits);
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(v[e], s)), -8.f), 7.f) : 0.f;
    word |= (uint32_t)((int)q + 8) << (4 * e);
  }
  packed[i] = word;
  if (i % group_words == 0) scales[i / group_words] = (uint16_t)bits;
}

__global__ __launch_bounds__(256) void tile_w4_kernel(const uint32_t* __restrict__ packed, uint32_t* __restrict__ dst,
                                                      uint64_t words, uint32_t kb_count, uint32_t tile_mul,
                                                      uint32_t tile_add) {
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;  // word j of lane of tile (nb, kb)
  if (i >= words) return;
  const uint32_t j = i & 3, lane = (i >> 2) & 63;
  const uint64_t tile = i >> 8;
  const uint64_t nb = tile / kb_count, kb = tile % kb_count;
  const uint64_t n = nb * 16 + (lane & 15);
  const uint32_t s = packed[n * kb_count * 16 + kb * 16 + 4 * j + (lane >> 4)];
  uint32_t d = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) d |= ((s >> (4 * e)) & 15u) << (4 * (e / 2) + 16 * (e % 2));
  dst[((nb * tile_mul + tile_add) * kb_count + kb) * 256 + (i & 255)] = d;
}

// [n][groups] to [n / 16][groups][16].
template <typename T>
__global__ __launch_bounds__(256) void tile_groups_kernel(const T* __restrict__ src, T* __restrict__ dst,
                                                          uint64_t count, uint32_t groups, uint32_t tile_mul,
                                                          uint32_t tile_add) {
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  const uint32_t r = i & 15;
  const uint64_t g = (i >> 4) % groups, nb = (i >> 4) / groups;
  dst[((nb * tile_mul + tile_add) * groups + g) * 16 + r] = src[(nb * 16 + r) * groups + g];
}

template <int NT, int MT, int GB, bool ZP, int WAVES>
void launch_w4_kernel(const uint16_t* xt, const uint32_t* w, const uint16_t* scales, const uint8_t* zeros, uint32_t m,
                      uint32_t n, uint32_t k, uint32_t epi, uint32_t splits, const uint16_t* residual, void* out,
                      uint32_t ldo, uint32_t* err, hipStream_t s) {
  const uint32_t kb = k / 128;
  hipLaunchKernelGGL((gemm_w4_kernel<NT, MT, GB, ZP, WAVES>), dim3(n / (16 * NT), splits), dim3(WAVES * 64), 0, s, xt,
                     w, scales, zeros, m, kb, (kb + splits - 1) / splits, epi, residual, out, ldo, err);
}

template <int NT, int WAVES>
void launch_w4(const uint16_t* xt, const uint32_t* w, const uint16_t* scales, const uint8_t* zeros, uint32_t m,
               uint32_t n, uint32_t k, uint32_t group, uint32_t epi, uint32_t splits, const uint16_t* residual,
               void* out, uint32_t ldo, uint32_t* err, hipStream_t s) {
#define FH_W4(MT_, GB_)                                                                                            \
  (zeros ? launch_w4_kernel<NT, MT_, GB_, true, WAVES>(xt, w, scales, zeros, m, n, k, epi, splits, residual, out, \
                                                      ldo, err, s)                                                 \
         : launch_w4_kernel<NT, MT_, GB_, false, WAVES>(xt, w, scales, zeros, m, n, k, epi, splits, residual, out, \
                                                       ldo, err, s))
  if (m <= 16) {
    if (group == 32) FH_W4(1, 1); else if (group == 64) FH_W4(1, 2); else FH_W4(1, 4);
  } else {
    if (group == 32) FH_W4(2, 1); else if (group == 64) FH_W4(2, 2); else FH_W4(2, 4);
  }
#undef FH_W4
}

}  // namespace

uint32_t gemm_w4_default_splits(uint32_t n, uint32_t k) {
  // About 256 workgroups of two tiles, each split keeping 4 blocks of 128 columns.
  const uint32_t groups = n % 32 == 0 ? n / 32 : n / 16, most = k / 512 ? k / 512 : 1;
  const uint32_t s = groups ? 256 / groups : 1;
  return s < 1 ? 1 : s > most ? most : s;
}

hipError_t launch_gemm_w4(const uint16_t* x_tiled, const uint32_t* w_tiled, const uint16_t* scales,
                          const uint8_t* zeros, uint32_t m, uint32_t n, uint32_t k, uint32_t group, uint32_t epilogue,
                          uint32_t splits, const uint16_t* residual, void* out, uint32_t ldo, uint32_t* err,
                          hipStream_t s) {
  const uint64_t wide = (uint64_t)splits * n;
  const bool quad = n % 64 == 0 && wide / 64 >= (m > 8 ? kQuadFromWide : kQuadFrom);
  const bool pair = n % 32 == 0 && (epilogue == FH_EPI_SWIGLU || wide / 32 >= kPairFrom);
  const bool many = wide / (pair ? 32 : 16) >= kMany;
#define FH_NT(NT_, WAVES_)                                                                                          \
  launch_w4<NT_, WAVES_>(x_tiled, w_tiled, scales, zeros, m, n, k, group, epilogue, splits, residual, out, ldo, err, s)
  if (quad)
    FH_NT(4, kWavesMany);
  else if (pair && many)
    FH_NT(2, kWavesMany);
  else if (pair)
    FH_NT(2, kWavesFew);
  else if (many)
    FH_NT(1, kWavesMany);
  else
    FH_NT(1, kWavesFew);
#undef FH_NT
  return hipGetLastError();
}

hipError_t launch_quantize_w4(const uint16_t* src, uint8_t* packed, uint16_t* scales, uint32_t n, uint32_t k,
                              uint32_t group, uint32_t* err, hipStream_t s) {
  const uint64_t words = (uint64_t)n * k / 8;
  hipLaunchKernelGGL(quantize_w4_kernel, dim3((words + 255) / 256), dim3(256), 0, s, src,
                     reinterpret_cast<uint32_t*>(packed), scales, words, group / 8, err);
  return hipGetLastError();
}

hipError_t launch_tile_weight_w4(const uint8_t* packed, const uint16_t* scales, const uint8_t* zeros, uint32_t* w_tiled,
                                 uint16_t* scales_tiled, uint8_t* zeros_tiled, uint32_t n, uint32_t k, uint32_t group,
                                 uint32_t tile_mul, uint32_t tile_add, hipStream_t s) {
  const uint64_t words = (uint64_t)n * k / 8, count = (uint64_t)n * (k / group);
  hipLaunchKernelGGL(tile_w4_kernel, dim3((words + 255) / 256), dim3(256), 0, s,
                     reinterpret_cast<const uint32_t*>(packed), w_tiled, words, k / 128, tile_mul, tile_add);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(tile_groups_kernel<uint16_t>, dim3((count + 255) / 256), dim3(256), 0, s, scales, scales_tiled,
                     count, k / group, tile_mul, tile_add);
  if ((e = hipGetLastError()) != hipSuccess || !zeros) return e;
  hipLaunchKernelGGL(tile_groups_kernel<uint8_t>, dim3((count + 255) / 256), dim3(256), 0, s, zeros, zeros_tiled, count,
                     k / group, tile_mul, tile_add);
  return hipGetLastError();
}

}  // namespace fh
