// K1 projections with 4-bit weights and group scales for decode batches
// (m <= 32 token rows) on gfx950 MFMA with FP32 accumulation.
//
//   y[m][n] = sum over groups g of s[n][g] * sum_{k in g} (q[n][k] - z[n][g]) x[m][k]
//
// with q in 0..15, groups of 32, 64 or 128 consecutive columns, bf16 scales s
// and zero points z (8 where none are given).
//
// A 4-bit weight enters the MFMA as the bf16 number 128 + q, which is exact (8
// significant bits: 128..143) and one and-or for two weights: the nibble is the
// low end of the mantissa of 0x4300. The 128 and the zero point come off per
// group, in FP32: sum (q - z) x = sum (128 + q) x - (128 + z) sum x, where sum x
// is the MFMA of the activations with a tile of ones, shared by the wave's
// weight tiles. The subtraction cancels: the terms are up to 136 / 7 of what is
// left, so the group's sum carries about 20 roundings' worth of FP32 error
// (2e-6 relative to a group's result), 1/2000 of the bf16 output's.
//
// Layout (fh_op_tile_weight_w4): a 16-row x 128-column tile is 1 KiB, one
// 16-byte load per lane; lane = row + 16 (column % 32 / 8), its four words are
// the four 32-column k-blocks, so word j is the A operand of k-block j's MFMA
// before unpacking: columns 2 i and 2 i + 1 of a word's eight at bits 4 i and
// 16 + 4 i, which (word >> 4 i) & 0x000f000f takes out as a pair. Tiles run
// k-fastest. Scales and zero points: [n / 16][groups][16], so the four rows of
// a lane's accumulators are one 8-byte (4-byte) load. Activations in their tile
// order (common.hpp act_offset). Lanes of rows past m read the last row again
// (less to fetch; their output columns are not stored).
#include "common.hpp"
#include "kernels.hpp"

namespace fh {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ bf16x8 unpack_w4(uint32_t w) {
  // Eight nibbles to bf16 128 + q.
  const u32x4 v = {(w & 0x000f000fu) | 0x43004300u, ((w >> 4) & 0x000f000fu) | 0x43004300u,
                   ((w >> 8) & 0x000f000fu) | 0x43004300u, ((w >> 12) & 0x000f000fu) | 0x43004300u};
  return __builtin_bit_cast(bf16x8, v);
}

// One workgroup: NT consecutive 16-row weight tiles and one split of k, whose
// 128-column blocks its waves divide; wave partials are added in wave order
// through LDS. GB: 32-column k-blocks per group. MT: 16-row activation tiles.
template <int NT, int MT, int GB, bool ZP, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void gemm_w4_kernel(const uint16_t* __restrict__ xt,
                                                            const uint32_t* __restrict__ w,
                                                            const uint16_t* __restrict__ scales,
                                                            const uint8_t* __restrict__ zeros, uint32_t m,
                                                            uint32_t kb_count, uint32_t kb_split, uint32_t epi,
                                                            const uint16_t* residual, void* out, uint32_t ldo,
                                                            uint32_t* err) {
  constexpr int GP = 4 / GB;  // groups per 128 columns
  __shared__ float red[WAVES][NT * MT * 256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tile0 = blockIdx.x * NT, split = blockIdx.y;
  const uint32_t s_lo = min(split * kb_split, kb_count), s_hi = min(s_lo + kb_split, kb_count), s_n = s_hi - s_lo;
  const uint32_t kb_lo = s_lo + (s_n * wave) / WAVES, kb_hi = s_lo + (s_n * (wave + 1)) / WAVES;
  const uint32_t r16 = lane & 15, g16 = lane >> 4;

  struct Stage {
    u32x4 w[NT], x[4][MT];
    uint2 s[NT][GP];
    uint32_t z[ZP ? NT : 1][GP];
  };
  const uint64_t kg = (uint64_t)kb_count * GP;
  auto load = [&](Stage& st, uint32_t kb) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      st.w[nt] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w) +
                                            ((uint64_t)(tile0 + nt) * kb_count + kb) * 64 + lane);
#pragma unroll
      for (int p = 0; p < GP; ++p) {
        const uint64_t at = ((uint64_t)(tile0 + nt) * kg + kb * GP + p) * 16 + 4 * g16;
        st.s[nt][p] = *reinterpret_cast<const uint2*>(scales + at);
        if constexpr (ZP) st.z[nt][p] = *reinterpret_cast<const uint32_t*>(zeros + at);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint32_t row = min(16 * mt + r16, m - 1) & 15u;
        st.x[j][mt] = *(reinterpret_cast<const u32x4*>(xt) + ((uint64_t)(4 * kb + j) * 2 + mt) * 64 + row + 16 * g16);
      }
  };

  f32x4 acc[NT][MT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  auto compute = [&](const Stage& st) {
#pragma unroll
    for (int p = 0; p < GP; ++p) {
      f32x4 sx[MT], part[NT][MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        sx[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) part[nt][mt] = sx[mt];
      }
#pragma unroll
      for (int b = 0; b < GB; ++b) {
        const int j = p * GB + b;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          sx[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(bf16x8, st.x[j][mt]), sx[mt], 0, 0, 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const bf16x8 a = unpack_w4(st.w[nt][j]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            part[nt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, st.x[j][mt]),
                                                                  part[nt][mt], 0, 0, 0);
        }
      }
      // Lane: activation row r16, weight rows 4 g16 + e.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float s[4] = {lo_bf16(st.s[nt][p].x), hi_bf16(st.s[nt][p].x), lo_bf16(st.s[nt][p].y),
                            hi_bf16(st.s[nt][p].y)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z = ZP ? 128.f + (float)((st.z[ZP ? nt : 0][p] >> (8 * e)) & 0xffu) : 136.f;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            acc[nt][mt][e] = __builtin_fmaf(s[e], __builtin_fmaf(-z, sx[mt][e], part[nt][mt][e]), acc[nt][mt][e]);
        }
      }
    }
  };
  Stage a, b;
  if (kb_lo < kb_hi) load(a, kb_lo);
  for (uint32_t kb = kb_lo; kb < kb_hi; kb += 2) {
    if (kb + 1 < kb_hi) load(b, kb + 1);
    __builtin_amdgcn_sched_barrier(0);
    compute(a);
    __builtin_amdgcn_sched_barrier(0);
    if (kb + 1 < kb_hi) {
      if (kb + 2 < kb_hi) load(a, kb + 2);
      __builtin_amdgcn_sched_barrier(0);
      compute(b);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][(nt * MT + mt) * 256 + r16 * 16 + 4 * g16 + e] = acc[nt][mt][e];
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
  hipLaunchKernelGGL((gemm_w4_kernel<NT, MT, GB, ZP, WAVES>), dim3(n / (16 * NT), splits), dim3(WAVES * 64), 0, s, xt, w,
                     scales, zeros, m, kb, (kb + splits - 1) / splits, epi, residual, out, ldo, err);
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
  const bool pair = n % 32 == 0 && (epilogue == FH_EPI_SWIGLU || n / 32 * splits >= 256);
  if (pair)
    launch_w4<2, 8>(x_tiled, w_tiled, scales, zeros, m, n, k, group, epilogue, splits, residual, out, ldo, err, s);
  else
    launch_w4<1, 8>(x_tiled, w_tiled, scales, zeros, m, n, k, group, epilogue, splits, residual, out, ldo, err, s);
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
