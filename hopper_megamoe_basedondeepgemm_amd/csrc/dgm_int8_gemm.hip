// int8 x int8 product with a scale for each token and each channel (gfx950):
//   D[m][n] = sa[m] sb[n] sum_k A[m][k] B[n][k] (+ C[m][n] or C[n]),
// or, with SwiGLU over a gate and an up half of B's rows (I = N / 2 each),
//   D[m][i] = silu(min(g, c)) * clamp(u, -c, c), g = product with row i, u = with row I + i.
// Sums are exact in int32 (K <= 131071 keeps 128 * 128 K below 2^31); a sum is rounded to fp32 once, the
// scales, C and SwiGLU are fp32 and the result is rounded once to D's type.
//
// The weights are the matrix core's A operand and the tokens its B operand, so that a lane's result
// registers hold consecutive channels of one token.
#include "dgm_common.hpp"
#include "dgm_abi_internal.hpp"
#include <stdlib.h>

using namespace dgm;

namespace {

typedef int v16i __attribute__((ext_vector_type(16)));

DGM_DEV v16i mfma_i8_32x32x32(v4i a, v4i b, v16i c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }

DGM_DEV float swiglu(float g, float u, float clamp, bool fast) {
  g = fminf(g, clamp);
  u = fminf(fmaxf(u, -clamp), clamp);
  return g * (fast ? sigmoid<true>(g) : sigmoid<false>(g)) * u;
}

// Type of D (and C) and what is added, as compile-time values: f(integral_constant dtype, bool_constant add).
template <class F>
DGM_DEV void with_epilogue(const DgmInt8GemmArgs& P, F&& f) {
  using std::integral_constant;
  auto add = [&](auto t) {
    if (P.c) f(t, std::true_type{});
    else f(t, std::false_type{});
  };
  if (P.dtype == DGM_SRC_F32) add(integral_constant<int, DGM_SRC_F32>{});
  else if (P.dtype == DGM_SRC_F16) add(integral_constant<int, DGM_SRC_F16>{});
  else add(integral_constant<int, DGM_SRC_BF16>{});
}

// scales of channels n .. n + 3 (behind the last: its own)
DGM_DEV v4f load_scales(const DgmInt8GemmArgs& P, int64_t n, int64_t end) {
  v4f s;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = P.sfb[(n + i < end ? n + i : end - 1) * P.sfb_stride];
  return s;
}

template <int T>
DGM_DEV float c_value(const void* p, int64_t i) {
  if constexpr (T == DGM_SRC_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (T == DGM_SRC_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

// Orders a wave's LDS accesses before and after it, between its lanes.
DGM_DEV void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A 16-byte piece of token m's row from channel n on (eight channels, fp32: four), from LDS: C added, rounded,
// stored. vec: rows of D (and C) are 16-byte aligned.
template <int T, bool ADD>
DGM_DEV void put_piece(const DgmInt8GemmArgs& P, int64_t m, int64_t n, int64_t n_out, int vec, const float* from) {
  constexpr int E = T == DGM_SRC_F32 ? 4 : 8;
  if (n >= n_out) return;
  float v[E];
#pragma unroll
  for (int i = 0; i < E; i += 4) {
    const v4f f = *reinterpret_cast<const v4f*>(from + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[i + k] = f[k];
  }
  const int64_t at = m * P.d_stride + n, ct = m * P.c_stride + n;
  if (vec && n + E <= n_out) {
    if constexpr (T == DGM_SRC_F32) {
      if constexpr (ADD) {
        const v4f c = *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(P.c) + ct);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += c[i];
      }
      *reinterpret_cast<v4f*>(reinterpret_cast<float*>(P.d) + at) = v4f{v[0], v[1], v[2], v[3]};
    } else {
      if constexpr (ADD) {
        const v4i c = *reinterpret_cast<const v4i*>(reinterpret_cast<const uint16_t*>(P.c) + ct);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t w[1] = {(uint16_t)((uint32_t)c[i >> 1] >> (16 * (i & 1)))};
          v[i] += c_value<T>(w, 0);
        }
      }
      v4i o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = T == DGM_SRC_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) : __builtin_bit_cast(uint16_t, (__bf16)v[2 * i]);
        const uint32_t hi = T == DGM_SRC_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) : __builtin_bit_cast(uint16_t, (__bf16)v[2 * i + 1]);
        o[i] = (int)(lo | hi << 16);
      }
      *reinterpret_cast<v4i*>(reinterpret_cast<uint16_t*>(P.d) + at) = o;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (n + i >= n_out) continue;
      if constexpr (ADD) v[i] += c_value<T>(P.c, ct + i);
      if constexpr (T == DGM_SRC_F32) reinterpret_cast<float*>(P.d)[at + i] = v[i];
      else if constexpr (T == DGM_SRC_F16) reinterpret_cast<_Float16*>(P.d)[at + i] = (_Float16)v[i];
      else reinterpret_cast<__bf16*>(P.d)[at + i] = (__bf16)v[i];
    }
  }
}

// Channels n .. n + 3 of token m; WHOLE: all four exist and one store (one load of C) takes them.
template <int T, bool ADD, bool SWIGLU, bool WHOLE>
DGM_DEV void put4(const DgmInt8GemmArgs& P, int64_t m, int64_t n, int64_t n_out, float sa, v4f sb, v4f su, v4i acc, v4i up) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (float)acc[i] * (sa * sb[i]);
    if constexpr (SWIGLU) v[i] = swiglu(v[i], (float)up[i] * (sa * su[i]), P.clamp, P.fast_math);
  }
  const int64_t at = m * P.d_stride + n, ct = m * P.c_stride + n;
  if constexpr (WHOLE) {
    if constexpr (ADD) {
      if constexpr (T == DGM_SRC_F32) {
        const v4f c = *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(P.c) + ct);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += c[i];
      } else {
        const uint2 c = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(P.c) + ct);
        const uint16_t w[4] = {(uint16_t)c.x, (uint16_t)(c.x >> 16), (uint16_t)c.y, (uint16_t)(c.y >> 16)};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += c_value<T>(w, i);
      }
    }
    if constexpr (T == DGM_SRC_F32) {
      *reinterpret_cast<v4f*>(reinterpret_cast<float*>(P.d) + at) = v4f{v[0], v[1], v[2], v[3]};
    } else {
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        h[i] = T == DGM_SRC_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[i]) : __builtin_bit_cast(uint16_t, (__bf16)v[i]);
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(P.d) + at) = uint2{h[0] | h[1] << 16, h[2] | h[3] << 16};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n + i >= n_out) continue;
      if constexpr (ADD) v[i] += c_value<T>(P.c, ct + i);
      if constexpr (T == DGM_SRC_F32) reinterpret_cast<float*>(P.d)[at + i] = v[i];
      else if constexpr (T == DGM_SRC_F16) reinterpret_cast<_Float16*>(P.d)[at + i] = (_Float16)v[i];
      else reinterpret_cast<__bf16*>(P.d)[at + i] = (__bf16)v[i];
    }
  }
}

// 16 bytes of a row from k on. ALIGNED: K is a multiple of 16 and rows are 16-byte aligned. Behind K: zeros
// of a row whose partner may then hold anything (ZERO), else any bytes of the row.
template <bool ALIGNED, bool ZERO>
DGM_DEV v4i load16(const int8_t* row, int k, int K) {
  if constexpr (ALIGNED) {
    const v4i r = *reinterpret_cast<const v4i*>(row + (k < K ? k : K - 16));
    return !ZERO || k < K ? r : v4i{0, 0, 0, 0};
  } else {
    v4i r = {0, 0, 0, 0};
    if (k + 16 <= K) __builtin_memcpy(&r, row + k, 16);
    else
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (k + j < K) r[j >> 2] |= (int)((uint32_t)(uint8_t)row[k + j] << (8 * (j & 3)));
    return r;
  }
}

// Few tokens (16 MT at most per workgroup): the weights are read once, straight into registers. A
// workgroup takes 16 channels (SwiGLU: their gate and up rows), its eight waves the K blocks of 128 in
// turn (lane l: 32 bytes of row l % 16, so a block's rows are read in whole 128-byte lines); the waves'
// int32 sums meet in LDS.
template <int MT, bool SWIGLU, bool ALIGNED>
__global__ void __launch_bounds__(512) k_int8_gemm_rows(const DgmInt8GemmArgs P, int vec) {
  constexpr int W = 8, H = SWIGLU ? 2 : 1;
  __shared__ v4i sums[W][H * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4, K = (int)P.k;
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n, m0 = (int64_t)blockIdx.y * (16 * MT), n0 = (int64_t)blockIdx.x * 16;
  const int8_t* a[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + 16 * t + r;
    a[t] = P.a + (m < P.m ? m : P.m - 1) * P.a_stride;
  }
  const int8_t* b[H];
  b[0] = P.b + (n0 + r < n_out ? n0 + r : n_out - 1) * P.b_stride;
  if constexpr (SWIGLU) b[1] = b[0] + n_out * P.b_stride;
  v4i acc[H][MT];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[h][t] = v4i{0, 0, 0, 0};
  for (int k0 = wave * 128; k0 < K; k0 += W * 128) {
    const int k = k0 + 32 * g;
    v4i bv[H][2], av[MT][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int h = 0; h < H; ++h) bv[h][j] = load16<ALIGNED, false>(b[h], k + 16 * j, K);
#pragma unroll
      for (int t = 0; t < MT; ++t) av[t][j] = load16<ALIGNED, true>(a[t], k + 16 * j, K);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[h][t] = mfma_i8_16x16x64(bv[h][j], av[t][j], acc[h][t]);
  }
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[wave][h * MT + t][lane] = acc[h][t];
  __syncthreads();
  if (wave >= MT) return;
  const int64_t m = m0 + 16 * wave + r;
  if (m >= P.m) return;
  v4i s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int w = 0; w < W; ++w) s[h] += sums[w][h * MT + wave][lane];
  const int64_t n = n0 + 4 * g;
  if (n >= n_out) return;
  const float sa = P.sfa[m * P.sfa_stride];
  const v4f sb = load_scales(P, n, n_out), su = SWIGLU ? load_scales(P, n_out + n, 2 * n_out) : sb;
  with_epilogue(P, [&](auto t, auto add) {
    if (vec && n + 3 < n_out) put4<t.value, add.value, SWIGLU, true>(P, m, n, n_out, sa, sb, su, s[0], s[1]);
    else put4<t.value, add.value, SWIGLU, false>(P, m, n, n_out, sa, sb, su, s[0], s[1]);
  });
}

#ifndef SWZ
#define SWZ(r) (((r) >> 1) & 7)
#endif
__device__ const uint4 k_zeros = {0u, 0u, 0u, 0u};

// Many tokens: a workgroup computes BM tokens x BN channels over K steps of 128 bytes. Both operands' rows
// go from HBM / L2 straight into LDS, the next step's while the current one is multiplied (two buffers,
// one barrier a step). A row's eight 16-byte pieces lie permuted by the row's number, so that eight lanes
// reading one piece of eight rows meet eight different bank groups.
// SwiGLU: blocks of 32 channel rows alternate between gate and up rows, so that a wave holds both of a
// channel.
template <int BM, int BN, int WM, int WN, bool SWIGLU>
__global__ void __launch_bounds__(64 * WM * WN) k_int8_gemm_tiles(const DgmInt8GemmArgs P, int vec, int tiles_m, int tiles_n) {
  constexpr int W = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, ROWS = BM + BN, LOADS = ROWS / (8 * W);
  static_assert(ROWS % (8 * W) == 0 && BM % (8 * W) == 0 && (!SWIGLU || TN % 2 == 0), "whole loads per wave");
  __shared__ __attribute__((aligned(1024))) int8_t lds[2][ROWS * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), K = (int)P.k;
  // Workgroups go to the 8 XCDs in turn: each XCD gets a contiguous run of tiles, ordered in bands of 8
  // token tiles, so that the tiles an XCD works on at a time share rows in its L2.
  const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
  int tile = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (tile >= tiles) return;
  const int band = tile / (8 * tiles_n), in_band = tile - band * 8 * tiles_n, bm = min(8, tiles_m - 8 * band);
  const int64_t m0 = (int64_t)(8 * band + in_band % bm) * BM, n0 = (int64_t)(in_band / bm) * (SWIGLU ? BN / 2 : BN);
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n;
  // each wave's loads: LOADS times eight rows of the token tile, then of the channel tile
  const int piece = (lane & 7) ^ SWZ((wave & 1) * 8 + (lane >> 3));
  const int8_t* src[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = (i * W + wave) * 8 + (lane >> 3);
    if (i * W * 8 < BM) {
      const int64_t m = m0 + row;
      src[i] = P.a + (m < P.m ? m : P.m - 1) * P.a_stride + 16 * piece;
    } else {
      const int rb = row - BM;
      int64_t n = SWIGLU ? n0 + (rb >> 6) * 32 + (rb & 31) : n0 + rb;
      n = n < n_out ? n : n_out - 1;
      if (SWIGLU && (rb & 32)) n += n_out;
      src[i] = P.b + n * P.b_stride + 16 * piece;
    }
  }
  auto fetch = [&](int k0, int8_t* to) {
    if (k0 + 128 <= K) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[i] + k0),
                                         (__attribute__((address_space(3))) void*)(to + (i * W + wave) * 1024), 16, 0, 0);
    } else {
      // (the pieces behind K: zeros)
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(k0 + 16 * piece < K ? src[i] + k0 : (const int8_t*)&k_zeros),
            (__attribute__((address_space(3))) void*)(to + (i * W + wave) * 1024), 16, 0, 0);
    }
  };
  v16i acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m) acc[n][m] = v16i{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  const int r = lane & 31, half = lane >> 5, wm = wave % WM, wn = wave / WM;
  const int row_a = wm * (BM / WM) + r, row_b = BM + wn * (BN / WN) + r;
  auto multiply = [&](const int8_t* from) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const int at = ((2 * kk + half) ^ SWZ(r)) * 16;
      v4i av[TM], bv[TN];
#pragma unroll
      for (int m = 0; m < TM; ++m) av[m] = *reinterpret_cast<const v4i*>(from + (row_a + 32 * m) * 128 + at);
#pragma unroll
      for (int n = 0; n < TN; ++n) bv[n] = *reinterpret_cast<const v4i*>(from + (row_b + 32 * n) * 128 + at);
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[n][m] = mfma_i8_32x32x32(bv[n], av[m], acc[n][m]);
    }
  };
  fetch(0, lds[0]);
  for (int k0 = 0, turn = 0; k0 < K; k0 += 128, turn ^= 1) {
    __builtin_amdgcn_s_waitcnt(0x0F70);      // this wave's loads of the step have landed,
    __syncthreads();                         // everyone's, and the other buffer is read
    if (k0 + 128 < K) fetch(k0 + 128, lds[turn ^ 1]);
    multiply(lds[turn]);
  }
  // Results through LDS, 32 tokens of a wave at a time: from the lanes' four channels of 32 tokens to 16-byte
  // pieces of whole token rows (rows padded by 16 bytes, so that neither side meets bank conflicts).
  constexpr int H = SWIGLU ? 2 : 1, CW = 32 * TN / H, PITCH = CW + 4;
  static_assert(W * 32 * PITCH * 4 <= (int)sizeof(lds), "the waves' parts fit");
  __syncthreads();
  float* part = reinterpret_cast<float*>(&lds[0][0]) + wave * 32 * PITCH;
  const int64_t c0 = n0 + wn * CW, t0 = m0 + wm * (BM / WM);
  v4f sb[TN][4];
#pragma unroll
  for (int n = 0; n < TN; n += H)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t c = c0 + 32 * n / H + 8 * q + 4 * half;
      sb[n][q] = load_scales(P, c, n_out);
      if constexpr (SWIGLU) sb[n + 1][q] = load_scales(P, n_out + c, 2 * n_out);
    }
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int64_t token = t0 + 32 * m + r;
    const float sa = P.sfa[(token < P.m ? token : P.m - 1) * P.sfa_stride];
#pragma unroll
    for (int n = 0; n < TN; n += H)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v4f v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = (float)acc[n][m][4 * q + i] * (sa * sb[n][q][i]);
          if constexpr (SWIGLU) v[i] = swiglu(v[i], (float)acc[n + 1][m][4 * q + i] * (sa * sb[n + 1][q][i]), P.clamp, P.fast_math);
        }
        *reinterpret_cast<v4f*>(part + r * PITCH + 32 * n / H + 8 * q + 4 * half) = v;
      }
    wave_sync();
    with_epilogue(P, [&](auto t, auto add) {
      constexpr int E = t.value == DGM_SRC_F32 ? 4 : 8, L = CW / E;      // elements of a piece, pieces of a row
#pragma unroll
      for (int j = 0; j < 32 * L / 64; ++j) {
        const int row = (64 * j + lane) / L, col = (64 * j + lane) % L * E;
        if (t0 + 32 * m + row < P.m)
          put_piece<t.value, add.value>(P, t0 + 32 * m + row, c0 + col, n_out, vec, part + row * PITCH + col);
      }
    });
    wave_sync();
  }
}

template <int MT>
void launch_rows(const DgmInt8GemmArgs& A, bool aligned, int vec, hipStream_t stream) {
  const int64_t n_out = A.swiglu ? A.n / 2 : A.n;
  const dim3 grid((unsigned)((n_out + 15) / 16), (unsigned)((A.m + 16 * MT - 1) / (16 * MT)));
  if (A.swiglu && aligned) hipLaunchKernelGGL((k_int8_gemm_rows<MT, true, true>), grid, dim3(512), 0, stream, A, vec);
  else if (A.swiglu) hipLaunchKernelGGL((k_int8_gemm_rows<MT, true, false>), grid, dim3(512), 0, stream, A, vec);
  else if (aligned) hipLaunchKernelGGL((k_int8_gemm_rows<MT, false, true>), grid, dim3(512), 0, stream, A, vec);
  else hipLaunchKernelGGL((k_int8_gemm_rows<MT, false, false>), grid, dim3(512), 0, stream, A, vec);
}

template <int BM, int BN, int WM, int WN>
void launch_tiles(const DgmInt8GemmArgs& A, int vec, hipStream_t stream) {
  const int tiles_m = (int)((A.m + BM - 1) / BM), tiles_n = (int)((A.n + BN - 1) / BN);
  const dim3 grid((unsigned)((tiles_m * tiles_n + 7) / 8 * 8));
  if (A.swiglu) hipLaunchKernelGGL((k_int8_gemm_tiles<BM, BN, WM, WN, true>), grid, dim3(64 * WM * WN), 0, stream, A, vec, tiles_m, tiles_n);
  else hipLaunchKernelGGL((k_int8_gemm_tiles<BM, BN, WM, WN, false>), grid, dim3(64 * WM * WN), 0, stream, A, vec, tiles_m, tiles_n);
}

}  // namespace

extern "C" {

int dgm_int8_gemm_struct_size(size_t* args) {
  DGM_CHECK_ARG(args, "null pointer");
  *args = sizeof(DgmInt8GemmArgs);
  return 0;
}

int dgm_int8_gemm_nt(const DgmInt8GemmArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmInt8GemmArgs A = *args;
  DGM_CHECK_ARG(A.dtype >= DGM_SRC_BF16 && A.dtype <= DGM_SRC_F32, "dtype 0 bf16, 1 fp16, 2 fp32");
  DGM_CHECK_ARG(A.m >= 0 && A.m < (1 << 20) && A.n >= 0 && A.n < (1 << 24), "m below 2^20, n below 2^24");
  DGM_CHECK_ARG(A.k > 0 && A.k <= DGM_INT8_GEMM_MAX_K, "k 1 to 131071 (int32 sums)");
  DGM_CHECK_ARG(!A.swiglu || (A.n % 2 == 0 && !A.c), "SwiGLU: a gate and an up half, no C");
  DGM_CHECK_ARG(A.a_stride >= 0 && A.b_stride >= 0 && A.sfa_stride >= 0 && A.sfb_stride >= 0 && A.c_stride >= 0 &&
                    A.d_stride >= 0, "strides >= 0");
  if (A.m == 0 || A.n == 0) return 0;
  DGM_CHECK_ARG(A.a && A.b && A.sfa && A.sfb && A.d, "null pointer");
  // 16-byte pieces of both operands; stores (and loads of C)
  const int e = A.dtype == DGM_SRC_F32 ? 4 : 2;
  const bool aligned = (A.k % 16 | A.a_stride % 16 | A.b_stride % 16) == 0 && (((uintptr_t)A.a | (uintptr_t)A.b) & 15) == 0;
  const int vec = (((uintptr_t)A.d | (uintptr_t)A.c | (uint64_t)(A.d_stride * e) | (uint64_t)(A.c_stride * e)) & 15) == 0;
  const char* force = getenv("DGM_GEMM");
  const int f = force ? atoi(force) : 0;
  if (f == 1 || (f == 0 && A.m >= 512 && aligned)) launch_tiles<256, 256, 2, 4>(A, vec, stream);
  else if (f == 2 || (f == 0 && A.m > 64 && aligned)) launch_tiles<128, 128, 2, 2>(A, vec, stream);
  else if (A.m <= 16) launch_rows<1>(A, aligned, vec, stream);
  else if (A.m <= 32) launch_rows<2>(A, aligned, vec, stream);
  else launch_rows<4>(A, aligned, vec, stream);
  return dgm_last_launch_status();
}

}  // extern "C"
