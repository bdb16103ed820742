// What follows the sums of a product of token rows with weight rows: SwiGLU, C added, results rounded once and stored.
// Args: the arguments of the product (dtype, c, c_stride, d, d_stride). Shared by the products around the layer.
#pragma once
#include "dgm_common.hpp"
#include "../../include/dgm_megamoe.h"

namespace dgm {

// (compared, not fminf / fmaxf, which put the clamp in the place of what is no number)
DGM_DEV float swiglu(float g, float u, float clamp, bool fast) {
  g = g > clamp ? clamp : g;
  u = u > clamp ? clamp : u < -clamp ? -clamp : u;
  return g * (fast ? sigmoid<true>(g) : sigmoid<false>(g)) * u;
}

// Type of D (and C) and what is added, as compile-time values: f(integral_constant dtype, bool_constant add).
template <class Args, class F>
DGM_DEV void with_epilogue(const Args& P, F&& f) {
  using std::integral_constant;
  auto add = [&](auto t) {
    if (P.c) f(t, std::true_type{});
    else f(t, std::false_type{});
  };
  if (P.dtype == DGM_SRC_F32) add(integral_constant<int, DGM_SRC_F32>{});
  else if (P.dtype == DGM_SRC_F16) add(integral_constant<int, DGM_SRC_F16>{});
  else add(integral_constant<int, DGM_SRC_BF16>{});
}

template <int T>
DGM_DEV float c_value(const void* p, int64_t i) {
  if constexpr (T == DGM_SRC_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (T == DGM_SRC_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

// 16 and 8 bytes of C or D, on 4 bytes at least
typedef int g4i __attribute__((ext_vector_type(4), aligned(4)));
typedef float g4f __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t g2u __attribute__((ext_vector_type(2), aligned(4)));

// Orders a wave's LDS accesses before and after it, between its lanes.
DGM_DEV void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A 16-byte piece of token m's row from channel n on (eight channels, fp32: four), from LDS: C added, rounded,
// stored. vec: rows of D (and C) are 4-byte aligned.
template <int T, bool ADD, class Args>
DGM_DEV void put_piece(const Args& P, int64_t m, int64_t n, int64_t n_out, int vec, const float* from) {
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
        const v4f c = *reinterpret_cast<const g4f*>(reinterpret_cast<const float*>(P.c) + ct);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += c[i];
      }
      *reinterpret_cast<g4f*>(reinterpret_cast<float*>(P.d) + at) = g4f{v[0], v[1], v[2], v[3]};
    } else {
      if constexpr (ADD) {
        const v4i c = *reinterpret_cast<const g4i*>(reinterpret_cast<const uint16_t*>(P.c) + ct);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t w[1] = {(uint16_t)((uint32_t)c[i >> 1] >> (16 * (i & 1)))};
          v[i] += c_value<T>(w, 0);
        }
      }
      g4i o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = T == DGM_SRC_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) : __builtin_bit_cast(uint16_t, (__bf16)v[2 * i]);
        const uint32_t hi = T == DGM_SRC_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) : __builtin_bit_cast(uint16_t, (__bf16)v[2 * i + 1]);
        o[i] = (int)(lo | hi << 16);
      }
      *reinterpret_cast<g4i*>(reinterpret_cast<uint16_t*>(P.d) + at) = o;
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
template <int T, bool ADD, bool WHOLE, class Args>
DGM_DEV void put4(const Args& P, int64_t m, int64_t n, int64_t n_out, float* v) {
  const int64_t at = m * P.d_stride + n, ct = m * P.c_stride + n;
  if constexpr (WHOLE) {
    if constexpr (ADD) {
      if constexpr (T == DGM_SRC_F32) {
        const v4f c = *reinterpret_cast<const g4f*>(reinterpret_cast<const float*>(P.c) + ct);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += c[i];
      } else {
        const g2u c = *reinterpret_cast<const g2u*>(reinterpret_cast<const uint16_t*>(P.c) + ct);
        const uint32_t lo = c[0], hi = c[1];
        const uint16_t w[4] = {(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += c_value<T>(w, i);
      }
    }
    if constexpr (T == DGM_SRC_F32) {
      *reinterpret_cast<g4f*>(reinterpret_cast<float*>(P.d) + at) = g4f{v[0], v[1], v[2], v[3]};
    } else {
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        h[i] = T == DGM_SRC_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[i]) : __builtin_bit_cast(uint16_t, (__bf16)v[i]);
      *reinterpret_cast<g2u*>(reinterpret_cast<uint16_t*>(P.d) + at) = g2u{h[0] | h[1] << 16, h[2] | h[3] << 16};
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

}  // namespace dgm
