// Rows of bf16, fp16 or fp32 elements as fp32, and reductions over a wave: shared by the row operators.
#pragma once
#include "dgm_common.hpp"
#include "../../include/dgm_megamoe.h"

namespace dgm {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

enum { T_BF16 = DGM_SRC_BF16, T_F16 = DGM_SRC_F16, T_F32 = DGM_SRC_F32 };

template <int T>
DGM_DEV float load1(const void* p, int64_t i) {
  if constexpr (T == T_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (T == T_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  else return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}
template <int T>
DGM_DEV void store1(void* p, int64_t i, float v) {
  if constexpr (T == T_F32) reinterpret_cast<float*>(p)[i] = v;
  else if constexpr (T == T_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
  else reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
}
// eight 16-bit elements as fp32
template <int T>
DGM_DEV void unpack8(u4 w, float* v) {
  static_assert(T != T_F32, "16-bit elements");
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t d = w[k];        // (a scalar: the cast of a vector's element reads its first one)
    if constexpr (T == T_F16) {
      const h2 f = __builtin_bit_cast(h2, d);
      v[2 * k] = (float)f[0];
      v[2 * k + 1] = (float)f[1];
    } else {
      v[2 * k] = __uint_as_float(d << 16);
      v[2 * k + 1] = __uint_as_float(d & 0xffff0000u);
    }
  }
}
// eight consecutive elements from element i (16-byte aligned) as fp32, and back (round to nearest even)
template <int T>
DGM_DEV void load8(const void* p, int64_t i, float* v) {
  if constexpr (T == T_F32) {
    const f4* q = reinterpret_cast<const f4*>(reinterpret_cast<const float*>(p) + i);
    const f4 a = q[0], b = q[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[4 + k] = b[k]; }
  } else {
    unpack8<T>(*reinterpret_cast<const u4*>(reinterpret_cast<const uint16_t*>(p) + i), v);
  }
}
template <int T>
DGM_DEV void store8(void* p, int64_t i, const float* v) {
  if constexpr (T == T_F32) {
    f4* q = reinterpret_cast<f4*>(reinterpret_cast<float*>(p) + i);
    q[0] = f4{v[0], v[1], v[2], v[3]};
    q[1] = f4{v[4], v[5], v[6], v[7]};
  } else {
    u4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f2 f = {v[2 * k], v[2 * k + 1]};
      if constexpr (T == T_F16) w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, h2));
      else w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf2));
    }
    *reinterpret_cast<u4*>(reinterpret_cast<uint16_t*>(p) + i) = w;
  }
}

// Eight consecutive elements as they lie in memory.
typedef uint32_t loose_u4 __attribute__((ext_vector_type(4), aligned(2)));
template <int T>
struct Piece {
  u4 w[T == T_F32 ? 2 : 1];
  static constexpr int SIZE = T == T_F32 ? 4 : 2;
  // from element i on: on 16 bytes, or on an element's alignment
  DGM_DEV void load(const void* p, int64_t i) {
    const u4* q = reinterpret_cast<const u4*>(reinterpret_cast<const char*>(p) + i * SIZE);
    w[0] = q[0];
    if constexpr (T == T_F32) w[1] = q[1];
  }
  DGM_DEV void load_loose(const void* p, int64_t i) {
    const loose_u4* q = reinterpret_cast<const loose_u4*>(reinterpret_cast<const char*>(p) + i * SIZE);
    w[0] = q[0];
    if constexpr (T == T_F32) w[1] = q[1];
  }
  // drops the first `by` elements (0 to 7), zeros behind the last
  DGM_DEV void shift(int by) {
    if (by == 0) return;
    if constexpr (T == T_F32) {
      auto drop = [&](bool some, int n) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t from = k + n < 8 ? w[(k + n) / 4 % 2][(k + n) % 4] : 0u;
          if (some) w[k / 4][k % 4] = from;
        }
      };
      drop(by & 4, 4);
      drop(by & 2, 2);
      drop(by & 1, 1);
    } else {
      if (by & 4) w[0] = u4{w[0][2], w[0][3], 0u, 0u};
      if (by & 2) w[0] = u4{w[0][1], w[0][2], w[0][3], 0u};
      if (by & 1)
        w[0] = u4{w[0][0] >> 16 | w[0][1] << 16, w[0][1] >> 16 | w[0][2] << 16, w[0][2] >> 16 | w[0][3] << 16, w[0][3] >> 16};
    }
  }
  DGM_DEV void unpack(float* v) const {
    if constexpr (T == T_F32) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t d = w[k / 4][k % 4];
        v[k] = __uint_as_float(d);
      }
    } else {
      unpack8<T>(w[0], v);
    }
  }
};
// eight elements at an element's alignment, rounded to nearest even
template <int T>
DGM_DEV void store8_loose(void* p, int64_t i, const float* v) {
  if constexpr (T == T_F32) {
    loose_u4* q = reinterpret_cast<loose_u4*>(reinterpret_cast<float*>(p) + i);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      q[h] = u4{__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3])};
  } else {
    u4 w;
    store8<T>(&w, 0, v);
    *reinterpret_cast<loose_u4*>(reinterpret_cast<uint16_t*>(p) + i) = w;
  }
}

// Sum and maximum over the 64 lanes (all active), in every lane, in a fixed order.
DGM_DEV float wave_sum(float v) {
  v += dpp_f32<0xB1>(v);        // quad_perm [1,0,3,2]
  v += dpp_f32<0x4E>(v);        // quad_perm [2,3,0,1]
  v += dpp_f32<0x141>(v);       // row_half_mirror
  v += dpp_f32<0x140>(v);       // row_mirror: every lane of a 16-lane row holds its sum
  const int u = __float_as_int(v);
  return (__int_as_float(__builtin_amdgcn_readlane(u, 0)) + __int_as_float(__builtin_amdgcn_readlane(u, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(u, 32)) + __int_as_float(__builtin_amdgcn_readlane(u, 48)));
}
DGM_DEV float wave_max(float v) {
  v = max_lanes16(v);
  const int u = __float_as_int(v);
  return fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(u, 0)), __int_as_float(__builtin_amdgcn_readlane(u, 16))),
               fmaxf(__int_as_float(__builtin_amdgcn_readlane(u, 32)), __int_as_float(__builtin_amdgcn_readlane(u, 48))));
}

}  // namespace dgm
