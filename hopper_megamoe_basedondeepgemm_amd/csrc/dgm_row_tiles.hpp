// Rows of up to 16384 elements, each in the registers of one workgroup: what the norms share.
#pragma once
#include "dgm_rows.hpp"

namespace dgm {

// The elements of a row that a thread holds. VEC: eight consecutive ones per 16-byte aligned chunk
// (H a multiple of 8), else single ones, a wave's loads contiguous in both.
template <int NV, int THREADS, bool VEC>
struct Row {
  static constexpr int N = 8 * NV;
  static DGM_DEV int index(int k) {
    if constexpr (VEC) return ((k >> 3) * THREADS + (int)threadIdx.x) * 8 + (k & 7);
    else return k * THREADS + (int)threadIdx.x;
  }
  template <int T>
  static DGM_DEV void load(const void* p, int64_t off, int H, float* v) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = (j * THREADS + (int)threadIdx.x) * 8;
        if constexpr (T == T_F32) {
          if (i < H) load8<T>(p, off + i, v + 8 * j);
          else
#pragma unroll
            for (int k = 0; k < 8; ++k) v[8 * j + k] = 0.f;
        } else {
          // (converted behind the branch: with the conversion in it the fp16 values of two chunks met through scratch
          // memory, 8192 x 4096 78 us instead of 46)
          u4 w = {0u, 0u, 0u, 0u};
          if (i < H) w = *reinterpret_cast<const u4*>(reinterpret_cast<const uint16_t*>(p) + off + i);
          unpack8<T>(w, v + 8 * j);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = index(k) < H ? load1<T>(p, off + index(k)) : 0.f;
    }
  }
  template <int T>
  static DGM_DEV void store(void* p, int64_t off, int H, const float* v) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = (j * THREADS + (int)threadIdx.x) * 8;
        if (i < H) store8<T>(p, off + i, v + 8 * j);
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (index(k) < H) store1<T>(p, off + index(k), v[k]);
    }
  }
  // norm weights: the rows' type or fp32
  template <int T>
  static DGM_DEV void weight(const void* p, bool f32, int H, float* v) {
    if (f32) load<T_F32>(p, 0, H, v);
    else load<T>(p, 0, H, v);
  }
};

// The same elements as Row<NV, THREADS, true> holds, of rows of any length at any alignment: 16 bytes at a time on the
// elements' alignment, a row's last piece from its last eight elements (up to seven are the thread's before it, which may
// be in another wave; they are dropped). Where a row's memory is written too, every thread has to have its elements first.
template <int NV, int THREADS>
struct LooseRow : Row<NV, THREADS, true> {
  template <int T>
  static DGM_DEV void load(const void* p, int64_t off, int H, float* v) {
    if (H < 8) {                                   // (thread 0's alone)
#pragma unroll
      for (int k = 0; k < 8 * NV; ++k) v[k] = LooseRow::index(k) < H ? load1<T>(p, off + LooseRow::index(k)) : 0.f;
      return;
    }
    Piece<T> piece[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) piece[j].load_loose(p, off + min(LooseRow::index(8 * j), H - 8));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = LooseRow::index(8 * j);
      piece[j].shift(min(max(i - (H - 8), 0), 7));
      piece[j].unpack(v + 8 * j);
      if (i >= H)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[8 * j + k] = 0.f;
    }
  }
  template <int T>
  static DGM_DEV void store(void* p, int64_t off, int H, const float* v) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = LooseRow::index(8 * j);
      if (i + 8 <= H) {
        store8_loose<T>(p, off + i, v + 8 * j);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i + k < H) store1<T>(p, off + i + k, v[8 * j + k]);
      }
    }
  }
  template <int T>
  static DGM_DEV void weight(const void* p, bool f32, int H, float* v) {
    if (f32) load<T_F32>(p, 0, H, v);
    else load<T>(p, 0, H, v);
  }
};

// Workgroup reductions of up to two values, in a fixed order, one barrier each. Two LDS sets taken in
// turn: a set is written again only after the barrier of the other one, which a wave reaches after it
// has read the first. Behind the barrier every lane takes a wave's value and they meet by lane exchange (each
// thread reading all of them in turn: 64 x 7168 with int8 rows 6.7 us, so 6.35).
template <int THREADS>
struct Reduce {
  static constexpr int W = THREADS / 64;
  float (*lds)[W][2];
  int turn = 0;
  // The waves' values meet across lanes: lane l takes that of wave l % W.
  template <bool MAX>
  static DGM_DEV float join(float v) {
    auto with = [&](float u) { v = MAX ? fmaxf(v, u) : v + u; };
    if constexpr (W >= 2) with(dpp_f32<0xB1>(v));        // quad_perm [1,0,3,2]
    if constexpr (W >= 4) with(dpp_f32<0x4E>(v));        // quad_perm [2,3,0,1]
    if constexpr (W >= 8) with(dpp_f32<0x141>(v));       // row_half_mirror
    if constexpr (W >= 16) with(dpp_f32<0x140>(v));      // row_mirror
    return v;
  }
  template <bool MAX = false>
  DGM_DEV void run(float& a) {
    a = MAX ? wave_max(a) : wave_sum(a);
    if constexpr (W > 1) {
      const int lane = threadIdx.x & 63;
      if (lane == 0) lds[turn][threadIdx.x >> 6][0] = a;
      __syncthreads();
      a = join<MAX>(lds[turn][lane & (W - 1)][0]);
      turn ^= 1;
    }
  }
  DGM_DEV void run(float& a, float& b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (W > 1) {
      const int lane = threadIdx.x & 63;
      if (lane == 0) {
        lds[turn][threadIdx.x >> 6][0] = a;
        lds[turn][threadIdx.x >> 6][1] = b;
      }
      __syncthreads();
      a = join<false>(lds[turn][lane & (W - 1)][0]);
      b = join<false>(lds[turn][lane & (W - 1)][1]);
      turn ^= 1;
    }
  }
};

// Eight elements of 16 bits as they were loaded (a row requested ahead of its turn).
struct Held {
  u4 w;
  DGM_DEV void load(const void* p, int64_t off, int H) {
    const int i = (int)threadIdx.x * 8;
    w = u4{0u, 0u, 0u, 0u};
    if (i < H) w = *reinterpret_cast<const u4*>(reinterpret_cast<const uint16_t*>(p) + off + i);
  }
};

// The same of any type T.
struct HeldRow {
  u4 a, b;
  template <int T>
  DGM_DEV void load(const void* p, int64_t off, int H) {
    const int i = (int)threadIdx.x * 8;
    a = b = u4{0u, 0u, 0u, 0u};
    if (i >= H) return;
    if constexpr (T == T_F32) {
      const u4* q = reinterpret_cast<const u4*>(reinterpret_cast<const float*>(p) + off + i);
      a = q[0], b = q[1];
    } else {
      a = *reinterpret_cast<const u4*>(reinterpret_cast<const uint16_t*>(p) + off + i);
    }
  }
  template <int T>
  DGM_DEV void unpack(float* v) const {
    if constexpr (T == T_F32) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = a[k], hi = b[k];
        v[k] = __uint_as_float(lo), v[4 + k] = __uint_as_float(hi);
      }
    } else {
      unpack8<T>(a, v);
    }
  }
};

static inline bool aligned(const void* p, int64_t stride, int size) {
  return !p || (((uintptr_t)p & 15) == 0 && (stride * size) % 16 == 0);
}

template <class F>
void dispatch_type(int dtype, bool vec, F&& f) {
  using std::integral_constant;
  auto v = [&](auto t) {
    if (vec) f(t, std::true_type{});
    else f(t, std::false_type{});
  };
  if (dtype == DGM_SRC_BF16) v(integral_constant<int, T_BF16>{});
  else if (dtype == DGM_SRC_F16) v(integral_constant<int, T_F16>{});
  else v(integral_constant<int, T_F32>{});
}

static inline int element_size(int dtype) { return dtype == DGM_SRC_F32 ? 4 : 2; }

}  // namespace dgm
