// Norms around a block (gfx950): the root-mean-square norm behind it, its gate, the scaled residual
// add and the norm before the next block in one pass over the rows, and the gradients of all of them.
//
// Row of H elements, n = x rstd1 w1 (rstd1 = rsqrt(mean x^2 + eps); n = x without w1), a = gate or
// sigmoid(gate), t = r + s a n, u = t rstd2, h = u w2. Everything between the loads and the stores is
// fp32 and t enters the second norm unrounded. A workgroup owns a row, a thread 8 NV of its elements in
// registers, so each input is read once whatever the number of norms; the bound is HBM.
// Gradients, with R = dL/dt (of the stored t) and D = dL/dh:
//   du = D w2, R' = R + rstd2 (du - u mean(du u)), dr = R', dw2 = sum D u,
//   da = s R' n, dn = s R' a, dw1 = sum dn z, dz = dn w1, dx = rstd1 (dz - z mean(dz z)), z = x rstd1.
#include "dgm_common.hpp"
#include "dgm_abi_internal.hpp"
#include "dgm_row_tiles.hpp"

using namespace dgm;

namespace {

// Gates. 16-bit rows: the hardware's exp2 and reciprocal, within (4 + |g|) 2^-24 of the value, far below half a step of
// their type (with IEEE expf and division 8192 x 4096 bf16 under a channel gate took 64 us, so 55). fp32 rows: the
// exponent's rounding put back, within 8 2^-24 (the exponential 4, the reciprocal 2, the sum and the product 1 each).
template <int T>
DGM_DEV float gate_sigmoid(float g) {
  if constexpr (T != T_F32) return sigmoid<true>(g);
  float x = -fabsf(g);
  x = x < -126.0f ? -126.0f : x;                 // (0 there; a gate that is no number stays one)
  const float h = x * 1.4426950408889634f;
  const float low = fmaf(x, 1.925963033500569e-8f, fmaf(x, 1.4426950408889634f, -h));
  float e = __builtin_amdgcn_exp2f(h);
  e = fmaf(e, low * 0.6931471805599453f, e);
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  return g < 0.f ? e * r : r;
}

enum { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_TOKEN = 2, GATE_FULL = 3 };

template <int T, int NV, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS) k_norm_fwd(const DgmNormArgs P) {
  using R = Row<NV, THREADS, VEC>;
  constexpr int N = R::N;
  __shared__ float lds[2][THREADS / 64][2];
  Reduce<THREADS> red{lds};
  const int H = P.hidden;
  const int64_t row = blockIdx.x;
  const bool wf = P.weights_f32;
  const float inv_h = 1.0f / (float)H;
  float t[N], w[N];
  // Rows of eight elements a thread: everything is requested at the start, so that a row waits for memory once
  // (64 x 4096 3.3 -> 3.0 us, 4096 x 4096 fp32 under a full gate 62.6 -> 60.7).
  constexpr bool EARLY = VEC && NV == 1;
  HeldRow hx, h1, hg, hr, h2;
  if constexpr (EARLY) {
    hx.load<T>(P.x, row * P.x_stride, H);
    if (P.residual) hr.load<T>(P.residual, row * P.residual_stride, H);
    if (P.post_weight) {
      if (wf) h1.load<T_F32>(P.post_weight, 0, H);
      else h1.load<T>(P.post_weight, 0, H);
    }
    if (P.gate_mode == GATE_CHANNEL || P.gate_mode == GATE_FULL) hg.load<T>(P.gate, P.gate_mode == GATE_FULL ? row * P.gate_stride : 0, H);
    if (P.pre_weight) {
      if (wf) h2.load<T_F32>(P.pre_weight, 0, H);
      else h2.load<T>(P.pre_weight, 0, H);
    }
  }
  auto get = [&](const HeldRow& held, const void* p, int64_t off, float* v) {
    if constexpr (EARLY) held.unpack<T>(v);
    else R::template load<T>(p, off, H, v);
  };
  auto get_weight = [&](const HeldRow& held, const void* p) {
    if constexpr (EARLY) {
      if (wf) held.unpack<T_F32>(w);
      else held.unpack<T>(w);
    } else {
      R::template weight<T>(p, wf, H, w);
    }
  };
  get(hx, P.x, row * P.x_stride, t);
  if (P.post_weight) {
    get_weight(h1, P.post_weight);
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) ss += t[k] * t[k];
    red.run(ss);
    const float rstd = 1.0f / sqrtf(ss * inv_h + P.eps);
    if (P.rstd_post && threadIdx.x == 0) P.rstd_post[row] = rstd;
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = t[k] * rstd * w[k];
  }
  if (P.gate_mode != GATE_NONE) {
    if (P.gate_mode == GATE_TOKEN) {
      float a = load1<T>(P.gate, row * P.gate_stride);
      if (P.gate_sigmoid) a = gate_sigmoid<T>(a);
#pragma unroll
      for (int k = 0; k < N; ++k) t[k] *= a;
    } else {
      get(hg, P.gate, P.gate_mode == GATE_FULL ? row * P.gate_stride : 0, w);
#pragma unroll
      for (int k = 0; k < N; ++k) t[k] *= P.gate_sigmoid ? gate_sigmoid<T>(w[k]) : w[k];
    }
  }
  if (P.residual) {
    get(hr, P.residual, row * P.residual_stride, w);
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = w[k] + P.residual_scale * t[k];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] *= P.residual_scale;
  }
  if (P.residual_out) R::template store<T>(P.residual_out, row * P.residual_out_stride, H, t);
  if (!P.pre_weight) return;
  get_weight(h2, P.pre_weight);
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (R::index(k) < H) ss += t[k] * t[k];
  red.run(ss);
  const float rstd = 1.0f / sqrtf(ss * inv_h + P.eps);
  if (P.rstd_pre && threadIdx.x == 0) P.rstd_pre[row] = rstd;
#pragma unroll
  for (int k = 0; k < N; ++k) t[k] = t[k] * rstd * w[k];
  if (P.h) R::template store<T>(P.h, row * P.h_stride, H, t);
  if constexpr (T == T_BF16) {
    if (!P.q) return;
    // int8 rows of the rounded h (the rule of dgm_cast_int8_rows): sf = max(amax, 1e-30) / 127,
    // q = clamp(rne(h / sf), +-127)
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      t[k] = round_bf16(t[k]);
      amax = fmaxf(amax, R::index(k) < H ? fabsf(t[k]) : 0.f);
    }
    red.template run<true>(amax);
    const float s = fmaxf(amax, 1e-30f) / 127.0f;
    if (threadIdx.x == 0) P.q_sf[row] = s;
    // h / s by the reciprocal and one correction: rounded to a whole number it is the quotient's for every bf16
    // amax and every bf16 h up to it (all 5.3e8 pairs compared on the CPU; the reciprocal alone misses 5464).
    // amax infinite: step 0 leaves 0, and NaN for the infinite ones. (A division each: 1024 x 7168 17.4 us.)
    const float inv = 1.0f / s, step = s == INFINITY ? 0.f : s;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float quotient = t[k] * inv;
      t[k] = fminf(fmaxf(rintf(fmaf(fmaf(-quotient, step, t[k]), inv, quotient)), -127.f), 127.f);
    }
    int8_t* q = P.q + row * (int64_t)H;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = (j * THREADS + (int)threadIdx.x) * 8;
        uint32_t d[2] = {0u, 0u};
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k >> 2] |= ((uint32_t)(int)t[8 * j + k] & 0xffu) << (8 * (k & 3));
        if (i < H) *reinterpret_cast<uint2*>(q + i) = uint2{d[0], d[1]};
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (R::index(k) < H) q[R::index(k)] = (int8_t)t[k];
    }
  }
}

// Gradients: workgroup g takes rows g, g + G, ...; the columns' sums over its rows stay in registers and
// go to partial[set][g][H] (set 0 pre weight, 1 post weight, 2 channel gate), which k_norm_columns adds up
// in a fixed order.
// SIG: a gate, under a sigmoid (a kernel of its own: with it in the others' way, those that spill take up to 17 % longer
// for rows without one).
template <int T, int NV, int THREADS, bool VEC, bool SIG>
__global__ void __launch_bounds__(THREADS) k_norm_bwd(const DgmNormGradArgs P) {
  using R = Row<NV, THREADS, VEC>;
  constexpr int N = R::N;
  __shared__ float lds[2][THREADS / 64][2];
  Reduce<THREADS> red{lds};
  const DgmNormArgs& F = P.forward;
  const int H = F.hidden;
  const float inv_h = 1.0f / (float)H;
  float dw2[N], dw1[N], dg[N];
#pragma unroll
  for (int k = 0; k < N; ++k) dw2[k] = dw1[k] = dg[k] = 0.f;
  // 16-bit rows of eight elements a thread: the next row, with its rstd and token gate, is requested before
  // the current one is worked on, and the weights wait in LDS (each thread's own): loads are awaited in
  // their order, so weights read from memory in the loop would wait for the next row first.
  constexpr bool AHEAD = VEC && T != T_F32 && NV == 1;
  // A channel gate waits in LDS in all rows of eight elements a thread: its sigmoid and derivative are one row's work,
  // not every row's.
  constexpr bool HELD_GATE = NV == 1;
  constexpr int GATE = AHEAD ? 2 : 0;            // the gate's two sets, behind the weights'
  __shared__ f4 held_w[AHEAD ? 4 : HELD_GATE ? 2 : 1][2][HELD_GATE ? THREADS : 1];
  Held hx, hr, hd, hg, ha;
  float next_rstd1 = 1.f, next_rstd2 = 0.f, next_gate = 1.f;
  auto scalars = [&](int64_t row) {
    if (F.post_weight) next_rstd1 = F.rstd_post[row];
    if (P.d_h) next_rstd2 = F.rstd_pre[row];
    if (F.gate_mode == GATE_TOKEN) next_gate = load1<T>(F.gate, row * F.gate_stride);
  };
  auto request = [&](int64_t row) {
    hx.load(F.x, row * F.x_stride, H);
    if (F.residual && P.d_h) hr.load(F.residual, row * F.residual_stride, H);
    if (P.d_h) hd.load(P.d_h, row * P.d_h_stride, H);
    if (P.d_residual_out) hg.load(P.d_residual_out, row * P.d_residual_out_stride, H);
    if (F.gate_mode == GATE_FULL) ha.load(F.gate, row * F.gate_stride, H);
    scalars(row);
  };
  auto keep = [&](const float* v, int set) {
    held_w[set][0][threadIdx.x] = f4{v[0], v[1], v[2], v[3]};
    held_w[set][1][threadIdx.x] = f4{v[4], v[5], v[6], v[7]};
  };
  auto keep_weight = [&](const void* p, bool f32, int set) {
    float v[N];
    R::template weight<T>(p, f32, H, v);
    keep(v, set);
  };
  auto held = [&](int set, float* v) {
    const f4 lo = held_w[set][0][threadIdx.x], hi = held_w[set][1][threadIdx.x];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = lo[k], v[4 + k] = hi[k];
  };
  auto weight = [&](const void* p, bool f32, int set, float* v) {
    if constexpr (AHEAD) held(set, v);
    else R::template weight<T>(p, f32, H, v);
  };
  if constexpr (AHEAD) {
    if (F.post_weight) keep_weight(F.post_weight, F.weights_f32, 0);
    if (F.pre_weight) keep_weight(F.pre_weight, F.weights_f32, 1);
  }
  if constexpr (HELD_GATE) {
    if (F.gate_mode == GATE_CHANNEL) {
      float v[N], d[N];
      R::template load<T>(F.gate, 0, H, v);
      if constexpr (SIG) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float rest = gate_sigmoid<T>(-v[k]);
          v[k] = gate_sigmoid<T>(v[k]);
          d[k] = v[k] * rest;
        }
        keep(d, GATE + 1);
      }
      keep(v, GATE);
    }
  }
  if constexpr (AHEAD) {
    if ((int64_t)blockIdx.x < F.rows) request(blockIdx.x);
  }
  for (int64_t row = blockIdx.x; row < F.rows; row += gridDim.x) {
    float x[N], t[N], a[N], w[N], g[N];
    Held cx, cr, cd, cg, ca;
    if constexpr (!AHEAD) scalars(row);
    // (the same in every lane: scalar registers, as the vector ones are short)
    auto scalar = [](float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); };
    const float rstd1 = scalar(next_rstd1), rstd2 = scalar(next_rstd2), token_gate = scalar(next_gate);
    if constexpr (AHEAD) {
      cx = hx, cr = hr, cd = hd, cg = hg, ca = ha;
      const int64_t next = row + gridDim.x;
      if (next < F.rows) request(next);
      unpack8<T>(cx.w, x);
    } else {
      R::template load<T>(F.x, row * F.x_stride, H, x);
    }
    // z (kept in x), n (in t), a
#pragma unroll
    for (int k = 0; k < N; ++k) { x[k] *= rstd1; t[k] = x[k]; a[k] = 1.f; }
    if (F.post_weight) {
      weight(F.post_weight, F.weights_f32, 0, w);
#pragma unroll
      for (int k = 0; k < N; ++k) t[k] *= w[k];
    }
    if (F.gate_mode == GATE_TOKEN) {
      const float v = SIG ? gate_sigmoid<T>(token_gate) : token_gate;
#pragma unroll
      for (int k = 0; k < N; ++k) a[k] = v;
    } else if (F.gate_mode != GATE_NONE) {
      if (F.gate_mode == GATE_CHANNEL) {
        if constexpr (HELD_GATE) held(GATE, a);    // (behind the sigmoid)
        else R::template load<T>(F.gate, 0, H, a);
      } else if constexpr (AHEAD) {
        unpack8<T>(ca.w, a);
        if constexpr (SIG) keep(a, GATE);         // (the row's gate, for its derivative)
      } else {
        R::template load<T>(F.gate, row * F.gate_stride, H, a);
      }
      if (SIG && !(HELD_GATE && F.gate_mode == GATE_CHANNEL))
#pragma unroll
        for (int k = 0; k < N; ++k) a[k] = gate_sigmoid<T>(a[k]);
    }
    // g = R' = the gradient of t
    if (P.d_residual_out) {
      if constexpr (AHEAD) unpack8<T>(cg.w, g);
      else R::template load<T>(P.d_residual_out, row * P.d_residual_out_stride, H, g);
    } else
#pragma unroll
      for (int k = 0; k < N; ++k) g[k] = 0.f;
    if (P.d_h) {
      float d[N], u[N];
      if constexpr (AHEAD) unpack8<T>(cd.w, d);
      else R::template load<T>(P.d_h, row * P.d_h_stride, H, d);
      if (F.residual) {
        if constexpr (AHEAD) unpack8<T>(cr.w, u);
        else R::template load<T>(F.residual, row * F.residual_stride, H, u);
      } else
#pragma unroll
        for (int k = 0; k < N; ++k) u[k] = 0.f;
      weight(F.pre_weight, F.weights_f32, 1, w);
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        u[k] = (u[k] + F.residual_scale * a[k] * t[k]) * rstd2;
        dw2[k] += d[k] * u[k];
        d[k] *= w[k];
        dot += d[k] * u[k];
      }
      red.run(dot);
      dot *= inv_h;
#pragma unroll
      for (int k = 0; k < N; ++k) g[k] += rstd2 * (d[k] - u[k] * dot);
    }
    if (P.d_residual) R::template store<T>(P.d_residual, row * P.d_residual_stride, H, g);
    // g = s R'; da = g n, dn = g a
    float dot = 0.f, tok = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) g[k] *= F.residual_scale;
    if (F.gate_mode != GATE_NONE) {
      if constexpr (SIG) {
        // the gate's derivative a (1 - a), with 1 - a = sigmoid(-gate): a difference keeps no bits of it beyond a gate
        // of 17 (computed here: held from above, or by the smaller of the two, every row would pay for it)
        if (F.gate_mode == GATE_TOKEN) {
          const float rest = gate_sigmoid<T>(-token_gate);
#pragma unroll
          for (int k = 0; k < N; ++k) t[k] *= a[k] * rest;
        } else if (HELD_GATE && F.gate_mode == GATE_CHANNEL) {
          held(GATE + 1, w);
#pragma unroll
          for (int k = 0; k < N; ++k) t[k] *= w[k];
        } else {
          if constexpr (AHEAD) held(GATE, w);
          else R::template load<T>(F.gate, F.gate_mode == GATE_FULL ? row * F.gate_stride : 0, H, w);
#pragma unroll
          for (int k = 0; k < N; ++k) t[k] *= a[k] * gate_sigmoid<T>(-w[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float da = g[k] * t[k];
        g[k] *= a[k];
        a[k] = da;
      }
      if (F.gate_mode == GATE_TOKEN) {
#pragma unroll
        for (int k = 0; k < N; ++k) tok += a[k];
      } else if (F.gate_mode == GATE_CHANNEL) {
#pragma unroll
        for (int k = 0; k < N; ++k) dg[k] += a[k];
      } else if (P.d_gate) {
        R::template store<T>(P.d_gate, row * P.d_gate_stride, H, a);
      }
    }
    if (F.post_weight) {
      weight(F.post_weight, F.weights_f32, 0, w);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        dw1[k] += g[k] * x[k];
        g[k] *= w[k];
        dot += g[k] * x[k];
      }
    }
    if (F.post_weight || F.gate_mode == GATE_TOKEN) {
      red.run(dot, tok);
      dot *= inv_h;
      if (F.gate_mode == GATE_TOKEN && P.d_gate && threadIdx.x == 0) store1<T>(P.d_gate, row * P.d_gate_stride, tok);
      if (F.post_weight)
#pragma unroll
        for (int k = 0; k < N; ++k) g[k] = rstd1 * (g[k] - x[k] * dot);
    }
    if (P.d_x) R::template store<T>(P.d_x, row * P.d_x_stride, H, g);
  }
  const int64_t set = (int64_t)gridDim.x * H, off = (int64_t)blockIdx.x * H;
  if (P.d_pre_weight) R::template store<T_F32>(P.workspace, off, H, dw2);
  if (P.d_post_weight) R::template store<T_F32>(P.workspace, set + off, H, dw1);
  if (P.d_gate && F.gate_mode == GATE_CHANNEL) R::template store<T_F32>(P.workspace, 2 * set + off, H, dg);
}

// Column sums of partial[G][H]: a workgroup takes C columns, its thread groups of C the rows in turn.
template <int T, int C>
__global__ void __launch_bounds__(1024) k_norm_columns(const DgmNormGradArgs P, int groups) {
  const DgmNormArgs& F = P.forward;
  constexpr int R = 1024 / C;
  __shared__ float lds[R][C];
  const int H = F.hidden, c = threadIdx.x % C, r = threadIdx.x / C, col = blockIdx.x * C + c, set = blockIdx.y;
  void* out = set == 0 ? P.d_pre_weight : set == 1 ? P.d_post_weight : F.gate_mode == GATE_CHANNEL ? P.d_gate : nullptr;
  if (!out) return;                               // (the whole workgroup)
  const float* src = (const float*)P.workspace + (int64_t)set * groups * H;
  float s = 0.f;
  if (col < H)
#pragma unroll 8
    for (int i = r; i < groups; i += R) s += src[(int64_t)i * H + col];
  lds[r][c] = s;
  __syncthreads();
  if (r == 0 && col < H) {
#pragma unroll 8
    for (int i = 1; i < R; ++i) s += lds[i][c];
    if (set < 2 && F.weights_f32) store1<T_F32>(out, col, s);
    else store1<T>(out, col, s);
  }
}

int check_forward(const DgmNormArgs* A) {
  DGM_CHECK_ARG(A->dtype >= DGM_SRC_BF16 && A->dtype <= DGM_SRC_F32, "dtype 0 bf16, 1 fp16, 2 fp32");
  // (a launch has fewer than 2^32 threads, a row up to 1024 of them)
  DGM_CHECK_ARG(A->rows >= 0 && A->rows < (1 << 22), "rows below 2^22");
  DGM_CHECK_ARG(A->hidden > 0 && A->hidden <= DGM_NORM_MAX_HIDDEN, "hidden 1 to 16384");
  DGM_CHECK_ARG(A->gate_mode >= 0 && A->gate_mode <= GATE_FULL, "gate_mode 0 none, 1 channel, 2 token, 3 full");
  DGM_CHECK_ARG(A->eps >= 0.f, "eps >= 0");
  if (A->rows == 0) return 0;
  DGM_CHECK_ARG(A->x, "null x");
  DGM_CHECK_ARG((A->gate != nullptr) == (A->gate_mode != GATE_NONE), "gate and gate_mode");
  return 0;
}

// Threads of a row's workgroup: eight elements each up to 8192, then sixteen (unaligned rows alike). Backward, sixteen
// elements with their column sums do not fit the 128 registers that 1024 threads leave: 106 to 144 of them are kept in
// scratch memory (aligned; unaligned 196 to 266, and 14 to 50 for rows of 4097 to 8192), and 2048 x 16384 bf16 takes 264
// us, 1.5 TB/s.
template <class F>
void dispatch_hidden(int H, F&& f) {
  using std::integral_constant;
  if (H <= 512) f(integral_constant<int, 1>{}, integral_constant<int, 64>{});
  else if (H <= 1024) f(integral_constant<int, 1>{}, integral_constant<int, 128>{});
  else if (H <= 2048) f(integral_constant<int, 1>{}, integral_constant<int, 256>{});
  else if (H <= 4096) f(integral_constant<int, 1>{}, integral_constant<int, 512>{});
  else if (H <= 8192) f(integral_constant<int, 1>{}, integral_constant<int, 1024>{});
  else f(integral_constant<int, 2>{}, integral_constant<int, 1024>{});
}
// Forward rows of 16 bits, many of them: half the threads with sixteen elements each (bf16, 8192 x 4096: 57 -> 51
// us, 4096 x 7168: 52 -> 46 us; fp16 takes bf16's time; one row of 4096 takes 5.4 us the other way and 5.8 this one, fp32 rows 48 and
// 49 us at 4096 x 4096).
template <class F>
void dispatch_hidden_pairs(int H, F&& f) {
  using std::integral_constant;
  if (H <= 512) f(integral_constant<int, 1>{}, integral_constant<int, 64>{});
  else if (H <= 1024) f(integral_constant<int, 2>{}, integral_constant<int, 64>{});
  else if (H <= 2048) f(integral_constant<int, 2>{}, integral_constant<int, 128>{});
  else if (H <= 4096) f(integral_constant<int, 2>{}, integral_constant<int, 256>{});
  else if (H <= 8192) f(integral_constant<int, 2>{}, integral_constant<int, 512>{});
  else f(integral_constant<int, 2>{}, integral_constant<int, 1024>{});
}
bool forward_aligned(const DgmNormArgs* A) {
  const int e = element_size(A->dtype);
  return A->hidden % 8 == 0 && aligned(A->x, A->x_stride, e) && aligned(A->residual, A->residual_stride, e) &&
         aligned(A->post_weight, 0, e) && aligned(A->pre_weight, 0, e) &&
         (A->gate_mode == GATE_TOKEN || aligned(A->gate, A->gate_mode == GATE_FULL ? A->gate_stride : 0, e)) &&
         aligned(A->residual_out, A->residual_out_stride, e) && aligned(A->h, A->h_stride, e) &&
         ((uintptr_t)A->q & 7) == 0;
}

}  // namespace

extern "C" {

int dgm_norm_struct_sizes(size_t* norm_args, size_t* norm_grad_args) {
  DGM_CHECK_ARG(norm_args && norm_grad_args, "null pointer");
  *norm_args = sizeof(DgmNormArgs);
  *norm_grad_args = sizeof(DgmNormGradArgs);
  return 0;
}

int dgm_rms_norm_residual(const DgmNormArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  if (int st = check_forward(args)) return st;
  const DgmNormArgs A = *args;
  DGM_CHECK_ARG(!A.q || (A.dtype == DGM_SRC_BF16 && A.q_sf && A.pre_weight), "int8 rows: of bf16 rows with a pre weight");
  if (A.rows == 0) return 0;
  dispatch_type(A.dtype, forward_aligned(&A), [&](auto t, auto vec) {
    auto launch = [&](auto nv, auto threads) {
      hipLaunchKernelGGL((k_norm_fwd<t.value, nv.value, threads.value, vec.value>), dim3((unsigned)A.rows),
                         dim3(threads.value), 0, stream, A);
    };
    if constexpr (vec.value && t.value != T_F32) {
      if (A.rows > 256) return dispatch_hidden_pairs(A.hidden, launch);
    }
    dispatch_hidden(A.hidden, launch);
  });
  return dgm_last_launch_status();
}

// As many workgroups as the CUs hold (16 waves each), a row each at least: 32768 x 512 with 512 of them
// took 174 us, 4096 x 7168 103 us.
int dgm_rms_norm_residual_groups(int64_t rows, int hidden) {
  int64_t most = 4096;
  dispatch_hidden(hidden, [&](auto, auto threads) { most = 4096 / (threads.value / 64); });
  return (int)(rows < 1 ? 1 : rows < most ? rows : most);
}

int dgm_rms_norm_residual_backward(const DgmNormGradArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmNormGradArgs A = *args;
  const DgmNormArgs& F = A.forward;
  if (int st = check_forward(&F)) return st;
  const bool columns = A.d_pre_weight || A.d_post_weight || (A.d_gate && F.gate_mode == GATE_CHANNEL);
  const int groups = dgm_rms_norm_residual_groups(F.rows, F.hidden);
  if (F.rows > 0) {
    DGM_CHECK_ARG(!F.post_weight || F.rstd_post, "rstd_post of the forward pass");
    DGM_CHECK_ARG(!A.d_h || (F.pre_weight && F.rstd_pre), "pre weight and rstd_pre of the forward pass");
    DGM_CHECK_ARG(!A.d_residual || F.residual, "d_residual without a residual");
  }
  DGM_CHECK_ARG(!A.d_pre_weight || F.pre_weight, "d_pre_weight without its weight");
  DGM_CHECK_ARG(!A.d_post_weight || F.post_weight, "d_post_weight without its weight");
  DGM_CHECK_ARG(!A.d_gate || F.gate_mode != GATE_NONE, "d_gate without a gate");
  // (read before the first row is, so also where there is none)
  DGM_CHECK_ARG(F.gate_mode != GATE_CHANNEL || F.gate, "gate and gate_mode");
  DGM_CHECK_ARG(!columns || (A.workspace && A.workspace_bytes >= (int64_t)groups * F.hidden * 12 &&
                             ((uintptr_t)A.workspace & 15) == 0),
                "workspace of 3 x groups x hidden floats, 16-byte aligned");
  const int e = element_size(F.dtype);
  const bool vec = forward_aligned(&F) && aligned(A.d_residual_out, A.d_residual_out_stride, e) &&
                   aligned(A.d_h, A.d_h_stride, e) && aligned(A.d_x, A.d_x_stride, e) &&
                   aligned(A.d_residual, A.d_residual_stride, e) &&
                   (F.gate_mode != GATE_FULL || aligned(A.d_gate, A.d_gate_stride, e));
  // (no rows: the partial sums of the one group are written as zeros)
  dispatch_type(F.dtype, vec, [&](auto t, auto v) {
    dispatch_hidden(F.hidden, [&](auto nv, auto threads) {
      if (F.gate_mode != GATE_NONE && F.gate_sigmoid)
        hipLaunchKernelGGL((k_norm_bwd<t.value, nv.value, threads.value, v.value, true>), dim3(groups), dim3(threads.value), 0,
                           stream, A);
      else
        hipLaunchKernelGGL((k_norm_bwd<t.value, nv.value, threads.value, v.value, false>), dim3(groups), dim3(threads.value), 0,
                           stream, A);
    });
    if (columns) {
      // (narrow rows have many groups: 16 columns a workgroup, so that there are enough of them)
      if (groups > 1024)
        hipLaunchKernelGGL((k_norm_columns<t.value, 16>), dim3((F.hidden + 15) / 16, 3), dim3(1024), 0, stream, A, groups);
      else
        hipLaunchKernelGGL((k_norm_columns<t.value, 64>), dim3((F.hidden + 63) / 64, 3), dim3(1024), 0, stream, A, groups);
    }
  });
  return dgm_last_launch_status();
}

}  // extern "C"
