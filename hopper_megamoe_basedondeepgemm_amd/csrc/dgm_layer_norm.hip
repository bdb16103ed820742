// Residual add and layer norm (gfx950) in one pass over the rows, and the gradients of both.
//
// Row of H elements: t = residual + s x (t = s x without residual), mu = mean t, rstd = rsqrt(mean (t - mu)^2 + eps),
// u = (t - mu) rstd, h = u w + b (w, b: 1 and 0 if absent). Everything between the loads and the stores is fp32; t
// enters the norm unrounded and stays in registers, so that the variance is that of the differences from the mean (no
// cancellation) and each input is read once. A workgroup owns a row; the bound is HBM.
// Gradients, with R = dL/dt (of the stored t) and D = dL/dh:
//   du = D w, R' = R + rstd (du - mean du - u mean(du u)), dresidual = R', dx = s R', dw = sum D u, db = sum D.
#include "dgm_abi_internal.hpp"
#include "dgm_mxfp4.hpp"
#include "dgm_row_tiles.hpp"

#include <algorithm>

using namespace dgm;

namespace {

// t, in fp32 and in this order wherever it is computed: forward and backward see the same bits.
DGM_DEV float total(float r, float s, float x) { return fmaf(s, x, r); }

// Forward: one read of x and residual, one write of r and h; two sums over the row one behind the other (the variance
// waits for the mean, which costs the second exchange but no cancellation). Over 800 MB of rows in turn, which no cache
// holds: bf16 8192 x 4096 51.8 us, fp32 8192 x 2880 72.9, bf16 2048 x 16384 52.6, 5.1 to 5.2 TB/s each; rows off 16 bytes
// are loaded on the elements' alignment, 4096 x 5001 54.4 us, 3.0 TB/s. Three sets of rows in turn, partly in the last
// cache: 8192 x 4096 48.2 (51.2 with the residual and the weights requested with x), 4096 x 5001 47.6 (by single
// elements 70).
// Rows of one wave: four of them a workgroup are no faster (100 000 x 256 56 us, one 54; half its lanes have no elements).
template <int T, int NV, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS) k_layer_norm_fwd(const DgmLayerNormArgs P) {
  using R = std::conditional_t<VEC, Row<NV, THREADS, true>, LooseRow<NV, THREADS>>;
  constexpr int N = R::N;
  __shared__ float lds[2][THREADS / 64][2];
  Reduce<THREADS> red{lds};
  const int H = P.hidden;
  const int64_t row = blockIdx.x;
  const bool wf = P.weights_f32;
  const float inv_h = 1.0f / (float)H;
  float t[N], w[N];
  R::template load<T>(P.x, row * P.x_stride, H, t);
  if (P.residual) {
    R::template load<T>(P.residual, row * P.residual_stride, H, w);
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = total(w[k], P.residual_scale, t[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] *= P.residual_scale;
  }
  // (loose rows: a thread also reads elements of the one before it, which may be another wave's, and residual_out may be
  // the row itself: stored behind the sum, which waits for every thread's elements)
  if (VEC && P.residual_out) R::template store<T>(P.residual_out, row * P.residual_out_stride, H, t);
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) sum += t[k];       // (zeros behind H)
  red.run(sum);
  if (!VEC && P.residual_out) R::template store<T>(P.residual_out, row * P.residual_out_stride, H, t);
  const float mean = sum / (float)H;              // (by 1 / H, a row of equal elements would not have them for its mean)
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    t[k] = R::index(k) < H ? t[k] - mean : 0.f;
    ss += t[k] * t[k];
  }
  red.run(ss);
  const float rstd = 1.0f / sqrtf(ss * inv_h + P.eps);
  if (P.mean && threadIdx.x == 0) P.mean[row] = mean, P.rstd[row] = rstd;
#pragma unroll
  for (int k = 0; k < N; ++k) t[k] *= rstd;
  if (P.weight) {
    R::template weight<T>(P.weight, wf, H, w);
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] *= w[k];
  }
  if (P.bias) {
    R::template weight<T>(P.bias, wf, H, w);
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] += w[k];
  }
  if (P.h) R::template store<T>(P.h, row * P.h_stride, H, t);
  if constexpr (T == T_BF16 && VEC) {
    if (!P.codes) return;
    // MXFP4 rows of the rounded h: a thread's eight elements are a quarter of a block (zeros behind H)
    const int64_t blocks = (H + 31) / 32;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < 8; ++k) t[8 * j + k] = round_bf16(t[8 * j + k]);
      const uint32_t code = mx_scale_code(max_u32_lanes4(magnitude8(t + 8 * j)), __float_as_uint(1e-30f));
      const int64_t piece = j * THREADS + (int)threadIdx.x;
      if (piece >= 4 * blocks) continue;
      reinterpret_cast<uint32_t*>(P.codes)[row * blocks * 4 + piece] = e2m1_codes8<T>(t + 8 * j, code);
      if ((piece & 3) == 0) P.scales[row * blocks + (piece >> 2)] = (uint8_t)code;
    }
  }
}

// Gradients: workgroup g takes rows g, g + G, ...; the columns' sums over its rows stay in registers and go to
// partial[set][g][H] (set 0 weight, 1 bias), which k_layer_norm_columns adds up in a fixed order: atomics would give
// another order every time. Both sums (du and du u) meet in one exchange. bf16 8192 x 4096, six tensors of rows (403 MB):
// 81 us with the column sums, 4.9 TB/s; fp32 4096 x 4096: 84, 4.8; off 16 bytes 4096 x 5001: 85, 2.9 TB/s (by single
// elements 186). Beyond hidden 8192 registers go to scratch memory, 9 to 11 a lane of aligned rows (2048 x 16384 bf16 105
// us, 3.8 TB/s; fp32 188, 4.3), 27 to 91 of others (2048 x 12345 bf16 135 us, 2.3 TB/s; fp16 233, 1.3).
template <int T, int NV, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS) k_layer_norm_bwd(const DgmLayerNormGradArgs P) {
  using R = std::conditional_t<VEC, Row<NV, THREADS, true>, LooseRow<NV, THREADS>>;
  constexpr int N = R::N;
  __shared__ float lds[2][THREADS / 64][2];
  Reduce<THREADS> red{lds};
  const DgmLayerNormArgs& F = P.forward;
  const int H = F.hidden;
  const float inv_h = 1.0f / (float)H;
  float dw[N], db[N];
#pragma unroll
  for (int k = 0; k < N; ++k) dw[k] = db[k] = 0.f;
  // Rows of eight 16-bit elements a thread: the next row is requested before the current one is worked on, and the weight
  // stays in registers (100 000 bf16 rows of 256: 70 us instead of 103; 4096 rows of 7168: 74 instead of 84; 8192 of 4096:
  // 85 instead of 90). Sixteen elements, or fp32 ones, are too many for two rows (fp32 8192 rows of 2880: 112 us
  // without, 116 with).
  constexpr bool AHEAD = VEC && NV == 1 && T != T_F32;
  HeldRow hx, hr, hd, hg;
  float next_mean = 0.f, next_rstd = 0.f, held_w[AHEAD ? N : 1];
  auto request = [&](int64_t row) {
    if (P.d_residual_out) hg.load<T>(P.d_residual_out, row * P.d_residual_out_stride, H);
    if (!P.d_h) return;
    hx.load<T>(F.x, row * F.x_stride, H);
    if (F.residual) hr.load<T>(F.residual, row * F.residual_stride, H);
    hd.load<T>(P.d_h, row * P.d_h_stride, H);
    next_mean = F.mean[row];
    next_rstd = F.rstd[row];
  };
  if constexpr (AHEAD) {
    if (F.weight) R::template weight<T>(F.weight, F.weights_f32, H, held_w);
    if ((int64_t)blockIdx.x < F.rows) request(blockIdx.x);
  }
  for (int64_t row = blockIdx.x; row < F.rows; row += gridDim.x) {
    float g[N];
    HeldRow cx, cr, cd, cg;
    float mean = next_mean, rstd = next_rstd;
    if constexpr (AHEAD) {
      cx = hx, cr = hr, cd = hd, cg = hg;
      const int64_t next = row + gridDim.x;
      if (next < F.rows) request(next);
    }
    auto get = [&](const HeldRow& held, const void* p, int64_t stride, float* v) {
      if constexpr (AHEAD) held.unpack<T>(v);
      else R::template load<T>(p, row * stride, H, v);
    };
    if (P.d_residual_out) get(cg, P.d_residual_out, P.d_residual_out_stride, g);
    else
#pragma unroll
      for (int k = 0; k < N; ++k) g[k] = 0.f;
    if (P.d_h) {
      float u[N], d[N], w[N];
      get(cx, F.x, F.x_stride, u);
      if (F.residual) {
        get(cr, F.residual, F.residual_stride, w);
#pragma unroll
        for (int k = 0; k < N; ++k) u[k] = total(w[k], F.residual_scale, u[k]);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) u[k] *= F.residual_scale;
      }
      get(cd, P.d_h, P.d_h_stride, d);
      if constexpr (!AHEAD) mean = F.mean[row], rstd = F.rstd[row];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        u[k] = (u[k] - mean) * rstd;
        dw[k] += d[k] * u[k];
        db[k] += d[k];
      }
      if (F.weight) {
        if constexpr (!AHEAD) R::template weight<T>(F.weight, F.weights_f32, H, w);
#pragma unroll
        for (int k = 0; k < N; ++k) d[k] *= AHEAD ? held_w[AHEAD ? k : 0] : w[k];
      }
      float sum = 0.f, dot = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) {          // (d is zero behind H)
        sum += d[k];
        dot += d[k] * u[k];
      }
      red.run(sum, dot);
      sum *= inv_h;
      dot *= inv_h;
#pragma unroll
      for (int k = 0; k < N; ++k) g[k] += rstd * (d[k] - sum - u[k] * dot);
    }
    if (P.d_residual) R::template store<T>(P.d_residual, row * P.d_residual_stride, H, g);
    if (P.d_x) {
#pragma unroll
      for (int k = 0; k < N; ++k) g[k] *= F.residual_scale;
      R::template store<T>(P.d_x, row * P.d_x_stride, H, g);
    }
  }
  const int64_t set = (int64_t)gridDim.x * H, off = (int64_t)blockIdx.x * H;
  if (P.d_weight) R::template store<T_F32>(P.workspace, off, H, dw);
  if (P.d_bias) R::template store<T_F32>(P.workspace, set + off, H, db);
}

// Column sums of partial[G][H]: a workgroup takes C columns, its thread groups of C the rows in turn (4096 columns of
// 512 groups: 4.6 us, most of it a launch and the latency of eight loads at a time).
template <int T, int C>
__global__ void __launch_bounds__(1024) k_layer_norm_columns(const DgmLayerNormGradArgs P, int groups) {
  const DgmLayerNormArgs& F = P.forward;
  constexpr int R = 1024 / C;
  __shared__ float lds[R][C];
  const int H = F.hidden, c = threadIdx.x % C, r = threadIdx.x / C, col = blockIdx.x * C + c, set = blockIdx.y;
  void* out = set == 0 ? P.d_weight : P.d_bias;
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
    if (F.weights_f32) store1<T_F32>(out, col, s);
    else store1<T>(out, col, s);
  }
}

// Threads of a row's workgroup: eight elements each up to 8192, then sixteen.
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

int check_forward(const DgmLayerNormArgs* A) {
  DGM_CHECK_ARG(A->dtype >= DGM_SRC_BF16 && A->dtype <= DGM_SRC_F32, "dtype 0 bf16, 1 fp16, 2 fp32");
  // (a launch has fewer than 2^32 threads, a row up to 1024 of them)
  DGM_CHECK_ARG(A->rows >= 0 && A->rows < (1 << 22), "rows below 2^22");
  DGM_CHECK_ARG(A->hidden > 0 && A->hidden <= DGM_NORM_MAX_HIDDEN, "hidden 1 to 16384");
  DGM_CHECK_ARG(A->eps >= 0.f, "eps >= 0");
  DGM_CHECK_ARG(A->rows == 0 || A->x, "null x");
  return 0;
}

bool forward_aligned(const DgmLayerNormArgs* A) {
  const int e = element_size(A->dtype);
  return A->hidden % 8 == 0 && aligned(A->x, A->x_stride, e) && aligned(A->residual, A->residual_stride, e) &&
         aligned(A->weight, 0, e) && aligned(A->bias, 0, e) && aligned(A->residual_out, A->residual_out_stride, e) &&
         aligned(A->h, A->h_stride, e);
}

}  // namespace

extern "C" {

int dgm_layer_norm_struct_sizes(size_t* norm_args, size_t* norm_grad_args) {
  DGM_CHECK_ARG(norm_args && norm_grad_args, "null pointer");
  *norm_args = sizeof(DgmLayerNormArgs);
  *norm_grad_args = sizeof(DgmLayerNormGradArgs);
  return 0;
}

int dgm_layer_norm_residual(const DgmLayerNormArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  if (int st = check_forward(args)) return st;
  const DgmLayerNormArgs A = *args;
  const bool vec = forward_aligned(&A);
  DGM_CHECK_ARG((A.codes != nullptr) == (A.scales != nullptr), "codes with their scales");
  DGM_CHECK_ARG((A.mean != nullptr) == (A.rstd != nullptr), "mean with rstd");
  DGM_CHECK_ARG(!A.codes || (A.dtype == DGM_SRC_BF16 && vec && ((uintptr_t)A.codes & 3) == 0), "MXFP4 rows: of 16-byte aligned bf16 rows of whole eights");
  if (A.rows == 0) return 0;
  dispatch_type(A.dtype, vec, [&](auto t, auto v) {
    auto launch = [&](auto nv, auto threads) {
      hipLaunchKernelGGL((k_layer_norm_fwd<t.value, nv.value, threads.value, v.value>), dim3((unsigned)A.rows),
                         dim3(threads.value), 0, stream, A);
    };
    // Many 16-bit rows of 4096 < hidden <= 8192: 512 threads of sixteen elements. Two workgroups of 1024 fill a CU and wait
    // together at their sums, four of 512 less so (4096 rows of 7168: 45.7 us instead of 47.0). Up to 4096 eight elements
    // a thread are as fast (8192 rows of 4096: 48.2, sixteen 48.4), and few rows want the shorter wait.
    if constexpr (v.value && t.value != T_F32) {
      if (A.rows > 256 && A.hidden > 4096 && A.hidden <= 8192)
        return launch(std::integral_constant<int, 2>{}, std::integral_constant<int, 512>{});
    }
    dispatch_hidden(A.hidden, launch);
  });
  return dgm_last_launch_status();
}

// As many workgroups as the CUs hold (16 waves each), two rows each at least (one, where there is no second).
int dgm_layer_norm_residual_groups(int64_t rows, int hidden) {
  // Two rows a workgroup at least: its column sums are as many bytes as two 16-bit rows, written and read again (300 x
  // 4096 15.0 us with one, 11.9; 64 x 7168 10.2 and 10.4). And no more than the CUs hold at a time.
  int64_t most = 0;
  dispatch_hidden(hidden, [&](auto, auto threads) { most = 4096 / (threads.value / 64); });
  rows = (rows + 1) / 2;
  return (int)(rows < 1 ? 1 : rows < most ? rows : most);
}

int dgm_layer_norm_residual_backward(const DgmLayerNormGradArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmLayerNormGradArgs A = *args;
  const DgmLayerNormArgs& F = A.forward;
  if (int st = check_forward(&F)) return st;
  const bool columns = A.d_weight || A.d_bias;
  int groups = dgm_layer_norm_residual_groups(F.rows, F.hidden);
  if (F.rows > 0) {
    DGM_CHECK_ARG(!A.d_h || (F.mean && F.rstd), "mean and rstd of the forward pass");
    DGM_CHECK_ARG(!A.d_residual || F.residual, "d_residual without a residual");
  }
  DGM_CHECK_ARG(!A.d_weight || F.weight, "d_weight without its weight");
  DGM_CHECK_ARG(!A.d_bias || F.bias, "d_bias without its bias");
  DGM_CHECK_ARG(!columns || (A.workspace && A.workspace_bytes >= (int64_t)groups * F.hidden * 8 &&
                             ((uintptr_t)A.workspace & 15) == 0),
                "workspace of 2 x groups x hidden floats, 16-byte aligned");
  const int e = element_size(F.dtype);
  const bool vec = forward_aligned(&F) && aligned(A.d_residual_out, A.d_residual_out_stride, e) &&
                   aligned(A.d_h, A.d_h_stride, e) && aligned(A.d_x, A.d_x_stride, e) &&
                   aligned(A.d_residual, A.d_residual_stride, e);
  // Rows requested ahead need half the waves, at least a workgroup a CU (bf16 8192 x 4096 80.5 us, twice as many groups
  // 85, half as many 100; 4096 x 2048 23.4 and 26; 4096 x 7168 with 128 groups 90, 256 74.5); others all they can have
  // (fp32 8192 x 2880 112 us, half 122).
  if (vec && F.dtype != DGM_SRC_F32 && F.hidden <= 8192)
    dispatch_hidden(F.hidden, [&](auto, auto threads) { groups = std::min(groups, std::max(2048 / (threads.value / 64), 256)); });
  // (no rows: the partial sums of the one group are written as zeros)
  dispatch_type(F.dtype, vec, [&](auto t, auto v) {
    dispatch_hidden(F.hidden, [&](auto nv, auto threads) {
      hipLaunchKernelGGL((k_layer_norm_bwd<t.value, nv.value, threads.value, v.value>), dim3(groups), dim3(threads.value), 0,
                         stream, A);
    });
    if (columns) {
      // (narrow rows have many groups: 16 columns a workgroup, so that there are enough of them)
      if (groups > 1024)
        hipLaunchKernelGGL((k_layer_norm_columns<t.value, 16>), dim3((F.hidden + 15) / 16, 2), dim3(1024), 0, stream, A, groups);
      else
        hipLaunchKernelGGL((k_layer_norm_columns<t.value, 64>), dim3((F.hidden + 63) / 64, 2), dim3(1024), 0, stream, A, groups);
    }
  });
  return dgm_last_launch_status();
}

}  // extern "C"
