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

using namespace dgm;

namespace {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));

DGM_DEV void store_out(void* d, int dtype, int64_t i, float v) {
  if (dtype == DGM_SRC_F32) reinterpret_cast<float*>(d)[i] = v;
  else if (dtype == DGM_SRC_F16) reinterpret_cast<_Float16*>(d)[i] = (_Float16)v;
  else reinterpret_cast<uint16_t*>(d)[i] = f32_to_bf16(v);
}
DGM_DEV float load_c(const void* c, int dtype, int64_t i) {
  if (dtype == DGM_SRC_F32) return reinterpret_cast<const float*>(c)[i];
  if (dtype == DGM_SRC_F16) return (float)reinterpret_cast<const _Float16*>(c)[i];
  return bf16_to_f32(reinterpret_cast<const uint16_t*>(c)[i]);
}
DGM_DEV float swiglu(float g, float u, float clamp, bool fast) {
  g = fminf(g, clamp);
  u = fminf(fmaxf(u, -clamp), clamp);
  return g * (fast ? sigmoid<true>(g) : sigmoid<false>(g)) * u;
}

// 16 bytes of a row from k on, zeros behind K, at any alignment.
DGM_DEV v4i load16_any(const int8_t* row, int64_t k, int64_t K) {
  v4i r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t d = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (k + 4 * j + b < K) d |= (uint32_t)(uint8_t)row[k + 4 * j + b] << (8 * b);
    r[j] = (int)d;
  }
  return r;
}

// Any size, stride and alignment: a wave takes 16 tokens x 16 channels (SwiGLU: their gate and up rows)
// and reads both operands byte by byte.
__global__ void __launch_bounds__(256) k_int8_gemm_any(const DgmInt8GemmArgs P) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int64_t n_out = P.swiglu ? P.n / 2 : P.n, m0 = (int64_t)blockIdx.y * 16, n0 = ((int64_t)blockIdx.x * 4 + wave) * 16;
  if (n0 >= n_out) return;
  const int64_t m = m0 + r < P.m ? m0 + r : P.m - 1, n = n0 + r < n_out ? n0 + r : n_out - 1;
  const int8_t* a = P.a + m * P.a_stride;
  const int8_t* b = P.b + n * P.b_stride;
  const int8_t* up = b + n_out * P.b_stride;
  v4i acc = {0, 0, 0, 0}, acc_up = {0, 0, 0, 0};
  for (int64_t k = 16 * g; k - 16 * g < P.k; k += 64) {
    const v4i av = load16_any(a, k, P.k);
    acc = mfma_i8_16x16x64(load16_any(b, k, P.k), av, acc);
    if (P.swiglu) acc_up = mfma_i8_16x16x64(load16_any(up, k, P.k), av, acc_up);
  }
  if (m0 + r >= P.m) return;
  const float sa = P.sfa[(m0 + r) * P.sfa_stride];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = n0 + 4 * g + i;
    if (c >= n_out) continue;
    float v = (float)acc[i] * (sa * P.sfb[c * P.sfb_stride]);
    if (P.swiglu) v = swiglu(v, (float)acc_up[i] * (sa * P.sfb[(n_out + c) * P.sfb_stride]), P.clamp, P.fast_math);
    else if (P.c) v += load_c(P.c, P.dtype, (m0 + r) * P.c_stride + c);
    store_out(P.d, P.dtype, (m0 + r) * P.d_stride + c, v);
  }
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
  const int64_t n_out = A.swiglu ? A.n / 2 : A.n;
  hipLaunchKernelGGL(k_int8_gemm_any, dim3((unsigned)((n_out + 63) / 64), (unsigned)((A.m + 15) / 16)), dim3(256), 0, stream, A);
  return dgm_last_launch_status();
}

}  // extern "C"
