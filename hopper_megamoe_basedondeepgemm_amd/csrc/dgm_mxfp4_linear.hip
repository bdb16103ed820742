// A linear layer on MXFP4 products, host side: the launches of a forward or a backward pass behind one call (a training
// step of a small layer is the host's time: seven calls of its parts from Python took 190 us, two take 125 us).
#include "dgm_abi_internal.hpp"

namespace {

int64_t pad256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t blocks(int64_t k) { return (k + 31) / 32; }

// Rows of k elements as they lie in the workspace: codes, then scales.
struct Quantised {
  int64_t rows, k;
  int64_t codes_bytes() const { return pad256(rows * blocks(k) * 16); }
  int64_t bytes() const { return codes_bytes() + pad256(rows * blocks(k)); }
  uint8_t* codes(void* at) const { return (uint8_t*)at; }
  uint8_t* scales(void* at) const { return (uint8_t*)at + codes_bytes(); }
};

int64_t product_bytes(int64_t m, int64_t n, int64_t k) { return dgm_mxfp4_gemm_workspace_bytes(m, n, 32 * blocks(k), 0); }

int product(const uint8_t* a, const uint8_t* sfa, const uint8_t* b, const uint8_t* sfb, void* d, int64_t m, int64_t n, int64_t k, int dtype,
            void* workspace, hipStream_t stream) {
  DgmMxfp4GemmArgs P = {};
  const int64_t kb = blocks(k);
  P.a = a, P.sfa = sfa, P.b = b, P.sfb = sfb, P.d = d;
  P.m = m, P.n = n, P.k = 32 * kb;
  P.a_stride = P.b_stride = 16 * kb;
  P.sfa_stride = P.sfb_stride = kb;
  P.d_stride = n;
  P.dtype = dtype;
  P.clamp = INFINITY;
  P.workspace = (float*)workspace;
  P.workspace_bytes = product_bytes(m, n, k);
  return dgm_mxfp4_gemm_nt(&P, stream);
}

int quantise(const void* x, int64_t rows, int64_t cols, int64_t stride, int dtype, uint8_t* codes, uint8_t* scales, uint8_t* t_codes,
             uint8_t* t_scales, hipStream_t stream) {
  const DgmMxfp4QuantArgs Q = {x, codes, scales, t_codes, t_scales, rows, cols, stride, dtype, 1e-30f};
  return dgm_mxfp4_quantize(&Q, stream);
}

int check(const DgmMxfp4LinearArgs& A, int backward) {
  DGM_CHECK_ARG(A.x_dtype >= DGM_SRC_BF16 && A.x_dtype <= DGM_SRC_F32 && A.w_dtype >= DGM_SRC_BF16 && A.w_dtype <= DGM_SRC_F32,
                "dtypes 0 bf16, 1 fp16, 2 fp32");
  DGM_CHECK_ARG(A.m >= 0 && A.m < (1 << 24) && A.n > 0 && A.n < (1 << 24) && A.k > 0 && A.k < (1 << 24), "m, n and k below 2^24, a feature at least");
  DGM_CHECK_ARG((A.x_columns != nullptr) == (A.x_column_scales != nullptr) && (A.w_columns != nullptr) == (A.w_column_scales != nullptr),
                "columns with their scales");
  DGM_CHECK_ARG(A.m == 0 || (A.workspace && ((uintptr_t)A.workspace & 15) == 0 &&
                             A.workspace_bytes >= dgm_mxfp4_linear_workspace_bytes(A.m, A.n, A.k, backward)), "workspace, 16-byte aligned");
  // (before anything is enqueued: what a product refuses)
  auto fits = [](int64_t m, int64_t n) { return ((m + 63) / 64) * ((n + 63) / 64) < (1 << 23); };
  DGM_CHECK_ARG(backward ? (!A.d_x || fits(A.m, A.k)) && (!A.d_w || fits(A.n, A.k)) : fits(A.m, A.n), "a product's limits");
  return 0;
}

}  // namespace

extern "C" {

int dgm_mxfp4_linear_struct_size(size_t* args) {
  DGM_CHECK_ARG(args, "null pointer");
  *args = sizeof(DgmMxfp4LinearArgs);
  return 0;
}

int64_t dgm_mxfp4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int backward) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  if (!backward) return Quantised{m, k}.bytes() + Quantised{n, k}.bytes() + product_bytes(m, n, k);
  const int64_t d_x = product_bytes(m, k, n), d_w = product_bytes(n, k, m);
  return Quantised{m, n}.bytes() + Quantised{n, m}.bytes() + (d_x > d_w ? d_x : d_w);
}

int dgm_mxfp4_linear(const DgmMxfp4LinearArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmMxfp4LinearArgs A = *args;
  if (int st = check(A, 0)) return st;
  DGM_CHECK_ARG(A.w && (A.m == 0 || (A.x && A.y)), "null pointer");
  const Quantised x = {A.m, A.k}, w = {A.n, A.k};
  if (A.m == 0)                                    // (the weight's columns alone)
    return A.w_columns ? quantise(A.w, A.n, A.k, A.w_stride, A.w_dtype, nullptr, nullptr, A.w_columns, A.w_column_scales, stream) : 0;
  uint8_t *xq = (uint8_t*)A.workspace, *wq = xq + x.bytes(), *sums = wq + w.bytes();
  if (int st = quantise(A.x, A.m, A.k, A.x_stride, A.x_dtype, x.codes(xq), x.scales(xq), A.x_columns, A.x_column_scales, stream)) return st;
  if (int st = quantise(A.w, A.n, A.k, A.w_stride, A.w_dtype, w.codes(wq), w.scales(wq), A.w_columns, A.w_column_scales, stream)) return st;
  return product(x.codes(xq), x.scales(xq), w.codes(wq), w.scales(wq), A.y, A.m, A.n, A.k, A.x_dtype, sums, stream);
}

int dgm_mxfp4_linear_backward(const DgmMxfp4LinearArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmMxfp4LinearArgs A = *args;
  if (int st = check(A, 1)) return st;
  DGM_CHECK_ARG(A.m > 0 || !A.d_w, "d_w of no tokens is zeros: left to the caller");
  DGM_CHECK_ARG((!A.d_x || A.w_columns) && (!A.d_w || A.x_columns), "columns of the forward pass");
  if (A.m == 0 || (!A.d_x && !A.d_w)) return 0;
  DGM_CHECK_ARG(A.d_y, "null pointer");
  const Quantised r = {A.m, A.n}, c = {A.n, A.m};
  uint8_t *rows = (uint8_t*)A.workspace, *columns = rows + r.bytes(), *sums = columns + c.bytes();
  if (int st = quantise(A.d_y, A.m, A.n, A.d_y_stride, A.x_dtype, A.d_x ? r.codes(rows) : nullptr, A.d_x ? r.scales(rows) : nullptr,
                        A.d_w ? c.codes(columns) : nullptr, A.d_w ? c.scales(columns) : nullptr, stream))
    return st;
  if (A.d_x)
    if (int st = product(r.codes(rows), r.scales(rows), A.w_columns, A.w_column_scales, A.d_x, A.m, A.k, A.n, A.x_dtype, sums, stream)) return st;
  if (!A.d_w) return 0;
  return product(c.codes(columns), c.scales(columns), A.x_columns, A.x_column_scales, A.d_w, A.n, A.k, A.m, A.w_dtype, sums, stream);
}

}  // extern "C"
