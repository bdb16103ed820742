// Rows, or columns, of a matrix as MXFP4 (gfx950): blocks of 32 values along a row (column) become E2M1 codes, two a
// byte, under one E8M0 scale,
//   e = least integer with max(amax, floor) <= 6 2^e (at least -126),  code = nearest E2M1 of x / 2^e,
// midpoints to the smaller magnitude; a block that holds an infinity or NaN gets scale 255 and zeros. Behind the last
// element a block holds zeros. About ten operations a value: the bound is HBM, at 2 (fp32 4) bytes read and 17 / 32
// written a value (both ways: twice 17 / 32).
#include "dgm_abi_internal.hpp"
#include "dgm_mxfp4.hpp"
#include "dgm_row_tiles.hpp"

#include <algorithm>

using namespace dgm;

namespace {

// eight elements of row `row` from column c on, zeros outside the matrix
template <int T>
DGM_DEV void load_piece(const DgmMxfp4QuantArgs& P, int64_t row, int64_t c, float* v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = row < P.rows && c + i < P.cols ? load1<T>(P.x, row * P.x_stride + c + i) : 0.f;
}

// The same as loaded, without a branch (a load in one is awaited at its end).
template <int T>
struct RawPiece : Piece<T> {
  using Piece<T>::w;
  DGM_DEV void clear_unless(bool some) {
    const u4 none = {0u, 0u, 0u, 0u};
    w[0] = some ? w[0] : none;
    if constexpr (T == T_F32) w[1] = some ? w[1] : none;
  }
  // the largest magnitude's fp32 bits
  DGM_DEV uint32_t magnitude() const {
    if constexpr (T == T_F32) {
      float v[8];
      this->unpack(v);
      return magnitude8(v);
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) m = max_pairs(m, w[0][k]);
      return magnitude_bits<T>(max_u32(m & 0xffffu, m >> 16));
    }
  }
};
// Where a row's eight elements from column c on are loaded: at c, or where they do not all exist (rows of eight
// elements at least) at the row's last eight, which are then shifted by `by`.
struct Place {
  int64_t at;
  int by;
  DGM_DEV Place(int64_t c, int64_t cols) : at(c + 8 <= cols ? c : cols - 8), by((int)min(c - at, (int64_t)8)) {}
};

// Rows: a thread takes eight values, four neighbours a block, whose maximum goes by lane exchange; nothing is kept
// between threads, so the loads of many waves are in flight (bf16 8192 x 4096, from the last cache: 15.2 us, 5.6 TB/s;
// 8192 x 7168 from HBM: 28.3 us, 5.2 TB/s). 2^log_row threads a row of the workgroup, `runs` workgroups along a row.
template <int T, bool VEC>
__global__ void __launch_bounds__(256) k_mxfp4_rows(const DgmMxfp4QuantArgs P, int log_row, int runs) {
  const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x;       // (the last of gridDim.y may be behind the last row)
  const int64_t group = id / (unsigned)runs;
  const int run = (int)(id - group * runs);
  const int64_t row = (group << (8 - log_row)) + (threadIdx.x >> log_row);
  const int64_t piece = ((int64_t)run << log_row) + (threadIdx.x & ((1 << log_row) - 1));
  const int64_t blocks = (P.cols + 31) / 32;
  if (row >= P.rows || piece >= 4 * blocks) return;           // (whole blocks: four lanes share one)
  float v[8];
  uint32_t m;
  const bool some = piece * 8 < P.cols;
  if (VEC || P.cols >= 8) {
    RawPiece<T> raw;
    if constexpr (VEC) {
      raw.load(P.x, row * P.x_stride + (some ? piece * 8 : 0));
    } else {
      const Place place(piece * 8, P.cols);
      raw.load_loose(P.x, row * P.x_stride + place.at);
      raw.shift(place.by);
    }
    raw.clear_unless(some);
    raw.unpack(v);
    m = raw.magnitude();
  } else {
    load_piece<T>(P, row, piece * 8, v);
    m = magnitude8(v);
  }
  const uint32_t code = mx_scale_code(max_u32_lanes4(m), __float_as_uint(P.amax_floor));
  reinterpret_cast<uint32_t*>(P.codes)[row * blocks * 4 + piece] = e2m1_codes8<T>(v, code);
  if ((piece & 3) == 0) P.scales[row * blocks + (piece >> 2)] = (uint8_t)code;
}

// Columns, and rows with them (BOTH): a tile of R rows x 128 columns is read once, its rows' codes are made on the
// way into LDS, and a thread then takes 32 rows of a column (16 bits: of two, a dword a row). The columns' codes meet in
// LDS again, so that what is stored for a column lies together (64 bytes; fp32 32). All of a tile's loads are requested
// before the first is used (with a branch around each, awaited at its end, columns took 20.2 us and both 33.8).
// bf16 8192 x 4096: columns 15.1 us, 5.6 TB/s; both 26.9, 3.8 TB/s: each value is rounded twice, and the vector units are
// as busy as memory. An order of tiles by XCD is no faster (27.8). Rows off 16 bytes are loaded on the elements'
// alignment (777 x 1234: columns 4.0 us, both 5.9; by single elements 8.3 and 10.1).
template <int T, bool VEC, bool BOTH>
__global__ void __launch_bounds__(256) k_mxfp4_columns(const DgmMxfp4QuantArgs P, int tiles_c) {
  constexpr int R = T == T_F32 ? 64 : 128, C = 128, B = R / 32, PAIR = T == T_F32 ? 1 : 2;
  using E = std::conditional_t<T == T_F32, uint32_t, uint16_t>;
  // (the columns' codes and scales take the tile's place: five workgroups a CU)
  __shared__ __attribute__((aligned(16))) uint8_t memory[R * C * sizeof(E)];
  E(*tile)[C] = reinterpret_cast<E(*)[C]>(memory);
  u4(*codes)[C + 1] = reinterpret_cast<u4(*)[C + 1]>(memory);
  uint8_t(*scales)[B] = reinterpret_cast<uint8_t(*)[B]>(memory + B * (C + 1) * 16);
  static_assert(B * (C + 1) * 16 + C * B <= (int)sizeof(memory), "they fit");
  const int64_t r0 = (int64_t)(blockIdx.x / (unsigned)tiles_c) * R, c0 = (int64_t)(blockIdx.x % (unsigned)tiles_c) * C;
  const int64_t row_blocks = (P.cols + 31) / 32, col_blocks = (P.rows + 31) / 32;
  const uint32_t floor_bits = __float_as_uint(P.amax_floor);
  const int at = (threadIdx.x & 15) * 8, first = threadIdx.x >> 4;
  const int most = (int)min(P.rows - r0, (int64_t)R) - 1;              // last row of the tile
  const bool inside = c0 + at < P.cols;
  const bool pieces = VEC || P.cols >= 8;
  RawPiece<T> raw[R / 16];                       // (all requested before the first is used)
  int by = 0;
  if (pieces) {
    int64_t from = r0 * P.x_stride + (inside ? c0 + at : 0);
    if constexpr (!VEC) {
      const Place place(c0 + at, P.cols);
      from = r0 * P.x_stride + place.at;
      by = place.by;
    }
#pragma unroll
    for (int i = 0; i < R / 16; ++i) {
      const int64_t place = from + (int64_t)min(i * 16 + first, most) * P.x_stride;
      if constexpr (VEC) raw[i].load(P.x, place);
      else raw[i].load_loose(P.x, place);
    }
  }
  const int64_t piece = (c0 + at) / 8;
  uint32_t* const row_codes = reinterpret_cast<uint32_t*>(P.codes) + r0 * row_blocks * 4 + piece;
  uint8_t* const row_scales = P.scales + r0 * row_blocks + (piece >> 2);
#pragma unroll
  for (int i = 0; i < R / 16; ++i) {
    const int r = i * 16 + first;
    float v[8];
    uint32_t m;
    if (pieces) {
      if constexpr (!VEC) raw[i].shift(by);
      raw[i].clear_unless(inside && r <= most);
      u4* to = reinterpret_cast<u4*>(&tile[r][at]);
      to[0] = raw[i].w[0];
      if constexpr (T == T_F32) to[1] = raw[i].w[1];
      if constexpr (BOTH) {
        raw[i].unpack(v);
        m = raw[i].magnitude();
      }
    } else {
      load_piece<T>(P, r0 + r, c0 + at, v);
      store8<T>(&tile[r][0], at, v);              // (exact: the values are of type T)
      m = magnitude8(v);
    }
    if constexpr (BOTH) {
      const uint32_t code = mx_scale_code(max_u32_lanes4(m), floor_bits);
      if (r <= most && piece < 4 * row_blocks) {
        row_codes[(int64_t)r * row_blocks * 4] = e2m1_codes8<T>(v, code);
        if ((piece & 3) == 0) row_scales[(int64_t)r * row_blocks] = (uint8_t)code;
      }
    }
  }
  __syncthreads();
  {
    const int c = threadIdx.x % (C / PAIR) * PAIR, b = threadIdx.x / (C / PAIR);
    static_assert(C / PAIR * B == 256, "a thread for each");
    uint32_t w[32];
#pragma unroll
    for (int k = 0; k < 32; ++k) w[k] = *reinterpret_cast<const uint32_t*>(&tile[32 * b + k][c]);
    __syncthreads();
    uint32_t pairs = 0;                            // 16 bits: both columns' magnitudes
    if constexpr (PAIR == 2)
#pragma unroll
      for (int k = 0; k < 32; ++k) pairs = max_pairs(pairs, w[k]);
#pragma unroll
    for (int h = 0; h < PAIR; ++h) {
      float v[32];
      uint32_t m = 0;
      if constexpr (PAIR == 2) m = magnitude_bits<T>(h ? pairs >> 16 : pairs & 0xffffu);
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        if constexpr (T == T_F32) v[k] = __uint_as_float(w[k]), m = max_u32(m, magnitude(v[k]));
        else if constexpr (T == T_F16) v[k] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[k] >> (16 * h)));
        else v[k] = __uint_as_float(h ? w[k] & 0xffff0000u : w[k] << 16);
      }
      const uint32_t code = mx_scale_code(m, floor_bits);
      u4 q;
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = e2m1_codes8<T>(v + 8 * k, code);
      codes[b][c + h] = q;
      scales[c + h][b] = (uint8_t)code;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < C * B; i += 256) {
    const int c = i / B, b = i % B;
    if (c0 + c >= P.cols || r0 / 32 + b >= col_blocks) continue;
    const int64_t block = (c0 + c) * col_blocks + r0 / 32 + b;
    reinterpret_cast<u4*>(P.t_codes)[block] = codes[b][c];
    P.t_scales[block] = scales[c][b];
  }
}

}  // namespace

extern "C" {

int dgm_mxfp4_quant_struct_size(size_t* args) {
  DGM_CHECK_ARG(args, "null pointer");
  *args = sizeof(DgmMxfp4QuantArgs);
  return 0;
}

int dgm_mxfp4_quantize(const DgmMxfp4QuantArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmMxfp4QuantArgs A = *args;
  DGM_CHECK_ARG(A.dtype >= DGM_SRC_BF16 && A.dtype <= DGM_SRC_F32, "dtype 0 bf16, 1 fp16, 2 fp32");
  DGM_CHECK_ARG(A.rows >= 0 && A.rows < (1 << 24) && A.cols >= 0 && A.cols < (1 << 24), "rows and columns below 2^24");
  DGM_CHECK_ARG(A.x_stride >= 0, "stride >= 0");
  DGM_CHECK_ARG(A.amax_floor >= 0.f && A.amax_floor < INFINITY, "amax_floor a number, at least 0");
  DGM_CHECK_ARG((A.codes != nullptr) == (A.scales != nullptr) && (A.t_codes != nullptr) == (A.t_scales != nullptr),
                "codes with their scales");
  if (A.rows == 0 || A.cols == 0) return 0;
  DGM_CHECK_ARG(A.x && (A.codes || A.t_codes), "null pointer");
  DGM_CHECK_ARG((((uintptr_t)A.codes | (uintptr_t)A.t_codes) & 15) == 0, "codes on 16 bytes");
  const bool vec = A.cols % 8 == 0 && aligned(A.x, A.x_stride, element_size(A.dtype));
  const int64_t pieces = (A.cols + 31) / 32 * 4;
  // threads a row: the most that leave few without a piece
  int log_row = 2, runs = 1;
  double best = 0;
  for (int l = 2; l <= 8; ++l) {
    const int64_t n = (pieces + (1 << l) - 1) >> l;
    const double used = (double)pieces / (double)(n << l);
    if (used >= best - 0.05) log_row = l, runs = (int)n, best = used > best ? used : best;
  }
  const int64_t groups = (A.rows + (256 >> log_row) - 1) >> (8 - log_row);
  const int tile_rows = A.dtype == DGM_SRC_F32 ? 64 : 128;
  const int64_t tiles_c = (A.cols + 127) / 128, tiles_r = (A.rows + tile_rows - 1) / tile_rows;
  DGM_CHECK_ARG(A.t_codes ? tiles_c * tiles_r < (1 << 24) : groups * runs < ((int64_t)1 << 32) - (1 << 23), "a launch has fewer than 2^32 threads (rows alone: workgroups)");
  // (a launch has fewer than 2^32 threads along a grid's axis)
  const unsigned grid_x = (unsigned)std::min(groups * runs, (int64_t)1 << 23);
  dispatch_type(A.dtype, vec, [&](auto t, auto v) {
    const unsigned tiles = (unsigned)(tiles_c * tiles_r);
    if (!A.t_codes)
      hipLaunchKernelGGL((k_mxfp4_rows<t.value, v.value>), dim3(grid_x, (unsigned)((groups * runs + grid_x - 1) / grid_x)), dim3(256), 0, stream,
                         A, log_row, runs);
    else if (A.codes)
      hipLaunchKernelGGL((k_mxfp4_columns<t.value, v.value, true>), dim3(tiles), dim3(256), 0, stream, A, (int)tiles_c);
    else
      hipLaunchKernelGGL((k_mxfp4_columns<t.value, v.value, false>), dim3(tiles), dim3(256), 0, stream, A, (int)tiles_c);
  });
  return dgm_last_launch_status();
}

}  // extern "C"
