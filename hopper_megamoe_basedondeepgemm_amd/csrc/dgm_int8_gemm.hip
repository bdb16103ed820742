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
#include "dgm_epilogue.hpp"

using namespace dgm;

namespace {

// scales of channels n .. n + 3 (behind the last: its own)
DGM_DEV v4f load_scales(const DgmInt8GemmArgs& P, int64_t n, int64_t end) {
  v4f s;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = P.sfb[(n + i < end ? n + i : end - 1) * P.sfb_stride];
  return s;
}

// Channels n .. n + 3 of token m with their scales.
template <int T, bool ADD, bool SWIGLU, bool WHOLE>
DGM_DEV void put4_scaled(const DgmInt8GemmArgs& P, int64_t m, int64_t n, int64_t n_out, float sa, v4f sb, v4f su, v4i acc, v4i up) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (float)acc[i] * (sa * sb[i]);
    if constexpr (SWIGLU) v[i] = swiglu(v[i], (float)up[i] * (sa * su[i]), P.clamp, P.fast_math);
  }
  put4<T, ADD, WHOLE>(P, m, n, n_out, v);
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

// Few tokens, or rows off 16-byte alignment (16 MT tokens per workgroup): the weights are read once per
// workgroup row, straight into registers. A workgroup's eight waves take K blocks of 128 in turn (lane l: 32
// bytes of row l % 16, so a block's rows are read in whole 128-byte lines); the waves' int32 sums meet in LDS.
// KP parts of K share a fragment: its 16 rows are 16 / KP weight rows in each part, its 16 token columns 16 / KP
// tokens in each, and of the products those of a part with itself count. A workgroup has CH channels; SwiGLU with
// CH below the rows of a part holds gate and up rows in one fragment, else in one each.
// One token, 4096 x 2048: 4.2 us, 2.0 TB/s. (Two or four K blocks requested at once: no faster, or slower.)
template <int MT, int KP, int CH, bool SWIGLU, bool ALIGNED>
__global__ void __launch_bounds__(512) k_int8_gemm_rows(const DgmInt8GemmArgs P, int vec) {
  constexpr int W = 8, ROWS = 16 / KP, H = SWIGLU && CH == ROWS ? 2 : 1;
  static_assert(KP == 1 || MT == 1, "parts of K share the token columns");
  static_assert(CH % 4 == 0 && (CH == ROWS || (SWIGLU && 2 * CH == ROWS)), "four channels a lane");
  __shared__ v4i sums[W][H * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4, K = (int)P.k;
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n, m0 = (int64_t)blockIdx.y * (ROWS * MT), n0 = (int64_t)blockIdx.x * CH;
  const int part = (K + 128 * KP - 1) / (128 * KP) * 128;      // of K
  const int8_t* a[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + 16 * t + r % ROWS;
    a[t] = P.a + (m < P.m ? m : P.m - 1) * P.a_stride;
  }
  const int8_t* b[H];
  const int64_t n_row = n0 + r % CH < n_out ? n0 + r % CH : n_out - 1;
  b[0] = P.b + (r % ROWS < CH ? n_row : n_out + n_row) * P.b_stride;
  if constexpr (H == 2) b[1] = b[0] + n_out * P.b_stride;
  v4i acc[H][MT];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[h][t] = v4i{0, 0, 0, 0};
  for (int k0 = wave * 128; k0 < part; k0 += W * 128) {
    const int k = r / ROWS * part + k0 + 32 * g;
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
  if (wave >= MT || g >= CH / 4 || r >= ROWS) return;
  const int64_t m = m0 + 16 * wave + r;
  if (m >= P.m) return;
  // (part q: rows 4 g .. behind ROWS q, token column r behind ROWS q)
  v4i s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int q = 0; q < KP; ++q) {
      const int at = lane + q * (ROWS / 4 * 16 + ROWS);
      s[0] += sums[w][wave][at];
      if constexpr (SWIGLU) s[1] += H == 2 ? sums[w][MT + wave][at] : sums[w][wave][at + CH / 4 * 16];
    }
  const int64_t n = n0 + 4 * g;
  if (n >= n_out) return;
  const float sa = P.sfa[m * P.sfa_stride];
  const v4f sb = load_scales(P, n, n_out), su = SWIGLU ? load_scales(P, n_out + n, 2 * n_out) : sb;
  with_epilogue(P, [&](auto t, auto add) {
    if (vec && n + 3 < n_out) put4_scaled<t.value, add.value, SWIGLU, true>(P, m, n, n_out, sa, sb, su, s[0], s[1]);
    else put4_scaled<t.value, add.value, SWIGLU, false>(P, m, n, n_out, sa, sb, su, s[0], s[1]);
  });
}

__device__ const uint4 k_zeros = {0u, 0u, 0u, 0u};

// More tokens: a workgroup computes BM tokens x BN channels over K steps of 128 bytes (whole 128-byte lines:
// half lines, 64-byte steps, cost as many cycles of a CU's 64 B / clock). Both operands' rows go from HBM /
// L2 straight into LDS, STAGES - 1 steps ahead of the one that is multiplied, with one barrier a step. A
// row's eight 16-byte pieces lie permuted by the row's number, so that the lanes reading one piece of 16
// rows meet 16 different bank groups (no conflicts counted). The 16 x 16 x 64 matrix instruction, whose
// accumulators move half as often per product as those of 32 x 32 x 32: the large products run at the clock
// that the card's power allows, and 8192 x 8192 x 4096 takes 246 us with it instead of 276.
// SwiGLU: blocks of 16 channel rows alternate between gate and up rows, so that a wave holds both of a
// channel.
// Few tiles: gridDim.y workgroups share a tile, each a range of K, and leave their int32 sums in the
// workspace [split][token][channel] for k_int8_gemm_join.
template <int BM, int BN, int WM, int WN, int STAGES, bool SWIGLU>
__global__ void __launch_bounds__(64 * WM * WN) k_int8_gemm_tiles(const DgmInt8GemmArgs P, int vec, int tiles_m, int tiles_n,
                                                                  int steps_per_split) {
  constexpr int W = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, ROWS = BM + BN, LOADS = ROWS / (8 * W);
  static_assert(ROWS % (8 * W) == 0 && BM % (8 * W) == 0 && W % 2 == 0 && TM % 2 == 0 && (!SWIGLU || TN % 2 == 0), "whole loads per wave");
  __shared__ __attribute__((aligned(1024))) int8_t lds[STAGES][ROWS * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.y, k_begin = split * steps_per_split * 128;
  const int K = min((int)P.k, k_begin + steps_per_split * 128);          // end of this workgroup's range
  // Workgroups go to the 8 XCDs in turn: each XCD gets a contiguous run of tiles, ordered in bands of 8
  // token tiles, so that the tiles an XCD works on at a time share rows in its L2.
  const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
  int tile = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (tile >= tiles) return;
  const int band = tile / (8 * tiles_n), in_band = tile - band * 8 * tiles_n, bm = min(8, tiles_m - 8 * band);
  const int64_t m0 = (int64_t)(8 * band + in_band % bm) * BM, n0 = (int64_t)(in_band / bm) * (SWIGLU ? BN / 2 : BN);
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n;
  // each wave's loads: LOADS times eight rows of the token tile, then of the channel tile
  const int piece = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4));
  const int8_t* src[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = (i * W + wave) * 8 + (lane >> 3);
    if (i * W * 8 < BM) {
      const int64_t m = m0 + row;
      src[i] = P.a + (m < P.m ? m : P.m - 1) * P.a_stride + 16 * piece;
    } else {
      const int rb = row - BM;
      int64_t n = SWIGLU ? n0 + (rb >> 5) * 16 + (rb & 15) : n0 + rb;
      n = n < n_out ? n : n_out - 1;
      if (SWIGLU && (rb & 16)) n += n_out;
      src[i] = P.b + n * P.b_stride + 16 * piece;
    }
  }
  auto load = [&](const int8_t* from, int8_t* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  };
  // Pieces behind K are zeros. (Their address is kept from the compiler's view: it would branch on a lane's
  // piece and issue two loads, and the waits below count them.)
  uint64_t zeros = (uint64_t)&k_zeros;
  asm("" : "+v"(zeros));
  auto fetch = [&](int k0, int8_t* to) {
    if (k0 + 128 <= K) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) load(src[i] + k0, to + (i * W + wave) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        load((const int8_t*)(k0 + 16 * piece < K ? (uint64_t)src[i] + (uint64_t)k0 : zeros), to + (i * W + wave) * 1024);
    }
  };
  v4i acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m) acc[n][m] = v4i{0, 0, 0, 0};
  const int r = lane & 15, g = lane >> 4, wm = wave % WM, wn = wave / WM;
  const int row_a = wm * (BM / WM) + r, row_b = BM + wn * (BN / WN) + r;
  auto multiply = [&](const int8_t* from) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int at = ((4 * kk + g) ^ ((r >> 1) & 7)) * 16;
      v4i av[TM], bv[TN];
#pragma unroll
      for (int n = 0; n < TN; ++n) bv[n] = *reinterpret_cast<const v4i*>(from + (row_b + 16 * n) * 128 + at);
#pragma unroll
      for (int m = 0; m < TM; ++m) av[m] = *reinterpret_cast<const v4i*>(from + (row_a + 16 * m) * 128 + at);
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[n][m] = mfma_i8_16x16x64(bv[n], av[m], acc[n][m]);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(k_begin + 128 * i, lds[i]);
  // A step: this wave's loads of it have landed (those of the STAGES - 2 steps behind it may be under way)
  // and its LDS reads of the step before have returned; behind the barrier that holds for every wave, so
  // the step can be read and the buffer of the step before filled again.
  for (int k0 = k_begin, turn = 0; k0 < K; k0 += 128) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * LOADS) : "memory");
    fetch(k0 + 128 * (STAGES - 1), lds[turn == 0 ? STAGES - 1 : turn - 1]);
    multiply(lds[turn]);
    turn = turn + 1 == STAGES ? 0 : turn + 1;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // (the zeros behind the last step)
  // Results through LDS, 32 tokens of a wave at a time: from the lanes' four channels of 32 tokens to 16-byte
  // pieces of whole token rows (stored from the lanes, a 8192 x 8192 output took 80 us longer). Rows are
  // padded by 16 bytes, so that neither side meets bank conflicts.
  constexpr int H = SWIGLU ? 2 : 1, CW = 16 * TN / H, PITCH = CW + 4;
  // (SwiGLU: the wave's fragments of 16 channels are gate and up rows in turn)
  auto frag = [](int n, int h) { return SWIGLU ? 2 * n + h : n; };
  static_assert(W * 32 * PITCH * 4 <= (int)sizeof(lds), "the waves' parts fit");
  __syncthreads();
  float* part = reinterpret_cast<float*>(&lds[0][0]) + wave * 32 * PITCH;
  const int64_t c0 = n0 + wn * CW, t0 = m0 + wm * (BM / WM);
  if (gridDim.y > 1) {
    int* ws = P.workspace + (int64_t)split * P.m * P.n;
#pragma unroll
    for (int m = 0; m < TM / 2; ++m)
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int n = 0; n < TN / H; ++n)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            *reinterpret_cast<v4i*>(part + (16 * q + r) * PITCH + 16 * n + 4 * g) = acc[frag(n, h)][2 * m + q];
        wave_sync();
        constexpr int L = CW / 4;
#pragma unroll
        for (int j = 0; j < 32 * L / 64; ++j) {
          const int row = (64 * j + lane) / L, col = (64 * j + lane) % L * 4;
          const int64_t token = t0 + 32 * m + row, c = c0 + col;
          if (token >= P.m || c >= n_out) continue;
          const v4i v = *reinterpret_cast<const v4i*>(part + row * PITCH + col);
          int* to = ws + token * P.n + (h ? n_out : 0) + c;
          if (P.n % 4 == 0 && n_out % 4 == 0) *reinterpret_cast<v4i*>(to) = v;
          else
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c + i < n_out) to[i] = v[i];
        }
        wave_sync();
      }
    return;
  }
  v4f sb[TN];
#pragma unroll
  for (int n = 0; n < TN / H; ++n) {
    const int64_t c = c0 + 16 * n + 4 * g;
    sb[frag(n, 0)] = load_scales(P, c, n_out);
    if constexpr (SWIGLU) sb[frag(n, 1)] = load_scales(P, n_out + c, 2 * n_out);
  }
#pragma unroll
  for (int m = 0; m < TM / 2; ++m) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t token = t0 + 32 * m + 16 * q + r;
      const float sa = P.sfa[(token < P.m ? token : P.m - 1) * P.sfa_stride];
#pragma unroll
      for (int n = 0; n < TN / H; ++n) {
        v4f v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = (float)acc[frag(n, 0)][2 * m + q][i] * (sa * sb[frag(n, 0)][i]);
          if constexpr (SWIGLU) v[i] = swiglu(v[i], (float)acc[frag(n, 1)][2 * m + q][i] * (sa * sb[frag(n, 1)][i]), P.clamp, P.fast_math);
        }
        *reinterpret_cast<v4f*>(part + (16 * q + r) * PITCH + 16 * n + 4 * g) = v;
      }
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

// The splits' sums added, then as the tiles' epilogue: a thread takes four channels of a token.
template <bool SWIGLU>
__global__ void __launch_bounds__(256) k_int8_gemm_join(const DgmInt8GemmArgs P, int vec, int splits) {
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n, quads = (n_out + 3) / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= quads * P.m) return;
  const int64_t m = id / quads, n = (id - m * quads) * 4;
  v4i s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  const bool four = P.n % 4 == 0 && n_out % 4 == 0;
#pragma unroll 4
  for (int k = 0; k < splits; ++k)
#pragma unroll
    for (int h = 0; h < (SWIGLU ? 2 : 1); ++h) {
      const int* from = P.workspace + ((int64_t)k * P.m + m) * P.n + (h ? n_out : 0) + n;
      if (four) s[h] += *reinterpret_cast<const v4i*>(from);
      else
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < n_out) s[h][i] += from[i];
    }
  const float sa = P.sfa[m * P.sfa_stride];
  const v4f sb = load_scales(P, n, n_out), su = SWIGLU ? load_scales(P, n_out + n, 2 * n_out) : sb;
  with_epilogue(P, [&](auto t, auto add) {
    if (vec && n + 3 < n_out) put4_scaled<t.value, add.value, SWIGLU, true>(P, m, n, n_out, sa, sb, su, s[0], s[1]);
    else put4_scaled<t.value, add.value, SWIGLU, false>(P, m, n, n_out, sa, sb, su, s[0], s[1]);
  });
}

// Parts of K and channels of a workgroup of the rows kernel (us, neighbour first).
// Two parts: half the rows a workgroup, twice the workgroups. Where 16 channels each leave CUs without one, or up
// to 2 tokens (whose rows cost nothing): 1 x 1024, K 8192 7.2 -> 5.3; 8 x 2048, K 4096 5.9 -> 5.0; 1 x 14336, K 4096
// 15.2 -> 13.2; but 4 x 8192, K 8192 16 -> 20 and, with too little K for the waves, 1 x 4096, K 2048 4.2 -> 4.5.
// SwiGLU with gate and up rows in one fragment: up to 8 tokens, or where it is needed to fill the CUs: 1 x 4096,
// K 7168 15.4 -> 10.4; 16 x 4096, K 7168 16.6 -> 12.1; but 16 x 8192, K 4096 12.8 -> 14.1 (token rows are read twice
// as often).
struct Rows { int parts, channels; };
Rows rows_form(int64_t m, int64_t n, int64_t k, bool swiglu) {
  const int parts = (m <= 8 && n <= 2048 && k >= 2048) || (m <= 2 && k >= 4096) ? 2 : 1;
  const bool one = swiglu && (parts == 2 || m <= 8 || n <= 4096);
  return {parts, 16 / parts / (one ? 2 : 1)};
}

template <int MT, int KP, int CH, bool SWIGLU>
void launch_rows(const DgmInt8GemmArgs& A, bool aligned, int vec, hipStream_t stream) {
  const int64_t n_out = SWIGLU ? A.n / 2 : A.n, tokens = 16 / KP * MT;
  const dim3 grid((unsigned)((n_out + CH - 1) / CH), (unsigned)((A.m + tokens - 1) / tokens));
  if (aligned) hipLaunchKernelGGL((k_int8_gemm_rows<MT, KP, CH, SWIGLU, true>), grid, dim3(512), 0, stream, A, vec);
  else hipLaunchKernelGGL((k_int8_gemm_rows<MT, KP, CH, SWIGLU, false>), grid, dim3(512), 0, stream, A, vec);
}
template <int MT>
void launch_rows(const DgmInt8GemmArgs& A, bool aligned, int vec, hipStream_t stream) {
  const Rows f = rows_form(A.m, A.n, A.k, A.swiglu != 0);
  if constexpr (MT == 1)
    if (f.parts == 2) return A.swiglu ? launch_rows<1, 2, 4, true>(A, aligned, vec, stream) : launch_rows<1, 2, 8, false>(A, aligned, vec, stream);
  if (!A.swiglu) launch_rows<MT, 1, 16, false>(A, aligned, vec, stream);
  else if (f.channels == 8) launch_rows<MT, 1, 8, true>(A, aligned, vec, stream);
  else launch_rows<MT, 1, 16, true>(A, aligned, vec, stream);
}

template <int BM, int BN, int WM, int WN, int STAGES>
void launch_tiles(const DgmInt8GemmArgs& A, int vec, int splits, hipStream_t stream) {
  const int tiles_m = (int)((A.m + BM - 1) / BM), tiles_n = (int)((A.n + BN - 1) / BN), steps = (int)((A.k + 127) / 128);
  const int per = (steps + splits - 1) / splits;
  splits = (steps + per - 1) / per;                // (every split has a step)
  const dim3 grid((unsigned)((tiles_m * tiles_n + 7) / 8 * 8), (unsigned)splits), block(64 * WM * WN);
  if (A.swiglu) hipLaunchKernelGGL((k_int8_gemm_tiles<BM, BN, WM, WN, STAGES, true>), grid, block, 0, stream, A, vec, tiles_m, tiles_n, per);
  else hipLaunchKernelGGL((k_int8_gemm_tiles<BM, BN, WM, WN, STAGES, false>), grid, block, 0, stream, A, vec, tiles_m, tiles_n, per);
  if (splits == 1) return;
  const int64_t quads = ((A.swiglu ? A.n / 2 : A.n) + 3) / 4 * A.m;
  const dim3 join((unsigned)((quads + 255) / 256));
  if (A.swiglu) hipLaunchKernelGGL(k_int8_gemm_join<true>, join, dim3(256), 0, stream, A, vec, splits);
  else hipLaunchKernelGGL(k_int8_gemm_join<false>, join, dim3(256), 0, stream, A, vec, splits);
}

// Which kernel takes an aligned product, from estimates of its time in us (256 CUs). A tile form takes `alone`
// us per K step while every workgroup has a CU to itself, `full` us when the CUs hold as many as fit, and 4.2 us
// around it; splitting K costs a second launch, 0.35 us a split and the sums' way through memory (3.2 TB/s). The times are
// fitted to 300 products of 1 to 12000 tokens with every form and split, none warm in the caches: the estimates'
// choice takes 0.5 % longer than the best form on average.
// Where each form is the best (us; next best):
//   64 x 64, 4 stages:    256 x 4096, K 2048: 8.8 (64 x 128 9.7);    200 x 2880, K 2880: 10.6 (12.1)
//   64 x 128, 3 stages:   300 x 5120, K 2880: 12.7 (64 x 64 15.9);   512 x 4096, K 2048: 10.4 (11.5)
//   128 x 128, 4 stages:  1024 x 4096, K 7168: 38.8 (192 x 128 46);  512 x 8192, K 4096: 25.4 (30)
//   128 x 128, 2 stages:  2048 x 4096, K 2048: 23.2 (128 x 256 24.3); 777 x 7168, K 2048: 20.8 (64 x 128 22)
//   192 x 128:            1000 x 5120, K 2880: 25.1 (128 x 128 28);  1536 x 4096, K 7168: 52 (58)
//   128 x 256:            512 x 16384, K 4096: 40 (128 x 128 45);    4096 x 2048, K 4096: 38 (41)
//   192 x 256:            1536 x 8192, K 4096: 53 (256 x 256 61);    4096 x 5120, K 2880: 82 (256 x 192 93)
//   256 x 192:            8192 x 2880, K 2880: 88 (192 x 128 98);    4096 x 2880, K 2880: 45 (256 x 256 50)
//   256 x 256:            8192 x 8192, K 4096: 243 (192 x 256 266);  2048 x 8192, K 4096: 69 (128 x 128 82)
// Up to 192 x 128 a step takes 2.5 to 3 times what the matrix instructions need; more stages, so more loads in flight,
// are no faster, and the cause is not known.
// The rows form takes 2 us and, per 1024 of a part of K and round of 256 workgroups, 0.75 us up to 4 tokens, 1.25
// up to 16, 1.65 up to 32 and 2.8 up to 64 (SwiGLU with a fragment each for gate and up rows 1.75 times the first
// two and twice the others): 16 x 4096, K 7168: 11.5 us (64 x 64, 4 splits 13); 32 x 8192, K 4096: 16.5 us (64 x 64,
// 2 splits 13.7).
struct Form { int kind, splits; };
enum { ROWS = 0, T64, T64_128, T128_DEEP, T128, T192_128, T128_256, T192_256, T256_192, T256 };
Form choose(int64_t m, int64_t n, int64_t k, bool swiglu, int64_t workspace_bytes) {
  static const struct { int bm, bn, per_cu; double alone, full; } tiles[] = {
      {0, 0, 0, 0, 0},           {64, 64, 2, 0.36, 0.64},  {64, 128, 2, 0.55, 0.88}, {128, 128, 1, 0.67, 0.67}, {128, 128, 2, 0.86, 1.14},
      {192, 128, 1, 0.85, 0.85}, {128, 256, 1, 1.1, 1.1},  {192, 256, 1, 1.28, 1.28}, {256, 192, 1, 1.35, 1.5},  {256, 256, 1, 1.65, 1.65}};
  const int64_t steps = (k + 127) / 128;
  Form best = {ROWS, 1};
  double least = 1e30;
  if (m <= 64) {
    const Rows f = rows_form(m, n, k, swiglu);
    const double c = (m <= 4 ? 0.75 : m <= 16 ? 1.25 : m <= 32 ? 1.65 : 2.8) *
                     (!swiglu || f.channels < 16 / f.parts ? 1.0 : m <= 16 ? 1.75 : 2.0);
    const int64_t wgs = (n / (swiglu ? 2 : 1) + f.channels - 1) / f.channels;
    least = 2 + (double)((k + 1024 * f.parts - 1) / (1024 * f.parts)) * c * (double)((wgs + 255) / 256);
  }
  for (int t = T64; t <= T256; ++t)
    for (int s = 1; s <= 8; s *= 2) {
      if (s > 1 && (steps < 2 * s || (int64_t)s * m * n * 4 > workspace_bytes)) break;
      const int64_t wgs = ((m + tiles[t].bm - 1) / tiles[t].bm) * ((n + tiles[t].bn - 1) / tiles[t].bn) * s;
      const int64_t rounds = (wgs + 256 * tiles[t].per_cu - 1) / (256 * tiles[t].per_cu);
      double us = 4.2 + (double)((steps + s - 1) / s) * (wgs <= 256 ? tiles[t].alone : tiles[t].full * (double)rounds);
      if (s > 1) us += 2.4 + 0.35 * s + 8e-6 / 3.2 * (double)s * (double)m * (double)n;
      if (us < least) least = us, best = {t, s};
    }
  return best;
}
// Sums of a split call above this are not worth their way through memory.
constexpr int64_t MOST_WORKSPACE = 64 << 20;

}  // namespace

extern "C" {

int dgm_int8_gemm_struct_size(size_t* args) {
  DGM_CHECK_ARG(args, "null pointer");
  *args = sizeof(DgmInt8GemmArgs);
  return 0;
}

int64_t dgm_int8_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k, int swiglu) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Form f = choose(m, n, k, swiglu != 0, MOST_WORKSPACE);
  return f.splits == 1 ? 0 : (int64_t)f.splits * m * n * 4;
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
  const int64_t held = A.workspace && ((uintptr_t)A.workspace & 15) == 0 ? A.workspace_bytes : 0;
  const Form f = aligned ? choose(A.m, A.n, A.k, A.swiglu != 0, held < MOST_WORKSPACE ? held : MOST_WORKSPACE) : Form{ROWS, 1};
  if (f.kind == T64) launch_tiles<64, 64, 2, 2, 4>(A, vec, f.splits, stream);
  else if (f.kind == T64_128) launch_tiles<64, 128, 2, 4, 3>(A, vec, f.splits, stream);
  else if (f.kind == T128_DEEP) launch_tiles<128, 128, 2, 4, 4>(A, vec, f.splits, stream);
  else if (f.kind == T128) launch_tiles<128, 128, 2, 4, 2>(A, vec, f.splits, stream);
  else if (f.kind == T192_128) launch_tiles<192, 128, 2, 4, 3>(A, vec, f.splits, stream);
  else if (f.kind == T128_256) launch_tiles<128, 256, 2, 4, 3>(A, vec, f.splits, stream);
  else if (f.kind == T192_256) launch_tiles<192, 256, 2, 4, 2>(A, vec, f.splits, stream);
  else if (f.kind == T256_192) launch_tiles<256, 192, 4, 2, 2>(A, vec, f.splits, stream);
  else if (f.kind == T256) launch_tiles<256, 256, 2, 4, 2>(A, vec, f.splits, stream);
  else if (A.m <= 16) launch_rows<1>(A, aligned, vec, stream);
  else if (A.m <= 32) launch_rows<2>(A, aligned, vec, stream);
  else launch_rows<4>(A, aligned, vec, stream);
  return dgm_last_launch_status();
}

}  // extern "C"
