// MXFP4 x MXFP4 product (gfx950): rows of E2M1 codes, two a byte, with an E8M0 scale for each 32 of them,
//   D[m][n] = sum over blocks b of 2^(sa[m][b] - 127) 2^(sb[n][b] - 127) sum_k A[m][k] B[n][k]   (+ C[m][n] or C[n]),
// or, with SwiGLU over a gate and an up half of B's rows (I = N / 2 each),
//   D[m][i] = silu(min(g, c)) * clamp(u, -c, c), g = product with row i, u = with row I + i.
// Products and scales go through the block-scaled matrix instruction, sums are fp32, and C and SwiGLU too; the result
// is rounded once to D's type.
//
// The weights are the matrix core's A operand and the tokens its B operand, so that a lane's result registers hold
// consecutive channels of one token. The instruction sums 128 of K: lane group g (lanes 16 g ..) brings one block of 32
// and its scale byte. Which block that is does not matter to the sum, so a step of 256 gives group g the two
// neighbouring blocks 2 g and 2 g + 1 (32 bytes of codes and 2 of scales), one for each of two instructions.
#include "dgm_common.hpp"
#include "dgm_abi_internal.hpp"
#include "dgm_epilogue.hpp"

using namespace dgm;

namespace {

DGM_DEV v8i operand(v4i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
template <int J>
DGM_DEV v4f mfma_fp4(v4i a, v4i b, v4f c, int sa, int sb) {
  return mfma_scale_16x16x128_sel<4, 4, J, J>(operand(a), operand(b), c, sa, sb);
}

// Scale bytes of blocks b and b + 1 of a row of n: 1.0 behind the last.
DGM_DEV int load_scales2(const uint8_t* row, int b, int n) {
  const int lo = b < n ? row[b] : 127, hi = b + 1 < n ? row[b + 1] : 127;
  return lo | hi << 8;
}

template <int T, bool ADD, bool SWIGLU, bool WHOLE>
DGM_DEV void put4_sums(const DgmMxfp4GemmArgs& P, int64_t m, int64_t n, int64_t n_out, v4f acc, v4f up) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = SWIGLU ? swiglu(acc[i], up[i], P.clamp, P.fast_math) : acc[i];
  put4<T, ADD, WHOLE>(P, m, n, n_out, v);
}

// Few tokens (16 MT per workgroup): the weights are read once per workgroup row, straight into registers. A
// workgroup's eight waves take steps of 256 of K in turn (lane l: 32 bytes of row l % 16, so a step's rows are read
// in whole 128-byte lines); the waves' sums meet in LDS in a fixed order.
// KP parts of K share a fragment: its 16 rows are 16 / KP weight rows in each part, its 16 token columns 16 / KP
// tokens in each, and of the products those of a part with itself count. A workgroup has CH channels; SwiGLU with
// CH below the rows of a part holds gate and up rows in one fragment, else in one each.
template <int MT, int KP, int CH, bool SWIGLU>
__global__ void __launch_bounds__(512) k_mxfp4_gemm_rows(const DgmMxfp4GemmArgs P, int vec) {
  constexpr int W = 8, ROWS = 16 / KP, H = SWIGLU && CH == ROWS ? 2 : 1;
  static_assert(KP == 1 || MT == 1, "parts of K share the token columns");
  static_assert(CH % 4 == 0 && (CH == ROWS || (SWIGLU && 2 * CH == ROWS)), "four channels a lane");
  __shared__ v4f sums[W][H * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int K = (int)P.k / 2, blocks = (int)P.k / 32;          // bytes of a row, blocks
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n, m0 = (int64_t)blockIdx.y * (ROWS * MT), n0 = (int64_t)blockIdx.x * CH;
  const int part = (K + 128 * KP - 1) / (128 * KP) * 128;      // of a row
  const uint8_t *a[MT], *sa[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + 16 * t + r % ROWS, row = m < P.m ? m : P.m - 1;
    a[t] = P.a + row * P.a_stride;
    sa[t] = P.sfa + row * P.sfa_stride;
  }
  const uint8_t *b[H], *sb[H];
  const int64_t n_row = n0 + r % CH < n_out ? n0 + r % CH : n_out - 1;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int64_t row = h == 0 && r % ROWS < CH ? n_row : n_out + n_row;
    b[h] = P.b + row * P.b_stride;
    sb[h] = P.sfb + row * P.sfb_stride;
  }
  v4f acc[H][MT];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[h][t] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave * 128; k0 < part; k0 += W * 128) {
    const int k = r / ROWS * part + k0 + 32 * g;
    v4i bv[H][2], av[MT][2];
    int bs[H], as[MT];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      // (behind K: any codes of the row against a token's zeros)
      const int at = k + 16 * j < K ? k + 16 * j : K - 16;
#pragma unroll
      for (int h = 0; h < H; ++h) bv[h][j] = *reinterpret_cast<const v4i*>(b[h] + at);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        av[t][j] = *reinterpret_cast<const v4i*>(a[t] + at);
        if (k + 16 * j >= K) av[t][j] = v4i{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int h = 0; h < H; ++h) bs[h] = load_scales2(sb[h], k / 16, blocks);
#pragma unroll
    for (int t = 0; t < MT; ++t) as[t] = load_scales2(sa[t], k / 16, blocks);
    static_for<2>([&](auto j) {
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[h][t] = mfma_fp4<j.value>(bv[h][j.value], av[t][j.value], acc[h][t], bs[h], as[t]);
    });
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
  v4f s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
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
  with_epilogue(P, [&](auto t, auto add) {
    if (vec && n + 3 < n_out) put4_sums<t.value, add.value, SWIGLU, true>(P, m, n, n_out, s[0], s[1]);
    else put4_sums<t.value, add.value, SWIGLU, false>(P, m, n, n_out, s[0], s[1]);
  });
}

__device__ const uint4 k_zeros = {0u, 0u, 0u, 0u};

// More tokens: a workgroup computes BM tokens x BN channels over steps of 256 of K (128 bytes a row, whole lines).
// Both operands' codes go from HBM / L2 straight into LDS, STAGES - 1 steps ahead of the one that is multiplied, with
// one barrier a step. A row's eight 16-byte pieces lie permuted by the row's number, so that the lanes reading one
// piece of 16 rows meet 16 different bank groups. Scales take the way through registers, a row's 16 bytes for two
// steps by one thread, two steps ahead: any alignment, and 1.0 behind K.
// SwiGLU: blocks of 16 channel rows alternate between gate and up rows, so that a wave holds both of a channel.
// Few tiles: gridDim.y workgroups share a tile, each a range of K, and leave their sums in the workspace
// [split][token][channel] for k_mxfp4_gemm_join.
template <int BM, int BN, int WM, int WN, int STAGES, bool SWIGLU>
__global__ void __launch_bounds__(64 * WM * WN) k_mxfp4_gemm_tiles(const DgmMxfp4GemmArgs P, int vec, int tiles_m, int tiles_n,
                                                                   int steps_per_split) {
  constexpr int W = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, ROWS = BM + BN, LOADS = ROWS / (8 * W);
  static_assert(ROWS % (8 * W) == 0 && BM % (8 * W) == 0 && W % 2 == 0 && TM % 2 == 0 && (!SWIGLU || TN % 2 == 0), "whole loads per wave");
  static_assert(64 * W >= ROWS, "a thread for each row's scales");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES][ROWS * 128];
  __shared__ __attribute__((aligned(16))) uint8_t lds_scales[2][ROWS * 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.y, k_begin = split * steps_per_split * 128;               // (bytes of a row)
  const int K = min((int)P.k / 2, k_begin + steps_per_split * 128);      // end of this workgroup's range
  // Workgroups go to the 8 XCDs in turn: each XCD gets a contiguous run of tiles, ordered in bands of 8
  // token tiles, so that the tiles an XCD works on at a time share rows in its L2.
  const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
  const int tile = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (tile >= tiles) return;
  const int band = tile / (8 * tiles_n), in_band = tile - band * 8 * tiles_n, bm = min(8, tiles_m - 8 * band);
  const int64_t m0 = (int64_t)(8 * band + in_band % bm) * BM, n0 = (int64_t)(in_band / bm) * (SWIGLU ? BN / 2 : BN);
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n;
  // memory row of the tile's row
  auto token_row = [&](int row) { const int64_t m = m0 + row; return m < P.m ? m : P.m - 1; };
  auto channel_row = [&](int rb) {
    int64_t n = SWIGLU ? n0 + (rb >> 5) * 16 + (rb & 15) : n0 + rb;
    n = n < n_out ? n : n_out - 1;
    return SWIGLU && (rb & 16) ? n + n_out : n;
  };
  // each wave's loads: LOADS times eight rows of the token tile, then of the channel tile
  const int piece = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4));
  const uint8_t* src[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = (i * W + wave) * 8 + (lane >> 3);
    src[i] = (i * W * 8 < BM ? P.a + token_row(row) * P.a_stride : P.b + channel_row(row - BM) * P.b_stride) + 16 * piece;
  }
  const int scale_row = min((int)threadIdx.x, ROWS - 1);
  const uint8_t* scales = scale_row < BM ? P.sfa + token_row(scale_row) * P.sfa_stride : P.sfb + channel_row(scale_row - BM) * P.sfb_stride;
  auto load = [&](const uint8_t* from, uint8_t* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  };
  // Pieces behind K are zeros. (Their address is kept from the compiler's view: it would branch on a lane's
  // piece and issue two loads, and the waits below count them.)
  uint64_t zeros = (uint64_t)&k_zeros;
  asm("" : "+v"(zeros));
  auto fetch = [&](int k0, uint8_t* to) {
    if (k0 + 128 <= K) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) load(src[i] + k0, to + (i * W + wave) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        load((const uint8_t*)(k0 + 16 * piece < K ? (uint64_t)src[i] + (uint64_t)k0 : zeros), to + (i * W + wave) * 1024);
    }
  };
  // a row's scales of the 16 blocks from byte k0 of its codes on
  auto fetch_scales = [&](int k0) {
    v4i s = {0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f};
    if (k0 + 256 <= K) __builtin_memcpy(&s, scales + k0 / 16, 16);
    else if (k0 < K)
      for (int i = 0; i < (K - k0) / 16; ++i) {
        const uint32_t byte = scales[k0 / 16 + i];
        const uint32_t shift = 8 * (i & 3);
#pragma unroll
        for (int d = 0; d < 4; ++d)
          if (d == i >> 2) s[d] = (int)(((uint32_t)s[d] & ~(0xffu << shift)) | byte << shift);
      }
    return s;
  };
  auto keep_scales = [&](v4i s, int set) {
    if ((int)threadIdx.x < ROWS) *reinterpret_cast<v4i*>(&lds_scales[set][threadIdx.x * 16]) = s;
  };
  v4f acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m) acc[n][m] = v4f{0.f, 0.f, 0.f, 0.f};
  const int r = lane & 15, g = lane >> 4, wm = wave % WM, wn = wave / WM;
  const int row_a = wm * (BM / WM) + r, row_b = BM + wn * (BN / WN) + r;
  auto multiply = [&](const uint8_t* from, const uint8_t* sc) {
    int as[TM], bs[TN];
#pragma unroll
    for (int n = 0; n < TN; ++n) bs[n] = *reinterpret_cast<const uint16_t*>(sc + (row_b + 16 * n) * 16 + 2 * g);
#pragma unroll
    for (int m = 0; m < TM; ++m) as[m] = *reinterpret_cast<const uint16_t*>(sc + (row_a + 16 * m) * 16 + 2 * g);
    static_for<2>([&](auto j) {
      const int at = ((2 * g + j.value) ^ ((r >> 1) & 7)) * 16;
      v4i av[TM], bv[TN];
#pragma unroll
      for (int n = 0; n < TN; ++n) bv[n] = *reinterpret_cast<const v4i*>(from + (row_b + 16 * n) * 128 + at);
#pragma unroll
      for (int m = 0; m < TM; ++m) av[m] = *reinterpret_cast<const v4i*>(from + (row_a + 16 * m) * 128 + at);
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[n][m] = mfma_fp4<j.value>(bv[n], av[m], acc[n][m], bs[n], as[m]);
    });
  };
  keep_scales(fetch_scales(k_begin), 0);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(k_begin + 128 * i, lds[i]);
  // A step: this wave's loads of it have landed (those of the STAGES - 2 steps behind it may be under way)
  // and its LDS accesses of the step before are done; behind the barrier that holds for every wave, so
  // the step can be read and the buffer of the step before filled again. Scales come before the codes that are
  // requested behind them, so the count below covers them too; they are kept in LDS in the second of a pair of steps.
  v4i next_scales = {0, 0, 0, 0};
  for (int k0 = k_begin, turn = 0, step = 0; k0 < K; k0 += 128, ++step) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * LOADS) : "memory");
    if ((step & 1) == 0) next_scales = fetch_scales(k0 + 256);
    fetch(k0 + 128 * (STAGES - 1), lds[turn == 0 ? STAGES - 1 : turn - 1]);
    multiply(lds[turn], &lds_scales[(step >> 1) & 1][8 * (step & 1)]);
    if (step & 1) keep_scales(next_scales, ((step >> 1) & 1) ^ 1);
    turn = turn + 1 == STAGES ? 0 : turn + 1;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // (the zeros behind the last step)
  // Results through LDS, 32 tokens of a wave at a time: from the lanes' four channels of 32 tokens to 16-byte
  // pieces of whole token rows. Rows are padded by 16 bytes, so that neither side meets bank conflicts.
  constexpr int H = SWIGLU ? 2 : 1, CW = 16 * TN / H, PITCH = CW + 4;
  // (SwiGLU: the wave's fragments of 16 channels are gate and up rows in turn)
  auto frag = [](int n, int h) { return SWIGLU ? 2 * n + h : n; };
  static_assert(W * 32 * PITCH * 4 <= (int)sizeof(lds), "the waves' parts fit");
  __syncthreads();
  float* part = reinterpret_cast<float*>(&lds[0][0]) + wave * 32 * PITCH;
  const int64_t c0 = n0 + wn * CW, t0 = m0 + wm * (BM / WM);
  if (gridDim.y > 1) {
    float* ws = P.workspace + (int64_t)split * P.m * P.n;
#pragma unroll
    for (int m = 0; m < TM / 2; ++m)
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int n = 0; n < TN / H; ++n)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            *reinterpret_cast<v4f*>(part + (16 * q + r) * PITCH + 16 * n + 4 * g) = acc[frag(n, h)][2 * m + q];
        wave_sync();
        constexpr int L = CW / 4;
#pragma unroll
        for (int j = 0; j < 32 * L / 64; ++j) {
          const int row = (64 * j + lane) / L, col = (64 * j + lane) % L * 4;
          const int64_t token = t0 + 32 * m + row, c = c0 + col;
          if (token >= P.m || c >= n_out) continue;
          const v4f v = *reinterpret_cast<const v4f*>(part + row * PITCH + col);
          float* to = ws + token * P.n + (h ? n_out : 0) + c;
          if (P.n % 4 == 0 && n_out % 4 == 0) *reinterpret_cast<v4f*>(to) = v;
          else
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c + i < n_out) to[i] = v[i];
        }
        wave_sync();
      }
    return;
  }
#pragma unroll
  for (int m = 0; m < TM / 2; ++m) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int n = 0; n < TN / H; ++n) {
        v4f v = acc[frag(n, 0)][2 * m + q];
        if constexpr (SWIGLU)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = swiglu(v[i], acc[frag(n, 1)][2 * m + q][i], P.clamp, P.fast_math);
        *reinterpret_cast<v4f*>(part + (16 * q + r) * PITCH + 16 * n + 4 * g) = v;
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

// The splits' sums added in their order, then as the tiles' epilogue: a thread takes four channels of a token.
template <bool SWIGLU>
__global__ void __launch_bounds__(256) k_mxfp4_gemm_join(const DgmMxfp4GemmArgs P, int vec, int splits) {
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n, quads = (n_out + 3) / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= quads * P.m) return;
  const int64_t m = id / quads, n = (id - m * quads) * 4;
  v4f s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  const bool four = P.n % 4 == 0 && n_out % 4 == 0;
#pragma unroll 4
  for (int k = 0; k < splits; ++k)
#pragma unroll
    for (int h = 0; h < (SWIGLU ? 2 : 1); ++h) {
      const float* from = P.workspace + ((int64_t)k * P.m + m) * P.n + (h ? n_out : 0) + n;
      if (four) s[h] += *reinterpret_cast<const v4f*>(from);
      else
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < n_out) s[h][i] += from[i];
    }
  with_epilogue(P, [&](auto t, auto add) {
    if (vec && n + 3 < n_out) put4_sums<t.value, add.value, SWIGLU, true>(P, m, n, n_out, s[0], s[1]);
    else put4_sums<t.value, add.value, SWIGLU, false>(P, m, n, n_out, s[0], s[1]);
  });
}

// Parts of K and channels of a workgroup of the rows kernel.
struct Rows { int parts, channels; };
Rows rows_form(int64_t m, int64_t n, int64_t k, bool swiglu) {
  const int parts = (m <= 8 && n <= 2048 && k >= 4096) || (m <= 2 && k >= 8192) ? 2 : 1;
  const bool one = swiglu && (parts == 2 || m <= 8 || n <= 4096);
  return {parts, 16 / parts / (one ? 2 : 1)};
}

template <int MT, int KP, int CH, bool SWIGLU>
void launch_rows(const DgmMxfp4GemmArgs& A, int vec, hipStream_t stream) {
  const int64_t n_out = SWIGLU ? A.n / 2 : A.n, tokens = 16 / KP * MT;
  const dim3 grid((unsigned)((n_out + CH - 1) / CH), (unsigned)((A.m + tokens - 1) / tokens));
  hipLaunchKernelGGL((k_mxfp4_gemm_rows<MT, KP, CH, SWIGLU>), grid, dim3(512), 0, stream, A, vec);
}
template <int MT>
void launch_rows(const DgmMxfp4GemmArgs& A, int vec, hipStream_t stream) {
  const Rows f = rows_form(A.m, A.n, A.k, A.swiglu != 0);
  if constexpr (MT == 1)
    if (f.parts == 2) return A.swiglu ? launch_rows<1, 2, 4, true>(A, vec, stream) : launch_rows<1, 2, 8, false>(A, vec, stream);
  if (!A.swiglu) launch_rows<MT, 1, 16, false>(A, vec, stream);
  else if (f.channels == 8) launch_rows<MT, 1, 8, true>(A, vec, stream);
  else launch_rows<MT, 1, 16, true>(A, vec, stream);
}

template <int BM, int BN, int WM, int WN, int STAGES>
void launch_tiles(const DgmMxfp4GemmArgs& A, int vec, int splits, hipStream_t stream) {
  const int tiles_m = (int)((A.m + BM - 1) / BM), tiles_n = (int)((A.n + BN - 1) / BN), steps = (int)((A.k + 255) / 256);
  const int per = (steps + splits - 1) / splits;
  splits = (steps + per - 1) / per;                // (every split has a step)
  const dim3 grid((unsigned)((tiles_m * tiles_n + 7) / 8 * 8), (unsigned)splits), block(64 * WM * WN);
  if (A.swiglu) hipLaunchKernelGGL((k_mxfp4_gemm_tiles<BM, BN, WM, WN, STAGES, true>), grid, block, 0, stream, A, vec, tiles_m, tiles_n, per);
  else hipLaunchKernelGGL((k_mxfp4_gemm_tiles<BM, BN, WM, WN, STAGES, false>), grid, block, 0, stream, A, vec, tiles_m, tiles_n, per);
  if (splits == 1) return;
  const int64_t quads = ((A.swiglu ? A.n / 2 : A.n) + 3) / 4 * A.m;
  const dim3 join((unsigned)((quads + 255) / 256));
  if (A.swiglu) hipLaunchKernelGGL(k_mxfp4_gemm_join<true>, join, dim3(256), 0, stream, A, vec, splits);
  else hipLaunchKernelGGL(k_mxfp4_gemm_join<false>, join, dim3(256), 0, stream, A, vec, splits);
}

// Which kernel takes a product, from estimates of its time in us (256 CUs): a tile form takes `alone` us per step of
// K while every workgroup has a CU to itself, `full` us when the CUs hold as many as fit, and 4.2 us around it;
// splitting K costs a second launch, 0.35 us a split and the sums' way through memory.
struct Form { int kind, splits; };
enum { ROWS = 0, T64, T64_128, T128, T128_256, T256 };
Form choose(int64_t m, int64_t n, int64_t k, bool swiglu, int64_t workspace_bytes) {
  static const struct { int bm, bn, per_cu; double alone, full; } tiles[] = {
      {0, 0, 0, 0, 0}, {64, 64, 2, 0.36, 0.64}, {64, 128, 2, 0.55, 0.88}, {128, 128, 1, 0.67, 0.67}, {128, 256, 1, 1.1, 1.1}, {256, 256, 1, 1.65, 1.65}};
  const int64_t steps = (k + 255) / 256;
  Form best = {ROWS, 1};
  double least = 1e30;
  if (m <= 64) {
    const Rows f = rows_form(m, n, k, swiglu);
    const double c = (m <= 4 ? 0.75 : m <= 16 ? 1.25 : m <= 32 ? 1.65 : 2.8) *
                     (!swiglu || f.channels < 16 / f.parts ? 1.0 : m <= 16 ? 1.75 : 2.0);
    const int64_t wgs = (n / (swiglu ? 2 : 1) + f.channels - 1) / f.channels;
    least = 2 + (double)((k + 2048 * f.parts - 1) / (2048 * f.parts)) * c * (double)((wgs + 255) / 256);
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

int dgm_mxfp4_gemm_struct_size(size_t* args) {
  DGM_CHECK_ARG(args, "null pointer");
  *args = sizeof(DgmMxfp4GemmArgs);
  return 0;
}

int64_t dgm_mxfp4_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k, int swiglu) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Form f = choose(m, n, k, swiglu != 0, MOST_WORKSPACE);
  return f.splits == 1 ? 0 : (int64_t)f.splits * m * n * 4;
}

int dgm_mxfp4_gemm_nt(const DgmMxfp4GemmArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmMxfp4GemmArgs A = *args;
  DGM_CHECK_ARG(A.dtype >= DGM_SRC_BF16 && A.dtype <= DGM_SRC_F32, "dtype 0 bf16, 1 fp16, 2 fp32");
  DGM_CHECK_ARG(A.m >= 0 && A.m < (1 << 24) && A.n >= 0 && A.n < (1 << 24), "m and n below 2^24");
  DGM_CHECK_ARG(A.k > 0 && A.k < (1 << 24) && A.k % 32 == 0, "k a multiple of 32 below 2^24");
  DGM_CHECK_ARG(!A.swiglu || (A.n % 2 == 0 && !A.c), "SwiGLU: a gate and an up half, no C");
  DGM_CHECK_ARG(A.a_stride >= 0 && A.b_stride >= 0 && A.sfa_stride >= 0 && A.sfb_stride >= 0 && A.c_stride >= 0 &&
                    A.d_stride >= 0, "strides >= 0");
  DGM_CHECK_ARG(((uint64_t)A.a_stride | (uint64_t)A.b_stride | (uintptr_t)A.a | (uintptr_t)A.b) % 16 == 0, "code rows on 16 bytes");
  if (A.m == 0 || A.n == 0) return 0;
  DGM_CHECK_ARG(A.a && A.b && A.sfa && A.sfb && A.d, "null pointer");
  // (a launch has fewer than 2^32 threads; the smallest tile has 64 x 64 results and 256 of them)
  DGM_CHECK_ARG(((A.m + 63) / 64) * ((A.n + 63) / 64) < (1 << 23), "m n / 4096 below 2^23");
  const int e = A.dtype == DGM_SRC_F32 ? 4 : 2;
  const int vec = (((uintptr_t)A.d | (uintptr_t)A.c | (uint64_t)(A.d_stride * e) | (uint64_t)(A.c_stride * e)) & 15) == 0;
  const int64_t held = A.workspace && ((uintptr_t)A.workspace & 15) == 0 ? A.workspace_bytes : 0;
  const Form f = choose(A.m, A.n, A.k, A.swiglu != 0, held < MOST_WORKSPACE ? held : MOST_WORKSPACE);
  if (f.kind == T64) launch_tiles<64, 64, 2, 2, 4>(A, vec, f.splits, stream);
  else if (f.kind == T64_128) launch_tiles<64, 128, 2, 4, 3>(A, vec, f.splits, stream);
  else if (f.kind == T128) launch_tiles<128, 128, 2, 4, 4>(A, vec, f.splits, stream);
  else if (f.kind == T128_256) launch_tiles<128, 256, 2, 4, 3>(A, vec, f.splits, stream);
  else if (f.kind == T256) launch_tiles<256, 256, 2, 4, 2>(A, vec, f.splits, stream);
  else if (A.m <= 16) launch_rows<1>(A, vec, stream);
  else if (A.m <= 32) launch_rows<2>(A, vec, stream);
  else launch_rows<4>(A, vec, stream);
  return dgm_last_launch_status();
}

}  // extern "C"
