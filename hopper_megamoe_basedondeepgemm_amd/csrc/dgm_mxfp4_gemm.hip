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

#include <algorithm>

using namespace dgm;

namespace {

DGM_DEV v8i operand(v4i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
template <int J>
DGM_DEV v4f mfma_fp4(v4i a, v4i b, v4f c, int sa, int sb) {
  return mfma_scale_16x16x128_sel<4, 4, J, J>(operand(a), operand(b), c, sa, sb);
}

// J scale bytes of a row of n from byte b on, zeros behind the last.
template <int J>
DGM_DEV int load_scales(const uint8_t* row, int b, int n) {
  uint32_t s = 0;
  if (b + J <= n) {
    __builtin_memcpy(&s, row + b, J);
  } else {
#pragma unroll
    for (int i = 0; i + 1 < J; ++i)
      if (b + i < n) s |= (uint32_t)row[b + i] << (8 * i);
  }
  return (int)s;
}

template <int T, bool ADD, bool SWIGLU, bool WHOLE>
DGM_DEV void put4_sums(const DgmMxfp4GemmArgs& P, int64_t m, int64_t n, int64_t n_out, v4f acc, v4f up) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = SWIGLU ? swiglu(acc[i], up[i], P.clamp, P.fast_math) : acc[i];
  put4<T, ADD, WHOLE>(P, m, n, n_out, v);
}

// Few tokens (16 MT per workgroup): the weights are read once per workgroup row, straight into registers. A
// workgroup's eight waves take steps of 128 J of K in turn, J = 2 or 4 instructions of 128 (lane l: J blocks of row
// l % 16 one behind the other, so a step's rows are read in whole 128-byte lines); the waves' sums meet in LDS in a
// fixed order.
// KP parts of K share a fragment: its 16 rows are 16 / KP weight rows in each part, its 16 token columns 16 / KP
// tokens in each, and of the products those of a part with itself count. A workgroup has CH channels; SwiGLU with
// CH below the rows of a part holds gate and up rows in one fragment, else in one each.
// One token, 4096 x 2048: 3.2 us; 4 tokens, 7168 x 7168: 8.5 us, 3.2 TB/s.
template <int MT, int KP, int CH, int J, bool SWIGLU>
__global__ void __launch_bounds__(512) k_mxfp4_gemm_rows(const DgmMxfp4GemmArgs P, int vec) {
  constexpr int W = 8, ROWS = 16 / KP, H = SWIGLU && CH == ROWS ? 2 : 1, STEP = 64 * J;
  static_assert(KP == 1 || MT == 1, "parts of K share the token columns");
  static_assert(CH % 4 == 0 && (CH == ROWS || (SWIGLU && 2 * CH == ROWS)), "four channels a lane");
  __shared__ v4f sums[W][H * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int K = (int)P.k / 2, blocks = (int)P.k / 32;          // bytes of a row, blocks
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n, m0 = (int64_t)blockIdx.y * (ROWS * MT), n0 = (int64_t)blockIdx.x * CH;
  const int part = (K + STEP * KP - 1) / (STEP * KP) * STEP;   // of a row
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
  for (int k0 = wave * STEP; k0 < part; k0 += W * STEP) {
    const int k = r / ROWS * part + k0 + 16 * J * g;
    v4i bv[H][J], av[MT][J];
    int bs[H], as[MT];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      // (behind K: any codes of the row against a token's zeros)
      const int at = k + 16 * j < K ? k + 16 * j : K - 16;
#pragma unroll
      for (int h = 0; h < H; ++h) bv[h][j] = *reinterpret_cast<const v4i*>(b[h] + at);
#pragma unroll
      for (int t = 0; t < MT; ++t) av[t][j] = *reinterpret_cast<const v4i*>(a[t] + at);
    }
#pragma unroll
    for (int h = 0; h < H; ++h) bs[h] = load_scales<J>(sb[h], k / 16, blocks);
#pragma unroll
    for (int t = 0; t < MT; ++t) as[t] = load_scales<J>(sa[t], k / 16, blocks);
    static_for<J>([&](auto j) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const v4i v = k + 16 * j.value < K ? av[t][j.value] : v4i{0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < H; ++h) acc[h][t] = mfma_fp4<j.value>(bv[h][j.value], v, acc[h][t], bs[h], as[t]);
      }
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

// More tokens: a workgroup computes BM tokens x BN channels over steps of 256 of K (128 bytes a row, whole lines).
// Both operands' codes go from HBM / L2 straight into LDS, STAGES - 1 steps ahead of the one that is multiplied, with
// one barrier a step. A row's eight 16-byte pieces (block 2 g + j at place 4 j + g) lie permuted by the row's number, so
// that the lanes of a read meet different banks (at place 2 g + j half of the LDS cycles were conflicts). Scales take the
// way through registers, a row's 16 bytes for two steps by one thread, a pair of steps ahead: any alignment.
// Behind K a row's last piece stands in for the missing ones (any finite codes), under scale bytes of 0 in both
// operands: 2^-127 each, so that such products are below 2^-240 and add nothing to an fp32 sum.
// SwiGLU: blocks of 16 channel rows alternate between gate and up rows, so that a wave holds both of a channel.
// Few tiles: gridDim.y workgroups share a tile, each a range of K, and leave their sums in the workspace
// [split][token][channel] for k_mxfp4_gemm_join.
// Bound: up to some hundred tokens the latency of a step (0.24 to 0.6 us, the loads' way from L2 and one barrier). Of
// 8192 x 8192, K 4096, 159 us (3.5 PFLOP/s), the instructions take 81 on such data (6.8 PFLOP/s from registers, where the
// card's power holds the clock; on zeros 61). Without results the kernel takes 120 (zeros 96): by count a step's 192 KB of
// reads from LDS and 64 KB into it are as many cycles as its products. The results' 39 us are under nothing else: a CU
// holds one workgroup and takes four tiles in turn.
// In the compiler's own order, everything read first and accumulators in scratch memory, it took 343. Not faster at their
// step: 256 workgroups that loop over tiles and request the next one's first step ahead (192 -> 197; 8192 x 4096 78 ->
// 87), whole 16-bit rows through LDS, four waves of 128 x 128 (the statements that keep the order hold accumulators in the
// 256 ordinary registers, which they fill; with them in the other 256 it is not tried) or sixteen of 64 x 64, fragments
// read three ahead.
// Eight waves a tile: with four, tiles of 128 x 128 wait longer for each step (8192 x 512, K 7168 23.6 -> 37; 777 x 5120,
// K 7168 by 192 x 128 25.5 -> 46); sixteen are 1 to 5 % slower.
template <int BM, int BN, int WM, int WN, int STAGES, bool SWIGLU>
__global__ void __launch_bounds__(64 * WM * WN) k_mxfp4_gemm_tiles(const DgmMxfp4GemmArgs P, int vec, int tiles_m, int tiles_n,
                                                                   int steps_per_split) {
  constexpr int W = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, ROWS = BM + BN, LOADS = ROWS / (8 * W), SCALES = (ROWS + 64 * W - 1) / (64 * W);
  static_assert(ROWS % (8 * W) == 0 && BM % (8 * W) == 0 && W % 2 == 0 && TM % 2 == 0 && (!SWIGLU || TN % 2 == 0), "whole loads per wave");
  // (one array: of two, the compiler knows which one the direct loads write and awaits them before every read of it)
  __shared__ __attribute__((aligned(1024))) uint8_t memory[STAGES * ROWS * 128 + 2 * ROWS * 16];
  uint8_t* const lds_scales = memory + STAGES * ROWS * 128;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.y, k_begin = split * steps_per_split * 128;               // (bytes of a row)
  const int K = min((int)P.k / 2, k_begin + steps_per_split * 128);      // end of this workgroup's range
  const int k_last = k_begin + (K - 1 - k_begin) / 128 * 128;            // its last step
  // Workgroups go to the 8 XCDs in turn: each XCD gets a contiguous run of tiles, ordered in bands of 8
  // token tiles, so that the tiles an XCD works on at a time share rows in its L2.
  const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
  const int tile = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (tile >= tiles) return;
  const int band = tile / (8 * tiles_n), in_band = tile - band * 8 * tiles_n, bm = min(8, tiles_m - 8 * band);
  const int64_t m0 = (int64_t)(8 * band + in_band % bm) * BM, n0 = (int64_t)(in_band / bm) * (SWIGLU ? BN / 2 : BN);
  const int64_t n_out = SWIGLU ? P.n / 2 : P.n;
  // rows of the tile from its first on, those behind the last token or channel being the last
  const int most_m = (int)min(P.m - m0, (int64_t)BM) - 1, most_n = (int)min(n_out - n0, (int64_t)BN) - 1;
  auto token_row = [&](int row) { return min(row, most_m); };
  auto channel_row = [&](int rb) { return min(SWIGLU ? (rb >> 5) * 16 + (rb & 15) : rb, most_n); };
  const uint8_t* const a0 = P.a + m0 * P.a_stride;
  const uint8_t* const b0 = P.b + n0 * P.b_stride;
  const uint8_t* const up0 = b0 + n_out * P.b_stride;
  auto buffer = [](const uint8_t* p) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, -1, 0x00020000); };
  const __amdgpu_buffer_rsrc_t tokens = buffer(a0), channels = buffer(b0), ups = buffer(up0);
  // each wave's loads: LOADS times eight rows of the token tile, then of the channel tile, at 32-bit offsets (buffer
  // instructions: behind the global ones into LDS the compiler awaits every load in flight for any value it needs)
  const int place = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4)), piece = 2 * (place & 3) + (place >> 2);
  uint32_t row_at[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = (i * W + wave) * 8 + (lane >> 3);
    row_at[i] = i * W * 8 < BM ? (uint32_t)token_row(row) * (uint32_t)P.a_stride : (uint32_t)channel_row(row - BM) * (uint32_t)P.b_stride;
  }
  auto fetch = [&](int i, int k0, uint8_t* to) {
    k0 = min(k0, k_last);
    const uint32_t k = (uint32_t)min(16 * piece, K - 16 - k0);
    const __amdgpu_buffer_rsrc_t from = i * W * 8 < BM ? tokens : SWIGLU && (((i * W + wave) * 8 - BM) & 16) ? ups : channels;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)(to + (i * W + wave) * 1024), 16,
                                             (int)(row_at[i] + k), k0, 0, 0);
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) fetch(i, k_begin + 128 * s, memory + s * (ROWS * 128));
  // scales: SCALES rows a thread, 64 W apart; 16 blocks from byte k0 of a row's codes on (whole pairs of steps), and what
  // is behind the last pair
  const int k_pairs = k_begin + (K - k_begin) / 256 * 256;
  struct Scales { v4i row[SCALES]; };
  const uint8_t* scales[SCALES];
  Scales rest;
#pragma unroll
  for (int i = 0; i < SCALES; ++i) {
    const int row = min((int)threadIdx.x + 64 * W * i, ROWS - 1), rb = row - BM;
    scales[i] = row < BM ? P.sfa + (m0 + token_row(row)) * P.sfa_stride
                         : P.sfb + (n0 + channel_row(rb) + (SWIGLU && (rb & 16) ? n_out : 0)) * P.sfb_stride;
    rest.row[i] = v4i{0, 0, 0, 0};
    if (k_pairs < K)
#pragma unroll
      for (int d = 0; d < 4; ++d) rest.row[i][d] = load_scales<4>(scales[i], k_pairs / 16 + 4 * d, K / 16);
  }
  auto fetch_scales = [&](int k0) {
    Scales s;
#pragma unroll
    for (int i = 0; i < SCALES; ++i) __builtin_memcpy(&s.row[i], scales[i] + k0 / 16, 16);
    return s;
  };
  // (in LDS a row's dword g holds blocks 2 g and 2 g + 1 of the first step, then of the second: group g's, one byte for
  // each of four instructions)
  auto keep_scales = [&](const Scales& s, int set) {
#pragma unroll
    for (int i = 0; i < SCALES; ++i) {
      const int row = threadIdx.x + 64 * W * i;
      v4i v;
#pragma unroll
      for (int g = 0; g < 4; ++g)
        v[g] = (int)__builtin_amdgcn_perm((uint32_t)s.row[i][2 + g / 2], (uint32_t)s.row[i][g / 2], g & 1 ? 0x07060302u : 0x05040100u);
      if (row < ROWS) *reinterpret_cast<v4i*>(lds_scales + set * (ROWS * 16) + row * 16) = v;
    }
  };
  v4f acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m) acc[n][m] = v4f{0.f, 0.f, 0.f, 0.f};
  const int r = lane & 15, g = lane >> 4, wm = wave % WM, wn = wave / WM;
  const int row_a = wm * (BM / WM) + r, row_b = BM + wn * (BN / WN) + r;
  int as[TM], bs[TN];
  auto read_scales = [&](const uint8_t* sc) {
#pragma unroll
    for (int n = 0; n < TN; ++n) bs[n] = *reinterpret_cast<const int*>(sc + (row_b + 16 * n) * 16 + 4 * g);
#pragma unroll
    for (int m = 0; m < TM; ++m) as[m] = *reinterpret_cast<const int*>(sc + (row_a + 16 * m) * 16 + 4 * g);
  };
  // Step S of a pair, and the requests of a later one: for each token fragment the products with all channel
  // fragments, while the next fragments are read from LDS and a request goes out. In this order and no other (the
  // compiler reads everything first, and spills).
  auto multiply = [&](auto S, const uint8_t* from, int k_next, uint8_t* to) {
    auto read = [&](int row, int j) {
      return *reinterpret_cast<const v4i*>(from + row * 128 + ((4 * j + g) ^ ((r >> 1) & 7)) * 16);
    };
    v4i av[2 * TM], bv[2][TN];           // (a fragment is read AHEAD fragments before its use)
    constexpr int AHEAD = 2;
#pragma unroll
    for (int n = 0; n < TN; ++n) bv[0][n] = read(row_b + 16 * n, 0);
#pragma unroll
    for (int m = 0; m < AHEAD; ++m) av[m] = read(row_a + 16 * (m % TM), m / TM);
    static_for<2 * TM>([&](auto f) {
      constexpr int j = f.value / TM, m = f.value % TM, ahead = f.value + AHEAD;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (ahead < 2 * TM) av[ahead] = read(row_a + 16 * (ahead % TM), ahead / TM);
      if constexpr (j == 0) {
#pragma unroll
        for (int n = 0; n < TN; ++n)
          if (n * TM / TN == m) bv[1][n] = read(row_b + 16 * n, 1);
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        if (i * 2 * TM / LOADS == f.value) fetch(i, k_next, to);
#pragma unroll
      for (int n = 0; n < TN; ++n) acc[n][m] = mfma_fp4<2 * S.value + j>(bv[j][n], av[f.value], acc[n][m], bs[n], as[m]);
      // (no instruction: the products stay before the next fragment's reads and the next barrier)
#pragma unroll
      for (int n = 0; n < TN; ++n) asm volatile("" : "+v"(acc[n][m]));
    });
    __builtin_amdgcn_sched_barrier(0);
  };
  keep_scales(k_pairs > k_begin ? fetch_scales(k_begin) : rest, 0);
  // A step: this wave's loads of it have landed (those of the STAGES - 2 steps behind it may be under way)
  // and its LDS accesses of the step before are done; behind the barrier that holds for every wave, so
  // the step can be read and the buffer of the step before filled again. Scales are requested in the first of a pair of
  // steps, before its codes, and kept in LDS in the second.
  auto ready = [&] { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * LOADS) : "memory"); };
  int turn = 0, set = 0;
  auto step = [&](auto S, int k0) {
    multiply(S, memory + turn * (ROWS * 128), k0 + 128 * (STAGES - 1), memory + (turn == 0 ? STAGES - 1 : turn - 1) * (ROWS * 128));
    turn = turn + 1 == STAGES ? 0 : turn + 1;
  };
  constexpr std::integral_constant<int, 0> first{};
  constexpr std::integral_constant<int, 1> second{};
  int k0 = k_begin;
  for (; k0 < k_pairs; k0 += 256) {
    ready();
    Scales next = fetch_scales(min(k0 + 256, k_pairs - 256));
    read_scales(lds_scales + set * (ROWS * 16));
    step(first, k0);
    ready();
    step(second, k0 + 128);
    set ^= 1;
    if (k0 + 256 == k_pairs) next = rest;
    keep_scales(next, set);
  }
  if (k0 < K) {
    ready();
    read_scales(lds_scales + set * (ROWS * 16));
    step(first, k0);
    if (k0 + 128 < K) {
      ready();
      step(second, k0 + 128);
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // (what was requested behind the last step)
  // Results through LDS, 32 tokens of a wave at a time: from the lanes' four channels of 32 tokens to 16-byte
  // pieces of whole token rows. Rows are padded by 16 bytes, so that neither side meets bank conflicts.
  constexpr int H = SWIGLU ? 2 : 1, CW = 16 * TN / H, PITCH = CW + 4;
  // (SwiGLU: the wave's fragments of 16 channels are gate and up rows in turn)
  auto frag = [](int n, int h) { return SWIGLU ? 2 * n + h : n; };
  static_assert(W * 32 * PITCH * 4 <= (int)sizeof(memory), "the waves' parts fit");
  __syncthreads();
  float* part = reinterpret_cast<float*>(memory) + wave * 32 * PITCH;
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

// The splits' sums added in their order, then as the tiles' epilogue: a thread takes four channels of a token. A second
// launch (3 to 4 us): a counter that lets the last workgroup join would have to be zero between calls, and two captured
// graphs would share it.
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

// Parts of K, channels of a workgroup and blocks of a lane's step of the rows kernel (us, neighbour first).
// Two parts: half the rows a workgroup, twice the workgroups. Where 16 channels each leave CUs without one, or up to 2
// tokens (whose rows cost nothing): 1 x 1024, K 8192 4.9 -> 3.7; 8 x 512, K 4096 4.1 -> 3.5; 1 x 14336, K 4096
// 8.3 -> 7.4; but 4 x 7168, K 7168 8.5 -> 8.9; SwiGLU 1 x 8192, K 4096 6.0 -> 6.2.
// SwiGLU with gate and up rows in one fragment: up to 8 tokens, or where it is needed to fill the CUs: 1 x 4096, K 7168
// 7.9 -> 5.6; 16 x 4096, K 7168 9.8 -> 7.5; but 16 x 8192, K 4096 7.2 -> 8.0 (token rows are read twice as often).
// Four blocks a lane, so that more loads are in flight: 4 x 4096, K 4096 4.3 -> 4.0; 16 x 1024, K 8192 7.4 -> 6.6; but
// where they leave a wave without a step 64 x 2880, K 2880 5.5 -> 7.0. More than 32 tokens under SwiGLU with two
// fragments have no form of four: by the estimates below tiles are ahead of it at every size.
struct Rows { int parts, channels, blocks; };
Rows rows_form(int64_t m, int64_t n, int64_t k, bool swiglu) {
  const int parts = k >= 2048 && m <= 8 && (n <= 2048 || (m <= 2 && !swiglu)) ? 2 : 1;
  const bool one = swiglu && (parts == 2 || m <= 8 || n <= 4096);
  const bool four = (k % 512 == 0 || k >= 4096) && !(m > 32 && swiglu && !one);
  return {parts, 16 / parts / (one ? 2 : 1), four ? 4 : 2};
}

// Threads of a tile's workgroup.
constexpr int TILE_THREADS = 512;

// A launch, or with `told` not the launch but what it would be (dgm_mxfp4_gemm_form).
struct Launch {
  int vec;
  hipStream_t stream;
  int64_t* told;
};

template <int MT, int KP, int CH, int J, bool SWIGLU>
void launch_rows(const DgmMxfp4GemmArgs& A, const Launch& L) {
  const int64_t n_out = SWIGLU ? A.n / 2 : A.n, tokens = 16 / KP * MT;
  const dim3 grid((unsigned)((n_out + CH - 1) / CH), (unsigned)((A.m + tokens - 1) / tokens));
  if (L.told) {
    const int64_t form[7] = {tokens, CH, 0, 1, KP, J, (int64_t)grid.x * 512};
    std::copy(form, form + 7, L.told);
    return;
  }
  hipLaunchKernelGGL((k_mxfp4_gemm_rows<MT, KP, CH, J, SWIGLU>), grid, dim3(512), 0, L.stream, A, L.vec);
}
template <int MT, int J>
void launch_rows(const DgmMxfp4GemmArgs& A, const Rows& f, const Launch& L) {
  if constexpr (MT == 1)
    if (f.parts == 2) return A.swiglu ? launch_rows<1, 2, 4, J, true>(A, L) : launch_rows<1, 2, 8, J, false>(A, L);
  if (!A.swiglu) launch_rows<MT, 1, 16, J, false>(A, L);
  else if (f.channels == 8) launch_rows<MT, 1, 8, J, true>(A, L);
  else if constexpr (MT < 4 || J < 4) launch_rows<MT, 1, 16, J, true>(A, L);
}
template <int MT>
void launch_rows(const DgmMxfp4GemmArgs& A, const Launch& L) {
  const Rows f = rows_form(A.m, A.n, A.k, A.swiglu != 0);
  if (f.blocks == 4) launch_rows<MT, 4>(A, f, L);
  else launch_rows<MT, 2>(A, f, L);
}

template <int BM, int BN, int WM, int WN, int STAGES>
void launch_tiles(const DgmMxfp4GemmArgs& A, int splits, const Launch& L) {
  static_assert(64 * WM * WN == TILE_THREADS, "as choose counts them");
  const int vec = L.vec;
  const hipStream_t stream = L.stream;
  const int tiles_m = (int)((A.m + BM - 1) / BM), tiles_n = (int)((A.n + BN - 1) / BN), steps = (int)((A.k + 255) / 256);
  const int per = (steps + splits - 1) / splits;
  splits = (steps + per - 1) / per;                // (every split has a step)
  const dim3 grid((unsigned)((tiles_m * tiles_n + 7) / 8 * 8), (unsigned)splits), block(64 * WM * WN);
  if (L.told) {
    const int64_t form[7] = {BM, BN, STAGES, splits, 1, 1, (int64_t)grid.x * block.x};
    std::copy(form, form + 7, L.told);
    return;
  }
  if constexpr (BN / WN % 32 == 0)                 // (a wave's gate and up fragments)
    if (A.swiglu) hipLaunchKernelGGL((k_mxfp4_gemm_tiles<BM, BN, WM, WN, STAGES, true>), grid, block, 0, stream, A, vec, tiles_m, tiles_n, per);
  if (!A.swiglu) hipLaunchKernelGGL((k_mxfp4_gemm_tiles<BM, BN, WM, WN, STAGES, false>), grid, block, 0, stream, A, vec, tiles_m, tiles_n, per);
  if (splits == 1) return;
  const int64_t quads = ((A.swiglu ? A.n / 2 : A.n) + 3) / 4 * A.m;
  const dim3 join((unsigned)((quads + 255) / 256));
  if (A.swiglu) hipLaunchKernelGGL(k_mxfp4_gemm_join<true>, join, dim3(256), 0, stream, A, vec, splits);
  else hipLaunchKernelGGL(k_mxfp4_gemm_join<false>, join, dim3(256), 0, stream, A, vec, splits);
}

// Which kernel takes a product, from estimates of its time in us (256 CUs). A tile form takes `around` us and, for each
// step of 256 of K, `alone` us while every workgroup has a CU to itself; when the CUs hold as many as fit, each round
// of them takes `full` us a step and `out` us for its results. Splitting K costs a second launch and the sums' way
// through memory. The times were fitted to 93 products of 1 to 8192 tokens before 64 x 64 took eight waves and launches
// went into a graph: they rank the forms, and are off by up to a third themselves (1000 x 5120, K 2880: 12.6, takes 17.5).
// Over 102 products the choice takes 1.3 % longer than the best form on average; 17 to 128 tokens 3.9 %, where rows, one
// range of 64 x 64 and several are close: 48 x 512, K 2880 64 x 64, 6.5 (rows 4.8); 64 x 4096, K 7168 four ranges, 11.6
// (one 10.6).
// Where each form is taken and the best (us; next best):
//   64 x 64:              64 x 8192, K 4096: 8.1 (64 x 128 9.6);     128 x 4096, K 2880: 7.2 (64 x 128 8.3)
//   64 x 128, 3 stages:   200 x 5120, K 2880: 9.2 (128 x 128 11.5);  777 x 1234, K 2880: 10.0 (64 x 64 12.1)
//   128 x 128, 4 stages:  512 x 7168, K 7168: 20.3 (64 x 128 24.7);  777 x 2880, K 4096: 12.8 (15.2 with 2 stages)
//   128 x 128, 2 stages:  1234 x 2880, K 800: 7.6 (7.8 with 4);      2048 x 2048, K 1024, SwiGLU: 7.0 (7.3 with 4)
//   256 x 128:            2048 x 4096, K 4096: 23.8 (128 x 128 26.2); 777 x 8192, K 8192: 39.4 (128 x 128 40.6)
//   192 x 128:            777 x 5120, K 7168: 27.2 (256 x 128 29.3); 1536 x 4096, K 2880: 18.2 (256 x 128 19.0)
//   192 x 256:            3000 x 2880, K 2880: 23.9 (256 x 256 26.5); 1536 x 7168, K 2048: 18.4 (256 x 256 20.8)
//   256 x 256:            8192 x 8192, K 4096: 159 (192 x 256 172);  4096 x 4096, K 8192: 66 (256 x 128 79)
// The rows form takes 2.4 us and the longer of a wave's steps (a time for each 4096 of a part of K) and the weights at
// the rate at which that many tokens can be multiplied with them (SwiGLU with a fragment each for gate and up rows:
// 1.75 times the former, 1.35 times the rate).
struct Form { int kind, splits; };
enum { ROWS = 0, T64, T64_128, T128_DEEP, T128, T256_128, T192_128, T192_256, T256 };
Form choose(int64_t m, int64_t n, int64_t k, bool swiglu, int64_t workspace_bytes) {
  static const struct { int bm, bn, per_cu; double around, alone, full, out; } tiles[] = {
      {0, 0, 0, 0, 0, 0, 0},                {64, 64, 2, 4.6, 0.24, 0.48, 1.0},
      {64, 128, 2, 4.3, 0.32, 0.75, 1.4},  {128, 128, 1, 4.8, 0.46, 0.68, 1.8}, {128, 128, 2, 4.2, 0.6, 1.14, 2.0},
      {256, 128, 1, 5.4, 0.77, 1.18, 1.4}, {192, 128, 1, 5.0, 0.63, 0.87, 1.5}, {192, 256, 1, 5.8, 1.11, 1.47, 1.6}, {256, 256, 1, 6.4, 1.36, 2.24, 0}};
  const int64_t steps = (k + 255) / 256;
  Form best = {ROWS, 1};
  double least = 1e30;
  if (m <= 64) {
    const Rows f = rows_form(m, n, k, swiglu);
    const bool two = swiglu && f.channels == 16 / f.parts;
    const double wave = (m <= 4 ? 1.5 : m <= 8 ? 1.7 : m <= 16 ? 2.1 : m <= 32 ? 3.5 : 6.0) * (two ? 1.75 : 1.0);
    const double rate = (m <= 4 ? 4.5 : m <= 8 ? 4.0 : m <= 16 ? 3.0 : m <= 32 ? 1.95 : 1.1) * (two ? 1.35 : 1.0);      // TB/s
    const double steps_us = (double)((k + 1024 * f.blocks * f.parts - 1) / (1024 * f.blocks * f.parts)) * wave * f.blocks / 4;
    const double weights_us = (double)n * (double)k * 17 / 32 * 1e-6 / rate;
    least = 2.4 + (steps_us > weights_us ? steps_us : weights_us);
  }
  for (int t = swiglu ? T64_128 : T64; t <= T256; ++t)           // (64 x 64: a wave has 16 channels, so no gate and up rows)
    for (int s = 1; s <= 8; s *= 2) {
      if (s > 1 && (steps < 2 * s || (int64_t)s * m * n * 4 > workspace_bytes)) break;
      const int64_t grid = ((m + tiles[t].bm - 1) / tiles[t].bm) * ((n + tiles[t].bn - 1) / tiles[t].bn), wgs = grid * s;
      // (a launch has fewer than 2^32 threads, and its tiles are rounded up to eights; only 64 x 64 tiles come that far
      // within the call's limit: 128 channels a tile need at most two thirds as many, or one column of 2^18)
      if ((grid + 7) / 8 * 8 * TILE_THREADS >= (int64_t)1 << 32) break;
      const int64_t rounds = (wgs + 256 * tiles[t].per_cu - 1) / (256 * tiles[t].per_cu), each = (steps + s - 1) / s;
      double us = tiles[t].around + (wgs <= 256 ? (double)each * tiles[t].alone : (double)rounds * ((double)each * tiles[t].full + tiles[t].out));
      if (s > 1) us += 3.4 + 0.1 * s + 1.06e-6 * (double)s * (double)m * (double)n;
      if (us < least) least = us, best = {t, s};
    }
  return best;
}
// Sums of a split call above this are not worth their way through memory.
constexpr int64_t MOST_WORKSPACE = 64 << 20;

void launch(const DgmMxfp4GemmArgs& A, const Form& f, const Launch& L) {
  if (f.kind == T64) launch_tiles<64, 64, 2, 4, 4>(A, f.splits, L);
  else if (f.kind == T64_128) launch_tiles<64, 128, 2, 4, 3>(A, f.splits, L);
  else if (f.kind == T128_DEEP) launch_tiles<128, 128, 2, 4, 4>(A, f.splits, L);
  else if (f.kind == T128) launch_tiles<128, 128, 2, 4, 2>(A, f.splits, L);
  else if (f.kind == T256_128) launch_tiles<256, 128, 4, 2, 3>(A, f.splits, L);
  else if (f.kind == T192_128) launch_tiles<192, 128, 2, 4, 3>(A, f.splits, L);
  else if (f.kind == T192_256) launch_tiles<192, 256, 2, 4, 2>(A, f.splits, L);
  else if (f.kind == T256) launch_tiles<256, 256, 2, 4, 2>(A, f.splits, L);
  else if (A.m <= 16) launch_rows<1>(A, L);
  else if (A.m <= 32) launch_rows<2>(A, L);
  else launch_rows<4>(A, L);
}

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

int dgm_mxfp4_gemm_form(int64_t m, int64_t n, int64_t k, int swiglu, int64_t workspace_bytes, int64_t* form) {
  DGM_CHECK_ARG(form, "null pointer");
  DGM_CHECK_ARG(m > 0 && m < (1 << 24) && n > 0 && n < (1 << 24) && k > 0 && k < (1 << 24) && k % 32 == 0 && (!swiglu || n % 2 == 0),
                "sizes of a product");
  DGM_CHECK_ARG(((m + 63) / 64) * ((n + 63) / 64) < (1 << 23), "m n / 4096 below 2^23");
  DgmMxfp4GemmArgs A = {};
  A.m = m, A.n = n, A.k = k, A.swiglu = swiglu;
  launch(A, choose(m, n, k, swiglu != 0, std::min(workspace_bytes, MOST_WORKSPACE)), {0, nullptr, form});
  return 0;
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
  // (256 rows of a tile lie within 31-bit offsets)
  DGM_CHECK_ARG(A.a_stride < (1 << 23) && A.b_stride < (1 << 23), "code rows less than 2^23 bytes apart");
  if (A.m == 0 || A.n == 0) return 0;
  DGM_CHECK_ARG(A.a && A.b && A.sfa && A.sfb && A.d, "null pointer");
  // (choose leaves out tiles whose launch would have 2^32 threads)
  DGM_CHECK_ARG(((A.m + 63) / 64) * ((A.n + 63) / 64) < (1 << 23), "m n / 4096 below 2^23");
  const int e = A.dtype == DGM_SRC_F32 ? 4 : 2;
  // 16-byte stores (and loads of C), which need 4-byte alignment (777 x 1234, K 2880: 11.1 us, single elements 12.3). Past
  // the caches, without regard to size, results are no faster: 8192 x 8192, K 4096 (134 MB) 160 -> 164 us, K 1024 64 -> 75;
  // 8192 x 4096, K 4096 76 -> 79; 16384 x 8192, K 4096 317 -> 307.
  const int vec = (((uintptr_t)A.d | (uintptr_t)A.c | (uint64_t)(A.d_stride * e) | (uint64_t)(A.c_stride * e)) & 3) == 0;
  const int64_t held = A.workspace && ((uintptr_t)A.workspace & 15) == 0 ? A.workspace_bytes : 0;
  const Form f = choose(A.m, A.n, A.k, A.swiglu != 0, held < MOST_WORKSPACE ? held : MOST_WORKSPACE);
  launch(A, f, {vec, stream, nullptr});
  return dgm_last_launch_status();
}

}  // extern "C"
