// The router's balance loss, its per-expert counts and the gradient of the logits (gfx950).
//
// Sequence b holds tokens [cu[b], cu[b+1]) (without cu: one sequence of all tokens). A token with a slot in
// [0, E) is routed; n_b routed tokens, c_be their slots of expert e, S_b = sum_e c_be, f_be = E c_be / S_b,
// p = softmax(l) or sigmoid(l) / sum sigmoid(l), B' sequences with n_b > 0, N = sum n_b:
//   loss = alpha / B' sum_b sum_e f_be mean_t p_te + beta / N sum_t lse_t^2
//   dl_te = alpha / (B' n_b) p_te (f_be - sum_j f_bj p_tj) (sigmoid: times 1 - sigmoid(l_te)) + 2 beta / N lse_t p_te
// An expert masked with -inf has p = 0; a row of nothing else adds to the counts alone.
//
// Sixteen lanes take a token, in 16-byte pieces of its row (a whole wave per token spent most of its time on
// the reductions and the scalar work of a token: 65536 x 256 bf16 76 us for loss and gradient, now 50); all
// passes read the logits once, so the bound is HBM. Sums over tokens: a workgroup's waves add their tokens of
// one sequence in registers and leave one row of sums per (chunk, sequence) at slot chunk + sequence (a walk
// that takes one step per slot, so slots are distinct), which k_balance_columns adds up in a fixed order: no
// atomics on floats, no cleared memory.
#include "dgm_common.hpp"
#include "dgm_abi_internal.hpp"
#include "dgm_rows.hpp"

using namespace dgm;

namespace {

// Waves of a workgroup over tokens: 16 while a lane's values fit the registers that this leaves (128).
__host__ __device__ constexpr int waves_for(int values) { return values <= 24 ? 16 : 8; }

// Row of the workspace: per slot E floats of p sums, E counts; then per slot lse^2 sum and n.
struct Slots {
  float* p;
  int* c;
  float* z;
  int* n;
  double* part;        // per (sequence, 64 experts): sum c P
  int* part_c;         // sum c
  int64_t bytes;
};
__host__ __device__ inline int64_t up16(int64_t x) { return (x + 15) & ~(int64_t)15; }
__host__ __device__ inline Slots slots_of(void* ws, int64_t slots, int seqs, int E) {
  char* b = (char*)ws;
  const int64_t blocks = (int64_t)seqs * ((E + 63) / 64);
  Slots s;
  int64_t at = 0;
  s.part = (double*)(b + at);
  at += up16(blocks * 8);
  s.part_c = (int*)(b + at);
  at += up16(blocks * 4);
  s.p = (float*)(b + at);
  at += up16(slots * E * 4);
  s.c = (int*)(b + at);
  at += up16(slots * E * 4);
  s.z = (float*)(b + at);
  at += up16(slots * 4);
  s.n = (int*)(b + at);
  at += up16(slots * 4);
  s.bytes = at;
  return s;
}

// Tokens of a chunk: whole rounds of a workgroup's waves (64 tokens), up to 512 chunks.
__host__ __device__ inline int64_t chunk_tokens(int64_t tokens) {
  const int64_t c = (tokens + 64 * 512 - 1) / (64 * 512) * 64;
  return c < 64 ? 64 : c;
}

DGM_DEV int64_t seq_begin(const DgmBalanceArgs& P, int b) {
  if (!P.cu_seqlens) return b == 0 ? 0 : P.tokens;
  const int64_t v = P.cu_seqlens[b];
  return v < 0 ? 0 : v > P.tokens ? P.tokens : v;
}
// The first sequence that ends behind token t (seqs if none), by a whole wave: 64 ends are looked at a step.
DGM_DEV int seq_of(const DgmBalanceArgs& P, int64_t t) {
  if (!P.cu_seqlens) return t < P.tokens ? 0 : P.seqs;
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = P.seqs;
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const uint64_t behind = __ballot(at < hi && seq_begin(P, at + 1) > t);
    const int probes = (hi - lo + step - 1) / step, first = behind ? __builtin_ctzll(behind) : probes;
    if (behind) hi = lo + first * step;
    if (first > 0) lo += (first - 1) * step + 1;
  }
  return lo;
}

// The slot's expert of lane `lane` (< topk), or -1.
DGM_DEV int slot_expert(const DgmBalanceArgs& P, int64_t t, int k) {
  const int64_t at = t * P.idx_stride + k;
  const int64_t e = P.idx_i64 ? reinterpret_cast<const int64_t*>(P.topk_idx)[at]
                              : (int64_t)reinterpret_cast<const int32_t*>(P.topk_idx)[at];
  return e >= 0 && e < P.experts ? (int)e : -1;
}
// What sixteen lanes read of a token: its logits (-inf behind the last expert) and its slots; `hit` is the
// lane's (of the first 16). VEC: rows of whole, aligned 16-byte pieces.
template <int T, int NV, bool VEC>
struct Token {
  static constexpr int V = T == T_F32 ? 4 : 8;             // experts of a piece
  float l[NV];
  int hit;
  static DGM_DEV int expert(int i) { return (i / V) * 16 * V + (int)(threadIdx.x & 15) * V + i % V; }
  DGM_DEV void load(const DgmBalanceArgs& P, int64_t t) {
    const int sub = threadIdx.x & 15;
    hit = sub < P.topk ? slot_expert(P, t, sub) : -1;
    const int64_t row = t * P.logits_stride;
#pragma unroll
    for (int c = 0; c < NV; c += V) {
      if constexpr (VEC) {
        if (expert(c) < P.experts) {
          if constexpr (T == T_F32) {
            const f4 v = *reinterpret_cast<const f4*>(reinterpret_cast<const float*>(P.logits) + row + expert(c));
#pragma unroll
            for (int i = 0; i < 4; ++i) l[c + i] = v[i];
          } else {
            load8<T>(P.logits, row + expert(c), l + c);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) l[c + i] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) l[c + i] = expert(c + i) < P.experts ? load1<T>(P.logits, row + expert(c + i)) : -INFINITY;
      }
    }
  }
  DGM_DEV bool routed(const DgmBalanceArgs& P, int64_t t) const {
    bool any = hit >= 0;
    for (int k = (threadIdx.x & 15) + 16; k < P.topk; k += 16) any |= slot_expert(P, t, k) >= 0;
    return ((__ballot(any) >> (threadIdx.x & 48)) & 0xffffu) != 0;
  }
};

DGM_DEV float sum_lanes16(float v) {
  v += dpp_f32<0xB1>(v);        // quad_perm [1,0,3,2]
  v += dpp_f32<0x4E>(v);        // quad_perm [2,3,0,1]
  v += dpp_f32<0x141>(v);       // row_half_mirror
  return v + dpp_f32<0x140>(v); // row_mirror
}
// over the four groups of sixteen lanes
DGM_DEV float sum_groups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// e^x by the hardware's exp2: within (2 + |x|) 2^-24 of the value, so a probability's error stays that of its
// rounded fp32 exponent (a third of the instructions of expf).
DGM_DEV float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

template <int NV>
DGM_DEV float highest(const float* l) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) m = fmaxf(m, l[i]);
  return max_lanes16(m);
}
DGM_DEV float inverse(float s) { return s != 0.f ? 1.0f / s : 0.f; }

// A token's softmax and its log-sum-exp (0 where nothing is left). A sum of zero (all masked) gives zeros.
template <int NV>
DGM_DEV void softmax(const float* l, float* p, float& lse) {
  float s = 0.f;
  const float m = highest<NV>(l), shift = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    p[i] = exp_fast(l[i] - shift);
    s += p[i];
  }
  s = sum_lanes16(s);
  lse = s != 0.f ? m + logf(s) : 0.f;
  const float inv = inverse(s);
#pragma unroll
  for (int i = 0; i < NV; ++i) p[i] *= inv;
}

// Sigmoid scores of a token, 1 / (1 + e^-l). Below -17 each is e^l to the last bit, and from -88 on out of fp32's range,
// which their shares are not: the scores of a row that lies there are taken times e^-m, as 1 / (0 + e^(m - l)).
// (A constant and a shift for each row: a select for each element and a branch for such rows both cost more.)
struct Sigmoid {
  float one, shift;
  template <int NV>
  DGM_DEV static Sigmoid of(const float* l) {
    const float m = highest<NV>(l);
    const bool low = m < -17.5f && m != -INFINITY;
    return {low ? 0.f : 1.0f, low ? m : 0.f};
  }
  // e^(m - l) (the difference first: m log2 e may be beyond fp32); score: the scaled one
  DGM_DEV float exponential(float l) const { return exp_fast(shift - l); }
  DGM_DEV float score(float e) const { return __builtin_amdgcn_rcpf(one + e); }
  // 1 - score, without a difference, which keeps no bits of it beyond l = 17 (from e = 2^25 on it is 1, and the score
  // may have left the range)
  DGM_DEV float rest(float e, float score) const { return e >= 0x1p25f ? 1.0f : e * score; }
};

// Sums of tokens [lo, hi) by the workgroup's waves, four tokens at a time, into rows of the experts' values
// (and counts in LDS).
template <int T, int NV, bool VEC, bool SOFTMAX, int W>
DGM_DEV void sum_tokens(const DgmBalanceArgs& P, int64_t lo, int64_t hi, float (*wave_p)[16 * NV], int* hist, float* wave_z,
                        int* wave_n) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & 15;
  float acc[NV], z = 0.f;
  int n = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.f;
  // (the next tokens are requested before the current ones are worked on; behind the last one it again)
  auto token = [&](int64_t base) { return base + (lane >> 4) < hi ? base + (lane >> 4) : hi - 1; };
  Token<T, NV, VEC> cur, next;
  const int64_t first = lo + 4 * wave;
  if (first < hi) cur.load(P, token(first));
  for (int64_t base = first; base < hi; base += 4 * W, cur = next) {
    if (base + 4 * W < hi) next.load(P, token(base + 4 * W));
    const int64_t t = token(base);
    const bool live = base + (lane >> 4) < hi, counted = cur.routed(P, t) && live;
    if (live) {
      if (cur.hit >= 0) atomicAdd(&hist[cur.hit], 1);
      for (int k = sub + 16; k < P.topk; k += 16) {
        const int e = slot_expert(P, t, k);
        if (e >= 0) atomicAdd(&hist[e], 1);
      }
    }
    float p[NV], lse = 0.f;
    if constexpr (SOFTMAX) {
      softmax<NV>(cur.l, p, lse);
    } else {
      const Sigmoid f = Sigmoid::of<NV>(cur.l);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) s += p[i] = f.score(f.exponential(cur.l[i]));
      const float inv = inverse(sum_lanes16(s));
#pragma unroll
      for (int i = 0; i < NV; ++i) p[i] *= inv;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] += counted ? p[i] : 0.f;      // (an unrouted row may hold anything)
    z += counted ? lse * lse : 0.f;
    n += counted;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float v = sum_groups(acc[i]);
    if (lane < 16) wave_p[wave][Token<T, NV, VEC>::expert(i)] = v;
  }
  z = sum_groups(z);
  n += __shfl_xor(n, 16);
  n += __shfl_xor(n, 32);
  if (lane == 0) {
    wave_z[wave] = z;
    wave_n[wave] = n;
  }
}

template <int T, int NV, bool VEC, bool SOFTMAX>
__global__ void __launch_bounds__(64 * waves_for(NV)) k_balance_tokens(const DgmBalanceArgs P, int64_t chunk, int64_t slots) {
  constexpr int WAVES = waves_for(NV);
  __shared__ float wave_p[WAVES][16 * NV];
  __shared__ int hist[16 * NV];
  __shared__ float wave_z[WAVES];
  __shared__ int wave_n[WAVES];
  const Slots S = slots_of(P.workspace, slots, P.seqs, P.experts);
  const int64_t c0 = (int64_t)blockIdx.x * chunk, c1 = c0 + chunk < P.tokens ? c0 + chunk : P.tokens;
  for (int b = seq_of(P, c0); b < P.seqs; ++b) {
    int64_t lo = seq_begin(P, b), hi = seq_begin(P, b + 1);
    if (lo >= c1) break;
    lo = lo < c0 ? c0 : lo;
    hi = hi > c1 ? c1 : hi;
    if (lo >= hi) continue;                      // (the whole workgroup)
    for (int e = threadIdx.x; e < 16 * NV; e += 64 * WAVES) hist[e] = 0;
    __syncthreads();
    sum_tokens<T, NV, VEC, SOFTMAX, WAVES>(P, lo, hi, wave_p, hist, wave_z, wave_n);
    __syncthreads();
    const int64_t slot = (int64_t)blockIdx.x + b;
    for (int e = threadIdx.x; e < P.experts; e += 64 * WAVES) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += wave_p[w][e];
      S.p[slot * P.experts + e] = s;
      S.c[slot * P.experts + e] = hist[e];
    }
    if (threadIdx.x == 0) {
      float z = 0.f;
      int n = 0;
      for (int w = 0; w < WAVES; ++w) z += wave_z[w], n += wave_n[w];
      S.z[slot] = z;
      S.n[slot] = n;
    }
    __syncthreads();
  }
}

DGM_DEV double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}
DGM_DEV int wave_sum_i32(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// Sequence blockIdx.x, experts 64 blockIdx.y ..: the slots' rows added up (16 waves, rows in turn).
__global__ void __launch_bounds__(1024) k_balance_columns(const DgmBalanceArgs P, int64_t chunk, int64_t slots) {
  __shared__ double lds_p[16][64];
  __shared__ int lds_c[16][64];
  const Slots S = slots_of(P.workspace, slots, P.seqs, P.experts);
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.y * 64 + lane;
  const int64_t lo = seq_begin(P, b), hi = seq_begin(P, b + 1);
  double p = 0.0, z = 0.0;
  int c = 0, n = 0;
  if (hi > lo) {
    const int64_t first = lo / chunk + b, last = (hi - 1) / chunk + b;
    if (e < P.experts)
#pragma unroll 8
      for (int64_t s = first + wave; s <= last; s += 16) {
        p += (double)S.p[s * P.experts + e];
        c += S.c[s * P.experts + e];
      }
    if (blockIdx.y == 0 && wave == 0) {
      for (int64_t s = first + lane; s <= last; s += 64) z += (double)S.z[s], n += S.n[s];
      z = wave_sum_f64(z);
      n = wave_sum_i32(n);
    }
  }
  lds_p[wave][lane] = p;
  lds_c[wave][lane] = c;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < 16; ++w) p += lds_p[w][lane], c += lds_c[w][lane];
  if (e < P.experts) P.counts[(int64_t)b * P.experts + e] = c;
  const double cp = wave_sum_f64((double)c * p);
  const int cs = wave_sum_i32(c);
  if (lane == 0) {
    S.part[(int64_t)b * gridDim.y + blockIdx.y] = cp;
    S.part_c[(int64_t)b * gridDim.y + blockIdx.y] = cs;
    if (blockIdx.y == 0) {
      P.seq_stats[4 * (int64_t)b + 1] = n;
      P.seq_stats[4 * (int64_t)b + 2] = (int)__float_as_uint((float)z);
    }
  }
}

// The loss from the sequences' parts, and what the backward pass needs of them: totals = (B', N).
// seq_stats[b] = (S_b, n_b, lse^2 sum as fp32 bits, 0).
DGM_DEV void finish_loss(const DgmBalanceArgs& P, double f, double z, int live, int total) {
  P.totals[0] = live;
  P.totals[1] = total;
  const double a = live > 0 ? (double)P.balance_coef * f / (double)live : 0.0;
  // (without a z loss lse^2 may be beyond fp32: a row at its type's lowest value)
  const double b = total > 0 && P.z_coef != 0.f ? (double)P.z_coef * z / (double)total : 0.0;
  *P.loss = (float)(a + b);
}
__global__ void __launch_bounds__(256) k_balance_loss(const DgmBalanceArgs P, int64_t slots) {
  __shared__ double lds[4][2];
  __shared__ int lds_n[4][2];
  const Slots S = slots_of(P.workspace, slots, P.seqs, P.experts);
  const int blocks = (P.experts + 63) / 64;
  double f = 0.0, z = 0.0;
  int live = 0, total = 0;
  for (int b = threadIdx.x; b < P.seqs; b += 256) {
    double cp = 0.0;
    int cs = 0;
    for (int i = 0; i < blocks; ++i) cp += S.part[(int64_t)b * blocks + i], cs += S.part_c[(int64_t)b * blocks + i];
    const int n = P.seq_stats[4 * (int64_t)b + 1];
    P.seq_stats[4 * (int64_t)b] = cs;
    if (n > 0) {
      f += (double)P.experts * cp / ((double)cs * (double)n);
      z += (double)__uint_as_float((uint32_t)P.seq_stats[4 * (int64_t)b + 2]);
      ++live;
      total += n;
    }
  }
  f = wave_sum_f64(f), z = wave_sum_f64(z), live = wave_sum_i32(live), total = wave_sum_i32(total);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) lds[wave][0] = f, lds[wave][1] = z, lds_n[wave][0] = live, lds_n[wave][1] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) f += lds[w][0], z += lds[w][1], live += lds_n[w][0], total += lds_n[w][1];
    finish_loss(P, f, z, live, total);
  }
}

// One sequence of few tokens: all of it by one workgroup, in one launch.
template <int T, int NV, bool VEC, bool SOFTMAX>
__global__ void __launch_bounds__(64 * waves_for(NV)) k_balance_small(const DgmBalanceArgs P) {
  constexpr int W = waves_for(NV);
  __shared__ float wave_p[W][16 * NV];
  __shared__ int hist[16 * NV];
  __shared__ float wave_z[W];
  __shared__ int wave_n[W];
  __shared__ double lds_cp[W];
  __shared__ int lds_c[W];
  for (int e = threadIdx.x; e < 16 * NV; e += 64 * W) hist[e] = 0;
  __syncthreads();
  sum_tokens<T, NV, VEC, SOFTMAX, W>(P, seq_begin(P, 0), seq_begin(P, 1), wave_p, hist, wave_z, wave_n);
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  double cp = 0.0;
  int c = 0;
  for (int e = threadIdx.x; e < P.experts; e += 64 * W) {
    double p = 0.0;
    for (int w = 0; w < W; ++w) p += (double)wave_p[w][e];
    c += hist[e];
    cp += (double)hist[e] * p;
    P.counts[e] = hist[e];
  }
  cp = wave_sum_f64(cp);
  c = wave_sum_i32(c);
  if ((threadIdx.x & 63) == 0) lds_cp[wave] = cp, lds_c[wave] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    double z = 0.0;
    int n = 0;
    cp = 0.0, c = 0;
    for (int w = 0; w < W; ++w) cp += lds_cp[w], c += lds_c[w], z += (double)wave_z[w], n += wave_n[w];
    P.seq_stats[0] = c;
    P.seq_stats[1] = n;
    P.seq_stats[2] = (int)__float_as_uint((float)z);
    finish_loss(P, n > 0 ? (double)P.experts * cp / ((double)c * (double)n) : 0.0, z, n > 0, n);
  }
}

// Gradient of the logits: a wave takes `per` consecutive tokens, four at a time; f of their sequence stays in
// registers.
template <int T, int NV, bool VEC, bool SOFTMAX>
__global__ void __launch_bounds__(256) k_balance_grad(const DgmBalanceArgs P, int64_t per) {
  using Tok = Token<T, NV, VEC>;
  const int lane = threadIdx.x & 63;
  const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * per;
  const int64_t last = first + per < P.tokens ? first + per : P.tokens;
  if (first >= last) return;
  const float g = *P.d_loss;
  const int live = P.totals[0], total = P.totals[1];
  const float zc = SOFTMAX && total > 0 ? 2.0f * P.z_coef / (float)total : 0.f;
  int b = seq_of(P, first) - 1, n = 0;           // (per group of lanes from here on)
  int64_t begin = 0, end = first;                // of the sequence whose f is held
  float f[NV], coef = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) f[i] = 0.f;
  auto token = [&](int64_t base) { return base + (lane >> 4) < last ? base + (lane >> 4) : last - 1; };
  Tok cur, next;
  cur.load(P, token(first));
  for (int64_t base = first; base < last; base += 4, cur = next) {
    if (base + 4 < last) next.load(P, token(base + 4));
    const int64_t t = token(base);
    if (t >= end) {
      do {
        ++b;
        begin = b < P.seqs ? seq_begin(P, b) : P.tokens;
        end = b < P.seqs ? seq_begin(P, b + 1) : P.tokens;
      } while (b < P.seqs && end <= t);
      n = b < P.seqs ? P.seq_stats[4 * (int64_t)b + 1] : 0;
      if (n > 0) {
        const float scale = (float)P.experts / (float)P.seq_stats[4 * (int64_t)b];
        const int* counts = P.counts + (int64_t)b * P.experts;
#pragma unroll
        for (int c = 0; c < NV; c += 4) {
          if constexpr (VEC) {
            v4i v = {0, 0, 0, 0};
            if (Tok::expert(c) < P.experts) v = *reinterpret_cast<const v4i*>(counts + Tok::expert(c));
#pragma unroll
            for (int i = 0; i < 4; ++i) f[c + i] = (float)v[i] * scale;
          } else {
#pragma unroll
            for (int i = c; i < c + 4; ++i) f[i] = Tok::expert(i) < P.experts ? (float)counts[Tok::expert(i)] * scale : 0.f;
          }
        }
        coef = P.balance_coef / ((float)live * (float)n);
      }
    }
    const bool counted = cur.routed(P, t) && n > 0 && t >= begin;
    float p[NV], dot = 0.f;
    if constexpr (SOFTMAX) {
      float lse;
      softmax<NV>(cur.l, p, lse);
#pragma unroll
      for (int i = 0; i < NV; ++i) dot += f[i] * p[i];
      dot = sum_lanes16(dot);
#pragma unroll
      for (int i = 0; i < NV; ++i) p[i] = g * (p[i] * (coef * (f[i] - dot) + zc * lse));
    } else {
      // (p: score times 1 - score, which is all that is left to use of them behind the sums)
      const Sigmoid of = Sigmoid::of<NV>(cur.l);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float e = of.exponential(cur.l[i]), score = of.score(e);
        s += score;
        dot += f[i] * score;
        p[i] = score * of.rest(e, score);
      }
      const float inv = inverse(sum_lanes16(s)), scale = g * (coef * inv);
      dot = sum_lanes16(dot) * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) p[i] *= scale * (f[i] - dot);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) p[i] = counted ? p[i] : 0.f;          // (an unrouted row may hold anything)
    if (base + (lane >> 4) >= last) continue;
    const int64_t row = t * P.d_logits_stride;
#pragma unroll
    for (int c = 0; c < NV; c += Tok::V) {
      if constexpr (VEC) {
        if (Tok::expert(c) < P.experts) {
          if constexpr (T == T_F32)
            *reinterpret_cast<f4*>(reinterpret_cast<float*>(P.d_logits) + row + Tok::expert(c)) = f4{p[c], p[c + 1], p[c + 2], p[c + 3]};
          else
            store8<T>(P.d_logits, row + Tok::expert(c), p + c);
        }
      } else {
#pragma unroll
        for (int i = c; i < c + Tok::V; ++i)
          if (Tok::expert(i) < P.experts) store1<T>(P.d_logits, row + Tok::expert(i), p[i]);
      }
    }
  }
}

int check(const DgmBalanceArgs& A) {
  DGM_CHECK_ARG(A.dtype >= DGM_SRC_BF16 && A.dtype <= DGM_SRC_F32, "dtype 0 bf16, 1 fp16, 2 fp32");
  DGM_CHECK_ARG(A.experts >= 1 && A.experts <= DGM_BALANCE_MAX_EXPERTS, "experts 1 to 1024");
  DGM_CHECK_ARG(A.topk >= 1 && A.topk <= A.experts, "topk 1 to experts");
  DGM_CHECK_ARG(A.tokens >= 0 && A.tokens * A.topk < (int64_t)1 << 31, "tokens x topk below 2^31");
  // (a launch has fewer than 2^32 threads, a sequence 1024 of them)
  DGM_CHECK_ARG(A.seqs >= 1 && A.seqs < (1 << 21) && (A.cu_seqlens || A.seqs == 1), "seqs 1 to 2^21, more than one with cu_seqlens");
  DGM_CHECK_ARG(A.score == 0 || (A.score == 1 && A.z_coef == 0.f), "score 0 softmax, 1 sigmoid (without z_coef)");
  DGM_CHECK_ARG(A.counts && A.seq_stats && A.totals, "null pointer");
  DGM_CHECK_ARG(A.tokens == 0 || (A.logits && A.topk_idx), "null pointer");
  return 0;
}

// Values a lane holds (sixteen lanes a token), alignment and score as compile-time values.
template <class F>
void dispatch(const DgmBalanceArgs& A, F&& f) {
  using std::integral_constant;
  const int e = A.dtype == DGM_SRC_F32 ? 4 : 2;
  const bool vec = A.experts % (16 / e) == 0 &&
                   (((uintptr_t)A.logits | (uintptr_t)A.d_logits | (uintptr_t)A.counts | (uint64_t)(A.logits_stride * e) |
                     (uint64_t)(A.d_logits_stride * e)) & 15) == 0;
  auto score = [&](auto t, auto nv, auto v) {
    if (A.score == 0) f(t, nv, v, std::true_type{});
    else f(t, nv, v, std::false_type{});
  };
  auto align = [&](auto t, auto nv) {
    if (vec) score(t, nv, std::true_type{});
    else score(t, nv, std::false_type{});
  };
  auto experts = [&](auto t) {
    if (A.experts <= 128) align(t, integral_constant<int, 8>{});
    else if (A.experts <= 256) align(t, integral_constant<int, 16>{});
    else if (A.experts <= 384) align(t, integral_constant<int, 24>{});
    else if (A.experts <= 512) align(t, integral_constant<int, 32>{});
    else align(t, integral_constant<int, 64>{});
  };
  if (A.dtype == DGM_SRC_BF16) experts(integral_constant<int, T_BF16>{});
  else if (A.dtype == DGM_SRC_F16) experts(integral_constant<int, T_F16>{});
  else experts(integral_constant<int, T_F32>{});
}

// One sequence up to this many tokens is one workgroup's.
constexpr int64_t SMALL_TOKENS = 256;

}  // namespace

extern "C" {

int dgm_balance_struct_size(size_t* args) {
  DGM_CHECK_ARG(args, "null pointer");
  *args = sizeof(DgmBalanceArgs);
  return 0;
}

int64_t dgm_router_balance_workspace_bytes(int64_t tokens, int seqs, int experts) {
  if (tokens < 0 || seqs < 1 || experts < 1 || (seqs == 1 && tokens <= SMALL_TOKENS)) return 0;
  const int64_t chunk = chunk_tokens(tokens);
  return slots_of(nullptr, (tokens + chunk - 1) / chunk + seqs, seqs, experts).bytes;
}

int dgm_router_balance_loss(const DgmBalanceArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmBalanceArgs A = *args;
  if (int st = check(A)) return st;
  DGM_CHECK_ARG(A.loss, "null loss");
  if (A.seqs == 1 && A.tokens <= SMALL_TOKENS) {
    dispatch(A, [&](auto t, auto nv, auto v, auto softmax) {
      hipLaunchKernelGGL((k_balance_small<t.value, nv.value, v.value, softmax.value>), dim3(1),
                         dim3(64 * waves_for(nv.value)), 0, stream, A);
    });
    return dgm_last_launch_status();
  }
  DGM_CHECK_ARG(A.workspace && ((uintptr_t)A.workspace & 15) == 0 &&
                    A.workspace_bytes >= dgm_router_balance_workspace_bytes(A.tokens, A.seqs, A.experts),
                "workspace of dgm_router_balance_workspace_bytes, 16-byte aligned");
  const int64_t chunk = chunk_tokens(A.tokens), chunks = (A.tokens + chunk - 1) / chunk, slots = chunks + A.seqs;
  if (chunks > 0)
    dispatch(A, [&](auto t, auto nv, auto v, auto softmax) {
      hipLaunchKernelGGL((k_balance_tokens<t.value, nv.value, v.value, softmax.value>), dim3((unsigned)chunks),
                         dim3(64 * waves_for(nv.value)), 0, stream, A, chunk, slots);
    });
  hipLaunchKernelGGL(k_balance_columns, dim3((unsigned)A.seqs, (unsigned)((A.experts + 63) / 64)), dim3(1024), 0, stream, A,
                     chunk, slots);
  hipLaunchKernelGGL(k_balance_loss, dim3(1), dim3(256), 0, stream, A, slots);
  return dgm_last_launch_status();
}

int dgm_router_balance_loss_backward(const DgmBalanceArgs* args, hipStream_t stream) {
  DGM_CHECK_ARG(args, "null arguments");
  const DgmBalanceArgs A = *args;
  if (int st = check(A)) return st;
  if (A.tokens == 0) return 0;
  DGM_CHECK_ARG(A.d_loss && A.d_logits, "null pointer");
  // (consecutive tokens of a wave share their sequence's f: 4096 waves, four tokens each at least)
  const int64_t per = (A.tokens + 16383) / 16384 * 4;
  const int64_t waves = (A.tokens + per - 1) / per;
  dispatch(A, [&](auto t, auto nv, auto v, auto softmax) {
    hipLaunchKernelGGL((k_balance_grad<t.value, nv.value, v.value, softmax.value>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0,
                       stream, A, per);
  });
  return dgm_last_launch_status();
}

}  // extern "C"
