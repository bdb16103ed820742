// The router's balance loss, its per-expert counts and the gradient of the logits (gfx950).
//
// Sequence b holds tokens [cu[b], cu[b+1]) (without cu: one sequence of all tokens). A token with a slot in
// [0, E) is routed; n_b routed tokens, c_be their slots of expert e, S_b = sum_e c_be, f_be = E c_be / S_b,
// p = softmax(l) or sigmoid(l) / sum sigmoid(l), B' sequences with n_b > 0, N = sum n_b:
//   loss = alpha / B' sum_b sum_e f_be mean_t p_te + beta / N sum_t lse_t^2
//   dl_te = alpha / (B' n_b) p_te (f_be - sum_j f_bj p_tj) (sigmoid: times 1 - sigmoid(l_te)) + 2 beta / N lse_t p_te
// An expert masked with -inf has p = 0; a row of nothing else adds to the counts alone.
//
// A wave takes a token, its lanes the experts (up to 16 each); all passes read the logits once, so the bound
// is HBM. Sums over tokens: a workgroup's waves add their tokens of one sequence in registers and leave one
// row of sums per (chunk, sequence) at slot chunk + sequence (a walk that takes one step per slot, so slots
// are distinct), which k_balance_columns adds up in a fixed order: no atomics on floats, no cleared memory.
#include "dgm_common.hpp"
#include "dgm_abi_internal.hpp"
#include "dgm_rows.hpp"

using namespace dgm;

namespace {

constexpr int WAVES = 16;                // of a workgroup over tokens

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

// Tokens of a chunk: about 512 chunks, 16 tokens at least.
__host__ __device__ inline int64_t chunk_tokens(int64_t tokens) {
  const int64_t c = (tokens + 511) / 512;
  return c < 16 ? 16 : c;
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
// What a wave reads of a token: its logits (lane: experts lane + 64 i, -inf behind the last) and whether it
// is routed; `hit` its lane's slot (of the first 64).
template <int T, int NE>
struct Token {
  float l[NE];
  int hit;
  DGM_DEV void load(const DgmBalanceArgs& P, int64_t t, int lane) {
    hit = lane < P.topk ? slot_expert(P, t, lane) : -1;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = lane + 64 * i;
      l[i] = e < P.experts ? load1<T>(P.logits, t * P.logits_stride + e) : -INFINITY;
    }
  }
  DGM_DEV bool routed(const DgmBalanceArgs& P, int64_t t, int lane) const {
    bool any = hit >= 0;
    for (int k = lane + 64; k < P.topk; k += 64) any |= slot_expert(P, t, k) >= 0;
    return __ballot(any) != 0;
  }
};

// e^x by the hardware's exp2: within (2 + |x|) 2^-24 of the value, so a probability's error stays that of its
// rounded fp32 exponent (a third of the instructions of expf, and these passes were bound by them).
DGM_DEV float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// A token's probabilities and its log-sum-exp (softmax; 0 where nothing is left). A sum of zero (all masked)
// gives zeros. sig: sigmoid(l), of the sigmoid form.
template <int NE, bool SOFTMAX>
DGM_DEV void probabilities(const float* l, float* p, float* sig, float& lse) {
  float s = 0.f;
  lse = 0.f;
  if constexpr (SOFTMAX) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i) m = fmaxf(m, l[i]);
    m = wave_max(m);
    const float shift = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      p[i] = exp_fast(l[i] - shift);
      s += p[i];
    }
    s = wave_sum(s);
    if (s != 0.f) lse = m + logf(s);
  } else {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      sig[i] = p[i] = __builtin_amdgcn_rcpf(1.0f + exp_fast(-l[i]));
      s += p[i];
    }
    s = wave_sum(s);
  }
  const float inv = s != 0.f ? 1.0f / s : 0.f;
#pragma unroll
  for (int i = 0; i < NE; ++i) p[i] *= inv;
}

// Sums of tokens [lo, hi) by the workgroup's waves, into rows of E values (and counts in LDS).
template <int T, int NE, bool SOFTMAX, int W>
DGM_DEV void sum_tokens(const DgmBalanceArgs& P, int64_t lo, int64_t hi, float (*wave_p)[64 * NE], int* hist, float* wave_z,
                        int* wave_n) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float acc[NE], z = 0.f;
  int n = 0;
#pragma unroll
  for (int i = 0; i < NE; ++i) acc[i] = 0.f;
  // (the next token is requested before the current one is worked on)
  Token<T, NE> cur, next;
  if (lo + wave < hi) cur.load(P, lo + wave, lane);
  for (int64_t t = lo + wave; t < hi; t += W, cur = next) {
    next.load(P, t + W < hi ? t + W : t, lane);
    if (cur.hit >= 0) atomicAdd(&hist[cur.hit], 1);
    for (int k = lane + 64; k < P.topk; k += 64) {
      const int e = slot_expert(P, t, k);
      if (e >= 0) atomicAdd(&hist[e], 1);
    }
    if (!cur.routed(P, t, lane)) continue;
    float p[NE], sig[NE], lse;
    probabilities<NE, SOFTMAX>(cur.l, p, sig, lse);
#pragma unroll
    for (int i = 0; i < NE; ++i) acc[i] += p[i];
    z += lse * lse;
    ++n;
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) wave_p[wave][lane + 64 * i] = acc[i];
  if (lane == 0) {
    wave_z[wave] = z;
    wave_n[wave] = n;
  }
}

template <int T, int NE, bool SOFTMAX>
__global__ void __launch_bounds__(64 * WAVES) k_balance_tokens(const DgmBalanceArgs P, int64_t chunk, int64_t slots) {
  __shared__ float wave_p[WAVES][64 * NE];
  __shared__ int hist[64 * NE];
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
    for (int e = threadIdx.x; e < 64 * NE; e += 64 * WAVES) hist[e] = 0;
    __syncthreads();
    sum_tokens<T, NE, SOFTMAX, WAVES>(P, lo, hi, wave_p, hist, wave_z, wave_n);
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
  const double b = total > 0 ? (double)P.z_coef * z / (double)total : 0.0;
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

// One sequence of few tokens: all of it by one workgroup of 16 waves, in one launch.
template <int T, int NE, bool SOFTMAX>
__global__ void __launch_bounds__(1024) k_balance_small(const DgmBalanceArgs P) {
  __shared__ float wave_p[16][64 * NE];
  __shared__ int hist[64 * NE];
  __shared__ float wave_z[16];
  __shared__ int wave_n[16];
  __shared__ double lds_cp[16];
  __shared__ int lds_c[16];
  for (int e = threadIdx.x; e < 64 * NE; e += 1024) hist[e] = 0;
  __syncthreads();
  const int64_t lo = seq_begin(P, 0), hi = seq_begin(P, 1);
  sum_tokens<T, NE, SOFTMAX, 16>(P, lo, hi, wave_p, hist, wave_z, wave_n);
  __syncthreads();
  const int e = threadIdx.x, wave = threadIdx.x >> 6;
  double cp = 0.0;
  int c = 0;
  if (e < 64 * NE) {
    double p = 0.0;
    for (int w = 0; w < 16; ++w) p += (double)wave_p[w][e];
    c = hist[e];
    cp = (double)c * p;
    if (e < P.experts) P.counts[e] = c;
  }
  cp = wave_sum_f64(cp);
  c = wave_sum_i32(c);
  if ((e & 63) == 0) lds_cp[wave] = cp, lds_c[wave] = c;
  __syncthreads();
  if (e == 0) {
    double z = 0.0;
    int n = 0;
    cp = 0.0, c = 0;
    for (int w = 0; w < 16; ++w) cp += lds_cp[w], c += lds_c[w], z += (double)wave_z[w], n += wave_n[w];
    P.seq_stats[0] = c;
    P.seq_stats[1] = n;
    P.seq_stats[2] = (int)__float_as_uint((float)z);
    finish_loss(P, n > 0 ? (double)P.experts * cp / ((double)c * (double)n) : 0.0, z, n > 0, n);
  }
}

// Gradient of the logits: a wave takes `per` consecutive tokens; f of their sequence stays in registers.
template <int T, int NE, bool SOFTMAX>
__global__ void __launch_bounds__(256) k_balance_grad(const DgmBalanceArgs P, int64_t per) {
  const int lane = threadIdx.x & 63;
  const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * per;
  const int64_t last = first + per < P.tokens ? first + per : P.tokens;
  if (first >= last) return;
  const float g = *P.d_loss;
  const int live = P.totals[0], total = P.totals[1];
  const float zc = SOFTMAX && total > 0 ? 2.0f * P.z_coef / (float)total : 0.f;
  int b = seq_of(P, first) - 1, n = 0;
  int64_t begin = 0, end = first;          // (of the sequence whose f is held)
  float f[NE], coef = 0.f;
#pragma unroll
  for (int i = 0; i < NE; ++i) f[i] = 0.f;
  Token<T, NE> cur, next;
  cur.load(P, first, lane);
  for (int64_t t = first; t < last; ++t, cur = next) {
    next.load(P, t + 1 < last ? t + 1 : t, lane);
    if (t >= end) {
      do {
        ++b;
        begin = b < P.seqs ? seq_begin(P, b) : P.tokens;
        end = b < P.seqs ? seq_begin(P, b + 1) : P.tokens;
      } while (b < P.seqs && end <= t);
      n = b < P.seqs ? P.seq_stats[4 * (int64_t)b + 1] : 0;
      if (n > 0) {
        const float scale = (float)P.experts / (float)P.seq_stats[4 * (int64_t)b];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
          const int e = lane + 64 * i;
          f[i] = e < P.experts ? (float)P.counts[(int64_t)b * P.experts + e] * scale : 0.f;
        }
        coef = P.balance_coef / ((float)live * (float)n);
      }
    }
    float d[NE];
    if (n > 0 && t >= begin && cur.routed(P, t, lane)) {
      float p[NE], sig[NE], lse, dot = 0.f;
      probabilities<NE, SOFTMAX>(cur.l, p, sig, lse);
#pragma unroll
      for (int i = 0; i < NE; ++i) dot += f[i] * p[i];
      dot = wave_sum(dot);
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        if constexpr (SOFTMAX) d[i] = g * (p[i] * (coef * (f[i] - dot) + zc * lse));
        else d[i] = g * (p[i] * (coef * (f[i] - dot)) * (1.0f - sig[i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < NE; ++i) d[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = lane + 64 * i;
      if (e < P.experts) store1<T>(P.d_logits, t * P.d_logits_stride + e, d[i]);
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

template <class F>
void dispatch(const DgmBalanceArgs& A, F&& f) {
  using std::integral_constant;
  auto score = [&](auto t, auto ne) {
    if (A.score == 0) f(t, ne, std::true_type{});
    else f(t, ne, std::false_type{});
  };
  auto experts = [&](auto t) {
    if (A.experts <= 64) score(t, integral_constant<int, 1>{});
    else if (A.experts <= 128) score(t, integral_constant<int, 2>{});
    else if (A.experts <= 256) score(t, integral_constant<int, 4>{});
    else if (A.experts <= 512) score(t, integral_constant<int, 8>{});
    else score(t, integral_constant<int, 16>{});
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
    dispatch(A, [&](auto t, auto ne, auto softmax) {
      hipLaunchKernelGGL((k_balance_small<t.value, ne.value, softmax.value>), dim3(1), dim3(1024), 0, stream, A);
    });
    return dgm_last_launch_status();
  }
  DGM_CHECK_ARG(A.workspace && ((uintptr_t)A.workspace & 15) == 0 &&
                    A.workspace_bytes >= dgm_router_balance_workspace_bytes(A.tokens, A.seqs, A.experts),
                "workspace of dgm_router_balance_workspace_bytes, 16-byte aligned");
  const int64_t chunk = chunk_tokens(A.tokens), chunks = (A.tokens + chunk - 1) / chunk, slots = chunks + A.seqs;
  if (chunks > 0)
    dispatch(A, [&](auto t, auto ne, auto softmax) {
      hipLaunchKernelGGL((k_balance_tokens<t.value, ne.value, softmax.value>), dim3((unsigned)chunks), dim3(64 * WAVES), 0,
                         stream, A, chunk, slots);
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
  // (consecutive tokens of a wave share their sequence's f: 8192 waves, a token each at least)
  const int64_t per = (A.tokens + 8191) / 8192;
  const int64_t waves = (A.tokens + per - 1) / per;
  dispatch(A, [&](auto t, auto ne, auto softmax) {
    hipLaunchKernelGGL((k_balance_grad<t.value, ne.value, softmax.value>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0,
                       stream, A, per);
  });
  return dgm_last_launch_status();
}

}  // extern "C"
