// The router's losses, counts and weights of a training step, and their
// gradient in the logits.
//
//   softmax: p = softmax(l)                sigmoid: s = sigmoid(l), p = s / sum s
//   sequence q of n tokens: c_e = #{(t, k): ids = e},  P_e = mean_t p_te,
//     L_q = E / (K n) sum_e c_e P_e;  balance = mean of L_q over non-empty ones
//   z = mean over the sequences' tokens of (logsumexp l)^2          (softmax)
//   w_k = f u_k, u the selected p (sigmoid: s), over their sum if renormalised
//
// Forward: one pass over the logits.  A token belongs to L lanes, each with V of
// its experts in registers (L V >= E), a wave takes 64 / L tokens at a time, and
// each lane keeps the sums of its experts over the tokens that it sees, so a
// workgroup writes one row of sums per chunk of tokens and sequence
// (router_stats_kernel).  A second launch adds the rows in their order, in fp64
// (router_finish_kernel): no floating-point atomics, the same bits every time.
// Backward: one pass, logits and the selected experts' gradients in, the logits'
// gradient out (router_grad_kernel); a row's maximum and sum come from the forward.
//
// A row of -inf has p = 0, no z and no gradient; so has one whose sigmoids vanish in 64
// bits.  NaN gives NaN, +inf with softmax too (sigmoid: its score is 1).
#include <cfloat>
#include <type_traits>

#include "xtu_common.hpp"

#include "../../include/xtu_moe_amd.h"

namespace xtu {
namespace rt {
namespace {

constexpr int kMaxE = 1024, kMaxK = 16;
// Forward: 16 waves a workgroup, so that 32 waves a CU write only two rows of sums.
constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr int kMaxChunks = 512;    // workgroups: two a CU, more where
constexpr int kLaneRows = 256;     // a lane would add more rows than this in fp32 (fp64 from there)
constexpr int kOneTurns = 4;       // turns of a workgroup that does without the second launch
constexpr int kOneSeqs = 64;       // and the sequences that it writes
// Second launch: 16 experts a workgroup, 16 partial rows at a time.
constexpr int kCols = 16, kSumThreads = 256;
// Backward: nothing is shared between waves.
constexpr int kGradWaves = 4, kGradThreads = 64 * kGradWaves, kGradChunks = 2048;

struct Rows {
  const void* logits;   // [T][E], rows ld apart
  long ld;
  int bf16, vec;        // vec: rows start on 4 elements, E % 4 == 0
  const int32_t* ids;   // [T][K]
  const int32_t* starts;   // [S + 1], or null: all rows are one sequence
  int T, E, K, S, sigmoid, renorm;
  float scale;
};

constexpr float kLog2e = 1.44269504f;
// A row whose sigmoids are all below 64 bits' normal numbers (e^-708) has no scores to speak
// of, as one of -inf: a mask's lowest value is no score.
constexpr float kNoScore = -708.f;

// e^(l - m) for l <= m.  Near zero as 2^(l log2 e - m log2 e): the rounding of the second
// product is the same for all of a row and leaves its probabilities alone, that of the
// difference would be |l - m| 2^-24.  That common factor leaves fp32's range from |m| of
// 1e9 on, so from 256 on the difference comes first: it is exact wherever e^(l - m) does not
// vanish (l is then within a factor of two of m), and zero for a row wholly at the lowest
// value.  Three instructions each instead of eight with the difference's rounding made good.
__device__ __forceinline__ float exp_from(float l, float m) {
  const float a = fabsf(m) < 256.f ? 0.f : m;
  return __builtin_amdgcn_exp2f(__builtin_fmaf(l - a, kLog2e, (a - m) * kLog2e));
}

// v of the lane across: within quads, halves of a row of 16, rows, and rows by
// row (every lane below that size holds the same value by then).
template <int D>
__device__ __forceinline__ float across(float v) {
  const int x = __float_as_int(v);
  if constexpr (D == 1) return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0xB1, 0xF, 0xF, false));
  if constexpr (D == 2) return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0x4E, 0xF, 0xF, false));
  if constexpr (D == 4) return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0x141, 0xF, 0xF, false));
  return __int_as_float(__builtin_amdgcn_mov_dpp(x, 0x140, 0xF, 0xF, false));   // 8
}

// The op of all of the L lanes of a token, in each of them.  Register moves only: by
// way of LDS (__shfl_xor) the six steps take longer than the rest of a row.
template <int L, class F>
__device__ __forceinline__ float reduce_over(float v, F op) {
  if constexpr (L >= 2) v = op(v, across<1>(v));
  if constexpr (L >= 4) v = op(v, across<2>(v));
  if constexpr (L >= 8) v = op(v, across<4>(v));
  if constexpr (L >= 16) v = op(v, across<8>(v));
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

template <int L>
__device__ __forceinline__ float sum_over(float v) {
  return reduce_over<L>(v, [](float x, float y) { return x + y; });
}

template <int L>
__device__ __forceinline__ float max_over(float v) {
  return reduce_over<L>(v, [](float x, float y) { return fmaxf(x, y); });
}

// The same for two's worth of bits.
template <int D>
__device__ __forceinline__ double across2(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  uint32_t lo = (uint32_t)b, hi = (uint32_t)(b >> 32);
  if constexpr (D == 16) {
    lo = __builtin_amdgcn_ds_swizzle(lo, 0x401F);   // lanes ^ 16
    hi = __builtin_amdgcn_ds_swizzle(hi, 0x401F);
  } else if constexpr (D == 32) {
    const int other = ((int)__lane_id() ^ 32) * 4;
    lo = __builtin_amdgcn_ds_bpermute(other, lo);
    hi = __builtin_amdgcn_ds_bpermute(other, hi);
  } else {
    lo = __float_as_uint(across<D>(__uint_as_float(lo)));
    hi = __float_as_uint(across<D>(__uint_as_float(hi)));
  }
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ double wave_sum(double v) {
  v += across2<1>(v);
  v += across2<2>(v);
  v += across2<4>(v);
  v += across2<8>(v);
  v += across2<16>(v);
  return v + across2<32>(v);
}

// The sums over a block's threads of N values each, in every thread and a fixed order;
// red: not in use.
template <int WAVES, int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double (*red)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = wave_sum(v[n]);
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64][n] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = 0.;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v[n] += red[w][n];
  }
}

__device__ __forceinline__ void lds_order() {
  __builtin_amdgcn_wave_barrier();
  __asm__ __volatile__("" ::: "memory");
}

// A lane's V logits of row t: experts 4 (i + L v) .. + 3; -inf past E.
template <int L, int V>
struct Raw {
  u32x4_t r[V / 4];
};

template <int L, int V>
__device__ __forceinline__ void load_row(const Rows& a, long t, int i, Raw<L, V>& raw) {
  if (a.vec) {
#pragma unroll
    for (int v = 0; v < V / 4; ++v) {
      const int c = 4 * (i + L * v);
      if (c >= a.E) {
        raw.r[v] = a.bf16 ? u32x4_t{0xff80ff80u, 0xff80ff80u, 0u, 0u}
                          : u32x4_t{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
      } else if (a.bf16) {
        const uint2 w = *reinterpret_cast<const uint2*>(
            reinterpret_cast<const uint16_t*>(a.logits) + t * a.ld + c);
        raw.r[v] = u32x4_t{w.x, w.y, 0u, 0u};
      } else {
        raw.r[v] = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const float*>(a.logits) +
                                                     t * a.ld + c);
      }
    }
    return;
  }
#pragma unroll
  for (int v = 0; v < V / 4; ++v) {
    raw.r[v] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 4 * (i + L * v) + e;
      if (a.bf16) {
        const uint32_t x = c < a.E ? reinterpret_cast<const uint16_t*>(a.logits)[t * a.ld + c]
                                   : 0xff80u;
        raw.r[v][e / 2] |= x << (16 * (e % 2));
      } else {
        raw.r[v][e] = c < a.E ? reinterpret_cast<const uint32_t*>(a.logits)[t * a.ld + c]
                              : 0xff800000u;
      }
    }
  }
}

template <int L, int V>
__device__ __forceinline__ void values(const Rows& a, const Raw<L, V>& raw, float (&l)[V]) {
#pragma unroll
  for (int v = 0; v < V / 4; ++v)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.bf16) {
        const uint32_t w = raw.r[v][e / 2];
        l[4 * v + e] = __uint_as_float(e % 2 ? w & 0xffff0000u : w << 16);
      } else {
        l[4 * v + e] = __uint_as_float(raw.r[v][e]);
      }
    }
}

// The score of a logit before its row's sum divides it.  softmax: e^(l - m), m the
// row's maximum.  sigmoid: sigmoid(l) e^-m with m = min(maximum, 0), so that a row
// of very negative logits keeps its ratios (kNoScore); sigmoid(l) = score e^m.  rest: 1 -
// sigmoid(l), without the cancellation.
template <bool SIG>
__device__ __forceinline__ float score(float l, float m, float& rest) {
  if constexpr (!SIG) {
    rest = 1.f;
    return exp_from(l, m);
  }
  const float e = __builtin_amdgcn_exp2f(-fabsf(l) * kLog2e);
  const float r = __builtin_amdgcn_rcpf(1.f + e), er = e * r;
  rest = l >= 0.f ? er : r;
  if (m < 0.f) return exp_from(l, m) * r;   // (every l < 0)
  return l >= 0.f ? r : er;
}

__device__ __forceinline__ int start_of(const Rows& a, int q) {
  return a.starts ? a.starts[q] : q ? a.T : 0;
}

// First sequence whose end lies behind row t (S: none), over ends clamped to T.
__device__ __forceinline__ int seq_of(const Rows& a, int t) {
  int lo = 0, hi = a.S;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (min(start_of(a, mid + 1), a.T) > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Rows [begin, end) of sequence q, inside [0, T].
__device__ __forceinline__ void seq_rows(const Rows& a, int q, int& begin, int& end) {
  begin = min(max(start_of(a, q), 0), a.T);
  end = min(max(start_of(a, q + 1), begin), a.T);
}

// Ids of a row that a lane takes: k = i, i + L, ..; -1: none.
template <int L>
struct Ids {
  static constexpr int N = (kMaxK + L - 1) / L;
  int e[N];
};

template <int L>
__device__ __forceinline__ void load_ids(const Rows& a, long t, int i, Ids<L>& ids) {
#pragma unroll
  for (int n = 0; n < Ids<L>::N; ++n) {
    const int k = i + L * n;
    const int e = k < a.K ? a.ids[t * a.K + k] : -1;
    ids.e[n] = (unsigned)e < (unsigned)a.E ? e : -1;
  }
}

struct Sums {
  float* part_p;       // [chunks + S][E]
  int32_t* part_c;
  float* part_z;       // [chunks + S]
  double* loss;        // [S][ceil(E / 16)]
  double* zsum;        // [S]
  unsigned* ticket;
  int32_t* counts;     // [S][E]
  float* probs;        // [S][E]
  float* balance;
  float* z;
  float* norm;         // [2]: non-empty sequences, their rows
};

__device__ __forceinline__ void write_losses(const Sums& o, double loss, double z, double rows,
                                             double seqs) {
  *o.balance = seqs > 0. ? (float)(loss / seqs) : 0.f;
  if (o.z) *o.z = rows > 0. ? (float)(z / rows) : 0.f;
  o.norm[0] = (float)seqs;
  o.norm[1] = (float)rows;
}

// Chunk g holds rows [g C, (g + 1) C).  Its part of sequence q writes row g + q
// of the partial sums: both grow along the rows, so no two parts share one.  ONE: the
// only chunk, whose sums are the sequences' own, and which writes the losses too.
template <int L, int V, bool SIG, bool ONE>
__global__ __launch_bounds__(kThreads, ONE || V > 8 ? 4 : 8) void router_stats_kernel(Rows a, int C, float* weights,
                                                                float2* stat, Sums o) {
  constexpr int G = 64 / L, NG = kWaves * G, COLS = L * V;
  // a token's scores; then a wave's sums
  __shared__ __attribute__((aligned(16))) float buf[NG][COLS];
  __shared__ int32_t hist[COLS];
  __shared__ float zs[kWaves];
  __shared__ double red[kWaves][4];
  const int tid = threadIdx.x, lane = tid % 64, w = tid / 64;
  const int i = lane % L, g = w * G + lane / L;
  const int c0 = blockIdx.x * C, c1 = min(c0 + C, a.T);
  Raw<L, V> next;
  Ids<L> nid;
  int t = c0 + g;
  if (t < c1) {   // ahead of the sequences' bounds
    load_row(a, t, i, next);
    load_ids(a, t, i, nid);
  }
  if (!ONE && blockIdx.x == 0 && tid == 0) *o.ticket = 0;   // of the next launch
  for (int c = tid; c < COLS; c += kThreads) hist[c] = 0;
  double loss = 0., zsum = 0.;
  if (ONE) {
    for (int k = tid; k < a.S * a.E; k += kThreads) {   // empty sequences stay so
      o.counts[k] = 0;
      o.probs[k] = 0.f;
    }
  }
  int q = seq_of(a, c0);
  int at = c0;   // rows before are done
  while (at < c1) {
    // rows [at, end) are sequence q's, or no one's (q == S, or before its start)
    int end = c1, n = 0;
    bool in = false;
    if (q < a.S) {
      int b, e;
      seq_rows(a, q, b, e);
      n = e - b;
      in = at >= b;
      end = min(c1, in ? e : b);
      if (end <= at) {   // an empty sequence (or starts that do not ascend)
        ++q;
        continue;
      }
    }
    __syncthreads();   // hist is zero, buf free
    float acc[V], z = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.f;
    t = at + g;
    if (at != c0 && t < end) {
      load_row(a, t, i, next);
      load_ids(a, t, i, nid);
    }
    for (int t0 = at; t0 < end; t0 += NG, t += NG) {   // every lane of a wave takes each turn
      const bool on = t < end;
      float l[V];
      values(a, next, l);
      const Ids<L> id = nid;
      if (t + NG < end) {
        load_row(a, t + NG, i, next);
        load_ids(a, t + NG, i, nid);
      }
      float m = l[0];
#pragma unroll
      for (int v = 1; v < V; ++v) m = fmaxf(m, l[v]);
      m = max_over<L>(m);
      if (m < (SIG ? kNoScore : -FLT_MAX)) m = 0.f;   // (the scores are zero then)
      if (SIG) m = fminf(m, 0.f);
      float s = 0.f, rest;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        l[v] = score<SIG>(l[v], m, rest);
        s += l[v];
      }
      lds_order();
#pragma unroll
      for (int v = 0; v < V / 4; ++v)
        *reinterpret_cast<f32x4_t*>(&buf[g][4 * (i + L * v)]) =
            f32x4_t{l[4 * v], l[4 * v + 1], l[4 * v + 2], l[4 * v + 3]};
      lds_order();
      s = sum_over<L>(s);
      const float inv = s == 0.f ? 0.f : 1.f / s;
      // the selected experts: lanes 0 .. K - 1 of the token, L at a time
      float sel[Ids<L>::N], total = 0.f;
#pragma unroll
      for (int n = 0; n < Ids<L>::N; ++n) {
        sel[n] = on && id.e[n] >= 0 ? buf[g][id.e[n]] : 0.f;
        total += sel[n];
      }
      if (a.renorm) total = sum_over<L>(total);
      float f = a.renorm ? (total == 0.f ? 0.f : a.scale / total)
                         : a.scale * (SIG ? __builtin_amdgcn_exp2f(m * kLog2e) : inv);
      if (!SIG && s != s) f = s;   // a probability of such a row is NaN, whoever is selected
      if (!on) continue;
#pragma unroll
      for (int n = 0; n < Ids<L>::N; ++n) {
        const int k = i + L * n;
        if (k < a.K) weights[(long)t * a.K + k] = id.e[n] >= 0 ? sel[n] * f : 0.f;
        if (in && id.e[n] >= 0) atomicAdd(&hist[id.e[n]], 1);
      }
      if (i == 0) stat[t] = make_float2(m, inv);
      if (!in) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = __builtin_fmaf(l[v], inv, acc[v]);
      if (!SIG && i == 0 && s != 0.f) {
        const float lse = m + logf(s);
        z = __builtin_fmaf(lse, lse, z);
      }
    }
    if (in) {
      __syncthreads();   // the scores are read, hist is whole
      // the wave's tokens' sums, then the waves'
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int d = L; d < 64; d *= 2) acc[v] += __shfl_xor(acc[v], d, 64);
      z = sum_over<64>(z);
      if (lane < L)
#pragma unroll
        for (int v = 0; v < V / 4; ++v)
          *reinterpret_cast<f32x4_t*>(&buf[w * G][4 * (i + L * v)]) =
              f32x4_t{acc[4 * v], acc[4 * v + 1], acc[4 * v + 2], acc[4 * v + 3]};
      if (lane == 0) zs[w] = z;
      __syncthreads();
      const long slot = ONE ? q : (long)blockIdx.x + q;
      for (int c = tid; c < a.E; c += kThreads) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) s += buf[k * G][c];
        const int32_t cnt = hist[c];
        hist[c] = 0;
        if (ONE) {
          const double p = (double)s / n;
          o.probs[slot * a.E + c] = (float)p;
          o.counts[slot * a.E + c] = cnt;
          loss += p * cnt * a.E / ((double)a.K * n);
        } else {
          o.part_p[slot * a.E + c] = s;
          o.part_c[slot * a.E + c] = cnt;
        }
      }
      if (tid == 0) {
        float s = 0.f;
        for (int k = 0; k < kWaves; ++k) s += zs[k];
        if (ONE) zsum += s;
        else o.part_z[slot] = s;
      }
    }
    at = end;
  }
  if (ONE) {
    double rows = 0., seqs = 0.;
    for (int k = tid; k < a.S; k += kThreads) {
      int b, e;
      seq_rows(a, k, b, e);
      rows += e - b;
      seqs += e > b;
    }
    double v[4] = {loss, zsum, rows, seqs};
    block_sums<kWaves>(v, red);
    if (tid == 0) write_losses(o, v[0], v[1], v[2], v[3]);
  }
}

// Stores and loads that other XCDs' L2s see without a write-back of this one's.
__device__ __forceinline__ void store_far(double* p, double v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double load_far(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sixteen experts of a sequence per workgroup: thread (r, c) adds every 16th
// partial row of expert c.  The workgroup that ends last adds the losses.
__global__ __launch_bounds__(kSumThreads) void router_finish_kernel(Rows a, int C, Sums o) {
  constexpr int R = kSumThreads / kCols, WAVES = kSumThreads / 64;
  __shared__ double sp[R][kCols];
  __shared__ int32_t sc[R][kCols];
  __shared__ double red1[WAVES][1], red4[WAVES][4];
  __shared__ bool last;
  const int tid = threadIdx.x, nb = (a.E + kCols - 1) / kCols;
  const int q = blockIdx.x / nb, b = blockIdx.x % nb;
  const int col = tid % kCols, e = b * kCols + col, r = tid / kCols;
  int begin, end;
  seq_rows(a, q, begin, end);
  const int n = end - begin;
  const int g0 = begin / C, g1 = n > 0 ? (end - 1) / C + 1 : g0;
  double p = 0., zz[1] = {0.};
  int32_t c = 0;
  if (e < a.E) {
#pragma unroll 8
    for (int g = g0 + r; g < g1; g += R) {
      const long at = ((long)g + q) * a.E + e;
      p += o.part_p[at];
      c += o.part_c[at];
    }
  }
  if (b == 0)
    for (int g = g0 + tid; g < g1; g += kSumThreads) zz[0] += o.part_z[(long)g + q];
  sp[r][col] = p;
  sc[r][col] = c;
  if (b == 0) block_sums<WAVES>(zz, red1);   // (the same for the whole workgroup)
  else __syncthreads();
  if (tid < 64) {
    double loss = 0.;
    if (tid < kCols && e < a.E) {
#pragma unroll
      for (int k = 1; k < R; ++k) {
        p += sp[k][tid];
        c += sc[k][tid];
      }
      p = n > 0 ? p / n : 0.;
      o.probs[(long)q * a.E + e] = (float)p;
      o.counts[(long)q * a.E + e] = c;
      loss = n > 0 ? p * c * a.E / ((double)a.K * n) : 0.;
    }
    loss = wave_sum(loss);
    if (tid == 0) {
      store_far(&o.loss[blockIdx.x], loss);
      if (b == 0) store_far(&o.zsum[q], zz[0]);
      __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");   // they are there before the ticket
      last = __hip_atomic_fetch_add(o.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!last) return;
  double v[4] = {0., 0., 0., 0.};   // losses, z, rows, sequences
  for (long k = tid; k < (long)a.S * nb; k += kSumThreads) v[0] += load_far(&o.loss[k]);
  for (int k = tid; k < a.S; k += kSumThreads) {
    int x, y;
    seq_rows(a, k, x, y);
    v[1] += load_far(&o.zsum[k]);
    v[2] += y - x;
    v[3] += y > x;
  }
  block_sums<WAVES>(v, red4);
  if (tid == 0) write_losses(o, v[0], v[1], v[2], v[3]);
}

struct Grads {
  const float2* stat;
  const float* weights;
  const int32_t* counts;
  const float* norm;
  const float* g_weights;   // [T][K] or null
  const float* g_balance;   // one value or null
  const float* g_z;
  void* out;                // [T][E], the logits' type
};

// A lane's selected experts of a row with their weights and gradients.
template <int L>
struct Picks {
  Ids<L> id;
  float w[Ids<L>::N], g[Ids<L>::N];
  float2 stat;
};

template <int L>
__device__ __forceinline__ void load_picks(const Rows& a, const Grads& o, long t, int i,
                                           Picks<L>& p) {
  p.stat = o.stat[t];
  if (!o.g_weights) return;
  load_ids(a, t, i, p.id);
#pragma unroll
  for (int n = 0; n < Ids<L>::N; ++n) {
    const int k = i + L * n;
    p.w[n] = k < a.K ? o.weights[t * a.K + k] : 0.f;
    p.g[n] = k < a.K ? o.g_weights[t * a.K + k] : 0.f;
  }
}

// One token per L lanes again.  The selected experts' parts meet the row's
// through LDS: lanes 0 .. K - 1 add them where their experts' owners read.
//   softmax: d_j = p_j (h_j - sum p h + z' - sum_k g_k w_k [not renormalised]) + sel_j
//   sigmoid: d_j = (1 - s_j) (p_j (h_j - sum p h) + sel_j)
template <int L, int V, bool SIG>
__global__ __launch_bounds__(kGradThreads) void router_grad_kernel(Rows a, int C, Grads o) {
  constexpr int G = 64 / L, NG = kGradWaves * G, COLS = L * V;
  __shared__ __attribute__((aligned(16))) float buf[NG][COLS];
  const int tid = threadIdx.x, lane = tid % 64, w = tid / 64;
  const int i = lane % L, g = w * G + lane / L;
  const int c0 = blockIdx.x * C, c1 = min(c0 + C, a.T);
  Raw<L, V> next;
  Picks<L> npick;
  int t = c0 + g;
  if (t < c1) {
    load_row(a, t, i, next);
    load_picks(a, o, t, i, npick);
  }
#pragma unroll
  for (int v = 0; v < V / 4; ++v)
    *reinterpret_cast<f32x4_t*>(&buf[g][4 * (i + L * v)]) = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float gb = o.g_balance ? *o.g_balance : 0.f;
  const float seqs = o.norm[0], rows = o.norm[1];
  const float gz = o.g_z && rows > 0.f ? 2.f * *o.g_z / rows : 0.f;
  float h[V];
  int q = -1, qb = 0, qe = 0;   // the sequence whose h is in registers, and its rows
  for (int t0 = c0; t0 < c1; t0 += NG, t += NG) {
    const bool on = t < c1;
    float l[V];
    values(a, next, l);
    const Picks<L> pick = npick;
    if (t + NG < c1) {
      load_row(a, t + NG, i, next);
      load_picks(a, o, t + NG, i, npick);
    }
    if (on && (q < 0 || (t >= qe && q < a.S))) {
      q = seq_of(a, t);
      if (q < a.S) seq_rows(a, q, qb, qe);
      const bool some = q < a.S && qe > qb && gb != 0.f;
      const float n = (float)(qe - qb);
      const float f = some ? gb * (float)a.E / ((float)a.K * n * n * seqs) : 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = 4 * (i + L * (v / 4)) + v % 4;
        h[v] = some && c < a.E ? f * (float)o.counts[(long)q * a.E + c] : 0.f;
      }
    }
    const bool in = on && q < a.S && t >= qb && t < qe;
    const float2 st = pick.stat;
    float rest[V], dot = 0.f;   // 1 - s
#pragma unroll
    for (int v = 0; v < V; ++v) {
      l[v] = score<SIG>(l[v], st.x, rest[v]) * st.y;   // p
      dot = __builtin_fmaf(l[v], h[v], dot);
    }
    dot = sum_over<L>(dot);
    // sum_k w_k g_k
    float wg = 0.f;
    if (o.g_weights) {
#pragma unroll
      for (int n = 0; n < Ids<L>::N; ++n)
        if (on && pick.id.e[n] >= 0) wg = __builtin_fmaf(pick.w[n], pick.g[n], wg);
      wg = sum_over<L>(wg);
      const float mean = a.renorm ? wg / a.scale : 0.f;
#pragma unroll
      for (int n = 0; n < Ids<L>::N; ++n)
        if (on && pick.id.e[n] >= 0) atomicAdd(&buf[g][pick.id.e[n]], pick.w[n] * (pick.g[n] - mean));
    }
    const float lse = !SIG && in && st.y != 0.f ? st.x - logf(st.y) : 0.f;
    const float base = (in ? -dot : 0.f) + (gz != 0.f ? gz * lse : 0.f) -
                       (!SIG && !a.renorm ? wg : 0.f);
    lds_order();
#pragma unroll
    for (int v = 0; v < V / 4; ++v) {
      const f32x4_t sel = *reinterpret_cast<const f32x4_t*>(&buf[g][4 * (i + L * v)]);
      f32x4_t d;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 4 * v + e;
        d[e] = __builtin_fmaf(l[k], (in ? h[k] : 0.f) + base, sel[e]);
        if (SIG) d[e] *= rest[k];
      }
      const int c = 4 * (i + L * v);
      if (!on || c >= a.E) continue;
      const long at = (long)t * a.E + c;
      if (a.bf16) {
        uint16_t* p = reinterpret_cast<uint16_t*>(o.out) + at;
        if (a.E % 4 == 0) {
          uint2 x;
          x.x = f32_to_bf16(d[0]) | (uint32_t)f32_to_bf16(d[1]) << 16;
          x.y = f32_to_bf16(d[2]) | (uint32_t)f32_to_bf16(d[3]) << 16;
          *reinterpret_cast<uint2*>(p) = x;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < a.E) p[e] = f32_to_bf16(d[e]);
        }
      } else {
        float* p = reinterpret_cast<float*>(o.out) + at;
        if (a.E % 4 == 0) {
          *reinterpret_cast<f32x4_t*>(p) = d;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < a.E) p[e] = d[e];
        }
      }
    }
    lds_order();
    if (o.g_weights)
#pragma unroll
      for (int n = 0; n < Ids<L>::N; ++n)
        if (on && pick.id.e[n] >= 0) buf[g][pick.id.e[n]] = 0.f;
    lds_order();
  }
}

// Lanes of a token and its experts a lane, by E.
struct Layout {
  int lanes, vals;
};
Layout layout_of(int E) {
  if (E <= 16) return {4, 4};
  if (E <= 32) return {8, 4};
  if (E <= 64) return {16, 4};
  if (E <= 128) return {32, 4};
  if (E <= 256) return {64, 4};
  if (E <= 512) return {64, 8};
  return {64, 16};
}

// Rows of a chunk: whole turns of a workgroup, about `chunks` chunks.
int chunk_rows(int T, int E, int waves, int chunks) {
  const int ng = waves * 64 / layout_of(E).lanes;
  const int c = T > 0 ? (int)(((long)T + chunks - 1) / chunks) : 1;
  return (c + ng - 1) / ng * ng;
}
int forward_rows(int T, int E) {
  const int c = chunk_rows(T, E, kWaves, kMaxChunks);
  const int most = kLaneRows * (kWaves * 64 / layout_of(E).lanes);
  return c < most ? c : most;
}

// Whether one workgroup does it all.
bool one_fits(int T, int E, int S) {
  return T <= kOneTurns * kWaves * 64 / layout_of(E).lanes && S <= kOneSeqs;
}

// The workspace: partial rows, losses, ticket.
struct Space {
  size_t p, c, z, loss, zsum, ticket, bytes;
};
Space space_of(int T, int E, int S) {
  const int C = forward_rows(T, E);
  const size_t slots = ((size_t)T + C - 1) / C + S, nb = (E + kCols - 1) / kCols;
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Space s;
  s.p = 0;
  s.c = s.p + up(slots * E * 4);
  s.z = s.c + up(slots * E * 4);
  s.loss = s.z + up(slots * 4);
  s.zsum = s.loss + up((size_t)S * nb * 8);
  s.ticket = s.zsum + up((size_t)S * 8);
  s.bytes = s.ticket + 256;
  return s;
}

template <bool SIG, class F>
hipError_t by_layout(int E, F f) {
  switch (layout_of(E).lanes * 100 + layout_of(E).vals) {
    case 404: return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
    case 804: return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
    case 1604: return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
    case 3204: return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{});
    case 6404: return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    case 6408: return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
    default: return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
  }
}

// The second launch: a workgroup per sequence and kCols experts, below 2^32 threads.
bool grid_ok(int E, int S) { return (long)S * ((E + kCols - 1) / kCols) * kSumThreads < (1L << 32); }

bool rows_of(const xtu_router_args& t, Rows& a) {
  if (t.T < 0 || t.T > (1 << 30) || t.E < 1 || t.E > kMaxE || t.K < 1 || t.K > kMaxK ||
      t.S < 1 || t.mode < 0 || t.mode > 1 || !(t.scale > 0.f) ||
      !(t.scale < INFINITY))
    return false;
  if (!grid_ok(t.E, t.S)) return false;
  if (t.T > 0 && (!t.logits || !t.ids || t.ld < 0)) return false;
  if (!t.starts && t.S != 1) return false;
  const size_t size = t.logits_bf16 ? 2 : 4;
  a = Rows{t.logits, t.ld, t.logits_bf16, 0, t.ids, t.starts, t.T, t.E, t.K, t.S, t.mode,
           t.renormalize, t.scale};
  if (reinterpret_cast<uintptr_t>(t.logits) % size || reinterpret_cast<uintptr_t>(t.ids) % 4 ||
      reinterpret_cast<uintptr_t>(t.starts) % 4)
    return false;
  a.vec = t.E % 4 == 0 && (t.T <= 1 || t.ld % 4 == 0) &&
          reinterpret_cast<uintptr_t>(t.logits) % (4 * size) == 0;
  return true;
}

}  // namespace
}  // namespace rt
}  // namespace xtu

using namespace xtu;
using namespace xtu::rt;

extern "C" {

size_t xtu_router_workspace_bytes(int T, int E, int S) {
  if (T < 0 || T > (1 << 30) || E < 1 || E > kMaxE || S < 1 || !grid_ok(E, S)) return 0;
  return space_of(T, E, S).bytes;
}

hipError_t xtu_router_losses(const xtu_router_args* args, hipStream_t stream) {
  XTU_CHECK_ARG(args);
  const xtu_router_args& t = *args;
  Rows a;
  XTU_CHECK_ARG(rows_of(t, a));
  XTU_CHECK_ARG(t.counts && t.probs && t.balance && t.norm && t.workspace);
  XTU_CHECK_ARG(t.T == 0 || (t.weights && t.stat));
  XTU_CHECK_ARG((t.mode == 0) == (t.z != nullptr));
  const Space s = space_of(t.T, t.E, t.S);
  XTU_CHECK_ARG(t.workspace_bytes >= s.bytes && reinterpret_cast<uintptr_t>(t.workspace) % 16 == 0);
  uint8_t* ws = reinterpret_cast<uint8_t*>(t.workspace);
  const Sums o{reinterpret_cast<float*>(ws + s.p), reinterpret_cast<int32_t*>(ws + s.c),
               reinterpret_cast<float*>(ws + s.z), reinterpret_cast<double*>(ws + s.loss),
               reinterpret_cast<double*>(ws + s.zsum), reinterpret_cast<unsigned*>(ws + s.ticket),
               t.counts, t.probs, t.balance, t.z, t.norm};
  const bool one = one_fits(t.T, t.E, t.S);
  const int C = one ? (t.T ? t.T : 1) : forward_rows(t.T, t.E);
  const int chunks = one ? 1 : (int)(((long)t.T + C - 1) / C);
  const int grid = chunks ? chunks : 1;   // (one writes the ticket)
  (void)hipGetLastError();
  const auto go = [&](auto sig) {
    return by_layout<decltype(sig)::value>(t.E, [&](auto l, auto v) {
      constexpr int L = decltype(l)::value, V = decltype(v)::value;
      constexpr bool SIG = decltype(sig)::value;
      const auto k = one ? router_stats_kernel<L, V, SIG, true> : router_stats_kernel<L, V, SIG, false>;
      k<<<grid, kThreads, 0, stream>>>(a, C, t.weights, reinterpret_cast<float2*>(t.stat), o);
      return hipPeekAtLastError();
    });
  };
  const hipError_t e = t.mode ? go(std::true_type{}) : go(std::false_type{});
  if (e != hipSuccess || one) return e;
  const int nb = (t.E + kCols - 1) / kCols;
  router_finish_kernel<<<(unsigned)t.S * nb, kSumThreads, 0, stream>>>(a, C, o);
  return hipPeekAtLastError();
}

hipError_t xtu_router_grad(const xtu_router_args* args, const float* g_weights,
                           const float* g_balance, const float* g_z, void* dlogits,
                           hipStream_t stream) {
  XTU_CHECK_ARG(args);
  const xtu_router_args& t = *args;
  Rows a;
  XTU_CHECK_ARG(rows_of(t, a));
  if (t.T == 0) return hipSuccess;
  XTU_CHECK_ARG(t.counts && t.norm && t.weights && t.stat && dlogits);
  XTU_CHECK_ARG(t.mode == 0 || !g_z);
  XTU_CHECK_ARG(reinterpret_cast<uintptr_t>(dlogits) % 16 == 0);
  const int C = chunk_rows(t.T, t.E, kGradWaves, kGradChunks);
  const int chunks = (int)(((long)t.T + C - 1) / C);
  const Grads o{reinterpret_cast<const float2*>(t.stat), t.weights, t.counts, t.norm, g_weights,
                g_balance, g_z, dlogits};
  (void)hipGetLastError();
  const auto go = [&](auto sig) {
    return by_layout<decltype(sig)::value>(t.E, [&](auto l, auto v) {
      router_grad_kernel<decltype(l)::value, decltype(v)::value, decltype(sig)::value>
          <<<chunks, kGradThreads, 0, stream>>>(a, C, o);
      return hipPeekAtLastError();
    });
  };
  return t.mode ? go(std::true_type{}) : go(std::false_type{});
}

}  // extern "C"
