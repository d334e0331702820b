// The MoE block of a few tokens in two launches, from hidden states:
//
//   logits = x Wg^T;  (ids, w) = selection(logits)
//   y[t] = sum_k w[t][k] E_{ids[t][k]}(x[t]) + sum_s g[t][s] S_s(x[t])
//
// with g = sigmoid(x . v_s) where the shared experts have a gate, else 1.
//
// Launch 1 (few_router_kernel) does what needs no routing: the router product
// (and the shared gates' rows), in panels of a few rows so that every CU has
// one, and the shared experts' gate/up.  It also clears launch 2's counters, so
// a workspace needs no state from one call to the next.
//
// Launch 2 (few_experts_kernel) is persistent: every workgroup selects the
// batch's experts in LDS for itself (same code, same logits: all agree), then
// draws work items: first the routed gate/up panels, expert by expert, then the
// output panels (down projection and weighted sum).  Before its first output
// panel a workgroup waits until every gate/up panel is done, and before that
// wait it has seen every gate/up panel drawn: those waited for are in the hands
// of workgroups that run and wait for nothing, so the wait ends whatever else
// shares the device, also where part of this launch is not resident yet.
//
// Items are dealt into eight groups, item i to group i % 8, with a counter each
// (one address takes about 100 atomics in a microsecond: all workgroups on one
// counter spent 10 us on their first items); a workgroup draws from the group of
// its XCD, and from the others' gate/up items when that is used up.
//
// Both phases are weight streams (the arithmetic is decode.hpp's): a wave's
// loads for its next item are issued as the registers of the present one are
// used up, so the stream does not pause at item ends, and a workgroup's first
// output panel is loaded while it waits.
//
// gate/up: an item is (expert, 16 gate and the 16 up rows); four waves split K
// for each half.  Down: an item is 16 output columns over a chunk of the active
// experts; the eight waves take (expert, up to 4 x 128 k) segments in turn and
// multiply by the token's weight as they add up.  The chunk's activation rows sit
// in LDS; with more than one chunk the chunks' sums go to memory and the last
// one to finish a panel adds them in chunk order, so results do not depend on
// timing.
#pragma once
#include "decode.hpp"

#include <cmath>

namespace xtu {
namespace few {

struct FewArgs {
  const uint16_t* x;        // [T][H]
  const uint16_t* gate;     // [E][H]
  const uint16_t* sgate;    // [NS][H] or null
  const float* bias;        // [E] or null
  int T, H, I, E, NS, K;
  int mode, renorm, n_group, topk_group;   // mode 0 softmax, 1 grouped sigmoid
  float scale;
  const uint8_t *w13, *s13, *w2, *s2;
  const float *gs13, *gs2;
  long w13_es, s13_es, w2_es, s2_es;
  float limit, alpha, beta;
  float* logits;            // [T][ldl]: E router logits, then the shared gates'
  int ldl;
  uint16_t* act;            // [T K + NS T][I]: routed rows by expert, then the shared experts'
  float* part;              // [chunks][T][H] (chunks > 1)
  unsigned* ctl;
  int ctl_words;
  int32_t* ids;
  float* wts;
  void* out;
  int out_bf16;
  int rp, n_sh;             // launch 1: router rows per panel; its shared gate/up items
  int epl;                  // experts per lane of the wave router (0: any E)
  int rows_per_chunk, chunks;              // launch 2: activation rows in LDS
  size_t stage_bytes;
};

// LDS and chunk plan of launch 2.  Two workgroups share a CU where the x rows
// and all activation rows fit half its LDS; otherwise one takes what it needs.
struct Plan {
  size_t stage, lds;
  int rows_per_chunk, chunks, occ;
};

namespace {

constexpr int kMaxT = 16, kMaxPairs = 256, kMaxShared = 4, kMaxE = 1024, kMaxGroups = 64;
constexpr int kThreads = 512, kWaves = 8, kKS = 4;   // waves along K per gate/up half
constexpr int kLine = 64;                            // words of a counter's own 256 bytes

// Counters (words): per group the gate/up items drawn, the output items drawn
// and the gate/up items done; a flag set if a wait ever ran out; then the chunks
// done per output panel.
constexpr int kGroups = 8;
constexpr int kTicket = 0, kTicket3 = 8 * kLine, kDone = 16 * kLine, kFlag = 24 * kLine,
              kPanels = 25 * kLine;
constexpr int kSpin = 1 << 20;


// The x rows to LDS, 16 bytes of padding each; a thread's loads go out eight
// at a time.
__device__ __forceinline__ void stage_x(const FewArgs& f, uint16_t* xs) {
  const int ldx = f.H + 8, per_row = f.H / 8, pieces = f.T * per_row;
  constexpr int SB = 8;
  for (int c0 = threadIdx.x; c0 < pieces; c0 += SB * kThreads) {
    u32x4_t v[SB];
#pragma unroll
    for (int k = 0; k < SB; ++k)
      v[k] = *reinterpret_cast<const u32x4_t*>(f.x + 8L * min(c0 + k * kThreads, pieces - 1));
#pragma unroll
    for (int k = 0; k < SB; ++k) {
      const int p = c0 + k * kThreads;
      if (p < pieces) {
        const int r = p / per_row;
        *reinterpret_cast<u32x4_t*>(xs + r * ldx + (p - r * per_row) * 8) = v[k];
      }
    }
  }
}

// ---------------------------------------------------------------- launch 1
template <int FMT, int NU>
__global__ __launch_bounds__(kThreads, 2) void few_router_kernel(FewArgs f) {
  using F = WFmt<FMT>;
  extern __shared__ __attribute__((aligned(16))) uint16_t xs[];   // [T][H + 8]
  __shared__ f32x4_t red[kWaves][kWave];
  const int tid = threadIdx.x;
  const int w = wave_id();
  const uint32_t lane = tid % kWave;
  const int q = lane / 16, m = lane % 16;
  const int ldx = f.H + 8;
  if (blockIdx.x == gridDim.x - 1)
    for (int i = tid; i < f.ctl_words; i += kThreads) f.ctl[i] = 0u;
  const uint16_t* xrow = xs + min(m, f.T - 1) * ldx;

  if ((int)blockIdx.x < f.n_sh) {   // a shared expert's gate/up panel, all T rows
    const int npan = f.I / 16;
    const int sh = blockIdx.x / npan, sub = blockIdx.x - sh * npan, ws = f.E + sh;
    DecodeArgs a{};
    a.w = f.w13;
    a.s = f.s13;
    a.gs = f.gs13;
    a.out = f.act;
    a.H = f.H;
    a.I = f.I;
    a.w_estride = f.w13_es;
    a.s_estride = f.s13_es;
    a.limit = f.limit;
    a.alpha = f.alpha;
    a.beta = f.beta;
    a.ksplit = kKS;
    const int half = w / kKS, ks = w % kKS, nunits = f.H / 128;
    const int u0 = ks * nunits / kKS, u1 = (ks + 1) * nunits / kKS;
    const Stream<FMT> st = make_stream<FMT>(a, ws, half ? npan + sub : sub, f.H);
    Round<FMT, NU> r;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    if (u0 < u1) issue_round<FMT, NU>(r, st, u0, u1, lane);
    __builtin_amdgcn_sched_barrier(0);
    stage_x(f, xs);
    __syncthreads();
    const uint16_t* xa = xrow + q * F::kCK;
    if (u0 < u1) {
      consume_round<FMT, NU, true>(r, acc, u0, u1, xa, nullptr);
      if (u0 + NU < u1) acc = more_rounds<FMT, NU, true>(acc, st, u0 + NU, u1, lane, xa, nullptr);
    }
    gate_up_epilogue<FMT>(a, red, acc, w, lane, f.T * f.K + sh * f.T, f.T, ws, sub);
    return;
  }

  // router rows [row0, row0 + rp): eight waves along K, w rows as the MFMA's A
  // operand (rows past the panel repeat its last one), the tokens as B
  const int er = f.E + (f.sgate ? f.NS : 0);
  const int row0 = (blockIdx.x - f.n_sh) * f.rp;
  const int row = min(row0 + min(m, f.rp - 1), er - 1);
  const uint16_t* wr = (row < f.E ? f.gate + (long)row * f.H : f.sgate + (long)(row - f.E) * f.H) +
                       8 * q;
  const int nst = f.H / 32 / kWaves, s0 = w * nst;   // H % 256 == 0
  constexpr int U = 8;
  u32x4_t wv[U];
#pragma unroll
  for (int i = 0; i < U; ++i)
    wv[i] = *reinterpret_cast<const u32x4_t*>(wr + 32 * (s0 + min(i, nst - 1)));
  __builtin_amdgcn_sched_barrier(0);
  stage_x(f, xs);
  __syncthreads();
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  auto use = [&](int i, int s) {
    if (s < nst) {
      const u32x4_t xv = *reinterpret_cast<const u32x4_t*>(xrow + 32 * (s0 + s) + 8 * q);
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(wv[i]), as_bf16x8(xv), acc, 0, 0, 0);
    }
  };
  int s = 0;
  for (; s + U < nst; s += U) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      use(i, s + i);
      wv[i] = *reinterpret_cast<const u32x4_t*>(wr + 32 * (s0 + min(s + U + i, nst - 1)));
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) use(i, s + i);
  red[w][lane] = acc;
  __syncthreads();
  if (tid < 256) {
    const int e = tid / 64, nl = 4 * q + e, n = row0 + nl;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) v += red[k][lane][e];
    if (m < f.T && nl < f.rp && n < er) f.logits[(long)m * f.ldl + n] = v;
  }
}

// ---------------------------------------------------------------- selection
// One wave selects one token's experts for any E <= 1024 (lane l holds experts
// l, l + 64, ..): K rounds of a wave-wide maximum of order-preserving keys,
// equal ones to the lowest index.  Scores, group scores and weights are
// route_token_wave's, in the same fp32 sequences (the sum over all experts,
// where the weights are not renormalised, lane by lane).
__device__ void select_any(const FewArgs& f, const float* l, int lane, int* ids_lds,
                           float* wts_lds, float* scr) {
#pragma clang fp contract(off)
  constexpr int N = kMaxE / kWave;
  const int E = f.E, K = f.K;
  uint32_t key[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = lane + kWave * i;
    key[i] = 0u;
    if (e < E) {
      float sc = l[e];
      if (f.mode == 1) {
        sc = xtu_sigmoid(sc) + (f.bias ? f.bias[e] : 0.0f);
        if (f.n_group > 1) scr[e] = sc;   // E floats of this wave's own
      }
      key[i] = max(tiny::score_key(sc), 1u);   // 0: no expert, or taken
    }
  }
  if (f.mode == 1 && f.n_group > 1) {
    // group score: the two best of the group, added; the topk_group best stay
    tiny::lds_wave_order();
    const int gsz = E / f.n_group;
    float gs = 0.f;
    if (lane < f.n_group) {
      float v1 = -__builtin_inff(), v2 = v1;
      for (int j = 0; j < gsz; ++j) {
        const float v = scr[lane * gsz + j];
        if (v > v1) {
          v2 = v1;
          v1 = v;
        } else if (v > v2) {
          v2 = v;
        }
      }
      gs = gsz >= 2 ? v1 + v2 : v1;
    }
    int r = 0;
    for (int j = 0; j < f.n_group; ++j) {
      const float o = tiny::readlane_f(gs, j);
      r += (o > gs || (o == gs && j < lane)) ? 1 : 0;
    }
    const unsigned long long kept = __ballot(lane < f.n_group && r < f.topk_group);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = lane + kWave * i;
      if (e < E && !((kept >> (e / gsz)) & 1ull)) key[i] = 0u;
    }
  }
  int my_e = 0;
  for (int k = 0; k < K; ++k) {
    uint32_t best = 0u;
    int bi = 0;
#pragma unroll
    for (int i = N - 1; i >= 0; --i)
      if (key[i] >= best) {   // equal keys: the lower i
        best = key[i];
        bi = i;
      }
    const uint32_t top = tiny::wave_max_u32(best);
    // lowest index among the lanes that hold the maximum (none left, which
    // NaN groups can bring about: expert k)
    const uint32_t e_inv = best == top ? (uint32_t)(kMaxE - (lane + kWave * bi)) : 0u;
    const int e = top ? kMaxE - (int)tiny::wave_max_u32(e_inv) : k;
    if (lane == k) my_e = e;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + kWave * i == e) key[i] = 0u;
  }
  const float my_l = lane < K ? l[my_e] : 0.f;
  float w = 0.f;
  if (f.mode == 0) {
    const float lmax = tiny::readlane_f(my_l, 0);
    const float ev = lane < K ? xtu_expf(my_l - lmax) : 0.f;
    float sum = 0.0f;
    if (f.renorm) {
      for (int k = 0; k < K; ++k) sum = sum + tiny::readlane_f(ev, k);
    } else {   // over all E: each lane's experts, then the lanes
      for (int e = lane; e < E; e += kWave) sum = sum + xtu_expf(l[e] - lmax);
      for (int o = 32; o; o >>= 1) sum = sum + __shfl_xor(sum, o, kWave);
    }
    w = __fdiv_rn(ev, sum);
  } else {
    const float sg = lane < K ? xtu_sigmoid(my_l) : 0.f;
    float sum = 0.0f;
    for (int k = 0; k < K; ++k) sum = sum + tiny::readlane_f(sg, k);
    w = f.renorm ? __fdiv_rn(sg, sum) * f.scale : sg * f.scale;
  }
  if (lane < K) {
    ids_lds[lane] = my_e;
    wts_lds[lane] = w;
  }
}

template <int EPL>
__device__ __forceinline__ void select_wave(const FewArgs& f, const float* l, int lane, int* ids,
                                            float* wts) {
  if (f.mode == 1)
    tiny::route_token_wave<1, EPL>(l, f.bias, f.K, f.n_group, f.topk_group, f.scale, f.renorm,
                                   lane, nullptr, nullptr, ids, wts);
  else
    tiny::route_token_wave<0, EPL>(l, nullptr, f.K, 1, 1, 1.0f, 1, lane, nullptr, nullptr, ids,
                                   wts);
}

// The batch's selection, as every workgroup of launch 2 holds it.  A slot is an
// active expert: the routed ones ascending, then the shared ones.
struct Sel {
  int ids[kMaxPairs];
  float wts[kMaxPairs];
  int rank[kMaxPairs];                       // earlier pairs of the same expert
  int slot_e[kMaxPairs + kMaxShared];
  int slot_r0[kMaxPairs + kMaxShared + 1];   // first activation row
  int row_tok[kMaxPairs + kMaxShared * kMaxT];
  int first[kMaxPairs];
  int n_routed;                              // slots of routed experts
  int ticket[2];
  int last;
};

// One thread of a workgroup draws an item of group g: which = kTicket (gate/up)
// or kTicket3 (output panels).
__device__ __forceinline__ int draw(const FewArgs& f, int which, int g) {
  return kGroups * (int)__hip_atomic_fetch_add(f.ctl + which + kLine * g, 1u, __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT) + g;
}

// rowof / wof: [slot][16] activation row and weight of token t in that slot
// (weight 0: the token does not use it).
// stage gets the x rows; scr: E floats per wave for select_any's groups.
// The workgroup's first two tickets are drawn on the way, the second once the
// first is back: by then every workgroup has drawn its first, so work spreads
// over all of them before anyone takes a second item.
__device__ __forceinline__ void build_selection(const FewArgs& f, Sel& g, uint16_t* rowof,
                                                float* wof, uint16_t* stage, float* scr) {
  const int tid = threadIdx.x, lane = tid % kWave, wv = wave_id();
  const int T = f.T, K = f.K, A = T * K, NS = f.NS;
  const bool drawer = tid == kThreads - kWave;
  int t0 = 0;
  const int grp = blockIdx.x % kGroups;
  if (drawer) t0 = draw(f, kTicket, grp);
  stage_x(f, stage);
  for (int t = wv; t < T; t += kWaves) {
    const float* l = f.logits + (long)t * f.ldl;
    int* ids = g.ids + t * K;
    float* wts = g.wts + t * K;
    switch (f.epl) {
      case 2: select_wave<2>(f, l, lane, ids, wts); break;
      case 4: select_wave<4>(f, l, lane, ids, wts); break;
      case 8: select_wave<8>(f, l, lane, ids, wts); break;
      default: select_any(f, l, lane, ids, wts, scr + wv * f.E); break;
    }
  }
  if (drawer) {
    g.ticket[0] = t0;
    __asm__ __volatile__("" ::"v"(t0) : "memory");   // the first ticket is back
    g.ticket[1] = draw(f, kTicket, grp);
  }
  for (int i = tid; i < kMaxPairs; i += kThreads)
    if (i >= A) g.ids[i] = 0x7fffffff;
  const int max_slots = min(f.E, A) + NS;
  for (int i = tid; i < max_slots * kMaxT; i += kThreads) {
    rowof[i] = 0;
    wof[i] = 0.f;
  }
  __syncthreads();
  const int A4 = (A + 3) / 4;
  int r0 = 0, rank = 0, e = 0;
  if (tid < A) {   // thread p: pair p
    e = g.ids[tid];
#pragma unroll 4
    for (int j = 0; j < A4; ++j) {
      const i32x4_t v = *reinterpret_cast<const i32x4_t*>(g.ids + 4 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r0 += v[i] < e ? 1 : 0;
        rank += v[i] == e && 4 * j + i < tid ? 1 : 0;
      }
    }
    g.rank[tid] = rank;
    g.first[tid] = rank == 0 ? e : 0x7fffffff;   // an expert's first pair
  } else if (tid < kMaxPairs) {
    g.first[tid] = 0x7fffffff;
  }
  __syncthreads();
  if (tid < A) {
    int slot = 0;   // experts below e
#pragma unroll 4
    for (int j = 0; j < A4; ++j) {
      const i32x4_t v = *reinterpret_cast<const i32x4_t*>(g.first + 4 * j);
      slot += (v[0] < e) + (v[1] < e) + (v[2] < e) + (v[3] < e);
    }
    const int t = tid / K, row = r0 + rank;
    g.row_tok[row] = t;
    rowof[slot * kMaxT + t] = (uint16_t)row;
    wof[slot * kMaxT + t] = g.wts[tid];
    if (rank == 0) {
      g.slot_e[slot] = e;
      g.slot_r0[slot] = r0;
    }
  }
  if (wv == kWaves - 1) {   // the shared experts' slots, behind the routed ones
    int n = 0;
    for (int i = 0; i < kMaxPairs; i += kWave)
      n += __popcll(__ballot(g.first[i + lane] != 0x7fffffff));
    if (lane == 0) {
      g.n_routed = n;
      g.slot_r0[n + NS] = A + NS * T;
    }
    if (lane < NS) {
      g.slot_e[n + lane] = f.E + lane;
      g.slot_r0[n + lane] = A + lane * T;
    }
    for (int i = lane; i < NS * T; i += kWave) {
      const int s = i / T, t = i - s * T;
      rowof[(n + s) * kMaxT + t] = (uint16_t)(A + i);
      wof[(n + s) * kMaxT + t] =
          f.sgate ? xtu_sigmoid(f.logits[(long)t * f.ldl + f.E + s]) : 1.0f;
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------- launch 2
// A round of the gate/up stream with the next one's loads rolling in: unit i
// of the next round (nst, [nub, nu1)) takes the registers of unit i as soon as
// it is multiplied.  A dead next stream has zero-length buffers.
template <int FMT, int NU>
__device__ __forceinline__ void roll_round(Round<FMT, NU>& r, f32x4_t& acc, int ub, int u1,
                                           const uint16_t* xa, const Stream<FMT>& nst, int nub,
                                           int nu1, uint32_t lane) {
  using F = WFmt<FMT>;
  using R = Round<FMT, NU>;
  R n;   // scales only
  if constexpr (R::kGroups > 0) {
    const int g0 = nub / F::kUG;
#pragma unroll
    for (int j = 0; j < R::kGroups; ++j) {
      const u32x4_t v = __builtin_bit_cast(
          u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(nst.s, (int)lane * 16, (g0 + j) * 1024,
                                                         kAuxNontemporal));
#pragma unroll
      for (int i = 0; i < 4; ++i) n.sw[4 * j + i] = v[i];
    }
    shift_bytes_down(r.sw, (ub % F::kUG) * F::kSBY);
  } else if constexpr (FMT == kFP8) {
    n.bsv = __builtin_bit_cast(
        float, __builtin_amdgcn_raw_buffer_load_b32(nst.s, (int)lane * 4, nub * 4, 0));
  }
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if (ub + i < u1) {
      uint32_t sraw = 0u;
      float bs = 1.0f;
      if constexpr (FMT == kMXFP4) sraw = r.sw[i / 4] >> (8 * (i % 4));
      else if constexpr (FMT == kNVFP4) sraw = r.sw[i / 2] >> (16 * (i % 2));
      else if constexpr (FMT == kFP8)
        bs = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, r.bsv), i));
      mma_unit<FMT, true>(r.w[i], sraw, bs, acc, ub + i, xa, nullptr);
    }
    const int u = nub + i < nu1 ? nub + i : max(nu1 - 1, 0);
#pragma unroll
    for (int j = 0; j < F::kSPU; ++j)
      r.w[i][j] = __builtin_bit_cast(
          u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(nst.w, (int)lane * 16,
                                                         (u * F::kSPU + j) * 1024,
                                                         kAuxNontemporal));
  }
  if constexpr (R::kGroups > 0) {
#pragma unroll
    for (int j = 0; j < 4 * R::kGroups; ++j) r.sw[j] = n.sw[j];
  } else if constexpr (FMT == kFP8) {
    r.bsv = n.bsv;
  }
}

// A segment of the down stream: up to NPER units of one expert's panel.
template <int FMT, int NPER>
struct Seg {
  u32x4_t w[NPER][WFmt<FMT>::kSPU];
  uint32_t sc0, sc1;   // fp4: the units' scale bytes
  float bsv;           // fp8: lane i holds the block scale of unit u0 + i
};

template <int FMT, int NPER>
__device__ __forceinline__ void issue_seg(Seg<FMT, NPER>& r, const FewArgs& f, int ws, bool live,
                                          int panel, int u0, uint32_t lane) {
  using F = WFmt<FMT>;
  const int nu = f.I / 128;
  const long nsb = f.I / F::kSB;
  const uint8_t* sx = f.s2 + (long)ws * f.s2_es;
  const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(f.w2 + (long)ws * f.w2_es + (long)panel * nsb * 1024), 0,
      live ? (int)(nsb * 1024) : 0, kRawBufferFlags);
  if constexpr (FMT == kMXFP4 || FMT == kNVFP4) {
    const long gbytes = scale_groups(f.I, F::kUG) * 1024;
    const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(sx + (long)panel * gbytes), 0, live ? (int)gbytes : 0, kRawBufferFlags);
    const int off = (u0 % F::kUG) * F::kSBY;   // the units' bytes sit in one aligned word of 8
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(
        sr, (int)lane * 16 + (off & 8), (u0 / F::kUG) * 1024, kAuxNontemporal);
    const uint64_t b = ((uint64_t)v[1] << 32 | v[0]) >> (8 * (off & 7));
    r.sc0 = (uint32_t)b;
    r.sc1 = (uint32_t)(b >> 32);
  } else if constexpr (FMT == kFP8) {
    const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(sx + (long)(panel / 8) * nu * 4), 0, live ? nu * 4 : 0, kRawBufferFlags);
    r.bsv = __builtin_bit_cast(
        float, __builtin_amdgcn_raw_buffer_load_b32(sr, (int)(lane + u0) * 4, 0, 0));
  }
#pragma unroll
  for (int i = 0; i < NPER; ++i)
#pragma unroll
    for (int j = 0; j < F::kSPU; ++j)
      r.w[i][j] = __builtin_bit_cast(
          u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                       wr, (int)lane * 16, (min(u0 + i, nu - 1) * F::kSPU + j) * 1024,
                       kAuxNontemporal));
}

template <int FMT, int NPER>
__device__ __forceinline__ f32x4_t use_seg(const Seg<FMT, NPER>& r, int u0, int nu,
                                           const uint16_t* xa) {
  f32x4_t pe = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NPER; ++i) {
    if (u0 + i < nu) {
      uint32_t sraw = 0u;
      float bs = 1.0f;
      if constexpr (FMT == kMXFP4) sraw = r.sc0 >> (8 * i);
      else if constexpr (FMT == kNVFP4) sraw = (i < 2 ? r.sc0 : r.sc1) >> (16 * (i % 2));
      else if constexpr (FMT == kFP8)
        bs = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, r.bsv), i));
      mma_unit<FMT, true>(r.w[i], sraw, bs, pe, u0 + i, xa, nullptr);
    }
  }
  return pe;
}

// Segments in flight per wave: as many as keep the kernel at 128 VGPRs.
template <int FMT, int NPER>
constexpr int ring_depth() {
  return FMT == kBF16 ? 2 : FMT == kFP8 ? (NPER == 4 ? 2 : 4) : (NPER == 4 ? 4 : 6);
}

constexpr int kAuxDev = 16;   // buffer access at device scope (sc1)

// Fixed LDS of launch 2 behind the stage: the selection, then rowof and wof.
__host__ __device__ constexpr size_t sel_bytes() { return (sizeof(Sel) + 15) / 16 * 16; }
__host__ __device__ inline size_t table_bytes(int max_slots) {
  return (size_t)max_slots * kMaxT * 6;
}

// OCC: workgroups that are to share a CU (128 or 256 VGPRs).
template <int FMT, int NU, int NPER, int OCC>
__global__ __launch_bounds__(kThreads, 2 * OCC) void few_experts_kernel(FewArgs f) {
  using F = WFmt<FMT>;
  constexpr int D = ring_depth<FMT, NPER>();
  extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
  __shared__ f32x4_t red[2][kWaves][kWave];
  uint16_t* stage = reinterpret_cast<uint16_t*>(dyn);   // x rows, then activation rows
  Sel& g = *reinterpret_cast<Sel*>(dyn + f.stage_bytes);
  float* wof = reinterpret_cast<float*>(dyn + f.stage_bytes + sel_bytes());
  const int tid = threadIdx.x;
  const int w = wave_id();
  const uint32_t lane = tid % kWave;
  const int q = lane / 16, m = lane % 16;
  const int T = f.T, H = f.H, I = f.I;
  const int max_slots = min(f.E, T * f.K) + f.NS;
  uint16_t* rowof = reinterpret_cast<uint16_t*>(wof + max_slots * kMaxT);
  build_selection(f, g, rowof, wof, stage,
                  reinterpret_cast<float*>(dyn + (size_t)T * (H + 8) * 2));
  if (blockIdx.x == 0) {
    for (int i = tid; i < T * f.K; i += kThreads) {
      f.ids[i] = g.ids[i];
      f.wts[i] = g.wts[i];
    }
  }
  int cur = __builtin_amdgcn_readfirstlane(g.ticket[0]);
  int nxt = __builtin_amdgcn_readfirstlane(g.ticket[1]);
  __syncthreads();   // the words are read before an item's draw takes one
  const int n_routed = __builtin_amdgcn_readfirstlane(g.n_routed);
  const int npan = I / 16, hpan = H / 16;
  const int n2 = n_routed * npan, n3 = f.chunks * hpan;
  const int grp = blockIdx.x % kGroups;
  int t_new = 0;
  int it = 0;   // items done: which half of red, which ticket word

  // ---- routed gate/up
  {
    DecodeArgs a{};
    a.w = f.w13;
    a.s = f.s13;
    a.gs = f.gs13;
    a.out = f.act;
    a.H = H;
    a.I = I;
    a.w_estride = f.w13_es;
    a.s_estride = f.s13_es;
    a.limit = f.limit;
    a.alpha = f.alpha;
    a.beta = f.beta;
    a.ksplit = kKS;
    const int half = w / kKS, ks = w % kKS, nunits = H / 128;
    const int u0 = ks * nunits / kKS, u1 = (ks + 1) * nunits / kKS;
    const int rounds = max((u1 - u0 + NU - 1) / NU, 1);
    auto stream_of = [&](int item) {
      const bool live = item < n2;
      const int slot = live ? item / npan : 0, sub = live ? item - slot * npan : 0;
      const int e = __builtin_amdgcn_readfirstlane(g.slot_e[slot]);
      return make_stream<FMT>(a, e, half ? npan + sub : sub, H, live);
    };
    const int ldx = H + 8;
    int count = 0;
    Round<FMT, NU> r;
    while (true) {
      if (cur >= n2) {
        // the own group is used up: an item of another one, if any is left
        nxt = n2;
        if (w == 0) {
          int got = n2;
          while (true) {
            const int left = (int)lane < kGroups
                                 ? (int)__hip_atomic_load(f.ctl + kTicket + kLine * lane,
                                                          __ATOMIC_RELAXED,
                                                          __HIP_MEMORY_SCOPE_AGENT) * kGroups +
                                       (int)lane
                                 : n2;
            const unsigned long long some = __ballot(left < n2);
            if (!some) break;
            int t = 0;
            if (lane == 0) t = draw(f, kTicket, __builtin_ctzll(some));
            got = __builtin_amdgcn_readfirstlane(t);
            if (got < n2) break;   // (else someone was quicker: look again)
          }
          if (lane == 0) g.ticket[it & 1] = got;
        }
        __syncthreads();
        cur = __builtin_amdgcn_readfirstlane(g.ticket[it & 1]);
        __syncthreads();
        if (cur >= n2) break;
      }
      Stream<FMT> st = stream_of(cur);
      if (u0 < u1) issue_round<FMT, NU>(r, st, u0, u1, lane);
      __builtin_amdgcn_sched_barrier(0);
      while (true) {   // cur is loaded; nxt rolls in behind it
        if (tid == 0) t_new = nxt < n2 ? draw(f, kTicket, grp) : n2;
        const int slot = cur / npan, sub = cur - slot * npan;
        const int r0 = g.slot_r0[slot], na = g.slot_r0[slot + 1] - r0;
        const int ws = g.slot_e[slot];
        const int tok = g.row_tok[r0 + min(m, na - 1)];
        const uint16_t* xa = stage + tok * ldx + q * F::kCK;
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (int rd = 0; rd + 1 < rounds; ++rd) {
          const int ub = u0 + rd * NU;
          roll_round<FMT, NU>(r, acc, ub, u1, xa, st, ub + NU, u1, lane);
        }
        const Stream<FMT> sn = stream_of(nxt);
        roll_round<FMT, NU>(r, acc, u0 + (rounds - 1) * NU, u1, xa, sn, u0, u1, lane);
        st = sn;
        if (tid == 0) g.ticket[it & 1] = t_new;
        // (ends with every wave past a barrier: the ticket is visible)
        gate_up_epilogue<FMT, true>(a, red[it & 1], acc, w, lane, r0, na, ws, sub);
        ++count;
        cur = nxt;
        nxt = __builtin_amdgcn_readfirstlane(g.ticket[it & 1]);
        ++it;
        if (cur >= n2) break;
      }
    }
    // this workgroup's rows are written: count its items; and draw its first
    // output panel
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      if (count)
        __hip_atomic_fetch_add(f.ctl + kDone + kLine * grp, (unsigned)count, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
      g.ticket[0] = draw(f, kTicket3, grp);
    }
    __syncthreads();
  }

  // ---- output panels
  cur = __builtin_amdgcn_readfirstlane(g.ticket[0]);
  if (cur >= n3) return;   // whole workgroup
  const int nu = I / 128, nseg = (nu + NPER - 1) / NPER;   // segments of an expert
  const int n_slots = n_routed + f.NS;
  // first slot of chunk c: rows of a slot belong to the chunk of its first row
  auto chunk_slot = [&](int c) {
    int lo = 0, hi = n_slots;
    const int row = c * f.rows_per_chunk;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (g.slot_r0[mid] < row) lo = mid + 1;
      else hi = mid;
    }
    return __builtin_amdgcn_readfirstlane(lo);
  };
  Seg<FMT, NPER> ring[D];
  // segment i of this wave in an item over slots [j0, j1), panel p
  auto issue_item = [&](int d, int i, int j0, int j1, int p, bool live) {
    const int fl = w + kWaves * i, j = j0 + fl / nseg;
    const bool ok = live && j < j1;
    const int e = __builtin_amdgcn_readfirstlane(g.slot_e[ok ? j : 0]);
    issue_seg<FMT, NPER>(ring[d], f, e, ok, p, (fl % nseg) * NPER, lane);
  };
  int c = cur / hpan, p = cur - c * hpan;
  int j0 = chunk_slot(c), j1 = chunk_slot(c + 1);
#pragma unroll
  for (int d = 0; d < D; ++d) issue_item(d, d, j0, j1, p, true);
  __builtin_amdgcn_sched_barrier(0);

  // wait for every gate/up item: all are drawn (see the top)
  if (w == 0) {
    for (int n = 0;; ++n) {
      unsigned v = 0u;
      if (lane < 8)
        v = __hip_atomic_load(f.ctl + kDone + kLine * lane, __ATOMIC_RELAXED,
                              __HIP_MEMORY_SCOPE_AGENT);
      v += __shfl_xor(v, 1, kWave);
      v += __shfl_xor(v, 2, kWave);
      v += __shfl_xor(v, 4, kWave);
      if (__builtin_amdgcn_readfirstlane(v) == (unsigned)n2) break;
      if (n == kSpin) {
        if (lane == 0)
          __hip_atomic_store(f.ctl + kFlag, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        break;
      }
      __builtin_amdgcn_s_sleep(2);
    }
    // the second panel, drawn when every workgroup has come this far
    if (lane == 0) g.ticket[1] = draw(f, kTicket3, grp);
  }
  __syncthreads();
  nxt = __builtin_amdgcn_readfirstlane(g.ticket[1]);
  __syncthreads();   // read before an item's draw takes the word

  const int lda = I + 8, per_row = I / 8;
  const __amdgpu_buffer_rsrc_t ract = __builtin_amdgcn_make_buffer_rsrc(
      (void*)f.act, 0, (T * f.K + f.NS * T) * I * 2, kRawBufferFlags);
  int staged = -1, row0 = 0;
  while (true) {
    if (c != staged) {   // the chunk's activation rows, read at device scope
      if (staged >= 0) __syncthreads();   // the old chunk's are used
      staged = c;
      row0 = g.slot_r0[j0];
      const int pieces = (g.slot_r0[j1] - row0) * per_row;
      constexpr int SB = 8;
      for (int c0 = tid; c0 < pieces; c0 += SB * kThreads) {
        u32x4_t v[SB];
#pragma unroll
        for (int k = 0; k < SB; ++k)
          v[k] = __builtin_bit_cast(
              u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                           ract, (row0 * per_row + min(c0 + k * kThreads, pieces - 1)) * 16, 0,
                           kAuxDev));
#pragma unroll
        for (int k = 0; k < SB; ++k) {
          const int pc = c0 + k * kThreads;
          if (pc < pieces) {
            const int rr = pc / per_row;
            *reinterpret_cast<u32x4_t*>(stage + rr * lda + (pc - rr * per_row) * 8) = v[k];
          }
        }
      }
      __syncthreads();
    }
    if (tid == 0) t_new = draw(f, kTicket3, grp);
    // next item
    const bool more = nxt < n3;
    const int cn = more ? nxt / hpan : c, pn = more ? nxt - cn * hpan : p;
    const int jn0 = cn == c ? j0 : chunk_slot(cn), jn1 = cn == c ? j1 : chunk_slot(cn + 1);
    const int total = (j1 - j0) * nseg;
    const int rounds = ((total + kWaves - 1) / kWaves + D - 1) / D;
    f32x4_t tacc = {0.f, 0.f, 0.f, 0.f};   // tokens 4q + i, column m of the panel
    auto use_item = [&](int d, int i) {
      const int fl = w + kWaves * i;
      if (fl < total) {
        const int j = j0 + fl / nseg, sg = fl % nseg;
        const uint16_t* xa =
            stage + max((int)rowof[j * kMaxT + m] - row0, 0) * lda + q * F::kCK;
        f32x4_t pe = use_seg<FMT, NPER>(ring[d], sg * NPER, nu, xa);
        if constexpr (FMT == kNVFP4) {
          if (f.gs2) pe = pe * f.gs2[__builtin_amdgcn_readfirstlane(g.slot_e[j])];
        }
        const f32x4_t wv = *reinterpret_cast<const f32x4_t*>(wof + j * kMaxT + 4 * q);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tacc[k] = wv[k] != 0.f ? __builtin_fmaf(wv[k], pe[k], tacc[k]) : tacc[k];
      }
    };
    for (int rd = 0; rd + 1 < rounds; ++rd) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        use_item(d, rd * D + d);
        issue_item(d, (rd + 1) * D + d, j0, j1, p, true);
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (rounds > 0) use_item(d, (rounds - 1) * D + d);
      issue_item(d, d, jn0, jn1, pn, more);
    }
    // the waves' sums, in their order
    f32x4_t(*rd_)[kWave] = red[it & 1];
    rd_[w][lane] = tacc;
    if (tid == 0) g.ticket[it & 1] = t_new;
    __syncthreads();
    if (tid < 256) {
      const int tok = tid / 16, n = tid % 16;
      if (tok < T) {
        const int l = (tok / 4) * 16 + n, k = tok % 4;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) v += rd_[i][l][k];
        const long o = (long)tok * H + 16 * p + n;
        if (f.chunks > 1)
          __hip_atomic_store(f.part + (long)c * T * H + o, v, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
        else if (f.out_bf16)
          reinterpret_cast<uint16_t*>(f.out)[o] = f32_to_bf16(v);
        else
          reinterpret_cast<float*>(f.out)[o] = v;
      }
    }
    const int nn = __builtin_amdgcn_readfirstlane(g.ticket[it & 1]);
    ++it;
    if (f.chunks > 1) {
      // the last chunk of a panel to get here adds them all up, in order
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      if (tid == 0)
        g.last = __hip_atomic_fetch_add(f.ctl + kPanels + p, 1u, __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT) == (unsigned)f.chunks - 1;
      __syncthreads();
      if (g.last && tid < 256) {
        const int tok = tid / 16, n = tid % 16;
        if (tok < T) {
          const long o = (long)tok * H + 16 * p + n;
          float v = 0.f;
          for (int i = 0; i < f.chunks; ++i)
            v += __hip_atomic_load(f.part + (long)i * T * H + o, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
          if (f.out_bf16) reinterpret_cast<uint16_t*>(f.out)[o] = f32_to_bf16(v);
          else reinterpret_cast<float*>(f.out)[o] = v;
        }
      }
    }
    if (!more) break;
    c = cn;
    p = pn;
    j0 = jn0;
    j1 = jn1;
    nxt = nn;
  }
}

// ---------------------------------------------------------------- host

// bits: of a weight, with its scales.  More chunks than the LDS asks for give
// the output panels more items: where there are fewer panels than CUs, or their
// last round leaves CUs idle.  Times in us: a CU streams about 25 GB/s, an item
// costs 0.7 beside its stream, the joining of chunks 2.
inline bool make_plan(int T, int E, int K, int NS, int H, int I, float bits, bool groups,
                      Plan& p) {
  if (T < 1 || T > kMaxT || K < 1 || K > 16 || K > E || E > kMaxE || T * K > kMaxPairs ||
      NS < 0 || NS > kMaxShared || H < 256 || H % 256 || H > 16384 || I < 128 || I % 128 ||
      I > 16384)
    return false;
  const int slots = std::min(E, T * K) + NS, R = T * (K + NS);
  const size_t fixed = (size_t)2 * kWaves * kWave * 16 + sel_bytes() + table_bytes(slots) + 256;
  const size_t half = 80 * 1024, full = 160 * 1024;
  // x rows, and behind them select_any's scores
  const size_t xb = (size_t)T * (H + 8) * 2 + (groups ? (size_t)kWaves * E * 4 : 0);
  const size_t row = (size_t)(I + 8) * 2;
  if (fixed + xb > full) return false;
  const int cap = (int)((full - fixed) / row);
  int least = 1;
  if (cap < R) {   // a chunk's last slot may begin on its last row
    const int rpc = cap - (T - 1);
    if (rpc < 1) return false;
    least = (R + rpc - 1) / rpc;
  }
  const double active = E * (1.0 - std::pow(1.0 - (double)K / E, T)) + NS;
  const double panel_us = active * I * 16 * bits / 8 / 25e3;
  const int hpan = H / 16, cus = cu_count();
  double best = 1e30;
  for (int c = least; c <= std::min(least + 7, R); ++c) {
    const double t = (c * hpan + cus - 1) / cus * (panel_us / c + 0.7) + (c > 1 ? 2.0 : 0.0);
    if (t < best - 0.01) {
      best = t;
      p.chunks = c;
    }
  }
  p.rows_per_chunk = (R + p.chunks - 1) / p.chunks;
  const int rows = p.chunks == 1 ? R : p.rows_per_chunk + T - 1;
  p.stage = (std::max(xb, rows * row) + 15) / 16 * 16;
  p.occ = fixed + p.stage <= half ? 2 : 1;
  p.lds = p.stage + sel_bytes() + table_bytes(slots);
  return true;
}

template <int FMT, int NU>
void launch_router(const FewArgs& f, hipStream_t stream) {
  const int er = f.E + (f.sgate ? f.NS : 0);
  const int grid = f.n_sh + (er + f.rp - 1) / f.rp;
  few_router_kernel<FMT, NU><<<grid, kThreads, (size_t)f.T * (f.H + 8) * 2, stream>>>(f);
}

template <int FMT, int NU, int NPER>
void launch_experts(const FewArgs& f, const Plan& p, hipStream_t stream) {
  const long items = std::max<long>((long)std::min(f.E, f.T * f.K) * (f.I / 16),
                                    (long)p.chunks * (f.H / 16));
  const int grid = (int)std::min<long>((long)p.occ * cu_count(), items);
  if (p.occ == 2) few_experts_kernel<FMT, NU, NPER, 2><<<grid, kThreads, p.lds, stream>>>(f);
  else few_experts_kernel<FMT, NU, NPER, 1><<<grid, kThreads, p.lds, stream>>>(f);
}

template <int FMT, int NU>
hipError_t launch_nu(const FewArgs& f, const Plan& p, hipStream_t stream) {
  launch_router<FMT, NU>(f, stream);
  const hipError_t e = hipPeekAtLastError();
  if (e != hipSuccess) return e;
  if constexpr (FMT != kBF16) {
    if (f.I / 128 % 4 == 0) {
      launch_experts<FMT, NU, 4>(f, p, stream);
      return hipPeekAtLastError();
    }
  }
  launch_experts<FMT, NU, 2>(f, p, stream);
  return hipPeekAtLastError();
}

// Units of a wave's gate/up share that are in flight at once.
template <int FMT>
hipError_t launch_few(FewArgs f, const Plan& p, hipStream_t stream) {
  using F = WFmt<FMT>;
  f.w13_es = F::w_bytes(2L * f.I, f.H);
  f.s13_es = F::s_bytes(2L * f.I, f.H);
  f.w2_es = F::w_bytes(f.H, f.I);
  f.s2_es = F::s_bytes(f.H, f.I);
  const int units = (f.H / 128 + kKS - 1) / kKS;
  if constexpr (FMT == kMXFP4 || FMT == kNVFP4) {
    if (units > 8) return launch_nu<FMT, 16>(f, p, stream);
  }
  if constexpr (FMT != kBF16) {
    if (units > 4) return launch_nu<FMT, 8>(f, p, stream);
  }
  return launch_nu<FMT, 4>(f, p, stream);
}

}  // namespace

// one translation unit per weight format
hipError_t run_mxfp4(const FewArgs& f, const Plan& p, hipStream_t stream);
hipError_t run_nvfp4(const FewArgs& f, const Plan& p, hipStream_t stream);
hipError_t run_fp8(const FewArgs& f, const Plan& p, hipStream_t stream);
hipError_t run_bf16(const FewArgs& f, const Plan& p, hipStream_t stream);

}  // namespace few
}  // namespace xtu
