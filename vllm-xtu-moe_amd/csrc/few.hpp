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
// for each half.  The MFMA's rows are the batch's tokens, the same x rows for
// every expert; a row is written where its token uses the expert.  Down: an item
// is 16 output columns over a range of K (a chunk) of all active experts; the
// eight waves take (expert, up to 4 x 128 k) segments in turn and multiply by the
// token's weight as they add up.  The chunk's part of the activation rows sits in
// LDS, and a workgroup stays with its chunk while that has panels left; with more
// than one chunk the chunks' sums go to memory and the last one to finish a panel
// adds them in chunk order, so results do not depend on timing.
// (They do depend on the batch, in the last bits: a token's experts are added in
// the order in which the batch's tokens bring them up.)
//
// Up to eight tokens leave half of the down projection's 16 MFMA rows unused:
// there every activation row is kept in two bf16 parts, the rounded value and the
// rest, and row t + 8 multiplies the rest.  That takes the rows' rounding (2^-9 of
// each value, as much as the output's own) out of the result, and matters most
// where a few large values make up an output (one token: up to 1.6 times the
// error of fp32 rows).  It costs the second part's place in LDS, so it is done
// where the rows fit with no other split into chunks (E = 512, H = 2048, I = 512,
// one token: 26 us either way; in more chunks, E = 256, H = 7168, I = 2048, two
// tokens: 101 us, 84 with one part).  Otherwise the rows are rounded to bf16, as
// everywhere else in this library.
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
  uint16_t* act;            // [parts][T K + NS T][I]: row t K + k, then T K + s T + t
  float* part;              // [chunks][T][H] (chunks > 1)
  unsigned* ctl;
  int ctl_words;
  int32_t* ids;
  float* wts;
  void* out;
  int out_bf16;
  int rp, n_sh;             // launch 1: router rows per panel; its shared gate/up items
  int epl;                  // experts per lane of the wave router (0: any E)
  int chunk_units, chunks;  // launch 2: 128-k units of a chunk of the down projection
  int parts;                // bf16 parts of an activation row
  size_t stage_bytes;
};

// LDS and chunk plan of launch 2.  Two workgroups share a CU where the x rows
// and all activation rows fit half its LDS; otherwise one takes what it needs.
struct Plan {
  size_t stage, lds;
  int nper, chunk_units, chunks, occ, parts;
};

namespace {

constexpr int kMaxT = 16, kMaxPairs = 256, kMaxShared = 4, kMaxE = 1024, kMaxGroups = 64;
constexpr int kThreads = 512, kWaves = 8, kKS = 4;   // waves along K per gate/up half
constexpr int kLine = 64;                            // words of a counter's own 256 bytes

// Counters (words): per group the gate/up items drawn and those done; per chunk
// and group the output panels drawn; then the chunks done per output panel.
constexpr int kGroups = 8, kMaxChunks = 8;
constexpr int kTicket = 0, kDone = kGroups * kLine, kTicket3 = 2 * kGroups * kLine,
              kPanels = kTicket3 + kMaxChunks * kGroups * kLine;
// Looks at the counters before a wait is given up: a look takes 0.27 us with one
// workgroup looking, 0.30 with 256, so about 0.3 s (the wait ends by itself as long
// as the workgroups that run make progress).
constexpr int kSpin = 1 << 20;

// Column col of activation row `row`, in its parts; read by other workgroups in
// the same launch.
__device__ __forceinline__ void store_act(const FewArgs& f, int row, int col, float v) {
  uint16_t* p = f.act + (long)row * f.I + col;
  const uint16_t hi = f32_to_bf16(v);
  __hip_atomic_store(p, hi, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (f.parts == 2) {
    const float rest = v - bf16_to_f32(hi);   // (no number where v is none: hi says so)
    __hip_atomic_store(p + (long)f.T * (f.K + f.NS) * f.I,
                       f32_to_bf16(fabsf(rest) < INFINITY ? rest : 0.f), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  }
}


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

// SwiGLU of a gate/up panel from the K splits' sums, added in their order:
// thread tid < 256 takes token tid / 16, column tid % 16 (row < 0: none).
template <int FMT>
__device__ __forceinline__ void finish_act(const FewArgs& f, const f32x4_t (*red)[kWave], int e,
                                           int row, int sub, int tid) {
  if (tid >= 256 || row < 0) return;
  const int t = tid / 16, n = tid % 16, l = (t / 4) * 16 + n, i = t % 4;
  float gv = 0.f, uv = 0.f;
#pragma unroll
  for (int k = 0; k < kKS; ++k) {
    gv += red[k][l][i];
    uv += red[kKS + k][l][i];
  }
  if constexpr (FMT == kNVFP4) {
    if (f.gs13) {
      gv *= f.gs13[2 * e];
      uv *= f.gs13[2 * e + 1];
    }
  }
  store_act(f, row, 16 * sub + n, silu_gate(gv, uv, f.limit, f.alpha, f.beta));
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
    a.w_estride = f.w13_es;
    a.s_estride = f.s13_es;
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
    red[w][lane] = acc;
    __syncthreads();
    finish_act<FMT>(f, red, ws, tid / 16 < f.T ? f.T * f.K + sh * f.T + tid / 16 : -1, sub, tid);
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
// l, l + 64, .. as order-preserving keys in kb, E words of this wave's own): K
// rounds of a wave-wide maximum, equal keys to the lowest index.  Scores, group
// scores and weights are route_token_wave's, in the same fp32 sequences (the sum
// over all experts, where the weights are not renormalised, lane by lane).
__device__ __forceinline__ void select_any(const FewArgs& f, const float* l, int lane,
                                           int* ids_lds, float* wts_lds, uint32_t* kb) {
#pragma clang fp contract(off)
  const int E = f.E, K = f.K;
#pragma unroll 1
  for (int e = lane; e < E; e += kWave) {
    float sc = l[e];
    if (f.mode == 1) sc = xtu_sigmoid(sc) + (f.bias ? f.bias[e] : 0.0f);
    kb[e] = max(tiny::score_key(sc), 1u);   // 0: taken, or not in a kept group
  }
  if (f.mode == 1 && f.n_group > 1) {
    // group score: the two best of the group, added; the topk_group best stay
    tiny::lds_wave_order();
    const int gsz = E / f.n_group;
    float gs = 0.f;
    if (lane < f.n_group) {
      uint32_t k1 = 0u, k2 = 0u;
#pragma unroll 1
      for (int j = 0; j < gsz; ++j) {
        const uint32_t k = kb[lane * gsz + j];
        k2 = max(k2, min(k1, k));
        k1 = max(k1, k);
      }
      const auto value = [](uint32_t k) {
        return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
      };
      gs = gsz >= 2 ? value(k1) + value(k2) : value(k1);
    }
    int r = 0;
#pragma unroll 1
    for (int j = 0; j < f.n_group; ++j) {
      const float o = tiny::readlane_f(gs, j);
      r += (o > gs || (o == gs && j < lane)) ? 1 : 0;
    }
    const unsigned long long kept = __ballot(lane < f.n_group && r < f.topk_group);
    tiny::lds_wave_order();
#pragma unroll 1
    for (int e = lane; e < E; e += kWave)
      if (!((kept >> (e / gsz)) & 1ull)) kb[e] = 0u;
  }
  int my_e = 0;
#pragma unroll 1
  for (int k = 0; k < K; ++k) {
    tiny::lds_wave_order();
    uint32_t best = 0u;
    int be = 0;
#pragma unroll 1
    for (int e = lane; e < E; e += kWave) {
      const uint32_t v = kb[e];
      if (v > best) {   // equal keys: the lower index
        best = v;
        be = e;
      }
    }
    const uint32_t top = tiny::wave_max_u32(best);
    // the lowest index of the lanes that hold the maximum (none left, which NaN
    // groups can bring about: expert k)
    const uint32_t inv = top && best == top ? (uint32_t)(kMaxE - be) : 0u;
    const int e = top ? kMaxE - (int)tiny::wave_max_u32(inv) : k;
    if (lane == k) my_e = e;
    if (lane == 0) kb[e] = 0u;
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
// active expert: the routed ones in the order of their first pairs, then the
// shared ones.
struct Sel {
  int ids[kMaxPairs];                        // of pair t K + k
  float wts[kMaxPairs];
  unsigned long long first[kMaxPairs / kWave];   // pairs that are their expert's first
  int slot_e[kMaxPairs + kMaxShared];
  int ticket[2];
  int last;
  int late;        // the wait for the gate/up items ran out
};

// One thread of a workgroup draws an item of group g: which = kTicket (gate/up),
// or for the output panels of chunk c kTicket3 + c * kGroups * kLine.
__device__ __forceinline__ int draw(const FewArgs& f, int which, int g) {
  return kGroups * (int)__hip_atomic_fetch_add(f.ctl + which + kLine * g, 1u, __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT) + g;
}

// rowof / wof: [slot][16] activation row and weight of token t in that slot
// (weight 0: the token does not use it).  stage gets the x rows; scr: E words
// per wave for select_any.  Returns the routed slots.  The workgroup's
// first two items are drawn on the way, the second once the first is back: by
// then every workgroup has drawn its first, so work spreads over all of them
// before anyone takes a second item.
__device__ __forceinline__ int build_selection(const FewArgs& f, Sel& g, uint16_t* rowof,
                                               float* wof, uint16_t* stage, uint32_t* scr) {
  const int tid = threadIdx.x, lane = tid % kWave, wv = wave_id();
  const int T = f.T, K = f.K, A = T * K, NS = f.NS;
  const bool drawer = tid == kThreads - kWave;
  const int grp = blockIdx.x % kGroups;
  int t0 = 0;
  if (drawer) t0 = draw(f, kTicket, grp);
  stage_x(f, stage);
  const int max_slots = min(f.E, A) + NS;
  for (int i = tid; i < max_slots * kMaxT; i += kThreads) {
    rowof[i] = 0;
    wof[i] = 0.f;
  }
  if (tid < kMaxPairs && tid >= A) g.ids[tid] = -1;
  if (tid == 0) g.late = 0;
  for (int t = wv; t < T; t += kWaves) {
    const float* l = f.logits + (long)t * f.ldl;
    int* ids = g.ids + t * K;
    float* wts = g.wts + t * K;
    switch (f.epl) {
      case 2: select_wave<2>(f, l, lane, ids, wts); break;
      case 4: select_wave<4>(f, l, lane, ids, wts); break;
      case 8: select_wave<8>(f, l, lane, ids, wts); break;
      default:
        select_any(f, l, lane, ids, wts, scr + wv * f.E);
    }
  }
  if (drawer) {
    g.ticket[0] = t0;
    __asm__ __volatile__("" ::"v"(t0) : "memory");   // the first item is back
    g.ticket[1] = draw(f, kTicket, grp);
  }
  __syncthreads();
  // thread p: pair p; its expert's first pair
  int fp = tid, e = 0;
  if (tid < A) {
    e = g.ids[tid];
    const int q1 = (tid + 3) / 4;
#pragma unroll 4
    for (int j = q1 - 1; j >= 0; --j) {
      const i32x4_t v = *reinterpret_cast<const i32x4_t*>(g.ids + 4 * j);
#pragma unroll
      for (int i = 3; i >= 0; --i)
        if (v[i] == e) fp = min(fp, 4 * j + i);
    }
  }
  const unsigned long long mine = __ballot(tid < A && fp == tid);
  if (lane == 0 && wv < kMaxPairs / kWave) g.first[wv] = mine;
  __syncthreads();
  int n = 0, slot = 0;   // slots in all; slots before pair fp's
#pragma unroll
  for (int i = 0; i < kMaxPairs / kWave; ++i) {
    const unsigned long long mk = g.first[i];
    const int c = __popcll(mk);
    n += c;
    slot += fp >= kWave * (i + 1) ? c
            : fp > kWave * i      ? __popcll(mk & ((1ull << (fp - kWave * i)) - 1))
                                  : 0;
  }
  if (tid < A) {
    const int t = tid / K;
    rowof[slot * kMaxT + t] = (uint16_t)tid;
    wof[slot * kMaxT + t] = g.wts[tid];
    if (fp == tid) g.slot_e[slot] = e;
  } else if (wv == kWaves - 1) {   // the shared experts' slots, behind the routed ones
    if (lane < NS) g.slot_e[n + lane] = f.E + lane;
    for (int s = 0; s < NS; ++s)
      if (lane < T) {
        rowof[(n + s) * kMaxT + lane] = (uint16_t)(A + s * T + lane);
        wof[(n + s) * kMaxT + lane] =
            f.sgate ? xtu_sigmoid(f.logits[(long)lane * f.ldl + f.E + s]) : 1.0f;
      }
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(n);
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
        sr, (int)lane * 16 + (off & 8), (u0 / F::kUG) * 1024, 0);   // cached: chunks share lines
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
  return FMT == kBF16   ? 2
         : FMT == kFP8  ? (NPER == 4 ? 2 : 4)
         : FMT == kNVFP4 ? (NPER == 4 ? 2 : 4)
                         : (NPER == 4 ? 4 : 6);
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
  const int n_routed = build_selection(
      f, g, rowof, wof, stage, reinterpret_cast<uint32_t*>(dyn + (size_t)T * (H + 8) * 2));
  if (blockIdx.x == 0) {
    for (int i = tid; i < T * f.K; i += kThreads) {
      f.ids[i] = g.ids[i];
      f.wts[i] = g.wts[i];
    }
  }
  int cur = __builtin_amdgcn_readfirstlane(g.ticket[0]);
  int nxt = __builtin_amdgcn_readfirstlane(g.ticket[1]);
  __syncthreads();   // the words are read before an item's draw takes one
  const int npan = I / 16, hpan = H / 16;
  const int n2 = n_routed * npan;
  const int grp = blockIdx.x % kGroups;
  int chunk = blockIdx.x / kGroups % f.chunks;   // of the down projection
  int t_new = 0;
  int it = 0;   // items done: which half of red, which ticket word

  // ---- routed gate/up
  {
    DecodeArgs a{};
    a.w = f.w13;
    a.s = f.s13;
    a.w_estride = f.w13_es;
    a.s_estride = f.s13_es;
    const int half = w / kKS, ks = w % kKS, nunits = H / 128;
    const int u0 = ks * nunits / kKS, u1 = (ks + 1) * nunits / kKS;
    const int rounds = max((u1 - u0 + NU - 1) / NU, 1);
    auto stream_of = [&](int item) {
      const bool live = item < n2;
      const int slot = live ? item / npan : 0, sub = live ? item - slot * npan : 0;
      const int e = __builtin_amdgcn_readfirstlane(g.slot_e[slot]);
      return make_stream<FMT>(a, e, half ? npan + sub : sub, H, live);
    };
    const uint16_t* xa = stage + min(m, T - 1) * (H + 8) + q * F::kCK;
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
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
        // (one copy of the round's code: what is run through once costs more to
        // fetch than to run)
#pragma unroll 1
        for (int rd = 0; rd < rounds; ++rd) {
          const int ub = u0 + rd * NU;
          const bool last = rd + 1 == rounds;
          if (last) st = stream_of(nxt);
          roll_round<FMT, NU>(r, acc, ub, u1, xa, st, last ? u0 : ub + NU, u1, lane);
        }
        if (tid == 0) g.ticket[it & 1] = t_new;
        // the rows of the tokens that use the expert
        f32x4_t(*rd_)[kWave] = red[it & 1];
        rd_[w][lane] = acc;
        __syncthreads();
        const int t = tid / 16 % kMaxT;
        finish_act<FMT>(f, rd_, g.slot_e[slot],
                        t < T && wof[slot * kMaxT + t] != 0.f ? rowof[slot * kMaxT + t] : -1, sub,
                        tid);
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
      g.ticket[0] = draw(f, kTicket3 + chunk * kGroups * kLine, grp);
    }
    __syncthreads();
  }

  // ---- output panels
  const int nu = I / 128, n_slots = n_routed + f.NS, cun = f.chunk_units;
  const int parts = f.parts, lda = cun * 128 + 8;
  const int rows = parts * T * (f.K + f.NS);
  // MFMA row m: token m & tmask, of part m / 8 if there are two
  const int tmask = parts == 2 ? 7 : 15, part_row = parts == 2 && m >= 8 ? rows / 2 : 0;
  const __amdgpu_buffer_rsrc_t ract = __builtin_amdgcn_make_buffer_rsrc(
      (void*)f.act, 0, rows * I * 2, kRawBufferFlags);
  Seg<FMT, NPER> ring[D];
  bool waited = false;
  // the own chunk first, then what the others have left
  for (int tries = 0; tries < f.chunks; ++tries, chunk = (chunk + 1) % f.chunks) {
    const int which = kTicket3 + chunk * kGroups * kLine;
    if (tries) {
      __syncthreads();
      if (tid == 0) g.ticket[0] = draw(f, which, grp);
      __syncthreads();
    }
    int p = __builtin_amdgcn_readfirstlane(g.ticket[0]);
    if (p >= hpan) continue;
    // segment i of this wave in a panel: all slots, nseg each
    const int units = min(cun, nu - chunk * cun), nseg = (units + NPER - 1) / NPER;
    const int total = n_slots * nseg;
    const int rounds = ((total + kWaves - 1) / kWaves + D - 1) / D;
    auto issue_item = [&](int d, int i, int pn, bool live) {
      const int fl = w + kWaves * i, j = fl / nseg;
      const bool ok = live && j < n_slots;
      const int e = __builtin_amdgcn_readfirstlane(g.slot_e[ok ? j : 0]);
      issue_seg<FMT, NPER>(ring[d], f, e, ok, pn, chunk * cun + (fl - j * nseg) * NPER, lane);
    };
#pragma unroll
    for (int d = 0; d < D; ++d) issue_item(d, d, p, true);
    __builtin_amdgcn_sched_barrier(0);
    if (!waited) {
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
            if (lane == 0) g.late = 1;
            break;
          }
          __builtin_amdgcn_s_sleep(2);
        }
      }

      waited = true;
    }
    // the second panel: drawn when every workgroup has come this far
    if (tid == 0) g.ticket[1] = draw(f, which, grp);
    __syncthreads();   // the wait is over for all; the old chunk's rows are used
    {   // the rows' part of the chunk, read at device scope
      const int per_row = units * 16, pieces = rows * per_row;
      constexpr int SB = 8;
      for (int c0 = tid; c0 < pieces; c0 += SB * kThreads) {
        u32x4_t v[SB];
        int at[SB];
#pragma unroll
        for (int k = 0; k < SB; ++k) {
          const int pc = min(c0 + k * kThreads, pieces - 1);
          const int rr = pc / per_row, kk = (pc - rr * per_row) * 8;
          at[k] = rr * lda + kk;
          v[k] = __builtin_bit_cast(
              u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                           ract, (rr * I + chunk * cun * 128 + kk) * 2, 0, kAuxDev));
        }
#pragma unroll
        for (int k = 0; k < SB; ++k)
          if (c0 + k * kThreads < pieces) *reinterpret_cast<u32x4_t*>(stage + at[k]) = v[k];
      }
    }
    int next = __builtin_amdgcn_readfirstlane(g.ticket[1]);
    __syncthreads();
    while (true) {
      if (tid == 0) t_new = next < hpan ? draw(f, which, grp) : hpan;
      const bool more = next < hpan;
      f32x4_t tacc = {0.f, 0.f, 0.f, 0.f};   // tokens 4q + i, column m of the panel
      auto use_item = [&](int d, int i) {
        const int fl = w + kWaves * i;
        if (fl < total) {
          const int j = fl / nseg, u0 = (fl - j * nseg) * NPER;   // within the chunk
          const int row = (int)rowof[j * kMaxT + (m & tmask)] + part_row;
          const uint16_t* xa = stage + row * lda + q * F::kCK;
          f32x4_t pe = use_seg<FMT, NPER>(ring[d], u0, units, xa);
          if constexpr (FMT == kNVFP4) {
            if (f.gs2) pe = pe * f.gs2[__builtin_amdgcn_readfirstlane(g.slot_e[j])];
          }
          const f32x4_t wv = *reinterpret_cast<const f32x4_t*>(wof + j * kMaxT + (4 * q & tmask));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tacc[k] = wv[k] != 0.f ? __builtin_fmaf(wv[k], pe[k], tacc[k]) : tacc[k];
        }
      };
#pragma unroll 1
      for (int rd = 0; rd < rounds; ++rd) {
        const bool last = rd + 1 == rounds;
        const int pn = last && more ? next : p, base = last ? 0 : (rd + 1) * D;
#pragma unroll
        for (int d = 0; d < D; ++d) {
          use_item(d, rd * D + d);
          issue_item(d, base + d, pn, !last || more);
        }
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
          if (parts == 2) {
            float rest = 0.f;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) rest += rd_[i][l + 32][k];
            v += rest;
          }
          if (g.late) v = NAN;   // rows may be missing: no answer that looks like one
          const long o = (long)tok * H + 16 * p + n;
          if (f.chunks > 1)
            __hip_atomic_store(f.part + (long)chunk * T * H + o, v, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
          else if (f.out_bf16)
            reinterpret_cast<uint16_t*>(f.out)[o] = f32_to_bf16(v);
          else
            reinterpret_cast<float*>(f.out)[o] = v;
        }
      }
      const int after = __builtin_amdgcn_readfirstlane(g.ticket[it & 1]);
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
      p = next;
      next = after;
    }
  }
}


// ---------------------------------------------------------------- host

// bits: of a weight, with its scales.  A segment is four units where the LDS
// holds all rows of four units and their number divides (BF16: two, by its
// registers).  More chunks than the LDS asks for give the output panels more
// items: where there are fewer panels than CUs, or their last round leaves CUs
// idle.  Times in us: a CU streams about 25 GB/s, an item costs 0.7 beside its
// stream, the joining of chunks 2.
__host__ inline bool plan_parts(int T, int E, int K, int NS, int H, int I, float bits, int parts,
                                Plan& p) {
  if (T < 1 || T > kMaxT || K < 1 || K > 16 || K > E || E > kMaxE || T * K > kMaxPairs ||
      NS < 0 || NS > kMaxShared || H < 256 || H % 256 || H > 16384 || I < 128 || I % 128 ||
      I > 16384)
    return false;
  const int slots = std::min(E, T * K) + NS, R = parts * T * (K + NS), nu = I / 128;
  const size_t fixed = (size_t)2 * kWaves * kWave * 16 + sel_bytes() + table_bytes(slots) + 256;
  const size_t half = 80 * 1024, full = 160 * 1024;
  // x rows, and behind them select_any's keys
  const size_t xb = (size_t)T * (H + 8) * 2 + (size_t)kWaves * E * 4;
  if (fixed + xb > full) return false;
  const auto stage_of = [&](int units) { return (size_t)R * (units * 128 + 8) * 2; };
  p.nper = bits < 16.0f && nu % 4 == 0 && fixed + stage_of(4) <= full ? 4 : 2;
  const double active = E * (1.0 - std::pow(1.0 - (double)K / E, T)) + NS;
  const double panel_us = active * I * 16 * bits / 8 / 25e3;
  const int hpan = H / 16, cus = cu_count();
  double best = 1e30;
  for (int units = (nu + p.nper - 1) / p.nper * p.nper; units >= p.nper; units -= p.nper) {
    if (fixed + stage_of(std::min(units, nu)) > full) continue;
    const int c = (nu + units - 1) / units;
    if (c > kMaxChunks) break;
    const double t = (c * hpan + cus - 1) / cus * (panel_us / c + 0.7) + (c > 1 ? 2.0 : 0.0);
    if (t < best - 0.01) {
      best = t;
      p.chunks = c;
      p.chunk_units = std::min(units, nu);
    }
  }
  if (best > 1e29) return false;
  p.stage = (std::max(xb, stage_of(p.chunk_units)) + 15) / 16 * 16;
  // two workgroups on a CU where LDS allows and they have about an item each;
  // with more, half as many workgroups end closer together
  p.occ = fixed + p.stage <= half && (active - NS) * (I / 16) <= 2.0 * cus ? 2 : 1;
  p.lds = p.stage + sel_bytes() + table_bytes(slots);
  p.parts = parts;
  return true;
}

__host__ inline bool make_plan(int T, int E, int K, int NS, int H, int I, float bits, Plan& p) {
  if (!plan_parts(T, E, K, NS, H, I, bits, 1, p)) return false;
  Plan two;
  if (T <= 8 && plan_parts(T, E, K, NS, H, I, bits, 2, two) && two.chunks == p.chunks &&
      two.nper == p.nper && two.occ == p.occ)
    p = two;
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
    if (p.nper == 4) {
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
