// The product with 4-bit weights for up to 64 rows of x at any alignment and row stride
// (linear4.hpp has the formula and the layout): every wave for itself.  A unit is two
// panels (swiglu: a gate and its up panel) times all MT blocks of 16 rows; the waves of
// a workgroup deal its blocks of 128 k among them and their sums are added through LDS
// in a fixed order.  Neither operand is staged: a wave takes w and x straight into the
// MFMA's registers, U blocks ahead, and waits for no other wave before the sums.  (For
// rows that start on 16 bytes linear4_block.hip takes half of its time: 47 x 7168 x
// 2048 NVFP4 8.4 us, 14.2 here.)
#include "linear4.hpp"

namespace xtu {
namespace l4 {
namespace {

template <int FMT, int G, bool GATED, int MT, int WV, int U>
__global__ __launch_bounds__(64 * WV) void linear4_rows_kernel(Linear4Args a) {
  constexpr int AK = GATED ? lin::kActSwiglu : lin::kActOther, REC = record_bytes(FMT, G);
  constexpr int COLS = GATED ? 16 : 32;   // output columns of a unit
  __shared__ f32x4_t red[WV][2][MT][64];
  const LinearArgs& e = a.e;
  const int tid = threadIdx.x, lane = tid % 64;
  const int w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int q = lane / 16, c = lane % 16;
  const int nb = blocks_of(e.K), units = (e.N + COLS - 1) / COLS;
  const int last = panels_of(e.N) * (GATED ? 2 : 1) - 1;   // panel
  const int steps = (nb + WV - 1) / WV;   // of a wave and unit
  const uint16_t* xrow[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) xrow[mt] = e.x + (long)min(16 * mt + c, e.M - 1) * e.ldx + 8 * q;
  struct Slot {
    Raw<FMT, G> w[2];
    u32x4_t x[4][MT];
  };
  Slot slot[U];
  // block w + WV i of a unit (past the end the last one again, not used)
  auto load = [&](int unit, int i, Slot& r) {
    const int s = min(w + WV * i, nb - 1);
#pragma unroll
    for (int p = 0; p < 2; ++p)
      r.w[p] = load_raw<FMT, G>(a.w + ((long)min(2 * unit + p, last) * nb + s) * REC, q, c, 4 * q);
    if (a.xvec && 128 * (s + 1) <= e.K) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          r.x[j][mt] = *reinterpret_cast<const u32x4_t*>(xrow[mt] + 128 * s + 32 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          r.x[j][mt] = load_x8(a, xrow[mt] - 8 * q, 128 * s + 32 * j + 8 * q);
    }
  };
  int unit = blockIdx.x;
#pragma unroll
  for (int i = 0; i < U; ++i) load(unit, i, slot[i]);
  const float g0 = a.gs ? a.gs[0] : 1.f, g1 = a.gs && GATED ? a.gs[1] : g0;

  for (; unit < units; unit += gridDim.x) {
    const int next = min(unit + (int)gridDim.x, units - 1);
    // what the epilogue reads beside the sums: wave w finishes panel w % 2, rows 16 (w / 2)
    const int fp = GATED ? 0 : w % 2, fm = 16 * (GATED ? w : w / 2) + c;
    const int fn = unit * COLS + 16 * fp + 4 * q;
    const bool fin = (GATED ? w : w / 2) < MT && fm < e.M && fn < e.N;
    u32x4_t bz = {0u, 0u, 0u, 0u}, bu = bz;
    lin::Row4 pre = {{0u, 0u, 0u, 0u}, 1.f};
    if (fin && e.vec) {
      lin::load_bias4<AK>(e, fn, bz, bu);
      pre = lin::load_row4(e, fm, fn);
    }
    f32x4_t acc[2][MT];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[p][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < steps; i0 += U) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (w + WV * (i0 + i) < nb)
          multiply<FMT, G, 2, MT>(slot[i].w, acc, [&](int j, int mt) { return slot[i].x[j][mt]; });
        // what comes U steps later, or the next unit's step of this slot
        const bool more = i0 + U < steps;
        if (more || unit != next) load(more ? unit : next, more ? i0 + U + i : i, slot[i]);
      }
    }
    __syncthreads();   // the sums of the unit before are read
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) red[w][p][mt][lane] = acc[p][mt];
    __syncthreads();
    if (!fin) continue;
    f32x4_t z[1] = {{0.f, 0.f, 0.f, 0.f}}, u[1] = {{0.f, 0.f, 0.f, 0.f}};
    const int mt = fm / 16;
#pragma unroll
    for (int k = 0; k < WV; ++k) {
      z[0] += red[k][fp][mt][lane];
      if constexpr (GATED) u[0] += red[k][1][mt][lane];
    }
    z[0] *= g0;
    if constexpr (GATED) u[0] *= g1;
    if (e.vec) {
      z[0] += lin::of_raw4(bz, e.bias_bf16);
      if constexpr (GATED) u[0] += lin::of_raw4(bu, e.bias_bf16);
      lin::act_all<AK>(e, z, u);
      lin::store_row4(e, fm, fn, z[0], pre);
    } else {
#pragma unroll 1
      for (int t = 0; t < 4; ++t) {
        if (fn + t < e.N) lin::finish_one<AK>(e, fm, fn + t, z[0][0], u[0][0]);
        z[0] = __builtin_shufflevector(z[0], z[0], 1, 2, 3, 0);
        u[0] = __builtin_shufflevector(u[0], u[0], 1, 2, 3, 0);
      }
    }
  }
}

template <int MT>
hipError_t launch(const Linear4Args& a, hipStream_t stream) {
  const LinearArgs& e = a.e;
  const bool gated = e.act == lin::kSwiglu;
  const long units = ((long)e.N + (gated ? 15 : 31)) / (gated ? 16 : 32);
  return by_format(a, [&](auto fmt, auto group, auto g) {
    constexpr int F = decltype(fmt)::value, G = decltype(group)::value;
    constexpr bool GATED = decltype(g)::value;
    // what the registers hold: INT4's scales take four times the others' and more
    constexpr int WV = MT == 1 && F != kI4 ? 16 : 8, U = F == kI4 && MT >= 3 ? 1 : 2;
    constexpr long kGrid = 256 * (MT == 1 ? 16 / WV : 1);   // what is resident
    auto k = blocks_of(e.K) <= WV ? linear4_rows_kernel<F, G, GATED, MT, WV, 1>
                                  : linear4_rows_kernel<F, G, GATED, MT, WV, U>;
    k<<<(unsigned)(units < kGrid ? units : kGrid), 64 * WV, 0, stream>>>(a);
    return hipPeekAtLastError();
  });
}

}  // namespace

hipError_t launch4_rows(const Linear4Args& a, hipStream_t stream) {
  if (a.e.M > 64) return hipErrorInvalidValue;
  if (a.e.M <= 16) return launch<1>(a, stream);
  if (a.e.M <= 32) return launch<2>(a, stream);
  if (a.e.M <= 48) return launch<3>(a, stream);
  return launch<4>(a, stream);
}

}  // namespace l4
}  // namespace xtu
