// The product with 4-bit weights for at most 16 rows of x (linear4.hpp has the
// formula and the layout): a stream of w.  All of x sits in LDS.  A unit is up to 16
// output columns (swiglu: of gate and up both); the waves of a workgroup deal its
// blocks of 128 k among them, their sums are added through LDS in a fixed order, and
// the workgroup takes further units in steps of the grid, with the next unit's first
// blocks already in flight.  Bound by HBM where there is much of w: 1 x 16384 gated x
// 7168 MXFP4 24 to 27 us (4.7 to 5.2 TB/s), 8 x 16384 x 7168 17.8.  Few columns: units of four or
// eight (the MFMA's other rows repeat the last one) put more CUs to work: 7 x 1171 x
// 1184 INT4 5.3 us.
#include "linear4.hpp"

namespace xtu {
namespace l4 {
namespace {

constexpr size_t kLds = 120 * 1024;
constexpr int kRowPad = 16;    // bf16 behind a row of x in LDS: rows 32 bytes apart in the banks

template <int FMT, int G, bool GATED, int WV, int U>
__global__ __launch_bounds__(64 * WV) void linear4_skinny_kernel(Linear4Args a, int rp) {
  constexpr int H = GATED ? 2 : 1, REC = record_bytes(FMT, G);
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ f32x4_t red[H][WV][64];
  const LinearArgs& e = a.e;
  const int tid = threadIdx.x, lane = tid % 64;
  const int w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int q = lane / 16, c = lane % 16;
  const int nb = blocks_of(e.K), per = 16 / rp;   // units of a panel
  const int units = panels_of(e.N) * per;
  const int steps = (nb + WV - 1) / WV;           // of a wave and unit
  Raw<FMT, G> raw[U][H];
  // block w + WV i of a unit (past the end the last one again, not used)
  auto load = [&](int unit, int i, Raw<FMT, G> (&r)[H]) {
    const int row = unit % per * rp;
    const uint8_t* rec = a.w + ((long)(unit / per) * H * nb + min(w + WV * i, nb - 1)) * REC;
#pragma unroll
    for (int h = 0; h < H; ++h)
      r[h] = load_raw<FMT, G>(rec + (long)h * nb * REC, q, row + min(c, rp - 1),
                              min(row + 4 * q, 12));
  };
  int unit = blockIdx.x;
#pragma unroll
  for (int i = 0; i < U; ++i) load(unit, min(i, steps - 1), raw[i]);
  __builtin_amdgcn_sched_barrier(0);   // x after the first loads of w
  // x to LDS, zeros behind K
  const int ldx = nb * 128 + kRowPad, pieces = nb * 16;
  uint16_t* xs = reinterpret_cast<uint16_t*>(lds);
  for (int p = tid; p < e.M * pieces; p += 64 * WV) {
    const int r = p / pieces, k8 = p - r * pieces;
    *reinterpret_cast<u32x4_t*>(xs + r * ldx + 8 * k8) = load_x8(a, e.x + (long)r * e.ldx, 8 * k8);
  }
  __syncthreads();
  const uint16_t* xl = xs + min(c, e.M - 1) * ldx + 8 * q;
  const float g0 = a.gs ? a.gs[0] : 1.f, g1 = a.gs && GATED ? a.gs[1] : g0;

  for (; unit < units; unit += gridDim.x) {
    const int next = min(unit + (int)gridDim.x, units - 1);
    f32x4_t acc[H][1];
#pragma unroll
    for (int h = 0; h < H; ++h) acc[h][0] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < steps; i0 += U) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int s = w + WV * (i0 + i);
        if (s < nb) {
          const uint16_t* xb = xl + 128 * s;
          multiply<FMT, G, H, 1>(raw[i], acc, [&](int j, int) {
            return *reinterpret_cast<const u32x4_t*>(xb + 32 * j);
          });
        }
        // what comes U steps later, or the next unit's step of this slot
        const bool more = i0 + U < steps;
        load(more ? unit : next, min(more ? i0 + U + i : i, steps - 1), raw[i]);
      }
    }
    __syncthreads();   // the sums of the unit before are read
#pragma unroll
    for (int h = 0; h < H; ++h) red[h][w][lane] = acc[h][0];
    __syncthreads();
    if (tid < 256) {
      const int t = tid / 64, nl = 4 * q + t, n = unit / per * 16 + unit % per * rp + nl;
      float z = 0.f, u = 0.f;
      if (c < e.M && nl < rp && n < e.N) {
#pragma unroll
        for (int k = 0; k < WV; ++k) {
          z += red[0][k][lane][t];
          if constexpr (GATED) u += red[H - 1][k][lane][t];
        }
        lin::finish_one<GATED ? lin::kActSwiglu : lin::kActOther>(e, c, n, z * g0, u * g1);
      }
    }
  }
}

template <int WV>
hipError_t launch(const Linear4Args& a, const SkinnyPlan& p, size_t lds, hipStream_t stream) {
  const bool one = WV < 16 || blocks_of(a.e.K) <= WV;   // a block per wave and unit
  return by_format(a, [&](auto fmt, auto group, auto g) {
    constexpr int F = decltype(fmt)::value, G = decltype(group)::value;
    constexpr bool GATED = decltype(g)::value;
    auto k = linear4_skinny_kernel<F, G, GATED, WV, 1>;
    if constexpr (WV == 16)
      if (!one) k = linear4_skinny_kernel<F, G, GATED, WV, 2>;
    k<<<(unsigned)p.grid, 64 * WV, lds, stream>>>(a, p.rows);
    return hipPeekAtLastError();
  });
}

size_t x_bytes(const Shape4& s) {
  return (size_t)s.M * ((size_t)blocks_of(s.K) * 128 + kRowPad) * 2;
}

}  // namespace

SkinnyPlan skinny4_plan(const Shape4& s) {
  SkinnyPlan p{4, 0, 0, 0};
  const size_t x = x_bytes(s);
  if (s.M > 16 || x > kLds) return p;
  // columns of a unit: about one unit per CU, 16 at most
  while (p.rows < 16 && (long)panels_of(s.N) * (16 / p.rows) > 256) p.rows *= 2;
  p.units = (long)panels_of(s.N) * (16 / p.rows);
  const int nb = blocks_of(s.K);
  p.waves = nb > 8 ? 16 : nb > 4 ? 8 : 4;
  const int fit = (int)(160 * 1024 / (x + (size_t)(s.gated ? 2 : 1) * p.waves * 1024));
  const long all = 256L * (fit < 32 / p.waves ? fit : 32 / p.waves);   // what is resident
  p.grid = p.units < all ? p.units : all;
  return p;
}

hipError_t launch4_skinny(const Linear4Args& a, hipStream_t stream) {
  const Shape4 s = shape_of(a);
  const SkinnyPlan p = skinny4_plan(s);
  if (p.grid == 0) return hipErrorInvalidValue;
  if (p.waves == 16) return launch<16>(a, p, x_bytes(s), stream);
  if (p.waves == 8) return launch<8>(a, p, x_bytes(s), stream);
  return launch<4>(a, p, x_bytes(s), stream);
}

}  // namespace l4
}  // namespace xtu
