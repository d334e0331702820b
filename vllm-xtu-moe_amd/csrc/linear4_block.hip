// The product with 4-bit weights for few rows of x or few units (linear4.hpp has the
// formula and the layout), every wave for itself.  A workgroup has one unit, two panels
// (swiglu: a gate and its up panel), times 4 LX rows of x; its waves deal the blocks of
// 128 k among them.  A wave brings its blocks of x straight to its own part of LDS, NB
// of them at a time, and waits for those alone: no barrier before the sums are added,
// in a fixed order.  What bounds it is x: a unit's rows of it come to every CU.  Loads
// that go to LDS come in at 40 to 65 KB a us and CU, loads to registers at 25 (the same
// kernel with x in registers, 47 x 7168 x 2048 NVFP4 14.2 us, 8.4 so; 64 x 7168 x 2048
// MXFP4 17.1 and 9.4; two panels also share x's operands).  16 x 7168 x 7168 NVFP4 13.3
// us, 9.9 with the weights in the caches.  Where units are fewer than CUs, x is split
// instead (block4_plan): w is read again, from the caches, and each CU takes in less.  In
// parts of 16 / 32 / 48 / 64 rows, MXFP4: 64 x 2048 x 7168 9.5 / 11.0 / 12.4 / 15.3 us,
// 128 x 2048 x 7168 16.6 / 11.9 / 13.0 / 15.7, 80 x 7168 x 2048 22.7 / 16.5 / 13.5 / 15.5,
// 128 x 4096 x 4096 24.2 / 15.9 / 16.5 / 12.7.
#include "linear4.hpp"

namespace xtu {
namespace l4 {
namespace {

template <int FMT, int G, int AK, int LX, int WV, int NB>
__global__ __launch_bounds__(64 * WV) void linear4_block_kernel(Linear4Args a) {
  constexpr bool GATED = AK == lin::kActSwiglu;
  constexpr int REC = record_bytes(FMT, G), COLS = GATED ? 16 : 32;
  constexpr int LW = 2 * (1 + (FMT == kI4 ? 128 / G : 1));   // loads of a block's records
  constexpr int MT = (LX + 3) / 4, SIZE = LX * 1024;          // its x: LX loads of four rows
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const LinearArgs& e = a.e;
  const int tid = threadIdx.x, lane = tid % 64;
  const int w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int q = lane / 16, c = lane % 16;
  const int nb = blocks_of(e.K), unit = blockIdx.x;
  const int m0 = 4 * LX * (int)blockIdx.y, rows = min(4 * LX, e.M - m0);
  const int last = panels_of(e.N) * (GATED ? 2 : 1) - 1;   // panel
  const int mine = (nb - w + WV - 1) / WV;                 // blocks w, w + WV, ..
  // x: load r of a block brings rows 4 r and on, a piece of 16 bytes a lane
  // (linear_tile.hip has the slots)
  const u32x4_t xr = lin::raw_buffer(e.x + (long)m0 * e.ldx,
                                     (uint32_t)(((long)(rows - 1) * e.ldx + e.K) * 2));
  uint8_t* xs = lds + w * (NB * SIZE);
  auto load_x = [&](int i) {
    const int s = w + WV * min(i, mine - 1);
#pragma unroll
    for (int r = 0; r < LX; ++r) {
      const int row = 4 * r + lane / 16, k = 8 * (lane % 16 ^ (row & 7) << 1);
      const uint32_t off = (uint32_t)min(row, rows - 1) * (uint32_t)(e.ldx * 2) + 2 * k;
      lin::buf_to_lds(xr, k < e.K - 128 * s ? off : 0x80000000u, (uint32_t)s * 256u,
                      xs + i % NB * SIZE + r * 1024);
    }
  };
  const uint8_t* wp[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) wp[p] = a.w + (long)min(2 * unit + p, last) * nb * REC;
  Raw<FMT, G> raw[2][2];
  auto load_w = [&](int i, Raw<FMT, G> (&r)[2]) {
    const long o = (long)(w + WV * min(i, mine - 1)) * REC;
#pragma unroll
    for (int p = 0; p < 2; ++p) r[p] = load_raw<FMT, G>(wp[p] + o, q, c, 4 * q);
  };
  // what the epilogue reads beside the sums: wave w finishes panel w % 2, rows 16 (w / 2)
  // (swiglu: rows 16 w)
  const int fp = GATED ? 0 : w % 2, fm = 16 * (GATED ? w : w / 2) + c;
  const int fn = unit * COLS + 16 * fp + 4 * q;
  const bool fin = (GATED ? w : w / 2) < MT && fm < rows && fn < e.N;
  u32x4_t bz = {0u, 0u, 0u, 0u}, bu = bz;
  lin::Row4 pre = {{0u, 0u, 0u, 0u}, 1.f};
  if (fin && e.vec) {
    lin::load_bias4<AK>(e, fn, bz, bu);
    pre = lin::load_row4(e, m0 + fm, fn);
  }
  const float g0 = a.gs ? a.gs[0] : 1.f, g1 = a.gs && GATED ? a.gs[1] : g0;

  f32x4_t acc[2][MT];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[p][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int xc = LX < 4 ? c % (4 * LX) : c;   // (rows past M repeat others: not written)
  const uint8_t* xl = xs + xc * 256;
  const int slot0 = (q ^ (xc & 7) << 1) * 16;   // of place 4 j + q: j moves bits 2 and 3
  if (mine > 0) {   // (loads past the end bring the last block again, where no one reads)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (n < NB) load_x(n);
      load_w(n, raw[n]);
    }
    for (int i = 0; i < mine; i += 2) {
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        if (i + d >= mine) break;
        // block i + d of x landed: behind it only the next one's loads are in flight
        __builtin_amdgcn_s_waitcnt(lin::wait_vm(NB == 2 ? LX + LW : LW));
        __asm__ __volatile__("" ::: "memory");
        const uint8_t* xb = xl + (NB == 2 ? d * SIZE : 0);
        multiply<FMT, G, 2, MT>(raw[d], acc, [&](int j, int mt) {
          return *reinterpret_cast<const u32x4_t*>(xb + 4096 * mt + (slot0 ^ 64 * j));
        });
        __asm__ __volatile__("s_waitcnt lgkmcnt(0)" ::: "memory");   // it is read
        load_x(i + d + NB);
        load_w(i + d + 2, raw[d]);
      }
    }
    __builtin_amdgcn_s_waitcnt(lin::wait_vm(0));
  }
  __syncthreads();   // every wave is done with x
  f32x4_t* red = reinterpret_cast<f32x4_t*>(lds);   // [WV][2][MT][64]
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) red[((w * 2 + p) * MT + mt) * 64 + lane] = acc[p][mt];
  __syncthreads();
  if (!fin) return;
  f32x4_t z[1] = {{0.f, 0.f, 0.f, 0.f}}, u[1] = {{0.f, 0.f, 0.f, 0.f}};
  const int mt = fm / 16;
#pragma unroll
  for (int k = 0; k < WV; ++k) {
    z[0] += red[((k * 2 + fp) * MT + mt) * 64 + lane];
    if constexpr (GATED) u[0] += red[((k * 2 + 1) * MT + mt) * 64 + lane];
  }
  z[0] *= g0;
  if constexpr (GATED) u[0] *= g1;
  if (e.vec) {
    z[0] += lin::of_raw4(bz, e.bias_bf16);
    if constexpr (GATED) u[0] += lin::of_raw4(bu, e.bias_bf16);
    lin::act_all<AK>(e, z, u);
    lin::store_row4(e, m0 + fm, fn, z[0], pre);
  } else {
#pragma unroll 1
    for (int t = 0; t < 4; ++t) {
      if (fn + t < e.N) lin::finish_one<AK>(e, m0 + fm, fn + t, z[0][0], u[0][0]);
      z[0] = __builtin_shufflevector(z[0], z[0], 1, 2, 3, 0);
      u[0] = __builtin_shufflevector(u[0], u[0], 1, 2, 3, 0);
    }
  }
}

template <int LX>
hipError_t launch(const Linear4Args& a, hipStream_t stream) {
  const LinearArgs& e = a.e;
  const int cols = e.act == lin::kSwiglu ? 16 : 32;
  const long units = ((long)e.N + cols - 1) / cols, parts = (e.M + 4 * LX - 1) / (4 * LX);
  return by_format(a, [&](auto fmt, auto group, auto g) {
    constexpr int F = decltype(fmt)::value, G = decltype(group)::value;
    // what LDS and the registers hold
    // (block4_waves)
    constexpr int MT = (LX + 3) / 4, WV = MT == 1 && !(F == kI4 && G == 32) ? 16 : 8, NB = MT <= 2 ? 2 : 1;
    constexpr size_t kX = (size_t)WV * NB * LX * 1024, kSums = (size_t)WV * MT * 2048;
    constexpr size_t kAll = kX > kSums ? kX : kSums;   // the sums take x's place
    static_assert(kAll <= 160 * 1024, "LDS of a CU");
    if (!lin::grid_fits(units * parts, 64 * WV)) return hipErrorInvalidConfiguration;
    auto k = linear4_block_kernel<F, G, decltype(g)::value ? lin::kActSwiglu : lin::kActOther, LX,
                                  WV, NB>;
    k<<<dim3((unsigned)units, (unsigned)parts), 64 * WV, kAll, stream>>>(a);
    return hipPeekAtLastError();
  });
}

}  // namespace

int block4_waves(const Shape4& s, int rows) {
  return rows <= 16 && !(s.fmt == kI4 && s.group == 32) ? 16 : 8;
}

hipError_t launch4_block(const Linear4Args& a, hipStream_t stream) {
  if (a.e.M > kBlockM) return hipErrorInvalidValue;
  const int rows = block4_plan(shape_of(a)).rows;
  if (rows == 4) return launch<1>(a, stream);
  if (rows == 8) return launch<2>(a, stream);
  if (rows == 16) return launch<4>(a, stream);
  if (rows == 32) return launch<8>(a, stream);
  if (rows == 48) return launch<12>(a, stream);
  return launch<16>(a, stream);
}

}  // namespace l4
}  // namespace xtu
