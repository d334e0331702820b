// The product with 4-bit weights for many rows of x (linear4.hpp has the formula and
// the layout).  A workgroup of 2 x 4 waves computes 128 rows of x times 64 NP rows of
// w, K in blocks of 128: a wave 64 rows times NP panels.  Its records go from memory
// to its registers, two blocks ahead, and become operands there: expanded in registers
// they take a quarter of the LDS traffic that bf16 tiles of w would, and a quarter of
// their bytes from memory, for being expanded by both waves of a column.  x goes
// straight to LDS, three stages (linear_tile.hip has the slots).  2048 x 2048 gated x
// 7168 MXFP4, one round of 256 tiles: 91 us, 1.32 PFLOP/s, MFMAs busy 54% of the cycles,
// other VALU instructions 44% (NVFP4 115 us, INT4 with groups of 128 121; 98, 125 and 130 on
// a card whose bf16 product of 8192 cubed reaches 1.34 PFLOP/s, not 1.42).
// Tiles of 128 x 128 in waves of 128 x 32, x by way of registers: 194.  The next
// operand expanded by quarters between the MFMAs of this one: 105.
#include "linear4.hpp"

namespace xtu {
namespace l4 {
namespace {

constexpr int kBM = 128, kMT = 4, kStages = 3, kNT = 512;
constexpr int kStage = kBM * 256, kLoads = kBM * 16 / kNT;   // bytes; per thread and stage

template <int FMT, int G, int AK, int NP>
__global__ __launch_bounds__(kNT, 2) void linear4_wide_kernel(Linear4Args a, int per, float* part) {
  constexpr bool GATED = AK == lin::kActSwiglu;
  constexpr int REC = record_bytes(FMT, G);
  constexpr int LW = NP * (1 + (FMT == kI4 ? 128 / G : 1));   // loads of a block's records
  constexpr int W = GATED ? 8 * NP : 16 * NP;                 // output columns of a wave
  constexpr int LD = 16 * NP + 4;                             // floats of an LDS row of sums
  static_assert(8 * 16 * LD * 4 <= kStages * kStage, "the epilogue's rows fit the stages");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const LinearArgs& e = a.e;
  const int tid = threadIdx.x, lane = tid % 64;
  const int w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int wn = w % 4, wm = w / 4, q = lane / 16, c = lane % 16;
  // contiguous ranges of tiles per XCD (workgroup b runs on XCD b % 8), eight m tiles
  // side by side so that concurrent workgroups share rows of both
  const int gm = (e.M + kBM - 1) / kBM, gn = (e.N + 4 * W - 1) / (4 * W), total = gm * gn;
  int t = blockIdx.x;
  {
    const int each = total / 8, rem = total % 8, x = t % 8;
    t = x * each + min(x, rem) + t / 8;
  }
  const int grp = t / (8 * gn), rows_g = min(8, gm - 8 * grp), in_g = t - grp * 8 * gn;
  const int m0 = (grp * 8 + in_g % rows_g) * kBM, tn = in_g / rows_g;
  const int nw = (tn * 4 + wn) * W;   // first output column of the wave
  const int nb = blocks_of(e.K);
  const int s0 = (int)blockIdx.y * per, s1 = min(nb, s0 + per);

  // panels past the last one read it again
  const int np = panels_of(e.N) * (GATED ? 2 : 1);
  const uint8_t* wp[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    int pan = (tn * 4 + wn) * NP + p;
    if (pan >= np) pan = GATED ? np - 2 + p % 2 : np - 1;
    wp[p] = a.w + (long)pan * nb * REC;
  }
  Raw<FMT, G> raw[2][NP];
  auto load_w = [&](int s, Raw<FMT, G> (&r)[NP]) {
    const long o = (long)min(s, s1 - 1) * REC;
#pragma unroll
    for (int p = 0; p < NP; ++p) r[p] = load_raw<FMT, G>(wp[p] + o, q, c, 4 * q);
  };
  // x: load j of a stage brings rows 32 j + 4 w and on, four a wave, a piece a lane
  const int mrows = min(kBM, e.M - m0);
  const u32x4_t xr = lin::raw_buffer(e.x + (long)m0 * e.ldx,
                                     (uint32_t)(((long)(mrows - 1) * e.ldx + e.K) * 2));
  uint32_t off[kLoads];
  const int xrow = 4 * w + lane / 16;
  const int kof = 8 * (lane % 16 ^ (xrow & 7) << 1);   // (rows 32 j on: the same & 7)
#pragma unroll
  for (int j = 0; j < kLoads; ++j)
    off[j] = (uint32_t)min(32 * j + xrow, mrows - 1) * (uint32_t)(e.ldx * 2) + 2 * kof;
  auto load_x = [&](int s) {
    const int sc = min(s, s1 - 1), st = (s - s0) % kStages;
    // (past the end the last block again, into a stage that no one reads)
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      lin::buf_to_lds(xr, kof < e.K - 128 * sc ? off[j] : 0x80000000u, (uint32_t)sc * 256u,
                      lds + st * kStage + (8 * j + w) * 1024);
  };
  f32x4_t acc[NP][kMT];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) acc[p][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  load_x(s0);
  load_w(s0, raw[0]);
  load_x(s0 + 1);
  load_w(s0 + 1, raw[1]);
  const int slot0 = (q ^ (c & 7) << 1) * 16;   // of place 4 j + q: j moves bits 2 and 3
  for (int s = s0; s < s1; s += 2) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      if (s + d >= s1) break;
      // block s + d of x landed: behind it only block s + d + 1's loads are in flight
      __builtin_amdgcn_s_waitcnt(lin::wait_vm(kLoads + LW));
      __syncthreads();   // all of it; and the stage of block s + d + 2 is read
      const uint8_t* xs = lds + (s + d - s0) % kStages * kStage + (64 * wm + c) * 256;
      multiply<FMT, G, NP, kMT>(
          raw[d], acc,
          [&](int j, int mt) {
            return *reinterpret_cast<const u32x4_t*>(xs + 16 * 256 * mt + (slot0 ^ 64 * j));
          },
          [&] { load_x(s + d + 2); });
      load_w(s + d + 2, raw[d]);
    }
  }
  __builtin_amdgcn_s_waitcnt(lin::wait_vm(0));   // (loads past the end)

  // Epilogue, 16 rows of x at a time: the wave lays its sums out as rows in its part
  // of LDS and takes them with consecutive lanes along a row.
  __syncthreads();
  const float g0 = a.gs ? a.gs[0] : 1.f, g1 = a.gs && GATED ? a.gs[1] : g0;
  float* eb = reinterpret_cast<float*>(lds) + w * (16 * LD);
  float* plane = part ? part + (long)blockIdx.y * lin::part_plane(e) : nullptr;
  constexpr int CG = W / 4, RS = 64 / CG, IT = 16 / RS;   // lanes of a row, rows at once, turns
  static_assert(RS <= 16, "a turn of at most 16 rows");
#pragma unroll 1
  for (int j = 0; j < kMT; ++j) {
    lin::lds_order();
#pragma unroll
    for (int jj = 0; jj < kMT; ++jj) {
      if (jj != j) continue;
#pragma unroll
      for (int p = 0; p < NP; ++p)
        *reinterpret_cast<f32x4_t*>(eb + c * LD + 16 * p + 4 * q) =
            acc[p][jj] * (GATED && p % 2 ? g1 : g0);
    }
    lin::lds_order();
    const int mb = m0 + 64 * wm + 16 * j;
    if (mb >= e.M) break;
    const auto place = [](int col) { return GATED ? col / 16 * 32 + col % 16 : col; };
    if (e.vec) {
      const int cv = lane % CG * 4, n = nw + cv, r = lane / CG;
      if (n >= e.N) continue;
      u32x4_t bz, bu;
      lin::load_bias4<AK>(e, n, bz, bu);
      // what the rows need is read before any is written
      lin::Row4 x[IT];
      if (!plane)
#pragma unroll
        for (int b = 0; b < IT; ++b) x[b] = lin::load_row4(e, min(mb + r + b * RS, e.M - 1), n);
      f32x4_t z[IT], u[IT];
#pragma unroll
      for (int b = 0; b < IT; ++b) {
        const float* row = eb + (r + b * RS) * LD + place(cv);
        z[b] = *reinterpret_cast<const f32x4_t*>(row);
        u[b] = z[b];
        if constexpr (GATED) u[b] = *reinterpret_cast<const f32x4_t*>(row + 16);
      }
      if (plane) {
#pragma unroll
        for (int b = 0; b < IT; ++b) {
          const int m = mb + r + b * RS;
          if (m >= e.M) break;
          float* pr = plane + (long)m * e.N * (GATED ? 2 : 1) + n;
          *reinterpret_cast<f32x4_t*>(pr) = z[b];
          if constexpr (GATED) *reinterpret_cast<f32x4_t*>(pr + e.N) = u[b];
        }
        continue;
      }
#pragma unroll
      for (int b = 0; b < IT; ++b) {
        z[b] += lin::of_raw4(bz, e.bias_bf16);
        if constexpr (GATED) u[b] += lin::of_raw4(bu, e.bias_bf16);
      }
      lin::act_all<AK>(e, z, u);
#pragma unroll
      for (int b = 0; b < IT; ++b) {
        const int m = mb + r + b * RS;
        if (m < e.M) lin::store_row4(e, m, n, z[b], x[b]);
      }
    } else {
#pragma unroll 1
      for (int i = lane; i < 16 * W; i += 64) {
        const int r = i / W, col = i % W, m = mb + r, n = nw + col;
        if (n >= e.N || m >= e.M) continue;
        const float z = eb[r * LD + place(col)], u = GATED ? eb[r * LD + place(col) + 16] : 0.f;
        if (plane) {
          float* pr = plane + (long)m * e.N * (GATED ? 2 : 1) + n;
          pr[0] = z;
          if constexpr (GATED) pr[e.N] = u;
        } else {
          lin::finish_one<AK>(e, m, n, z, u);
        }
      }
    }
  }
}

template <int NP>
hipError_t launch(const Linear4Args& a, int split, float* part, hipStream_t stream) {
  const LinearArgs& e = a.e;
  const int cols = 4 * (e.act == lin::kSwiglu ? 8 : 16) * NP, nb = blocks_of(e.K);
  const int per = (nb + split - 1) / split;
  split = (nb + per - 1) / per;   // no empty range
  const long tiles = ((long)e.M + kBM - 1) / kBM * (((long)e.N + cols - 1) / cols);
  if (!lin::grid_fits(tiles, kNT)) return hipErrorInvalidConfiguration;
  float* to = split > 1 ? part : nullptr;
  const hipError_t r = by_format(a, [&](auto fmt, auto group, auto g) {
    constexpr int F = decltype(fmt)::value, G = decltype(group)::value;
    if constexpr (NP == 4 && F == kI4 && G != 128) {
      return hipErrorInvalidValue;   // no room for its sums (not planned)
    } else {
      auto k = linear4_wide_kernel<F, G, lin::kActSwiglu, NP>;
      if constexpr (!decltype(g)::value)
        k = to || e.act == lin::kNone ? linear4_wide_kernel<F, G, lin::kActNone, NP>
                                      : linear4_wide_kernel<F, G, lin::kActOther, NP>;
      k<<<dim3((unsigned)tiles, (unsigned)split), kNT, kStages * kStage, stream>>>(a, per, to);
      return hipPeekAtLastError();
    }
  });
  if (r == hipSuccess && split > 1) return lin::launch_join(e, split, part, stream);
  return r;
}

}  // namespace

hipError_t launch4_wide(const Plan4& p, const Linear4Args& a, float* part, hipStream_t stream) {
  return p.kind == kWide4 ? launch<4>(a, p.split, part, stream) : launch<2>(a, p.split, part, stream);
}

}  // namespace l4
}  // namespace xtu
