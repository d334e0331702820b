// The product with 4-bit weights on tiles of 64 rows of x, at any alignment and row
// stride (linear4.hpp has the formula and the layout): for rows that do not start on 16
// bytes where there is no workspace to copy them to, or that are too far apart for
// 32-bit offsets.  Four waves, each with two panels of w times all of the tile's rows, K
// in blocks of 128.  A wave's records go from memory to its registers, two blocks ahead,
// and are made operands there; x goes through registers to LDS, which all waves read, one
// block ahead.  2048 x 4096 x 7168 MXFP4 at odd 2-byte addresses 265 us (copied first and
// in linear4_wide.hip 107).
#include "linear4.hpp"

namespace xtu {
namespace l4 {
namespace {

constexpr int kAhead = 2;   // blocks of w in registers

// Eight k of a row of x at any 2-byte address (one load, which the hardware splits where
// it has to), zeros past K.
__device__ __forceinline__ u32x4_t load_any8(const Linear4Args& a, const uint16_t* row, int k) {
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (k < a.e.K) __builtin_memcpy(&v, row + k, 16);   // (K % 8 == 0)
  return v;
}

template <int FMT, int G, bool GATED, int MT, int NP>
__global__ __launch_bounds__(256) void linear4_tile_kernel(Linear4Args a) {
  constexpr int AK = GATED ? lin::kActSwiglu : lin::kActOther;
  constexpr int BM = 16 * MT, REC = record_bytes(FMT, G);
  constexpr int W = GATED ? 8 * NP : 16 * NP;   // output columns of a wave
  constexpr int LD = 16 * NP + 4;               // floats of an LDS row of sums
  constexpr int STAGE = BM * 256, EPI = 4 * 16 * LD * 4;
  static_assert(!GATED || NP % 2 == 0, "a wave has gate panels with their up panels");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE > EPI ? 2 * STAGE : EPI];
  const LinearArgs& e = a.e;
  const int tid = threadIdx.x, lane = tid % 64;
  const int w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int q = lane / 16, c = lane % 16;
  const int gm = (e.M + BM - 1) / BM, gn = (e.N + 4 * W - 1) / (4 * W), total = gm * gn;
  // contiguous ranges of tiles per XCD (workgroup b runs on XCD b % 8), m tiles of the
  // same columns side by side
  int t = blockIdx.x;
  {
    const int each = total / 8, rem = total % 8, x = t % 8;
    t = x * each + min(x, rem) + t / 8;
  }
  const int m0 = t % gm * BM, tn = t / gm;
  const int nw = (tn * 4 + w) * W;   // first output column of the wave
  const int nb = blocks_of(e.K);
  const int s0 = 0, s1 = nb;

  // panels past the last one read it again
  const int np = panels_of(e.N) * (GATED ? 2 : 1);
  const uint8_t* wp[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    int pan = (tn * 4 + w) * NP + p;
    if (pan >= np) pan = GATED ? np - 2 + p % 2 : np - 1;
    wp[p] = a.w + (long)pan * nb * REC;
  }
  Raw<FMT, G> raw[kAhead][NP];
  auto load_w = [&](int s, Raw<FMT, G> (&r)[NP]) {
    const long o = (long)min(s, s1 - 1) * REC;
#pragma unroll
    for (int p = 0; p < NP; ++p) r[p] = load_raw<FMT, G>(wp[p] + o, q, c, 4 * q);
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d) load_w(s0 + d, raw[d]);

  // x: thread t stages piece t % 16 of rows t / 16, + 16, ..
  const int xp = tid % 16, xr = tid / 16;
  const uint16_t* xrow[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    xrow[i] = e.x + (long)min(m0 + 16 * i + xr, e.M - 1) * e.ldx;
  u32x4_t xv[MT];
  auto load_x = [&](int s) {
#pragma unroll
    for (int i = 0; i < MT; ++i) xv[i] = load_any8(a, xrow[i], 128 * s + 8 * xp);
  };
  // (16 lanes that read a block's rows at one place touch all banks: linear_tile.hip)
  const auto slot = [](int place, int row) { return (place ^ (row & 7) << 1) * 16; };
  auto store_x = [&](int st) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
      *reinterpret_cast<u32x4_t*>(lds + st * STAGE + (16 * i + xr) * 256 +
                                  slot(xp, xr)) = xv[i];
  };
  f32x4_t acc[NP][MT];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[p][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  load_x(s0);
  store_x(0);
  for (int s = s0; s < s1; s += kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      if (s + d >= s1) break;
      const int st = (s + d - s0) & 1;
      if (s + d + 1 < s1) load_x(s + d + 1);
      __syncthreads();   // block s + d is staged; the other stage is read
      const uint8_t* xs = lds + st * STAGE;
      multiply<FMT, G, NP, MT>(raw[d], acc, [&](int j, int mt) {
        return *reinterpret_cast<const u32x4_t*>(xs + (16 * mt + c) * 256 + slot(4 * j + q, c));
      });
      load_w(s + d + kAhead, raw[d]);
      if (s + d + 1 < s1) store_x(st ^ 1);
    }
  }

  // Epilogue, 16 rows of x at a time: the wave lays its sums out as rows in its part
  // of LDS and takes them with consecutive lanes along a row.
  __syncthreads();
  const float g0 = a.gs ? a.gs[0] : 1.f, g1 = a.gs && GATED ? a.gs[1] : g0;
  float* eb = reinterpret_cast<float*>(lds) + w * (16 * LD);
  constexpr int CG = W / 4, RS = 64 / CG > 16 ? 16 : 64 / CG;
#pragma unroll 1
  for (int j = 0; j < MT; ++j) {
    lin::lds_order();
#pragma unroll
    for (int jj = 0; jj < MT; ++jj) {
      if (jj != j) continue;
#pragma unroll
      for (int p = 0; p < NP; ++p)
        *reinterpret_cast<f32x4_t*>(eb + c * LD + 16 * p + 4 * q) =
            acc[p][jj] * (GATED && p % 2 ? g1 : g0);
    }
    lin::lds_order();
    const int mb = m0 + 16 * j;
    if (mb >= e.M) break;
    const auto place = [](int col) { return GATED ? col / 16 * 32 + col % 16 : col; };
    if (e.vec) {
      const int cv = lane % CG * 4, n = nw + cv;
#pragma unroll 1
      for (int r = lane / CG; r < 16; r += RS) {
        const int m = mb + r;
        if (n >= e.N || m >= e.M || lane / CG >= RS) break;
        const f32x4_t z = *reinterpret_cast<const f32x4_t*>(eb + r * LD + place(cv));
        f32x4_t u = z;
        if constexpr (GATED) u = *reinterpret_cast<const f32x4_t*>(eb + r * LD + place(cv) + 16);
        lin::finish4<AK>(e, m, n, z, u);
      }
    } else {
#pragma unroll 1
      for (int i = lane; i < 16 * W; i += 64) {
        const int r = i / W, col = i % W, m = mb + r, n = nw + col;
        if (n >= e.N || m >= e.M) continue;
        const float z = eb[r * LD + place(col)], u = GATED ? eb[r * LD + place(col) + 16] : 0.f;
        lin::finish_one<AK>(e, m, n, z, u);
      }
    }
  }
}

}  // namespace

hipError_t launch4_tile(const Linear4Args& a, hipStream_t stream) {
  constexpr int MT = 4, NP = 2;
  const int cols = 4 * (a.e.act == lin::kSwiglu ? 8 : 16) * NP;
  const long tiles = ((long)a.e.M + 16 * MT - 1) / (16 * MT) * (((long)a.e.N + cols - 1) / cols);
  if (!lin::grid_fits(tiles, 256)) return hipErrorInvalidConfiguration;
  return by_format(a, [&](auto fmt, auto group, auto g) {
    linear4_tile_kernel<decltype(fmt)::value, decltype(group)::value, decltype(g)::value, MT, NP>
        <<<(unsigned)tiles, 256, 0, stream>>>(a);
    return hipPeekAtLastError();
  });
}

}  // namespace l4
}  // namespace xtu
