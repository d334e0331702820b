// The product with 4-bit weights for up to 64 rows of x (linear4.hpp has the formula
// and the layout).  A workgroup of eight waves holds a range of K of all rows of x in
// LDS; each wave streams that range of its own two panels (swiglu: a gate and its up
// panel) to its registers, U blocks ahead, and meets no barrier on the way.
//
// What bounds it is what a CU takes in: its share of w, which is fixed, and the
// workgroup's part of x.  Splitting K makes the latter smaller and costs partial sums,
// which linear_join_kernel adds (linear4.hip weighs them): 16 x 16384 gated x 7168 MXFP4
// 32 us in 2 ranges (blocks 47), 24 x 16384 x 4096 16.5 in 2 (18.4), 16 x 2048 x 16384
// 13.1 in 16 (19.5).  More records ahead change nothing (U = 5, 7).
#include "linear4.hpp"

namespace xtu {
namespace l4 {
namespace {

constexpr int kWv = kSlabWaves;

template <int FMT, int G, int AK, int MT, int U>
__global__ __launch_bounds__(64 * kWv) void linear4_slab_kernel(Linear4Args a, int per, float* part) {
  constexpr bool GATED = AK == lin::kActSwiglu;
  constexpr int REC = record_bytes(FMT, G), COLS = GATED ? 16 : 32;
  constexpr int LW = 2 * (1 + (FMT == kI4 ? 128 / G : 1));   // loads of a block's records
  static_assert(U * LW <= 63, "vmcnt");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const LinearArgs& e = a.e;
  const int tid = threadIdx.x, lane = tid % 64;
  const int w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int q = lane / 16, c = lane % 16;
  const int nb = blocks_of(e.K), s0 = (int)blockIdx.y * per, s1 = min(nb, s0 + per);
  const int unit = blockIdx.x * kWv + w;
  const int last = panels_of(e.N) * (GATED ? 2 : 1) - 1;   // panel
  const uint8_t* wp[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) wp[p] = a.w + (long)min(2 * unit + p, GATED ? last - 1 + p : last) * nb * REC;
  Raw<FMT, G> raw[U][2];
  auto load = [&](int s, Raw<FMT, G> (&r)[2]) {
    const long o = (long)min(s, s1 - 1) * REC;
#pragma unroll
    for (int p = 0; p < 2; ++p) r[p] = load_raw<FMT, G>(wp[p] + o, q, c, 4 * q);
  };
  // x straight to LDS, block by block: a load brings four rows, a piece of 16 bytes a
  // lane (linear_tile.hip has the slots); the waves take turns
  const u32x4_t xr = lin::raw_buffer(e.x, (uint32_t)(((long)(e.M - 1) * e.ldx + e.K) * 2));
  const int quads = (e.M + 3) / 4, size = quads * 1024;   // of a block
  int r = w % quads, s = s0 + w / quads;
  const int dr = kWv % quads, ds = kWv / quads;
#pragma unroll 1
  while (s < s1) {
    const int row = 4 * r + lane / 16, k = 8 * (lane % 16 ^ (row & 7) << 1);
    const uint32_t off = (uint32_t)min(row, e.M - 1) * (uint32_t)(e.ldx * 2) + 2 * k;
    lin::buf_to_lds(xr, k < e.K - 128 * s ? off : 0x80000000u, (uint32_t)s * 256u,
                    lds + (s - s0) * size + r * 1024);
    r += dr;
    s += ds;
    if (r >= quads) {
      r -= quads;
      ++s;
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) load(s0 + i, raw[i]);
  __builtin_amdgcn_s_waitcnt(lin::wait_vm(U * LW));   // x; loads come back in order
  __syncthreads();
  const uint8_t* xl[MT];   // (rows past M repeat the last one: not written)
  int slot[MT];            // of place 4 j + q: j moves bits 2 and 3
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = min(16 * mt + c, e.M - 1);
    xl[mt] = lds + row * 256;
    slot[mt] = (q ^ (row & 7) << 1) * 16;
  }
  f32x4_t acc[2][MT];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[p][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (s = s0; s < s1; s += U) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (s + i >= s1) break;
      const int o = (s + i - s0) * size;
      multiply<FMT, G, 2, MT>(raw[i], acc, [&](int j, int mt) {
        return *reinterpret_cast<const u32x4_t*>(xl[mt] + o + (slot[mt] ^ 64 * j));
      });
      load(s + i + U, raw[i]);
    }
  }

  const float g0 = a.gs ? a.gs[0] : 1.f, g1 = a.gs && GATED ? a.gs[1] : g0;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    acc[0][mt] *= g0;
    acc[1][mt] *= GATED ? g1 : g0;
  }
  const int n0 = unit * COLS + 4 * q;
  const auto whole = [&](int n) { return e.vec && n < e.N; };   // N % 4 == 0: four or none
  if (part) {
    float* plane = part + (long)blockIdx.y * lin::part_plane(e);
    const long row = (long)e.N * (GATED ? 2 : 1);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int m = 16 * mt + c;
      if (m >= e.M) break;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int n = n0 + (GATED ? 0 : 16 * p);
        float* to = plane + m * row + (GATED && p ? e.N : 0) + n;
        if (whole(n)) {
          *reinterpret_cast<f32x4_t*>(to) = acc[p][mt];
        } else if (!e.vec) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (n + t < e.N) to[t] = acc[p][mt][t];
        }
      }
    }
    return;
  }
  constexpr int F = GATED ? 1 : 2;   // vectors of results per row
  if constexpr (AK != lin::kActOther) {
    // what all of them read beside the sums is asked for at once
    u32x4_t bz[F], bu[F];
    lin::Row4 pre[F][MT];
    if (e.vec) {
#pragma unroll
      for (int p = 0; p < F; ++p) {
        const int n = min(n0 + 16 * p, e.N - 4);
        lin::load_bias4<AK>(e, n, bz[p], bu[p]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) pre[p][mt] = lin::load_row4(e, min(16 * mt + c, e.M - 1), n);
      }
#pragma unroll
      for (int p = 0; p < F; ++p)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int m = 16 * mt + c, n = n0 + 16 * p;
          if (m >= e.M || n >= e.N) continue;
          f32x4_t z[1] = {acc[p][mt] + lin::of_raw4(bz[p], e.bias_bf16)}, u[1] = {z[0]};
          if constexpr (GATED) u[0] = acc[1][mt] + lin::of_raw4(bu[p], e.bias_bf16);
          lin::act_all<AK>(e, z, u);
          lin::store_row4(e, m, n, z[0], pre[p][mt]);
        }
      return;
    }
  }
  // the others one at a time, their code once (linear.hpp, ActKind)
#pragma unroll 1
  for (int k = 0; k < F * MT; ++k) {
    f32x4_t z = acc[0][0], u = acc[1][0];
#pragma unroll
    for (int i = 0; i < F * MT; ++i) {
      if (i != k) continue;
      z = acc[GATED ? 0 : i % 2][i / F];
      u = acc[1][i / F];
    }
    const int m = 16 * (k / F) + c, n = n0 + (GATED ? 0 : 16 * (k % 2));
    if (m >= e.M) break;
    if (whole(n)) {
      lin::finish4<AK>(e, m, n, z, u);
    } else if (!e.vec) {
#pragma unroll 1
      for (int t = 0; t < 4; ++t) {
        if (n + t < e.N) lin::finish_one<AK>(e, m, n + t, z[0], u[0]);
        z = __builtin_shufflevector(z, z, 1, 2, 3, 0);
        u = __builtin_shufflevector(u, u, 1, 2, 3, 0);
      }
    }
  }
}

template <int MT>
hipError_t launch(const Linear4Args& a, int split, float* part, hipStream_t stream) {
  const LinearArgs& e = a.e;
  const int nb = blocks_of(e.K), per = (nb + split - 1) / split;
  split = (nb + per - 1) / per;   // no empty range
  const int cols = (e.act == lin::kSwiglu ? 16 : 32) * kWv;
  const dim3 grid((unsigned)(((long)e.N + cols - 1) / cols), (unsigned)split);
  const size_t lds = slab4_lds(e.M, per);
  if (e.M > 64 || lds > kSlabLds) return hipErrorInvalidValue;
  float* to = split > 1 ? part : nullptr;
  const hipError_t r = by_format(a, [&](auto fmt, auto group, auto g) {
    constexpr int F = decltype(fmt)::value, G = decltype(group)::value;
    constexpr int U = F == kI4 && G == 32 ? 2 : 3;   // what the registers hold
    auto k = linear4_slab_kernel<F, G, lin::kActSwiglu, MT, U>;
    if constexpr (!decltype(g)::value)
      k = to || e.act == lin::kNone ? linear4_slab_kernel<F, G, lin::kActNone, MT, U>
                                    : linear4_slab_kernel<F, G, lin::kActOther, MT, U>;
    k<<<grid, 64 * kWv, lds, stream>>>(a, per, to);
    return hipPeekAtLastError();
  });
  if (r == hipSuccess && split > 1) return lin::launch_join(e, split, part, stream);
  return r;
}

}  // namespace

hipError_t launch4_slab(const Linear4Args& a, int split, float* part, hipStream_t stream) {
  if (a.e.M <= 16) return launch<1>(a, split, part, stream);
  if (a.e.M <= 32) return launch<2>(a, split, part, stream);
  if (a.e.M <= 48) return launch<3>(a, split, part, stream);
  return launch<4>(a, split, part, stream);
}

}  // namespace l4
}  // namespace xtu
