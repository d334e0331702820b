// The dense product with its epilogue: dispatch, the join of K splits, and what
// rows that do not start on 16 bytes need: a copy that makes them (linear_pack_kernel),
// or, without a workspace for it, the kernel for any operands (linear_any_kernel).
#include "linear.hpp"

#include "../../include/xtu_moe_amd.h"

namespace xtu {
namespace lin {
namespace {

constexpr int kAnyM = 64, kAnyN = 64, kAnyK = 64;
constexpr int kAnyLd = kAnyK + 8;   // bf16 of an LDS row

// Any sizes, strides and alignment: 64 rows of x times 64 rows of w (swiglu:
// 32 gate and their 32 up rows) per workgroup, four waves of 32 x 32, K in
// steps of 64 through LDS with the next step's loads in registers.  The MFMA
// takes w as its A operand, so a lane holds four consecutive output columns
// of one row.  Rows past M or N read the last row; what they give is not
// written.
template <bool GATED>
__global__ __launch_bounds__(256) void linear_any_kernel(LinearArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t xs[kAnyM][kAnyLd];
  __shared__ __attribute__((aligned(16))) uint16_t wsm[kAnyN][kAnyLd];
  constexpr int NB = GATED ? kAnyN / 2 : kAnyN;   // output columns of the tile
  const int tid = threadIdx.x, lane = tid % 64, w = tid / 64;
  const int q = lane / 16, c = lane % 16;
  const int wm = w & 1, wn = w >> 1;
  const int gn = (a.N + NB - 1) / NB;
  const int m0 = blockIdx.x / gn * kAnyM, n0 = blockIdx.x % gn * NB;
  const int r = tid / 4, kc = (tid % 4) * 16;
  // LDS row r of the w tile: 16-row blocks alternate gate, up
  int wr;
  if (GATED) wr = (r / 16 % 2) * a.N + min(n0 + r / 32 * 16 + r % 16, a.N - 1);
  else wr = min(n0 + r, a.N - 1);
  const uint16_t* xrow = a.x + (long)min(m0 + r, a.M - 1) * a.ldx;
  const uint16_t* wrow = a.w + (long)wr * a.ldw;
  u32x4_t xv[2], wv[2];
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xv[i] = load8(xrow, k0 + kc + 8 * i, a.K);
      wv[i] = load8(wrow, k0 + kc + 8 * i, a.K);
    }
  };
  f32x4_t acc[2][2] = {};
  load(0);
  for (int k0 = 0; k0 < a.K; k0 += kAnyK) {
    __syncthreads();   // the previous step is read
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<u32x4_t*>(&xs[r][kc + 8 * i]) = xv[i];
      *reinterpret_cast<u32x4_t*>(&wsm[r][kc + 8 * i]) = wv[i];
    }
    __syncthreads();
    if (k0 + kAnyK < a.K) load(k0 + kAnyK);
#pragma unroll
    for (int kk = 0; kk < kAnyK; kk += 32) {
      u32x4_t av[2], bv[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        av[i] = *reinterpret_cast<const u32x4_t*>(&wsm[32 * wn + 16 * i + c][kk + 8 * q]);
        bv[i] = *reinterpret_cast<const u32x4_t*>(&xs[32 * wm + 16 * i + c][kk + 8 * q]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(av[i]), as_bf16x8(bv[j]),
                                                              acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int m = m0 + 32 * wm + 16 * j + c;
    if (m >= a.M) continue;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (GATED) {
        const int n = n0 + 16 * wn + 4 * q + t;
        if (n < a.N) finish_one<kActSwiglu>(a, m, n, acc[0][j][t], acc[1][j][t]);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = n0 + 32 * wn + 16 * i + 4 * q + t;
          if (n < a.N) finish_one<kActOther>(a, m, n, acc[i][j][t], 0.f);
        }
      }
    }
  }
}

// Adds the partial sums of the K splits, in their order, and finishes the
// elements; one thread per V (4 or 1) columns of a row.
template <int AK, int V>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a, int split,
                                                          const float* part) {
  constexpr bool GATED = AK == kActSwiglu;
  const int gn = a.N / V;
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  if (t >= (long)a.M * gn) return;
  const int m = (int)(t / gn), n = (int)(t % gn) * V;
  const long plane = part_plane(a);
  const float* p = part + (long)m * a.N * (GATED ? 2 : 1) + n;
  if constexpr (V == 4) {
    f32x4_t z = {0.f, 0.f, 0.f, 0.f}, u = z;
    for (int k = 0; k < split; ++k, p += plane) {
      z += *reinterpret_cast<const f32x4_t*>(p);
      if constexpr (GATED) u += *reinterpret_cast<const f32x4_t*>(p + a.N);
    }
    finish4<AK>(a, m, n, z, u);
  } else {
    float z = 0.f, u = 0.f;
    for (int k = 0; k < split; ++k, p += plane) {
      z += p[0];
      if constexpr (GATED) u += p[a.N];
    }
    finish_one<AK>(a, m, n, z, u);
  }
}

// x and w as rows of K8 = K rounded up to 8, zeros behind K: what the tile
// kernels read.  1013 x 1187 by 771 rows of it: the two launches take 16 us (with bias,
// gelu and residual) where linear_any_kernel takes 24.
__global__ __launch_bounds__(256) void linear_pack_kernel(const uint16_t* x, long ldx, int M,
                                                          const uint16_t* w, long ldw, int rows,
                                                          int K, uint16_t* out) {
  const int per = (K + 7) / 8;
  const long p = (long)blockIdx.x * 256 + threadIdx.x;
  if (p >= ((long)M + rows) * per) return;
  const long r = p / per;
  const int k = (int)(p - r * per) * 8;
  const uint16_t* row = r < M ? x + r * ldx : w + (r - M) * ldw;
  *reinterpret_cast<u32x4_t*>(out + p * 8) = load8<true>(row, k, K);
}

}  // namespace

hipError_t launch_join(const LinearArgs& a, int split, const float* part, hipStream_t stream) {
  const long n = (long)a.M * (a.vec ? a.N / 4 : a.N);
  if (!grid_fits((n + 255) / 256, 256)) return hipErrorInvalidConfiguration;
  void (*k)(LinearArgs, int, const float*);
  if (a.act == kSwiglu) k = a.vec ? linear_join_kernel<kActSwiglu, 4> : linear_join_kernel<kActSwiglu, 1>;
  else if (a.act == kNone) k = a.vec ? linear_join_kernel<kActNone, 4> : linear_join_kernel<kActNone, 1>;
  else k = a.vec ? linear_join_kernel<kActOther, 4> : linear_join_kernel<kActOther, 1>;
  k<<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a, split, part);
  return hipPeekAtLastError();
}

hipError_t launch_any(const LinearArgs& a, hipStream_t stream) {
  const int nb = a.act == kSwiglu ? kAnyN / 2 : kAnyN;
  const long gm = (a.M + (long)kAnyM - 1) / kAnyM, gn = ((long)a.N + nb - 1) / nb;
  const unsigned grid = (unsigned)(gm * gn);
  if (!grid_fits(gm * gn, 256)) return hipErrorInvalidConfiguration;
  if (a.act == kSwiglu) linear_any_kernel<true><<<grid, 256, 0, stream>>>(a);
  else linear_any_kernel<false><<<grid, 256, 0, stream>>>(a);
  return hipPeekAtLastError();
}

}  // namespace lin
}  // namespace xtu

namespace xtu {
namespace lin {
namespace {

// Rows past M, up to a tile's 256, are ints too.
constexpr int kMaxM = 0x7fffffff - 511;

size_t pack_bytes(int M, long rows, int K) { return (size_t)(M + rows) * ((K + 7) / 8) * 16; }

size_t split_bytes(const TilePlan& p, int M, long rows) {
  return p.split > 1 ? (size_t)p.split * M * rows * 4 : 0;
}

hipError_t launch_pack(LinearArgs& a, long rows, void* ws, hipStream_t stream) {
  const long K8 = (a.K + 7) / 8 * 8, pieces = (a.M + rows) * (K8 / 8);
  uint16_t* out = reinterpret_cast<uint16_t*>(ws);
  if (!grid_fits((pieces + 255) / 256, 256)) return hipErrorInvalidConfiguration;
  linear_pack_kernel<<<(unsigned)((pieces + 255) / 256), 256, 0, stream>>>(
      a.x, a.ldx, a.M, a.w, a.ldw, (int)rows, a.K, out);
  a.x = out;
  a.w = out + a.M * K8;
  a.ldx = a.ldw = K8;
  a.K = (int)K8;
  return hipPeekAtLastError();
}

}  // namespace
}  // namespace lin
}  // namespace xtu

using namespace xtu;
using namespace xtu::lin;

extern "C" {

size_t xtu_linear_workspace_bytes(int M, int N, int K, int act, int aligned) {
  if (M <= 0 || M > kMaxM || N <= 0 || K <= 0 || N > (1 << 28) || K > (1 << 28)) return 0;
  LinearArgs a{};
  a.M = M;
  a.N = N;
  a.K = K;
  a.act = act;
  if (skinny_fits(a)) return 0;
  const long rows = (long)N * (act == kSwiglu ? 2 : 1);
  const size_t pack = aligned ? 0 : pack_bytes(M, rows, K);
  return pack + split_bytes(plan_tile(M, N, K, act == kSwiglu, true), M, rows);
}

int xtu_linear_plan(int M, int N, int K, int act) {
  if (M <= 0 || M > kMaxM || N <= 0 || K <= 0 || N > (1 << 28) || K > (1 << 28)) return -1;
  LinearArgs a{};
  a.M = M;
  a.N = N;
  a.K = K;
  if (skinny_fits(a)) return 0;
  const TilePlan p = plan_tile(M, N, K, act == kSwiglu, true);
  return 256 * p.split + 1 + p.kind;
}

hipError_t xtu_linear(const xtu_linear_args* args, hipStream_t stream) {
  XTU_CHECK_ARG(args);
  const xtu_linear_args& t = *args;
  const int M = t.M, N = t.N, K = t.K, act = t.act;
  XTU_CHECK_ARG(M >= 0 && N >= 1 && K >= 1 && act >= kNone && act <= kSwiglu);
  XTU_CHECK_ARG(M <= kMaxM && N <= (1 << 28) && K <= (1 << 28));
  if (M == 0) return hipSuccess;
  XTU_CHECK_ARG(t.x && t.w && t.out && t.ldx >= 0 && t.ldw >= 0 && t.ldr >= 0 &&
                t.scale_stride >= 0);
  XTU_CHECK_ARG(M == 1 || t.ldo >= N);
  XTU_CHECK_ARG(reinterpret_cast<uintptr_t>(t.workspace) % 16 == 0);
  const bool gated = act == kSwiglu;
  const long gm = (M + (long)kAnyM - 1) / kAnyM, gn = ((long)N + kAnyN / 2 - 1) / (kAnyN / 2);
  XTU_CHECK_ARG(gm * gn < (1L << 31) && (long)M * N < (1L << 38));   // grids
  const auto al = [](const void* p, long bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0;
  };
  // vectors of four elements in the epilogue
  const int vec = N % 4 == 0 && al(t.out, t.out_bf16 ? 8 : 16) && (M == 1 || t.ldo % 4 == 0) &&
                  (!t.residual || (al(t.residual, t.residual_bf16 ? 8 : 16) &&
                                   (M == 1 || t.ldr % 4 == 0))) &&
                  (!t.bias || al(t.bias, t.bias_bf16 ? 8 : 16));
  LinearArgs a{(const uint16_t*)t.x, (const uint16_t*)t.w, t.ldx, t.ldw, M, N, K, act, t.bias,
               t.bias_bf16, t.row_scale, t.scale_stride, t.residual, t.residual_bf16, t.ldr,
               t.out, t.out_bf16, t.ldo, t.limit, t.alpha, t.beta, vec};
  (void)hipGetLastError();
  if (skinny_fits(a)) return launch_skinny(a, stream);
  const long rows = (long)N * (gated ? 2 : 1);
  uint8_t* ws = reinterpret_cast<uint8_t*>(t.workspace);
  size_t left = ws ? t.workspace_bytes : 0;
  if (!tile_fits(a)) {
    const size_t need = pack_bytes(M, rows, K);
    const long K8 = (K + 7) / 8 * 8;
    if (left < need || 256 * K8 * 2 + K8 * 2 >= (1L << 31) ||
        (M + rows) * (K8 / 8) >= (1L << 38))
      return launch_any(a, stream);
    const hipError_t e = launch_pack(a, rows, ws, stream);
    if (e != hipSuccess) return e;
    ws += need;
    left -= need;
  }
  TilePlan p = plan_tile(M, N, a.K, gated, true);
  if (split_bytes(p, M, rows) > left) p = plan_tile(M, N, a.K, gated, false);
  return launch_tile_kind(p.kind, a, p.split, reinterpret_cast<float*>(ws), stream);
}

}  // extern "C"
