// The dense product with its epilogue: dispatch and the kernel for any shape.
#include "linear.hpp"

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
        if (n < a.N) finish_one(a, m, n, acc[0][j][t], acc[1][j][t]);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = n0 + 32 * wn + 16 * i + 4 * q + t;
          if (n < a.N) finish_one(a, m, n, acc[i][j][t], 0.f);
        }
      }
    }
  }
}

}  // namespace
}  // namespace lin
}  // namespace xtu

using namespace xtu;
using namespace xtu::lin;

extern "C" {

hipError_t xtu_linear(const void* x, long ldx, const void* w, long ldw, int M, int N, int K,
                      int act, const void* bias, int bias_bf16, const float* row_scale,
                      long scale_stride, const void* residual, int residual_bf16, long ldr,
                      void* out, int out_bf16, long ldo, float limit, float alpha, float beta,
                      hipStream_t stream) {
  XTU_CHECK_ARG(M >= 0 && N >= 1 && K >= 1 && act >= kNone && act <= kSwiglu);
  XTU_CHECK_ARG(N <= (1 << 28) && K <= (1 << 28));
  if (M == 0) return hipSuccess;
  XTU_CHECK_ARG(x && w && out && ldx >= 0 && ldw >= 0 && ldr >= 0 && scale_stride >= 0);
  XTU_CHECK_ARG(M == 1 || ldo >= N);
  const int nb = act == kSwiglu ? kAnyN / 2 : kAnyN;
  const long gm = (M + (long)kAnyM - 1) / kAnyM, gn = ((long)N + nb - 1) / nb;
  XTU_CHECK_ARG(gm * gn < (1L << 31));
  (void)hipGetLastError();
  LinearArgs a{(const uint16_t*)x, (const uint16_t*)w, ldx, ldw, M, N, K, act, bias, bias_bf16,
               row_scale, scale_stride, residual, residual_bf16, ldr, out, out_bf16, ldo, limit,
               alpha, beta};
  const unsigned grid = (unsigned)(gm * gn);
  if (act == kSwiglu) linear_any_kernel<true><<<grid, 256, 0, stream>>>(a);
  else linear_any_kernel<false><<<grid, 256, 0, stream>>>(a);
  return hipPeekAtLastError();
}

}  // extern "C"
