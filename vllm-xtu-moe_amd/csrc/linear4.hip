// The product with 4-bit weights: argument checks and dispatch.
#include "linear4.hpp"

#include "../../include/xtu_moe_amd.h"

using namespace xtu;
using namespace xtu::l4;

namespace {

// Rows past M, up to a tile's 128, are ints too; columns and k as the dense product.
constexpr int kMaxM = 0x7fffffff - 511, kMaxN = 1 << 28, kMaxK = 1 << 28;

bool format_ok(int fmt, int group) {
  if (fmt == kMx) return group == 32;
  if (fmt == kNv) return group == 16;
  return fmt == kI4 && (group == 32 || group == 64 || group == 128);
}

bool sizes_ok(int M, int N, int K, int act, int fmt, int group) {
  return M >= 0 && M <= kMaxM && N >= 1 && N <= kMaxN && K >= 1 && K <= kMaxK &&
         act >= lin::kNone && act <= lin::kSwiglu && format_ok(fmt, group) && K % group == 0;
}

size_t split_bytes(const Plan4& p, int M, int N, bool gated) {
  return p.split > 1 ? (size_t)p.split * M * N * (gated ? 2 : 1) * 4 : 0;
}

}  // namespace

extern "C" {

size_t xtu_linear4_weight_bytes(int N, int K, int act, int fmt, int group) {
  if (!sizes_ok(0, N, K, act, fmt, group)) return 0;
  return (size_t)panels_of(N) * (act == lin::kSwiglu ? 2 : 1) * blocks_of(K) *
         record_bytes(fmt, group);
}

size_t xtu_linear4_workspace_bytes(int M, int N, int K, int act, int fmt, int group) {
  if (!sizes_ok(M, N, K, act, fmt, group) || M == 0) return 0;
  const bool gated = act == lin::kSwiglu;
  LinearArgs e{};
  e.M = M;
  e.K = K;
  if (skinny4_fits(e) || rows4_fits(e)) return 0;
  return split_bytes(plan4_tile(M, N, K, gated, true), M, N, gated);
}

hipError_t xtu_linear4(const xtu_linear4_args* args, hipStream_t stream) {
  XTU_CHECK_ARG(args);
  const xtu_linear4_args& t = *args;
  const int M = t.M, N = t.N, K = t.K;
  XTU_CHECK_ARG(sizes_ok(M, N, K, t.act, t.fmt, t.group));
  if (M == 0) return hipSuccess;
  XTU_CHECK_ARG(t.x && t.w && t.out && t.ldx >= 0 && t.ldr >= 0 && t.scale_stride >= 0);
  XTU_CHECK_ARG((t.fmt == kNv) == (t.gs != nullptr));
  XTU_CHECK_ARG(M == 1 || t.ldo >= N);
  const auto al = [](const void* p, long bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0;
  };
  XTU_CHECK_ARG(al(t.w, 16) && al(t.workspace, 16) && al(t.x, 2) && al(t.gs, 4));
  const bool gated = t.act == lin::kSwiglu;
  XTU_CHECK_ARG((long)M * N < (1L << 38));   // grids
  // vectors of four elements in the epilogue
  const int vec = N % 4 == 0 && al(t.out, t.out_bf16 ? 8 : 16) && (M == 1 || t.ldo % 4 == 0) &&
                  (!t.residual || (al(t.residual, t.residual_bf16 ? 8 : 16) &&
                                   (M == 1 || t.ldr % 4 == 0))) &&
                  (!t.bias || al(t.bias, t.bias_bf16 ? 8 : 16));
  Linear4Args a{};
  a.e = lin::LinearArgs{(const uint16_t*)t.x, nullptr, t.ldx, 0, M, N, K, t.act, t.bias,
                        t.bias_bf16, t.row_scale, t.scale_stride, t.residual, t.residual_bf16,
                        t.ldr, t.out, t.out_bf16, t.ldo, t.limit, t.alpha, t.beta, vec};
  a.w = reinterpret_cast<const uint8_t*>(t.w);
  a.gs = t.gs;
  a.fmt = t.fmt;
  a.group = t.group;
  a.xvec = al(t.x, 16) && K % 8 == 0 && (M == 1 || t.ldx % 8 == 0);
  (void)hipGetLastError();
#ifdef L4_NOSKINNY
  if (rows4_fits(a.e)) return launch4_rows(a, stream);
#endif
  if (skinny4_fits(a.e)) return launch4_skinny(a, stream);
  if (rows4_fits(a.e)) return launch4_rows(a, stream);
  Plan4 p = plan4_tile(M, N, K, gated, true);
  if (split_bytes(p, M, N, gated) > (t.workspace ? t.workspace_bytes : 0))
    p = plan4_tile(M, N, K, gated, false);
  return launch4_tile(p, a, reinterpret_cast<float*>(t.workspace), stream);
}

}  // extern "C"
