// The MoE block of a few tokens: entry points (few.hpp has the kernels).
#include "few.hpp"

#include "../../include/xtu_moe_amd.h"

namespace xtu {
namespace few {
namespace {

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// bits of a weight with its scales
float format_bits(int fmt) {
  return fmt == kBF16 ? 16.0f : fmt == kFP8 ? 8.0f : fmt == kMXFP4 ? 4.25f : 4.5f;
}

struct Layout {
  int ldl, ctl_words;
  size_t logits, act, part, ctl, total;   // byte offsets
};

Layout layout_of(const Plan& p, int T, int E, int K, int NS, int H, int I) {
  Layout l;
  l.ldl = (E + NS + 3) / 4 * 4;   // 16-byte rows
  l.ctl_words = kPanels + H / 16;
  l.logits = 0;
  l.act = up256((size_t)T * l.ldl * 4);
  l.part = l.act + up256((size_t)p.parts * T * (K + NS) * I * 2);
  l.ctl = l.part + (p.chunks > 1 ? up256((size_t)p.chunks * T * H * 4) : 0);
  l.total = l.ctl + up256((size_t)l.ctl_words * 4);
  return l;
}

}  // namespace
}  // namespace few
}  // namespace xtu

using namespace xtu;
using namespace xtu::few;

extern "C" {

size_t xtu_few_workspace_bytes(int fmt, int T, int E, int K, int n_shared, int H, int I) {
  Plan p;
  if (fmt < 0 || fmt > 3 ||
      !make_plan(T, E, K, n_shared, H, I, format_bits(fmt), p))
    return 0;
  return layout_of(p, T, E, K, n_shared, H, I).total;
}

hipError_t xtu_few_block(const xtu_few_args* args, hipStream_t stream) {
  XTU_CHECK_ARG(args);
  const xtu_few_args& t = *args;
  Plan p;
  XTU_CHECK_ARG(t.fmt >= 0 && t.fmt <= 3 && (t.mode == 0 || t.mode == 1));
  XTU_CHECK_ARG(make_plan(t.T, t.E, t.K, t.n_shared, t.H, t.I, format_bits(t.fmt), p));
  XTU_CHECK_ARG(t.x && t.gate && t.w13 && t.w2 && t.out && t.ids && t.weights && t.workspace);
  XTU_CHECK_ARG(t.fmt == kBF16 || (t.s13 && t.s2));
  XTU_CHECK_ARG(!t.shared_gate || t.n_shared > 0);
  const auto al16 = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  XTU_CHECK_ARG(al16(t.x) && al16(t.gate) && al16(t.shared_gate) && al16(t.workspace) &&
                al16(t.w13) && al16(t.w2) && al16(t.s13) && al16(t.s2));
  if (t.mode == 1)
    XTU_CHECK_ARG(t.n_group >= 1 && t.n_group <= kMaxGroups && t.E % t.n_group == 0 &&
                  t.topk_group >= 1 && t.topk_group <= t.n_group &&
                  t.K <= t.topk_group * (t.E / t.n_group));
  const Layout l = layout_of(p, t.T, t.E, t.K, t.n_shared, t.H, t.I);
  XTU_CHECK_ARG(t.workspace_bytes >= l.total);
  (void)hipGetLastError();
  uint8_t* ws = reinterpret_cast<uint8_t*>(t.workspace);
  FewArgs f{};
  f.x = (const uint16_t*)t.x;
  f.gate = (const uint16_t*)t.gate;
  f.sgate = (const uint16_t*)t.shared_gate;
  f.bias = t.mode == 1 ? t.bias : nullptr;
  f.T = t.T;
  f.H = t.H;
  f.I = t.I;
  f.E = t.E;
  f.NS = t.n_shared;
  f.K = t.K;
  f.mode = t.mode;
  f.renorm = t.renormalize;
  f.n_group = t.mode == 1 ? t.n_group : 1;
  f.topk_group = t.mode == 1 ? t.topk_group : 1;
  f.scale = t.mode == 1 ? t.routed_scaling : 1.0f;
  f.w13 = (const uint8_t*)t.w13;
  f.s13 = (const uint8_t*)t.s13;
  f.w2 = (const uint8_t*)t.w2;
  f.s2 = (const uint8_t*)t.s2;
  f.gs13 = t.gs13;
  f.gs2 = t.gs2;
  f.limit = t.limit;
  f.alpha = t.alpha;
  f.beta = t.beta;
  f.ldl = l.ldl;
  f.logits = reinterpret_cast<float*>(ws + l.logits);
  f.act = reinterpret_cast<uint16_t*>(ws + l.act);
  f.part = reinterpret_cast<float*>(ws + l.part);
  f.ctl = reinterpret_cast<unsigned*>(ws + l.ctl);
  f.ctl_words = l.ctl_words;
  f.ids = t.ids;
  f.wts = t.weights;
  f.out = t.out;
  f.out_bf16 = t.out_bf16;
  f.n_sh = t.n_shared * (t.I / 16);
  const int er = t.E + (t.shared_gate ? t.n_shared : 0);
  f.rp = 1;   // router rows per panel: a CU each, beside the shared panels
  while (f.rp < 16 && f.n_sh + (er + f.rp - 1) / f.rp > cu_count()) f.rp *= 2;
  f.epl = tiny::wave_epl(t.mode, t.E, f.n_group, t.renormalize, f.logits, f.bias);
  f.chunk_units = p.chunk_units;
  f.chunks = p.chunks;
  f.parts = p.parts;
  f.stage_bytes = p.stage;
  switch (t.fmt) {
    case kMXFP4: return run_mxfp4(f, p, stream);
    case kNVFP4: return run_nvfp4(f, p, stream);
    case kFP8: return run_fp8(f, p, stream);
    case kBF16: return run_bf16(f, p, stream);
  }
  return hipErrorInvalidValue;
}

}  // extern "C"
