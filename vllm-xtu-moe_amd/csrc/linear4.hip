// The product with 4-bit weights: argument checks and the choice of a kernel.
#include "linear4.hpp"

#include "../../include/xtu_moe_amd.h"

using namespace xtu;
using namespace xtu::l4;

namespace xtu {
namespace l4 {
namespace {

// Rows past M, up to a tile's 128, are ints too; columns and k as the dense product.
constexpr int kMaxM = 0x7fffffff - 511, kMaxN = 1 << 28, kMaxK = 1 << 28;
constexpr int kCus = 256;

bool format_ok(int fmt, int group) {
  if (fmt == kMx) return group == 32;
  if (fmt == kNv) return group == 16;
  return fmt == kI4 && (group == 32 || group == 64 || group == 128);
}

bool sizes_ok(int M, int N, int K, int act, int fmt, int group) {
  return M >= 0 && M <= kMaxM && N >= 1 && N <= kMaxN && K >= 1 && K <= kMaxK &&
         act >= lin::kNone && act <= lin::kSwiglu && format_ok(fmt, group) && K % group == 0;
}

long up(long n, long d) { return (n + d - 1) / d; }

// Estimated times in us.  All CUs together take in w at 6.2 GB a ms, one of them rows
// of x that are staged whole at 50 KB a us, and what it loads straight to LDS at 65 to
// 80; a launch and its latencies are 3 to 6, the launch that adds K splits 3 and its
// partial sums' way.  A workgroup of blocks after the first on its CU adds 3.5.

float join_time(const Shape4& s, int split, float rate) {
  if (split == 1) return 0.f;
  return 3.0f + 2.f * split * s.M * (float)s.N * (s.gated ? 2 : 1) * 4.f / rate;
}

float larger(float a, float b) { return a > b ? a : b; }

float skinny_time(const Shape4& s) {
  const SkinnyPlan p = skinny4_plan(s);
  if (p.grid == 0) return 1e30f;
  const int nb = blocks_of(s.K);
  const long rounds = up(p.grid, kCus);
  const float x = s.M * (float)s.K * 2e-3f;
  const float w = (s.gated ? 2 : 1) * (float)nb * record_bytes(s.fmt, s.group) * p.rows / 16 * 1e-3f;
  return 3.0f + 0.1f * (nb < 16 ? nb : 16) + rounds * x / 50.f +
         larger(p.units * w / 6200.f, rounds * up(p.units, p.grid) * w / 50.f);
}

float block_time(const Shape4& s, int rows) {
  const int nb = blocks_of(s.K);
  const long parts = up(s.M, rows), units = up(s.N, s.gated ? 16 : 32);
  const long rounds = up(units * parts, kCus);
  const float x = rows * 0.256f * nb, w = 2.f * nb * record_bytes(s.fmt, s.group) * 1e-3f;
  // (past 64 rows: all of x comes to every XCD that has a unit)
  const float far = s.M > 64 ? (units < 8 ? units : 8) * s.M * 0.256f * nb : 0.f;
  return 3.2f + larger(rounds * x / 80.f, far / 4500.f) +
         larger(units * w / 6200.f, rounds * w / 75.f) +
         0.35f * up(nb, block4_waves(s, rows)) + 3.5f * (rounds - 1);
}

// The split of K with the least time, 0 where no range of K fits LDS.
constexpr float kSlabBase = 6.0f;
int slab_split(const Shape4& s, bool may_split, float& time) {
  const int nb = blocks_of(s.K);
  const long gx = up(s.N, (s.gated ? 16 : 32) * kSlabWaves);
  int best = 0;
  time = 1e30f;
  for (int split = 1; split <= nb && split <= (may_split ? 64 : 1); ++split) {
    const int per = (int)up(nb, split);
    if (up(nb, per) != split || slab4_lds(s.M, per) > kSlabLds) continue;
    const long rounds = up(gx * split, kCus);
    const float x = slab4_lds(s.M, per) * 1e-3f;
    const float w = 2e-3f * kSlabWaves * per * record_bytes(s.fmt, s.group);
    const float t = kSlabBase + rounds * x / 65.f + larger(gx * split * w / 6200.f, rounds * w / 50.f) +
                    1.f * (rounds - 1) + join_time(s, split, 4e6f);
    if (t < time) {
      time = t;
      best = split;
    }
  }
  return best;
}

// Up to 64 rows.  Measured, in us (stream of w / blocks / slabs, MXFP4): M 1: 512 gated x
// 2048 5.6 / 4.5 / -, 7168 x 7168 9.1 / 8.8 / -, 16384 gated x 7168 25 / 30 / 29; M 4: 7168
// x 7168 10.5 / 9.3 / 11.2; M 8: 7168 x 2048 6.3 / 5.3 / -, 16384 x 7168 17.8 / 18.7 / 17.1;
// M 16: 7168 x 7168 - / 12.8 / 12.5, 2048 x 16384 - / 19.5 / 13.1, 16384 gated x 7168 - / 47 /
// 32; M 24: 16384 x 4096 - / 18.4 / 16.5; M 64: 7168 x 2048 - / 9.4 / 14.5, 7168 x 7168 -
// / 20.6 / 20.4.  (The estimates' choice is the fastest of three or within 4% of it there.)
Plan4 plan_few(const Shape4& s, bool may_split) {
  const float skinny = skinny_time(s), block = block4_plan(s).time;
  float slab = 1e30f;
  int split = 0;
  if (skinny > kSlabBase && block > kSlabBase) split = slab_split(s, may_split, slab);
  if (skinny <= block && skinny <= slab) return {kSkinny4, 1};
  if (block <= slab) return {kBlock4, 1};
  return {kSlab4, split};
}

// Steps of 128 k of a tile of 128 rows and 256 or 128 rows of w, alone on its CU, in us
// (2048 x 2048 gated x 7168, one round of the larger and two of the smaller: MXFP4 91 /
// 122, NVFP4 115 / 140, INT4 with groups of 128 121 / 148; 128 x 7168 x 2048 in 28 and
// 56 tiles: 29 / 20).  INT4's finer groups have no room for the larger one's sums: 198 us
// with groups of 32, 168 with 64, two rounds of steps of 1.70 and 1.43 us.
// Blocks against the better of the two, MXFP4: 128 x 2048 x 7168 11.9 / 20.0, 192 x 4096 x
// 4096 18.2 / 21.5, 256 x 512 x 7168 10.4 / 16.4, 512 x 1024 x 2048 9.8 / 16.8, 192 x 7168 x
// 2048 22.4 / 20.2, 512 x 2048 x 7168 30.8 / 26.6; x large: 2048 x 128 x 2048 9.6 / 14.7,
// 4096 x 128 x 2048 19.5 / 16.9.
Plan4 plan_many(const Shape4& s, bool may_split) {
  const bool fine = s.fmt == kI4 && s.group != 128;
  const float step4 = s.fmt == kMx ? 1.5f : s.fmt == kNv ? 1.95f : 2.1f;
  const float step2 = s.fmt == kMx ? 1.03f : s.fmt == kNv ? 1.2f : fine ? 1.7f : 1.3f;
  const int nb = blocks_of(s.K);
  Plan4 best{kBlock4, 1};
  float time = block4_plan(s).time;
  for (int kind : {kWide4, kWide2}) {
    if (kind == kWide4 && fine) continue;
    const long tiles = up(s.M, 128) * up(s.N, (s.gated ? 32 : 64) * (kind == kWide4 ? 4 : 2));
    for (int split : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (split > 1 && (!may_split || nb < 2 * split || tiles >= 2 * kCus)) break;
      const int per = (int)up(nb, split), real = (int)up(nb, per);
      const float t = 4.0f + up(tiles * real, kCus) * (per * (kind == kWide4 ? step4 : step2) + 2.f) +
                      join_time(s, real, 5e6f);
      if (t < time) {
        time = t;
        best = Plan4{kind, real};
      }
    }
  }
  return best;
}

Plan4 plan(const Shape4& s, bool may_split) {
  return s.M <= 64 ? plan_few(s, may_split) : plan_many(s, may_split);
}

size_t split_bytes(const Plan4& p, const Shape4& s) {
  return p.split > 1 ? (size_t)p.split * s.M * s.N * (s.gated ? 2 : 1) * 4 : 0;
}

// A copy of x.
size_t pack_bytes(int M, int K) { return (size_t)M * ((K + 7) / 8) * 16; }

// Rows of x on 16 bytes and, 128 of them, in reach of 32-bit offsets.
bool x_fits(const LinearArgs& e) {
  return reinterpret_cast<uintptr_t>(e.x) % 16 == 0 && e.K % 8 == 0 &&
         (e.M == 1 || e.ldx % 8 == 0) && ((e.M == 1 ? 0 : 128 * e.ldx) + e.K) * 2 < (1L << 31);
}

Shape4 shape_of(int M, int N, int K, int act, int fmt, int group) {
  return Shape4{M, N, K, act == lin::kSwiglu, fmt, group};
}

}  // namespace

// The rows of a part of x with the least time.
BlockPlan block4_plan(const Shape4& s) {
  if (s.M > kBlockM) return {0, 1e30f};
  if (s.M <= 8) {
    const int rows = s.M <= 4 ? 4 : 8;
    return {rows, block_time(s, rows)};
  }
  BlockPlan best{0, 1e30f};
  for (int rows = 64; rows >= 16; rows -= 16) {
    const float time = block_time(s, rows);
    if (rows < s.M + 16 && time < best.time) best = {rows, time};
  }
  return best;
}

}  // namespace l4
}  // namespace xtu

extern "C" {

size_t xtu_linear4_weight_bytes(int N, int K, int act, int fmt, int group) {
  if (!sizes_ok(0, N, K, act, fmt, group)) return 0;
  return (size_t)panels_of(N) * (act == lin::kSwiglu ? 2 : 1) * blocks_of(K) *
         record_bytes(fmt, group);
}

size_t xtu_linear4_workspace_bytes(int M, int N, int K, int act, int fmt, int group, int aligned) {
  if (!sizes_ok(M, N, K, act, fmt, group) || M == 0) return 0;
  const Shape4 s = shape_of(M, N, K, act, fmt, group);
  return split_bytes(plan(s, true), s) + (aligned ? 0 : pack_bytes(M, K));
}

int xtu_linear4_plan(int M, int N, int K, int act, int fmt, int group) {
  if (!sizes_ok(M, N, K, act, fmt, group) || M == 0) return -1;
  const Plan4 p = plan(shape_of(M, N, K, act, fmt, group), true);
  return 16 * p.split + p.kind;
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
  (void)hipGetLastError();
  const Shape4 s = shape_of(M, N, K, t.act, t.fmt, t.group);
  uint8_t* ws = reinterpret_cast<uint8_t*>(t.workspace);
  size_t left = ws ? t.workspace_bytes : 0;
  if (!x_fits(a.e)) {
    const size_t need = pack_bytes(M, K);
    LinearArgs copy = a.e;
    copy.x = reinterpret_cast<const uint16_t*>(ws);
    copy.ldx = K;
    if (left < need || !x_fits(copy)) return launch4_tile(a, stream);
    const hipError_t e = lin::launch_pack_x(a.e.x, a.e.ldx, M, K, reinterpret_cast<uint16_t*>(ws), stream);
    if (e != hipSuccess) return e;
    a.e = copy;
    ws += need;
    left -= need;
  }
  Plan4 p = plan(s, true);
  if (split_bytes(p, s) > left) p = plan(s, false);
  float* part = reinterpret_cast<float*>(ws);
  switch (p.kind) {
    case kSkinny4: return launch4_skinny(a, stream);
    case kBlock4: return launch4_block(a, stream);
    case kSlab4: return launch4_slab(a, p.split, part, stream);
    default: return launch4_wide(p, a, part, stream);
  }
}

}  // extern "C"
