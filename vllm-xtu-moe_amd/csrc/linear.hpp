// Dense product with a fused epilogue: what the kernels of linear*.hip share.
//
//   y[m][n] = residual[m][n] + row_scale[m] * act(sum_k x[m][k] w[n][k] + bias[n])
//
// x, w bf16 with row strides, fp32 sums.  "swiglu": w holds 2N rows, the gate
// rows [0, N) and the up rows [N, 2N) (bias alike), act = the expert MLP's
// clamped gated SiLU.  Everything after the product stays in fp32 and is
// rounded once, to the output's type.
#pragma once
#include "xtu_common.hpp"

namespace xtu {
namespace lin {

enum Act : int { kNone = 0, kRelu, kSilu, kGelu, kGeluTanh, kSigmoid, kSwiglu };

struct LinearArgs {
  const uint16_t* x;      // [M][K] bf16, rows ldx apart
  const uint16_t* w;      // [N or 2N][K] bf16, rows ldw apart
  long ldx, ldw;
  int M, N, K, act;
  const void* bias;       // [N or 2N] bf16 or fp32, or null
  int bias_bf16;
  const float* scale;     // [M], elements sstride apart, or null
  long sstride;
  const void* res;        // [M][N] bf16 or fp32, rows ldr apart, or null
  int res_bf16;
  long ldr;
  void* out;              // [M][N] bf16 or fp32, rows ldo apart
  int out_bf16;
  long ldo;
  float limit, alpha, beta;
};

// NaN stays NaN in every activation (relu: the comparison is false for it).
__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case kRelu: return z < 0.f ? 0.f : z;
    case kSilu: return z / (1.f + __expf(-z));
    case kGelu: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case kGeluTanh:
      return 0.5f * z * (1.f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
    case kSigmoid: return 1.f / (1.f + __expf(-z));
    default: return z;
  }
}

__device__ __forceinline__ float load_bias(const LinearArgs& a, int n) {
  return a.bias_bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(a.bias)[n])
                     : reinterpret_cast<const float*>(a.bias)[n];
}

// One output element from its product(s): z, and for swiglu the up product u.
__device__ __forceinline__ void finish_one(const LinearArgs& a, int m, int n, float z, float u) {
  if (a.bias) {
    z += load_bias(a, n);
    if (a.act == kSwiglu) u += load_bias(a, a.N + n);
  }
  float y = a.act == kSwiglu ? silu_gate(z, u, a.limit, a.alpha, a.beta) : activate(a.act, z);
  if (a.scale) y *= a.scale[(long)m * a.sstride];
  if (a.res) {
    const long o = (long)m * a.ldr + n;
    y += a.res_bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(a.res)[o])
                    : reinterpret_cast<const float*>(a.res)[o];
  }
  const long o = (long)m * a.ldo + n;
  if (a.out_bf16) reinterpret_cast<uint16_t*>(a.out)[o] = f32_to_bf16(y);
  else reinterpret_cast<float*>(a.out)[o] = y;
}

// Eight consecutive k of one row from k on, zeros past K.  Rows need not start
// on 16 bytes: global loads take any alignment, at more than one transaction.
__device__ __forceinline__ u32x4_t load8(const uint16_t* row, int k, int K) {
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (k + 8 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) v[i / 2] |= (uint32_t)row[k + i] << (16 * (i % 2));
  }
  return v;
}

}  // namespace lin
}  // namespace xtu
