// The dense product with 4-bit weights and group scales: what the kernels of
// linear4*.hip share.
//
//   y[m][n] = residual[m][n] + row_scale[m] *
//             act(g sum_k x[m][k] v[n][k] s[n][k / G] + bias[n])
//
//   MXFP4: v = e2m1 of the code, G = 32,  s = 2^(byte - 127)
//   NVFP4: v = e2m1 of the code, G = 16,  s = e4m3 of the byte, g the second-level scale
//   INT4:  v = code - 8,         G = 32, 64 or 128, s fp32
//
// v s is exact in bf16 for MXFP4 and NVFP4 (significands of 2 and 2 x 4 bits), so the
// bf16 MFMA multiplies exact operands; INT4's v is, and its scale multiplies the
// group's fp32 sum.  The epilogue is linear.hpp's.
//
// Layout.  Rows in panels of 16 (swiglu: gate and up panels in turn), K in blocks
// of 128; a block of a panel is one record: 1024 bytes of codes [4 q][16 row][4 j][4 B],
// lane 16 q + row of a wave takes 16 of them, dword j the codes of k = 32 j + 8 q .. + 7
// (low nibble first; INT4: as code ^ 8, two's complement), which are an MFMA operand's.
// So an MFMA's 32 k are consecutive, x is read as it lies, and an INT4 group is whole
// MFMAs.  Then the record's scales, a dword of four for the lanes that share them:
//   MXFP4: [16 row][4 j] bytes        NVFP4: [2 q / 2][16 row][4 j] bytes
//   INT4:  fp32 [128 / G][16 row], times 16 (i4x8_to_bf16)
// A panel's records are consecutive: a wave walks one stream.  Rows and k past the
// matrix are zero codes under scale one (NVFP4, INT4: zero).
#pragma once
#include <type_traits>

#include "linear.hpp"

namespace xtu {
namespace l4 {

using lin::LinearArgs;

// as the formats of the expert layer
enum Format : int { kMx = 2, kNv = 3, kI4 = 4 };

struct Linear4Args {
  LinearArgs e;           // x, sizes, epilogue; w and ldw unused
  const uint8_t* w;       // records
  const float* gs;        // NVFP4: [1], swiglu [2] (gate, up); else null
  int fmt, group;
  int xvec;               // rows of x start on 16 bytes, K % 8 == 0
};

__host__ __device__ constexpr int scale_bytes(int fmt, int group) {
  return fmt == kMx ? 64 : fmt == kNv ? 128 : 8192 / group;
}
__host__ __device__ constexpr int record_bytes(int fmt, int group) {
  return 1024 + scale_bytes(fmt, group);
}
__host__ __device__ __forceinline__ int blocks_of(int K) { return (K + 127) / 128; }
// 16-row panels of a half (swiglu: of the gate half; else of all rows)
__host__ __device__ __forceinline__ int panels_of(int N) { return (N + 15) / 16; }

// Eight two's complement nibbles of a dword, low nibble first, as bf16 pairs of v / 16:
// the converter reads a byte's low four bits as a fraction.
__device__ __forceinline__ u32x4_t i4x8_to_bf16(uint32_t w) {
  const uint32_t o = w >> 4;
  u32x4_t r;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const float lo = __builtin_amdgcn_cvt_off_f32_i4((int)(w >> (8 * b)));
    const float hi = __builtin_amdgcn_cvt_off_f32_i4((int)(o >> (8 * b)));
    r[b] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  }
  return r;
}

// A lane's part of a record as it lies in memory.
template <int FMT, int G>
struct Raw {
  u32x4_t c;
  uint32_t s;
};
template <int G>
struct Raw<kI4, G> {
  u32x4_t c;
  f32x4_t s[128 / G];   // of the four rows that the lane's sums are of
};

// row: the row that the lane's codes are of; srow: the first of its sums' four.
template <int FMT, int G>
__device__ __forceinline__ Raw<FMT, G> load_raw(const uint8_t* rec, int q, int row, int srow) {
  Raw<FMT, G> r;
  r.c = *reinterpret_cast<const u32x4_t*>(rec + (16 * q + row) * 16);
  const uint8_t* sc = rec + 1024;
  if constexpr (FMT == kMx) {
    r.s = *reinterpret_cast<const uint32_t*>(sc + 4 * row);
  } else if constexpr (FMT == kNv) {
    r.s = *reinterpret_cast<const uint32_t*>(sc + 64 * (q / 2) + 4 * row);
  } else {
#pragma unroll
    for (int g = 0; g < 128 / G; ++g)
      r.s[g] = *reinterpret_cast<const f32x4_t*>(sc + 64 * g + 4 * srow);
  }
  return r;
}

// The MFMA operand of dword j.
template <int FMT, int G>
__device__ __forceinline__ u32x4_t operand(const Raw<FMT, G>& r, int j) {
  if constexpr (FMT == kI4) {
    return i4x8_to_bf16(r.c[j]);
  } else {
    uint32_t o[4];
    // (the converter takes the exponent bits alone: a byte 0 means 2^-127 to it)
    if constexpr (FMT == kMx)
      fp4x8_to_bf16(r.c[j], __uint_as_float((j < 3 ? r.s << (23 - 8 * j) : r.s >> 1) & 0x7f800000u), o);
    else fp4x8_to_bf16_mul(r.c[j], e4m3_to_f32(r.s >> (8 * j)), o);
    return u32x4_t{o[0], o[1], o[2], o[3]};
  }
}

// One block of NP panels times MT blocks of 16 rows of x; x(j, mt) gives the operand
// of dword j.  acc[p][mt] += the products.
template <int FMT, int G, int NP, int MT, class X>
__device__ __forceinline__ void multiply(const Raw<FMT, G> (&r)[NP], f32x4_t (&acc)[NP][MT], X x) {
  constexpr int GM = FMT == kI4 ? G / 32 : 4;   // MFMAs that share a scale
#pragma unroll
  for (int g = 0; g < 4 / GM; ++g) {
    f32x4_t t[NP][MT];
#pragma unroll
    for (int jj = 0; jj < GM; ++jj) {
      const int j = GM * g + jj;
      u32x4_t xv[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) xv[mt] = x(j, mt);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const bf16x8_t w = as_bf16x8(operand(r[p], j));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          if constexpr (FMT == kI4) {
            const f32x4_t z = {0.f, 0.f, 0.f, 0.f};
            t[p][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, as_bf16x8(xv[mt]),
                                                               jj ? t[p][mt] : z, 0, 0, 0);
          } else {
            acc[p][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, as_bf16x8(xv[mt]), acc[p][mt],
                                                                 0, 0, 0);
          }
        }
      }
    }
    if constexpr (FMT == kI4) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[p][mt][e] = __builtin_fmaf(t[p][mt][e], r[p].s[g][e], acc[p][mt][e]);
    }
  }
}

// Eight k of a row of x, zeros past K.
__device__ __forceinline__ u32x4_t load_x8(const Linear4Args& a, const uint16_t* row, int k) {
  if (a.xvec) {
    u32x4_t v = {0u, 0u, 0u, 0u};
    if (k < a.e.K) v = *reinterpret_cast<const u32x4_t*>(row + k);
    return v;
  }
  return lin::load8(row, k, a.e.K);
}

// At most 16 rows of x, all of x in LDS.
constexpr size_t kSkinny4Lds = 120 * 1024;
bool skinny4_fits(const LinearArgs& e);
hipError_t launch4_skinny(const Linear4Args& a, hipStream_t stream);

// At most 64 rows of x.
bool rows4_fits(const LinearArgs& e);
hipError_t launch4_rows(const Linear4Args& a, hipStream_t stream);

struct Plan4 {
  int kind, split;   // kind: blocks of 16 rows of a tile
};
Plan4 plan4_tile(int M, int N, int K, bool gated, bool may_split);
hipError_t launch4_tile(const Plan4& p, const Linear4Args& a, float* part, hipStream_t stream);

// f(format, group, gated) with the three as constants.
template <class F>
hipError_t by_format(const Linear4Args& a, F f) {
  const auto g = [&](auto fmt, auto group) {
    return a.e.act == lin::kSwiglu ? f(fmt, group, std::true_type{}) : f(fmt, group, std::false_type{});
  };
  if (a.fmt == kMx) return g(std::integral_constant<int, kMx>{}, std::integral_constant<int, 32>{});
  if (a.fmt == kNv) return g(std::integral_constant<int, kNv>{}, std::integral_constant<int, 16>{});
  if (a.group == 32) return g(std::integral_constant<int, kI4>{}, std::integral_constant<int, 32>{});
  if (a.group == 64) return g(std::integral_constant<int, kI4>{}, std::integral_constant<int, 64>{});
  return g(std::integral_constant<int, kI4>{}, std::integral_constant<int, 128>{});
}

}  // namespace l4
}  // namespace xtu
