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
// (low nibble first; INT4: i4x8_to_bf16), which are an MFMA operand's.
// So an MFMA's 32 k are consecutive, x is read as it lies, and an INT4 group is whole
// MFMAs.  Then the record's scales, a dword of four for the lanes that share them:
//   MXFP4: [16 row][4 j] bytes        NVFP4: [2 q / 2][16 row][4 j] bytes
//   INT4:  fp32 [128 / G][16 row]
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

// Eight INT4 codes of a dword as bf16: k = b in byte b's low nibble, 4 + b in its high
// one.  Code c >= 8 is stored as c - 8 (v = 0 .. 7), c < 8 as 15 - c (8 + |v| - 1), so
// that a byte of sign and magnitude, 0 .. 8, takes a mask and two sums for four codes at
// once; as e4m3 that byte is v 2^-9 (subnormal, and 8 2^-9 the first normal), which the
// converter scales back.  15 instructions; the converter of single nibbles
// (v_cvt_off_f32_i4) needs fewer but runs at a quarter of the rate.
__device__ __forceinline__ u32x4_t i4x8_to_bf16(uint32_t w) {
  const uint32_t h0 = w >> 3 & 0x01010101u, h1 = w >> 7 & 0x01010101u;
  const uint32_t b0 = (h0 << 7) + ((w & 0x07070707u) + h0);
  const uint32_t b1 = (h1 << 7) + ((w >> 4 & 0x07070707u) + h1);
  const auto two = [](uint32_t b, auto hi) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(
                                            b, 512.f, decltype(hi)::value));
  };
  return u32x4_t{two(b0, std::false_type{}), two(b0, std::true_type{}),
                 two(b1, std::false_type{}), two(b1, std::true_type{})};
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

__device__ __forceinline__ float e4m3_of(uint32_t s, int j) {
  switch (j) {
    case 0: return __builtin_amdgcn_cvt_f32_fp8(s, 0);
    case 1: return __builtin_amdgcn_cvt_f32_fp8(s, 1);
    case 2: return __builtin_amdgcn_cvt_f32_fp8(s, 2);
    default: return __builtin_amdgcn_cvt_f32_fp8(s, 3);
  }
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
    else fp4x8_to_bf16_mul(r.c[j], e4m3_of(r.s, j), o);
    return u32x4_t{o[0], o[1], o[2], o[3]};
  }
}

// One block of NP panels times MT blocks of 16 rows of x; x(j, mt) gives the operand
// of dword j.  acc[p][mt] += the products.  after(): called behind the first dword's
// operands, when every record has been waited for.
template <int FMT, int G, int NP, int MT, class X, class A>
__device__ __forceinline__ void multiply(const Raw<FMT, G> (&r)[NP], f32x4_t (&acc)[NP][MT], X x,
                                         A after) {
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
      if (j == 0) after();
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

template <int FMT, int G, int NP, int MT, class X>
__device__ __forceinline__ void multiply(const Raw<FMT, G> (&r)[NP], f32x4_t (&acc)[NP][MT], X x) {
  multiply<FMT, G, NP, MT>(r, acc, x, [] {});
}

// Eight k of a row of x that starts on 16 bytes, zeros past K.
__device__ __forceinline__ u32x4_t load_x8(const Linear4Args& a, const uint16_t* row, int k) {
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (k < a.e.K) v = *reinterpret_cast<const u32x4_t*>(row + k);
  return v;
}

struct Shape4 {
  int M, N, K;
  bool gated;
  int fmt, group;
};

// The kernels, for rows of x on 16 bytes and in reach of 32-bit offsets, and the ranges
// of K that are summed apart.
enum Kind4 : int { kSkinny4 = 0, kBlock4, kSlab4, kWide2, kWide4 };
struct Plan4 {
  int kind, split;
};

// Up to 16 rows of x, all of it in LDS: units of `rows` output columns; grid 0: no.
struct SkinnyPlan {
  int rows, waves;
  long units, grid;
};
SkinnyPlan skinny4_plan(const Shape4& s);
hipError_t launch4_skinny(const Linear4Args& a, hipStream_t stream);
// Up to kBlockM rows of x, 4, 8, 16, 32, 48 or 64 to a workgroup, blocks of them a wave's
// own in LDS; `time` in us.
constexpr int kBlockM = 65536;
struct BlockPlan {
  int rows;
  float time;
};
BlockPlan block4_plan(const Shape4& s);
int block4_waves(const Shape4& s, int rows);
hipError_t launch4_block(const Linear4Args& a, hipStream_t stream);
// Up to 64 rows of x, a range of `per` blocks of K in LDS.
constexpr int kSlabWaves = 8;
constexpr size_t kSlabLds = 160 * 1024;
inline size_t slab4_lds(int M, int per) { return (size_t)((M + 3) / 4) * 1024 * per; }
hipError_t launch4_slab(const Linear4Args& a, int split, float* part, hipStream_t stream);
// More rows: tiles of 128 rows and 64 NP rows of w.
hipError_t launch4_wide(const Plan4& p, const Linear4Args& a, float* part, hipStream_t stream);
// Any rows, without a workspace.
hipError_t launch4_tile(const Linear4Args& a, hipStream_t stream);

inline Shape4 shape_of(const Linear4Args& a) {
  return Shape4{a.e.M, a.e.N, a.e.K, a.e.act == lin::kSwiglu, a.fmt, a.group};
}

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
