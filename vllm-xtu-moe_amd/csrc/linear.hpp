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
  int vec;                // bias, residual and out take vectors of 4 elements
};

// Split K: the partial sums of one split, [M][rows of w] fp32.
__host__ __device__ __forceinline__ long part_plane(const LinearArgs& a) {
  return (long)a.M * a.N * (a.act == kSwiglu ? 2 : 1);
}

// NaN stays NaN in every activation (relu: the comparison is false for it).
// __expf is 2^(z log2 e) on the exponential unit, also where the output is fp32: its
// argument's rounding leaves a relative error of |z| 2^-24 beside the unit's own.
// In 1 / (1 + e^-z) that shows for negative z only, where the result is about e^z
// (z = -16: 2^-20 of 1e-7); the exp without it is longer code, which an epilogue
// pays for (ActKind).
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

// What a kernel's epilogue is compiled for: no activation, swiglu, or any of
// the others (chosen at run time).  An epilogue's code is run through once per
// tile, so its size counts: instructions fetched for the first time cost more
// than they take to run (a 256 x 256 tile's epilogue took 24 us with every
// activation inlined at each of its four row blocks).
enum ActKind : int { kActNone = 0, kActSwiglu, kActOther };

template <int AK>
__device__ __forceinline__ float act_of(const LinearArgs& a, float z, float u) {
  if constexpr (AK == kActNone) return z;
  else if constexpr (AK == kActSwiglu) return silu_gate(z, u, a.limit, a.alpha, a.beta);
  else return activate(a.act, z);
}

// One output element from its product(s): z, and for swiglu the up product u.
template <int AK>
__device__ __forceinline__ void finish_one(const LinearArgs& a, int m, int n, float z, float u) {
  if (a.bias) {
    z += load_bias(a, n);
    if constexpr (AK == kActSwiglu) u += load_bias(a, a.N + n);
  }
  float y = act_of<AK>(a, z, u);
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

// What an epilogue reads ahead stays as it is in memory until it is used: to
// convert it is to wait for it.
__device__ __forceinline__ u32x4_t load_raw4(const void* p, long o, int is_bf16) {
  if (!is_bf16) return *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const float*>(p) + o);
  const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + o);
  return u32x4_t{v.x, v.y, 0u, 0u};
}

__device__ __forceinline__ f32x4_t of_raw4(u32x4_t v, int is_bf16) {
  if (!is_bf16) return __builtin_bit_cast(f32x4_t, v);
  return f32x4_t{__uint_as_float(v[0] << 16), __uint_as_float(v[0] & 0xffff0000u),
                 __uint_as_float(v[1] << 16), __uint_as_float(v[1] & 0xffff0000u)};
}

__device__ __forceinline__ uint32_t load_raw1(const void* p, long o, int is_bf16) {
  return is_bf16 ? reinterpret_cast<const uint16_t*>(p)[o] : reinterpret_cast<const uint32_t*>(p)[o];
}

__device__ __forceinline__ float of_raw1(uint32_t v, int is_bf16) {
  return __uint_as_float(is_bf16 ? v << 16 : v);
}

// Four columns' bias: of z, and for swiglu of u.
template <int AK>
__device__ __forceinline__ void load_bias4(const LinearArgs& a, int n, u32x4_t& bz, u32x4_t& bu) {
  bz = bu = u32x4_t{0u, 0u, 0u, 0u};   // zero in both types
  if (!a.bias) return;
  bz = load_raw4(a.bias, n, a.bias_bf16);
  if constexpr (AK == kActSwiglu) bu = load_raw4(a.bias, a.N + n, a.bias_bf16);
}

// What the epilogue of four columns of a row reads, and of a single one.
struct Row4 {
  u32x4_t res;
  float scale;
};
struct Row1 {
  uint32_t res;
  float scale;
};

__device__ __forceinline__ Row4 load_row4(const LinearArgs& a, int m, int n) {
  Row4 r = {{0u, 0u, 0u, 0u}, 1.f};
  if (a.res) r.res = load_raw4(a.res, (long)m * a.ldr + n, a.res_bf16);
  if (a.scale) r.scale = a.scale[(long)m * a.sstride];
  return r;
}

__device__ __forceinline__ Row1 load_row1(const LinearArgs& a, int m, int n) {
  Row1 r = {0u, 1.f};
  if (a.res) r.res = load_raw1(a.res, (long)m * a.ldr + n, a.res_bf16);
  if (a.scale) r.scale = a.scale[(long)m * a.sstride];
  return r;
}

// z[] = act(z[], u[]), the choice of an activation outside the loops.
template <int AK, int C>
__device__ __forceinline__ void act_all(const LinearArgs& a, f32x4_t (&z)[C], f32x4_t (&u)[C]) {
  const auto each = [&](auto f) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) z[c][e] = f(z[c][e], u[c][e]);
  };
  if constexpr (AK == kActSwiglu) {
    each([&](float g, float v) { return silu_gate(g, v, a.limit, a.alpha, a.beta); });
  } else if constexpr (AK == kActOther) {
    switch (a.act) {
      case kRelu: each([](float g, float) { return activate(kRelu, g); }); break;
      case kSilu: each([](float g, float) { return activate(kSilu, g); }); break;
      case kGelu: each([](float g, float) { return activate(kGelu, g); }); break;
      case kGeluTanh: each([](float g, float) { return activate(kGeluTanh, g); }); break;
      case kSigmoid: each([](float g, float) { return activate(kSigmoid, g); }); break;
    }
  }
}

__device__ __forceinline__ void store_row4(const LinearArgs& a, int m, int n, f32x4_t y,
                                           const Row4& r) {
  if (a.scale) y *= r.scale;
  if (a.res) y += of_raw4(r.res, a.res_bf16);
  const long o = (long)m * a.ldo + n;
  if (a.out_bf16) {
    uint2 v;
    v.x = f32_to_bf16(y[0]) | (uint32_t)f32_to_bf16(y[1]) << 16;
    v.y = f32_to_bf16(y[2]) | (uint32_t)f32_to_bf16(y[3]) << 16;
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + o) = v;
  } else {
    *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(a.out) + o) = y;
  }
}

// Columns n .. n + 3 of row m, all of them there (a.vec: N % 4 == 0).
template <int AK>
__device__ __forceinline__ void finish4(const LinearArgs& a, int m, int n, f32x4_t z, f32x4_t u) {
  u32x4_t bz, bu;
  load_bias4<AK>(a, n, bz, bu);
  const Row4 r = load_row4(a, m, n);
  f32x4_t zz[1] = {z + of_raw4(bz, a.bias_bf16)}, uu[1] = {u + of_raw4(bu, a.bias_bf16)};
  act_all<AK>(a, zz, uu);
  store_row4(a, m, n, zz[0], r);
}

// Order this wave's LDS writes before its later LDS reads by other lanes: a
// wave's LDS instructions execute in issue order, so only the compiler must
// not move them.
__device__ __forceinline__ void lds_order() {
  __builtin_amdgcn_wave_barrier();
  __asm__ __volatile__("" ::: "memory");
}

// 16 bytes at p, which need only be a multiple of 2 bytes.  Loads that start on
// a word run at the speed of aligned ones, others at less than half (2467 rows of
// 6341 values, two rows of x: 24.4 us, 11.1 for 6342); the five words around them
// and a shift take 15.1.  A word that holds a byte of the row is inside its
// allocation.
typedef unsigned int u32x4_w __attribute__((ext_vector_type(4), aligned(4)));

struct Words5 {
  u32x4_t v;
  uint32_t t;
};

__device__ __forceinline__ Words5 load_words(const uint8_t* p, uint32_t shift) {
  const uint8_t* a = p - shift;   // shift = 2 where p is no multiple of 4, else 0
  Words5 r;
  r.v = *reinterpret_cast<const u32x4_w*>(a);
  r.t = *reinterpret_cast<const uint32_t*>(a + (shift ? 16 : 0));
  return r;
}

__device__ __forceinline__ u32x4_t shifted(const Words5& r, uint32_t shift) {
  return u32x4_t{__builtin_amdgcn_alignbyte(r.v[1], r.v[0], shift),
                 __builtin_amdgcn_alignbyte(r.v[2], r.v[1], shift),
                 __builtin_amdgcn_alignbyte(r.v[3], r.v[2], shift),
                 __builtin_amdgcn_alignbyte(r.t, r.v[3], shift)};
}

// Eight consecutive k of one row from k on, zeros past K; any alignment.  SHIFT:
// by load_words, for streams; else one load that the hardware splits, for code
// that waits for its loads anyway (two loads of each cost it more).
template <bool SHIFT = false>
__device__ __forceinline__ u32x4_t load8(const uint16_t* row, int k, int K) {
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (k + 8 <= K) {
    if constexpr (SHIFT) {
      const uint8_t* p = reinterpret_cast<const uint8_t*>(row + k);
      const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(p) & 2u;
      v = shifted(load_words(p, shift), shift);
    } else {
      __builtin_memcpy(&v, row + k, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) v[i / 2] |= (uint32_t)row[k + i] << (16 * (i % 2));
  }
  return v;
}

// 16 bytes per lane to LDS at dst + 16 * lane, from the buffer's base + off +
// soff (zeros out of range).
__device__ __forceinline__ void buf_to_lds(u32x4_t rsrc, uint32_t off, uint32_t soff,
                                           const uint8_t* dst) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
               :: "v"(off), "s"(rsrc), "s"(soff), "{m0}"((uint32_t)(uintptr_t)dst)
               : "memory");
}

// Raw buffer over [base, base + bytes), wave-uniform.
__device__ __forceinline__ u32x4_t raw_buffer(const void* base, uint32_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  u32x4_t r = {(uint32_t)p, (uint32_t)(p >> 32) & 0xffffu, bytes, 0x00020000u};
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);
  return r;
}

// s_waitcnt immediates: vmcnt(n), and vmcnt(n) with lgkmcnt(0)
constexpr int wait_vm(int n) { return 0x0f70 | (n & 15) | ((n >> 4) << 14); }
constexpr int wait_vm_lgkm0(int n) { return 0x0070 | (n & 15) | ((n >> 4) << 14); }

// A launch has fewer than 2^32 threads along x.
__host__ inline bool grid_fits(long blocks, int threads) {
  return blocks * threads < (1L << 32);
}

struct TilePlan {
  int kind, split;
};
TilePlan plan_tile(int M, int N, int K, bool gated, bool may_split);
// Whether the tile kernels take the operands (16-byte rows, K % 8 == 0).
bool tile_fits(const LinearArgs& a);
// `split` K ranges; part: split * part_plane(a) floats when split > 1.
hipError_t launch_tile_kind(int kind, const LinearArgs& a, int split, float* part,
                            hipStream_t stream);
// At most 16 rows of x, all of x in LDS; any alignment.
constexpr int kSkinnyM = 16;
constexpr size_t kSkinnyLds = 120 * 1024;
bool skinny_fits(const LinearArgs& a);
hipError_t launch_skinny(const LinearArgs& a, hipStream_t stream);
hipError_t launch_any(const LinearArgs& a, hipStream_t stream);
hipError_t launch_join(const LinearArgs& a, int split, const float* part, hipStream_t stream);
// Rows of x at any alignment as rows of K rounded up to 8, zeros behind K.
hipError_t launch_pack_x(const uint16_t* x, long ldx, int M, int K, uint16_t* out,
                         hipStream_t stream);

}  // namespace lin
}  // namespace xtu
