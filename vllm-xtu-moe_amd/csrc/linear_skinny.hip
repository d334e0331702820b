// The dense product for at most 16 rows of x (linear.hpp has the formula): a
// stream of w.  One workgroup of sixteen waves per panel of up to 16 output
// columns (further panels in steps of the grid); the waves split K (swiglu:
// eight on the gate rows, eight on the matching up rows) and their sums are
// added through LDS in a fixed order.  All of x sits in LDS.  A wave keeps U MFMA
// steps of 32 k of w in flight: a lane loads 16 bytes of its w row straight
// into the operand registers, and each slot is loaded again, for what comes U
// steps later, over panel ends too, as soon as it is used.  Rows past M or N
// repeat the last one; what they give is not written.
//
// Few columns: a CU takes in about 25 GB/s whatever its waves ask for, so a
// product of 256 columns by 7168 k in panels of 16 waits 14 us for 16 CUs; panels
// of fewer columns, down to two (the MFMA's other rows repeat the panel's last row,
// at no further traffic), for about one a CU take 6.6 us: 128 panels here, half the
// CUs.  512 gated columns by 2048 k 7.8 -> 5.1 us.  What such products wait for
// besides is x: every workgroup brings all of it to LDS before its first MFMA (4
// rows of 7168: 57 KB beside 28 KB of w).  Cached loads of w beat non-temporal ones here (28672
// columns by 7168 k 73 us = 5.65 TB/s against 91).
#include "linear.hpp"

namespace xtu {
namespace lin {
namespace {

constexpr int kSkW = 16;           // waves per workgroup
constexpr int kSkinnyGrid = 256;   // one workgroup per CU

// A slot of the stream: 16 bytes of a row that starts on a word (WORDS), or the
// five words around them.
template <bool WORDS>
struct Slot {
  u32x4_t v;
};
template <>
struct Slot<false> {
  Words5 v;
};

template <bool GATED, bool WORDS, int U>
__global__ __launch_bounds__(64 * kSkW) void linear_skinny_kernel(LinearArgs a, int rp) {
  constexpr int KW = GATED ? kSkW / 2 : kSkW;   // waves along K
  extern __shared__ __attribute__((aligned(16))) uint16_t xs[];   // [M][K32 + 8]
  __shared__ f32x4_t red[2][kSkW][64];
  const int tid = threadIdx.x, lane = tid % 64;
  const int w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int kw = GATED ? w % KW : w;
  const long up = GATED && w >= KW ? a.N : 0;   // first row of the wave's half
  const int q = lane / 16, c = lane % 16;
  const int npan = (a.N + rp - 1) / rp;
  // whole steps of 32 k, dealt to the waves; the partial last one, if any,
  // goes to the last wave along K
  const int nst = a.K / 32;
  const int s0 = kw * nst / KW, s1 = (kw + 1) * nst / KW;
  const int nch = max((s1 - s0 + U - 1) / U, 1);
  auto wbase = [&](int pan) { return a.w + (up + (long)rp * pan) * a.ldw; };
  auto woffs = [&](int pan) {
    return (uint32_t)(min(min(c, rp - 1), a.N - 1 - rp * pan) * a.ldw + 8 * q) * 2u;
  };
  // loads are unconditional (past the wave's range: its last step again, or
  // for a wave without steps the row's start, not used), so that every wait
  // is for exactly the slot about to be used
  Slot<WORDS> wv[U];
  const int k_last = max(s1 - 1, s0 > 0 ? s0 - 1 : 0);
  auto issue = [&](int i, const uint16_t* wb, uint32_t wo, int s) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(wb + 32L * min(s, k_last)) + wo;
    if constexpr (WORDS) wv[i].v = *reinterpret_cast<const u32x4_w*>(p);
    else wv[i].v = load_words(p, (uint32_t)reinterpret_cast<uintptr_t>(p) & 2u);
  };
  int pan = blockIdx.x;
  const uint16_t* wb = wbase(pan);
  uint32_t wo = woffs(pan);
  const bool any = nst > 0;   // K < 32: the partial step alone
  if (any) {
#pragma unroll
    for (int i = 0; i < U; ++i) issue(i, wb, wo, s0 + i);
  }
  __builtin_amdgcn_sched_barrier(0);   // x after the first loads of w
  // x to LDS, zeros behind K up to a whole step
  const int k32 = (a.K + 31) / 32 * 32, ldx = k32 + 8, per_row = k32 / 8;
  for (int p = tid; p < a.M * per_row; p += 64 * kSkW) {
    const int r = p / per_row, k = (p - r * per_row) * 8;
    *reinterpret_cast<u32x4_t*>(xs + r * ldx + k) = load8(a.x + (long)r * a.ldx, k, a.K);
  }
  __syncthreads();
  const uint16_t* xl = xs + min(c, a.M - 1) * ldx + 8 * q;

  for (int it = 0; pan < npan; pan += gridDim.x, ++it) {
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    // of this lane's row of the panel (k steps are whole words)
    const uint32_t wshift = ((uint32_t)reinterpret_cast<uintptr_t>(wb) + wo) & 2u;
    auto use = [&](int i, int s) {
      if (s < s1) {
        const u32x4_t xv = *reinterpret_cast<const u32x4_t*>(xl + 32 * s);
        u32x4_t v;
        if constexpr (WORDS) v = wv[i].v;
        else v = shifted(wv[i].v, wshift);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(v), as_bf16x8(xv), acc, 0, 0, 0);
      }
    };
    const int next = pan + (int)gridDim.x;
    const uint16_t* nb = wbase(next < npan ? next : pan);
    const uint32_t no = woffs(next < npan ? next : pan);
    if (any) {
      for (int ch = 0; ch + 1 < nch; ++ch) {
        const int s = s0 + ch * U;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          use(i, s + i);
          issue(i, wb, wo, s + U + i);
        }
      }
      const int s = s0 + (nch - 1) * U;
      if (next < npan) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          use(i, s + i);
          issue(i, nb, no, s0 + i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i) use(i, s + i);
      }
    }
    if (a.K % 32 && kw == KW - 1) {
      const u32x4_t tw =
          load8(wb + min(min(c, rp - 1), a.N - 1 - rp * pan) * a.ldw, 32 * nst + 8 * q, a.K);
      const u32x4_t tx = *reinterpret_cast<const u32x4_t*>(xl + 32 * nst);
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(tw), as_bf16x8(tx), acc, 0, 0, 0);
    }
    red[it & 1][w][lane] = acc;
    __syncthreads();   // the other half of red is written before the next barrier
    if (tid < 256) {
      const int e = tid / 64, nl = 4 * q + e, n = rp * pan + nl;
      float z = 0.f, u = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        z += red[it & 1][k][lane][e];
        if constexpr (GATED) u += red[it & 1][KW + k][lane][e];
      }
      if (c < a.M && nl < rp && n < a.N) finish_one<GATED ? kActSwiglu : kActOther>(a, c, n, z, u);
    }
    wb = nb;
    wo = no;
  }
}

size_t skinny_lds(const LinearArgs& a) { return (size_t)a.M * ((a.K + 31) / 32 * 32 + 8) * 2; }

template <bool GATED, bool WORDS>
hipError_t launch(const LinearArgs& a, hipStream_t stream) {
  int rp = 2;   // columns of a panel: about one panel per CU, 16 at most
  while (rp < 16 && (a.N + rp - 1) / rp > kSkinnyGrid) rp *= 2;
  const int npan = (a.N + rp - 1) / rp;
  const int grid = npan < kSkinnyGrid ? npan : kSkinnyGrid;
  const size_t lds = skinny_lds(a);
  // steps of a wave: U of them in flight
  const bool few = a.K / 32 <= 4 * (GATED ? kSkW / 2 : kSkW);
  auto k = few ? linear_skinny_kernel<GATED, WORDS, 4> : linear_skinny_kernel<GATED, WORDS, 8>;
  k<<<grid, 64 * kSkW, lds, stream>>>(a, rp);
  return hipPeekAtLastError();
}

}  // namespace

bool skinny_fits(const LinearArgs& a) {
  return a.M <= kSkinnyM && a.K <= (1 << 20) && skinny_lds(a) <= kSkinnyLds &&
         16 * a.ldw * 2 < (1L << 31);
}

hipError_t launch_skinny(const LinearArgs& a, hipStream_t stream) {
  const bool words = reinterpret_cast<uintptr_t>(a.w) % 4 == 0 && a.ldw % 2 == 0;
  if (a.act == kSwiglu) return words ? launch<true, true>(a, stream) : launch<true, false>(a, stream);
  return words ? launch<false, true>(a, stream) : launch<false, false>(a, stream);
}

}  // namespace lin
}  // namespace xtu
