// The dense product on matrix tiles staged through LDS (linear.hpp has the
// formula).  A workgroup computes BM rows of x times BN rows of w, K in steps
// of BK; the loads go from global memory straight to LDS, STAGES - 1 steps
// ahead of the MFMAs.
//
// LDS: a stage holds BM + BN rows of BK k, x rows first.  The 16-byte pieces of
// a row are permuted by the row (slot_of).  A 16-byte LDS read serves 16 lanes
// at once: lanes 0-3, 12-15 and 20-27, then 4-11, 16-19 and 28-31, and the same
// of the upper half.  Lane l reads row l % MB of a block, piece l / MB, and with
// these slots the 16 lanes touch all 64 banks once: 4.2 cycles a read instead of
// 8.2 (p ^ (r & 7) with MB = 32).  The loads write LDS linearly, so the
// permutation is in each lane's global address.  Pieces past K are loaded out of
// the buffer's range, which gives zeros; rows past M or N repeat the last row and
// are not written.
//
// The MFMA takes w as its A operand and x as B: a lane then holds four
// consecutive output columns of one row, which the epilogue reads and writes
// as vectors.  swiglu: the w rows of a tile alternate between gate and up in
// blocks of 32 (16 on the 16-row blocks), so both products of an element sit
// in one lane.
#include "linear.hpp"

namespace xtu {
namespace lin {
namespace {

// Slot of piece p of row r in an LDS row of PCS pieces, for MB rows a read.
template <int PCS, int MB>
__device__ __forceinline__ int slot_of(int p, int r) {
  static_assert(PCS == 8 || (PCS == 16 && MB == 16), "rows of 128 or 256 bytes");
  if (PCS == 16) return p ^ (r & 7) << 1;
  return p ^ (r & 7) ^ (MB == 32 ? r >> 4 & 1 : 0);
}

// LDS row of the epilogue's sums, in floats (16 bytes of padding: eight
// lanes' 16-byte writes to consecutive rows touch all banks).
template <int WN>
__host__ __device__ constexpr int epi_ld() { return WN + 4; }

template <int MB>
struct AccOf { typedef f32x16_t type; };
template <>
struct AccOf<16> { typedef f32x4_t type; };

// WM x WN of x rows x w rows per wave, in MB x MB blocks (MB 32: the 32x32x16
// MFMA, 16: 16x16x32).  SPLIT: the K range of blockIdx.y only, fp32 sums to
// a plane of the workspace [split][M][w rows] (finished by linear_join_kernel).
template <int BM, int BN, int WM, int WN, int MB, int BK, int STAGES, bool PIPE, int AK,
          bool SPLIT, int OCC>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64, OCC) void linear_tile_kernel(
    LinearArgs a, int kstep_per, float* part) {
  constexpr bool GATED = AK == kActSwiglu;
  constexpr int WAVES = BM / WM * (BN / WN), NT = WAVES * 64;
  constexpr int PCS = BK / 8, LROW = BK * 2;   // 16-byte pieces and bytes of an LDS row
  constexpr int ROWS = BM + BN, STAGE = ROWS * LROW;
  constexpr int LOADS = ROWS * PCS / NT;       // per thread and step
  constexpr int LEAD = STAGES - 1;
  constexpr int NI = WN / MB, NJ = WM / MB;   // blocks of a wave
  constexpr int KK = MB == 32 ? 16 : 32;      // k of an MFMA
  constexpr int NB = GATED ? BN / 2 : BN;     // output columns of the tile
  static_assert(ROWS * PCS % NT == 0 && BM * PCS % 64 == 0, "whole waves of loads");
  static_assert(!PIPE || (BK / KK) % 2 == 0, "two sets of fragments in turn");
  static_assert((STAGES - 1) * LOADS <= 63, "vmcnt");
  static_assert(!GATED || NI % 2 == 0, "gate and up blocks pair up in a wave");
  typedef typename AccOf<MB>::type acc_t;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid % 64;
  const int w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int wn = w % (BN / WN), wm = w / (BN / WN);

  // tile: contiguous ranges of tiles per XCD (workgroup b runs on XCD b % 8),
  // eight m tiles side by side so that concurrent workgroups share rows of both
  const int gm = (a.M + BM - 1) / BM, gn = (a.N + NB - 1) / NB, total = gm * gn;
  int t = blockIdx.x;
  {
    const int per = total / 8, rem = total % 8, x = t % 8;
    t = x * per + min(x, rem) + t / 8;
  }
  const int grp = t / (8 * gn), rows_g = min(8, gm - 8 * grp), in_g = t - grp * 8 * gn;
  const int m0 = (grp * 8 + in_g % rows_g) * BM, n0 = in_g / rows_g * NB;

  // k steps of this workgroup
  const int nk = (a.K + BK - 1) / BK;
  const int s0 = SPLIT ? (int)blockIdx.y * kstep_per : 0;
  const int s1 = SPLIT ? min(nk, s0 + kstep_per) : nk;

  const int mrows = min(BM, a.M - m0);
  const u32x4_t xr = raw_buffer(a.x + (long)m0 * a.ldx,
                                (uint32_t)(((long)(mrows - 1) * a.ldx + a.K) * 2));
  // w rows of the tile: from its first row, swiglu the same of the up half too
  const int ncols = min(NB, a.N - n0);
  const uint32_t wbytes = (uint32_t)(((long)(ncols - 1) * a.ldw + a.K) * 2);
  const u32x4_t wr = raw_buffer(a.w + (long)n0 * a.ldw, wbytes);
  const u32x4_t ur = GATED ? raw_buffer(a.w + (long)(a.N + n0) * a.ldw, wbytes) : wr;

  // load j of a step takes rows RPJ j and on, RPW of them a wave, a piece a lane:
  // all of x or all of w.  swiglu: gate or up goes by the wave, or by j
  constexpr int RPW = 64 / PCS, RPJ = RPW * WAVES;
  static_assert(BM % RPJ == 0 && BN % RPJ == 0, "a load is of x or of w");
  static_assert(!GATED || RPJ % (2 * MB) == 0 || RPJ == MB, "a wave's load is of gate or of up");
  uint32_t off[LOADS];
  int kof[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = RPJ * j + RPW * w + lane / PCS;
    const int p = slot_of<PCS, MB>(lane % PCS, RPJ * j % 32 + RPW * w + lane / PCS);
    kof[j] = 8 * p;
    if (RPJ * j < BM) {
      off[j] = (uint32_t)min(r, mrows - 1) * (uint32_t)(a.ldx * 2) + 16 * p;
    } else {
      const int rr = r - BM;
      const int col = GATED ? rr / (2 * MB) * MB + rr % MB : rr;
      off[j] = (uint32_t)min(col, ncols - 1) * (uint32_t)(a.ldw * 2) + 16 * p;
    }
  }
  const u32x4_t wave_wr = GATED && RPW * w / MB % 2 ? ur : wr;
  const int kend = min(a.K, BK * s1);
  auto issue_one = [&](int s, int st, int j) {
    const uint32_t o = kof[j] < kend - BK * s ? off[j] : 0x80000000u;
    const uint8_t* to = lds + st * STAGE + (WAVES * j + w) * 1024;
    // (past the end the last step's, which stays inside the buffer: the range
    // check is of o against what is left of it)
    const uint32_t k = (uint32_t)min(s, s1 - 1) * (uint32_t)LROW;
    if (RPJ * j < BM) buf_to_lds(xr, o, k, to);
    else if (GATED && RPJ == MB) buf_to_lds((RPJ * j - BM) / MB % 2 ? ur : wr, o, k, to);
    else buf_to_lds(wave_wr, o, k, to);
  };
  auto issue = [&](int s, int st) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) issue_one(s, st, j);
  };

  // The epilogue's part of the wave.  Vectors: CG lanes along a row, RS rows at a
  // time, BT such in one pass; single columns: RS1 rows, BT1 such.  A wave of one
  // row block reads what it needs beside the sums here, ahead of the operands.
  constexpr int W = GATED ? WN / 2 : WN;   // output columns of the wave
  constexpr int CG = W / 4, RS = 64 / CG, IT = MB / RS, RS1 = 64 / W, IT1 = MB / RS1;
  constexpr int BT = IT < 4 ? IT : AK == kActOther ? 2 : 4, BT1 = 4;
  constexpr bool PRE = NJ == 1 && !SPLIT;
  static_assert(IT1 % BT1 == 0 && (!PRE || IT == BT), "whole passes");
  const int nw = n0 + W * wn, mw = m0 + WM * wm;
  const int cv = lane % CG * 4, nv = nw + cv;   // a lane's four columns
  const int c1 = lane % W, n1 = nw + c1;        // or its single one
  u32x4_t bz = {0u, 0u, 0u, 0u}, bu = bz;
  Row4 pre[PRE ? IT : 1];
  Row1 pre1[PRE ? IT1 : 1];
  if (!SPLIT && a.vec && nv < a.N) {
    load_bias4<AK>(a, nv, bz, bu);
    if constexpr (PRE)
#pragma unroll
      for (int b = 0; b < IT; ++b)
        pre[b] = load_row4(a, min(mw + b * RS + lane / CG, a.M - 1), nv);
  }
  if (!SPLIT && !a.vec && n1 < a.N) {
    if (a.bias) {
      bz[0] = load_raw1(a.bias, n1, a.bias_bf16);
      if constexpr (GATED) bu[0] = load_raw1(a.bias, (long)a.N + n1, a.bias_bf16);
    }
    if constexpr (PRE)
#pragma unroll
      for (int b = 0; b < IT1; ++b)
        pre1[b] = load_row1(a, min(mw + b * RS1 + lane / W, a.M - 1), n1);
  }

  acc_t acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int k = 0; k < (MB == 32 ? 16 : 4); ++k) acc[i][j][k] = 0.f;

  const int rl = lane % MB, h = lane / MB;   // row of a block, k group of 8
  const uint8_t* xb = lds + (WM * wm + rl) * LROW;
  const uint8_t* wb = lds + (BM + WN * wn + rl) * LROW;
  struct Frags {
    u32x4_t w[NI], x[NJ];
  };
  // fragment f of k group kk: w block f, then x block f - NI
  auto read_one = [&](Frags& fr, int st, int kk, int f) {
    const int o = st * STAGE + slot_of<PCS, MB>(kk * (KK / 8) + h, rl) * 16;
    if (f < NI) fr.w[f] = *reinterpret_cast<const u32x4_t*>(wb + o + f * MB * LROW);
    else fr.x[f - NI] = *reinterpret_cast<const u32x4_t*>(xb + o + (f - NI) * MB * LROW);
  };
  auto mma_one = [&](const Frags& fr, int n) {
    const int i = n / NJ, j = n % NJ;
    if constexpr (MB == 32)
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(fr.w[i]), as_bf16x8(fr.x[j]),
                                                          acc[i][j], 0, 0, 0);
    else
      acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(fr.w[i]), as_bf16x8(fr.x[j]),
                                                          acc[i][j], 0, 0, 0);
  };

  if constexpr (!PIPE) {
    // Step s: wait for its loads (the later LEAD - 1 steps' may be in
    // flight), meet the barrier (every wave is done with step s - 1, whose
    // stage the loads of step s + LEAD take), issue them, multiply.
#pragma unroll
    for (int p = 0; p < LEAD; ++p)
      if (s0 + p < s1) issue(s0 + p, p);
    int st = 0, sl = LEAD % STAGES;
    for (int s = s0; s < s1; ++s) {
      if (s + LEAD <= s1) __builtin_amdgcn_s_waitcnt(wait_vm((LEAD - 1) * LOADS));
      else __builtin_amdgcn_s_waitcnt(wait_vm(0));
      __syncthreads();
      if (s + LEAD < s1) issue(s + LEAD, sl);
#pragma unroll
      for (int kk = 0; kk < BK / KK; ++kk) {
        Frags fr;
#pragma unroll
        for (int f = 0; f < NI + NJ; ++f) read_one(fr, st, kk, f);
#pragma unroll
        for (int n = 0; n < NI * NJ; ++n) mma_one(fr, n);
      }
      st = st + 1 == STAGES ? 0 : st + 1;
      sl = sl + 1 == STAGES ? 0 : sl + 1;
    }
  } else {
    // 16 x 16 blocks: 361 us at 8192 x 4096 x 7168, in 32 x 32 ones 378, though
    // half the fragment registers are then enough; four waves of 128 x 128 with
    // 32 x 32 blocks, which read LDS less, take 393.
    // The barrier sits before a step's last k group: by then the fragments of
    // all its groups are read (each group's between the MFMAs of the one
    // before), so behind it the loads of step s + STAGES may take its stage;
    // step s + 1 has landed, and its group 0 is read between the last group's
    // MFMAs, as are the loads issued.  The MFMAs wait for nothing but the
    // barrier itself.
    constexpr int M = NI * NJ, R = NI + NJ, KG = BK / KK;
    // reads of a group behind its n'th MFMA, in the order of their use: the
    // last quarter of the MFMAs covers their latency
    auto read_at = [&](Frags& fr, int stage, int g, int n) {
#pragma unroll
      for (int k = n * R * 4 / (3 * M); k < min(R, (n + 1) * R * 4 / (3 * M)); ++k)
        read_one(fr, stage, g, k == 0 ? 0 : k <= NJ ? NI + k - 1 : k - NJ);
    };
#pragma unroll
    for (int p = 0; p < STAGES; ++p) issue(s0 + p, p);
    __builtin_amdgcn_s_waitcnt(wait_vm((STAGES - 1) * LOADS));
    __syncthreads();
    Frags f[2];
#pragma unroll
    for (int k = 0; k < R; ++k) read_one(f[0], 0, 0, k);
    int st = 0;
    for (int s = s0; s < s1; ++s) {
#pragma unroll
      for (int g = 0; g + 1 < KG; ++g)
#pragma unroll
        for (int n = 0; n < M; ++n) {
          mma_one(f[g & 1], n);
          read_at(f[(g + 1) & 1], st, g + 1, n);
          __builtin_amdgcn_sched_barrier(0);
        }
      // step s + 1 landed (the STAGES - 2 after it may be in flight), the reads done
      __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((STAGES - 2) * LOADS));
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      const int nst = st + 1 == STAGES ? 0 : st + 1;
#pragma unroll
      for (int n = 0; n < M; ++n) {
        mma_one(f[(KG - 1) & 1], n);
        // (the last step reads what lies in the next stage; not used)
        read_at(f[0], nst, 0, n);
        // (between the first quarter: spread over all of the group's MFMAs
        // 361 us become 376 at 8192 x 4096 x 7168, over two groups 397)
#pragma unroll
        for (int d = n * LOADS * 4 / M; d < min(LOADS, (n + 1) * LOADS * 4 / M); ++d)
          issue_one(s + STAGES, st, d);
        __builtin_amdgcn_sched_barrier(0);
      }
      st = nst;
    }
    __builtin_amdgcn_s_waitcnt(wait_vm(0));   // (loads past the end bring zeros)
  }

  // Epilogue, MB rows of x at a time: the wave lays its sums out as rows in
  // its own part of LDS, then takes them with consecutive lanes along a row
  // (whole lines to memory).  The loops stay rolled (ActKind).
  constexpr int LD = epi_ld<WN>();
  __syncthreads();   // every wave is done with the stages
  float* eb = reinterpret_cast<float*>(lds) + w * (MB * LD);
  float* plane = SPLIT ? part + (long)blockIdx.y * part_plane(a) : nullptr;
#pragma unroll 1
  for (int j = 0; j < NJ; ++j) {
    lds_order();
#pragma unroll
    for (int jj = 0; jj < NJ; ++jj) {
      if (jj != j) continue;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int g = 0; g < (MB == 32 ? 4 : 1); ++g) {
          const f32x4_t v = {acc[i][jj][4 * g], acc[i][jj][4 * g + 1], acc[i][jj][4 * g + 2],
                             acc[i][jj][4 * g + 3]};
          *reinterpret_cast<f32x4_t*>(eb + rl * LD + MB * i + (MB == 32 ? 8 * g : 0) + 4 * h) = v;
        }
    }
    lds_order();
    const int mb = mw + MB * j;
    // column col of the wave: its gate (or only) sum's place in the row
    const auto place = [&](int col) { return GATED ? col / MB * 2 * MB + col % MB : col; };
    if (a.vec) {
      // what BT rows need is read before any is written
#pragma unroll 1
      for (int it = 0; it < IT && nv < a.N; it += BT) {
        f32x4_t z[BT], u[BT];
        Row4 x[BT];
        const int r = it * RS + lane / CG, m = mb + r;
#pragma unroll
        for (int b = 0; b < BT; ++b) {
          const float* row = eb + (r + b * RS) * LD + place(cv);
          z[b] = *reinterpret_cast<const f32x4_t*>(row);
          u[b] = z[b];
          if constexpr (GATED) u[b] = *reinterpret_cast<const f32x4_t*>(row + MB);
          if constexpr (PRE) x[b] = pre[b];
          else if constexpr (!SPLIT) x[b] = load_row4(a, min(m + b * RS, a.M - 1), nv);
        }
        if constexpr (!SPLIT) {
#pragma unroll
          for (int b = 0; b < BT; ++b) {
            z[b] += of_raw4(bz, a.bias_bf16);
            u[b] += of_raw4(bu, a.bias_bf16);
          }
          act_all<AK>(a, z, u);
        }
#pragma unroll
        for (int b = 0; b < BT; ++b) {
          if (m + b * RS >= a.M) break;
          if constexpr (SPLIT) {
            float* pr = plane + (long)(m + b * RS) * a.N * (GATED ? 2 : 1) + nv;
            *reinterpret_cast<f32x4_t*>(pr) = z[b];
            if constexpr (GATED) *reinterpret_cast<f32x4_t*>(pr + a.N) = u[b];
          } else {
            store_row4(a, m + b * RS, nv, z[b], x[b]);
          }
        }
      }
    } else {
      // the same by single columns
#pragma unroll PRE ? IT1 / BT1 : 1
      for (int it = 0; it < IT1; it += BT1) {
        if (n1 >= a.N) break;
        f32x4_t z[1], u[1];
        Row1 x[BT1];
        const int r = it * RS1 + lane / W, m = mb + r;
#pragma unroll
        for (int b = 0; b < BT1; ++b) {
          const float* row = eb + (r + b * RS1) * LD + place(c1);
          z[0][b] = row[0];
          u[0][b] = GATED ? row[MB] : 0.f;
          if constexpr (PRE) x[b] = pre1[it + b];
          else if constexpr (!SPLIT) x[b] = load_row1(a, min(m + b * RS1, a.M - 1), n1);
        }
        if constexpr (!SPLIT) {
          z[0] += of_raw1(bz[0], a.bias_bf16);
          u[0] += of_raw1(bu[0], a.bias_bf16);
          act_all<AK>(a, z, u);
#pragma unroll
          for (int b = 0; b < BT1; ++b) {
            if (a.scale) z[0][b] *= x[b].scale;
            if (a.res) z[0][b] += of_raw1(x[b].res, a.res_bf16);
          }
        }
#pragma unroll
        for (int b = 0; b < BT1; ++b) {
          const long mm = m + b * RS1;
          if (mm >= a.M) break;
          if constexpr (SPLIT) {
            float* pr = plane + mm * a.N * (GATED ? 2 : 1) + n1;
            pr[0] = z[0][b];
            if constexpr (GATED) pr[a.N] = u[0][b];
          } else if (a.out_bf16) {
            reinterpret_cast<uint16_t*>(a.out)[mm * a.ldo + n1] = f32_to_bf16(z[0][b]);
          } else {
            reinterpret_cast<float*>(a.out)[mm * a.ldo + n1] = z[0][b];
          }
        }
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, int MB, int BK, int STAGES, bool PIPE, int OCC>
hipError_t launch_tile(const LinearArgs& a, int split, float* part, hipStream_t stream) {
  const bool gated = a.act == kSwiglu;
  const int nb = gated ? BN / 2 : BN;
  const long gm = ((long)a.M + BM - 1) / BM, gn = ((long)a.N + nb - 1) / nb;
  const int nk = (a.K + BK - 1) / BK;
  const int per = (nk + split - 1) / split;
  split = (nk + per - 1) / per;   // no empty range
  constexpr int WAVES = BM / WM * (BN / WN), NT = WAVES * 64;
  constexpr size_t kStages = (size_t)STAGES * (BM + BN) * BK * 2;
  constexpr size_t kEpi = (size_t)WAVES * MB * epi_ld<WN>() * 4;
  constexpr size_t lds = kStages > kEpi ? kStages : kEpi;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  if (!grid_fits(gm * gn, NT)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)(gm * gn), (unsigned)split);
  void (*k)(LinearArgs, int, float*) = nullptr;
  if (split > 1)
    k = gated ? linear_tile_kernel<BM, BN, WM, WN, MB, BK, STAGES, PIPE, kActSwiglu, true, OCC>
              : linear_tile_kernel<BM, BN, WM, WN, MB, BK, STAGES, PIPE, kActNone, true, OCC>;
  else if (gated)
    k = linear_tile_kernel<BM, BN, WM, WN, MB, BK, STAGES, PIPE, kActSwiglu, false, OCC>;
  else if (a.act == kNone)
    k = linear_tile_kernel<BM, BN, WM, WN, MB, BK, STAGES, PIPE, kActNone, false, OCC>;
  else
    k = linear_tile_kernel<BM, BN, WM, WN, MB, BK, STAGES, PIPE, kActOther, false, OCC>;
  k<<<grid, NT, lds, stream>>>(a, per, part);
  hipError_t e = hipPeekAtLastError();
  if (e == hipSuccess && split > 1) e = launch_join(a, split, part, stream);
  return e;
}

}  // namespace

bool tile_fits(const LinearArgs& a) {
  const auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!al(a.x) || !al(a.w) || a.K % 8) return false;
  if ((a.M > 1 && a.ldx % 8) || a.ldw % 8) return false;
  // 32-bit offsets inside a tile
  return (256 * a.ldx + a.K) * 2 < (1L << 31) && (256 * a.ldw + a.K) * 2 < (1L << 31);
}

namespace {

// The variants: tile, k of a step, workgroups that share a CU, and what they
// cost on MI355X, in us: t[i] a step, o[i] a round beside its steps, with i + 1
// workgroups on a CU.  Fitted to products that fill the chip one to three times
// over at K = 256, 1024 and 4096 (64 x 64: one per CU 4.7 / 8.0 / 19.5, two
// 6.5 / 10.9 / 29.8; 128 x 128 in two stages, two per CU 13.1 / 23.8 / 73.0, in
// four stages, alone on its CU 9.3 / 15.1 / 42.5; 256 x 256: 23.9 / 40.5 / 117).
struct TileKind {
  int m, n, k, occ;
  float t[2], o[2];
};
constexpr TileKind kTileKinds[] = {
    {64, 32, 128, 1, {0.36f, 0.36f}, {1.3f, 1.3f}},
    {64, 64, 64, 2, {0.24f, 0.39f}, {1.9f, 2.3f}},
    {128, 64, 64, 2, {0.32f, 0.73f}, {3.1f, 1.8f}},
    {128, 128, 64, 2, {0.77f, 1.03f}, {2.6f, 5.0f}},
    {128, 128, 64, 1, {0.56f, 0.56f}, {3.7f, 3.7f}},
    {256, 256, 64, 1, {1.55f, 1.55f}, {11.0f, 11.0f}},
};
constexpr float kLaunch = 2.3f;
constexpr int kCus = 256;

}  // namespace

// The variant and K split with the least estimated time.  A split costs the
// second launch that adds the partial sums, and their way through memory.
TilePlan plan_tile(int M, int N, int K, bool gated, bool may_split) {
  TilePlan best{0, 1};
  float best_t = 1e30f;
  for (int kind = 0; kind < (int)(sizeof(kTileKinds) / sizeof(kTileKinds[0])); ++kind) {
    const TileKind& v = kTileKinds[kind];
    const int nb = gated ? v.n / 2 : v.n;
    const long tiles1 = (((long)M + v.m - 1) / v.m) * (((long)N + nb - 1) / nb);
    const int nk = (K + v.k - 1) / v.k;
    for (int split : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (split > 1 && (!may_split || nk < 2 * split || tiles1 >= 2 * kCus)) break;
      const int steps = (nk + split - 1) / split;
      const long tiles = tiles1 * ((nk + steps - 1) / steps);
      const long full = tiles / (kCus * v.occ), rem = tiles % (kCus * v.occ);
      float t = kLaunch + full * (v.t[v.occ - 1] * steps + v.o[v.occ - 1]);
      if (rem) {
        const int i = (int)((rem + kCus - 1) / kCus) - 1;
        t += v.t[i] * steps + v.o[i];
      }
      if (split > 1) t += 3.0f + 2.0f * split * M * (float)N * (gated ? 2 : 1) * 4.0f / 5e6f;
      if (t < best_t) {
        best_t = t;
        best = TilePlan{kind, split};
      }
    }
  }
  return best;
}

hipError_t launch_tile_kind(int kind, const LinearArgs& a, int split, float* part,
                            hipStream_t stream) {
  switch (kind) {
    case 0: return launch_tile<64, 32, 16, 32, 16, 128, 4, false, 1>(a, split, part, stream);
    case 1: return launch_tile<64, 64, 16, 32, 16, 64, 4, true, 4>(a, split, part, stream);
    case 2: return launch_tile<128, 64, 32, 32, 16, 64, 3, true, 4>(a, split, part, stream);
    case 3: return launch_tile<128, 128, 32, 64, 16, 64, 2, true, 4>(a, split, part, stream);
    case 4: return launch_tile<128, 128, 64, 32, 16, 64, 4, true, 2>(a, split, part, stream);
    case 5: return launch_tile<256, 256, 128, 64, 16, 64, 2, true, 2>(a, split, part, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace lin
}  // namespace xtu
