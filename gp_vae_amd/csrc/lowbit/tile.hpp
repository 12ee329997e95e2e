// tile.hpp — the products of skinny.hpp for many rows: tiles of 64 rows x 128 outputs on the bf16 matrix pipe.
//
// Bound by the matrix pipe (2 M K N flop per piece), so the loop must feed it: the floating operand is split into its
// planes ONCE by split_planes_kernel (a workgroup splitting its own rows would repeat that for every 128 outputs, and
// vector instructions compete with the matrix ones) and staged through LDS, double buffered, 64 reduction indices at a time,
// 16-byte chunks at chunk ^ (row / 2 % 8) so that fragment reads and stage writes are free of bank conflicts; the codes go
// straight from memory to registers, one step ahead, and are decoded a half step before they are used.
// Measured, float32 (three pieces): 1024 x 4096 x 4096 87-91 us in all, the tiles alone 83, 1240 TFLOP/s issued (a library product
// of two 8192 x 8192 bfloat16 matrices: 1213).  1024 x 1024 x 4096 33 us: tiles 28.1, of which 11 do not depend on the depth
// (launch, first loads, last stores), planes 5.5; transposed 45 us: tiles 31.4, planes 8.0 and the sum of four parts 6.6.
// 4096 x 4096 x 4096 bfloat16 (in place) 140 us, 983 TFLOP/s, transposed 179; float16 235 us, 1170 TFLOP/s over its two pieces.  1024 x 1024 x 4096
// transposed: bfloat16 27 us, float16 35, most of it the parts and their sum.  Before the halves of a step were interleaved (all reads, all
// decoding, all products, all writes) and addresses took 50 instructions a step: 104, 36.7 and 50.2 us.  Tiles of 128 rows
// (wave tiles 64 x 64, one workgroup a unit): 125 and 41.
#pragma once
#include "frag.hpp"

namespace gpvae_lb {

// planes[p][k / 64][m][k % 64] of X [M, ldx], zero past L (Lp a multiple of 128): what a step stages is contiguous.
// A block of 256 threads takes 256 >> qsh rows (blockIdx.x) x 1024 columns (blockIdx.y), 4 elements a thread.
template <typename T>
__global__ __launch_bounds__(256) void split_planes_kernel(int64_t M, int64_t L, int64_t Lp, int qsh, const T *__restrict__ X, int64_t ldx,
                                                           u32x2 *__restrict__ planes) {
  constexpr int P = Split<T>::P;
  const int64_t q = Lp / 4, m = ((int64_t)blockIdx.x << (8 - qsh)) + (threadIdx.x >> qsh);
  if (m >= M) return;
  for (int64_t k4 = (int64_t)blockIdx.y * 256 + (threadIdx.x & ((1 << qsh) - 1)); k4 < q; k4 += (int64_t)gridDim.y * 256) {
    const Vec4<T> v = load4(X + m * ldx, k4 * 4, L);
    uint32_t a[P], b[P];
    Split<T>::two(v.v[0], v.v[1], a);
    Split<T>::two(v.v[2], v.v[3], b);
#pragma unroll
    for (int p = 0; p < P; ++p) planes[p * M * q + ((k4 >> 4) * M + m) * 16 + (k4 & 15)] = u32x2{a[p], b[p]};
  }
}

constexpr int TL_WM = 2, TL_MT = 2;  // TL_WM x 2 waves, each 16 TL_MT rows x 64 outputs

// Addresses are a scalar base that moves with the step plus a fixed 32-bit offset per lane, so that the loop spends no vector
// instruction on them.  Operand element (piece p, row m, reduction index k) is at byte p ps + (k / 64) ss + m rs + 2 (k % 64).
template <typename T, bool VJP>
__global__ __launch_bounds__(128 * TL_WM, 2) void tile_kernel(int64_t M, int64_t O, const char *__restrict__ planes, int64_t rs,
                                                           int64_t ss, int64_t ps, const char *__restrict__ codes,
                                                           const char *__restrict__ exps, int64_t Np, int64_t kbs, int mtiles,
                                                           int64_t s_all, int steps, float *__restrict__ part,
                                                           Epilogue<T, VJP> ep) {
  constexpr int P = Split<T>::P, WM = TL_WM, MT = TL_MT, NT = 128 * WM, BM = 16 * MT * WM;
  constexpr int CH = P * BM * 8, NLD = CH / NT;  // 16-byte chunks of a stage, and of one thread's share
  static_assert(BM % (NT / 8) == 0 && NT / 8 % 8 == 0, "whole shares");
  __shared__ __align__(16) unsigned char lds[2][CH * 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wo = wave & 1, c = lane >> 4, l16 = lane & 15;
  const uint32_t ot = __builtin_amdgcn_readfirstlane(blockIdx.x / (uint32_t)mtiles);  // row tiles fastest
  const int64_t m0 = (int64_t)(blockIdx.x - ot * (uint32_t)mtiles) * BM, o0 = (int64_t)ot * 128 + wo * 64;
  const int64_t s_lo = (int64_t)blockIdx.y * steps, s_hi = s_lo + steps < s_all ? s_lo + steps : s_all;
  Tr8 tr;
  if (VJP) tr.init(lane);
  const int lab = tr8_label(lane), half = l16 >> 3;

  // stage share: thread -> 16-byte chunk tid % 8 of rows tid / 8 + RP i of every plane
  constexpr int RP = NT / 8, NR = BM / RP;
  const int ck8 = tid & 7, trow = tid >> 3;
  uint32_t src[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int64_t row = trow + i * RP;
    src[i] = (uint32_t)((m0 + row < M ? row : M - 1 - m0) * rs) + ck8 * 16;  // rows past the last: results unused
  }
  // lane group c reads chunk 2 c + t (product) or 4 t + c: either is kept at 4 t + c, so that the reads of the lane groups that
  // share a cycle never meet in a bank
  const int pk8 = VJP ? ck8 : (ck8 >> 1) | (ck8 & 1) << 2;
  const int dst = (trow * 8 + (pk8 ^ ((trow >> 1) & 7))) * 16;
  // Codes of one step: product: 8 bytes (two groups of 8 rows) of each of 4 columns 16 apart, lane group c taking rows
  // 32 (c / 2) + 16 (c % 2) + ...; transposed product: 8 bytes of a column for two blocks of 32 columns x two of 32 rows.
  // What lies past the last block is loaded as zero; columns (rows) past the last repeat the last one or its block, unused.
  uint32_t coff[4], eoff[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (!VJP) {
      const int64_t n = o0 + t * 16 + l16 < Np ? o0 + t * 16 + l16 : Np - 1;
      coff[t] = (uint32_t)(((c >> 1) * Np + n) * 16 + (c & 1) * 8);
      eoff[t] = (uint32_t)(((c >> 1) * (Np / 8) + n / 8) * 4 + 2 * (c & 1));
    } else {
      coff[t] = ((t >> 1) * 32 + c * 8 + lab) * 16 + half * 8;
      eoff[t] = ((t >> 1) * 4 + c) * 4 + 2 * half;
    }
  }
  struct Ahead {  // what is in flight for a step: its share of the stage, its codes and tile exponents
    u32x4 st[NLD];
    u32x2 cw[4];
    uint32_t ce[4];  // the exponents of both halves' tiles
  };
  // No branch may surround these loads: the wait for a step's loads counts the younger ones behind them, and a load that
  // may not have been issued does not count, so that the wait would reach into the step just issued.  The steps are loaded in
  // order, each by scalar bases that move on by themselves; past the last one nothing is read.
  const char *pb = planes + m0 * rs + s_lo * ss;
  int stages = (int)(s_all - s_lo);  // steps from here to the planes' end
  auto issue_stage = [&](Ahead &h) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NLD; ++i)
      h.st[i] = __builtin_amdgcn_raw_buffer_load_b128(buffer(pb + (i / NR) * ps, stages > 0 ? 0x7fffffff : 0), src[i % NR], 0, 0);
    pb += ss;
    --stages;
  };
  const int64_t kbv0 = o0 / 32 < kbs ? o0 / 32 : kbs - 1, kbv1 = o0 / 32 + 1 < kbs ? o0 / 32 + 1 : kbs - 1;
  const int64_t cat0 = VJP ? kbv0 * Np + s_lo * 64 : 2 * s_lo * Np, cat1 = kbv1 * Np + s_lo * 64;
  const char *cb0 = codes + cat0 * 16, *cb1 = codes + cat1 * 16, *eb0 = exps + cat0 / 2, *eb1 = exps + cat1 / 2;
  int ends = (int)(VJP ? Np - s_lo * 64 : kbs - 2 * s_lo);  // columns (blocks of 32 rows) from here to the codes' end
  auto issue_codes = [&](Ahead &h) __attribute__((always_inline)) {
    if (!VJP) {
      const int bytes = ends >= 2 ? (int)Np : ends == 1 ? (int)Np / 2 : 0;  // of exponents; 32 times as many of codes
      const rsrc_t rc = buffer(cb0, bytes * 32), re = buffer(eb0, bytes);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        h.cw[t] = __builtin_amdgcn_raw_buffer_load_b64(rc, coff[t], 0, 0);
        h.ce[t] = __builtin_amdgcn_raw_buffer_load_b16(re, eoff[t], 0, 0);
      }
      cb0 += Np * 32, eb0 += Np;
      ends -= 2;
    } else {
      const int nc = __builtin_amdgcn_readfirstlane(ends >= 64 ? 64 : ends > 0 ? ends : 0);  // (a vector instruction clamps)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        h.cw[t] = __builtin_amdgcn_raw_buffer_load_b64(buffer(t & 1 ? cb1 : cb0, nc * 16), coff[t], 0, 0);
        h.ce[t] = __builtin_amdgcn_raw_buffer_load_b16(buffer(t & 1 ? eb1 : eb0, nc / 2), eoff[t], 0, 0);
      }
      cb0 += 1024, cb1 += 1024, eb0 += 32, eb1 += 32;
      ends -= 64;
    }
  };
  auto put = [&](const Ahead &h, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) *reinterpret_cast<u32x4 *>(lds[b] + dst + i * RP * 128) = h.st[i];
  };

  f32x4_t acc[MT][4];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = f32x4_t{0, 0, 0, 0};
  const int arow = (wm * MT * 16 + l16) * 128, sw = l16 >> 1;
  u32x4 x[2][P][MT], f[2][4];
  auto read = [&](int t, int b) __attribute__((always_inline)) {
    const int ck = ((t * 4 + c) ^ sw) * 16;
#pragma unroll
    for (int p = P - 1; p >= 0; --p)
#pragma unroll
      for (int a = 0; a < MT; ++a) x[t][p][a] = *reinterpret_cast<const u32x4 *>(lds[b] + p * BM * 128 + arow + a * 2048 + ck);
  };
  auto decode = [&](const Ahead &h, int t) __attribute__((always_inline)) {
    if (!VJP) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t e = h.ce[i];
        f[t][i] = w4_frag(t ? h.cw[i].y : h.cw[i].x, t ? w4_scale<1>(e) : w4_scale<0>(e));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t e = h.ce[2 * t + i];
        f[t][2 * i] = w4_frag(tr(h.cw[2 * t + i].x), w4_scale<0>(e));
        f[t][2 * i + 1] = w4_frag(tr(h.cw[2 * t + i].y), w4_scale<1>(e));
      }
    }
  };
  auto multiply = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int p = P - 1; p >= 0; --p)
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[a][i] = mfma(x[t][p][a], f[t][i], acc[a][i]);
  };
  // One step, in two halves of 32 indices.  Its first half's fragments are in registers, its stage in lds[b], its codes in `now`;
  // `next` holds step s + 1 in flight.  While a half is multiplied, the other's fragments are read and decoded and the next
  // stage is written, instruction by instruction: matrix, vector and LDS instructions overlap only when they alternate.  What
  // has been written and decoded is replaced: the stage by step s + 3's in `next`, the codes by step s + 2's in `now`.
  auto step = [&](Ahead &now, Ahead &next, int b) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);  // the unit's other workgroup is kept in the opposite half: 2-4 % faster
    read(1, b);
    decode(now, 1);
    put(next, b ^ 1);
    multiply(0);
#pragma unroll
    for (int g = 0; g < 2 * P; ++g) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // a fragment read
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // a stage write
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    read(0, b ^ 1);
    decode(next, 0);
    issue_stage(next);
    issue_codes(now);
    multiply(1);
#pragma unroll
    for (int g = 0; g < 2 * P; ++g) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, (2 * P + 8 + 2 * P - 1) / (2 * P), 0);  // loads
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  Ahead h0, h1;
  issue_stage(h0);
  issue_codes(h0);
  issue_stage(h1);
  issue_codes(h1);
  put(h0, 0);
  issue_stage(h0);
  __syncthreads();
  read(0, 0);
  decode(h0, 0);
  // an even number of steps: a loop that may leave after the first of two makes the compiler copy registers whose loads are in
  // flight, and wait for them
#pragma unroll 1
  for (int64_t s = s_lo; s < s_hi; s += 2) {
    step(h0, h1, 0);
    step(h1, h0, 1);
  }
  const bool whole = gridDim.y == 1;
  int64_t oi[4];
  float bv[4];
  uint32_t mask[MT][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    oi[i] = o0 + (VJP ? (i >> 1) * 32 + (2 * half + (i & 1)) * 8 + lab : i * 16 + l16);
    const int64_t oc = oi[i] < O ? oi[i] : O - 1;
    bv[i] = whole ? ep.bias_at(oc) : 0.0f;
#pragma unroll
    for (int a = 0; a < MT; ++a) {
      const int64_t m = m0 + (wm * MT + a) * 16 + 4 * c;
      mask[a][i] = whole ? ep.mask4_at(m < M ? m : 0, oc) : 0u;
    }
  }
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t m = m0 + (wm * MT + a) * 16 + 4 * c + r;
      if (m >= M) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (oi[i] >= O) continue;
        if (whole) ep.store(m, oi[i], acc[a][i][r], bv[i], (mask[a][i] >> (8 * r)) & 255u);
        else part[((int64_t)blockIdx.y * M + m) * O + oi[i]] = acc[a][i][r];
      }
    }
}

struct TilePlan {
  int mtiles, splits, steps;
  int64_t blocks, Lp, plane_bytes;
  bool direct;         // the operand itself is its only plane
};

// Rows of one launch; more are taken in turn.  Launches hold fewer than 2^32 threads (a workgroup of split_planes_kernel may have one
// row, one of tile_kernel 64 rows x 128 of the O outputs), and 2^20 rows fill the chip hundreds of times over.
static inline int64_t tile_rows(int64_t O) {
  const int64_t tiles = ((int64_t(1) << 32) / (128 * TL_WM) - 1) / cdiv(O, 128) * (16 * TL_MT * TL_WM);
  return tiles < 1 ? 16 * TL_MT * TL_WM : tiles < (1 << 20) ? tiles : 1 << 20;
}
// Into how many parts is the reduction split?  A step of 64 takes 0.25 + 0.22 P us where a compute unit has one workgroup and
// 0.20 + 0.31 P us where it has the two that fit, every full round of 512 workgroups anew; a split costs the launch that adds
// the parts (4 us) and writing and reading them.  The least of that estimate over powers of two and the numbers that give
// every unit one or two workgroups.  Measured, one part / two / four: float32 512 x 1024 x 4096 24.6 / 32.7 / 36.4 us,
// 512 x 4096 x 4096 58 / 59 / 63, 1024 x 1024 x 4096 transposed 68.6 / 51.3 / 47.8 (bfloat16 40.4 / 31.9 / 28.4); bfloat16 1024 x 1000 x 1000
// 14.6 / 20.6 / 23.5.
static inline TilePlan tile_plan(int P, int64_t M, int64_t L, int64_t O, bool direct) {
  TilePlan p;
  p.direct = direct;
  p.Lp = round_up(L, 128);
  p.mtiles = (int)cdiv(M, 16 * TL_MT * TL_WM);
  p.blocks = p.mtiles * cdiv(O, 128);
  const int64_t steps = p.Lp / 64;
  p.splits = 1;
  p.steps = (int)steps;
  double best = 0.0;
  for (int64_t i = 1; i <= 512; i *= 2)
    for (int64_t s : {i, i < 256 ? int64_t(0) : 256 * (i / 256) / p.blocks}) {
      if (s < 1 || (s > 1 && (s * p.blocks > 640 || s * 4 > steps))) continue;
      const int64_t per = round_up(cdiv(steps, s), 2), parts = cdiv(steps, per), b = parts * p.blocks;
      const double step = b <= 256 ? 0.25 + 0.22 * P : (double)cdiv(b, 512) * (0.20 + 0.31 * P);
      const double t = (double)per * step + (parts > 1 ? 4.0 + (double)parts * ((double)M * (double)O * (8 / 4.5e6) + 0.06) : 0.0);
      if (s == 1 || t < best) best = t, p.splits = (int)parts, p.steps = (int)per;
    }
  p.plane_bytes = direct ? 0 : round_up(P * M * p.Lp * 2, 256);
  return p;
}

template <typename T, bool VJP>
static void launch_tile(hipStream_t st, const TilePlan &p, int64_t M, int64_t L, int64_t O, const T *X, int64_t ldx,
                        const void *codes, const void *exps, int64_t Np, int64_t kbs, unsigned char *work,
                        const Epilogue<T, VJP> &ep) {
  const char *planes = reinterpret_cast<const char *>(X);
  int64_t rs = ldx * 2, ss = 128, ps = 0;
  if (!p.direct) {
    int qsh = 5;  // 2^qsh >= Lp / 4, at most 256 threads to a row
    while (qsh < 8 && (4 << qsh) < p.Lp) ++qsh;
    hipLaunchKernelGGL((split_planes_kernel<T>), dim3((unsigned)cdiv(M, 256 >> qsh), (unsigned)(p.Lp < 1024 * 65535ll ? cdiv(p.Lp, 1024) : 65535)), dim3(256), 0, st,
                       M, L, p.Lp, qsh, X, ldx, (u32x2 *)work);
    if (hipPeekAtLastError() != hipSuccess) return;  // reported by the caller; the planes are not written
    planes = reinterpret_cast<const char *>(work);
    rs = 128, ss = M * 128, ps = M * p.Lp * 2;
  }
  float *part = reinterpret_cast<float *>(work + p.plane_bytes);
  const dim3 grid((unsigned)p.blocks, (unsigned)p.splits);
  hipLaunchKernelGGL((tile_kernel<T, VJP>), grid, dim3(128 * TL_WM), 0, st, M, O, planes, rs, ss, ps, (const char *)codes,
                     (const char *)exps, Np, kbs, p.mtiles, p.Lp / 64, p.steps, part, ep);
  if (p.splits > 1 && hipPeekAtLastError() == hipSuccess)
    launch_split_sum<T, VJP>(st, M, O, p.splits, part, ep);
}

}  // namespace gpvae_lb
