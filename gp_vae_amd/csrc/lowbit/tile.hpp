// tile.hpp — the products of skinny.hpp for many rows: tiles of (16 MT WM) rows x 128 outputs on the bf16 matrix pipe.
//
// Bound by the matrix pipe (2 M K N flop per piece), so the loop must feed it: the floating operand is split into its
// planes ONCE by split_planes_kernel (a workgroup splitting its own rows would repeat that for every 128 outputs, and
// vector instructions compete with the matrix ones) and staged through LDS, double buffered, 64 reduction indices at a time,
// 16-byte chunks at chunk ^ (row & 7) so that fragment reads and stage writes are free of bank conflicts; the codes go
// straight from memory to registers, one step ahead, and are decoded where they are used.
#pragma once
#include "frag.hpp"

namespace gpvae_lb {

// planes[p][m][Lp] of X [M, ldx], zero past L (Lp a multiple of 64)
template <typename T>
__global__ __launch_bounds__(256) void split_planes_kernel(int64_t M, int64_t L, int64_t Lp, const T *__restrict__ X, int64_t ldx,
                                                           uint2 *__restrict__ planes) {
  constexpr int P = Split<T>::P;
  const int64_t q = Lp / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= M * q) return;
  const int64_t m = i / q, k4 = i - m * q;
  const Vec4<T> v = load4(X + m * ldx, k4 * 4, L);
  uint32_t a[P], b[P];
  Split<T>::two(v.v[0], v.v[1], a);
  Split<T>::two(v.v[2], v.v[3], b);
#pragma unroll
  for (int p = 0; p < P; ++p) planes[p * M * q + i] = make_uint2(a[p], b[p]);
}

// WM x 2 waves, each 16 MT rows x 64 outputs
template <typename T, bool VJP, int WM, int MT>
__global__ __launch_bounds__(128 * WM, WM == 4 ? 2 : 3) void tile_kernel(int64_t M, int64_t Lp, int64_t O, const uint16_t *__restrict__ planes,
                                                           int64_t ldp, int64_t plane, const uint4 *__restrict__ codes,
                                                           const uint32_t *__restrict__ exps, int64_t Np, int64_t kbs, int mtiles,
                                                           int steps, float *__restrict__ part, Epilogue<T, VJP> ep) {
  constexpr int P = Split<T>::P, NT = 128 * WM, BM = 16 * MT * WM;
  constexpr int CH = P * BM * 8, NLD = CH / NT;  // 16-byte chunks of a stage, and of one thread's share
  static_assert(CH % NT == 0, "whole shares");
  __shared__ __align__(16) unsigned char lds[2][CH * 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wo = wave & 1, c = lane >> 4, l16 = lane & 15;
  const int64_t bt = blockIdx.x, m0 = (bt % mtiles) * BM, o0 = (bt / mtiles) * 128 + wo * 64;  // row tiles fastest
  const int64_t s_all = Lp / 64, s_lo = (int64_t)blockIdx.y * steps;
  const int64_t s_hi = s_lo + steps < s_all ? s_lo + steps : s_all;
  Tr8 tr;
  if (VJP) tr.init(lane);
  const int lab = tr8_label(lane), half = l16 >> 3;

  // stage share: chunk id -> (piece, row, 16-byte chunk)
  uint4 st[NLD];
  const uint16_t *src[NLD];
  int dst[NLD];
#pragma unroll
  for (int i = 0; i < NLD; ++i) {
    const int id = i * NT + tid, ck = id & 7, row = (id >> 3) % BM, p = (id >> 3) / BM;
    const int64_t m = m0 + row < M ? m0 + row : M - 1;  // rows past the last: results unused
    src[i] = planes + p * plane + m * ldp + ck * 8;
    dst[i] = ((p * BM + row) * 8 + (ck ^ (row & 7))) * 16;
  }
  auto stage_load = [&](int64_t s) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) st[i] = *reinterpret_cast<const uint4 *>(src[i] + s * 64);
  };
  auto stage_store = [&](int b) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) *reinterpret_cast<uint4 *>(lds[b] + dst[i]) = st[i];
  };
  // codes of one step: product: 8 bytes (two groups of 8 rows) of each of 4 columns 16 apart, lane group c taking rows
  // 32 (c / 2) + 16 (c % 2) + ...; transposed product: 8 bytes of a column for two blocks of 32 columns x two of 32 rows
  uint2 cw[4];
  uint32_t ce[4];
  auto fetch = [&](int64_t s) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (!VJP) {
        const int64_t kb = 2 * s + (c >> 1), n = o0 + t * 16 + l16;
        const bool in = kb < kbs && n < Np;
        cw[t] = in ? reinterpret_cast<const uint2 *>(codes)[(kb * Np + n) * 2 + (c & 1)] : make_uint2(0, 0);
        ce[t] = in ? exps[kb * (Np / 8) + n / 8] >> (16 * (c & 1)) : 0u;
      } else {
        const int64_t n = s * 64 + (t >> 1) * 32, kb = o0 / 32 + (t & 1);
        const bool in = n < Np && kb < kbs;
        cw[t] = in ? reinterpret_cast<const uint2 *>(codes)[(kb * Np + n + c * 8 + lab) * 2 + half] : make_uint2(0, 0);
        ce[t] = in ? exps[kb * (Np / 8) + n / 8 + c] >> (16 * half) : 0u;
      }
    }
  };

  f32x4_t acc[MT][4];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = f32x4_t{0, 0, 0, 0};
  stage_load(s_lo);
  fetch(s_lo);
  stage_store(0);
  __syncthreads();
  const int arow = (wm * MT * 16 + l16) * 128, sw = l16 & 7;
  for (int64_t s = s_lo; s < s_hi; ++s) {
    const int b = (int)(s - s_lo) & 1;
    const uint2 w[4] = {cw[0], cw[1], cw[2], cw[3]};
    const uint32_t e[4] = {ce[0], ce[1], ce[2], ce[3]};
    const bool more = s + 1 < s_hi;
    if (more) {
      stage_load(s + 1);
      fetch(s + 1);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint4 f[4];
      if (!VJP) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = w4_frag(t ? w[i].y : w[i].x, t ? w4_scale<1>(e[i]) : w4_scale<0>(e[i]));
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f[2 * i] = w4_frag(tr(w[2 * t + i].x), w4_scale<0>(e[2 * t + i]));
          f[2 * i + 1] = w4_frag(tr(w[2 * t + i].y), w4_scale<1>(e[2 * t + i]));
        }
      }
      const int ck = ((VJP ? t * 4 + c : 2 * c + t) ^ sw) * 16;
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int a = 0; a < MT; ++a) {
          const uint4 x = *reinterpret_cast<const uint4 *>(lds[b] + p * BM * 128 + arow + a * 2048 + ck);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[a][i] = mfma(x, f[i], acc[a][i]);
        }
    }
    if (more) stage_store(b ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t o = o0 + (VJP ? (i >> 1) * 32 + (2 * half + (i & 1)) * 8 + lab : i * 16 + l16);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t m = m0 + (wm * MT + a) * 16 + 4 * c + r;
        if (m >= M || o >= O) continue;
        if (gridDim.y == 1) ep(m, o, acc[a][i][r]);
        else part[((int64_t)blockIdx.y * M + m) * O + o] = acc[a][i][r];
      }
    }
}

struct TilePlan {
  int wm, mt;          // kernel shape
  int mtiles, splits, steps;
  int64_t blocks, Lp, plane_bytes;
  bool direct;         // the operand itself is its only plane
};

static inline TilePlan tile_plan(int P, int64_t M, int64_t L, int64_t O, bool direct) {
  TilePlan p;
  p.direct = direct;
  p.wm = M <= 64 ? 2 : 4;
  p.mt = 2;
  p.Lp = round_up(L, 64);
  p.mtiles = (int)cdiv(M, 16 * p.mt * p.wm);
  p.blocks = p.mtiles * cdiv(O, 128);
  const int64_t steps = p.Lp / 64;
  int64_t s = p.blocks < 192 ? cdiv(256, p.blocks) : 1;
  if (s > steps / 4) s = steps / 4;
  if (s < 1) s = 1;
  p.steps = (int)cdiv(steps, s);
  p.splits = (int)cdiv(steps, p.steps);
  p.plane_bytes = direct ? 0 : round_up(P * M * p.Lp * 2, 256);
  return p;
}

template <typename T, bool VJP>
static void launch_tile(hipStream_t st, const TilePlan &p, int64_t M, int64_t L, int64_t O, const T *X, int64_t ldx,
                        const void *codes, const void *exps, int64_t Np, int64_t kbs, unsigned char *work,
                        const Epilogue<T, VJP> &ep) {
  const uint16_t *planes = reinterpret_cast<const uint16_t *>(X);
  int64_t ldp = ldx, plane = 0;
  if (!p.direct) {
    hipLaunchKernelGGL((split_planes_kernel<T>), dim3((unsigned)cdiv(M * p.Lp / 4, 256)), dim3(256), 0, st, M, L, p.Lp, X, ldx,
                       (uint2 *)work);
    planes = reinterpret_cast<const uint16_t *>(work);
    ldp = p.Lp;
    plane = M * p.Lp;
  }
  float *part = reinterpret_cast<float *>(work + p.plane_bytes);
  const dim3 grid((unsigned)p.blocks, (unsigned)p.splits);
#define GO(WM, MT)                                                                                                        \
  hipLaunchKernelGGL((tile_kernel<T, VJP, WM, MT>), grid, dim3(128 * WM), 0, st, M, p.Lp, O, planes, ldp, plane,        \
                     (const uint4 *)codes, (const uint32_t *)exps, Np, kbs, p.mtiles, p.steps, part, ep)
  if (p.wm == 2) GO(2, 2);
  else GO(4, 2);
#undef GO
  if (p.splits > 1)
    hipLaunchKernelGGL((split_sum_kernel<T, VJP>), dim3((unsigned)cdiv(M * O, 256)), dim3(256), 0, st, M, O, p.splits, part, ep);
}

}  // namespace gpvae_lb
