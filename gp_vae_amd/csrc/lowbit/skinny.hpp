// skinny.hpp — the product with 4-bit weights (VJP = false: Y = X W, reduction over K) and with their transpose
// (VJP = true: dX = dY W^T, reduction over N) for few rows.
//
// What it has to do is read the codes once: K N / 2 bytes.  So each wave owns 32 outputs, streams codes straight
// from memory into registers (2 KB per step of 128 reduction indices, the next step's loads in flight while this one
// is multiplied) and multiplies them on the matrix pipe, whose 16 A rows carry the floating rows AND their pieces:
// row p M + m of the operand image is piece p of row m, so one row of float32 costs one matrix instruction, not three.
// The image sits in LDS; the waves of a workgroup share it, and split the reduction (WK) as far as there are
// too few outputs to fill the chip; S workgroups split it further.  Pieces, waves and splits are added in a fixed order.
// Measured, float32: 1 x 4096 x 32768 17.0-19.4 us with the codes in memory (4.1-3.6 TB/s; a copy on this card: 4.8), 14.0 with
// part of them in the last-level cache; 16 x 4096 x 1024 7.7 us, 37 x 700 x 1025 transposed 6.7 us and 1 x 50 x 4096 4.2 us, bound by the
// chain launch - first loads - products - sums, not by a rate.  More rows: staging, the matrix pipe and the decoding take over
// (21 x 4096 x 32768 35 us; the image is written, waited for and multiplied in turn), see use_skinny.
#pragma once
#include "frag.hpp"

namespace gpvae_lb {

constexpr int SK_WAVES = 8, SK_MAXROWS = 64;

struct SkinnyPlan {
  int rt;        // tiles of 16 operand rows
  int wk;        // waves of a workgroup along the reduction (the others: along the outputs)
  int chunk;     // reduction indices staged at a time (a multiple of 128 wk)
  int splits;    // workgroups along the reduction
  int steps;     // steps of 128 reduction indices of one split (a multiple of chunk / 128 unless it is the only chunk)
  int64_t gx;    // workgroups along the outputs
  int groups, mg;  // groups of rows (each reads all codes) and rows of one
};
static constexpr int skinny_lds(int rt) { return rt <= 1 ? 40 << 10 : rt == 2 ? 56 << 10 : 72 << 10; }

// P pieces of M rows, L reduction indices, O outputs
static inline SkinnyPlan skinny_plan(int P, int64_t M, int64_t L, int64_t O) {
  SkinnyPlan p;
  const int64_t steps = cdiv(L, 128), tiles = cdiv(O, 32);
  // Smaller groups than fit where that leaves the chip idle: each decodes all codes again, but stages fewer rows.  Doubled while
  // there are at most 128 workgroups for a reduction of up to 16 steps, 64 for one of up to 32; beyond, splitting the reduction
  // is better.  Limits of 0 / 64 / 128, float32 40 rows x 1000 outputs: 9 steps 12.0 / 6.3 / 6.3 us, 32 steps 10.4 / 8.2 / 8.2 (float16 62 rows x 700:
  // 40 steps 15.1 / 15.9 / 15.9); 3000 outputs: 7 steps 10.4 (64) / 7.9 (128), 14 steps 13.6 / 11.9, 20 steps 14.4 / 15.5, 30 steps 17.5 / 19.2.
  const int64_t most_blocks = steps <= 16 ? 128 : steps <= 32 ? 64 : 0;
  int rows, room;
  for (p.groups = (int)cdiv(M, SK_MAXROWS / P);; p.groups *= 2) {
    p.mg = (int)cdiv(M, p.groups);
    p.groups = (int)cdiv(M, p.mg);
    rows = P * p.mg;
    p.rt = (int)cdiv(rows, 16);
    room = (int)((skinny_lds(p.rt) / rows - 16) / 256);  // steps whose image fits
    p.wk = 1;
    while (p.wk < SK_WAVES && 2 * p.wk <= steps && 2 * p.wk <= room && tiles * p.wk < 2048) p.wk *= 2;
    p.gx = cdiv(tiles, SK_WAVES / p.wk);
    if (p.rt == 1 || p.gx * p.groups > most_blocks) break;
  }
  int64_t s = p.gx * p.groups < 256 ? cdiv(512, p.gx * p.groups) : 1;
  // a split costs a second launch (3 us): worth it down to four steps of each wave for one operand tile, two for two, one for
  // three or four, whose steps take longer.  At four / two / one: float32 1 x 4096 x 1024 5.6 / 6.7 / 6.3 us, 16 x 1024 x 4096 transposed
  // 9.3 / 8.9 / 9.3, float16 40 x 8192 x 500 13.7 / 10.5 / 9.8.  Longer reductions of one or two operand tiles would bear a finer split:
  // bfloat16 8 x 8192 x 512 9.0 / 7.3 / 6.6, 24 x 500 x 8192 transposed 14.4 / 10.3 / 8.3.
  const int64_t most = steps / ((p.rt == 1 ? 4 : p.rt == 2 ? 2 : 1) * p.wk);
  if (s > most) s = most;
  if (s < 1) s = 1;
  if (s > 64) s = 64;
  if (steps < 3 * p.wk) s = 1;  // less than three steps a wave are not worth a launch
  int64_t per = cdiv(steps, s);
  per = round_up(per, p.wk);
  p.splits = (int)cdiv(steps, per);
  p.steps = (int)per;
  int64_t ch = room / p.wk * p.wk;
  if (ch > per) ch = per;
  p.chunk = (int)(ch * 128);
  return p;
}

template <typename T, bool VJP, int RT>
__global__ __launch_bounds__(64 * SK_WAVES) void skinny_kernel(int64_t M_all, int mg, int64_t L, int64_t O, const T *__restrict__ X,
                                                               int64_t ldx, const char *__restrict__ codes,
                                                               const char *__restrict__ exps, int64_t Np, int64_t kbs,
                                                               int wk_n, int steps, int chunk, uint32_t magic, float *__restrict__ part,
                                                               Epilogue<T, VJP> ep) {
  constexpr int P = Split<T>::P;
  __shared__ __align__(16) unsigned char lds[skinny_lds(RT)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave & (wk_n - 1), wn = wave / wk_n;
  const int c = lane >> 4, l16 = lane & 15;
  const int64_t m_lo = (int64_t)blockIdx.z * mg;  // this group of rows
  const int M = m_lo + mg <= M_all ? mg : (int)(M_all - m_lo);
  X += m_lo * ldx;
  const int64_t tile = (int64_t)blockIdx.x * (SK_WAVES / wk_n) + wn;  // 32 outputs
  const int64_t o0 = (tile * 32 < O ? tile : (O - 1) / 32) * 32;           // a wave past the last tile repeats it, unused
  const int rows = P * M;
  const int stride = chunk * 2 + 16;  // bytes of an image row: 16 more spread the rows over the banks
  const int64_t s_all = cdiv(L, 128), s_lo = (int64_t)blockIdx.y * steps;
  const int64_t s_hi = s_lo + steps < s_all ? s_lo + steps : s_all;
  Tr8 tr;
  if (VJP) tr.init(lane);
  const int lab = tr8_label(lane), half = l16 >> 3;

  u32x2 cw[4];  // codes of one step: 16 bytes for each of two columns, or 8 bytes for each of four
  uint32_t ce[VJP ? 4 : 2];
  const uint32_t coff = VJP ? (c * 8 + lab) * 16 + half * 8 : (uint32_t)((c * Np + l16) * 16);
  const uint32_t eoff = VJP ? c * 4 : (uint32_t)(c * (Np / 2) + (l16 >> 3) * 4);
  // last step with codes, and how many blocks of 32 rows (quarters of 32 columns) it has
  const int s_last = (int)((VJP ? Np - 1 : (kbs - 1) * 32) / 128);
  const int part_last = VJP ? (int)(Np - (int64_t)s_last * 128) / 32 - 1 : (int)(kbs - 1 - 4 * (int64_t)s_last);
  const char *const cbase = codes + (VJP ? o0 / 32 * Np : o0) * 16, *const ebase = exps + (VJP ? o0 / 32 * Np : o0) / 2;
  const uint32_t cstep = VJP ? 2048u : (uint32_t)(Np * 64), estep = VJP ? 64u : (uint32_t)(Np * 2);
  auto fetch = [&](int s) __attribute__((always_inline)) {
    const int sc = s < s_last ? s : s_last, last = s < s_last ? 3 : part_last;
    const char *const cb = cbase + (uint64_t)(uint32_t)sc * cstep, *const eb = ebase + (uint64_t)(uint32_t)sc * estep;
    if (!VJP) {
      const uint32_t back = c > last ? (uint32_t)(c - last) : 0u;  // blocks past the last: that one
      const uint32_t co = coff - back * (cstep / 4), eo = eoff - back * (estep / 4);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4 q = *reinterpret_cast<const u32x4 *>(cb + t * 256 + co);
        cw[2 * t] = u32x2{q.x, q.y};
        cw[2 * t + 1] = u32x2{q.z, q.w};
        ce[t] = *reinterpret_cast<const uint32_t *>(eb + t * 8 + eo);
      }
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t back = t > last ? (uint32_t)(t - last) : 0u;  // quarters past the last: that one
        cw[t] = *reinterpret_cast<const u32x2 *>(cb + (coff + (t - back) * 512));  // t >= back: no wrap before the addition
        ce[t] = *reinterpret_cast<const uint32_t *>(eb + (eoff + (t - back) * 16));
      }
    }
  };

  f32x4_t acc[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[r][t] = f32x4_t{0, 0, 0, 0};

  fetch((int)s_lo + wk);
  int a_off[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = r * 16 + l16;
    a_off[r] = (row < rows ? row : rows - 1) * stride + (VJP ? c * 16 : c * 64);  // rows past the last: results unused
  }
  const int chunk_steps = chunk / 128;
  for (int64_t s0 = s_lo; s0 < s_hi; s0 += chunk_steps) {
    if (s0 != s_lo) __syncthreads();
    {  // the image of reduction indices [128 s0, 128 s0 + chunk): 4 at a time, zeros past L
      const int q = chunk / 4;  // magic = ceil(2^32 / q): exact quotients, i < 2^32 / q
      auto put = [&](int m, int k4, const Vec4<T> &v) __attribute__((always_inline)) {
        uint32_t a[P], b[P];
        Split<T>::two(v.v[0], v.v[1], a);
        Split<T>::two(v.v[2], v.v[3], b);
#pragma unroll
        for (int p = 0; p < P; ++p)
          *reinterpret_cast<u32x2 *>(lds + (p * M + m) * stride + k4 * 8) = u32x2{a[p], b[p]};
      };
      const T *const x0 = X + s0 * 128;
      if (s0 * 128 + chunk <= L) {
#pragma unroll 2  // two vectors in flight: 21 x 4096 x 32768 float32 39.2 -> 34.6 us
        for (int i = tid; i < M * q; i += 64 * SK_WAVES) {
          const int m = (int)__umulhi((uint32_t)i, magic), k4 = i - m * q;
          put(m, k4, *reinterpret_cast<const Vec4<T> *>(x0 + m * ldx + k4 * 4));
        }
      } else {
        for (int i = tid; i < M * q; i += 64 * SK_WAVES) {
          const int m = (int)__umulhi((uint32_t)i, magic), k4 = i - m * q;
          put(m, k4, load4(x0 + m * ldx, k4 * 4, L - s0 * 128));
        }
      }
    }
    __syncthreads();
    for (int i = wk; i < chunk_steps; i += wk_n) {
      const int64_t s = s0 + i;
      if (s >= s_hi) break;
      u32x2 w[4];
      uint32_t e[VJP ? 4 : 2];
#pragma unroll
      for (int t = 0; t < 4; ++t) w[t] = cw[t];
#pragma unroll
      for (int t = 0; t < (VJP ? 4 : 2); ++t) e[t] = ce[t];
      fetch((int)s + wk_n);
      const unsigned char *img = lds + i * 256;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 f0, f1;
        if (!VJP) {
          const uint32_t d0 = j & 1 ? w[j >> 1].y : w[j >> 1].x, d1 = j & 1 ? w[2 + (j >> 1)].y : w[2 + (j >> 1)].x;
          f0 = w4_frag(d0, j == 0 ? w4_scale<0>(e[0]) : j == 1 ? w4_scale<1>(e[0]) : j == 2 ? w4_scale<2>(e[0]) : w4_scale<3>(e[0]));
          f1 = w4_frag(d1, j == 0 ? w4_scale<0>(e[1]) : j == 1 ? w4_scale<1>(e[1]) : j == 2 ? w4_scale<2>(e[1]) : w4_scale<3>(e[1]));
        } else {  // columns: row tiles 2 half and 2 half + 1 of the block of 32
          const uint32_t ej = e[VJP ? j : 0] >> (16 * half);
          f0 = w4_frag(tr(w[j].x), w4_scale<0>(ej));
          f1 = w4_frag(tr(w[j].y), w4_scale<1>(ej));
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const u32x4 a = *reinterpret_cast<const u32x4 *>(img + a_off[r] + (VJP ? j * 64 : j * 16));
          acc[r][0] = mfma(a, f0, acc[r][0]);
          acc[r][1] = mfma(a, f1, acc[r][1]);
        }
      }
    }
  }

  // [wave][operand row][output of the wave's 32] -> sums over the waves of one output tile, then over the pieces
  __syncthreads();
  float *red = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int row = r * 16 + 4 * c + v;
        const int o = VJP ? (2 * half + t) * 8 + lab : t * 16 + l16;
        if (row < rows) red[(wave * rows + row) * 32 + o] = acc[r][t][v];
      }
  __syncthreads();
  // a thread keeps its output column (the columns of a workgroup divide its threads), four rows at a time
  const int outs = SK_WAVES / wk_n * 32, oo = tid & (outs - 1), w = oo >> 5, col = oo & 31, dm = 64 * SK_WAVES / outs;
  const int64_t o = ((int64_t)blockIdx.x * (SK_WAVES / wk_n) + w) * 32 + col;
  if (o >= O) return;
  const bool whole = gridDim.y == 1;
  const float b = whole ? ep.bias_at(o) : 0.0f;
  for (int m0 = tid / outs; m0 < M; m0 += 4 * dm) {
    float v[4];
    uint32_t mask[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) mask[u] = m0 + u * dm < M && whole ? ep.mask_at(m_lo + m0 + u * dm, o) : 0u;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      v[u] = 0.0f;
      if (m0 + u * dm < M)
        for (int p = P - 1; p >= 0; --p)  // small pieces first
          for (int k = 0; k < wk_n; ++k) v[u] += red[((w * wk_n + k) * rows + p * M + m0 + u * dm) * 32 + col];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int m = m0 + u * dm;
      if (m >= M) break;
      if (whole) ep.store(m_lo + m, o, v[u], b, mask[u]);
      else part[((int64_t)blockIdx.y * M_all + m_lo + m) * O + o] = v[u];
    }
  }
}

template <typename T, bool VJP>
static void launch_skinny(hipStream_t st, const SkinnyPlan &p, int64_t M, int64_t L, int64_t O, const T *X, int64_t ldx,
                          const void *codes, const void *exps, int64_t Np, int64_t kbs, float *part,
                          const Epilogue<T, VJP> &ep) {
  const dim3 grid((unsigned)p.gx, (unsigned)p.splits, (unsigned)p.groups);
#define GO(RT)                                                                                                            \
  hipLaunchKernelGGL((skinny_kernel<T, VJP, RT>), grid, dim3(64 * SK_WAVES), 0, st, M, p.mg, L, O, X, ldx,              \
                     (const char *)codes, (const char *)exps, Np, kbs, p.wk, p.steps, p.chunk, (uint32_t)cdiv(int64_t(1) << 32, p.chunk / 4), part, ep)
  if (p.rt == 1) GO(1);
  else if (p.rt == 2) GO(2);
  else if (p.rt == 3) GO(3);
  else GO(4);
#undef GO
  if (p.splits > 1 && hipPeekAtLastError() == hipSuccess)
    launch_split_sum<T, VJP>(st, M, O, p.splits, part, ep);
}

}  // namespace gpvae_lb
