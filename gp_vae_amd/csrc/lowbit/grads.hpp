// grads.hpp — parameter gradients of a dense layer from the 8-bit checkpoint of its input:
//   dW[k][n] = sum_m X~[m][k] dY[m][n],   db[n] = sum_m dY[m][n].
//
// The reduction runs over the ROWS of both operands, the matrix instruction wants 8 consecutive reduction indices per lane.
// The checkpoint is laid out for that (8 rows of a column are 8 consecutive bytes); dY is transposed on its way into
// LDS: a thread loads 8 consecutive rows of a column (consecutive lanes: consecutive columns), splits them into their
// bfloat16 pieces and writes each piece's 8 values as 16 bytes.  Bound by the matrix pipe and LDS (one 128 x 128
// tile per workgroup, 64 rows a step): the conversions are vector work that is dealt between the matrix instructions of
// the step before.  All row tiles of a column tile run on one XCD (xcd_chunk), whose L2 then serves dY to them: dealt
// round-robin every XCD read all of dY from memory (4096 x 1024 x 4096 float32: 140 us; with it see the launch).
#pragma once
#include "frag.hpp"

namespace gpvae_lb {

constexpr int GR_THREADS = 512, GR_ROWS = 64;

struct GradsPlan {
  int ktiles, splits, steps;
  int64_t blocks;
};
static inline GradsPlan grads_plan(int64_t M, int64_t K, int64_t N) {
  GradsPlan p;
  p.ktiles = (int)cdiv(K, 128);
  p.blocks = p.ktiles * cdiv(N, 128);
  const int64_t steps = cdiv(M, GR_ROWS);
  int64_t s = p.blocks < 192 ? cdiv(256, p.blocks) : 1;
  if (s > steps / 2) s = steps / 2;  // a split keeps two steps
  if (s < 1) s = 1;
  p.steps = (int)cdiv(steps, s);
  p.splits = p.steps ? (int)cdiv(steps, p.steps) : 1;
  return p;
}

// 8 codes (bytes) -> 8 bfloat16 values times 2^e; exponent byte eb (255: NaN)
template <bool RELU> __device__ __forceinline__ u32x4 q8_frag(u32x2 q, uint32_t eb) {
  const float s = scale_of(eb);
  float v[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w = RELU ? q[h] : q[h] ^ 0x80808080u;  // two's complement -> offset by 128
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = (float)((w >> (8 * i)) & 255u);
      v[4 * h + i] = RELU ? u * s : __builtin_fmaf(u, s, -128.0f * s);  // exact: an integer below 256 times 2^e
    }
  }
  return u32x4{pack_hi(v[0], v[1]), pack_hi(v[2], v[3]), pack_hi(v[4], v[5]), pack_hi(v[6], v[7])};
}

template <typename T, bool RELU>
__global__ __launch_bounds__(GR_THREADS, 2) void grads_kernel(int64_t M, int64_t K, int64_t N, const char *__restrict__ codes,
                                                              const uint8_t *__restrict__ exps, const T *__restrict__ dY,
                                                              int64_t lddy, int ktiles, int s_all, int steps, float *dW,
                                                              int64_t lddw, float *db, int64_t part_stride) {
  constexpr int P = Split<T>::P, AB = 128 * 128, ST = AB * (1 + P);  // bytes of one image of 128 rows x 64; of a stage
  __shared__ __align__(16) unsigned char lds[2][ST];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave >> 2, wn = wave & 3, c = lane >> 4, l16 = lane & 15;  // wave: 64 rows of dW x 32 columns
  const int64_t bt = xcd_chunk(blockIdx.x, gridDim.x), kt = bt % ktiles, k0 = kt * 128, n0 = (bt / ktiles) * 128;
  const int s_lo = (int)blockIdx.y * steps, s_hi = s_lo + steps < s_all ? s_lo + steps : s_all;
  const int64_t Kp = q8_kp(K);
  const int mbs = (int)q8_mb(M);
  const bool sum_db = db != nullptr && kt == 0;
  dW += blockIdx.y * part_stride;
  if (db) db += blockIdx.y * part_stride;

  // dY share: columns lane and lane + 64, rows 8 wave .. + 7 of the step; checkpoint share: column tid % 128, blocks of
  // 8 rows tid / 128 and + 4.  Past the last column (row of dW): the last one again, results unused.
  uint32_t yoff[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) yoff[e] = (uint32_t)((n0 + lane + 64 * e < N ? lane + 64 * e : N - 1 - n0) * sizeof(T));
  const int xk = tid & 127, xb = wave >> 1;
  const int64_t kk = k0 + xk < Kp ? k0 + xk : Kp - 1;
  const uint32_t xoff = (uint32_t)(kk - k0) * 8, eoff = (uint32_t)(kk / 8 - k0 / 8);
  const int ydst = AB + lane * 128 + ((wave ^ ((lane >> 1) & 7)) * 16);   // lane + 64: same swizzle
  const int xsw = (xk >> 1) & 7;
  struct Ahead {
    T y[8][2];
    u32x2 q[2];
    uint32_t e[2];
  };
  // No branch may surround these loads: the wait for a step's loads counts the younger ones behind them, and a load that
  // may not have been issued does not count, so that the wait would reach into the step just issued.  Past the last step
  // and the last row the last ones are read again.  Addresses are scalar bases plus fixed lane offsets.
  const int64_t rb = lddy * (int64_t)sizeof(T);
  const char *const ybase = reinterpret_cast<const char *>(dY + n0);
  auto issue = [&](Ahead &h, int s) __attribute__((always_inline)) {
    s = s < s_hi ? s : s_hi - 1;
    const int m_ = s * GR_ROWS + wave * 8, m = __builtin_amdgcn_readfirstlane(m_ < (int)M ? m_ : (int)M - 1);
    const int rem = (int)M - 1 - m;
    const char *r = ybase + m * rb;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i) r += i <= rem ? rb : 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) h.y[i][e] = *reinterpret_cast<const T *>(r + yoff[e]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      int mb = s * (GR_ROWS / 8) + xb + 4 * j;
      mb = __builtin_amdgcn_readfirstlane(mb < mbs ? mb : mbs - 1);  // finite (or already NaN) times the zeros that put makes of rows past the last
      h.q[j] = *reinterpret_cast<const u32x2 *>(codes + (mb * Kp + k0) * 8 + xoff);
      h.e[j] = *(exps + (mb * Kp + k0) / 8 + eoff);
    }
  };
  float dbacc[2] = {0.0f, 0.0f};
  auto put = [&](Ahead &h, int s, int b) __attribute__((always_inline)) {
    if ((s + 1) * GR_ROWS > (int)M || s >= s_hi) {  // rows past the last, and a step past the last, add nothing
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s * GR_ROWS + wave * 8 + i >= (int)M || s >= s_hi) h.y[i][0] = h.y[i][1] = T(0.0f);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t w[4][P];
#pragma unroll
      for (int i = 0; i < 4; ++i) Split<T>::two(h.y[2 * i][e], h.y[2 * i + 1][e], w[i]);
#pragma unroll
      for (int p = 0; p < P; ++p)
        *reinterpret_cast<u32x4 *>(lds[b] + ydst + p * AB + e * 64 * 128) = u32x4{w[0][p], w[1][p], w[2][p], w[3][p]};
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      *reinterpret_cast<u32x4 *>(lds[b] + xk * 128 + (((xb + 4 * j) ^ xsw) * 16)) = q8_frag<RELU>(h.q[j], h.e[j]);
    if (sum_db) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) dbacc[e] += to_f32(h.y[i][e]);
    }
  };

  f32x4_t acc[4][2];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int i = 0; i < 2; ++i) acc[a][i] = f32x4_t{0, 0, 0, 0};
  const int arow = (wk * 64 + l16) * 128, brow = AB + (wn * 32 + l16) * 128, sw = l16 >> 1;
  auto step = [&](Ahead &now, Ahead &next, int s, int b) __attribute__((always_inline)) {
    u32x4 x[2][4], y[2][P][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int ck = ((t * 4 + c) ^ sw) * 16;
#pragma unroll
      for (int a = 0; a < 4; ++a) x[t][a] = *reinterpret_cast<const u32x4 *>(lds[b] + arow + a * 2048 + ck);
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < 2; ++i) y[t][p][i] = *reinterpret_cast<const u32x4 *>(lds[b] + brow + p * AB + i * 2048 + ck);
    }
    issue(now, s + 2);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[a][i] = mfma(x[t][a], y[t][p][i], acc[a][i]);
    put(next, s + 1, b ^ 1);
    __syncthreads();
  };
  Ahead h0, h1;
  if (s_lo < s_hi) {
    issue(h0, s_lo);
    issue(h1, s_lo + 1);
    put(h0, s_lo, 0);
  }
  __syncthreads();
  // two steps a turn whatever their number (a step past the last adds zeros): a loop that may leave after the first makes the
  // compiler copy registers whose loads are in flight, and wait for them
#pragma unroll 1
  for (int s = s_lo; s < s_hi; s += 2) {
    step(h0, h1, s, 0);
    step(h1, h0, s + 1, 1);
  }
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t k = k0 + wk * 64 + a * 16 + 4 * c + r;
      if (k >= K) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t n = n0 + wn * 32 + i * 16 + l16;
        if (n < N) dW[k * lddw + n] = acc[a][i][r];
      }
    }
  if (sum_db) {  // rows 8 wave .. of every step, added over the waves in order
    float *red = reinterpret_cast<float *>(lds);
    red[wave * 128 + lane] = dbacc[0];
    red[wave * 128 + 64 + lane] = dbacc[1];
    __syncthreads();
    if (tid < 128 && n0 + tid < N) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += red[w * 128 + tid];
      db[n0 + tid] = v;
    }
  }
}

// partial sums [splits][K + 1][N] (the last row: db) -> dW, db, in order
static __global__ __launch_bounds__(256) void grads_sum_kernel(int64_t K, int64_t N, int splits, const float *__restrict__ part,
                                                               float *__restrict__ dW, int64_t lddw, float *__restrict__ db) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  for (int64_t k = blockIdx.y; k < (db ? K + 1 : K); k += gridDim.y) {
    const float v = sum_parts(part + k * N + n, (K + 1) * N, splits);
    if (k < K) dW[k * lddw + n] = v;
    else db[n] = v;
  }
}

template <typename T, bool RELU>
static void launch_grads(hipStream_t st, const GradsPlan &p, int64_t M, int64_t K, int64_t N, const void *codes,
                         const void *exps, const T *dY, int64_t lddy, float *dW, int64_t lddw, float *db, float *work) {
  const bool split = p.splits > 1;
  const dim3 grid((unsigned)p.blocks, (unsigned)p.splits);
  hipLaunchKernelGGL((grads_kernel<T, RELU>), grid, dim3(GR_THREADS), 0, st, M, K, N, (const char *)codes,
                     (const uint8_t *)exps, dY, lddy, p.ktiles, (int)cdiv(M, GR_ROWS), p.steps, split ? work : dW,
                     split ? N : lddw, split ? (db ? work + K * N : nullptr) : db, split ? (K + 1) * N : 0);
  if (split)
    hipLaunchKernelGGL(grads_sum_kernel, dim3((unsigned)cdiv(N, 256), (unsigned)(K < 4096 ? K + 1 : 4096)), dim3(256), 0, st, K, N, p.splits, work, dW, lddw, db);
}

}  // namespace gpvae_lb
