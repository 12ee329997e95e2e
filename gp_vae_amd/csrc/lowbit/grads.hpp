// grads.hpp — parameter gradients of a dense layer from the 8-bit checkpoint of its input:
//   dW[k][n] = sum_m X~[m][k] dY[m][n],   db[n] = sum_m dY[m][n].
//
// The reduction runs over the ROWS of both operands, the matrix instruction wants 8 consecutive reduction indices per lane.
// The checkpoint is laid out for that (8 rows of a column are 8 consecutive bytes); dY is transposed on its way into
// LDS: a thread loads 8 consecutive rows of a column (consecutive lanes: consecutive columns), splits them into their
// bfloat16 pieces and writes each piece's 8 values as 16 bytes.  One 128 x 128 tile per workgroup, 64 rows a step, loaded
// one step ahead through buffer descriptors: scalar bases, and rows past the end read as zero without a test.
// float32 is bound by matrix and vector instructions, of which little overlaps (4096 x 1024 x 4096: 43 % and 37 % of the time; 103-107 us,
// 960-1000 TFLOP/s over the three pieces), the other types by instruction issue, LDS and the step's barrier (bfloat16 50 us, float16
// 74 us; a library product of two bfloat16 matrices of this size: 52 us).  All row tiles of a column tile run on one
// XCD (xcd_chunk), whose L2 then serves dY to them: dealt round-robin every XCD read all of dY from memory (140 us before,
// 122 after).  Tried without gain: 4 steps in flight, the two waves of a SIMD half a step apart, matrix and vector instructions
// alternating, the checkpoint decoded by a launch of its own.
#pragma once
#include "frag.hpp"

namespace gpvae_lb {

constexpr int GR_THREADS = 512, GR_ROWS = 64;

struct GradsPlan {
  int ktiles, splits, steps;
  int64_t blocks;
};
// Into how many parts are the rows split?  A step takes 0.35 + 0.38 P us (P pieces of dY), every full round of 256 workgroups
// anew; a split costs the launch that adds the parts (4 us) and writing and reading them.  The least of that estimate over
// powers of two and the number that gives every unit a workgroup.  Measured, one part / two / four: bfloat16 300 x 700 x 1001
// 10.1 / 15.2 / 15.0 us, float32 300 x 700 x 1000 14.2 / 18.3 / 17.0, 2000 x 1024 x 1024 52 / 39 / 28.5.
static inline GradsPlan grads_plan(int P, int64_t M, int64_t K, int64_t N) {
  GradsPlan p;
  p.ktiles = (int)cdiv(K, 128);
  p.blocks = p.ktiles * cdiv(N, 128);
  const int64_t steps = M > 0 ? cdiv(M, GR_ROWS) : 1;
  p.splits = 1;
  p.steps = (int)steps;
  double best = 0.0;
  for (int64_t i = 1; i <= 256; i *= 2)
    for (int64_t s : {i, i < 256 ? int64_t(0) : 256 / p.blocks}) {
      if (s < 1 || (s > 1 && (s * p.blocks > 320 || s * 2 > steps))) continue;
      const int64_t per = round_up(cdiv(steps, s), 2), parts = cdiv(steps, per);
      const double t = (double)(per * cdiv(parts * p.blocks, 256)) * (0.35 + 0.38 * P) +
                       (parts > 1 ? 4.0 + (double)parts * ((double)(K + 1) * (double)N * (8 / 4.5e6) + 0.06) : 0.0);
      if (s == 1 || t < best) best = t, p.splits = (int)parts, p.steps = (int)per;
    }
  return p;
}

// 8 codes (bytes) -> 8 bfloat16 values times 2^e; exponent byte eb (255: NaN).  A signed code is scaled as it is: taken as an
// offset and a correction of 128 2^e, the correction would overflow at the largest e.
template <bool RELU> __device__ __forceinline__ u32x4 q8_frag(u32x2 q, uint32_t eb) {
  const float s = scale_of(eb);
  float v[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w = q[h];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * h + i] = (RELU ? (float)((w >> (8 * i)) & 255u) : (float)(int8_t)(w >> (8 * i))) * s;  // exact
  }
  return u32x4{pack_hi(v[0], v[1]), pack_hi(v[2], v[3]), pack_hi(v[4], v[5]), pack_hi(v[6], v[7])};
}

// What a thread has loaded of dY for a step: 8 rows of two columns, which are lane and lane + 64, or, for two-byte types (PAIR),
// 2 lane and 2 lane + 1 with one load for both.
template <typename T, bool PAIR> struct RowsOf {
  uint32_t w[8][PAIR ? 1 : 2];
  // row i, whose columns lie o0 and o1 bytes from the base
  __device__ __forceinline__ void load(rsrc_t r, int i, uint32_t o0, uint32_t o1) {
    if constexpr (PAIR) {
      w[i][0] = __builtin_amdgcn_raw_buffer_load_b32(r, o0, 0, 0);
    } else if constexpr (sizeof(T) == 4) {
      w[i][0] = __builtin_amdgcn_raw_buffer_load_b32(r, o0, 0, 0);
      w[i][1] = __builtin_amdgcn_raw_buffer_load_b32(r, o1, 0, 0);
    } else {
      w[i][0] = __builtin_amdgcn_raw_buffer_load_b16(r, o0, 0, 0);
      w[i][1] = __builtin_amdgcn_raw_buffer_load_b16(r, o1, 0, 0);
    }
  }
  __device__ __forceinline__ T value(int i, int e) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, w[i][e]);
    else if constexpr (PAIR) return __builtin_bit_cast(T, (uint16_t)(w[i][0] >> (16 * e)));
    else return __builtin_bit_cast(T, (uint16_t)w[i][e]);
  }
  // rows i and i + 1 of a column -> one dword of each piece
  __device__ __forceinline__ void split(int i, int e, uint32_t *out) const {
    if constexpr (__is_same(T, __bf16))
      out[0] = PAIR ? __builtin_amdgcn_perm(w[i + 1][0], w[i][0], e ? 0x07060302u : 0x05040100u)
                    : __builtin_amdgcn_perm(w[i + 1][e], w[i][e], 0x05040100u);
    else Split<T>::two(value(i, e), value(i + 1, e), out);
  }
};

template <typename T, bool RELU, bool PAIR>
__global__ __launch_bounds__(GR_THREADS, 2) void grads_kernel(int64_t M, int64_t K, int64_t N, const char *__restrict__ codes,
                                                              const char *__restrict__ exps, const T *__restrict__ dY,
                                                              int64_t lddy, int ktiles, int s_all, int steps, float *dW,
                                                              int64_t lddw, float *db, int64_t part_stride) {
  constexpr int P = Split<T>::P, AB = 128 * 128, ST = AB * (1 + P);  // bytes of one image of 128 rows x 64; of a stage
  __shared__ __align__(16) unsigned char lds[2][ST];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave >> 2, wn = wave & 3, c = lane >> 4, l16 = lane & 15;  // wave: 64 rows of dW x 32 columns
  const uint32_t bt = (uint32_t)xcd_chunk(blockIdx.x, gridDim.x);
  const uint32_t nt = __builtin_amdgcn_readfirstlane(bt / (uint32_t)ktiles), kt = bt - nt * (uint32_t)ktiles;
  const int64_t k0 = (int64_t)kt * 128, n0 = (int64_t)nt * 128;
  const int s_lo = (int)blockIdx.y * steps, s_hi = s_lo + steps < s_all ? s_lo + steps : s_all;
  const int64_t Kp = q8_kp(K);
  const bool sum_db = db != nullptr && kt == 0;
  dW += blockIdx.y * part_stride;
  if (db) db += blockIdx.y * part_stride;

  // dY share: two columns, rows 8 wave .. + 7 of the step; checkpoint share: columns 2 lane and 2 lane + 1 of the same rows,
  // which are one tile row.  Everything outside the matrices, and a step past the last, is loaded as zero.
  const int ycol0 = PAIR ? 2 * lane : lane, ycol1 = PAIR ? ycol0 + 1 : lane + 64;
  // 16-byte chunks of an image row at chunk ^ (row / 2 % 8) where a thread writes two neighbouring rows, at chunk ^ (row % 8) where
  // neighbouring threads do: eight consecutive lanes then write to, and a fragment's lanes read from, different banks
  const int ydst0 = AB + ycol0 * 128 + ((wave ^ ((PAIR ? lane : ycol0) & 7)) * 16), ydst1 = ydst0 + (ycol1 - ycol0) * 128;
  const int xdst = lane * 256 + ((wave ^ (lane & 7)) * 16);
  struct Ahead {
    RowsOf<T, PAIR> y;
    u32x4 q;
    uint32_t e;
  };
  // No branch may surround these loads: the wait for a step's loads counts the younger ones behind them, and a load that
  // may not have been issued does not count, so that the wait would reach into the step just issued.  The steps are loaded in order:
  // the bases move on by themselves, and the loop spends few scalar instructions on addresses (a wave issues one instruction in
  // four cycles, and two waves share a SIMD).
  const uint32_t rb = (uint32_t)(lddy * (int64_t)sizeof(T));
  const int ybytes = (int)(N - n0 < 128 ? N - n0 : 128) * (int)sizeof(T), xcols = (int)(Kp - k0 < 128 ? Kp - k0 : 128);
  // columns past the last: the last one (pair) again, results unused
  const int yl0 = ycol0 * (int)sizeof(T), yl1 = ycol1 * (int)sizeof(T), ylast = ybytes - (PAIR ? 2 : 1) * (int)sizeof(T);
  uint32_t yo[8][2];  // lddy <= 2^26: 8 rows lie within a 32-bit offset (the scalar offset is not part of the range check)
#pragma unroll
  for (int i = 0; i < 8; ++i) yo[i][0] = (uint32_t)i * rb + (yl0 < ylast ? yl0 : ylast), yo[i][1] = (uint32_t)i * rb + (yl1 < ylast ? yl1 : ylast);
  int64_t m_end = (int64_t)s_hi * GR_ROWS;
  m_end = m_end < M ? m_end : M;
  int left = (int)(m_end - (int64_t)s_lo * GR_ROWS);  // rows from the next step's first to the last of this workgroup
  const char *yb = reinterpret_cast<const char *>(dY + n0) + ((int64_t)s_lo * GR_ROWS + wave * 8) * (int64_t)rb;
  const int64_t at = ((int64_t)s_lo * (GR_ROWS / 8) + wave) * Kp + k0;
  const char *qb = codes + at * 8, *eb = exps + at / 8;
  auto issue = [&](Ahead &h) __attribute__((always_inline)) {
    int rows = left - wave * 8;
    rows = rows < 8 ? rows : 8;
    const rsrc_t ry = buffer(yb, rows > 0 ? (int)((rows - 1) * rb + ybytes) : 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) h.y.load(ry, i, yo[i][0], yo[i][1]);
    h.q = __builtin_amdgcn_raw_buffer_load_b128(buffer(qb, rows > 0 ? xcols * 8 : 0), lane * 16, 0, 0);
    h.e = __builtin_amdgcn_raw_buffer_load_b8(buffer(eb, rows > 0 ? xcols / 8 : 0), lane / 4, 0, 0);
    qb += Kp * GR_ROWS;
    eb += Kp;
    yb += (int64_t)rb * GR_ROWS;
    left -= GR_ROWS;
  };
  float dbacc[2] = {0.0f, 0.0f};
  auto put = [&](const Ahead &h, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t w[4][P];
#pragma unroll
      for (int i = 0; i < 4; ++i) h.y.split(2 * i, e, w[i]);
#pragma unroll
      for (int p = 0; p < P; ++p)
        *reinterpret_cast<u32x4 *>(lds[b] + (e ? ydst1 : ydst0) + p * AB) = u32x4{w[0][p], w[1][p], w[2][p], w[3][p]};
    }
    *reinterpret_cast<u32x4 *>(lds[b] + xdst) = q8_frag<RELU>(u32x2{h.q.x, h.q.y}, h.e);
    *reinterpret_cast<u32x4 *>(lds[b] + xdst + 128) = q8_frag<RELU>(u32x2{h.q.z, h.q.w}, h.e);
    if (sum_db) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) dbacc[e] += to_f32(h.y.value(i, e));
    }
  };

  f32x4_t acc[4][2];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int i = 0; i < 2; ++i) acc[a][i] = f32x4_t{0, 0, 0, 0};
  const int arow = (wk * 64 + l16) * 128, brow = AB + (wn * 32 + l16) * 128, xrsw = l16 >> 1, yrsw = PAIR ? l16 >> 1 : l16 & 7;
  auto multiply = [&](int b) __attribute__((always_inline)) {
    u32x4 x[2][4], y[2][P][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int xc = ((t * 4 + c) ^ xrsw) * 16, yc = ((t * 4 + c) ^ yrsw) * 16;
#pragma unroll
      for (int a = 0; a < 4; ++a) x[t][a] = *reinterpret_cast<const u32x4 *>(lds[b] + arow + a * 2048 + xc);
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < 2; ++i) y[t][p][i] = *reinterpret_cast<const u32x4 *>(lds[b] + brow + p * AB + i * 2048 + yc);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[a][i] = mfma(x[t][a], y[t][p][i], acc[a][i]);
  };
  // Step s is in lds[b], `next` holds s + 1 in flight, s + 2 replaces `now`.
  auto step = [&](Ahead &now, Ahead &next, int b) __attribute__((always_inline)) {
    issue(now);
    multiply(b);
    put(next, b ^ 1);
    __syncthreads();
  };
  Ahead h0, h1;
  if (s_lo < s_hi) {
    issue(h0);
    issue(h1);
    put(h0, 0);
  }
  __syncthreads();
  // two steps a turn whatever their number (a step past the last adds zeros): a loop that may leave after the first makes the
  // compiler copy registers whose loads are in flight, and wait for them
#pragma unroll 1
  for (int s = s_lo; s < s_hi; s += 2) {
    step(h0, h1, 0);
    step(h1, h0, 1);
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
    red[wave * 128 + ycol0] = dbacc[0];
    red[wave * 128 + ycol1] = dbacc[1];
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
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(GR_THREADS), 0, st, M, K, N, (const char *)codes, (const char *)exps, dY, lddy,
                       p.ktiles, (int)cdiv(M, GR_ROWS), p.steps, split ? work : dW, split ? N : lddw,
                       split ? (db ? work + K * N : nullptr) : db, split ? (K + 1) * N : 0);
  };
  // Two-byte types: both columns of a pair exist or neither, and a pair is aligned to 4 bytes.  One load for two columns
  // against two: bfloat16 4096 x 1024 x 4096 50 us, 4096 x 1024 x 4095 59.  (float32 in pairs gained nothing.)
  if constexpr (sizeof(T) == 2) {
    if (N % 2 == 0 && lddy % 2 == 0 && ((uintptr_t)dY & 3) == 0) launch(grads_kernel<T, RELU, true>);
    else launch(grads_kernel<T, RELU, false>);
  } else {
    launch(grads_kernel<T, RELU, false>);
  }
  if (split && hipPeekAtLastError() == hipSuccess)
    hipLaunchKernelGGL(grads_sum_kernel, dim3((unsigned)cdiv(N, 256), (unsigned)(K < 4096 ? K + 1 : 4096)), dim3(256), 0, st, K, N, p.splits, work, dW, lddw, db);
}

}  // namespace gpvae_lb
