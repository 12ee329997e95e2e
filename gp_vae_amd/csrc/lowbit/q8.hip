// q8.hip — activation checkpoints in 8 bits: writer (with the ReLU), reader, parameter gradients of a dense layer.
#include "grads.hpp"

namespace gpvae_lb {

// Bound by memory: X is read once, Y and the codes are written once.  A thread owns a strip of 8 rows x 4 columns, half a
// tile: 8 loads of 4 elements (16 bytes of float32) cover the strip, the tile's largest magnitude is one exchange with the
// neighbouring lane, and its 4 columns of codes are 32 consecutive bytes.  Consecutive lanes take consecutive
// strips of the same rows, so that every row of a wave is one contiguous stretch.  Measured, float32 4096 x 4096 with the
// ReLU's output: 26.2 us, 5.8 TB/s (the matrices fit the last-level cache; 16384 x 4096 with the reader: 188 us, 5.0 TB/s).
template <typename T, bool RELU>
__global__ __launch_bounds__(256) void store_q8_kernel(int64_t M, int64_t K, const T *X, int64_t ldx, T *Y, int64_t ldy,
                                                       uint8_t *__restrict__ codes, uint8_t *__restrict__ exps) {
  const int64_t Kp = q8_kp(K), strips = Kp / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t all = q8_mb(M) * strips;
  const bool live = id < all;  // (an even number of strips: a pair of lanes is live or not together)
  const int64_t mb = live ? id / strips : 0, k0 = live ? (id - mb * strips) * 4 : 0, m0 = mb * 8;
  const bool whole = m0 + 8 <= M && k0 + 4 <= K;
  Vec4<T> v[8];
  if (whole) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const Vec4<T> *>(X + (m0 + i) * ldx + k0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) v[i].v[c] = live && m0 + i < M && k0 + c < K ? X[(m0 + i) * ldx + k0 + c] : T(0.0f);
  }
  if (RELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) v[i].v[c] = to_f32(v[i].v[c]) < 0.0f ? T(0.0f) : v[i].v[c];
    if (Y) {
      if (whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<Vec4<T> *>(Y + (m0 + i) * ldy + k0) = v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (live && m0 + i < M && k0 + c < K) Y[(m0 + i) * ldy + k0 + c] = v[i].v[c];
      }
    }
  }
  // the largest magnitude as bits: an infinity or a NaN is above every finite value
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t b = __builtin_bit_cast(uint32_t, to_f32(v[i].v[c])) & 0x7fffffffu;
      top = b > top ? b : top;
    }
  const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true);  // the lane next to it
  const float amax = __builtin_bit_cast(float, other > top ? other : top);
  const int eb = RELU ? tile_exp_byte<255, 7, -126>(amax) : tile_exp_byte<127, 6, -126>(amax);
  const int e = eb - 127, h = e >> 1;
  const float s1 = pow2f(-h), s2 = pow2f(h - e);
  uint32_t w[4][2];
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      w[c][g] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = to_f32(v[4 * g + i].v[c]);
        uint32_t q = 0;
        if (RELU) {
          q = (uint32_t)fminf(rintf(x * s1 * s2), 255.0f);
          q = eb == 255 ? 0u : q;
          q = q == 0 && !(x <= 0.0f) ? 1u : q;
        } else {
          q = (uint32_t)(int)fminf(fmaxf(rintf(x * s1 * s2), -127.0f), 127.0f) & 255u;
          q = eb == 255 ? 0u : q;
        }
        w[c][g] |= q << (8 * i);
      }
    }
  if (!live) return;
  u32x4 *dst = reinterpret_cast<u32x4 *>(codes + (mb * Kp + k0) * 8);
  dst[0] = u32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
  dst[1] = u32x4{w[2][0], w[2][1], w[3][0], w[3][1]};
  if ((id & 1) == 0) exps[mb * (Kp / 8) + k0 / 8] = (uint8_t)eb;
}

// The reverse: a thread reads its strip's 32 bytes of codes and writes 8 rows of 4 elements (4096 x 4096: 15.5 us, 5.4 TB/s).
template <typename T, bool RELU>
__global__ __launch_bounds__(256) void load_q8_kernel(int64_t M, int64_t K, const uint8_t *__restrict__ codes,
                                                      const uint8_t *__restrict__ exps, T *__restrict__ out, int64_t ldo) {
  const int64_t Kp = q8_kp(K), strips = Kp / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= q8_mb(M) * strips) return;
  const int64_t mb = id / strips, k0 = (id - mb * strips) * 4, m0 = mb * 8;
  const u32x4 *src = reinterpret_cast<const u32x4 *>(codes + (mb * Kp + k0) * 8);
  const u32x4 a = src[0], b = src[1];
  const uint32_t w[4][2] = {{a.x, a.y}, {a.z, a.w}, {b.x, b.y}, {b.z, b.w}};
  const float s = scale_of(exps[mb * (Kp / 8) + k0 / 8]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    Vec4<T> v;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t q = (w[c][i >> 2] >> (8 * (i & 3))) & 255u;
      v.v[c] = from_f32<T>((RELU ? (float)q : (float)(int8_t)q) * s);
    }
    if (m0 + i >= M) break;
    if (k0 + 4 <= K) {
      *reinterpret_cast<Vec4<T> *>(out + (m0 + i) * ldo + k0) = v;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (k0 + c < K) out[(m0 + i) * ldo + k0 + c] = v.v[c];
    }
  }
}

static int check_q8(const char *fn, int dtype, int64_t M, int64_t K) {
  LB_REQUIRE(dtype_ok(dtype), 2, "%s: dtype must be float32, bfloat16 or float16 (got %d)", fn, dtype);
  LB_REQUIRE(M >= 0 && M <= MAX_MK, 3, "%s: M must lie in [0, 2^30] (got %lld)", fn, (long long)M);
  LB_REQUIRE(K >= 1 && K <= MAX_MK, 4, "%s: K must lie in [1, 2^30] (got %lld)", fn, (long long)K);
  return 0;
}

}  // namespace gpvae_lb

using namespace gpvae_lb;

extern "C" int gpvae_store_q8(void *stream, int dtype, int64_t M, int64_t K, const void *X, int64_t ldx, int relu, void *Y,
                              int64_t ldy, void *codes, void *exps) {
  const char *fn = "gpvae_store_q8";
  if (const int rc = check_q8(fn, dtype, M, K)) return rc;
  if (M == 0) return 0;
  LB_REQUIRE(X, 5, "%s: X is NULL", fn);
  LB_REQUIRE(ldx >= K, 6, "%s: ldx < K", fn);
  LB_REQUIRE(relu || !Y, 8, "%s: Y is the ReLU's output: NULL without relu", fn);
  LB_REQUIRE(!Y || ldy >= K, 9, "%s: ldy < K", fn);
  LB_REQUIRE(Y != X || ldy == ldx, 9, "%s: in place needs ldy == ldx", fn);
  LB_REQUIRE(codes && aligned16(codes), 10, "%s: codes must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(exps && aligned16(exps), 11, "%s: exps must be a 16-byte aligned device pointer", fn);
  const int64_t strips = q8_mb(M) * (q8_kp(K) / 4);
  LB_REQUIRE(launchable(cdiv(strips, 256), 256), 3, "%s: matrix too large", fn);
#define GO2(T, R)                                                                                                        \
  hipLaunchKernelGGL((store_q8_kernel<T, R>), dim3((unsigned)cdiv(strips, 256)), dim3(256), 0, (hipStream_t)stream, M, K, \
                     (const T *)X, ldx, (T *)Y, ldy, (uint8_t *)codes, (uint8_t *)exps)
#define GO(T) do { if (relu) GO2(T, true); else GO2(T, false); } while (0)
  LB_BY_DTYPE(dtype, GO);
#undef GO
#undef GO2
  LB_CHECK_LAUNCH(fn);
  return 0;
}

extern "C" int gpvae_load_q8(void *stream, int dtype, int64_t M, int64_t K, int relu, const void *codes, const void *exps,
                             void *out, int64_t ldo) {
  const char *fn = "gpvae_load_q8";
  if (const int rc = check_q8(fn, dtype, M, K)) return rc;
  if (M == 0) return 0;
  LB_REQUIRE(codes && aligned16(codes), 6, "%s: codes must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(exps && aligned16(exps), 7, "%s: exps must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(out, 8, "%s: out is NULL", fn);
  LB_REQUIRE(ldo >= K, 9, "%s: ldo < K", fn);
  const int64_t strips = q8_mb(M) * (q8_kp(K) / 4);
  LB_REQUIRE(launchable(cdiv(strips, 256), 256), 3, "%s: matrix too large", fn);
  const dim3 grid((unsigned)cdiv(strips, 256));
#define GO2(T, R)                                                                                                  \
  hipLaunchKernelGGL((load_q8_kernel<T, R>), grid, dim3(256), 0, (hipStream_t)stream, M, K, (const uint8_t *)codes, \
                     (const uint8_t *)exps, (T *)out, ldo)
#define GO(T) do { if (relu) GO2(T, true); else GO2(T, false); } while (0)
  LB_BY_DTYPE(dtype, GO);
#undef GO
#undef GO2
  LB_CHECK_LAUNCH(fn);
  return 0;
}

extern "C" int64_t gpvae_dense_grads_q8_workspace_bytes(int dtype, int64_t M, int64_t K, int64_t N) {
  if (!dtype_ok(dtype) || M < 0 || M > MAX_MK || K < 1 || K > MAX_MK || N < 1 || N > MAX_N_GRADS) return 0;
  const GradsPlan p = grads_plan(pieces(dtype), M, K, N);
  return p.splits > 1 ? p.splits * (K + 1) * N * 4 : 0;
}

extern "C" int gpvae_dense_grads_q8(void *stream, int dtype, int64_t M, int64_t K, int64_t N, int relu, const void *codes,
                                    const void *exps, const void *dY, int64_t lddy, float *dW, int64_t lddw, float *db,
                                    void *work) {
  const char *fn = "gpvae_dense_grads_q8";
  if (const int rc = check_q8(fn, dtype, M, K)) return rc;
  LB_REQUIRE(N >= 1 && N <= MAX_N_GRADS, 5, "%s: N must lie in [1, 2^26] (got %lld)", fn, (long long)N);
  LB_REQUIRE(M == 0 || (codes && aligned16(codes)), 7, "%s: codes must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(M == 0 || (exps && aligned16(exps)), 8, "%s: exps must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(M == 0 || dY, 9, "%s: dY is NULL", fn);
  LB_REQUIRE(M == 0 || lddy >= N, 10, "%s: lddy < N", fn);
  if (M <= 1) lddy = N;
  LB_REQUIRE(lddy <= (1 << 26), 10, "%s: lddy must not exceed 2^26 (got %lld)", fn, (long long)lddy);
  LB_REQUIRE(dW, 11, "%s: dW is NULL", fn);
  LB_REQUIRE(lddw >= N, 12, "%s: lddw < N", fn);
  LB_REQUIRE(!gpvae_dense_grads_q8_workspace_bytes(dtype, M, K, N) || (work && aligned16(work)), 14,
             "%s: work must be a 16-byte aligned device pointer", fn);
  const GradsPlan p = grads_plan(pieces(dtype), M, K, N);
  LB_REQUIRE(launchable(p.blocks, GR_THREADS), 4, "%s: K x N too large (%lld tiles of 128 x 128)", fn, (long long)p.blocks);
#define GO2(T, R)                                                                                                       \
  launch_grads<T, R>((hipStream_t)stream, p, M, K, N, codes, exps, (const T *)dY, lddy, dW, lddw, db, (float *)work)
#define GO(T) do { if (relu) GO2(T, true); else GO2(T, false); } while (0)
  LB_BY_DTYPE(dtype, GO);
#undef GO
#undef GO2
  LB_CHECK_LAUNCH(fn);
  return 0;
}
