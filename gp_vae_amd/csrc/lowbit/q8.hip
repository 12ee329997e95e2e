// q8.hip — activation checkpoints in 8 bits: writer (with the ReLU), reader, parameter gradients of a dense layer.
#include "grads.hpp"

namespace gpvae_lb {

// One thread per tile of 8 x 8.
template <typename T, bool RELU>
__global__ __launch_bounds__(256) void store_q8_kernel(int64_t M, int64_t K, const T *X, int64_t ldx, T *Y, int64_t ldy,
                                                       uint8_t *__restrict__ codes, uint8_t *__restrict__ exps) {
  const int64_t Kp = q8_kp(K), kt = Kp / 8, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= q8_mb(M) * kt) return;
  const int64_t mb = id / kt, t = id % kt, m0 = mb * 8, k0 = t * 8;
  float amax = 0.0f;
  bool bad = false;
  for (int i = 0; i < 8; ++i)
    for (int c = 0; c < 8; ++c)
      if (m0 + i < M && k0 + c < K) {
        float v = to_f32(X[(m0 + i) * ldx + k0 + c]);
        if (RELU) v = v < 0.0f ? 0.0f : v;
        bad |= !(fabsf(v) <= 3.402823466e+38f);
        amax = fmaxf(amax, fabsf(v));
      }
  const int eb = bad ? 255 : (RELU ? tile_exp_byte<255, 7, -126>(amax) : tile_exp_byte<127, 6, -126>(amax));
  exps[mb * kt + t] = (uint8_t)eb;
  for (int c = 0; c < 8; ++c) {
    uint64_t w = 0;
    for (int i = 0; i < 8; ++i)
      if (m0 + i < M && k0 + c < K) {
        float v = to_f32(X[(m0 + i) * ldx + k0 + c]);
        if (RELU) {
          v = v < 0.0f ? 0.0f : v;
          if (Y) Y[(m0 + i) * ldy + k0 + c] = from_f32<T>(v);
        }
        int q = bad ? 0 : (int)rintf(unscale<RELU ? 255 : 127>(v, eb));
        if (RELU && q == 0 && !(v <= 0.0f)) q = 1;
        w |= (uint64_t)(uint8_t)q << (8 * i);
      }
    *reinterpret_cast<uint64_t *>(codes + (mb * Kp + k0 + c) * 8) = w;
  }
}

template <bool RELU>
__device__ __forceinline__ float q8_value(const uint8_t *codes, const uint8_t *exps, int64_t Kp, int64_t m, int64_t k) {
  const uint8_t q = codes[((m / 8) * Kp + k) * 8 + m % 8];
  return (RELU ? (float)q : (float)(int8_t)q) * scale_of(exps[(m / 8) * (Kp / 8) + k / 8]);
}

template <typename T, bool RELU>
__global__ __launch_bounds__(256) void load_q8_kernel(int64_t M, int64_t K, const uint8_t *__restrict__ codes,
                                                      const uint8_t *__restrict__ exps, T *__restrict__ out, int64_t ldo) {
  const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (k >= K) return;
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y) out[m * ldo + k] = from_f32<T>(q8_value<RELU>(codes, exps, q8_kp(K), m, k));
}

static int check_q8(const char *fn, int dtype, int64_t M, int64_t K) {
  LB_REQUIRE(dtype_ok(dtype), 2, "%s: dtype must be float32, bfloat16 or float16 (got %d)", fn, dtype);
  LB_REQUIRE(M >= 0 && M <= (1 << 30), 3, "%s: M must lie in [0, 2^30] (got %lld)", fn, (long long)M);
  LB_REQUIRE(K >= 1 && K <= (1 << 30), 4, "%s: K must lie in [1, 2^30] (got %lld)", fn, (long long)K);
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
  const int64_t tiles = q8_mb(M) * (q8_kp(K) / 8);
  LB_REQUIRE(cdiv(tiles, 256) <= 0x7fffffff, 3, "%s: matrix too large", fn);
#define GO2(T, R)                                                                                                        \
  hipLaunchKernelGGL((store_q8_kernel<T, R>), dim3((unsigned)cdiv(tiles, 256)), dim3(256), 0, (hipStream_t)stream, M, K, \
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
  const dim3 grid((unsigned)cdiv(K, 256), (unsigned)(M < 65535 ? M : 65535));
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
  if (!dtype_ok(dtype) || M < 0 || K < 1 || N < 1) return 0;
  const GradsPlan p = grads_plan(M, K, N);
  return p.splits > 1 ? p.splits * (K + 1) * N * 4 : 0;
}

extern "C" int gpvae_dense_grads_q8(void *stream, int dtype, int64_t M, int64_t K, int64_t N, int relu, const void *codes,
                                    const void *exps, const void *dY, int64_t lddy, float *dW, int64_t lddw, float *db,
                                    void *work) {
  const char *fn = "gpvae_dense_grads_q8";
  if (const int rc = check_q8(fn, dtype, M, K)) return rc;
  LB_REQUIRE(N >= 1 && N <= (1 << 30), 5, "%s: N must lie in [1, 2^30] (got %lld)", fn, (long long)N);
  LB_REQUIRE(M == 0 || (codes && aligned16(codes)), 7, "%s: codes must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(M == 0 || (exps && aligned16(exps)), 8, "%s: exps must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(M == 0 || dY, 9, "%s: dY is NULL", fn);
  LB_REQUIRE(M == 0 || lddy >= N, 10, "%s: lddy < N", fn);
  LB_REQUIRE(dW, 11, "%s: dW is NULL", fn);
  LB_REQUIRE(lddw >= N, 12, "%s: lddw < N", fn);
  LB_REQUIRE(!gpvae_dense_grads_q8_workspace_bytes(dtype, M, K, N) || (work && aligned16(work)), 14,
             "%s: work must be a 16-byte aligned device pointer", fn);
  const GradsPlan p = grads_plan(M, K, N);
#define GO2(T, R)                                                                                                       \
  launch_grads<T, R>((hipStream_t)stream, p, M, K, N, codes, exps, (const T *)dY, lddy, dW, lddw, db, (float *)work)
#define GO(T) do { if (relu) GO2(T, true); else GO2(T, false); } while (0)
  LB_BY_DTYPE(dtype, GO);
#undef GO
#undef GO2
  LB_CHECK_LAUNCH(fn);
  return 0;
}
