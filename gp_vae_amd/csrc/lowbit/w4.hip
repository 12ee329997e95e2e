// w4.hip — dense layers with weights in 4 bits: quantiser, reader, the product and the transposed product.
#include "skinny.hpp"
#include "tile.hpp"

namespace gpvae_lb {

// Bound by memory: W is read once.  A thread owns 32 rows x 4 columns, half of four tiles: rows are read 4 elements at a time
// (consecutive lanes: consecutive columns), a tile's largest magnitude is one exchange with the neighbouring lane, and
// the codes of its 4 columns are 64 consecutive bytes.  Measured, float32 4096 x 32768: 160 us, 3.8 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void quant_w4_kernel(int64_t K, int64_t N, const T *__restrict__ W, int64_t ldw,
                                                       u32x4 *__restrict__ codes, uint32_t *__restrict__ exps) {
  const int64_t Np = w4_np(N), strips = Np / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool live = id < w4_kb(K) * strips;  // (an even number of strips: a pair of lanes is live or not together)
  const int64_t kb = live ? id / strips : 0, n0 = live ? (id - kb * strips) * 4 : 0;
  const bool whole = kb * 32 + 32 <= K && n0 + 4 <= N;
  u32x4 out[4];
  uint32_t eall = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t k0 = kb * 32 + j * 8;
    Vec4<T> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (whole) {
        v[i] = *reinterpret_cast<const Vec4<T> *>(W + (k0 + i) * ldw + n0);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[i].v[c] = live && k0 + i < K && n0 + c < N ? W[(k0 + i) * ldw + n0 + c] : T(0.0f);
      }
    }
    uint32_t top = 0;  // the largest magnitude as bits: an infinity or a NaN is above every finite value
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t b = __builtin_bit_cast(uint32_t, to_f32(v[i].v[c])) & 0x7fffffffu;
        top = b > top ? b : top;
      }
    const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true);  // the lane next to it
    const int eb = tile_exp_byte<6, 2, -125>(__builtin_bit_cast(float, other > top ? other : top));
    eall |= (uint32_t)eb << (8 * j);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= e2m1_code(unscale<6>(to_f32(v[i].v[c]), eb)) << (4 * i);
      out[c][j] = eb == 255 ? 0u : w;
    }
  }
  if (!live) return;
#pragma unroll
  for (int c = 0; c < 4; ++c) codes[kb * Np + n0 + c] = out[c];
  if ((id & 1) == 0) exps[kb * (Np / 8) + n0 / 8] = eall;
}

// The reverse: a thread reads the 64 bytes of its 4 columns and writes 32 rows of 4 elements (4096 x 32768: 141 us, 4.3 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void load_w4_kernel(int64_t K, int64_t N, const u32x4 *__restrict__ codes,
                                                      const uint32_t *__restrict__ exps, T *__restrict__ out, int64_t ldo) {
  const int64_t Np = w4_np(N), strips = Np / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= w4_kb(K) * strips) return;
  const int64_t kb = id / strips, n0 = (id - kb * strips) * 4;
  u32x4 q[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) q[c] = codes[kb * Np + n0 + c];
  const uint32_t e = exps[kb * (Np / 8) + n0 / 8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float s = scale_of((e >> (8 * j)) & 255u);
    u32x4 f[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) f[c] = w4_frag(q[c][j], s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t k = kb * 32 + j * 8 + i;
      if (k >= K) return;
      Vec4<T> v;
#pragma unroll
      for (int c = 0; c < 4; ++c) v.v[c] = from_f32<T>(i & 1 ? bf_hi(f[c][i >> 1]) : bf_lo(f[c][i >> 1]));
      if (n0 + 4 <= N) {
        *reinterpret_cast<Vec4<T> *>(out + k * ldo + n0) = v;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n0 + c < N) out[k * ldo + n0 + c] = v.v[c];
      }
    }
  }
}

static int check_w4(const char *fn, int dtype, int64_t K, int64_t N, int kn_arg) {
  LB_REQUIRE(dtype_ok(dtype), 2, "%s: dtype must be float32, bfloat16 or float16 (got %d)", fn, dtype);
  LB_REQUIRE(K >= 1 && K <= MAX_MK, kn_arg, "%s: K must lie in [1, 2^30] (got %lld)", fn, (long long)K);
  LB_REQUIRE(N >= 1 && N <= MAX_N_W4, kn_arg + 1, "%s: N must lie in [1, 2^25] (got %lld)", fn, (long long)N);
  return 0;
}

}  // namespace gpvae_lb

using namespace gpvae_lb;

extern "C" int gpvae_quant_w4(void *stream, int dtype, int64_t K, int64_t N, const void *W, int64_t ldw, void *codes,
                              void *exps) {
  const char *fn = "gpvae_quant_w4";
  if (const int rc = check_w4(fn, dtype, K, N, 3)) return rc;
  LB_REQUIRE(W, 5, "%s: W is NULL", fn);
  LB_REQUIRE(ldw >= N, 6, "%s: ldw < N", fn);
  LB_REQUIRE(codes && aligned16(codes), 7, "%s: codes must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(exps && aligned16(exps), 8, "%s: exps must be a 16-byte aligned device pointer", fn);
  const int64_t strips = w4_kb(K) * (w4_np(N) / 4);
  LB_REQUIRE(launchable(cdiv(strips, 256), 256), 3, "%s: matrix too large", fn);
#define GO(T)                                                                                                         \
  hipLaunchKernelGGL(quant_w4_kernel<T>, dim3((unsigned)cdiv(strips, 256)), dim3(256), 0, (hipStream_t)stream, K, N,  \
                     (const T *)W, ldw, (u32x4 *)codes, (uint32_t *)exps)
  LB_BY_DTYPE(dtype, GO);
#undef GO
  LB_CHECK_LAUNCH(fn);
  return 0;
}

extern "C" int gpvae_load_w4(void *stream, int dtype, int64_t K, int64_t N, const void *codes, const void *exps, void *out,
                             int64_t ldo) {
  const char *fn = "gpvae_load_w4";
  if (const int rc = check_w4(fn, dtype, K, N, 3)) return rc;
  LB_REQUIRE(codes && aligned16(codes), 5, "%s: codes must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(exps && aligned16(exps), 6, "%s: exps must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(out, 7, "%s: out is NULL", fn);
  LB_REQUIRE(ldo >= N, 8, "%s: ldo < N", fn);
  const int64_t strips = w4_kb(K) * (w4_np(N) / 4);
  LB_REQUIRE(launchable(cdiv(strips, 256), 256), 3, "%s: matrix too large", fn);
  const dim3 grid((unsigned)cdiv(strips, 256));
#define GO(T)                                                                                                     \
  hipLaunchKernelGGL(load_w4_kernel<T>, grid, dim3(256), 0, (hipStream_t)stream, K, N, (const u32x4 *)codes,    \
                     (const uint32_t *)exps, (T *)out, ldo)
  LB_BY_DTYPE(dtype, GO);
#undef GO
  LB_CHECK_LAUNCH(fn);
  return 0;
}

// Few rows (skinny.hpp) or many (tile.hpp)?  Few: one launch (two where the reduction is split), every group of 64 / P rows
// decodes all codes, every workgroup stages the operand anew; many: the operand is split into planes first (a launch; none for
// most bfloat16 operands) and 64 rows share a decoded tile.  Measured on both sides, few / many in us (t: transposed):
//   bfloat16 16 x 4096 x 32768 21.2 / 26.2 (t 31.1 / 32.2), 32 x 4096 x 4096 13.0 / 13.0, 64 x 2048 x 4096 10.9 / 12.4 (t 11.3 / 14.4),
//     128 x 1024 x 4096 7.7 / 11.7 (t 13.9 / 14.3), 200 x 512 x 512 4.8 / 8.5, 24 x 4096 x 32768 25.9 / 28.4 (t 38.8 / 33.6),
//     64 x 4096 x 32768 49 / 35.6 (t 52 / 38.7);
//   float16 24 x 4096 x 32768 34 / 40 (t 40 / 44), 32 x 4096 x 8192 20.0 / 22.0 (t 21.1 / 23.7), 64 x 4096 x 32768 50 / 47 (t 81 / 51),
//     200 x 1024 x 4096 13.5 / 16.5 (t 19.8 / 21.5), 96 x 4096 x 32768 79 / 63 (t 148 / 80);
//   float32 21 x 4096 x 32768 35 / 47 (t 45 / 55), 42 x 1024 x 32768 18.4 / 22.0 (t 29 / 36), 42 x 4096 x 8192 25.9 / 24.4 (t 27.8 / 28.1),
//     42 x 4096 x 32768 49 / 51 (t 76 / 60), 42 x 8192 x 65536 152 / 160, 42 x 8192 x 32768 95 / 91, 42 x 8192 x 8192 44 / 32.5
//     (t 50 / 39), 64 x 4096 x 4096 21.6 / 21.8 (t 24.0 / 25.7), 256 x 1024 x 4096 23.2 / 22.0 (t 29.3 / 27.8),
//     128 x 4096 x 4096 32.7 / 25.8 (t 37.8 / 30.5).
// The rule takes the slower side of these for bfloat16 24 x 4096 x 32768 (by 10 %, so that its transposed product is not
// 15 % slower), float32 42 x 4096 x 8192 and 256 x 1024 x 4096 (by 6 %).
static inline bool use_skinny(int P, int64_t M, int64_t L, int64_t O, bool vjp) {
  const int64_t groups = cdiv(M, SK_MAXROWS / P);
  const double work = (double)P * (double)M * (double)L * (double)O;
  if (P == 1) return M <= 16 || (groups <= 4 && work <= 0x1p29);
  if (groups == 1) return P == 3 || M <= 24 || work <= 0x1p32;
  if (groups == 2) return work <= 0x1p32 || (P == 3 && !vjp && O >= 8 * L);
  return groups <= 16 && work <= 3 * 0x1p30;
}
static int64_t w4_workspace(int dtype, int64_t M, int64_t L, int64_t O, bool vjp) {
  const int64_t K = vjp ? O : L, N = vjp ? L : O;
  if (!dtype_ok(dtype) || M < 1 || M > MAX_MK || K < 1 || K > MAX_MK || N < 1 || N > MAX_N_W4) return 0;
  const int P = pieces(dtype);
  if (use_skinny(P, M, L, O, vjp)) {
    const SkinnyPlan p = skinny_plan(P, M, L, O);
    return p.splits > 1 ? p.splits * M * O * 4 : 0;
  }
  int64_t most = 0;  // the launches of a call follow one another and share it
  const int64_t slab = tile_rows(O);
  for (const int64_t m : {M < slab ? M : slab, M % slab}) {
    if (m == 0) continue;
    const TilePlan p = tile_plan(P, m, L, O, false);
    const int64_t bytes = p.plane_bytes + (p.splits > 1 ? p.splits * m * O * 4 : 0);
    if (bytes > most) most = bytes;
  }
  return most;
}
template <typename T, bool VJP>
static void run_w4(hipStream_t st, int64_t M, int64_t L, int64_t O, const void *X, int64_t ldx, const void *codes,
                   const void *exps, int64_t Np, int64_t kbs, void *work, const Epilogue<T, VJP> &ep) {
  constexpr int P = Split<T>::P;
  if (use_skinny(P, M, L, O, VJP)) {
    launch_skinny<T, VJP>(st, skinny_plan(P, M, L, O), M, L, O, (const T *)X, ldx, codes, exps, Np, kbs, (float *)work, ep);
  } else {
    // a bfloat16 operand is its own plane where its rows can be read 16 bytes at a time to the end of the last step and
    // 256 of them lie within a 32-bit offset
    const bool direct = P == 1 && L % 128 == 0 && ldx % 8 == 0 && ldx < (1 << 23) && aligned16(X);
    for (int64_t m = 0, slab = tile_rows(O); m < M; m += slab) {
      const int64_t rows = M - m < slab ? M - m : slab;
      launch_tile<T, VJP>(st, tile_plan(P, rows, L, O, direct), rows, L, O, (const T *)X + m * ldx, ldx, codes, exps, Np, kbs,
                          (unsigned char *)work, ep.from_row(m));
    }
  }
}
extern "C" int64_t gpvae_dense_w4_workspace_bytes(int dtype, int64_t M, int64_t K, int64_t N) {
  return w4_workspace(dtype, M, K, N, false);
}
extern "C" int64_t gpvae_dense_vjp_w4_workspace_bytes(int dtype, int64_t M, int64_t K, int64_t N) {
  return w4_workspace(dtype, M, N, K, true);
}

extern "C" int gpvae_dense_w4(void *stream, int dtype, int64_t M, int64_t K, int64_t N, const void *X, int64_t ldx,
                              const void *codes, const void *exps, const void *bias, int relu, void *Y, int64_t ldy,
                              void *work) {
  const char *fn = "gpvae_dense_w4";
  LB_REQUIRE(dtype_ok(dtype), 2, "%s: dtype must be float32, bfloat16 or float16 (got %d)", fn, dtype);
  LB_REQUIRE(M >= 0 && M <= MAX_MK, 3, "%s: M must lie in [0, 2^30] (got %lld)", fn, (long long)M);
  if (const int rc = check_w4(fn, dtype, K, N, 4)) return rc;
  if (M == 0) return 0;
  LB_REQUIRE(X, 6, "%s: X is NULL", fn);
  LB_REQUIRE(ldx >= K, 7, "%s: ldx < K", fn);
  LB_REQUIRE(codes && aligned16(codes), 8, "%s: codes must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(exps && aligned16(exps), 9, "%s: exps must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(Y && Y != X, 12, "%s: Y is NULL or X", fn);
  LB_REQUIRE(ldy >= N, 13, "%s: ldy < N", fn);
  LB_REQUIRE(!w4_workspace(dtype, M, K, N, false) || (work && aligned16(work)), 14, "%s: work must be a 16-byte aligned device pointer", fn);
#define GO(T)                                                                                                        \
  run_w4<T, false>((hipStream_t)stream, M, K, N, X, ldx, codes, exps, w4_np(N), w4_kb(K), work,                     \
                   Epilogue<T, false>{(const T *)bias, relu, nullptr, 0, (T *)Y, ldy})
  LB_BY_DTYPE(dtype, GO);
#undef GO
  LB_CHECK_LAUNCH(fn);
  return 0;
}

extern "C" int gpvae_dense_vjp_w4(void *stream, int dtype, int64_t M, int64_t K, int64_t N, const void *dY, int64_t lddy,
                                  const void *codes, const void *exps, const void *act_codes, void *dX, int64_t lddx,
                                  void *work) {
  const char *fn = "gpvae_dense_vjp_w4";
  LB_REQUIRE(dtype_ok(dtype), 2, "%s: dtype must be float32, bfloat16 or float16 (got %d)", fn, dtype);
  LB_REQUIRE(M >= 0 && M <= MAX_MK, 3, "%s: M must lie in [0, 2^30] (got %lld)", fn, (long long)M);
  if (const int rc = check_w4(fn, dtype, K, N, 4)) return rc;
  if (M == 0) return 0;
  LB_REQUIRE(dY, 6, "%s: dY is NULL", fn);
  LB_REQUIRE(lddy >= N, 7, "%s: lddy < N", fn);
  LB_REQUIRE(codes && aligned16(codes), 8, "%s: codes must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(exps && aligned16(exps), 9, "%s: exps must be a 16-byte aligned device pointer", fn);
  LB_REQUIRE(!act_codes || aligned16(act_codes), 10, "%s: act_codes must be 16-byte aligned", fn);
  LB_REQUIRE(dX && dX != dY, 11, "%s: dX is NULL or dY", fn);
  LB_REQUIRE(lddx >= K, 12, "%s: lddx < K", fn);
  LB_REQUIRE(!w4_workspace(dtype, M, N, K, true) || (work && aligned16(work)), 13, "%s: work must be a 16-byte aligned device pointer", fn);
#define GO(T)                                                                                                        \
  run_w4<T, true>((hipStream_t)stream, M, N, K, dY, lddy, codes, exps, w4_np(N), w4_kb(K), work,                    \
                  Epilogue<T, true>{nullptr, 0, (const uint8_t *)act_codes, q8_kp(K), (T *)dX, lddx})
  LB_BY_DTYPE(dtype, GO);
#undef GO
  LB_CHECK_LAUNCH(fn);
  return 0;
}
