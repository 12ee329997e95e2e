// lowbit.hpp — the two low-bit formats (include/gpvae_lowbit.h) and what their kernels share (gfx950 only).
//
// Everything here rests on one fact: a stored value is a small integer (q8: |q| <= 255) or an E2M1 magnitude (w4) times
// a power of two, hence EXACTLY a bfloat16 number.  A product of a floating matrix with a low-bit one therefore runs on
// the bf16 matrix pipe with the low-bit operand as ONE piece, and the floating operand as its exact sum of bf16
// pieces: three for float32 (8 + 8 + 8 significand bits), two for float16 (8 + 3), one for bfloat16.  Every piece
// product is exact in float32; only the accumulation rounds.
#pragma once
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#pragma GCC visibility push(default)  // the library is built with hidden visibility: it exports its C ABI only
#include "../../../include/gpvae_lowbit.h"
#pragma GCC visibility pop

namespace gpvae_lb {

void set_error(const char *fmt, ...);  // api.hip (thread-local buffer)

#define LB_REQUIRE(cond, argidx, ...)     \
  do {                                    \
    if (!(cond)) {                        \
      ::gpvae_lb::set_error(__VA_ARGS__); \
      return -(argidx);                   \
    }                                     \
  } while (0)

#define LB_CHECK_LAUNCH(name)                                                           \
  do {                                                                                  \
    hipError_t e__ = hipGetLastError();                                                 \
    if (e__ != hipSuccess) {                                                            \
      ::gpvae_lb::set_error("%s: launch failed: %s", name, hipGetErrorString(e__));     \
      return -1;                                                                        \
    }                                                                                   \
  } while (0)

static inline __host__ __device__ int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline __host__ __device__ int64_t round_up(int64_t a, int64_t b) { return cdiv(a, b) * b; }
// The largest sizes.  N: four rows of code words lie within a 32-bit offset; gradients: eight rows of float32.
constexpr int64_t MAX_MK = 1 << 30, MAX_N_W4 = 1 << 25, MAX_N_GRADS = 1 << 26;
// A dimension of a launch holds fewer than 2^32 threads: a larger one runs as its remainder, without an error.
static inline bool launchable(int64_t blocks, int threads) { return blocks < (int64_t(1) << 32) / threads; }
static inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static inline bool dtype_ok(int dt) { return dt == GPVAE_LB_F32 || dt == GPVAE_LB_BF16 || dt == GPVAE_LB_F16; }

// (the compiler keeps arrays of these in registers; of HIP's uint4 / uint2 structures it does not)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// ---- floating element types --------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }  // nearest, ties to even

// ---- tile exponents ------------------------------------------------------------------------------------------
// 2^e as a float, -126 <= e <= 127
__device__ __forceinline__ float pow2f(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
// The exponent byte of a tile whose largest magnitude is amax (inf or NaN: not finite).  LEAD: top lies in
// [2^LEAD, 2^(LEAD + 1)); LOWEST keeps 2^e (and half of it, for w4's 0.5) a normal float, HIGHEST keeps TOP 2^e finite
// (larger magnitudes saturate: unscale's clamp).
template <int TOP, int LEAD, int LOWEST> __device__ __forceinline__ int tile_exp_byte(float amax) {
  constexpr int HIGHEST = 127 - LEAD;
  if (!(amax <= 3.402823466e+38f)) return 255;
  if (amax == 0.0f) return 127;
  const int ex = (int)(__builtin_bit_cast(uint32_t, amax) >> 23);  // biased; 0: subnormal, below every LOWEST
  int e = ex - 127 - LEAD;
  e = e < LOWEST ? LOWEST : e;
  if (amax > (float)TOP * pow2f(e) && e < HIGHEST) ++e;
  return e + 127;
}
// the float 2^e of an exponent byte; 255 -> NaN (so is every product with it)
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 255u ? 0x7fc00000u : byte << 23);
}
// x * 2^-e for an exponent byte 1 .. 254 (2^-e itself may overflow: two exact factors), at most TOP in magnitude
template <int TOP> __device__ __forceinline__ float unscale(float x, int byte) {
  const int e = byte - 127, h = e >> 1;
  return fminf(fmaxf(x * pow2f(-h) * pow2f(h - e), (float)-TOP), (float)TOP);
}

// ---- w4 --------------------------------------------------------------------------------------------------------
// nearest E2M1 code (sign in bit 3) of v, |v| <= 6, ties to the even code: the edges whose upper code is even go up
__device__ __forceinline__ uint32_t e2m1_code(float v) {
  const float a = fabsf(v);
  const uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return c | (v < 0.0f ? 8u : 0u);
}
// two codes (byte SEL of w, low nibble first) times 2^e as bfloat16 pairs; scale = scale_of(byte), of which the
// instruction uses the exponent (exponent 255: NaN)
template <int SEL> __device__ __forceinline__ uint32_t w4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
__device__ __forceinline__ float bf_lo(uint32_t p) { return __builtin_bit_cast(float, p << 16); }
__device__ __forceinline__ float bf_hi(uint32_t p) { return __builtin_bit_cast(float, p & 0xffff0000u); }

static inline __host__ __device__ int64_t w4_np(int64_t N) { return round_up(N, 32); }
static inline __host__ __device__ int64_t w4_kb(int64_t K) { return cdiv(K, 32); }
static inline __host__ __device__ int64_t q8_kp(int64_t K) { return round_up(K, 32); }
static inline __host__ __device__ int64_t q8_mb(int64_t M) { return cdiv(M, 8); }

// dispatch on the floating type: FN(T)
#define LB_BY_DTYPE(dt, FN)                 \
  do {                                      \
    if ((dt) == GPVAE_LB_F32) FN(float);    \
    else if ((dt) == GPVAE_LB_BF16) FN(__bf16); \
    else FN(_Float16);                      \
  } while (0)

}  // namespace gpvae_lb
