// frag.hpp — fragments for v_mfma_f32_16x16x32_bf16 from the low-bit formats, and the exact split of floating operands.
//
// The instruction: lane l supplies A[l % 16][8 (l / 16) + i] and B[8 (l / 16) + i][l % 16], i = 0..7, and holds
// D[4 (l / 16) + r][l % 16], r = 0..3.  Which reduction indices the four lane groups take is free as long as A and B agree.
#pragma once
#include "lowbit.hpp"

namespace gpvae_lb {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t mfma(u32x4 a, u32x4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Workgroups are dealt to the 8 XCDs round-robin; this renumbers them so that an XCD gets a contiguous run.
__device__ __forceinline__ int64_t xcd_chunk(int64_t id, int64_t n) {
  const int64_t x = id & 7, q = n >> 3, r = n & 7;
  return x * q + (x < r ? x : r) + (id >> 3);
}

// A buffer of `bytes` at a wave-uniform base: what lies past it reads as zero, without an access.
typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t buffer(const char *base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, bytes, 0x00027000);
}

// ---- w4 -----------------------------------------------------------------------------------------------------------------
// 8 codes -> 8 bfloat16 values; byte J of the tile-exponent word e is their exponent.  The conversion uses the scale's exponent
// bits alone (checked over all exponents with random sign and mantissa bits): the neighbouring bytes need no masking.
template <int J> __device__ __forceinline__ float w4_scale(uint32_t e) {
  return __builtin_bit_cast(float, J == 0 ? e << 23 : J == 1 ? e << 15 : J == 2 ? e << 7 : e >> 1);
}
__device__ __forceinline__ u32x4 w4_frag(uint32_t w, float scale) {
  return u32x4{w4_pair<0>(w, scale), w4_pair<1>(w, scale), w4_pair<2>(w, scale), w4_pair<3>(w, scale)};
}

// 8 x 8 transpose of nibbles inside groups of 8 lanes: the lane labelled a holds in[i] = T(i, a) and gets out[b] = T(a, b).
// Labels are dealt so that the three exchange partners (label bit 0, 1, 2 flipped) are one DPP move each:
// lane i, bits i2 i1 i0, carries label (i2, i1 ^ i2, i0 ^ i2), and i -> 7 - i flips label bit 2 alone.
__device__ __forceinline__ int tr8_label(int lane) {
  const int i2 = (lane >> 2) & 1;
  return (i2 << 2) | ((((lane >> 1) & 1) ^ i2) << 1) | ((lane & 1) ^ i2);
}
struct Tr8 {
  uint32_t sel4, sel2, rot, own;
  __device__ __forceinline__ void init(int lane) {
    const int b = tr8_label(lane);
    sel4 = (b & 4) ? 0x03020706u : 0x05040100u;
    sel2 = (b & 2) ? 0x03070105u : 0x06020400u;
    rot = (b & 1) ? 4u : 28u;
    own = (b & 1) ? 0xf0f0f0f0u : 0x0f0f0f0fu;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
    uint32_t p = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true);  // row_half_mirror
    x = __builtin_amdgcn_perm(p, x, sel4);
    p = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true);            // quad_perm [2,3,0,1]
    x = __builtin_amdgcn_perm(p, x, sel2);
    p = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true);            // quad_perm [1,0,3,2]
    p = __builtin_amdgcn_alignbit(p, p, rot);
    return p ^ (own & (x ^ p));  // own ? x : p, bit by bit
  }
};

// ---- the floating operand as its exact sum of bfloat16 pieces -----------------------------------------------------------
// Truncation, not rounding: the top 16 bits of a finite float are a finite bfloat16 whatever its size, the remainder is
// exact, and float32's 24 bits are 8 + 8 + 8.  An infinity or a NaN goes into piece 0: the remainder is taken of
// the value clamped to the finite range, so that inf * w stays inf (inf - inf would make it NaN).  A float32 NaN is made a
// quiet one first: a signalling one may have its mantissa bits in the lower half only, and its upper half is an infinity.
// That instruction a value costs dense_grads_q8 4096 x 1024 x 4096 103.8 -> 107.4 us, dense_vjp_w4 42 x 1024 x 32768 27.8 -> 28.6 us,
// and nothing measurable where rows are split once or are few.  (float16: the conversion to float32 quiets.)
template <typename T> struct Split;
__device__ __forceinline__ uint32_t pack_hi(float a, float b) {  // top halves of a (low) and b (high)
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}
__device__ __forceinline__ float trunc_bf(float a) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, a) & 0xffff0000u);
}
__device__ __forceinline__ float finite(float a) {
  return __builtin_amdgcn_fmed3f(a, -3.402823466e+38f, 3.402823466e+38f);
}
template <> struct Split<float> {
  static constexpr int P = 3;
  // two values -> one dword of each piece
  __device__ static __forceinline__ void two(float a, float b, uint32_t *out) {
    a = __builtin_canonicalizef(a), b = __builtin_canonicalizef(b);
    out[0] = pack_hi(a, b);
    a = finite(a), b = finite(b);
    a -= trunc_bf(a), b -= trunc_bf(b);
    out[1] = pack_hi(a, b);
    a -= trunc_bf(a), b -= trunc_bf(b);
    out[2] = pack_hi(a, b);
  }
};
template <> struct Split<_Float16> {
  static constexpr int P = 2;
  __device__ static __forceinline__ void two(_Float16 ha, _Float16 hb, uint32_t *out) {
    float a = (float)ha, b = (float)hb;
    out[0] = pack_hi(a, b);
    a = finite(a), b = finite(b);
    out[1] = pack_hi(a - trunc_bf(a), b - trunc_bf(b));
  }
};
template <> struct Split<__bf16> {
  static constexpr int P = 1;
  __device__ static __forceinline__ void two(__bf16 a, __bf16 b, uint32_t *out) {
    out[0] = (uint32_t)__builtin_bit_cast(uint16_t, a) | ((uint32_t)__builtin_bit_cast(uint16_t, b) << 16);
  }
};
// pieces of an operand of this type
static inline int pieces(int dtype) { return dtype == GPVAE_LB_F32 ? 3 : dtype == GPVAE_LB_F16 ? 2 : 1; }

// four elements at any element-aligned address: one vector load (unaligned access is on)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Vec4 { T v[4]; };

// v[0..3] = row[k .. k + 3], zero from L on (k may lie past L)
template <typename T> __device__ __forceinline__ Vec4<T> load4(const T *row, int64_t k, int64_t L) {
  Vec4<T> v;
  if (k + 4 <= L) {
    v = *reinterpret_cast<const Vec4<T> *>(row + k);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v.v[i] = k + i < L ? row[k + i] : T(0.0f);
  }
  return v;
}

// The end of a dense layer's output element: bias and ReLU (NaN stays), or the checkpoint's mask; rounded once.  What an
// element needs from memory is loaded by the caller ahead of a batch of stores: a load behind a store waits for it.
template <typename T, bool VJP> struct Epilogue {
  const T *bias;
  int relu;
  const uint8_t *act;
  int64_t act_kp;
  T *out;
  int64_t ldo;
  Epilogue from_row(int64_t m) const {  // m a multiple of 8
    return Epilogue{bias, relu, act ? act + m * act_kp : nullptr, act_kp, out + m * ldo, ldo};
  }
  __device__ __forceinline__ float bias_at(int64_t o) const { return !VJP && bias ? to_f32(bias[o]) : 0.0f; }
  // mask byte of one element; the four bytes of rows m .. m + 3, m a multiple of 4
  __device__ __forceinline__ uint32_t mask_at(int64_t m, int64_t o) const {
    return VJP && act ? act[((m >> 3) * act_kp + o) * 8 + (m & 7)] : 1u;
  }
  __device__ __forceinline__ uint32_t mask4_at(int64_t m, int64_t o) const {
    return VJP && act ? *reinterpret_cast<const uint32_t *>(act + ((m >> 3) * act_kp + o) * 8 + (m & 7)) : 0x01010101u;
  }
  __device__ __forceinline__ void store(int64_t m, int64_t o, float v, float b, uint32_t mask) const {
    if (VJP) {
      if (!mask) v = 0.0f;
    } else {
      if (bias) v += b;
      if (relu) v = v < 0.0f ? 0.0f : v;
    }
    out[m * ldo + o] = from_f32<T>(v);
  }
};

// p[0] + p[stride] + ... (n terms) in order, eight loads in flight at a time
__device__ __forceinline__ float sum_parts(const float *p, int64_t stride, int n) {
  float v = 0.0f;
  for (int s = 0; s < n; s += 8) {
    float t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = p[(s + u < n ? s + u : n - 1) * stride];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (s + u < n) v += t[u];
  }
  return v;
}

// the sum of the partial outputs [splits][M][O] in order, and the epilogue
template <typename T, bool VJP>
__global__ __launch_bounds__(256) void split_sum_kernel(int64_t M, int64_t O, int splits, const float *__restrict__ part,
                                                        Epilogue<T, VJP> ep) {
  const int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (o >= O) return;
  const float b = ep.bias_at(o);
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
    const uint32_t mask = ep.mask_at(m, o);
    ep.store(m, o, sum_parts(part + m * O + o, M * O, splits), b, mask);
  }
}
template <typename T, bool VJP>
static void launch_split_sum(hipStream_t st, int64_t M, int64_t O, int splits, const float *part, const Epilogue<T, VJP> &ep) {
  hipLaunchKernelGGL((split_sum_kernel<T, VJP>), dim3((unsigned)cdiv(O, 256), (unsigned)(M < 4096 ? M : 4096)), dim3(256), 0, st,
                     M, O, splits, part, ep);
}

}  // namespace gpvae_lb
