// Shared device helpers and host-side error plumbing for libqattn (gfx950 only).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>
#include <string>

#include "qattn.h"

namespace qattn {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------------
// host: error reporting
// ------------------------------------------------------------------------------------------------
int set_error(int code, const char* fmt, ...);
int check_launch(const char* what);

#define QATTN_REQUIRE(cond, code, ...)        \
  do {                                        \
    if (!(cond)) return ::qattn::set_error((code), __VA_ARGS__); \
  } while (0)

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ------------------------------------------------------------------------------------------------
// device: half <-> float
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float bf16_to_f32(uint16_t h) { return __uint_as_float(((uint32_t)h) << 16); }

__device__ __forceinline__ float f16_to_f32(uint16_t h) {
  _Float16 x;
  __builtin_memcpy(&x, &h, 2);
  return (float)x;
}

template <bool IS_FP16>
__device__ __forceinline__ float half_to_f32(uint16_t h) {
  if constexpr (IS_FP16) return f16_to_f32(h);
  else return bf16_to_f32(h);
}

// round-to-nearest-even fp32 -> bf16 bits (NaN stays NaN)
__device__ __forceinline__ uint16_t f32_to_bf16(float f) {
  uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  u += 0x7fffu + ((u >> 16) & 1u);
  return (uint16_t)(u >> 16);
}

__device__ __forceinline__ uint16_t f32_to_f16(float f) {
  _Float16 x = (_Float16)f;  // v_cvt_f16_f32: round to nearest even
  uint16_t h;
  __builtin_memcpy(&h, &x, 2);
  return h;
}

template <bool IS_FP16>
__device__ __forceinline__ uint16_t f32_to_half(float f) {
  if constexpr (IS_FP16) return f32_to_f16(f);
  else return f32_to_bf16(f);
}

// ------------------------------------------------------------------------------------------------
// device: the quantizers' rounding (shared by the quantizer kernels and the attention kernels that
// quantize Q themselves)
// ------------------------------------------------------------------------------------------------
// v_cvt_i32_f32: truncate toward zero, saturate to the int32 range, NaN -> 0 (the hardware conversion; a C
// cast leaves NaN and out-of-range values undefined)
__device__ __forceinline__ int cvt_i32_trunc_sat(float t) {
  int r;
  asm("v_cvt_i32_f32 %0, %1" : "=v"(r) : "v"(t));
  return r;
}

// a / b, correctly rounded, from y1 = refined_rcp(b): the fma corrections of the IEEE division sequence
// without its range scaling (div_scale / div_fixup).  Exact wherever the residuals do not underflow: the
// quantizers divide |a| <= 127 b with b >= 1e-7, where only quotients below 2^-80 (which quantize to 0
// either way) can differ.
__device__ __forceinline__ float refined_rcp(float b) {
  const float y0 = __builtin_amdgcn_rcpf(b);
  return fmaf(fmaf(-b, y0, 1.0f), y0, y0);
}
__device__ __forceinline__ float div_by(float a, float b, float y1) {
  const float q0 = a * y1;
  const float q1 = fmaf(fmaf(-b, q0, a), y1, q0);
  return fmaf(fmaf(-b, q1, a), y1, q1);
}

// Scales of the per-block / per-warp (CUDA QuantInt8Kernel: amax / 127, codes RNE(x * 127 / amax)) and
// per-thread (Triton: amax / 127 + 1e-7, codes round-half-away(x / scale)) quantizers from the |x| maximum
__device__ __forceinline__ float quant_scale_cuda(float amax) { return amax / 127.0f; }
__device__ __forceinline__ float quant_recip_cuda(float amax) { return 127.0f / amax; }
__device__ __forceinline__ float quant_scale_triton(float amax) { return amax / 127.0f + 0.0000001f; }
__device__ __forceinline__ int quant_code_cuda(float x, float recip) { return cvt_i32_trunc_sat(__builtin_rintf(x * recip)); }
// HALF_X: x is a half-precision value.  With its 11 significant bits one correction of the quotient gives the correctly
// rounded one for every pair of mantissas and every rcp within an ulp, but for a power of two over 2 - 2^-23, whose
// neighbour has the same code (all 2^23 x 2^10 pairs were compared); half Q quantized inside the resident kernel spends
// half of that kernel's VALU work here.
template <bool HALF_X = false>
__device__ __forceinline__ int quant_code_triton(float x, float scale, float rcp_scale) {
  float t;
  if constexpr (HALF_X) {
    const float q0 = x * rcp_scale;
    t = fmaf(fmaf(-scale, q0, x), rcp_scale, q0);
  } else {
    t = div_by(x, scale, rcp_scale);
  }
  return cvt_i32_trunc_sat(t + __builtin_copysignf(0.5f, t));
}

// Rows [start, start + len) of sequence b of a packed variable-length batch: cu[b] .. cu[b + 1] clamped to
// the packed tensor's `total` rows and to `maxlen`, so that a malformed sequence table cannot address
// memory outside the packed tensors (every varlen kernel and the block-offset kernel use this).
__device__ __forceinline__ void varlen_range(const int32_t* cu, int64_t b, int64_t total, int64_t maxlen,
                                             int64_t& start, int64_t& len) {
  const int64_t s0 = min(max((int64_t)cu[b], (int64_t)0), total);
  const int64_t s1 = min(max((int64_t)cu[b + 1], s0), total);
  start = s0;
  len = min(s1 - s0, maxlen);
}

// Row quantization of the INT8 projections from the bits of max|x| (sign cleared): scale = max|x| / 127 and code =
// rint(127 x / max|x|), the quotient correctly rounded, so that the codes of half values are those of the real
// numbers.  A row of zeros has scale 0 and codes 0.  A row with an infinity or a NaN has scale NaN and codes 0: every
// product with it is NaN.  Rows of maximum below 1e-30 are scaled up first, where the quotient's corrections would
// underflow.
struct RowQuant {
  float scale, mult, top, rcp;
  bool fine;
  __device__ __forceinline__ explicit RowQuant(uint32_t top_bits) {
    const float t = __uint_as_float(top_bits);
    fine = top_bits != 0 && top_bits < 0x7f800000u;
    scale = top_bits < 0x7f800000u ? t / 127.0f : __uint_as_float(0x7fc00000u);
    const float pre = t < 1e-30f ? 0x1p80f : t > 1e30f ? 0x1p-40f : 1.0f;
    mult = 127.0f * pre;
    top = fine ? t * pre : 1.0f;
    rcp = refined_rcp(top);
  }
  // the code in the low byte.  127 x is exact for half values; its quotient takes one correction (as quant_code_triton's),
  // and adding 1.5 * 2^23 rounds it to an integer, ties to even, in the low bits
  __device__ __forceinline__ uint32_t code(float x) const {
    const float n = x * mult;
    const float q = n * rcp;
    return __float_as_uint(fmaf(fmaf(-top, q, n), rcp, q) + 12582912.0f);
  }
  // x times 127 / max|x| rounded to float32: for values that carry a float32 rounding of their own, which moves a code
  // across a border as often; where max|x| is not scaled up (127 / max|x| would not be finite)
  __device__ __forceinline__ bool nearable() const { return mult <= 127.0f; }
  __device__ __forceinline__ uint32_t near(float x) const { return __float_as_uint(fmaf(x, mult * rcp, 12582912.0f)); }
  // four codes, the first in the low byte
  __device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return fine ? lo | hi : 0u;
  }
  __device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) const {
    return pack4(code(a), code(b), code(c), code(d));
  }
  __device__ __forceinline__ uint32_t near4(float a, float b, float c, float d) const {
    return pack4(near(a), near(b), near(c), near(d));
  }
};

// wave64 reductions (DPP / permute through the compiler's shuffle lowering)
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The same over the DPP network, the result in a scalar register: within quads, rows of 16 (half mirror, mirror), then
// lane 15 of each row to the next one and lane 31 to the upper half; lane 63 ends with the whole wave's.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t old, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, ROWS, 0xf, false);
}
template <typename OP>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, uint32_t zero, OP op) {
  v = op(v, dpp<0xb1, 0xf>(zero, v));
  v = op(v, dpp<0x4e, 0xf>(zero, v));
  v = op(v, dpp<0x141, 0xf>(zero, v));
  v = op(v, dpp<0x140, 0xf>(zero, v));
  v = op(v, dpp<0x142, 0xa>(zero, v));
  v = op(v, dpp<0x143, 0xc>(zero, v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
  return wave_reduce(v, 0u, [](uint32_t a, uint32_t b) { return max(a, b); });
}

// of each half wave, in its last lane
__device__ __forceinline__ uint32_t half_wave_top(uint32_t v) {
  v = max(v, dpp<0xb1, 0xf>(0u, v));
  v = max(v, dpp<0x4e, 0xf>(0u, v));
  v = max(v, dpp<0x141, 0xf>(0u, v));
  v = max(v, dpp<0x140, 0xf>(0u, v));
  return max(v, dpp<0x142, 0xa>(0u, v));
}

}  // namespace qattn
