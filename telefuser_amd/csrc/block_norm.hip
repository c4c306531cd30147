// The row operators around a DiT block: the norm before it (LayerNorm or RMSNorm, weight, bias, adaLN scale and shift),
// the gated residual after it (optionally of the normalized output), both in one pass, and the row quantizer.
//
//   v    = x                                             or  residual_scale * x + gate * p(y),  p(y) = y or its norm
//   h    = v                                             (stored where wanted)
//   z    = n(v) * weight + bias, then z * (1 + scale) + shift
//   n(v) = v | (v - mean) / sqrt(var + eps) | v / sqrt(mean(v^2) + eps)
//   z is stored in bf16 / fp16 / fp32, or as INT8: code = rint(127 z / max|z|), row scale max|z| / 127
//
// Everything between the loads and the stores is fp32; v reaches the norm unrounded.  LayerNorm's mean is removed twice, the
// second time as what is left of it in the centred values, and the variance is that of the result.  Parameters are read with
// the strides of their broadcast shape.  A float32 y (a product that is not to be rounded before the sum) takes twice the
// bytes of a half one: gated residual + norm of 32760 x 1536 74 us, with a float32 y 95 (5.3 TB/s).
//
// Bound by memory: x (and y) read once, h and z written once.  At the rate of a copy (5.1 TB/s for 1 GiB) or above where
// the caches help (medians, inputs in turn): gated residual + norm of 75600 x 5120 bf16 0.58 ms (5.3 TB/s), modulated norm of
// it 304 us (5.1), of 32760 x 1536 36 us (from memory 42), row quantizer of 75600 x 5120 210 us (5.5).  What it took: every
// value loaded once and held in registers (8.4 ms with the row read again for each reduction); reductions over DPP instead of
// LDS; 16-byte accesses at any alignment (20000 x 5119, one element a load: 405 us, now 131); several narrow rows a wave
// (75600 x 64: 25 us, now 7.6); parameters in LDS for many rows; and few VALU instructions a value, which INT8 output has
// most of: masks only in groups that the row's end cuts, one fused multiply-add for a code of a normalized value (20000 x
// 5120 to INT8: 110 us, then 85, and 92 with the second part of the mean).
#include "attn_device.h"

namespace qattn {

// a parameter with the broadcast strides of its leading dimensions; the channels are contiguous
struct Param {
  const void* p;
  int dtype;
  int64_t sb, sl;
};

struct BlockNormParams {
  const void* x;
  int64_t xb, xl;
  const void* y;
  int64_t yb, yl;
  void* h;  // [B, L, C] in x's type, or null
  void* z;  // [B, L, C], INT8 [B * L, z_pitch], or null
  float* z_scale;
  int64_t z_pitch;
  int x_dtype, y_dtype, z_dtype;
  Param gate, weight, bias, scale, shift, post_weight, post_bias;
  int64_t L, rows;
  int C, norm, post_norm;
  float eps, post_eps, residual_scale;
  int staged[5], stage_half;  // offsets in LDS of the staged parameters (floats), or -1; floats of a half
};

__device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
  if (dtype == QATTN_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return dtype == QATTN_FP16 ? f16_to_f32(v) : bf16_to_f32(v);
}
__device__ __forceinline__ void store_elem(void* p, int dtype, int64_t i, float v) {
  if (dtype == QATTN_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = dtype == QATTN_FP16 ? f32_to_f16(v) : f32_to_bf16(v);
}
__device__ __forceinline__ float load_param(const Param& q, int64_t b, int64_t l, int c) {
  return load_elem(q.p, q.dtype, b * q.sb + l * q.sl + c);
}

// ------------------------------------------------------------------------------------------------
// rows held in registers
// ------------------------------------------------------------------------------------------------
// A thread holds NV groups of 8 consecutive channels of a row: every value is loaded once, the reductions run over
// registers, and the outputs are written from them.  A group is one 16-byte access (two for fp32) at whatever alignment
// its row has; only a group that the row's end cuts goes element by element.
enum YMode { Y_NONE, Y_SAME, Y_BF16, Y_FP16, Y_F32 };

typedef v4u v4u_any __attribute__((aligned(2)));  // rows of halves start anywhere
typedef v4u v4u_word __attribute__((aligned(4)));

template <int DT>
struct RawGroup {
  static constexpr int kWords = DT == QATTN_F32 ? 8 : 4;
  uint32_t w[kWords];
  // channels c .. c + 7 of the row at `at` of `C` channels, zeros past its end; whole: known to lie within
  __device__ __forceinline__ void load(const void* p, int64_t at, int c, int C, bool whole) {
    if (whole || c + 8 <= C) {
      if constexpr (DT == QATTN_F32) {
        const v4u_word* q = reinterpret_cast<const v4u_word*>(static_cast<const float*>(p) + at + c);
        const v4u a = q[0], b = q[1];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = a[e], w[4 + e] = b[e];
      } else {
        const v4u a = *reinterpret_cast<const v4u_any*>(static_cast<const uint16_t*>(p) + at + c);
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = a[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < kWords; e++) w[e] = 0;
#pragma unroll
      for (int e = 0; e < 7; e++)
        if (c + e < C) {
          if constexpr (DT == QATTN_F32) w[e] = static_cast<const uint32_t*>(p)[at + c + e];
          else w[e / 2] |= (uint32_t)static_cast<const uint16_t*>(p)[at + c + e] << (16 * (e & 1));
        }
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (DT == QATTN_F32) return __uint_as_float(w[e]);
    else return half_to_f32<DT == QATTN_FP16>((uint16_t)(w[e / 2] >> (16 * (e & 1))));
  }
};

__device__ __forceinline__ void load_param8(const Param& q, int64_t at, int c, int C, bool whole, float (&out)[8]) {
  if (q.dtype == QATTN_F32) {
    RawGroup<QATTN_F32> g;
    g.load(q.p, at, c, C, whole);
#pragma unroll
    for (int e = 0; e < 8; e++) out[e] = g.get(e);
  } else {
    RawGroup<QATTN_BF16> g;
    g.load(q.p, at, c, C, whole);
    if (q.dtype == QATTN_BF16) {
#pragma unroll
      for (int e = 0; e < 8; e++) out[e] = g.get(e);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) out[e] = f16_to_f32((uint16_t)(g.w[e / 2] >> (16 * (e & 1))));
    }
  }
}

__device__ __forceinline__ void store8(void* p, int dtype, int64_t at, int c, int C, bool whole, const float (&v)[8]) {
  if (whole || c + 8 <= C) {
    if (dtype == QATTN_F32) {
      v4u_word* q = reinterpret_cast<v4u_word*>(static_cast<float*>(p) + at + c);
      q[0] = v4u{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      q[1] = v4u{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
    } else {
      v4u o;
      if (dtype == QATTN_FP16) {
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = pack_half2<true>(v[2 * e], v[2 * e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = pack_half2<false>(v[2 * e], v[2 * e + 1]);
      }
      *reinterpret_cast<v4u_any*>(static_cast<uint16_t*>(p) + at + c) = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 7; e++)
      if (c + e < C) store_elem(p, dtype, at + c + e, v[e]);
  }
}

// Reductions over the lanes of a row: LANES of a wave, or whole waves (each call then has its own LDS slots, so one
// barrier separates write and read).
constexpr int kMaxRowWaves = 8;
constexpr int kRowSlots = 7;  // two LayerNorms of three sums, and the maximum
template <int LANES>
struct RowReduce {
  uint32_t (*slots)[kMaxRowWaves];
  int waves, wave;
  int used = 0;
  template <typename OP>
  __device__ __forceinline__ uint32_t reduce(uint32_t v, OP op) {
    if constexpr (LANES < 64) {
      v = op(v, dpp<0xb1, 0xf>(0u, v));
      v = op(v, dpp<0x4e, 0xf>(0u, v));
      v = op(v, dpp<0x141, 0xf>(0u, v));
      if constexpr (LANES > 8) v = op(v, dpp<0x140, 0xf>(0u, v));
      if constexpr (LANES > 16) v = op(v, (uint32_t)__shfl_xor((int)v, 16, 64));
      return v;
    } else {
      uint32_t t = wave_reduce(v, 0u, op);
      if (waves == 1) return t;
      uint32_t* s = slots[used++];
      if ((threadIdx.x & 63) == 0) s[wave] = t;
      __syncthreads();
      t = s[0];
      for (int i = 1; i < waves; i++) t = op(t, s[i]);
      return t;
    }
  }
  static __device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }
  __device__ __forceinline__ float sum(float v) { return __uint_as_float(reduce(__float_as_uint(v), plus)); }
  // both at one barrier
  __device__ __forceinline__ void sums(float& v, float& w) {
    if (LANES < 64 || waves == 1) {
      v = sum(v), w = sum(w);
      return;
    }
    const uint32_t a = wave_reduce(__float_as_uint(v), 0u, plus), b = wave_reduce(__float_as_uint(w), 0u, plus);
    uint32_t *s = slots[used], *t = slots[used + 1];
    used += 2;
    if ((threadIdx.x & 63) == 0) s[wave] = a, t[wave] = b;
    __syncthreads();
    v = __uint_as_float(s[0]), w = __uint_as_float(t[0]);
    for (int i = 1; i < waves; i++) v += __uint_as_float(s[i]), w += __uint_as_float(t[i]);
  }
  __device__ __forceinline__ uint32_t top(uint32_t v) {
    return reduce(v, [](uint32_t a, uint32_t b) { return max(a, b); });
  }
};

// Where a row's parameters come from: memory, with the strides of their broadcast shape, ...
struct DirectParams {
  const BlockNormParams& p;
  int64_t b, l;
  __device__ __forceinline__ void load(const Param& q, int c, bool whole, float (&t)[8]) const {
    load_param8(q, b * q.sb + l * q.sl, c, p.C, whole, t);
  }
  __device__ __forceinline__ bool post(int c, bool whole, float (&mul)[8], float (&add)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; e++) mul[e] = 1.0f, add[e] = 0.0f;
    if (p.post_weight.p) load(p.post_weight, c, whole, mul);
    if (p.post_bias.p) load(p.post_bias, c, whole, add);
    return p.post_weight.p || p.post_bias.p;
  }
  __device__ __forceinline__ bool gate(int c, bool whole, float (&t)[8]) const {
    if (p.gate.p) load(p.gate, c, whole, t);
    return p.gate.p;
  }
  // weight, bias, scale and shift as one multiplication and one addition
  __device__ __forceinline__ bool affine(int c, bool whole, float (&mul)[8], float (&add)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; e++) mul[e] = 1.0f, add[e] = 0.0f;
    if (p.weight.p) load(p.weight, c, whole, mul);
    if (p.bias.p) load(p.bias, c, whole, add);
    if (p.scale.p) {
      float t[8];
      load(p.scale, c, whole, t);
#pragma unroll
      for (int e = 0; e < 8; e++) mul[e] = fmaf(mul[e], t[e], mul[e]), add[e] = fmaf(add[e], t[e], add[e]);
    }
    if (p.shift.p) {
      float t[8];
      load(p.shift, c, whole, t);
#pragma unroll
      for (int e = 0; e < 8; e++) add[e] += t[e];
    }
    return p.weight.p || p.bias.p || p.scale.p || p.shift.p;
  }
};

// ... or LDS, where the workgroup has put them once for all of its rows: those that there are of [post mul, post add, gate,
// mul, add], each as the first halves of all 8-channel groups and then the second ones, so that a wave reads 16 bytes a
// lane side by side.
struct StagedParams {
  const BlockNormParams& p;
  const float* lds;
  __device__ __forceinline__ void load(int which, int c, float (&t)[8]) const {
    // (a thread past the row's end takes the last group's, and drops what it makes of them)
    const float* q = lds + p.staged[which] + min(c / 2, p.stage_half - 4);
    const v4f a = *reinterpret_cast<const v4f*>(q), b = *reinterpret_cast<const v4f*>(q + p.stage_half);
#pragma unroll
    for (int e = 0; e < 4; e++) t[e] = a[e], t[4 + e] = b[e];
  }
  __device__ __forceinline__ bool post(int c, bool, float (&mul)[8], float (&add)[8]) const {
    if (p.staged[0] < 0) return false;
    load(0, c, mul), load(1, c, add);
    return true;
  }
  __device__ __forceinline__ bool gate(int c, bool, float (&t)[8]) const {
    if (p.staged[2] < 0) return false;
    load(2, c, t);
    return true;
  }
  __device__ __forceinline__ bool affine(int c, bool, float (&mul)[8], float (&add)[8]) const {
    if (p.staged[3] < 0) return false;
    load(3, c, mul), load(4, c, add);
    return true;
  }
};

// 1 / sqrt(var + eps) from the mean square of values whose mean is `rest`; an infinite one stays
__device__ __forceinline__ float inv_deviation(float square, float rest, float eps) {
  const float var = square < __builtin_inff() ? fmaxf(fmaf(-rest, rest, square), 0.0f) : square;
  return 1.0f / sqrtf(var + eps);
}

// A thread's part of a row as loaded; `first` is its first channel, `step` the distance between its groups.  A group i of
// which no thread's lies past the row's end (a condition on scalars) takes no masks.
template <int XD, int YM, int NV>
struct RowValues {
  static constexpr int YD = YM == Y_BF16 ? QATTN_BF16 : YM == Y_FP16 ? QATTN_FP16 : YM == Y_F32 ? QATTN_F32 : XD;
  RawGroup<XD> x[NV];
  RawGroup<YD> y[YM == Y_NONE ? 1 : NV];
  __device__ __forceinline__ void load(const BlockNormParams& p, int64_t b, int64_t l, int first, int step) {
    const int64_t xo = b * p.xb + l * p.xl, yo = b * p.yb + l * p.yl;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const bool whole = (i + 1) * step <= p.C;
      x[i].load(p.x, xo, first + i * step, p.C, whole);
      if constexpr (YM != Y_NONE) y[i].load(p.y, yo, first + i * step, p.C, whole);
    }
  }
};

// One row.  r: its values, loaded; next() is called once they are used and may load others into r.
template <int XD, int YM, int NV, typename REDUCE, typename PARAMS, typename NEXT>
__device__ __forceinline__ void norm_row(const BlockNormParams& p, int64_t b, int64_t l, int first, int step, REDUCE red,
                                         const PARAMS& params, const RowValues<XD, YM, NV>& r, NEXT next) {
  const int C = p.C;
  const int64_t row = b * p.L + l;
  const float inv_c = 1.0f / (float)C;
  auto whole = [&](int i) __attribute__((always_inline)) { return (i + 1) * step <= C; };
  float v[NV][8];
  // v - mean (or v) in place and 1 / sqrt(var + eps); values past the row's end are zeros before, and anything after.  The
  // mean of a float32 sum is off by a few roundings of its own size, which a row of small variance beside its mean would
  // show (or a constant one, whose result is 0): what is left of it in the centred values, and of their variance, goes too.
  auto normalize = [&](int kind, float eps) __attribute__((always_inline)) {
    float s = 0.0f;
    if (kind == QATTN_NORM_LAYER) {
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) s += v[i][e];
      const float mean = red.sum(s) / (float)C;
      float rest = 0.0f, var = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; i++) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] -= mean;
        if (!whole(i)) {
          const int left = C - first - i * step;
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (e >= left) v[i][e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) rest += v[i][e], var = fmaf(v[i][e], v[i][e], var);
      }
      red.sums(rest, var);
      rest /= (float)C;
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] -= rest;
      return inv_deviation(var * inv_c, rest, eps);
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) s = fmaf(v[i][e], v[i][e], s);
    return 1.0f / sqrtf(red.sum(s) * inv_c + eps);
  };
  if constexpr (YM != Y_NONE) {
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = r.y[i].get(e);
    if (p.post_norm) {
      const float rstd = normalize(p.post_norm, p.post_eps);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        float mul[8], add[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] *= rstd;
        if (params.post(first + i * step, whole(i), mul, add))
#pragma unroll
          for (int e = 0; e < 8; e++) v[i][e] = fmaf(v[i][e], mul[e], add[e]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float t[8];
      if (params.gate(first + i * step, whole(i), t))
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] *= t[e];
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = fmaf(p.residual_scale, r.x[i].get(e), v[i][e]);
      if (!whole(i)) {  // past the row's end stay zeros, whatever the parameters made of them: the next norm sums them
        const int left = C - first - i * step;
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (e >= left) v[i][e] = 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = r.x[i].get(e);
  }
  next();
  if (p.h)
#pragma unroll
    for (int i = 0; i < NV; i++) store8(p.h, XD, row * C, first + i * step, C, whole(i), v[i]);
  if (!p.z) return;

  if (p.norm) {
    const float rstd = normalize(p.norm, p.eps);
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] *= rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; i++) {
    float mul[8], add[8];
    if (params.affine(first + i * step, whole(i), mul, add))
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = fmaf(v[i][e], mul[e], add[e]);
  }
  if (p.z_dtype != QATTN_I8) {
#pragma unroll
    for (int i = 0; i < NV; i++) store8(p.z, p.z_dtype, row * C, first + i * step, C, whole(i), v[i]);
    return;
  }
  // max|z| as an integer: the bits of |z| are ordered as the values, infinity and NaN above them all
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    if (!whole(i)) {
      const int left = C - first - i * step;
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e >= left) v[i][e] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      top = max(top, max(__float_as_uint(v[i][e]) & 0x7fffffffu, __float_as_uint(v[i][e + 1]) & 0x7fffffffu));
  }
  const RowQuant rq(red.top(top));
  int8_t* codes = static_cast<int8_t*>(p.z) + row * p.z_pitch;
  // up to the pitch, which divides by 8: the codes past the row's end are those of zeros
  auto put = [&](auto code4) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = first + i * step;
      if (whole(i) || c < p.z_pitch)
        *reinterpret_cast<v2u*>(codes + c) = v2u{code4(v[i][0], v[i][1], v[i][2], v[i][3]),
                                                 code4(v[i][4], v[i][5], v[i][6], v[i][7])};
    }
  };
  if (p.norm && rq.nearable()) put([&](float a, float b, float c, float d) { return rq.near4(a, b, c, d); });
  else put([&](float a, float b, float c, float d) { return rq.code4(a, b, c, d); });
  for (int64_t c = first + NV * step; c < p.z_pitch; c += step) *reinterpret_cast<v2u*>(codes + c) = v2u{0u, 0u};
  if (first == 0) p.z_scale[row] = rq.scale;
}

// Narrow rows: LANES lanes a row, several rows a wave.
template <int XD, int YM, int LANES>
__global__ __launch_bounds__(256) void narrow_row_kernel(BlockNormParams p) {
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  // a row past the last is the last one again: its lanes take part in the reductions and write what its own lanes write
  const int64_t at = min(row, p.rows - 1), b = at / p.L, l = at - b * p.L;
  const int first = threadIdx.x % LANES * 8;
  RowValues<XD, YM, 1> r;
  r.load(p, b, l, first, LANES * 8);
  norm_row<XD, YM, 1>(p, b, l, first, LANES * 8, RowReduce<LANES>{nullptr, 1, 0}, DirectParams{p, b, l}, r, [] {});
}

// A workgroup a row.
template <int XD, int YM, int NV>
__global__ __launch_bounds__(kMaxRowWaves * 64) void row_norm_kernel(BlockNormParams p) {
  __shared__ uint32_t slots[kRowSlots][kMaxRowWaves];
  const int64_t b = blockIdx.x / p.L, l = blockIdx.x - b * p.L;
  const int first = threadIdx.x * 8, step = blockDim.x * 8;
  RowValues<XD, YM, NV> r;
  r.load(p, b, l, first, step);
  norm_row<XD, YM, NV>(p, b, l, first, step, RowReduce<64>{slots, (int)blockDim.x >> 6, (int)threadIdx.x >> 6},
                       DirectParams{p, b, l}, r, [] {});
}

// Many rows with the same parameters: a workgroup folds them and puts them into LDS once, then its eight waves take rows of
// one batch entry in turn, `waves` of them a row, and load the next row while they work on this one.  Read from memory for
// every row they are 4 bytes a value and parameter beside the 2 of x, and L2 does not keep up with that.
template <int XD, int YM, int NV>
__global__ __launch_bounds__(512) void staged_row_kernel(BlockNormParams p, int waves, int turns) {
  extern __shared__ __attribute__((aligned(16))) float staged[];
  __shared__ uint32_t slots[8][2][kRowSlots][kMaxRowWaves];
  const int64_t b = blockIdx.y;
  const DirectParams from{p, b, 0};
  for (int c = threadIdx.x * 8; c < p.stage_half * 2; c += 512 * 8) {
    float mul[8], add[8];
    auto put = [&](int which, const float (&t)[8]) {
      float* q = staged + p.staged[which] + c / 2;
      *reinterpret_cast<v4f*>(q) = v4f{t[0], t[1], t[2], t[3]};
      *reinterpret_cast<v4f*>(q + p.stage_half) = v4f{t[4], t[5], t[6], t[7]};
    };
    if (p.staged[0] >= 0) from.post(c, false, mul, add), put(0, mul), put(1, add);
    if (p.staged[2] >= 0) from.gate(c, false, mul), put(2, mul);
    if (p.staged[3] >= 0) from.affine(c, false, mul, add), put(3, mul), put(4, add);
  }
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), per = 8 / waves, group = wave / waves;
  const int first = (threadIdx.x - group * waves * 64) * 8, step = waves * 512;
  // all groups take all turns, for the barriers between a row's waves; past the last row it is the last one again, and gets
  // the same values
  auto row = [&](int t) { return min(((int64_t)t * gridDim.x + blockIdx.x) * per + group, p.L - 1); };
  RowValues<XD, YM, NV> r;
  r.load(p, b, row(0), first, step);
  for (int t = 0; t < turns; t++) {
    // slots alternate: only one barrier may lie between the last read of a row and the next one's write
    norm_row<XD, YM, NV>(p, b, row(t), first, step, RowReduce<64>{slots[group][t & 1], waves, wave - group * waves},
                         StagedParams{p, staged}, r, [&] {
                           if (t + 1 < turns) r.load(p, b, row(t + 1), first, step);
                         });
  }
}

// ------------------------------------------------------------------------------------------------
// rows too wide for that: one wave per row, one element per lane and step, the row read again for each reduction, and codes
// from the corrected quotient for normalized values too.  The simple kernel that the others replaced, kept for widths that
// the framework's models do not have: latency of a row's steps bounds it (quantizer of 1 x 28672 228 us, of 500 x 28672 399).
// ------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void wide_row_kernel(BlockNormParams p) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const int lane = threadIdx.x & 63;
  const int64_t b = row / p.L, l = row - b * p.L;
  const float inv_c = 1.0f / (float)p.C;
  const int64_t xo = b * p.xb + l * p.xl, yo = b * p.yb + l * p.yl;

  // mean, what is left of it in the centred values, and 1 / sqrt(var + eps), of get(c); as in norm_row
  auto statistics = [&](int kind, float eps, auto get, float& mean, float& rest, float& rstd) {
    float s = 0.0f;
    if (kind == QATTN_NORM_LAYER) {
      for (int c = lane; c < p.C; c += 64) s += get(c);
      mean = wave_sum(s) / (float)p.C;
      s = 0.0f;
    }
    float var = 0.0f;
    for (int c = lane; c < p.C; c += 64) {
      const float d = get(c) - mean;
      s += d, var = fmaf(d, d, var);
    }
    if (kind == QATTN_NORM_LAYER) rest = wave_sum(s) / (float)p.C;
    rstd = inv_deviation(wave_sum(var) * inv_c, rest, eps);
  };
  float y_mean = 0.0f, y_rest = 0.0f, y_rstd = 1.0f;
  if (p.y && p.post_norm)
    statistics(p.post_norm, p.post_eps, [&](int c) { return load_elem(p.y, p.y_dtype, yo + c); }, y_mean, y_rest, y_rstd);
  auto value = [&](int c) {
    float v = load_elem(p.x, p.x_dtype, xo + c);
    if (p.y) {
      float t = load_elem(p.y, p.y_dtype, yo + c);
      if (p.post_norm) {
        t = (t - y_mean - y_rest) * y_rstd;
        if (p.post_weight.p) t *= load_param(p.post_weight, b, l, c);
        if (p.post_bias.p) t += load_param(p.post_bias, b, l, c);
      }
      if (p.gate.p) t *= load_param(p.gate, b, l, c);
      v = fmaf(p.residual_scale, v, t);
    }
    return v;
  };
  if (p.h)
    for (int c = lane; c < p.C; c += 64) store_elem(p.h, p.x_dtype, row * p.C + c, value(c));
  if (!p.z) return;

  float mean = 0.0f, rest = 0.0f, rstd = 1.0f;
  if (p.norm) statistics(p.norm, p.eps, value, mean, rest, rstd);
  auto out = [&](int c) {
    float z = (value(c) - mean - rest) * rstd;
    if (p.weight.p) z *= load_param(p.weight, b, l, c);
    if (p.bias.p) z += load_param(p.bias, b, l, c);
    if (p.scale.p) z = fmaf(z, load_param(p.scale, b, l, c), z);
    if (p.shift.p) z += load_param(p.shift, b, l, c);
    return z;
  };
  if (p.z_dtype != QATTN_I8) {
    for (int c = lane; c < p.C; c += 64) store_elem(p.z, p.z_dtype, row * p.C + c, out(c));
    return;
  }
  // max|z| as an integer: the bits of |z| are ordered as the values, infinity and NaN above them all
  uint32_t top = 0;
  for (int c = lane; c < p.C; c += 64) top = max(top, __float_as_uint(out(c)) & 0x7fffffffu);
  top = wave_top(top);
  const RowQuant rq(top);
  int8_t* codes = static_cast<int8_t*>(p.z) + row * p.z_pitch;
  for (int c = lane; c < p.C; c += 64) codes[c] = rq.fine ? (int8_t)rq.code(out(c)) : (int8_t)0;
  for (int64_t c = p.C + lane; c < p.z_pitch; c += 64) codes[c] = 0;
  if (lane == 0) p.z_scale[row] = rq.scale;
}

}  // namespace qattn

using namespace qattn;

static int check_param(const qattn_param& q, const char* name, int64_t B, int64_t L) {
  if (!q.data) return QATTN_OK;
  QATTN_REQUIRE(q.dtype >= QATTN_BF16 && q.dtype <= QATTN_F32, QATTN_ERR_DTYPE, "block_norm: %s has dtype code %d", name,
                q.dtype);
  const int64_t size = q.dtype == QATTN_F32 ? 4 : 2;
  QATTN_REQUIRE(reinterpret_cast<uintptr_t>(q.data) % size == 0, QATTN_ERR_ALIGN, "block_norm: %s is misaligned", name);
  QATTN_REQUIRE((q.sb >= 0 || B < 2) && (q.sl >= 0 || L < 2), QATTN_ERR_STRIDE, "block_norm: %s has a negative stride",
                name);
  return QATTN_OK;
}

// Waves per row and 8-channel groups per thread, by the groups of 8 lanes that they occupy (idle ones too) and by the
// waves.  A thread that has only x to read takes up to 5 groups, and a wave more costs as much as 12 lanes' worth of groups:
// reductions between waves take barriers (row quantizer of 39606 x 3328 with 7 / 4 / 3 / 2 waves: 134 / 99 / 96 / 79 us).
// One that reads y or parameters beside it takes 2 where 8 waves suffice: its registers then leave room for more waves
// (2 x 4680 x 5120, 5 / 2 groups at most: norm with per-token scale and shift 113 / 106 us).
static bool row_shape(int C, bool plain, int& waves, int& groups) {
  const int vecs = (C + 7) / 8;
  int64_t best = -1;
  for (int nv = 1; nv <= (plain || best < 0 ? 5 : 2); nv++) {
    const int w = (vecs + 64 * nv - 1) / (64 * nv);
    if (w > kMaxRowWaves) continue;
    const int64_t cost = (int64_t)w * nv * 16 + w * (plain ? 24 : 1);
    if (best < 0 || cost < best) best = cost, waves = w, groups = nv;
  }
  return best >= 0;
}

// Staging pays for many rows of a batch entry (microseconds, read per row / staged: norm of 4680 x 5120 26 / 30, of 9000 x
// 5120 45.5 / 45 from one input that the caches hold and 53 / 47 from several in turn, of 16384 x 5120 95 / 75, of 75600 x
// 5120 429 / 304, of 16384 x 1536 26 / 19; gated residual + norm of 75600 x 640 109 / 83, of 48306 x 7040 600 / 514).  The
// two are equal at about 9000 rows already: between that and this number some calls take up to a fifth longer than they
// could.  A batch entry counts by itself: 21 frames of 1560 x 1536 with parameters of their own read them for every row (62
// us, as one entry of 32760 rows 36).
constexpr int64_t kStagedRows = 16384;
constexpr int kStagedWidest = 8192;
constexpr size_t kLds = 163840, kSlotBytes = 8 * 2 * kRowSlots * kMaxRowWaves * 4;
// Groups a thread holds in the staged kernel, before a row takes two or four waves.
constexpr int staged_groups(int dtype, int ymode) { return dtype == QATTN_F32 || ymode == Y_F32 ? 3 : 5; }
constexpr int64_t kCus = 256;
// Offsets of the folded parameters in LDS, and its bytes; 0 where rows do not share them or LDS does not hold
// them.
static size_t stage(BlockNormParams& p, const Param* const* params) {
  for (int i = 0; i < 7; i++)
    if (params[i]->p && params[i]->sl) return 0;
  p.stage_half = (p.C + 7) / 8 * 4;
  int n = 0;
  auto take = [&](bool there) { return there ? 2 * p.stage_half * n++ : -1; };
  const bool post = p.post_norm && (p.post_weight.p || p.post_bias.p);
  const bool affine = p.z && (p.weight.p || p.bias.p || p.scale.p || p.shift.p);
  p.staged[0] = take(post), p.staged[1] = take(post);
  p.staged[2] = take(p.y && p.gate.p);
  p.staged[3] = take(affine), p.staged[4] = take(affine);
  const size_t bytes = (size_t)n * 2 * p.stage_half * 4;
  return bytes + kSlotBytes <= kLds ? bytes : 0;
}

template <int XD, int YM>
static void launch_rows(const BlockNormParams& p, int waves, int groups, size_t lds, hipStream_t stream) {
  if (lds) {
    constexpr int nvmax = staged_groups(XD, YM);
    const int vecs = (p.C + 511) / 512;  // at most 16 (kStagedWidest), so four waves hold up to four groups
    const int w = vecs <= nvmax ? 1 : vecs <= 2 * nvmax ? 2 : 4, nv = (vecs + w - 1) / w;
    // rows of a batch entry in turns, by two workgroups for each CU where LDS holds them.  Kernels of more than 128 registers
    // (four groups a thread or more, three with y) have room for one at a time: the second half of their grid then follows
    // the first and stages the parameters once more.
    const int64_t batches = p.rows / p.L, per = 8 / w;
    const int64_t hold = std::max((int64_t)1, kCus * std::min((int64_t)2, (int64_t)(kLds / (lds + kSlotBytes))) / batches);
    const int64_t turns = (p.L + per * hold - 1) / (per * hold);
    const dim3 grid((unsigned)((p.L + per * turns - 1) / (per * turns)), (unsigned)batches), block(512);
    if (nv == 1) staged_row_kernel<XD, YM, 1><<<grid, block, lds, stream>>>(p, w, (int)turns);
    else if (nv == 2) staged_row_kernel<XD, YM, 2><<<grid, block, lds, stream>>>(p, w, (int)turns);
    else if (nv == 3) staged_row_kernel<XD, YM, 3><<<grid, block, lds, stream>>>(p, w, (int)turns);
    else if (nv == 4) staged_row_kernel<XD, YM, 4><<<grid, block, lds, stream>>>(p, w, (int)turns);
    else if constexpr (nvmax > 4) staged_row_kernel<XD, YM, 5><<<grid, block, lds, stream>>>(p, w, (int)turns);
    return;
  }
  if (p.C <= 256) {
    const int lanes = p.C <= 64 ? 8 : p.C <= 128 ? 16 : 32, per = 256 / lanes;
    const dim3 grid((unsigned)((p.rows + per - 1) / per)), block(256);
    if (lanes == 8) narrow_row_kernel<XD, YM, 8><<<grid, block, 0, stream>>>(p);
    else if (lanes == 16) narrow_row_kernel<XD, YM, 16><<<grid, block, 0, stream>>>(p);
    else narrow_row_kernel<XD, YM, 32><<<grid, block, 0, stream>>>(p);
    return;
  }
  const dim3 grid((unsigned)p.rows), block(waves * 64);
  if (groups == 1) row_norm_kernel<XD, YM, 1><<<grid, block, 0, stream>>>(p);
  else if (groups == 2) row_norm_kernel<XD, YM, 2><<<grid, block, 0, stream>>>(p);
  else if (groups == 3) row_norm_kernel<XD, YM, 3><<<grid, block, 0, stream>>>(p);
  else if (groups == 4) row_norm_kernel<XD, YM, 4><<<grid, block, 0, stream>>>(p);
  else row_norm_kernel<XD, YM, 5><<<grid, block, 0, stream>>>(p);
}

// any_y: y may also be fp32 beside a half x
static int run_block_norm(const qattn_block_norm_args* a, bool any_y, qattn_stream_t stream) {
  QATTN_REQUIRE(a && a->size == sizeof(qattn_block_norm_args), QATTN_ERR_ARG,
                "block_norm: args missing or of another version of the header");
  QATTN_REQUIRE(a->x_dtype >= QATTN_BF16 && a->x_dtype <= QATTN_F32, QATTN_ERR_DTYPE, "block_norm: x has dtype code %d",
                a->x_dtype);
  QATTN_REQUIRE(!a->y || a->y_dtype == a->x_dtype ||
                    (a->x_dtype == QATTN_F32 && a->y_dtype >= QATTN_BF16 && a->y_dtype <= QATTN_F32) ||
                    (any_y && a->y_dtype == QATTN_F32),
                QATTN_ERR_DTYPE, "block_norm: y has dtype code %d beside x's %d", a->y_dtype, a->x_dtype);
  QATTN_REQUIRE(!a->z || (a->z_dtype >= QATTN_BF16 && a->z_dtype <= QATTN_I8), QATTN_ERR_DTYPE,
                "block_norm: z has dtype code %d", a->z_dtype);
  QATTN_REQUIRE(a->B >= 0 && a->L >= 0 && a->C >= 1 && a->C <= (1 << 24), QATTN_ERR_SHAPE,
                "block_norm: B = %lld, L = %lld, C = %lld", (long long)a->B, (long long)a->L, (long long)a->C);
  QATTN_REQUIRE(a->B == 0 || a->L <= ((int64_t)1 << 31) / a->B, QATTN_ERR_SHAPE, "block_norm: more than 2^31 rows");
  QATTN_REQUIRE(a->norm >= QATTN_NORM_NONE && a->norm <= QATTN_NORM_RMS && a->post_norm >= QATTN_NORM_NONE &&
                    a->post_norm <= QATTN_NORM_RMS,
                QATTN_ERR_ARG, "block_norm: norm codes %d, %d", a->norm, a->post_norm);
  QATTN_REQUIRE(a->h || a->z, QATTN_ERR_ARG, "block_norm: no output");
  if (a->B == 0 || a->L == 0) return QATTN_OK;
  QATTN_REQUIRE(a->x, QATTN_ERR_ARG, "block_norm: x is null");
  const uintptr_t xs = a->x_dtype == QATTN_F32 ? 4 : 2, ys = a->y_dtype == QATTN_F32 ? 4 : 2;
  QATTN_REQUIRE(reinterpret_cast<uintptr_t>(a->x) % xs == 0 && (!a->y || reinterpret_cast<uintptr_t>(a->y) % ys == 0),
                QATTN_ERR_ALIGN, "block_norm: x or y is misaligned");
  QATTN_REQUIRE(aligned16(a->h) && aligned16(a->z), QATTN_ERR_ALIGN, "block_norm: outputs must be 16-byte aligned");
  if (a->z && a->z_dtype == QATTN_I8) {
    QATTN_REQUIRE(a->z_scale && reinterpret_cast<uintptr_t>(a->z_scale) % 4 == 0, QATTN_ERR_ARG,
                  "block_norm: INT8 rows need a scale per row");
    QATTN_REQUIRE(a->z_pitch >= a->C && a->z_pitch % 16 == 0, QATTN_ERR_STRIDE,
                  "block_norm: the pitch of INT8 rows must be a multiple of 16, at least C");
  }
  const qattn_param* params[] = {&a->gate, &a->weight, &a->bias, &a->scale, &a->shift, &a->post_weight, &a->post_bias};
  const char* names[] = {"gate", "weight", "bias", "scale", "shift", "post_weight", "post_bias"};
  for (int i = 0; i < 7; i++)
    if (int rc = check_param(*params[i], names[i], a->B, a->L)) return rc;

  BlockNormParams p;
  // the stride of a dimension of one means nothing (and says nothing about alignment)
  p.x = a->x, p.xb = a->B > 1 ? a->x_sb : 0, p.xl = a->L > 1 ? a->x_sl : 0;
  p.y = a->y, p.yb = a->B > 1 ? a->y_sb : 0, p.yl = a->L > 1 ? a->y_sl : 0;
  p.h = a->h, p.z = a->z, p.z_scale = a->z_scale, p.z_pitch = a->z_pitch;
  p.x_dtype = a->x_dtype, p.y_dtype = a->y_dtype, p.z_dtype = a->z_dtype;
  Param* to[] = {&p.gate, &p.weight, &p.bias, &p.scale, &p.shift, &p.post_weight, &p.post_bias};
  for (int i = 0; i < 7; i++)
    *to[i] = Param{params[i]->data, params[i]->dtype, a->B > 1 ? params[i]->sb : 0, a->L > 1 ? params[i]->sl : 0};
  p.L = a->L, p.rows = a->B * a->L, p.C = (int)a->C;
  p.norm = a->norm, p.post_norm = a->y ? a->post_norm : QATTN_NORM_NONE;
  p.eps = a->eps, p.post_eps = a->post_eps, p.residual_scale = a->residual_scale;
  const hipStream_t st = (hipStream_t)stream;
  int waves = 1, groups;
  bool plain = !p.y;
  for (int i = 0; i < 7; i++) plain = plain && !to[i]->p;
  const bool wide = !row_shape(p.C, plain, waves, groups);
  QATTN_REQUIRE(p.rows * waves <= ((int64_t)1 << 25), QATTN_ERR_SHAPE,
                "block_norm: %lld rows of %d channels are more than one launch takes", (long long)p.rows, p.C);
  if (wide) {
    wide_row_kernel<<<dim3((unsigned)((p.rows + 3) / 4)), 256, 0, st>>>(p);
    return check_launch("block_norm");
  }
  const size_t lds = p.C > 256 && p.C <= kStagedWidest && p.L >= kStagedRows && a->B < 65536 ? stage(p, to) : 0;
  if (p.x_dtype == QATTN_F32) {
    if (!p.y) launch_rows<QATTN_F32, Y_NONE>(p, waves, groups, lds, st);
    else if (p.y_dtype == QATTN_F32) launch_rows<QATTN_F32, Y_SAME>(p, waves, groups, lds, st);
    else if (p.y_dtype == QATTN_BF16) launch_rows<QATTN_F32, Y_BF16>(p, waves, groups, lds, st);
    else launch_rows<QATTN_F32, Y_FP16>(p, waves, groups, lds, st);
  } else if (p.x_dtype == QATTN_BF16) {
    if (!p.y) launch_rows<QATTN_BF16, Y_NONE>(p, waves, groups, lds, st);
    else if (p.y_dtype == QATTN_F32) launch_rows<QATTN_BF16, Y_F32>(p, waves, groups, lds, st);
    else launch_rows<QATTN_BF16, Y_SAME>(p, waves, groups, lds, st);
  } else {
    if (!p.y) launch_rows<QATTN_FP16, Y_NONE>(p, waves, groups, lds, st);
    else if (p.y_dtype == QATTN_F32) launch_rows<QATTN_FP16, Y_F32>(p, waves, groups, lds, st);
    else launch_rows<QATTN_FP16, Y_SAME>(p, waves, groups, lds, st);
  }
  return check_launch("block_norm");
}

extern "C" int qattn_block_norm(const qattn_block_norm_args* args, qattn_stream_t stream) {
  return run_block_norm(args, false, stream);
}
extern "C" int qattn_block_norm_ex(const qattn_block_norm_args* args, qattn_stream_t stream) {
  return run_block_norm(args, true, stream);
}
