// The row operators around a DiT block: the norm before it (LayerNorm or RMSNorm, weight, bias, adaLN scale and shift),
// the gated residual after it (optionally of the normalized output), both in one pass, and the row quantizer.
//
//   v    = x                                             or  residual_scale * x + gate * p(y),  p(y) = y or its norm
//   h    = v                                             (stored where wanted)
//   z    = n(v) * weight + bias, then z * (1 + scale) + shift
//   n(v) = v | (v - mean) / sqrt(var + eps) | v / sqrt(mean(v^2) + eps)
//   z is stored in bf16 / fp16 / fp32, or as INT8: code = rint(127 z / max|z|), row scale max|z| / 127
//
// Everything between the loads and the stores is fp32; v reaches the norm unrounded.  The variance is that of the
// centred values.  Parameters are read with the strides of their broadcast shape.
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
// A workgroup of W waves takes a row, every thread NV groups of 8 channels: each value is loaded once, the reductions
// run over registers (DPP within a wave, LDS between waves), and the outputs are written from them.
//   VEC:  groups of 8 consecutive channels in 16-byte loads (32 for fp32); everything divides by 8 and is aligned.
//   else: channel (8 i + e) T + tid, one element per load: any width, stride and alignment.
constexpr int kRowGroup = 8;
constexpr int kMaxRowWaves = 8;

enum YMode { Y_NONE, Y_SAME, Y_BF16, Y_FP16 };

template <int DT, bool VEC>
struct RawGroup {
  static constexpr int kWords = DT == QATTN_F32 ? 8 : VEC ? 4 : 8;  // scalar halves: one word each
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* p, int64_t at, int c, int step, int C) {
    if constexpr (VEC) {
      if (c < C) {
        constexpr int kSize = DT == QATTN_F32 ? 4 : 2;
        const v4u* q = reinterpret_cast<const v4u*>(static_cast<const char*>(p) + (at + c) * kSize);
#pragma unroll
        for (int k = 0; k < kWords / 4; k++) {
          const v4u v = q[k];
#pragma unroll
          for (int e = 0; e < 4; e++) w[4 * k + e] = v[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < kWords; e++) w[e] = 0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int cc = c + e * step;
        if constexpr (DT == QATTN_F32) w[e] = cc < C ? static_cast<const uint32_t*>(p)[at + cc] : 0u;
        else w[e] = cc < C ? static_cast<const uint16_t*>(p)[at + cc] : 0u;
      }
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (DT == QATTN_F32) return __uint_as_float(w[e]);
    const uint16_t h = VEC ? (uint16_t)(w[e / 2] >> (16 * (e & 1))) : (uint16_t)w[e];
    return half_to_f32<DT == QATTN_FP16>(h);
  }
};

template <bool VEC>
__device__ __forceinline__ void load_param8(const Param& q, int64_t b, int64_t l, int c, int step, int C, float (&out)[8]) {
  const int64_t at = b * q.sb + l * q.sl;
  if (q.dtype == QATTN_F32) {
    RawGroup<QATTN_F32, VEC> g;
    g.load(q.p, at, c, step, C);
#pragma unroll
    for (int e = 0; e < 8; e++) out[e] = g.get(e);
  } else {
    RawGroup<QATTN_BF16, VEC> g;
    g.load(q.p, at, c, step, C);
    if (q.dtype == QATTN_BF16) {
#pragma unroll
      for (int e = 0; e < 8; e++) out[e] = g.get(e);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) out[e] = f16_to_f32(VEC ? (uint16_t)(g.w[e / 2] >> (16 * (e & 1))) : (uint16_t)g.w[e]);
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void store8(void* p, int dtype, int64_t at, int c, int step, int C, const float (&v)[8]) {
  if constexpr (VEC) {
    if (c >= C) return;
    if (dtype == QATTN_F32) {
      v4f* q = reinterpret_cast<v4f*>(static_cast<float*>(p) + at + c);
      q[0] = v4f{v[0], v[1], v[2], v[3]};
      q[1] = v4f{v[4], v[5], v[6], v[7]};
    } else {
      v4u o;
      if (dtype == QATTN_FP16) {
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = pack_half2<true>(v[2 * e], v[2 * e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = pack_half2<false>(v[2 * e], v[2 * e + 1]);
      }
      *reinterpret_cast<v4u*>(static_cast<uint16_t*>(p) + at + c) = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (c + e * step < C) store_elem(p, dtype, at + c + e * step, v[e]);
  }
}

// Reductions over the workgroup; each call has its own LDS slots, so one barrier separates write and read.
struct RowReduce {
  uint32_t (*slots)[kMaxRowWaves];
  int waves, wave;
  int used = 0;
  __device__ __forceinline__ float sum(float v) {
    float t = wave_total(v);
    if (waves == 1) return t;
    uint32_t* s = slots[used++];
    if ((threadIdx.x & 63) == 0) s[wave] = __float_as_uint(t);
    __syncthreads();
    t = 0.0f;
    for (int i = 0; i < waves; i++) t += __uint_as_float(s[i]);
    return t;
  }
  __device__ __forceinline__ uint32_t top(uint32_t v) {
    uint32_t t = wave_top(v);
    if (waves == 1) return t;
    uint32_t* s = slots[used++];
    if ((threadIdx.x & 63) == 0) s[wave] = t;
    __syncthreads();
    for (int i = 0; i < waves; i++) t = max(t, s[i]);
    return t;
  }
};

template <int XD, int YM, bool VEC, int NV>
__global__ __launch_bounds__(kMaxRowWaves * 64) void row_norm_kernel(BlockNormParams p) {
  constexpr int YD = YM == Y_BF16 ? QATTN_BF16 : YM == Y_FP16 ? QATTN_FP16 : XD;
  __shared__ uint32_t slots[5][kMaxRowWaves];
  const int T = blockDim.x, tid = threadIdx.x, step = VEC ? 1 : T;
  RowReduce red{slots, T >> 6, tid >> 6};
  const int64_t row = blockIdx.x;
  const int64_t b = row / p.L, l = row - b * p.L;
  const int C = p.C;
  const float inv_c = 1.0f / (float)C;
  auto first = [&](int i) { return VEC ? (i * T + tid) * 8 : i * 8 * T + tid; };
  // out-of-row values of the scalar form: element e of group i is beyond the row
  auto in_row = [&](int i, int e) { return first(i) + (VEC ? 0 : e * T) < C; };

  RawGroup<XD, VEC> xr[NV];
  RawGroup<YD, VEC> yr[YM == Y_NONE ? 1 : NV];
  const int64_t xo = b * p.xb + l * p.xl, yo = b * p.yb + l * p.yl;
#pragma unroll
  for (int i = 0; i < NV; i++) xr[i].load(p.x, xo, first(i), step, C);
  if constexpr (YM != Y_NONE)
#pragma unroll
    for (int i = 0; i < NV; i++) yr[i].load(p.y, yo, first(i), step, C);

  float v[NV][8];
  if constexpr (YM != Y_NONE) {
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = yr[i].get(e);
    if (p.post_norm) {
      float mean = 0.0f, s = 0.0f;
      if (p.post_norm == QATTN_NORM_LAYER) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) s += v[i][e];
        mean = red.sum(s) * inv_c;
        s = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          v[i][e] = in_row(i, e) ? v[i][e] - mean : 0.0f;
          s = fmaf(v[i][e], v[i][e], s);
        }
      const float rstd = 1.0f / sqrtf(red.sum(s) * inv_c + p.post_eps);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] *= rstd;
        if (p.post_weight.p) {
          load_param8<VEC>(p.post_weight, b, l, first(i), step, C, t);
#pragma unroll
          for (int e = 0; e < 8; e++) v[i][e] *= t[e];
        }
        if (p.post_bias.p) {
          load_param8<VEC>(p.post_bias, b, l, first(i), step, C, t);
#pragma unroll
          for (int e = 0; e < 8; e++) v[i][e] += t[e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (p.gate.p) {
        float t[8];
        load_param8<VEC>(p.gate, b, l, first(i), step, C, t);
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] *= t[e];
      }
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = fmaf(p.residual_scale, xr[i].get(e), v[i][e]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = xr[i].get(e);
  }
  if (p.h)
#pragma unroll
    for (int i = 0; i < NV; i++) store8<VEC>(p.h, XD, row * C, first(i), step, C, v[i]);
  if (!p.z) return;

  if (p.norm) {
    float mean = 0.0f, s = 0.0f;
    if (p.norm == QATTN_NORM_LAYER) {
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) s += v[i][e];
      mean = red.sum(s) * inv_c;
      s = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        v[i][e] = in_row(i, e) ? v[i][e] - mean : 0.0f;
        s = fmaf(v[i][e], v[i][e], s);
      }
    const float rstd = 1.0f / sqrtf(red.sum(s) * inv_c + p.eps);
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] *= rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; i++) {
    float t[8];
    if (p.weight.p) {
      load_param8<VEC>(p.weight, b, l, first(i), step, C, t);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] *= t[e];
    }
    if (p.bias.p) {
      load_param8<VEC>(p.bias, b, l, first(i), step, C, t);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] += t[e];
    }
    if (p.scale.p) {
      load_param8<VEC>(p.scale, b, l, first(i), step, C, t);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = fmaf(v[i][e], t[e], v[i][e]);
    }
    if (p.shift.p) {
      load_param8<VEC>(p.shift, b, l, first(i), step, C, t);
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] += t[e];
    }
  }
  if (p.z_dtype != QATTN_I8) {
#pragma unroll
    for (int i = 0; i < NV; i++) store8<VEC>(p.z, p.z_dtype, row * C, first(i), step, C, v[i]);
    return;
  }
  // max|z| as an integer: the bits of |z| are ordered as the values, infinity and NaN above them all
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; i++)
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (in_row(i, e)) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
  const RowQuant rq(red.top(top));
  int8_t* codes = static_cast<int8_t*>(p.z) + row * p.z_pitch;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int c = first(i);
    if constexpr (VEC) {
      if (c < C)
        *reinterpret_cast<v2u*>(codes + c) = v2u{rq.code4(v[i][0], v[i][1], v[i][2], v[i][3]),
                                                 rq.code4(v[i][4], v[i][5], v[i][6], v[i][7])};
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (c + e * T < C) codes[c + e * T] = rq.fine ? (int8_t)rq.code(v[i][e]) : (int8_t)0;
    }
  }
  for (int64_t c = C + tid; c < p.z_pitch; c += T) codes[c] = 0;
  if (tid == 0) p.z_scale[row] = rq.scale;
}

// ------------------------------------------------------------------------------------------------
// rows too wide for that: one wave per row, one element per lane and step, the row read again for each reduction
// ------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void wide_row_kernel(BlockNormParams p) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const int lane = threadIdx.x & 63;
  const int64_t b = row / p.L, l = row - b * p.L;
  const float inv_c = 1.0f / (float)p.C;
  const int64_t xo = b * p.xb + l * p.xl, yo = b * p.yb + l * p.yl;

  float y_mean = 0.0f, y_rstd = 1.0f;
  if (p.y && p.post_norm) {
    float s = 0.0f;
    if (p.post_norm == QATTN_NORM_LAYER) {
      for (int c = lane; c < p.C; c += 64) s += load_elem(p.y, p.y_dtype, yo + c);
      y_mean = wave_sum(s) * inv_c;
    }
    s = 0.0f;
    for (int c = lane; c < p.C; c += 64) {
      const float d = load_elem(p.y, p.y_dtype, yo + c) - y_mean;
      s = fmaf(d, d, s);
    }
    y_rstd = 1.0f / sqrtf(wave_sum(s) * inv_c + p.post_eps);
  }
  auto value = [&](int c) {
    float v = load_elem(p.x, p.x_dtype, xo + c);
    if (p.y) {
      float t = load_elem(p.y, p.y_dtype, yo + c);
      if (p.post_norm) {
        t = (t - y_mean) * y_rstd;
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

  float mean = 0.0f, rstd = 1.0f;
  if (p.norm) {
    float s = 0.0f;
    if (p.norm == QATTN_NORM_LAYER) {
      for (int c = lane; c < p.C; c += 64) s += value(c);
      mean = wave_sum(s) * inv_c;
    }
    s = 0.0f;
    for (int c = lane; c < p.C; c += 64) {
      const float d = value(c) - mean;
      s = fmaf(d, d, s);
    }
    rstd = 1.0f / sqrtf(wave_sum(s) * inv_c + p.eps);
  }
  auto out = [&](int c) {
    float z = (value(c) - mean) * rstd;
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

// Waves per row and 8-channel groups per thread: the pair that leaves the fewest lanes idle, of equal ones the one with
// fewer waves (a reduction between waves takes a barrier).
static bool row_shape(int C, int& waves, int& groups) {
  const int vecs = (C + 7) / 8;
  int64_t best = -1;
  for (int nv = 1; nv <= 4; nv++) {
    const int w = (vecs + 64 * nv - 1) / (64 * nv);
    if (w > kMaxRowWaves) continue;
    const int64_t cost = (int64_t)w * nv * 16 + w;
    if (best < 0 || cost < best) best = cost, waves = w, groups = nv;
  }
  return best >= 0;
}

template <int XD, int YM, bool VEC>
static void launch_rows(const BlockNormParams& p, int waves, int groups, hipStream_t stream) {
  const dim3 grid((unsigned)p.rows), block(waves * 64);
  if (groups == 1) row_norm_kernel<XD, YM, VEC, 1><<<grid, block, 0, stream>>>(p);
  else if (groups == 2) row_norm_kernel<XD, YM, VEC, 2><<<grid, block, 0, stream>>>(p);
  else if (groups == 3) row_norm_kernel<XD, YM, VEC, 3><<<grid, block, 0, stream>>>(p);
  else row_norm_kernel<XD, YM, VEC, 4><<<grid, block, 0, stream>>>(p);
}
template <int XD, int YM>
static void launch_rows(const BlockNormParams& p, bool vec, int waves, int groups, hipStream_t stream) {
  if (vec) launch_rows<XD, YM, true>(p, waves, groups, stream);
  else launch_rows<XD, YM, false>(p, waves, groups, stream);
}

// every row of 8-channel groups in 16-byte pieces
static bool vectors(const void* q, int dtype, int64_t sb, int64_t sl) {
  const int64_t per = 16 / (dtype == QATTN_F32 ? 4 : 2);
  return aligned16(q) && sb % per == 0 && sl % per == 0;
}

extern "C" int qattn_block_norm(const qattn_block_norm_args* a, qattn_stream_t stream) {
  QATTN_REQUIRE(a && a->size == sizeof(qattn_block_norm_args), QATTN_ERR_ARG,
                "block_norm: args missing or of another version of the header");
  QATTN_REQUIRE(a->x_dtype >= QATTN_BF16 && a->x_dtype <= QATTN_F32, QATTN_ERR_DTYPE, "block_norm: x has dtype code %d",
                a->x_dtype);
  QATTN_REQUIRE(!a->y || a->y_dtype == a->x_dtype || (a->x_dtype == QATTN_F32 && a->y_dtype >= QATTN_BF16 &&
                                                      a->y_dtype <= QATTN_F32),
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
  for (int i = 0; i < 7; i++) *to[i] = Param{params[i]->data, params[i]->dtype, a->B > 1 ? params[i]->sb : 0, a->L > 1 ? params[i]->sl : 0};
  p.L = a->L, p.rows = a->B * a->L, p.C = (int)a->C;
  p.norm = a->norm, p.post_norm = a->y ? a->post_norm : QATTN_NORM_NONE;
  p.eps = a->eps, p.post_eps = a->post_eps, p.residual_scale = a->residual_scale;
  const hipStream_t st = (hipStream_t)stream;
  int waves, groups;
  if (!row_shape(p.C, waves, groups)) {
    wide_row_kernel<<<dim3((unsigned)((p.rows + 3) / 4)), 256, 0, st>>>(p);
    return check_launch("block_norm");
  }
  bool vec = p.C % 8 == 0 && vectors(p.x, p.x_dtype, p.xb, p.xl) && (!p.y || vectors(p.y, p.y_dtype, p.yb, p.yl));
  for (int i = 0; i < 7; i++) vec = vec && vectors(to[i]->p, to[i]->dtype, to[i]->sb, to[i]->sl);
  if (p.x_dtype == QATTN_F32) {
    if (!p.y) launch_rows<QATTN_F32, Y_NONE>(p, vec, waves, groups, st);
    else if (p.y_dtype == QATTN_F32) launch_rows<QATTN_F32, Y_SAME>(p, vec, waves, groups, st);
    else if (p.y_dtype == QATTN_BF16) launch_rows<QATTN_F32, Y_BF16>(p, vec, waves, groups, st);
    else launch_rows<QATTN_F32, Y_FP16>(p, vec, waves, groups, st);
  } else if (p.x_dtype == QATTN_BF16) {
    if (p.y) launch_rows<QATTN_BF16, Y_SAME>(p, vec, waves, groups, st);
    else launch_rows<QATTN_BF16, Y_NONE>(p, vec, waves, groups, st);
  } else {
    if (p.y) launch_rows<QATTN_FP16, Y_SAME>(p, vec, waves, groups, st);
    else launch_rows<QATTN_FP16, Y_NONE>(p, vec, waves, groups, st);
  }
  return check_launch("block_norm");
}
