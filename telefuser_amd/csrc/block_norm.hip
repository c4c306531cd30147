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
#include "common.h"

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

// One wave per row, one element per lane and step; the row is read again for each reduction.
__global__ __launch_bounds__(256) void block_norm_kernel(BlockNormParams p) {
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
  top = wave_max_u32(top);
  const RowQuant rq(top);
  int8_t* codes = static_cast<int8_t*>(p.z) + row * p.z_pitch;
  for (int c = lane; c < p.C; c += 64) codes[c] = (int8_t)rq.code(out(c));
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
  p.x = a->x, p.xb = a->x_sb, p.xl = a->x_sl;
  p.y = a->y, p.yb = a->y_sb, p.yl = a->y_sl;
  p.h = a->h, p.z = a->z, p.z_scale = a->z_scale, p.z_pitch = a->z_pitch;
  p.x_dtype = a->x_dtype, p.y_dtype = a->y_dtype, p.z_dtype = a->z_dtype;
  Param* to[] = {&p.gate, &p.weight, &p.bias, &p.scale, &p.shift, &p.post_weight, &p.post_bias};
  for (int i = 0; i < 7; i++) *to[i] = Param{params[i]->data, params[i]->dtype, params[i]->sb, params[i]->sl};
  p.L = a->L, p.rows = a->B * a->L, p.C = (int)a->C;
  p.norm = a->norm, p.post_norm = a->y ? a->post_norm : QATTN_NORM_NONE;
  p.eps = a->eps, p.post_eps = a->post_eps, p.residual_scale = a->residual_scale;
  block_norm_kernel<<<dim3((unsigned)((p.rows + 3) / 4)), 256, 0, (hipStream_t)stream>>>(p);
  return check_launch("block_norm");
}
