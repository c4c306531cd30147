// INT8 linear: out[m, n] = act(x_scale[m] * w_scale[n] * sum_k x[m, k] w[n, k] + bias[n]) on v_mfma_i32_32x32x32_i8.
//
// A workgroup computes a TM x TN tile.  The weight is the MFMA's A operand and the activation its B operand, so a lane of
// the result holds one token and runs of four channels.  K advances by 128 bytes: both operands' rows come into LDS by
// DMA, a whole 128-byte line per row, double-buffered: the DMA of the next step runs while this one is multiplied.  Row r
// of a tile holds its 16-byte chunk c at position c ^ ((r >> 1) & 7), so that the 16-byte reads of the fragments (32 rows
// at one chunk) spread over the banks; the DMA's per-lane global address does the permutation.
// Rows past M or N lie behind the end of the buffer resource and read as zeros.
#include "attn_device.h"

namespace qattn {

struct LinearParams {
  const int8_t* x;
  int64_t x_pitch;
  const float* x_scale;
  const int8_t* w;
  int64_t w_pitch;
  const float* w_scale;
  const float* bias;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int64_t M, N;
  int K, act;
  int tiles_m, tiles_n;
};

constexpr int kLinK = 128;  // bytes of K per step

template <int ACT>
__device__ __forceinline__ float activate(float y) {
  if constexpr (ACT == QATTN_ACT_GELU_TANH) {
    // y (1 + tanh u) / 2 = y / (1 + exp(-2 u)), u = sqrt(2 / pi) (y + 0.044715 y^3)
    const float k = -2.0f * 0.7978845608f * 1.4426950409f;
    const float t = y * y;
    return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * fmaf(t, k * 0.044715f, k)));
  } else if constexpr (ACT == QATTN_ACT_SILU) {
    return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.4426950409f));
  } else {
    return y;
  }
}

template <int N>
__device__ __forceinline__ void wait_vm_barrier() {
  // the LDS reads too: a fragment read still in flight must not meet the next DMA into its buffer
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

template <int TM, int TN, int WM, int WN, int ACT>
__global__ __launch_bounds__(WM* WN * 64) void linear_int8_kernel(LinearParams p) {
  constexpr int kWaves = WM * WN;
  constexpr int NI = TN / WN / 32, MJ = TM / WM / 32;  // 32 x 32 results of a wave
  constexpr int kRows = TM + TN;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2][kRows * kLinK];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = xcd_remap(blockIdx.x, gridDim.x);
  const int64_t tm = id / p.tiles_n, tn = id - tm * p.tiles_n;
  const int64_t m0 = tm * TM, n0 = tn * TN;

  const int64_t rows_m = min((int64_t)TM, p.M - m0), rows_n = min((int64_t)TN, p.N - n0);
  const v4u rx = make_rsrc(p.x + m0 * p.x_pitch, (uint32_t)((rows_m - 1) * p.x_pitch + p.K));
  const v4u rw = make_rsrc(p.w + n0 * p.w_pitch, (uint32_t)((rows_n - 1) * p.w_pitch + p.K));
  const uint32_t base = lds_addr(lds);

  // one DMA instruction moves 8 rows; the wave's instructions are 8 * kWaves rows apart
  const int r8 = wave * 8 + (lane >> 3);
  const uint32_t chunk = (uint32_t)((lane & 7) ^ ((r8 >> 1) & 7)) * 16;
  const uint32_t vx = (uint32_t)(r8 * p.x_pitch) + chunk, vw = (uint32_t)(r8 * p.w_pitch) + chunk;
  auto fetch = [&](int buf, uint32_t k) {
    const uint32_t to = base + buf * kRows * kLinK + wave * 1024;
#pragma unroll
    for (int i = 0; i < TM / 8 / kWaves; i++)
      lds_dma16(vx + (uint32_t)(i * 8 * kWaves * p.x_pitch), rx, k, to + i * kWaves * 1024);
#pragma unroll
    for (int i = 0; i < TN / 8 / kWaves; i++)
      lds_dma16(vw + (uint32_t)(i * 8 * kWaves * p.w_pitch), rw, k, to + TM * kLinK + i * kWaves * 1024);
  };

  v16i acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; i++)
#pragma unroll
    for (int j = 0; j < MJ; j++) acc[i][j] = v16i{};

  const int wm = wave % WM, wn = wave / WM;
  const int row = lane & 31;
  const int swz = ((lane >> 5) ^ ((row >> 1) & 7)) * 16;
  const int xrow = (wm * (TM / WM) + row) * kLinK, wrow = (TM + wn * (TN / WN) + row) * kLinK;

  fetch(0, 0);
  const int steps = p.K / kLinK;
  for (int t = 0; t < steps; t++) {
    wait_vm_barrier<0>();
    if (t + 1 < steps) fetch((t + 1) & 1, (uint32_t)(t + 1) * kLinK);
    const uint8_t* tile = lds[t & 1];
#pragma unroll
    for (int s = 0; s < 4; s++) {
      v4i a[NI], b[MJ];
#pragma unroll
      for (int i = 0; i < NI; i++) a[i] = *reinterpret_cast<const v4i*>(tile + wrow + i * 32 * kLinK + (swz ^ (s * 32)));
#pragma unroll
      for (int j = 0; j < MJ; j++) b[j] = *reinterpret_cast<const v4i*>(tile + xrow + j * 32 * kLinK + (swz ^ (s * 32)));
#pragma unroll
      for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < MJ; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
    }
  }

  // element r of a result: channel 8 (r / 4) + 4 (lane / 32) + r % 4, token lane % 32
#pragma unroll
  for (int i = 0; i < NI; i++) {
    const int64_t n = n0 + wn * (TN / WN) + i * 32 + (lane >> 5) * 4;
#pragma unroll
    for (int j = 0; j < MJ; j++) {
      const int64_t m = m0 + wm * (TM / WM) + j * 32 + row;
      if (m >= p.M) continue;
      const float sx = p.x_scale[m];
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int64_t c = n + (r >> 2) * 8 + (r & 3);
        if (c >= p.N) continue;
        const float y = activate<ACT>(fmaf((float)acc[i][j][r] * sx, p.w_scale[c], p.bias ? p.bias[c] : 0.0f));
        const int64_t at = m * p.out_stride + c;
        if (p.out_dtype == QATTN_F32) static_cast<float*>(p.out)[at] = y;
        else static_cast<uint16_t*>(p.out)[at] = p.out_dtype == QATTN_FP16 ? f32_to_f16(y) : f32_to_bf16(y);
      }
    }
  }
}

}  // namespace qattn

using namespace qattn;

template <int TM, int TN, int WM, int WN>
static int launch_linear(LinearParams& p, hipStream_t stream) {
  const int64_t tm = (p.M + TM - 1) / TM, tn = (p.N + TN - 1) / TN;
  QATTN_REQUIRE(tm * tn < ((int64_t)1 << 31), QATTN_ERR_SHAPE, "linear_int8: more than 2^31 tiles");
  p.tiles_m = (int)tm, p.tiles_n = (int)tn;
  const dim3 grid((unsigned)(tm * tn)), block(WM * WN * 64);
  if (p.act == QATTN_ACT_GELU_TANH) linear_int8_kernel<TM, TN, WM, WN, QATTN_ACT_GELU_TANH><<<grid, block, 0, stream>>>(p);
  else if (p.act == QATTN_ACT_SILU) linear_int8_kernel<TM, TN, WM, WN, QATTN_ACT_SILU><<<grid, block, 0, stream>>>(p);
  else linear_int8_kernel<TM, TN, WM, WN, QATTN_ACT_NONE><<<grid, block, 0, stream>>>(p);
  return check_launch("linear_int8");
}

extern "C" int qattn_linear_int8(const int8_t* x, int64_t x_pitch, const float* x_scale, const int8_t* w,
                                 int64_t w_pitch, const float* w_scale, const float* bias, void* out, int out_dtype,
                                 int64_t out_stride, int64_t M, int64_t N, int64_t K, int act, qattn_stream_t stream) {
  QATTN_REQUIRE(out_dtype >= QATTN_BF16 && out_dtype <= QATTN_F32, QATTN_ERR_DTYPE, "linear_int8: out has dtype code %d",
                out_dtype);
  QATTN_REQUIRE(M >= 0 && N >= 1 && M <= ((int64_t)1 << 31) && N <= (1 << 24), QATTN_ERR_SHAPE,
                "linear_int8: M = %lld, N = %lld", (long long)M, (long long)N);
  QATTN_REQUIRE(K >= 128 && K <= 131072 && K % 128 == 0, QATTN_ERR_SHAPE,
                "linear_int8: K = %lld must be a multiple of 128 up to 131072 (int32 sums)", (long long)K);
  QATTN_REQUIRE(act >= QATTN_ACT_NONE && act <= QATTN_ACT_SILU, QATTN_ERR_ARG, "linear_int8: act code %d", act);
  if (M == 0) return QATTN_OK;
  QATTN_REQUIRE(x && x_scale && w && w_scale && out, QATTN_ERR_ARG, "linear_int8: a null operand");
  QATTN_REQUIRE(x_pitch >= K && w_pitch >= K && x_pitch % 16 == 0 && w_pitch % 16 == 0 && x_pitch <= (1 << 22) &&
                    w_pitch <= (1 << 22),
                QATTN_ERR_STRIDE, "linear_int8: pitches %lld, %lld must be multiples of 16 from K to 2^22",
                (long long)x_pitch, (long long)w_pitch);
  QATTN_REQUIRE(out_stride >= N, QATTN_ERR_STRIDE, "linear_int8: out_stride %lld below N", (long long)out_stride);
  QATTN_REQUIRE(aligned16(x) && aligned16(w), QATTN_ERR_ALIGN, "linear_int8: x and w must be 16-byte aligned");
  QATTN_REQUIRE(reinterpret_cast<uintptr_t>(out) % (out_dtype == QATTN_F32 ? 4 : 2) == 0 &&
                    (reinterpret_cast<uintptr_t>(x_scale) | reinterpret_cast<uintptr_t>(w_scale) |
                     reinterpret_cast<uintptr_t>(bias)) % 4 == 0,
                QATTN_ERR_ALIGN, "linear_int8: out, a scale or the bias is misaligned");
  LinearParams p{x, x_pitch, x_scale, w, w_pitch, w_scale, bias, out, out_dtype, out_stride, M, N, (int)K, act, 0, 0};
  return launch_linear<128, 128, 2, 2>(p, (hipStream_t)stream);
}
