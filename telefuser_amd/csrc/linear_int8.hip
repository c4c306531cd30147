// INT8 linear: out[m, n] = act(x_scale[m] * w_scale[n] * sum_k x[m, k] w[n, k] + bias[n]) on v_mfma_i32_16x16x64_i8.
//
// A workgroup computes TM x TN tiles, eight waves in a 2 x 4 grid.  The weight is the MFMA's A operand and the activation
// its B operand, so a lane of a 16 x 16 result holds one token and four channels.
//   * Instruction: with the matrix pipes busy the chip runs at its power limit (1.6 to 1.9 GHz), so energy per operation
//     decides.  16 x 16 x 64 does with less register traffic than 32 x 32 x 32 (its sum over K is twice as long):
//     75600 x 13824 x 5120 4.94 -> 4.23 ms, the same schedule otherwise.
//   * LDS: K advances by 128 bytes a stage, a whole line per row; both operands come by DMA into NB stages.  Row r holds
//     its 16-byte chunk c at position c ^ (r & 7) (the DMA's per-lane address does it), so the 16-byte fragment reads of
//     16 rows at one chunk meet no bank twice (counter SQ_LDS_BANK_CONFLICT: 0).
//   * Schedule: fragments are double-buffered in registers, one LDS read after each of the first MFMAs of a step, and the
//     order is frozen (sched_barrier): left to the compiler every read is followed by its wait (256 x 256: 1.86 -> 2.1
//     PFLOP/s).  One barrier a stage, before its last step: then every wave has this stage's last fragments in registers
//     and the next stage has landed, so its first fragments are read and the DMA of stage t + NB starts between the MFMAs
//     of that step.
//   * The large tile's workgroups stay and walk over tiles: the DMA runs ahead into the next tile while this one ends, so
//     its first stages load during the epilogue (32760 x 4608 x 1536: 224 -> 208 us).
//   * The weight's rows lie in LDS in an order that gives a lane 8 channels in a row from two results: one 16-byte store,
//     64 contiguous bytes for the four lanes of a token and its whole line in two stores (stores of 16 bytes at a stride
//     of 32: 245 us there).
//   * Scales and bias of a tile come into LDS by DMA with its first stage, four tiles deep.
// Tiles: 256 x 256, two stages (they fill 128 KiB); 128 x 128, three (512 x 5120 x 4096 17.6 us, with four 18.0), and 64 x
// 64, four (39606 x 64 x 3328 26.5 us, with three 28.1), where larger ones leave CUs without work.  A stage of the 128 x 128
// tile takes about 950 cycles for 512 of MFMA; reads, DMA and MFMAs overlap in part (without the MFMAs 32.4 of 34.5 us at
// 1560 x 1536 x 8960, without the LDS reads 29.4, without the DMA 25.8).  96 x 128 tiles, on 204 CUs there instead of 156,
// fetch a seventh more in all and take the same time.  The tiny tile fetches twice as much for its products, and runs one
// workgroup a CU as all of them do: two waves a SIMD is what the large tile's registers allow, and the attribute that says so
// holds for every instantiation, though this one's 54 registers and 67 KiB of LDS have room for two.  Rows past M or N lie
// behind the end of the buffer resource and read as zeros, and so does every stage past the last (the range check counts the
// scalar offset, and does not wrap where that is past the end).
// 75600 x 13824 x 5120 4.16 ms (2.57 PFLOP/s, the least of 30 launches 4.10 and 2.61), with GELU 4.23; one call after the
// other, 32760 x 1536 x 8960 365 us (2.47), 32760 x 4608 x 1536 212 us (2.19).  The power that a product takes depends on its
// values: launches apart from each other on codes spread evenly over the whole range take up to a third longer.
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
  v4i* part;         // split along K: [splits, tiles, 8 waves, NI * MJ, 64 lanes]
  int split_stages;  // stages of a split
};

constexpr int kLinK = 128;  // bytes of K per stage
// Tiles are walked down this many rows of them, then across: an XCD's 32 CUs share few rows of x and the weight passes by
// all XCDs at once (75600 x 13824 x 5120 in large tiles, group 1 / 2 / 3 / 4 / 8: 4.84 / 4.14 / 4.10 / 4.6 / 4.8 ms; 1560 x
// 1536 x 8960 in small ones, 1 / 3 / 5 / 13: 34.5 / 31.0 / 29.8 / 30.8 us).
constexpr int lin_group(int tile) { return tile == 256 ? 3 : 5; }

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

// A sum with its scales and bias.  The weight's scale comes first: the sum is a whole number below 2^31, so that the product
// neither overflows nor loses bits below the smallest normal value with any normal scale up to 2^96, and a row's scale, which
// large or tiny activations bring near either end, meets it where the result itself leaves the range.
__device__ __forceinline__ float scaled(int sum, float w_scale, float x_scale, float bias) {
  return fmaf((float)sum * w_scale, x_scale, bias);
}

// Waits until at most N of the wave's vector memory operations are under way, then for the other waves; the LDS reads
// too: a fragment read still in flight must not meet the next DMA into its stage.
template <int N>
__device__ __forceinline__ void wait_vm_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// Eight channels of a token, `left` of them within the row, in 16-byte stores at whatever alignment the row has (5234 x
// 3123 x 64, one element a store: 46 us, now 27).
__device__ __forceinline__ void store_out8(char* o, int dtype, int64_t left, const float (&y)[8]) {
  typedef v4u v4u_any __attribute__((aligned(2)));
  typedef v4u v4u_word __attribute__((aligned(4)));
  if (left >= 8) {
    if (dtype == QATTN_F32) {
      v4u_word* q = reinterpret_cast<v4u_word*>(o);
      q[0] = v4u{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])};
      q[1] = v4u{__float_as_uint(y[4]), __float_as_uint(y[5]), __float_as_uint(y[6]), __float_as_uint(y[7])};
      return;
    }
    v4u u;
    if (dtype == QATTN_FP16) {
#pragma unroll
      for (int e = 0; e < 4; e++) u[e] = pack_half2<true>(y[2 * e], y[2 * e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) u[e] = pack_half2<false>(y[2 * e], y[2 * e + 1]);
    }
    *reinterpret_cast<v4u_any*>(o) = u;
    return;
  }
#pragma unroll
  for (int e = 0; e < 7; e++)
    if (e < left) {
      if (dtype == QATTN_F32) reinterpret_cast<float*>(o)[e] = y[e];
      else reinterpret_cast<uint16_t*>(o)[e] = dtype == QATTN_FP16 ? f32_to_f16(y[e]) : f32_to_bf16(y[e]);
    }
}

template <int TM, int TN>
__device__ __forceinline__ void place_tile(const LinearParams& p, int slot, int tiles, int64_t& m0, int64_t& n0) {
  const uint32_t id = (uint32_t)xcd_remap(slot, tiles);
  constexpr uint32_t kGroup = lin_group(TM);
  const uint32_t per = kGroup * p.tiles_n, g = id / per, in = id - g * per;
  const uint32_t gm = min(kGroup, (uint32_t)p.tiles_m - g * kGroup);
  const uint32_t tn = in / gm;
  m0 = (int64_t)(g * kGroup + in - tn * gm) * TM;
  n0 = (int64_t)tn * TN;
}

// ACT = kSplit: a workgroup multiplies split_stages stages of a tile and leaves the int32 sums in p.part, each register of
// the wave as one 1 KiB line.
constexpr int kSplit = -1;
template <int TM, int TN, int WM, int NB, int ACT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void linear_int8_kernel(LinearParams p) {
  constexpr int kWaves = 8, WN = kWaves / WM;
  constexpr int NI = TN / WN / 16, MJ = TM / WM / 16;  // 16 x 16 results of a wave
  constexpr int kStage = (TM + TN) * kLinK;
  constexpr int IX = TM / 8 / kWaves, IW = TN / 8 / kWaves;  // DMA instructions of a wave and stage, 8 rows each
  constexpr int S = kLinK / 64, ND = IX + IW, NM = NI * MJ, NR = NI + MJ;
  constexpr int kVec = (2 * TN + TM) * 4;  // w_scale, bias and x_scale of a tile
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NB * kStage + 4 * kVec];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t base = lds_addr(lds);
  // the channel, within the tile, that row rho of the weight's part of a stage holds
  auto channel = [](int rho) {
    const int r = rho % (16 * NI), it = r / 16, a = r % 16;
    return rho - r + (it >> 1) * 32 + (a >> 2) * 8 + (it & 1) * 4 + (a & 3);
  };
  uint32_t vx[IX], vw[IW];
  const uint32_t chunk = (uint32_t)((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
  for (int i = 0; i < IX; i++) vx[i] = (uint32_t)(((i * kWaves + wave) * 8 + (lane >> 3)) * p.x_pitch) + chunk;
#pragma unroll
  for (int i = 0; i < IW; i++) vw[i] = (uint32_t)(channel((i * kWaves + wave) * 8 + (lane >> 3)) * p.w_pitch) + chunk;

  const int tiles = p.tiles_m * p.tiles_n;
  auto place = [&](int slot, int64_t& m0, int64_t& n0) { place_tile<TM, TN>(p, slot, tiles, m0, n0); };

  constexpr bool kWhole = ACT != kSplit;
  const int split = kWhole ? 0 : blockIdx.x / tiles;
  const int slot0 = kWhole ? blockIdx.x : blockIdx.x - split * tiles, stride = kWhole ? gridDim.x : tiles;
  const uint32_t k0 = kWhole ? 0 : (uint32_t)(split * p.split_stages * kLinK);
  const uint32_t k1 = kWhole ? (uint32_t)p.K : min((uint32_t)p.K, k0 + p.split_stages * kLinK);
  // where the DMA stands: the tile in slot fslot (the fn-th of this workgroup), byte fk of its rows
  int fslot = slot0, fn = 0;
  uint32_t fk = k0;
  v4u rx, rw;
  auto enter = [&]() {
    if (fslot >= tiles) {
      rx[2] = 0u, rw[2] = 0u;
      return;
    }
    int64_t m0, n0;
    place(fslot, m0, n0);
    const int64_t rm = min((int64_t)TM, p.M - m0), rn = min((int64_t)TN, p.N - n0);
    rx = make_rsrc(p.x + m0 * p.x_pitch, (uint32_t)((rm - 1) * p.x_pitch + p.K));
    rw = make_rsrc(p.w + n0 * p.w_pitch, (uint32_t)((rn - 1) * p.w_pitch + p.K));
    if constexpr (!kWhole) return;
    const v4u rs = make_rsrc(p.w_scale + n0, (uint32_t)rn * 4), rt = make_rsrc(p.x_scale + m0, (uint32_t)rm * 4);
    const v4u rb = make_rsrc(p.bias ? p.bias + n0 : p.w_scale, p.bias ? (uint32_t)rn * 4 : 0u);
    const uint32_t to = base + NB * kStage + (fn & 3) * kVec;
    for (int i = wave; i < TN / 64; i += kWaves) {
      lds_dma4(lane * 4, rs, i * 256, to + i * 256);
      lds_dma4(lane * 4, rb, i * 256, to + TN * 4 + i * 256);
    }
    for (int i = wave; i < TM / 64; i += kWaves) lds_dma4(lane * 4, rt, i * 256, to + TN * 8 + i * 256);
  };
  auto advance = [&]() {
    fk += kLinK;
    if (fk == k1) {
      fk = k0, fslot += stride, fn++;
      enter();
    }
  };
  auto fetch = [&](int d, uint32_t to) {
    if (d < IX) lds_dma16(vx[d], rx, fk, to + d * kWaves * 1024);
    else lds_dma16(vw[d - IX], rw, fk, to + TM * kLinK + (d - IX) * kWaves * 1024);
  };
  enter();
#pragma unroll
  for (int b = 0; b < NB; b++) {
    if (b) advance();
#pragma unroll
    for (int d = 0; d < ND; d++) fetch(d, base + b * kStage + wave * 1024);
  }
  wait_vm_barrier<NB == 2 ? 0 : (NB - 1) * ND>();

  const int wm = wave % WM, wn = wave / WM;
  const int row = lane & 15;
  const int swz = ((lane >> 4) ^ (row & 7)) * 16;
  const int xrow = (wm * (TM / WM) + row) * kLinK, wrow = (TM + wn * (TN / WN) + row) * kLinK;
  v4i a[2][NI], b[2][MJ];
  auto read = [&](uint32_t stage, int s, int r, v4i (&a)[NI], v4i (&b)[MJ]) {
    if (r < MJ) b[r] = *reinterpret_cast<const v4i*>(lds + stage + xrow + r * 16 * kLinK + (swz ^ (s * 64)));
    else a[r - MJ] = *reinterpret_cast<const v4i*>(lds + stage + wrow + (r - MJ) * 16 * kLinK + (swz ^ (s * 64)));
  };
#pragma unroll
  for (int r = 0; r < NR; r++) read(0, 0, r, a[0], b[0]);

  const int steps = (k1 - k0) / kLinK;
  uint32_t cur = 0;
  int n = 0;
  for (int slot = slot0; slot < tiles; slot += stride, n++) {
    v4i acc[NI][MJ];
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
      for (int j = 0; j < MJ; j++) acc[i][j] = v4i{};
    for (int t = 0; t < steps; t++) {
      const uint32_t nxt = NB == 2 ? cur ^ kStage : cur == (NB - 1) * kStage ? 0u : cur + kStage;
      advance();
#pragma unroll
      for (int s = 0; s < S; s++) {
        if (s == S - 1) {
          // stage t + 1 has landed when only the NB - 2 behind it are under way (more may lie behind: the wait is then
          // for more than it needs)
          __builtin_amdgcn_sched_barrier(0);
          wait_vm_barrier<(NB - 2) * ND>();
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int q = 0; q < NM; q++) {
          const int i = q / MJ, j = q % MJ;
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s & 1][i], b[s & 1][j], acc[i][j], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          constexpr int RQ = NM / 2 < NR ? NM / 2 : NR, DQ = NM / 2;  // MFMAs that carry reads, and the first with DMA
#pragma unroll
          for (int r = 0; r < NR; r++)
            if (r * RQ / NR == q) {
              if (s < S - 1) read(cur, s + 1, r, a[(s + 1) & 1], b[(s + 1) & 1]);
              else read(nxt, 0, r, a[(s + 1) & 1], b[(s + 1) & 1]);
              __builtin_amdgcn_sched_barrier(0);
            }
          if (s == S - 1)
#pragma unroll
            for (int d = 0; d < ND; d++)
              if (DQ + d * (NM - DQ) / ND == q) {
                fetch(d, base + cur + wave * 1024);
                __builtin_amdgcn_sched_barrier(0);
              }
        }
      }
      cur = nxt;
    }

    int64_t m0, n0;
    place(slot, m0, n0);
    if constexpr (!kWhole) {
      v4i* to = p.part + (((int64_t)split * tiles + slot) * kWaves + wave) * (NM * 64) + lane;
#pragma unroll
      for (int j = 0; j < MJ; j++)
        if (m0 + wm * (TM / WM) + j * 16 < p.M)
#pragma unroll
          for (int i = 0; i < NI; i++) to[(j * NI + i) * 64] = acc[i][j];
      continue;
    }
    const float* vec = reinterpret_cast<const float*>(lds + NB * kStage + (n & 3) * kVec);
    const int cl = wn * (TN / WN) + (lane >> 4) * 8, ml = wm * (TM / WM) + row;
    const int es = p.out_dtype == QATTN_F32 ? 4 : 2;
    char* out = static_cast<char*>(p.out) + ((m0 + ml) * p.out_stride + n0 + cl) * es;
#pragma unroll
    for (int j = 0; j < MJ; j++, out += p.out_stride * 16 * es) {
      if (m0 + ml + j * 16 >= p.M) continue;
      const float sx = vec[2 * TN + ml + j * 16];
#pragma unroll
      for (int i = 0; i < NI; i += 2) {
        const v4f* sw = reinterpret_cast<const v4f*>(vec + cl + 16 * i);
        const v4f* bi = reinterpret_cast<const v4f*>(vec + TN + cl + 16 * i);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
          y[e] = activate<ACT>(scaled(acc[i + e / 4][j][e % 4], sw[e / 4][e % 4], sx, bi[e / 4][e % 4]));
        store_out8(out + 16 * i * es, p.out_dtype, p.N - n0 - cl - 16 * i, y);
      }
    }
  }
  // the DMA of the stages past the last still writes (zeros) into this workgroup's LDS
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The sums of the splits of a tile, and what the tile kernel does with them at its end.  A wave takes what one wave of the
// tile kernel left of 16 tokens.
template <int TM, int TN, int WM, int ACT>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearParams p, int splits) {
  constexpr int WN = 8 / WM, NI = TN / WN / 16, MJ = TM / WM / 16;
  static_assert(NI == 2);
  const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int tiles = p.tiles_m * p.tiles_n;
  const int j = id % MJ, wave = id / MJ % 8, slot = id / (MJ * 8);
  if (slot >= tiles) return;
  int64_t m0, n0;
  place_tile<TM, TN>(p, slot, tiles, m0, n0);
  m0 += wave % WM * (TM / WM) + j * 16;
  n0 += wave / WM * (TN / WN) + (lane >> 4) * 8;
  if (m0 >= p.M) return;
  const v4i* from = p.part + ((int64_t)slot * 8 + wave) * (NI * MJ * 64) + j * NI * 64 + lane;
  v4i sum[NI]{};
#pragma unroll 4
  for (int s = 0; s < splits; s++)
#pragma unroll
    for (int i = 0; i < NI; i++) sum[i] += from[(int64_t)s * tiles * 8 * NI * MJ * 64 + i * 64];
  const int64_t m = m0 + (lane & 15), left = p.N - n0;
  if (m >= p.M) return;
  const float sx = p.x_scale[m];
  const int es = p.out_dtype == QATTN_F32 ? 4 : 2;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; e++)
    y[e] = e < left ? activate<ACT>(scaled(sum[e / 4][e % 4], p.w_scale[n0 + e], sx, p.bias ? p.bias[n0 + e] : 0.0f)) : 0.0f;
  store_out8(static_cast<char*>(p.out) + (m * p.out_stride + n0) * es, p.out_dtype, left, y);
}

// ------------------------------------------------------------------------------------------------
// few tokens
// ------------------------------------------------------------------------------------------------
// Up to 16 tokens the weight is what there is to read.  A workgroup takes 16 NI channels and all tokens; its eight waves
// take turns along K, 128 bytes a turn, and read the weight's fragments straight from global memory, whole lines, several
// turns ahead.  Their sums meet in LDS.  X: a floating x is quantized by every workgroup for itself, with the code of the
// row quantizer and so to the same bits, which saves the quantizer's launch and the rows' way through memory; for up to
// kFewValues values, where that costs less than the launch (channels x values: 9216 x 1 x 1536 6.1 us, against 5.5 from INT8
// rows and 2.7 for the quantizer; 13824 x 3 x 5120 16.9 against 14.3 and 3.7, 4.2 TB/s of weight).  32 channels a workgroup
// where that gives one to every CU.
constexpr int kFewRows = 16;
constexpr int kFewValues = 16384;

struct FewParams {
  LinearParams lin;  // x and x_scale: the INT8 rows (X < 0)
  const void* x;     // the floating rows, L of them to a batch entry
  int64_t xb, xl;
  int L, cols;
  bool vec;  // four values in a load
};

template <int X>
__device__ __forceinline__ void few_values4(const void* x, int64_t at, int left, bool vec, float (&v)[4]) {
  if constexpr (X == QATTN_F32) {
    const float* q = static_cast<const float*>(x) + at;
    if (vec && left >= 4) {
      const v4f r = *reinterpret_cast<const v4f*>(q);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = r[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = e < left ? q[e] : 0.0f;
    }
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(x) + at;
    uint16_t h[4];
    if (vec && left >= 4) {
      const v2u r = *reinterpret_cast<const v2u*>(q);
      __builtin_memcpy(h, &r, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) h[e] = e < left ? q[e] : (uint16_t)0;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = half_to_f32<X == QATTN_FP16>(h[e]);
  }
}

// X: element type of the floating x, or -1 for INT8 rows.
template <int NI, int X, int ACT>
__global__ __launch_bounds__(512) void linear_few_kernel(FewParams f) {
  const LinearParams& p = f.lin;
  constexpr int kWaves = 8, kAhead = 4 / NI;
  __shared__ __attribute__((aligned(16))) v4i part[kWaves][NI][64];
  __shared__ __attribute__((aligned(16))) uint8_t rows[X < 0 ? 16 : kFewValues + 16 * 16];  // 16 bytes apart: banks
  __shared__ uint32_t tops[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 16 * NI;
  const int M = (int)p.M, K = p.K;

  // the weight's first lines are under way while the rows are quantized
  const int8_t* w[NI];
#pragma unroll
  for (int i = 0; i < NI; i++) w[i] = p.w + min(n0 + i * 16 + (lane & 15), p.N - 1) * p.w_pitch + (lane >> 4) * 16;
  v4i a[kAhead][NI][2];
  auto load = [&](int k, v4i (&a)[NI][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; i++) {
      a[i][0] = *reinterpret_cast<const v4i*>(w[i] + k);
      a[i][1] = *reinterpret_cast<const v4i*>(w[i] + k + 64);
    }
  };
  constexpr int kTurn = kWaves * kLinK;
#pragma unroll
  for (int i = 0; i < kAhead; i++)
    if (wave * kLinK + i * kTurn < K) load(wave * kLinK + i * kTurn, a[i]);
  // and the scales of the four channels a lane ends with
  const int64_t c = n0 + wave * 16 + (lane >> 4) * 4;
  float sw[4], bias[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const bool in = wave < NI && c + e < p.N;
    sw[e] = in ? p.w_scale[c + e] : 0.0f;
    bias[e] = in && p.bias ? p.bias[c + e] : 0.0f;
  }

  const int pitch = K + 16;
  if constexpr (X >= 0) {
    // words of four values; 32 of them lie in one row.  The quotients are small: (n + 1/2) / d lies further from an integer
    // than float32 is off.
    constexpr int kWords = kFewValues / 4 / 512;
    const int per = K / 4, words = M * per;
    const float of_per = __builtin_amdgcn_rcpf((float)per), of_l = __builtin_amdgcn_rcpf((float)f.L);
    float v[kWords][4];
    int at[kWords], of[kWords];
    if (threadIdx.x < 16) tops[threadIdx.x] = 0;
#pragma unroll
    for (int i = 0; i < kWords; i++) {
      if (i * 512 >= words) break;
      const int id = threadIdx.x + i * 512;
      of[i] = id < words ? (int)(((float)id + 0.5f) * of_per) : -1;
      if (of[i] < 0) continue;
      const int c = (id - of[i] * per) * 4, b = (int)(((float)of[i] + 0.5f) * of_l);
      at[i] = of[i] * pitch + c;
      few_values4<X>(f.x, b * f.xb + (of[i] - b * f.L) * f.xl + c, f.cols - c, f.vec, v[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWords; i++) {
      if (i * 512 >= words) break;
      uint32_t top = 0;
      if (of[i] >= 0)
#pragma unroll
        for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
      top = half_wave_top(top);
      if ((lane & 31) == 31 && of[i] >= 0) atomicMax(&tops[of[i]], top);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWords; i++) {
      if (i * 512 >= words) break;
      if (of[i] >= 0)
        *reinterpret_cast<uint32_t*>(rows + at[i]) = RowQuant(tops[of[i]]).code4(v[i][0], v[i][1], v[i][2], v[i][3]);
    }
    __syncthreads();
  }
  const int64_t m = min(lane & 15, M - 1);  // tokens past the last repeat it and are dropped
  const int8_t* x = X >= 0 ? reinterpret_cast<const int8_t*>(rows) + m * pitch + (lane >> 4) * 16
                           : p.x + m * p.x_pitch + (lane >> 4) * 16;
  v4i acc[NI]{};
  for (int k0 = wave * kLinK; k0 < K; k0 += kAhead * kTurn) {
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
      const int k = k0 + i * kTurn;
      if (k < K) {
        const v4i b0 = *reinterpret_cast<const v4i*>(x + k), b1 = *reinterpret_cast<const v4i*>(x + k + 64);
#pragma unroll
        for (int n = 0; n < NI; n++) {
          acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i][n][0], b0, acc[n], 0, 0, 0);
          acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i][n][1], b1, acc[n], 0, 0, 0);
        }
        if (k + kAhead * kTurn < K) load(k + kAhead * kTurn, a[i]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NI; n++) part[wave][n][lane] = acc[n];
  __syncthreads();
  // a wave finishes 16 channels: four a lane
  if (wave >= NI || (lane & 15) >= M) return;
  v4i sum = part[0][wave][lane];
#pragma unroll
  for (int i = 1; i < kWaves; i++) sum += part[i][wave][lane];
  const float sx = X >= 0 ? RowQuant(tops[m]).scale : p.x_scale[m];
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (c + e < p.N) {
      const float y = activate<ACT>(scaled(sum[e], sw[e], sx, bias[e]));
      const int64_t at = m * p.out_stride + c + e;
      if (p.out_dtype == QATTN_F32) static_cast<float*>(p.out)[at] = y;
      else static_cast<uint16_t*>(p.out)[at] = p.out_dtype == QATTN_FP16 ? f32_to_f16(y) : f32_to_bf16(y);
    }
}

}  // namespace qattn

using namespace qattn;

template <int NI, int X>
static int launch_few(const FewParams& f, hipStream_t stream) {
  const dim3 grid((unsigned)((f.lin.N + 16 * NI - 1) / (16 * NI))), block(512);
  if (f.lin.act == QATTN_ACT_GELU_TANH) linear_few_kernel<NI, X, QATTN_ACT_GELU_TANH><<<grid, block, 0, stream>>>(f);
  else if (f.lin.act == QATTN_ACT_SILU) linear_few_kernel<NI, X, QATTN_ACT_SILU><<<grid, block, 0, stream>>>(f);
  else linear_few_kernel<NI, X, QATTN_ACT_NONE><<<grid, block, 0, stream>>>(f);
  return check_launch("linear_int8");
}
template <int X>
static int launch_few(const FewParams& f, hipStream_t stream) {
  // 32 channels a workgroup where that still gives one to every CU
  return f.lin.N >= 32 * 256 ? launch_few<2, X>(f, stream) : launch_few<1, X>(f, stream);
}

template <int TM, int TN, int WM, int NB>
static int launch_linear(LinearParams& p, int workgroups, hipStream_t stream) {
  p.tiles_m = (int)((p.M + TM - 1) / TM), p.tiles_n = (int)((p.N + TN - 1) / TN);
  const dim3 grid((unsigned)std::min(p.tiles_m * p.tiles_n, workgroups)), block(512);
  if (p.act == QATTN_ACT_GELU_TANH) linear_int8_kernel<TM, TN, WM, NB, QATTN_ACT_GELU_TANH><<<grid, block, 0, stream>>>(p);
  else if (p.act == QATTN_ACT_SILU) linear_int8_kernel<TM, TN, WM, NB, QATTN_ACT_SILU><<<grid, block, 0, stream>>>(p);
  else linear_int8_kernel<TM, TN, WM, NB, QATTN_ACT_NONE><<<grid, block, 0, stream>>>(p);
  return check_launch("linear_int8");
}

constexpr int kLinCus = 256;

static int64_t tiles_of(int64_t M, int64_t N, int64_t t) { return ((M + t - 1) / t) * ((N + t - 1) / t); }

// The checks that both entries share, and the parameters.
static int linear_params(LinearParams& p, const int8_t* w, int64_t w_pitch, const float* w_scale, const float* bias,
                         void* out, int out_dtype, int64_t out_stride, int64_t M, int64_t N, int64_t K, int act) {
  QATTN_REQUIRE(out_dtype >= QATTN_BF16 && out_dtype <= QATTN_F32, QATTN_ERR_DTYPE, "linear_int8: out has dtype code %d",
                out_dtype);
  QATTN_REQUIRE(M >= 0 && N >= 1 && M <= ((int64_t)1 << 31) && N <= (1 << 24), QATTN_ERR_SHAPE,
                "linear_int8: M = %lld, N = %lld", (long long)M, (long long)N);
  QATTN_REQUIRE(K >= 128 && K <= 131072 && K % 128 == 0, QATTN_ERR_SHAPE,
                "linear_int8: K = %lld must be a multiple of 128 up to 131072 (int32 sums)", (long long)K);
  QATTN_REQUIRE(act >= QATTN_ACT_NONE && act <= QATTN_ACT_SILU, QATTN_ERR_ARG, "linear_int8: act code %d", act);
  if (M == 0) return QATTN_OK;
  QATTN_REQUIRE(tiles_of(M, N, 64) < ((int64_t)1 << 23), QATTN_ERR_SHAPE, "linear_int8: more than 2^23 tiles of 64 x 64");
  QATTN_REQUIRE(w && w_scale && out, QATTN_ERR_ARG, "linear_int8: a null operand");
  QATTN_REQUIRE(w_pitch >= K && w_pitch % 16 == 0 && w_pitch <= (1 << 22), QATTN_ERR_STRIDE,
                "linear_int8: w_pitch %lld must be a multiple of 16 from K to 2^22", (long long)w_pitch);
  QATTN_REQUIRE(out_stride >= N, QATTN_ERR_STRIDE, "linear_int8: out_stride %lld below N", (long long)out_stride);
  QATTN_REQUIRE(aligned16(w), QATTN_ERR_ALIGN, "linear_int8: w must be 16-byte aligned");
  QATTN_REQUIRE(reinterpret_cast<uintptr_t>(out) % (out_dtype == QATTN_F32 ? 4 : 2) == 0 &&
                    (reinterpret_cast<uintptr_t>(w_scale) | reinterpret_cast<uintptr_t>(bias)) % 4 == 0,
                QATTN_ERR_ALIGN, "linear_int8: out, a scale or the bias is misaligned");
  p = LinearParams{nullptr, 0, nullptr, w, w_pitch, w_scale, bias, out, out_dtype, out_stride, M, N, (int)K, act, 0, 0, nullptr, 0};
  return QATTN_OK;
}

// Which kernel, by estimated microseconds: of a stage and of a tile's beginning and end, times the rounds of the chip; a
// split along K writes its int32 sums and the join reads them (5 TB/s, and 3 us for its launch).  Measured, large / small /
// tiny tile: 3000 x 3000 x 3000 38 / 42 / -, 32760 x 4608 x 1536 208 / 338 / -, 1560 x 1536 x 8960 85 / 30 / 46, 512 x 5120 x
// 4096 43 / 17 / 26, 600 x 1536 x 1536 19 / 8.3 / 6.1, 777 x 999 x 1027 - / 9.7 / 5.7, 1000 x 640 x 4096 - / 15.6 / 9.6; all
// with one workgroup a CU, which the rounds count too.
enum LinearKernel { LINEAR_FEW, LINEAR_LARGE, LINEAR_SMALL, LINEAR_TINY };
struct LinearPlan {
  LinearKernel kernel;
  int splits, split_stages;
};
static int64_t plan_tiles(const LinearPlan& plan, int64_t M, int64_t N) {
  return tiles_of(M, N, plan.kernel == LINEAR_SMALL ? 128 : 64);
}
static LinearPlan plan_linear(int64_t M, int64_t N, int64_t K) {
  if (M <= kFewRows) return {LINEAR_FEW, 1, 0};
  const int64_t stages = K / kLinK;
  auto cost = [](int64_t workgroups, int64_t stages, double stage, double ends) {
    return (double)((workgroups + kLinCus - 1) / kLinCus) * (stage * stages + ends);
  };
  LinearPlan best{LINEAR_LARGE, 1, (int)stages};
  double least = cost(tiles_of(M, N, 256), stages, 1.3, 5.0);
  for (const LinearKernel kernel : {LINEAR_SMALL, LINEAR_TINY}) {
    const double stage = kernel == LINEAR_SMALL ? 0.42 : 0.18, ends = kernel == LINEAR_SMALL ? 3.5 : 3.1;
    const int64_t tiles = tiles_of(M, N, kernel == LINEAR_SMALL ? 128 : 64);
    const double whole = cost(tiles, stages, stage, ends);
    if (whole < least) least = whole, best = {kernel, 1, (int)stages};
    for (int64_t s = 2; s <= 16 && s * tiles <= 2 * kLinCus && s * 4 <= stages; s++) {
      const int64_t per = (stages + s - 1) / s, splits = (stages + per - 1) / per;
      const double t = (cost(splits * tiles, per, stage, ends) + 3 + 8.0 * splits * M * N / 5e6) / 0.9;
      if (t < least) least = t, best = {kernel, (int)splits, (int)per};
    }
  }
  return best;
}
static size_t split_bytes(const LinearPlan& plan, int64_t M, int64_t N) {
  const size_t tile = plan.kernel == LINEAR_SMALL ? 128 : 64;
  return plan.splits > 1 ? plan.splits * plan_tiles(plan, M, N) * tile * tile * 4 : 0;
}

template <int TM, int TN, int WM, int NB>
static int launch_split(LinearParams& p, const LinearPlan& plan, void* workspace, hipStream_t stream) {
  p.part = static_cast<v4i*>(workspace), p.split_stages = plan.split_stages;
  p.tiles_m = (int)((p.M + TM - 1) / TM), p.tiles_n = (int)((p.N + TN - 1) / TN);
  const int tiles = p.tiles_m * p.tiles_n;
  linear_int8_kernel<TM, TN, WM, NB, kSplit><<<dim3((unsigned)(tiles * plan.splits)), dim3(512), 0, stream>>>(p);
  if (int rc = check_launch("linear_int8")) return rc;
  // one wave for each of a tile's eight and each of its groups of 16 tokens
  const dim3 grid((unsigned)(tiles * 2 * (TM / WM / 16))), block(256);
  if (p.act == QATTN_ACT_GELU_TANH) linear_join_kernel<TM, TN, WM, QATTN_ACT_GELU_TANH><<<grid, block, 0, stream>>>(p, plan.splits);
  else if (p.act == QATTN_ACT_SILU) linear_join_kernel<TM, TN, WM, QATTN_ACT_SILU><<<grid, block, 0, stream>>>(p, plan.splits);
  else linear_join_kernel<TM, TN, WM, QATTN_ACT_NONE><<<grid, block, 0, stream>>>(p, plan.splits);
  return check_launch("linear_int8");
}

static int run_linear(LinearParams& p, const LinearPlan& plan, void* workspace, hipStream_t stream) {
  if (plan.kernel == LINEAR_FEW) return launch_few<-1>(FewParams{p, nullptr, 0, 0, 1, 0, false}, stream);
  if (plan.kernel == LINEAR_LARGE) return launch_linear<256, 256, 2, 2>(p, kLinCus, stream);
  if (plan.splits > 1)
    return plan.kernel == LINEAR_SMALL ? launch_split<128, 128, 2, 3>(p, plan, workspace, stream)
                                       : launch_split<64, 64, 4, 4>(p, plan, workspace, stream);
  return plan.kernel == LINEAR_SMALL ? launch_linear<128, 128, 2, 3>(p, INT32_MAX, stream)
                                     : launch_linear<64, 64, 4, 4>(p, INT32_MAX, stream);
}

static int check_workspace(const void* workspace, size_t bytes, size_t need) {
  QATTN_REQUIRE(!need || (workspace && bytes >= need && aligned16(workspace)), QATTN_ERR_WORKSPACE,
                "linear_int8: workspace of %zu bytes, %zu needed (16-byte aligned)", bytes, need);
  return QATTN_OK;
}

extern "C" size_t qattn_linear_int8_workspace_size(int64_t M, int64_t N, int64_t K) {
  return M > 0 && N > 0 && K > 0 ? split_bytes(plan_linear(M, N, K), M, N) : 0;
}

extern "C" int qattn_linear_int8(const int8_t* x, int64_t x_pitch, const float* x_scale, const int8_t* w,
                                 int64_t w_pitch, const float* w_scale, const float* bias, void* out, int out_dtype,
                                 int64_t out_stride, int64_t M, int64_t N, int64_t K, int act, void* workspace,
                                 size_t workspace_bytes, qattn_stream_t stream) {
  LinearParams p;
  if (int rc = linear_params(p, w, w_pitch, w_scale, bias, out, out_dtype, out_stride, M, N, K, act)) return rc;
  if (M == 0) return QATTN_OK;
  QATTN_REQUIRE(x && x_scale, QATTN_ERR_ARG, "linear_int8: a null operand");
  QATTN_REQUIRE(x_pitch >= K && x_pitch % 16 == 0 && x_pitch <= (1 << 22), QATTN_ERR_STRIDE,
                "linear_int8: x_pitch %lld must be a multiple of 16 from K to 2^22", (long long)x_pitch);
  QATTN_REQUIRE(aligned16(x) && reinterpret_cast<uintptr_t>(x_scale) % 4 == 0, QATTN_ERR_ALIGN,
                "linear_int8: x or x_scale is misaligned");
  p.x = x, p.x_pitch = x_pitch, p.x_scale = x_scale;
  const LinearPlan plan = plan_linear(M, N, K);
  if (int rc = check_workspace(workspace, workspace_bytes, split_bytes(plan, M, N))) return rc;
  return run_linear(p, plan, workspace, (hipStream_t)stream);
}

static bool few_values(int64_t M, int64_t K) { return M <= kFewRows && M * K <= kFewValues; }
// the INT8 rows, their scales, and the split sums from a multiple of 16 on
static size_t rows_bytes(int64_t M, int64_t K) { return (size_t)(M * K + M * 4 + 15) / 16 * 16; }

extern "C" size_t qattn_linear_int8_rows_workspace_size(int64_t M, int64_t N, int64_t cols) {
  if (M <= 0 || N <= 0 || cols <= 0) return 0;
  const int64_t K = (cols + 127) / 128 * 128;
  return few_values(M, K) ? 0 : rows_bytes(M, K) + split_bytes(plan_linear(M, N, K), M, N);
}

extern "C" int qattn_linear_int8_rows(const void* x, int x_dtype, int64_t x_sb, int64_t x_sl, int64_t B, int64_t L,
                                      int64_t cols, const int8_t* w, int64_t w_pitch, const float* w_scale,
                                      const float* bias, void* out, int out_dtype, int64_t out_stride, int64_t N, int act,
                                      void* workspace, size_t workspace_bytes, qattn_stream_t stream) {
  QATTN_REQUIRE(x_dtype >= QATTN_BF16 && x_dtype <= QATTN_F32, QATTN_ERR_DTYPE, "linear_int8: x has dtype code %d", x_dtype);
  QATTN_REQUIRE(cols >= 1 && cols <= 131072 && B >= 0 && L >= 0 && (B == 0 || L <= ((int64_t)1 << 31) / B),
                QATTN_ERR_SHAPE, "linear_int8: x of %lld x %lld rows of %lld", (long long)B, (long long)L, (long long)cols);
  const int64_t M = B * L, K = (cols + 127) / 128 * 128;
  LinearParams p;
  if (int rc = linear_params(p, w, w_pitch, w_scale, bias, out, out_dtype, out_stride, M, N, K, act)) return rc;
  if (M == 0) return QATTN_OK;
  QATTN_REQUIRE(x, QATTN_ERR_ARG, "linear_int8: a null operand");
  QATTN_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == QATTN_F32 ? 4 : 2) == 0, QATTN_ERR_ALIGN,
                "linear_int8: x is misaligned");
  if (few_values(M, K)) {
    const int64_t xs = x_dtype == QATTN_F32 ? 4 : 2, xb = B > 1 ? x_sb : 0, xl = L > 1 ? x_sl : 0;
    const bool vec = (reinterpret_cast<uintptr_t>(x) | xb * xs | xl * xs) % (4 * xs) == 0;
    const FewParams f{p, x, xb, xl, (int)L, (int)cols, vec};
    return x_dtype == QATTN_F32 ? launch_few<QATTN_F32>(f, (hipStream_t)stream)
           : x_dtype == QATTN_FP16 ? launch_few<QATTN_FP16>(f, (hipStream_t)stream)
                                   : launch_few<QATTN_BF16>(f, (hipStream_t)stream);
  }
  const LinearPlan plan = plan_linear(M, N, K);
  if (int rc = check_workspace(workspace, workspace_bytes, rows_bytes(M, K) + split_bytes(plan, M, N))) return rc;
  qattn_block_norm_args q{};
  q.size = sizeof(q);
  q.x = x, q.x_dtype = x_dtype, q.x_sb = x_sb, q.x_sl = x_sl, q.B = B, q.L = L, q.C = cols;
  q.z = workspace, q.z_dtype = QATTN_I8, q.z_pitch = K, q.z_scale = reinterpret_cast<float*>(static_cast<char*>(workspace) + M * K);
  if (int rc = qattn_block_norm(&q, stream)) return rc;
  p.x = static_cast<const int8_t*>(workspace), p.x_pitch = K, p.x_scale = q.z_scale;
  return run_linear(p, plan, static_cast<char*>(workspace) + rows_bytes(M, K), (hipStream_t)stream);
}
