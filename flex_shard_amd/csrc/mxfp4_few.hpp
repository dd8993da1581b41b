// The product of few rows with a microscaled 4-bit weight: one token, or a few of
// every expert.  Bound by the weight's bytes, and where those are few by the chain
// of one launch: loads, products, sums.
//
// A workgroup owns 16 rows of the weight and all (at most 16 kTokenBlocks) rows of
// the activation; its waves take the contraction's steps of 256 columns in turn,
// so that what they load at a time is contiguous, straight from memory into the
// registers of the matrix instructions, and their sums are joined through LDS in a
// fixed order.  There is nothing to share through LDS: no weight is read twice.
#pragma once
#include "mxfp4_tiles.hpp"

namespace fsh {
namespace {

struct MxFewParams {
  const uint8_t* a;  // [a_rows][lda], or kQuantize: elements
  const uint8_t* as;
  const uint8_t* b;
  const uint8_t* bs;
  void* out;
  const void* bias;
  int64_t m, n, a_rows, b_rows, ld, ldo;  // ld: bytes of a quantized row
  int64_t cols, ldx;                      // kQuantize: columns and row stride of the activation, elements
  int32_t steps, tiles_n, waves;
  int32_t experts, top_k, vec;
  const int32_t* offsets;
  const int32_t* source;
};

constexpr int kFewRows = 16;  // of the weight, per workgroup
constexpr int kFewBatch = 4;  // steps that a wave has in flight
constexpr int kFewQuantize = FSH_MXFP4_FEW_ROWS;  // rows that a workgroup quantizes itself

// kQuantize: the activation comes as it is (at most kFewQuantize rows) and every
// workgroup quantizes it into its LDS: one launch instead of two.
template <int DT, int kTokenBlocks, bool kExperts, bool kQuantize>
__global__ __launch_bounds__(1024) void mxfp4_few_rows_kernel(const MxFewParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int r16 = lane & 15, group = lane >> 4;
  const int tile_n = static_cast<int>(blockIdx.x) % p.tiles_n, expert = static_cast<int>(blockIdx.x) / p.tiles_n;
  const int64_t n0 = static_cast<int64_t>(tile_n) * kFewRows;
  int64_t begin = 0, end = p.m, b_row0 = n0;
  if (kExperts) {
    begin = load_uniform(p.offsets + expert);
    end = expert < p.experts ? load_uniform(p.offsets + expert + 1) : p.m;
    if (expert == p.experts) {  // rows of no expert
      for (int64_t i = threadIdx.x; i < (end - begin) * kFewRows; i += blockDim.x)
        if (n0 + i % kFewRows < p.n) store_element<DT>(p.out, (begin + i / kFewRows) * p.ldo + n0 + i % kFewRows, 0.0f);
      return;
    }
    b_row0 = expert * p.n + n0;
  }
  const int64_t b_last = p.n - n0 < kFewRows ? p.n - n0 - 1 : kFewRows - 1;
  const int64_t b_row = b_row0 + (r16 < b_last ? r16 : b_last);
  const uint8_t* b_at = p.b + b_row * p.ld + group * 32;
  const uint8_t* bs_at = p.bs + b_row * 8 + group * 2;
  float* const sums = reinterpret_cast<float*>(few_lds);  // [waves][kTokenBlocks][16 rows][16 + 1]
  constexpr int kPitch = 17, kWaveSums = kTokenBlocks * 16 * kPitch;
  // kQuantize: rows of data, 16 bytes apart in the banks, then rows of scales
  uint8_t* const x_data = few_lds + p.waves * kWaveSums * 4;
  const int x_pitch = static_cast<int>(p.ld) + 16, s_pitch = 8 * p.steps;
  uint8_t* const x_scales = x_data + kFewQuantize * x_pitch;

  const auto load_b = [&](int step, u32x4 (&data)[2], int& scale) FSH_INLINE {
    const uint8_t* at = b_at + static_cast<int64_t>(step) * 128;
    data[0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
    data[1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at + 16));
    scale = *reinterpret_cast<const uint16_t*>(bs_at + static_cast<int64_t>(step) * p.b_rows * 8);
  };
  for (int64_t first = begin; first < end; first += 16 * kTokenBlocks) {
    f32x4 acc[kTokenBlocks];
    const uint8_t* a_at[kTokenBlocks];
    const uint8_t* as_at[kTokenBlocks];
#pragma unroll
    for (int t = 0; t < kTokenBlocks; ++t) {
      acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      int64_t row = first + 16 * t + r16;
      row = row < end ? row : end - 1;
      if (kQuantize) {
        a_at[t] = x_data + row * x_pitch + group * 32;
        as_at[t] = x_scales + row * s_pitch + group * 2;
      } else {
        if (kExperts && p.source) row = p.source[row] / p.top_k;
        a_at[t] = p.a + row * p.ld + group * 32;
        as_at[t] = p.as + row * 8 + group * 2;
      }
    }
    const int64_t as_step = kQuantize ? 8 : p.a_rows * 8;
    for (int s0 = wave; s0 < p.steps; s0 += kFewBatch * p.waves) {
      u32x4 bf[kFewBatch][2];
      int sb[kFewBatch];
#pragma unroll
      for (int i = 0; i < kFewBatch; ++i) {
        const int step = s0 + i * p.waves;
        load_b(step < p.steps ? step : s0, bf[i], sb[i]);
      }
      if (kQuantize && s0 == wave) {  // (every wave has a step; the weight's first loads are under way)
        const int pieces = p.steps * 32;  // of eight columns, per row
        for (int64_t i = threadIdx.x; i < (end - begin) * pieces; i += blockDim.x) {
          const int64_t row = i / pieces, col = (i - row * pieces) * 8;
          const Raw8<DT> raw = load_raw8<DT>(p.a + (row * p.ldx + col) * element_bytes<DT>(), p.cols - col, p.vec);
          float f[8];
          unpack_raw8<DT>(raw, f);
          uint32_t m = max_magnitude8(f);
          m = dpp_max_u32<0xB1, 0xF>(m);
          m = dpp_max_u32<0x4E, 0xF>(m);
          const uint32_t byte = mx_scale_byte(m);
          *reinterpret_cast<uint32_t*>(x_data + row * x_pitch + col / 2) = mx_quantize8(f, mx_scale(byte));
          if ((i & 3) == 0) x_scales[row * s_pitch + col / kMxBlock] = static_cast<uint8_t>(byte);
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < kFewBatch; ++i) {
        const int step = s0 + i * p.waves;
        if (step >= p.steps) break;
        const v8i32 b0 = {static_cast<int>(bf[i][0].x), static_cast<int>(bf[i][0].y), static_cast<int>(bf[i][0].z), static_cast<int>(bf[i][0].w), 0, 0, 0, 0};
        const v8i32 b1 = {static_cast<int>(bf[i][1].x), static_cast<int>(bf[i][1].y), static_cast<int>(bf[i][1].z), static_cast<int>(bf[i][1].w), 0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < kTokenBlocks; ++t) {
          const u32x4 x0 = *reinterpret_cast<const u32x4*>(a_at[t] + static_cast<int64_t>(step) * 128);
          const u32x4 x1 = *reinterpret_cast<const u32x4*>(a_at[t] + static_cast<int64_t>(step) * 128 + 16);
          const int sx = *reinterpret_cast<const uint16_t*>(as_at[t] + step * as_step);
          const v8i32 a0 = {static_cast<int>(x0.x), static_cast<int>(x0.y), static_cast<int>(x0.z), static_cast<int>(x0.w), 0, 0, 0, 0};
          const v8i32 a1 = {static_cast<int>(x1.x), static_cast<int>(x1.y), static_cast<int>(x1.z), static_cast<int>(x1.w), 0, 0, 0, 0};
          acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b0, a0, acc[t], 4, 4, 0, sb[i], 0, sx);
          acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b1, a1, acc[t], 4, 4, 1, sb[i], 1, sx);
        }
      }
    }
    // Lane (r, g) holds columns 4 g .. 4 g + 3 of row r of each block of the output.
#pragma unroll
    for (int t = 0; t < kTokenBlocks; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c) sums[wave * kWaveSums + (t * 16 + r16) * kPitch + 4 * group + c] = acc[t][c];
    __syncthreads();
    for (int i = threadIdx.x; i < kTokenBlocks * 256; i += blockDim.x) {
      const int64_t row = first + i / 16, col = n0 + i % 16;
      float sum = 0.0f;
      for (int w = 0; w < p.waves; ++w) sum += sums[w * kWaveSums + (i / 16) * kPitch + i % 16];
      if (row < end && col < p.n) {
        if (p.bias) sum += load_element<DT>(p.bias, col);
        store_element<DT>(p.out, row * p.ldo + col, sum);
      }
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace fsh
