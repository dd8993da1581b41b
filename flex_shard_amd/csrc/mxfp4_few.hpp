// The product of few rows with a microscaled 4-bit weight: a token, or a few.
// Bound by the weight's bytes, and where those are few by the chain of one launch:
// loads, products, sums.  One row: 14336, k 4096 (31 MB) 8.5 to 8.8 us, 3.6 TB/s;
// 4096, k 4096 4.1 to 4.3; 4096, k 14336 9.6; 1024, k 4096 3.2 to 3.5.
//
// A workgroup owns 16 rows of the weight and all (at most 16) rows of the
// activation; its waves take the contraction's steps of 256 columns in turn,
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
  int32_t steps, waves, vec;
  int32_t bias_f32;  // the bias is fp32, whatever the output
};

constexpr int kFewRows = 16;  // of the weight, per workgroup
constexpr int kFewBatch = 2;  // steps that a wave requests together
constexpr int kFewMaxWaves = 8;
constexpr int kFewQuantize = FSH_MXFP4_FEW_ROWS;  // rows that a workgroup quantizes itself

// A lane's part of 16 rows and a step of 256 columns: row lane & 15, in half h the
// 32 columns g + 4 h of the 8 times 32 (g = lane / 16; 64 contiguous bytes of a row
// per load), and the row's word of scales.
struct MxFewFragment {
  u32x4 half[2];
  u32x2 scales;
};
__device__ __forceinline__ v8i32 few_operand(const u32x4& v) {
  return v8i32{static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w), 0, 0, 0, 0};
}

// kQuantize: the activation comes as it is (at most kFewQuantize rows) and every
// workgroup quantizes it into its LDS: one launch instead of two.
template <int DT, bool kQuantize>
__global__ __launch_bounds__(64 * kFewMaxWaves) void mxfp4_few_rows_kernel(const MxFewParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int r16 = lane & 15, group = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kFewRows;
  const int64_t b_last = p.n - n0 < kFewRows ? p.n - n0 - 1 : kFewRows - 1;
  const int64_t b_row = n0 + (r16 < b_last ? r16 : b_last);
  const uint8_t* b_at = p.b + b_row * p.ld + group * 16;
  const uint8_t* bs_at = p.bs + b_row * 8;
  float* const sums = reinterpret_cast<float*>(few_lds);  // [waves][16 rows][16 + 1]
  constexpr int kPitch = 17, kWaveSums = 16 * kPitch;
  // kQuantize: rows of data, 16 bytes apart in the banks, then rows of scales
  uint8_t* const x_data = few_lds + p.waves * kWaveSums * 4;
  const int x_pitch = static_cast<int>(p.ld) + 16, s_pitch = 8 * p.steps;
  uint8_t* const x_scales = x_data + kFewQuantize * x_pitch;
  const uint32_t pick = 0x0C0C0000u | static_cast<uint32_t>((4 + group) << 8) | static_cast<uint32_t>(group);  // scale bytes g and 4 + g
  const auto scales_of = [&](const u32x2& word) FSH_INLINE { return static_cast<int>(__builtin_amdgcn_perm(word.y, word.x, pick)); };

  const int64_t row = r16 < p.m ? r16 : p.m - 1;
  const uint8_t* const a_at = kQuantize ? x_data + row * x_pitch + group * 16 : p.a + row * p.ld + group * 16;
  const uint8_t* const as_at = kQuantize ? x_scales + row * s_pitch : p.as + row * 8;
  const int64_t as_step = kQuantize ? 8 : p.a_rows * 8, bs_step = p.b_rows * 8;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  struct Batch {
    MxFewFragment a[kFewBatch], b[kFewBatch];
  };
  // Steps s, s + waves, ..; steps past the last are the last one again (and not used).
  const auto load_a = [&](MxFewFragment& to, int step) FSH_INLINE {
    const uint8_t* at = a_at + static_cast<int64_t>(step) * 128;
    to.half[0] = *reinterpret_cast<const u32x4*>(at);
    to.half[1] = *reinterpret_cast<const u32x4*>(at + 64);
    to.scales = *reinterpret_cast<const u32x2*>(as_at + step * as_step);
  };
  const auto load = [&](Batch& batch, int s) FSH_INLINE {
#pragma unroll
    for (int i = 0; i < kFewBatch; ++i) {
      const int step = s + i * p.waves < p.steps ? s + i * p.waves : p.steps - 1;
      const uint8_t* at = b_at + static_cast<int64_t>(step) * 128;
      batch.b[i].half[0] = *reinterpret_cast<const u32x4*>(at);
      batch.b[i].half[1] = *reinterpret_cast<const u32x4*>(at + 64);
      batch.b[i].scales = *reinterpret_cast<const u32x2*>(bs_at + step * bs_step);
      if (!kQuantize) load_a(batch.a[i], step);
    }
  };
  const auto multiply = [&](Batch& batch, int s) FSH_INLINE {
#pragma unroll
    for (int i = 0; i < kFewBatch; ++i) {
      const int step = s + i * p.waves;
      if (step >= p.steps) break;
      if (kQuantize) load_a(batch.a[i], step);
      const int sb = scales_of(batch.b[i].scales), sa = scales_of(batch.a[i].scales);
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(few_operand(batch.b[i].half[0]), few_operand(batch.a[i].half[0]), acc, 4, 4, 0,
                                                             sb, 0, sa);
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(few_operand(batch.b[i].half[1]), few_operand(batch.a[i].half[1]), acc, 4, 4, 1,
                                                             sb, 1, sa);
    }
  };
  const int stride = kFewBatch * p.waves;
  Batch even, odd;
  load(even, wave);  // (every wave has a step)
  if (wave + stride < p.steps) load(odd, wave + stride);
  if (kQuantize) {
    const int pieces = p.steps * 32;  // of eight columns, per row
    const int total = static_cast<int>(p.m) * pieces;
    for (int i0 = threadIdx.x; i0 < total; i0 += 4 * blockDim.x) {  // whole fours of lanes, a run each
      Raw8<DT> raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * static_cast<int>(blockDim.x), x_row = i / pieces, col = (i - x_row * pieces) * 8;
        raw[u] = load_raw8<DT>(p.a + (x_row * p.ldx + col) * element_bytes<DT>(), i < total ? p.cols - col : 0, p.vec);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * static_cast<int>(blockDim.x), x_row = i / pieces, col = (i - x_row * pieces) * 8;
        uint32_t m = max_magnitude8(raw[u]);
        m = dpp_max_u32<0xB1, 0xF>(m);
        m = dpp_max_u32<0x4E, 0xF>(m);
        const uint32_t byte = mx_scale_byte(magnitude_bits_to_f32<DT>(m));
        if (i >= total) break;
        *reinterpret_cast<uint32_t*>(x_data + x_row * x_pitch + col / 2) = mx_quantize8(raw[u], mx_scale(byte));
        if ((i & 3) == 0) x_scales[x_row * s_pitch + col / kMxBlock] = static_cast<uint8_t>(byte);
      }
    }
    __syncthreads();
  }
  for (int s = wave; s < p.steps; s += 2 * stride) {
    multiply(even, s);
    if (s + 2 * stride < p.steps) load(even, s + 2 * stride);
    if (s + stride < p.steps) multiply(odd, s + stride);
    if (s + 3 * stride < p.steps) load(odd, s + 3 * stride);
  }
  // Lane (r, g) holds columns 4 g .. 4 g + 3 of row r of the output.
#pragma unroll
  for (int c = 0; c < 4; ++c) sums[wave * kWaveSums + r16 * kPitch + 4 * group + c] = acc[c];
  __syncthreads();
  for (int i = threadIdx.x; i < 256; i += blockDim.x) {
    const int64_t out_row = i / 16, col = n0 + i % 16;
    float sum = 0.0f;
    for (int w = 0; w < p.waves; ++w) sum += sums[w * kWaveSums + (i / 16) * kPitch + i % 16];
    if (out_row < p.m && col < p.n) {
      if (p.bias) sum += load_bias<DT>(p.bias, col, p.bias_f32);
      store_element<DT>(p.out, out_row * p.ldo + col, sum);
    }
  }
}

}  // namespace
}  // namespace fsh
