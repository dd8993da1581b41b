// Microscaled 4-bit floats: E2M1 elements (magnitudes 0, 0.5, 1, 1.5, 2, 3, 4,
// 6), 32 of them under one E8M0 scale (a power of two, 2^(byte - 127)).
//
// A matrix lies in memory as
//   data    [rows][cols_padded / 2] bytes, the element of the lower column in
//           the low half; cols_padded = cols rounded up to 256, the pad zero
//   scales  [cols_padded / 256][rows][8] bytes: the eight scales of a row's 256
//           columns are one 8-byte word, the words of neighbouring rows adjacent
// so that a tile's k-step is 128 bytes of data and one word of scales per row.
#pragma once
#include "common.hpp"

#include <type_traits>

namespace fsh {
namespace {

constexpr int kMxBlock = 32;
constexpr int kMxColumns = 256;  // columns are padded to a multiple of this

inline bool known_dtype(int32_t dtype) { return dtype == FSH_DT_BF16 || dtype == FSH_DT_F32 || dtype == FSH_DT_F16; }
inline int dtype_bytes(int32_t dtype) { return dtype == FSH_DT_F32 ? 4 : 2; }
// launch(tag) with tag.value the dtype, for a template argument.
template <typename Launch>
void by_dtype(int32_t dtype, Launch launch) {
  if (dtype == FSH_DT_BF16) launch(std::integral_constant<int, FSH_DT_BF16>{});
  else if (dtype == FSH_DT_F16) launch(std::integral_constant<int, FSH_DT_F16>{});
  else launch(std::integral_constant<int, FSH_DT_F32>{});
}

// Eight consecutive elements of a row as they lie in memory.
template <int DT>
struct Raw8 {
  u32x4 v[DT == FSH_DT_F32 ? 2 : 1];
};
template <int DT>
constexpr int element_bytes() { return DT == FSH_DT_F32 ? 4 : 2; }

// Elements [0, count) of the eight at `at`, the others zero.  `vec`: `at` is
// 16-byte aligned whenever count is 8.
template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const uint8_t* at, int64_t count, bool vec) {
  Raw8<DT> r;
#pragma unroll
  for (auto& v : r.v) v = u32x4{0, 0, 0, 0};
  if (vec && count >= 8) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(r.v) / 16); ++i) r.v[i] = *reinterpret_cast<const u32x4*>(at + 16 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= count) break;
      if (DT == FSH_DT_F32)
        r.v[i / 4][i % 4] = reinterpret_cast<const uint32_t*>(at)[i];
      else
        r.v[0][i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(at)[i]) << (16 * (i % 2));
    }
  }
  return r;
}
// Element `half` (0: low, 1: high) of a pair of 16-bit elements.
template <int DT>
__device__ __forceinline__ float half_of_pair(uint32_t pair, int half) {
  if (DT == FSH_DT_F16) return f16_bits_to_f32(half ? pair >> 16 : pair & 0xFFFFu);
  return u32_as_f32(half ? pair & 0xFFFF0000u : pair << 16);
}
template <int DT>
__device__ __forceinline__ void unpack_raw8(const Raw8<DT>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = DT == FSH_DT_F32 ? u32_as_f32(r.v[i / 4][i % 4]) : half_of_pair<DT>(r.v[0][i / 2], i % 2);
}

template <int DT>
__device__ __forceinline__ float load_element(const void* base, int64_t i) {
  if (DT == FSH_DT_F32) return static_cast<const float*>(base)[i];
  const uint16_t bits = static_cast<const uint16_t*>(base)[i];
  return DT == FSH_DT_F16 ? f16_bits_to_f32(bits) : bf16_bits_to_f32(bits);
}
__device__ __forceinline__ uint32_t round_to_16_bits(float f, int dtype) {
  return dtype == FSH_DT_F16 ? f32_to_f16_bits(f) : f32_to_bf16_bits(f);
}
// Element i of a bias: of the output's type DT, or fp32.
template <int DT>
__device__ __forceinline__ float load_bias(const void* bias, int64_t i, int32_t is_f32) {
  return is_f32 ? load_element<FSH_DT_F32>(bias, i) : load_element<DT>(bias, i);
}
template <int DT>
__device__ __forceinline__ void store_element(void* base, int64_t i, float f) {
  if (DT == FSH_DT_F32) static_cast<float*>(base)[i] = f;
  else static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(round_to_16_bits(f, DT));
}
// Two floats to fp16, bit for bit f32_to_f16_bits (a NaN keeps its payload): the hardware's conversion, and below 2^-14,
// where it does not round ties to even, the sum with 0.5, whose low mantissa bits are the subnormal's.  A third of
// the instructions: 1000 x 5120, k 2048 17.1 us with the one, 14.1 so.
__device__ __forceinline__ uint32_t f32_to_f16_fast(float f) {
  const uint32_t h = __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  const uint32_t low = f32_as_u32(fabsf(f) + 0.5f) & 0x7FFFu;
  return fabsf(f) < 6.103515625e-05f ? (h & 0x8000u) | low : h;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) { return f32_to_f16_fast(lo) | (f32_to_f16_fast(hi) << 16); }
// Eight floats to 16-bit elements.
template <int DT>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  if constexpr (DT == FSH_DT_BF16) {
    return pack8_bf16(f);
  } else {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack_f16x2(f[2 * j], f[2 * j + 1]);
    return w;
  }
}

// The scale byte of a run from the largest magnitude's fp32 bits: the power of
// two at or below it, less 2 (6 = 1.5 * 2^2 is the largest element), not below
// 2^-127; 255 (not a number) if the run holds an infinity or a NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// The scale as a float; its exponent field is the byte.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return u32_as_f32(byte == 0u ? 0x00400000u : byte == 255u ? 0x7FC00000u : byte << 23);
}
// Eight elements over a scale, the first in the low bits: to nearest, ties to
// the even code, magnitudes above 6 to 6.
__device__ __forceinline__ uint32_t mx_quantize8(const float (&f)[8], float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0], f[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], scale, 3);
  return w;
}
// Eight elements as they lie in memory: 16-bit magnitudes compare as whole
// numbers, and pairs of bf16 or fp16 convert without being taken apart.
template <int DT>
__device__ __forceinline__ uint32_t magnitude_bits_to_f32(uint32_t m) {  // of a 16-bit magnitude, or fp32 bits
  if (DT == FSH_DT_F32) return m;
  return DT == FSH_DT_F16 ? f32_as_u32(f16_bits_to_f32(m)) : m << 16;
}
__device__ __forceinline__ uint32_t larger_half(uint32_t pair) { return (pair & 0xFFFFu) > (pair >> 16) ? pair & 0xFFFFu : pair >> 16; }
template <int DT>
__device__ __forceinline__ uint32_t max_magnitude8(const Raw8<DT>& r) {  // in the element's own bits
  if constexpr (DT == FSH_DT_F32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = r.v[i / 4][i % 4] & 0x7FFFFFFFu;
      m = b > m ? b : m;
    }
    return m;
  } else {
    const u32x4 a = r.v[0] & 0x7FFF7FFFu;
    return larger_half(pk_max_u16(pk_max_u16(a.x, a.y), pk_max_u16(a.z, a.w)));
  }
}
// Two neighbouring elements (16-bit: a dword that holds both) to byte kByte of `old`.
template <int DT, int kByte>
__device__ __forceinline__ uint32_t mx_quantize_pair(uint32_t old, uint32_t pair, float scale) {
  if constexpr (DT == FSH_DT_F16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, pair), scale, kByte);
  } else {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, pair), scale, kByte);
  }
}
template <int DT>
__device__ __forceinline__ uint32_t mx_quantize8(const Raw8<DT>& r, float scale) {
  if constexpr (DT == FSH_DT_F32) {
    float f[8];
    unpack_raw8<DT>(r, f);
    return mx_quantize8(f, scale);
  } else {
    uint32_t w = 0;
    w = mx_quantize_pair<DT, 0>(w, r.v[0].x, scale);
    w = mx_quantize_pair<DT, 1>(w, r.v[0].y, scale);
    w = mx_quantize_pair<DT, 2>(w, r.v[0].z, scale);
    return mx_quantize_pair<DT, 3>(w, r.v[0].w, scale);
  }
}

// Experts: the rows of expert e are [offsets[e], offsets[e + 1]) of the sorted
// rows.  How many of `count` ascending numbers are at most `at` (all lanes).
__device__ __forceinline__ int count_not_above(const int32_t* numbers, int count, int64_t at) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int found = 0;
  for (int first = 0; first < count; first += 64) {
    const bool below = first + lane < count && numbers[first + lane] <= at;
    found += __popcll(__ballot(below));
  }
  return __builtin_amdgcn_readfirstlane(found);
}

}  // namespace
}  // namespace fsh
