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
template <int DT>
__device__ __forceinline__ void store_element(void* base, int64_t i, float f) {
  if (DT == FSH_DT_F32) static_cast<float*>(base)[i] = f;
  else static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(round_to_16_bits(f, DT));
}
// Elements [0, count) of eight to `at`; `vec` as above.
template <int DT>
__device__ __forceinline__ void store_raw8(uint8_t* at, const float (&f)[8], int64_t count, bool vec) {
  if (vec && count >= 8) {
    if (DT == FSH_DT_F32) {
      reinterpret_cast<f32x4*>(at)[0] = f32x4{f[0], f[1], f[2], f[3]};
      reinterpret_cast<f32x4*>(at)[1] = f32x4{f[4], f[5], f[6], f[7]};
    } else if (DT == FSH_DT_BF16) {
      *reinterpret_cast<u32x4*>(at) = pack8_bf16(f);
    } else {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = f32_to_f16_bits(f[2 * j]) | (f32_to_f16_bits(f[2 * j + 1]) << 16);
      *reinterpret_cast<u32x4*>(at) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < count) store_element<DT>(at, i, f[i]);
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
__device__ __forceinline__ uint32_t max_magnitude8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = f32_as_u32(f[i]) & 0x7FFFFFFFu;
    m = b > m ? b : m;
  }
  return m;
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
