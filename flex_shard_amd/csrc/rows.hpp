// Rows of bf16, fp16 or fp32 elements in vectors of VEC, and sums and maxima
// over the lanes that share a row: helpers of the norm and optimizer kernels.
#pragma once
#include "common.hpp"

#include <type_traits>

namespace fsh {
namespace {

constexpr int kNoType = -1;  // of an operand that is not there

inline bool is_dtype(int32_t dtype) { return dtype == FSH_DT_BF16 || dtype == FSH_DT_F32 || dtype == FSH_DT_F16; }
constexpr int bytes_of(int dtype) { return dtype == FSH_DT_F32 ? 4 : dtype == kNoType ? 0 : 2; }

// Rows in memory (base null: none); whether two of them may share some of it.
struct RowSpan {
  const void* base;
  int64_t rows, cols, ld, size;
};
inline bool share(const RowSpan& a, const RowSpan& b) {
  if (!a.base || !b.base) return false;
  const auto from = [](const RowSpan& r) { return reinterpret_cast<uintptr_t>(r.base); };
  const auto to = [&](const RowSpan& r) { return from(r) + static_cast<uintptr_t>(((r.rows - 1) * r.ld + r.cols) * r.size); };
  return from(a) < to(b) && from(b) < to(a);
}
// `count` elements of `size` bytes.
inline RowSpan span_of(const void* base, int64_t count, int64_t size) { return {base, 1, count, count, size}; }
// Whether an output lies over an input or another output.
template <int M, int N>
bool outputs_overlap(const RowSpan (&inputs)[M], const RowSpan (&outputs)[N]) {
  for (int i = 0; i < N; ++i) {
    for (const RowSpan& in : inputs)
      if (share(in, outputs[i])) return true;
    for (int j = 0; j < i; ++j)
      if (share(outputs[j], outputs[i])) return true;
  }
  return false;
}

// VEC elements as they lie in memory.
template <int DT, int VEC>
struct RawVec {
  uint32_t w[DT == kNoType ? 1 : VEC * bytes_of(DT) / 4];
};

// 8 or 16 bytes, or several 16, at any address (global memory instructions may be
// unaligned).  STREAM: with the nontemporal hint, for what is not read again.
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));
template <bool STREAM, int N>
__device__ __forceinline__ void load_words(const uint8_t* src, uint32_t (&w)[N]) {
  if constexpr (!STREAM || N < 2) {
    __builtin_memcpy(w, src, sizeof(w));
  } else if constexpr (N == 2) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any*>(src));
    __builtin_memcpy(w, &v, 8);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(src + 4 * i));
      __builtin_memcpy(w + i, &v, 16);
    }
  }
}
template <bool STREAM, int N>
__device__ __forceinline__ void store_words(uint8_t* dst, const uint32_t (&w)[N]) {
  if constexpr (!STREAM || N < 2) {
    __builtin_memcpy(dst, w, sizeof(w));
  } else if constexpr (N == 2) {
    __builtin_nontemporal_store(u32x2{w[0], w[1]}, reinterpret_cast<u32x2_any*>(dst));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      __builtin_nontemporal_store(u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]}, reinterpret_cast<u32x4_any*>(dst + 4 * i));
  }
}

// Elements [0, count) of the VEC at element `at`, the others zero.
template <int DT, int VEC, bool STREAM = false>
__device__ __forceinline__ RawVec<DT, VEC> load_vec(const void* base, int64_t at, int64_t count) {
  RawVec<DT, VEC> r;
#pragma unroll
  for (auto& w : r.w) w = 0;
  if constexpr (DT != kNoType) {
    const uint8_t* src = static_cast<const uint8_t*>(base) + at * bytes_of(DT);
    if (count >= VEC) {
      load_words<STREAM>(src, r.w);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (j >= count) break;
        if (DT == FSH_DT_F32) {
          uint32_t v;
          __builtin_memcpy(&v, src + 4 * j, 4);
          r.w[j] = v;
        } else {
          uint16_t v;
          __builtin_memcpy(&v, src + 2 * j, 2);
          r.w[j / 2] |= static_cast<uint32_t>(v) << (16 * (j % 2));
        }
      }
    }
  }
  return r;
}

template <int DT, int VEC>
__device__ __forceinline__ float element(const RawVec<DT, VEC>& r, int j) {
  if (DT == FSH_DT_F32) return u32_as_f32(r.w[j]);
  const uint32_t half = (r.w[j / 2] >> (16 * (j % 2))) & 0xFFFFu;
  return DT == FSH_DT_BF16 ? bf16_bits_to_f32(half) : f16_bits_to_f32(half);
}

// fp32 to the bits of a type, to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t bits_of(float f) {
  return DT == FSH_DT_F32 ? f32_as_u32(f) : DT == FSH_DT_BF16 ? f32_to_bf16_bits(f) : f32_to_f16_bits(f);
}

// VEC floats rounded to a type once.
template <int DT, int VEC>
__device__ __forceinline__ RawVec<DT, VEC> to_vec(const float (&f)[VEC]) {
  RawVec<DT, VEC> r;
  if constexpr (DT == FSH_DT_F32) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) r.w[j] = f32_as_u32(f[j]);
  } else if constexpr (DT == FSH_DT_BF16) {
    bool nan = false;
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      r.w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{f[2 * j], f[2 * j + 1]}), bf16x2));
      nan |= __builtin_isunordered(f[2 * j], f[2 * j + 1]) != 0;
    }
    if (nan) {
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) r.w[j] = canonical_nan_pair(r.w[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) r.w[j] = f32_to_f16_bits(f[2 * j]) | (f32_to_f16_bits(f[2 * j + 1]) << 16);
  }
  return r;
}

template <int DT, int VEC, bool STREAM = false>
__device__ __forceinline__ void store_vec(void* base, int64_t at, int64_t count, const RawVec<DT, VEC>& r) {
  uint8_t* dst = static_cast<uint8_t*>(base) + at * bytes_of(DT);
  if (count >= VEC) {
    store_words<STREAM>(dst, r.w);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (j >= count) break;
      if (DT == FSH_DT_F32) {
        __builtin_memcpy(dst + 4 * j, &r.w[j], 4);
      } else {
        const uint16_t v = static_cast<uint16_t>(r.w[j / 2] >> (16 * (j % 2)));
        __builtin_memcpy(dst + 2 * j, &v, 2);
      }
    }
  }
}

// VEC elements of a type that is known at run time (the same for all lanes).
template <int VEC>
__device__ __forceinline__ void load_floats(const void* base, int32_t dtype, int64_t at, int64_t count, float (&f)[VEC]) {
  if (dtype == FSH_DT_F32) {
    const auto r = load_vec<FSH_DT_F32, VEC>(base, at, count);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = element<FSH_DT_F32, VEC>(r, j);
  } else if (dtype == FSH_DT_BF16) {
    const auto r = load_vec<FSH_DT_BF16, VEC>(base, at, count);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = element<FSH_DT_BF16, VEC>(r, j);
  } else {
    const auto r = load_vec<FSH_DT_F16, VEC>(base, at, count);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = element<FSH_DT_F16, VEC>(r, j);
  }
}

// Sums over 8 lanes, a row of 16, half a wave, a wave, in every lane of them: moves
// between lanes (DPP), always in the same order.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + u32_as_f32(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(f32_as_u32(v)), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ float sum8(float v) {
  v = dpp_add<0xB1>(v);      // quad_perm [1,0,3,2]
  v = dpp_add<0x4E>(v);      // quad_perm [2,3,0,1]
  return dpp_add<0x141>(v);  // row_half_mirror
}
__device__ __forceinline__ float sum16(float v) { return dpp_add<0x140>(sum8(v)); }  // row_mirror
__device__ __forceinline__ float sum32(float v) {
  v = sum16(v);
  return v + __shfl_xor(v, 16, kWave);
}
__device__ __forceinline__ float sum64(float v) {
  v = sum16(v);
  const int b = static_cast<int>(f32_as_u32(v));
  const float r0 = u32_as_f32(__builtin_amdgcn_readlane(b, 0)), r1 = u32_as_f32(__builtin_amdgcn_readlane(b, 16));
  const float r2 = u32_as_f32(__builtin_amdgcn_readlane(b, 32)), r3 = u32_as_f32(__builtin_amdgcn_readlane(b, 48));
  return (r0 + r1) + (r2 + r3);
}
// Largest of non-negative floats' bits over half a wave.
__device__ __forceinline__ uint32_t max32_u32(uint32_t v) {
  v = row16_max_u32(v);
  const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16, kWave));
  return o > v ? o : v;
}

// The sum over the LANES threads that share a row (8, 16, 32, 64, or a whole workgroup of
// several waves: then `lds` holds a float for each of them, twice over, used in turn).
template <int LANES>
__device__ __forceinline__ float sum_over_row(float v, float* lds, int turn) {
  if constexpr (LANES == 8) return sum8(v);
  if constexpr (LANES == 16) return sum16(v);
  if constexpr (LANES == 32) return sum32(v);
  if constexpr (LANES == 64) return sum64(v);
  constexpr int kWaves = LANES / 64;
  float* const mine = lds + (turn & 1) * kWaves;
  v = sum64(v);
  if ((threadIdx.x & 63) == 0) mine[threadIdx.x >> 6] = v;
  __syncthreads();
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sum += mine[w];
  return sum;
}

}  // namespace
}  // namespace fsh
