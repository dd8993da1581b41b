// How the rows of a norm are dealt out to threads: LANES threads share a row of
// up to LANES * PER columns, each with vectors of VEC, and keep it in registers;
// TURN rows are under way in a thread together.  Rows of more columns are read twice
// by 1024 threads (PER = 0).  ENDS: how a row's end falls into vectors.
#pragma once
#include "rows.hpp"

namespace fsh {
namespace {

// Rows of a multiple of VEC columns; of more than VEC; of fewer, which go in pieces.
enum RowEnds { kEven, kOverlapping, kPieces };

template <int ENDS_, int LANES_, int PER_, int VEC_, int TURN_ = 1>
struct NormLayout {
  static constexpr int LANES = LANES_, PER = PER_, VEC = VEC_, ITEMS = PER_ / VEC_, TURN = TURN_;
  static constexpr int THREADS = LANES < 256 ? 256 : LANES;
  static constexpr int ROWS = THREADS / LANES;  // side by side in a workgroup
  static constexpr int ENDS = ENDS_;
};

// A lane's vector of a row, for columns `col` on.  The last one of a row that is no
// multiple of VEC lies over the one before it, so that every access is a whole vector: the `skip`
// columns that both have are counted by the lane before, and written by both with the same bits.  (One
// access for each of the last columns, which wait for each other: the gradients of 12800 rows of
// 2301 bf16 take 98 us for 59, the norm of 60000 of 300 46 for 29.)
template <typename L>
struct NormVector {
  int at, skip, count;
  bool inside;
  __device__ __forceinline__ NormVector(int col, int cols) {
    inside = col < cols;
    at = L::ENDS == kOverlapping ? min(col, cols - L::VEC) : col;
    skip = L::ENDS == kOverlapping && inside ? col - at : 0;
    count = L::ENDS == kPieces ? cols - col : L::VEC;
  }
  template <int DT>
  __device__ __forceinline__ RawVec<DT, L::VEC> load(const void* base, int64_t row, bool live) const {
    if constexpr (L::ENDS == kPieces) return load_vec<DT, L::VEC, true>(base, row + at, live ? count : 0);
    RawVec<DT, L::VEC> r;
#pragma unroll
    for (auto& w : r.w) w = 0;
    if constexpr (DT != kNoType) {
      if (live && inside) load_words<true>(static_cast<const uint8_t*>(base) + (row + at) * bytes_of(DT), r.w);
    }
    return r;
  }
  template <int DT, bool STREAM>
  __device__ __forceinline__ void store(void* base, int64_t row, const RawVec<DT, L::VEC>& r) const {
    store_vec<DT, L::VEC, STREAM>(base, row + at, count, r);
  }
  // Ones outside the row.
  __device__ __forceinline__ void weights(const void* base, int32_t dtype, float (&w)[L::VEC]) const {
#pragma unroll
    for (int j = 0; j < L::VEC; ++j) w[j] = 1.0f;
    if (base && inside) load_floats<L::VEC>(base, dtype, at, count, w);
  }
};

// The lane once more, for a loop that works out again where its vectors lie rather than
// to keep that in registers since the loop before it.
template <bool AGAIN>
__device__ __forceinline__ int lane_again(int lane) {
  if constexpr (AGAIN) asm volatile("" : "+v"(lane));
  return lane;
}

// launch(ends) for rows of `cols` columns in vectors of VEC, as an integral constant.
template <int VEC, typename Launch>
void by_ends(int64_t cols, Launch launch) {
  if (cols < VEC) launch(std::integral_constant<int, kPieces>{});
  else if (cols % VEC) launch(std::integral_constant<int, kOverlapping>{});
  else launch(std::integral_constant<int, kEven>{});
}

}  // namespace
}  // namespace fsh
