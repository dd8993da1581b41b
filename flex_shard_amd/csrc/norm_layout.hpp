// How the rows of a norm are dealt out to threads: LANES threads share a row of
// up to LANES * PER columns, each with vectors of VEC, and keep it in registers;
// TURN rows are under way in a thread together.  Rows of more columns are read twice
// by 1024 threads (PER = 0).
#pragma once
#include "rows.hpp"

namespace fsh {
namespace {

template <int LANES_, int PER_, int VEC_, int TURN_ = 1>
struct NormLayout {
  static constexpr int LANES = LANES_, PER = PER_, VEC = VEC_, ITEMS = PER_ / VEC_, TURN = TURN_;
  static constexpr int THREADS = LANES < 256 ? 256 : LANES;
  static constexpr int ROWS = THREADS / LANES;  // side by side in a workgroup
};

}  // namespace
}  // namespace fsh
