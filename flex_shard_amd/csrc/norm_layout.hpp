// How the rows of a norm are dealt out to threads: LANES threads share a row of
// up to LANES * PER columns, each with vectors of VEC, and keep it in registers.
// Rows of more columns are read twice by 1024 threads (PER = 0).
#pragma once
#include "rows.hpp"

namespace fsh {
namespace {

template <int LANES_, int PER_, int VEC_>
struct NormLayout {
  static constexpr int LANES = LANES_, PER = PER_, VEC = VEC_, ITEMS = PER_ / VEC_;
  static constexpr int THREADS = LANES < 256 ? 256 : LANES;
  static constexpr int ROWS = THREADS / LANES;  // per workgroup and turn
};

// launch(layout) with the layout for rows of `cols` columns.
template <int VEC, typename Launch>
void by_columns(int64_t cols, Launch launch) {
  if (cols <= 128) launch(NormLayout<128 / VEC, VEC, VEC>{});
  else if (cols <= 512) launch(NormLayout<64, 8, VEC>{});
  else if (cols <= 1024) launch(NormLayout<64, 16, VEC>{});
  else if (cols <= 2048) launch(NormLayout<256, 8, VEC>{});
  else if (cols <= 4096) launch(NormLayout<256, 16, VEC>{});
  else if (cols <= 8192) launch(NormLayout<256, 32, VEC>{});
  else if (cols <= 16384) launch(NormLayout<1024, 16, VEC>{});
  else launch(NormLayout<1024, 0, VEC>{});
}

}  // namespace
}  // namespace fsh
