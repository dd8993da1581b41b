// The product of two microscaled 4-bit matrices, a tile at a time.
//
//   out[i][j] = sum over blocks b of 32 columns of
//               2^(sa[i][b] - 127) * 2^(sb[j][b] - 127) * dot(a[i][b], b[j][b])
//
// The matrix instruction takes the scales itself (one byte per row and 32
// columns of each operand), so a k-step is loads, fragment reads and MFMAs alone.
#pragma once
#include "mfma_tiles.hpp"
#include "mxfp4.hpp"

#include <utility>

namespace fsh {
namespace {

typedef int v8i32 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Lambdas of a kernel are always inlined: a real call would keep the registers that they refer to in memory.
#define FSH_INLINE __attribute__((always_inline))

// f(0), f(1) .. f(N - 1) with constants.
template <typename F, int... I>
__device__ __forceinline__ void static_for(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for(f, std::make_integer_sequence<int, N>{});
}

constexpr int at_most_63(int count) { return count < 63 ? count : 63; }  // what the wait instruction can count

// Waits until all loads but those of the `later` last steps have landed, kPer each (at most kSteps of them).
template <int kSteps, int kPer>
__device__ __forceinline__ void wait_but_steps(int later) {
  if constexpr (kSteps == 0) {
    wait_for_dma_loads();
  } else {
    if (later == kSteps) wait_for_dma_loads_but<kSteps * kPer>();
    else wait_but_steps<kSteps - 1, kPer>(later);
  }
}

enum MxProblem {
  kMxDense,      // one product
  kMxRows,       // rows of a in segments, one per expert, each against that expert's b
  kMxOverRows,   // per expert the product over its own (padded) columns of a and b: [experts][m][n]
};

// Division by a number that the host knows: x / d is x * factor >> shift for x
// below 2^31, with factor = ceil(2^shift / d) and shift = 31 + ceil(log2 d).
struct Divisor {
  uint32_t factor;
  int32_t shift;
  __host__ static Divisor of(uint32_t d) {
    int32_t b = 0;
    while ((1ULL << b) < d) ++b;
    return Divisor{static_cast<uint32_t>(((1ULL << (31 + b)) + d - 1) / d), 31 + b};
  }
  __device__ __forceinline__ int quotient(int x) const {
    return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(x)) * factor >> shift);
  }
};

// The order of the tiles: XCD x takes the run [x, x + 1) * items_per_xcd of an order in which kGroupTilesM tile rows are
// walked together, so that the tiles that its compute units hold at a time share operands in its L2.  Products of
// different lengths (kMxOverRows) are cut into runs of `run` tiles, and the first runs of all experts come before the
// second ones: every XCD then has an eighth of every expert, whatever their rows.
struct MxSchedule {
  int32_t tiles_m, tiles_n, items, items_per_xcd;  // items: tiles of all matrices
  int32_t run;
  Divisor by_span, by_run, by_round;  // kGroupTilesM tile rows, a run, the runs of all experts
};

struct MxGemmParams {
  const uint8_t* a;   // [a_rows][lda]
  const uint8_t* as;  // [k / 256][a_rows][8]
  const uint8_t* b;
  const uint8_t* bs;
  void* out;
  const void* bias;  // [n] of the output's type, or fp32 (bias_f32), or null
  int64_t m, n, k;   // k a multiple of 256; kMxOverRows: of all segments
  int64_t a_rows, b_rows, lda, ldb, ldo;
  int32_t out_dtype, bias_f32;
  int32_t experts, top_k;
  const int32_t* offsets;         // [experts + 1]
  const int32_t* padded_offsets;  // [experts + 1] (kMxOverRows)
  const int32_t* source;          // kMxRows: row r of the segments is row source[r] / top_k of a, or null
  Divisor by_top_k;
  MxSchedule schedule;
};

// A tile of WM x WN waves, each TM x TN blocks of 32 x 32.  A k-step is 256
// columns: 128 bytes and 8 scale bytes of every row.  A chunk is what one request
// of every wave fills.  The first kEarly chunks of a step have kDepth + 1 slots in
// LDS, the others and the scales kDepth.  kResident: a workgroup holds a compute
// unit and takes one tile after another.
template <int WM_, int WN_, int TM_, int TN_, int kDepth_, int kEarly_, bool kResident_>
struct MxTile {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, kDepth = kDepth_, kEarly = kEarly_;
  static constexpr bool kResident = kResident_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves, kWaveM = 32 * TM, kWaveN = 32 * TN;
  static constexpr int BM = WM * kWaveM, BN = WN * kWaveN, kRowBytes = 128;
  static constexpr int kChunkRows = 8 * kWaves, kChunkBytes = kChunkRows * kRowBytes;
  static constexpr int kChunksA = BM / kChunkRows, kChunks = (BM + BN) / kChunkRows, kLate = kChunks - kEarly;
  // Scales: two planes (the words' lower and upper half) of BM + BN dwords, 64 by a request.
  static constexpr int kScaleRequests = 2 * (BM + BN) / 64 / kWaves, kPlaneBytes = 4 * (BM + BN);
  static constexpr int kEarlyBytes = kEarly * kChunkBytes, kLateBytes = kLate * kChunkBytes, kScaleBytes = 2 * kPlaneBytes;
  static constexpr int kLateOffset = (kDepth + 1) * kEarlyBytes, kScaleOffset = kLateOffset + kDepth * kLateBytes;
  // Behind the slots: the bias of the tile's columns, or the first tile of every segment.
  static constexpr int kTableOffset = kScaleOffset + kDepth * kScaleBytes, kTableBytes = FSH_MAX_EXPERTS * 4;
  static constexpr int kLdsBytes = kTableOffset + kTableBytes;
  static constexpr int kRequests = kChunks + kScaleRequests;  // of a step, per wave
  // Epilogue staging of a wave: 32 rows of 128 bytes, in the last early slot of a resident tile (the next tile's first
  // steps fill the others meanwhile).
  static constexpr int kPitch = 144, kRegion = 32 * kPitch, kStageOffset = kResident ? kDepth * kEarlyBytes : 0;
  static_assert(kLdsBytes <= 160 * 1024, "LDS of a compute unit");
  static_assert(kWaves * kRegion <= (kResident ? kEarlyBytes : kTableOffset), "staging");
  static_assert(BM % kChunkRows == 0 && BN % kChunkRows == 0 && kChunkRows % 32 == 0, "whole requests, whole blocks");
  static_assert(BM % 64 == 0 && BN % 64 == 0 && kScaleRequests * kWaves * 32 == BM + BN, "scales by 64, the same for every wave");
  static_assert(kEarly <= kChunksA && BN <= kThreads, "operand B is late; a bias per thread");
  static_assert(kDepth >= 2 && (kDepth - 1) * kRequests + kEarly < 64, "requests in flight are counted in six bits");
  static_assert(!kResident || kDepth == 2, "the requests that the epilogue sends");
};

// Where a tile lies.
struct MxTilePlace {
  int64_t row0, rows;  // output rows [row0, row0 + rows); also the operand's (before `source`)
  int64_t col0, b_row0;  // output columns from col0 on; row of b that column 0 is
  int64_t out_offset;    // elements
  int64_t first_step;
  int steps;
  bool zero;  // rows without a product: zeros
};

// The first tile of BM rows of segments 1 to `experts` to `table`; the rows behind
// the last expert's are segment `experts`.  Returns the number of tiles (in every wave).
template <int BM>
__device__ __forceinline__ int fill_segment_table(const MxGemmParams& p, int32_t* table) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int before = 0;
  for (int first = 0; first <= p.experts; first += 64) {
    const int e = first + lane;
    int tiles = 0;
    if (e <= p.experts) {
      const int64_t end = e < p.experts ? p.offsets[e + 1] : p.m;
      tiles = static_cast<int>((end - p.offsets[e] + BM - 1) / BM);
    }
    int sum = tiles;  // inclusive scan over the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int other = __shfl_up(sum, off, kWave);
      if (lane >= off) sum += other;
    }
    if (threadIdx.x < 64 && e < p.experts) table[e] = before + sum;
    before += __shfl(sum, 63, kWave);
  }
  __syncthreads();
  return uniform_i32(before);
}

// A number that is the same in every lane, through the scalar cache: a vector load
// would be waited for together with all requests and stores in flight.
__device__ __forceinline__ int32_t load_uniform(const int32_t* at) {
  typedef const __attribute__((address_space(4))) int32_t* constant_address;
  return *(constant_address)(reinterpret_cast<uintptr_t>(at));
}

// How a finished tile leaves: in parts of 32 rows x kCols columns of a wave,
// kStores 16-byte stores of every lane each, and which of them follow the next
// tile's requests, which go out a few behind each part.
template <typename Cfg, int DT>
struct MxStores {
  static constexpr int kElement = element_bytes<DT>(), kCols = kElement == 2 && Cfg::TN > 1 ? 64 : 32;
  static constexpr int kPartBytes = kCols * kElement, kWords = kPartBytes / 8, kStores = kPartBytes / 32;
  static constexpr int kParts = Cfg::TM * Cfg::kWaveN / kCols;
  static constexpr int part_of_request(int r) { return r * kParts / (2 * Cfg::kRequests); }
  static constexpr int behind_step(int step) { return (kParts - part_of_request((step + 1) * Cfg::kRequests - 1)) * kStores; }
  static_assert(kPartBytes + 16 <= Cfg::kPitch, "staging");
};

// The tile of a workgroup's turn (0 for the first) in the order of `schedule`.
template <typename Cfg, int kProblem>
__device__ __forceinline__ bool place_of_turn(const MxGemmParams& p, const MxSchedule& schedule, const int32_t* table, int turn,
                                              MxTilePlace* place) {
  const int id = static_cast<int>(blockIdx.x) + turn * static_cast<int>(gridDim.x);
  const int item = id % kXcds * schedule.items_per_xcd + id / kXcds;
  if (id / kXcds >= schedule.items_per_xcd || item >= schedule.items) return false;
  const int tiles = schedule.tiles_m * schedule.tiles_n;
  int batch = 0, t = item;
  if (kProblem == kMxOverRows) {
    const int round = schedule.by_round.quotient(item), first = round * schedule.run, left = tiles - first;
    const int run = left < schedule.run ? left : schedule.run, of_round = item - first * p.experts;
    batch = run == schedule.run ? schedule.by_run.quotient(of_round) : of_round / run;
    t = first + of_round - batch * run;
  }
  const int first_m = schedule.by_span.quotient(t) * kGroupTilesM;
  const int within = t - first_m * schedule.tiles_n, rows = min(schedule.tiles_m - first_m, kGroupTilesM);
  static_assert(kGroupTilesM == 4, "the divisions");
  const int tn = rows == 4 ? within / 4 : rows == 3 ? within / 3 : rows == 2 ? within / 2 : within, tm = first_m + within - tn * rows;
  place->zero = false;
  place->out_offset = 0;
  place->first_step = 0;
  place->steps = static_cast<int>(p.k / kMxColumns);
  place->col0 = static_cast<int64_t>(tn) * Cfg::BN;
  place->b_row0 = 0;
  if (kProblem == kMxRows) {
    const int segment = count_not_above(table, p.experts, tm);  // the segments that end at or before tile tm
    const int first_tile = segment > 0 ? uniform_i32(table[segment - 1]) : 0;
    const int64_t end = segment < p.experts ? load_uniform(p.offsets + segment + 1) : p.m;
    place->row0 = load_uniform(p.offsets + segment) + static_cast<int64_t>(tm - first_tile) * Cfg::BM;
    place->rows = end - place->row0 < Cfg::BM ? end - place->row0 : Cfg::BM;
    place->zero = segment == p.experts;
    place->b_row0 = static_cast<int64_t>(segment) * p.n;
  } else {
    place->row0 = static_cast<int64_t>(tm) * Cfg::BM;
    place->rows = p.m - place->row0 < Cfg::BM ? p.m - place->row0 : Cfg::BM;
    if (kProblem == kMxOverRows) {
      const int expert = batch;
      const int32_t begin = load_uniform(p.padded_offsets + expert), end = load_uniform(p.padded_offsets + expert + 1);
      place->first_step = begin / kMxColumns;
      place->steps = (end - begin) / kMxColumns;
      place->zero = place->steps == 0;
      place->out_offset = expert * p.m * p.n;
    }
  }
  return true;
}

template <int DT, typename Cfg>
__device__ __forceinline__ void zero_tile(const MxGemmParams& p, const MxTilePlace& place) {
  for (int i = threadIdx.x; i < Cfg::BM * Cfg::BN; i += Cfg::kThreads) {
    const int64_t r = i / Cfg::BN, col = place.col0 + i % Cfg::BN;
    if (r < place.rows && col < p.n) store_element<DT>(p.out, place.out_offset + (place.row0 + r) * p.ldo + col, 0.0f);
  }
}

// The k loop is rotated: an iteration is the last of a step's four k-quarters and
// the first three of the next step.  The barrier that hands over step t + 1 sits
// behind the first MFMA of step t's last quarter, when all of step t's fragments
// are in registers; behind the barrier its slots are free, and the requests of
// step t + kDepth (scales and late chunks) and t + kDepth + 1 (early chunks) leave
// one by one behind the iteration's MFMAs.  The fragments of a quarter are read
// behind the MFMAs of the quarter before.
//
// A resident workgroup requests the first two steps of its next tile before it
// stores the one it has finished: the start of a tile (a chain of loads) and the
// end of one (128 KB of stores) then pass behind one another and behind products.
//
// Measured, 256 x 256 tiles: 2340 cycles a step (2048 of MFMA), 10 000 to 12 000 between
// two tiles' steps, at the 1.7 GHz that the power allows.  8192 x 4096, k 14336 206
// us, 4.7 PFLOP/s; 8192 x 14336, k 4096 250 us, 3.9; 4096 x 4096, k 4096 36 us, 3.9.
// Outputs go past the caches, which hold the operands: rows of 32 experts' weight
// gradients, [2048, 7168] each of 1024 rows, 484 us through them, 364 so.
// The staging pays for whole 128-byte stores: swapping halves and quarters of a
// wave instead (64-byte pieces, no LDS) took 63 us for 47, 14336 x 4096, k 1024.
template <typename Cfg, int kProblem, int DT>
__global__ __launch_bounds__(Cfg::kThreads, Cfg::kWaves / 4) void mxfp4_gemm_kernel(const MxGemmParams p) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds_bytes[];
  constexpr int TM = Cfg::TM, TN = Cfg::TN, kChunks = Cfg::kChunks, kChunksA = Cfg::kChunksA, kEarly = Cfg::kEarly, kDepth = Cfg::kDepth;
  constexpr int kRequests = Cfg::kRequests, kScaleRequests = Cfg::kScaleRequests;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
  int32_t* const table = reinterpret_cast<int32_t*>(lds_bytes + Cfg::kTableOffset);
  float* const bias_of_tile = reinterpret_cast<float*>(lds_bytes + Cfg::kTableOffset);

  MxSchedule schedule = p.schedule;
  if (kProblem == kMxRows) {
    // How many tiles the segments have is known here only.
    schedule.tiles_m = fill_segment_table<Cfg::BM>(p, table);
    schedule.items = schedule.tiles_m * schedule.tiles_n;
    schedule.items_per_xcd = (schedule.items + kXcds - 1) / kXcds;
  }
  MxTilePlace place;
  if (!place_of_turn<Cfg, kProblem>(p, schedule, table, 0, &place)) return;  // whole workgroup

  // Data: request c of a wave fills rows [kChunkRows c + 8 wave, +8), lane l slot
  // l & 7 of row l >> 3.  Slot s of row r holds the row's 16-byte chunk
  // s ^ ((r >> 1) & 7): the 32 rows that half a wave reads at a time then lie in
  // different banks, 16 by 16.
  const int fill_row = lane >> 3;
  const uint32_t fill_chunk = (lane & 7) ^ (((8 * wave + fill_row) >> 1) & 7);
  // Scales: request q = kScaleRequests wave + i fills plane q & 1 of rows [64 (q >> 1), +64).
  const bool gathered = kProblem == kMxRows && p.source;
  // The rows of A that this lane requests; rows past the last are read from the
  // last (their products are not stored).
  struct Rows {
    int32_t data[kChunksA], scales[kScaleRequests];  // from the tile's first row, or of the matrix where gathered
  };
  const auto rows_of = [&](const MxTilePlace& at) FSH_INLINE {
    Rows rows;
    const int last = static_cast<int>(at.rows) - 1;
#pragma unroll
    for (int c = 0; c < kChunksA; ++c) {
      const int r = Cfg::kChunkRows * c + 8 * wave + fill_row;
      rows.data[c] = r < last ? r : last;
      if (gathered) rows.data[c] = at.zero ? 0 : p.source[at.row0 + rows.data[c]];
    }
#pragma unroll
    for (int i = 0; i < kScaleRequests; ++i) {
      const int r = 64 * ((kScaleRequests * wave + i) >> 1) + lane;
      rows.scales[i] = r < last ? r : last;
      if (gathered && r < Cfg::BM) rows.scales[i] = at.zero ? 0 : p.source[at.row0 + rows.scales[i]];
    }
    return rows;
  };
  uint32_t voff[kChunks], scale_voff[kScaleRequests];
  const uint8_t* a_data = nullptr;
  const uint8_t* b_data = nullptr;
  const uint8_t* scale_src[kScaleRequests];
  int64_t scale_step[kScaleRequests];
  uint32_t scale_lds[kScaleRequests];
  const auto aim = [&](const MxTilePlace& at, const Rows& rows) FSH_INLINE {
    const int64_t a_first = gathered ? 0 : at.row0, b_first = at.b_row0 + at.col0;
    const int b_last = static_cast<int>(p.n - at.col0 < Cfg::BN ? p.n - at.col0 : Cfg::BN) - 1;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (c < kChunksA) {
        voff[c] = static_cast<uint32_t>(gathered ? p.by_top_k.quotient(rows.data[c]) : rows.data[c]) * static_cast<uint32_t>(p.lda);
      } else {
        const int r = Cfg::kChunkRows * (c - kChunksA) + 8 * wave + fill_row;
        voff[c] = static_cast<uint32_t>(r < b_last ? r : b_last) * static_cast<uint32_t>(p.ldb);
      }
      voff[c] += fill_chunk * 16;
    }
    a_data = uniform_ptr(p.a + a_first * p.lda + at.first_step * Cfg::kRowBytes);
    b_data = uniform_ptr(p.b + b_first * p.ldb + at.first_step * Cfg::kRowBytes);
#pragma unroll
    for (int i = 0; i < kScaleRequests; ++i) {
      const int q = kScaleRequests * wave + i, first = 64 * (q >> 1);
      const bool of_a = first < Cfg::BM;
      const int r = first - Cfg::BM + lane;
      const int row = of_a ? (gathered ? p.by_top_k.quotient(rows.scales[i]) : rows.scales[i]) : (r < b_last ? r : b_last);
      scale_voff[i] = static_cast<uint32_t>(row) * 8;
      scale_step[i] = (of_a ? p.a_rows : p.b_rows) * 8;
      scale_src[i] = uniform_ptr((of_a ? p.as + a_first * 8 : p.bs + b_first * 8) + at.first_step * scale_step[i] + 4 * (q & 1));
      scale_lds[i] = (q & 1) * Cfg::kPlaneBytes + first * 4;
    }
  };
  typedef __attribute__((address_space(3))) uint8_t* lds_address;
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_address)lds_bytes));
  // Where a step lies: the offsets of its early chunks, of its late ones and of its scales.
  struct Place {
    int early, late, scales;
  };
  constexpr Place kFirst{0, Cfg::kLateOffset, Cfg::kScaleOffset};
  constexpr Place kLast{kDepth * Cfg::kEarlyBytes, Cfg::kLateOffset + (kDepth - 1) * Cfg::kLateBytes,
                        Cfg::kScaleOffset + (kDepth - 1) * Cfg::kScaleBytes};
  const auto place_after = [](const Place& at) {
    return Place{at.early == kLast.early ? kFirst.early : at.early + Cfg::kEarlyBytes,
                 at.late == kLast.late ? kFirst.late : at.late + Cfg::kLateBytes,
                 at.scales == kLast.scales ? kFirst.scales : at.scales + Cfg::kScaleBytes};
  };
  const auto request = [&](int step, const Place& at, int c) FSH_INLINE {
    dma_load_16(voff[c], (c < kChunksA ? a_data : b_data) + static_cast<int64_t>(step) * Cfg::kRowBytes,
                lds_base + (c < kEarly ? at.early : at.late) + wave * 1024, (c < kEarly ? c : c - kEarly) * Cfg::kChunkBytes);
  };
  const auto request_scales = [&](int step, const Place& at, int i) FSH_INLINE {
    dma_touch_4(scale_voff[i], scale_src[i] + step * scale_step[i], lds_base + at.scales + scale_lds[i]);
  };
  // Request r of the first kDepth steps of a tile, of kRequests each; then the early chunks of one more.
  const auto request_first = [&](auto long_enough, int steps, auto r_tag) FSH_INLINE {
    constexpr int d = decltype(r_tag)::value / kRequests, q = decltype(r_tag)::value % kRequests;
    constexpr Place at{d * Cfg::kEarlyBytes, kFirst.late + d * Cfg::kLateBytes, kFirst.scales + d * Cfg::kScaleBytes};
    if (long_enough.value || d == 0 || d < steps) {
      if constexpr (q < kScaleRequests) request_scales(d, at, q);
      else request(d, at, q - kScaleRequests);
    }
  };
  const auto request_first_early = [&](int steps) FSH_INLINE {
#pragma unroll
    for (int c = 0; c < kEarly; ++c)
      if (kDepth < steps) request(kDepth, Place{kDepth * Cfg::kEarlyBytes, 0, 0}, c);
  };
  const auto request_all_first = [&](int steps) FSH_INLINE {
    static_for<kDepth * kRequests>([&](auto r) FSH_INLINE { request_first(std::false_type{}, steps, r); });
    request_first_early(steps);
  };

  // Lane l of a fragment has row l & 31 and, in quarter s of a step, the 32
  // columns 4 g + s of its 8 times 32 (g = l >> 5); its four scale bytes of the
  // step are then one dword.
  const int frag_row = lane & 31, group = lane >> 5;
  uint32_t frag_off[4];
#pragma unroll
  for (int s = 0; s < 4; ++s)
    frag_off[s] = static_cast<uint32_t>(frag_row * Cfg::kRowBytes + (((4 * group + s) ^ ((frag_row >> 1) & 7)) * 16));
  const uint32_t scale_off = static_cast<uint32_t>(group * Cfg::kPlaneBytes + frag_row * 4);
  const int a0 = wm * Cfg::kWaveM, b0 = Cfg::BM + wn * Cfg::kWaveN;
  // 32 rows from `row` of the tile (A's rows, then B's)
  const auto read_frag = [&](const Place& at, int row, int s) FSH_INLINE -> u32x4 {
    const int c = row / Cfg::kChunkRows;
    const int base = c < kEarly ? at.early + c * Cfg::kChunkBytes : at.late + (c - kEarly) * Cfg::kChunkBytes;
    return *reinterpret_cast<const u32x4*>(lds_bytes + base + row % Cfg::kChunkRows * Cfg::kRowBytes + frag_off[s]);
  };
  const auto read_scale = [&](const Place& at, int row) FSH_INLINE -> int {
    return *reinterpret_cast<const int*>(lds_bytes + at.scales + scale_off + row * 4);
  };

  constexpr int kBlocks = TM * TN, kCycle = 4 * kBlocks, kReads = TM + TN;
  // The MFMA of an iteration that request r goes out behind: behind the reads that follow the barrier.
  constexpr auto behind_mfma = [](int r) {
    constexpr int first = kBlocks > 1 ? kBlocks / 2 : 0, late = Cfg::kLate + kScaleRequests;
    constexpr int late_end = kEarly > 0 ? first + (kCycle - first) / 2 : kCycle;
    return r < late ? first + r * (late_end - first) / late : late_end + (r - late) * (kCycle - late_end) / (kEarly > 0 ? kEarly : 1);
  };
  constexpr std::integral_constant<int, 0> q0{};
  constexpr std::integral_constant<int, 1> q1{};
  constexpr std::integral_constant<int, 2> q2{};
  constexpr std::integral_constant<int, 3> q3{};
  constexpr std::true_type yes{};
  constexpr std::false_type no{};

  aim(place, rows_of(place));
  if (!place.zero) request_all_first(place.steps);
  using Stores = MxStores<Cfg, DT>;
  bool counted_stores = false;  // the last tile left between this one's first requests, in whole parts
  for (int turn = 1;; ++turn) {
    MxTilePlace next_place;
    bool more_tiles = false;
    Rows next_rows;
    float bias = 0.0f;
    if (Cfg::kResident) {
      more_tiles = place_of_turn<Cfg, kProblem>(p, schedule, table, turn, &next_place);
      if (more_tiles) next_rows = rows_of(next_place);
    }
    if (kProblem == kMxDense && p.bias && tid < Cfg::BN && place.col0 + tid < p.n) bias = load_bias<DT>(p.bias, place.col0 + tid, p.bias_f32);
    if (place.zero) {
      zero_tile<DT, Cfg>(p, place);
      if (!more_tiles) return;
      place = next_place;
      aim(place, next_rows);
      if (!place.zero) request_all_first(place.steps);
      counted_stores = false;
      continue;
    }
    const int steps = place.steps;
    // Lane (r = l & 31, g) accumulates, of row r of a block, columns 8 q + 4 g + 0 .. 3, q = 0 .. 3.
    f32x16 acc[TM][TN];
    constexpr f32x16 kZeros = {};
    // Step 0 has landed; what was queued behind it stays in flight.
    if (kDepth < steps) {
      if (Cfg::kResident && counted_stores) wait_for_dma_loads_but<at_most_63((kDepth - 1) * kRequests + kEarly + Stores::behind_step(0))>();
      else wait_for_dma_loads_but<(kDepth - 1) * kRequests + kEarly>();
    } else {
      wait_but_steps<kDepth - 1, kRequests>(steps - 1);
    }
    asm volatile("s_barrier" ::: "memory");

    u32x4 af[2][TM], bf[2][TN];
    int sa[TM], sb[TN], next_sa[TM], next_sb[TN];
    Place now = kFirst;
    const auto read_one = [&](const Place& at, int s, int r) FSH_INLINE {  // fragment r of quarter s: A's, then B's
      if (r < TM) af[s & 1][r] = read_frag(at, a0 + 32 * r, s);
      else bf[s & 1][r - TM] = read_frag(at, b0 + 32 * (r - TM), s);
    };
#pragma unroll
    for (int i = 0; i < TM; ++i) sa[i] = read_scale(now, a0 + 32 * i);
#pragma unroll
    for (int j = 0; j < TN; ++j) sb[j] = read_scale(now, b0 + 32 * j);
#pragma unroll
    for (int r = 0; r < kReads; ++r) read_one(now, 0, r);

    // Quarter s of a step.  Behind its MFMAs: the barrier and the first fragments
    // and scales of the step at `at`, the next one (quarter 3), or the fragments of
    // this one's next quarter; requests of the iteration that began with step
    // `left`, into that step's slots.
    const auto quarter = [&](auto s_tag, auto first_tag, auto more_tag, auto late_tag, auto early_tag, const Place& at, int left,
                             const Place& freed) FSH_INLINE {
      constexpr bool of_first = decltype(first_tag)::value;
      constexpr int s = decltype(s_tag)::value;
      constexpr bool more = decltype(more_tag)::value, late = decltype(late_tag)::value, early = decltype(early_tag)::value;
#pragma unroll
      for (int m = 0; m < kBlocks; ++m) {
        const int i = m % TM, j = m / TM;
        const u32x4 a = af[s & 1][i], b = bf[s & 1][j];
        const v8i32 av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
        const v8i32 bv = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(bv, av, s == 0 && of_first ? kZeros : acc[i][j], 4, 4, s, sb[j], s, sa[i]);
        __builtin_amdgcn_sched_barrier(0);
        if (s == 3 && more && m == 0) {
          if (late) {
            if (Cfg::kResident && counted_stores && left == 0) wait_for_dma_loads_but<at_most_63(kEarly + Stores::behind_step(1))>();
            else wait_for_dma_loads_but<(kDepth - 2) * kRequests + kEarly>();
          } else {
            wait_but_steps<kDepth - 2, kRequests>(steps - 2 - left);
          }
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        if (s < 3) {
          constexpr int per = (kReads + kBlocks - 1) / kBlocks;
#pragma unroll
          for (int q = 0; q < per; ++q)
            if (m * per + q < kReads) read_one(at, s + 1, m * per + q);
        } else if (more) {
          constexpr int per = (2 * kReads + kBlocks - 1) / kBlocks;
#pragma unroll
          for (int q = 0; q < per; ++q) {
            const int r = m * per + q;
            if (r < kReads) read_one(at, 0, r);
            else if (r < kReads + TM) next_sa[r - kReads] = read_scale(at, a0 + 32 * (r - kReads));
            else if (r < 2 * kReads) next_sb[r - kReads - TM] = read_scale(at, b0 + 32 * (r - kReads - TM));
          }
        }
#pragma unroll
        for (int r = 0; r < kRequests; ++r)
          if ((s == 3 ? 0 : s + 1) * kBlocks + m == behind_mfma(r)) {
            if (r < kScaleRequests) {
              if (late) request_scales(left + kDepth, freed, r);
            } else if (r < kScaleRequests + Cfg::kLate) {
              if (late) request(left + kDepth, freed, kEarly + r - kScaleRequests);
            } else if (early) {
              request(left + kDepth + 1, freed, r - kScaleRequests - Cfg::kLate);
            }
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const auto iteration = [&](int step, auto late, auto early) FSH_INLINE {
      const Place freed = now, next = place_after(now);
      quarter(q3, no, yes, late, early, next, step, freed);
#pragma unroll
      for (int i = 0; i < TM; ++i) sa[i] = next_sa[i];
#pragma unroll
      for (int j = 0; j < TN; ++j) sb[j] = next_sb[j];
      quarter(q0, no, yes, late, early, next, step, freed);
      quarter(q1, no, yes, late, early, next, step, freed);
      quarter(q2, no, yes, late, early, next, step, freed);
      now = next;
    };
    quarter(q0, yes, yes, no, no, now, 0, now);
    quarter(q1, yes, yes, no, no, now, 0, now);
    quarter(q2, yes, yes, no, no, now, 0, now);
    int step = 0;
    for (; step + kDepth + 1 < steps; ++step) iteration(step, yes, yes);
    if (step + kDepth < steps) iteration(step++, yes, no);
    for (; step + 1 < steps; ++step) iteration(step, no, no);
    quarter(q3, no, no, no, no, now, 0, now);
    if (kProblem == kMxDense && tid < Cfg::BN) bias_of_tile[tid] = bias;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the slots are free

    const MxTilePlace done = place;
    const bool request_next = Cfg::kResident && more_tiles && !next_place.zero;
    if (Cfg::kResident && more_tiles) {
      place = next_place;
      aim(place, next_rows);
    }
    // A part goes through LDS to leave as whole row pieces; while it is read back the next one is converted.
    constexpr int kElement = Stores::kElement, kCols = Stores::kCols, kParts = Stores::kParts;
    constexpr int kLanesPerRow = Stores::kPartBytes / 16, kRowsPerStore = 64 / kLanesPerRow, kPerLane = 16 / kElement;
    const int64_t wave_row = done.row0 + wm * Cfg::kWaveM, row_end = done.row0 + done.rows, wave_col = done.col0 + wn * Cfg::kWaveN;
    uint8_t* region = lds_bytes + Cfg::kStageOffset + wave * Cfg::kRegion;
    uint8_t* out = static_cast<uint8_t*>(p.out) + done.out_offset * kElement;
    const bool vec = p.ldo * kElement % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const bool whole = vec && wave_row + Cfg::kWaveM <= row_end && wave_col + Cfg::kWaveN <= p.n;
    const int store_row = lane / kLanesPerRow, store_col = lane % kLanesPerRow * kPerLane;
    const int rows_left = static_cast<int>(row_end - wave_row), cols_left = static_cast<int>(p.n - wave_col < Cfg::kWaveN ? p.n - wave_col : Cfg::kWaveN);
    const int vec_cols = vec ? (cols_left > 0 ? cols_left : 0) / kPerLane * kPerLane : 0;  // those that leave 16 bytes at a time
    uint8_t* const wave_out = out + (wave_row * p.ldo + wave_col) * kElement;
    uint8_t* const lane_out = wave_out + (store_row * p.ldo + store_col) * kElement;
    const int64_t row_bytes = p.ldo * kElement;
    u32x4 leaving[Stores::kStores];
    // (opaque: the compiler multiplies it out ahead of all tiles otherwise, and spills)
    int64_t store_bytes = kRowsPerStore * row_bytes;
    asm volatile("" : "+s"(store_bytes));
    const auto store_one = [&](auto plain, int part, int s) FSH_INLINE {
      const int row = part / (Cfg::kWaveN / kCols) * 32 + s * kRowsPerStore, col = part % (Cfg::kWaveN / kCols) * kCols;
      if (plain.value || (row + store_row < rows_left && col + store_col < vec_cols))
        __builtin_nontemporal_store(leaving[s], reinterpret_cast<u32x4*>(lane_out + row / kRowsPerStore * store_bytes + col * kElement));
    };
    const auto store_rest = [&](int part) FSH_INLINE {
      const int row = part / (Cfg::kWaveN / kCols) * 32, col = part % (Cfg::kWaveN / kCols) * kCols;
      // What is left of rows that are not whole 16-byte pieces, out of the staging.  Not unrolled: the code of whole
      // tiles has to stay in the instruction cache.
      if (vec_cols < cols_left) {
#pragma unroll 1
        for (int e = lane; e < 32 * kCols; e += 64) {
          const int r = e / kCols, c = e % kCols;
          if (row + r >= rows_left || col + c < vec_cols || col + c >= cols_left) continue;
          const uint8_t* from = region + r * Cfg::kPitch + c * kElement;
          uint8_t* there = wave_out + (row + r) * row_bytes + (col + c) * kElement;
          if (kElement == 4) *reinterpret_cast<uint32_t*>(there) = *reinterpret_cast<const uint32_t*>(from);
          else *reinterpret_cast<uint16_t*>(there) = *reinterpret_cast<const uint16_t*>(from);
        }
      }
    };
    const auto leave = [&](auto plain) FSH_INLINE {
      static_for<kParts>([&](auto part_tag) FSH_INLINE {
        constexpr int part = decltype(part_tag)::value;
        constexpr int i = part / (Cfg::kWaveN / kCols), j0 = part % (Cfg::kWaveN / kCols) * (kCols / 32);
        // (said to be in accumulation registers up to here: the compiler copies them all out ahead otherwise, and spills)
        float v[kCols / 32][16];
#pragma unroll
        for (int j = 0; j < kCols / 32; ++j) {
          asm volatile("" : "+a"(acc[i][j0 + j]));
#pragma unroll
          for (int t = 0; t < 16; ++t) v[j][t] = acc[i][j0 + j][t];
        }
        if (kProblem == kMxDense && p.bias) {
#pragma unroll
          for (int j = 0; j < kCols / 32; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 add = *reinterpret_cast<const f32x4*>(bias_of_tile + wn * Cfg::kWaveN + 32 * (j0 + j) + 8 * q + 4 * group);
#pragma unroll
              for (int t = 0; t < 4; ++t) v[j][4 * q + t] += add[t];
            }
        }
        // (the part before leaves between the conversions)
        uint32_t words[Stores::kWords];
        constexpr int kPerStore = Stores::kWords / Stores::kStores;
        static_for<Stores::kStores>([&](auto s_tag) FSH_INLINE {
          constexpr int s = decltype(s_tag)::value;
#pragma unroll
          for (int w = s * kPerStore; w < (s + 1) * kPerStore; ++w) {
            if (DT == FSH_DT_F32) words[w] = f32_as_u32(v[0][w]);
            else if (DT == FSH_DT_BF16) words[w] = pack_bf16x2(v[w / 8][2 * w % 16], v[w / 8][2 * w % 16 + 1]);
            else words[w] = pack_f16x2(v[w / 8][2 * w % 16], v[w / 8][2 * w % 16 + 1]);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (part > 0) store_one(plain, part - 1, s);
          __builtin_amdgcn_sched_barrier(0);
        });
        if (part > 0 && !plain.value) store_rest(part - 1);
        wave_lds_sync();
        constexpr int kPerPiece = kElement;  // dwords of four columns, less what 16 bits save: 2 or 4
#pragma unroll
        for (int piece = 0; piece < Stores::kWords / kPerPiece; ++piece) {
          uint8_t* at = region + frag_row * Cfg::kPitch + (32 * (piece / 4) + 8 * (piece % 4) + 4 * group) * kElement;
          const uint32_t* w = words + piece * kPerPiece;
          if constexpr (kElement == 4) *reinterpret_cast<u32x4*>(at) = u32x4{w[0], w[1], w[2], w[3]};
          else *reinterpret_cast<u32x2*>(at) = u32x2{w[0], w[1]};
        }
        wave_lds_sync();
#pragma unroll
        for (int s = 0; s < Stores::kStores; ++s)
          leaving[s] = *reinterpret_cast<const u32x4*>(region + (s * kRowsPerStore + store_row) * Cfg::kPitch + store_col * kElement);
        __builtin_amdgcn_sched_barrier(0);
        if (plain.value || request_next)
          static_for<2 * kRequests>([&](auto r) FSH_INLINE {
            if constexpr (Cfg::kResident && Stores::part_of_request(decltype(r)::value) == part) request_first(plain, place.steps, r);
          });
        __builtin_amdgcn_sched_barrier(0);
      });
      static_for<Stores::kStores>([&](auto s) FSH_INLINE { store_one(plain, kParts - 1, decltype(s)::value); });
      if (!plain.value) store_rest(kParts - 1);
    };
    // A whole tile before a tile of some length, as most are, leaves without a branch.
    if (Cfg::kResident && whole && request_next && kDepth < place.steps) leave(yes);
    else leave(no);
    counted_stores = whole;
    if (!more_tiles) return;
    // The staging's slot is the third step's: every wave has to be done with it.
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (!place.zero) request_first_early(place.steps);
  }
}

}  // namespace
}  // namespace fsh
