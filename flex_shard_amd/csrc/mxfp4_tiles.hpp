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

namespace fsh {
namespace {

typedef int v8i32 __attribute__((ext_vector_type(8)));

enum MxProblem {
  kMxDense,      // one product
  kMxRows,       // rows of a in segments, one per expert, each against that expert's b
  kMxOverRows,   // per expert the product over its own (padded) columns of a and b: [experts][m][n]
};

struct MxGemmParams {
  const uint8_t* a;   // [a_rows][lda]
  const uint8_t* as;  // [k / 256][a_rows][8]
  const uint8_t* b;
  const uint8_t* bs;
  void* out;
  const void* bias;  // [n] of the output's type, or null
  int64_t m, n, k;   // k a multiple of 256; kMxOverRows: of all segments
  int64_t a_rows, b_rows, lda, ldb, ldo;
  int32_t out_dtype;
  int32_t experts, top_k;
  const int32_t* offsets;         // [experts + 1]
  const int32_t* padded_offsets;  // [experts + 1] (kMxOverRows)
  const int32_t* source;          // kMxRows: row r of the segments is row source[r] / top_k of a, or null
  GemmParams schedule;            // tile order
};

// A tile of WM x WN waves, each TM x TN blocks of 16 x 16.  A k-step is 256
// columns: 128 bytes and 8 scale bytes of every row.
template <int WM_, int WN_, int TM_, int TN_, int kDepth_>
struct MxTile {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, kDepth = kDepth_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves, kWaveM = 16 * TM, kWaveN = 16 * TN;
  static constexpr int BM = WM * kWaveM, BN = WN * kWaveN, kRowBytes = 128;
  static constexpr int kRequestRows = 8 * kWaves;  // rows that one request of every wave fills
  static constexpr int kRequestsA = BM / kRequestRows, kRequests = (BM + BN) / kRequestRows;
  static constexpr int kDataBytes = (BM + BN) * kRowBytes;
  // Scales: two planes (the words' lower and upper half) of BM + BN dwords, 64 by a request.
  static constexpr int kScaleRequests = 2 * (BM + BN) / 64 / kWaves, kPlaneBytes = 4 * (BM + BN);
  static constexpr int kStageBytes = kDataBytes + 2 * kPlaneBytes;
  static constexpr int kLdsBytes = kDepth * kStageBytes;
  static constexpr int kPitch = kWaveN * 2 + 16, kRegion = 32 * kPitch;  // epilogue staging of a wave, bytes
  static_assert(kLdsBytes <= 160 * 1024 && kWaves * kRegion <= kLdsBytes, "LDS of a compute unit");
  static_assert(BM % kRequestRows == 0 && BN % kRequestRows == 0, "whole requests");
  static_assert(BM % 64 == 0 && BN % 64 == 0 && kScaleRequests * kWaves * 32 == BM + BN, "scales by 64, the same for every wave");
  static_assert(TM % 2 == 0, "the epilogue stages 32 rows at a time");
};

// Where a tile lies.
struct MxTilePlace {
  int64_t row0, rows;    // output rows [row0, row0 + rows) of those that exist
  int64_t a_row0;        // of the operand (before `source`)
  int64_t col0, b_row0;  // output columns from col0 on; row of b that column 0 is
  int64_t out_offset;    // elements
  int64_t first_step, steps;
  bool zero;             // rows without a product: zeros
};

// Which expert and rows m-tile t of segments cut into tiles of BM rows is.  The
// rows behind the last segment count as one more segment.
template <int BM>
__device__ __forceinline__ bool find_segment_tile(const MxGemmParams& p, int t, int* expert, int64_t* row0, int64_t* rows) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int before = 0;
  for (int first = 0; first <= p.experts; first += 64) {
    const int e = first + lane;
    int64_t begin = 0, end = 0;
    if (e <= p.experts) {
      begin = p.offsets[e];
      end = e < p.experts ? p.offsets[e + 1] : p.m;
    }
    const int tiles = static_cast<int>((end - begin + BM - 1) / BM);
    int sum = tiles;  // inclusive scan over the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int other = __shfl_up(sum, off, kWave);
      if (lane >= off) sum += other;
    }
    const uint64_t mine = __ballot(t < before + sum);
    if (mine) {
      const int owner = __builtin_ctzll(mine);
      const int at = t - before - (__shfl(sum, owner, kWave) - __shfl(tiles, owner, kWave));
      *expert = first + owner;
      const int64_t b0 = __shfl(static_cast<int>(begin), owner, kWave), e0 = __shfl(static_cast<int>(end), owner, kWave);
      *row0 = uniform_i64(b0 + static_cast<int64_t>(at) * BM);
      *rows = uniform_i64(e0) - *row0 < BM ? uniform_i64(e0) - *row0 : BM;
      *expert = uniform_i32(*expert);
      return true;
    }
    before += __shfl(sum, 63, kWave);
  }
  return false;
}

template <typename Cfg, int kProblem>
__device__ __forceinline__ bool place_of_workgroup(const MxGemmParams& p, MxTilePlace* place) {
  int64_t batch;
  int tm, tn;
  if (!tile_of_workgroup(p.schedule, blockIdx.x, &batch, &tm, &tn)) return false;
  tm = uniform_i32(tm);
  tn = uniform_i32(tn);
  place->zero = false;
  place->out_offset = 0;
  place->first_step = 0;
  place->steps = p.k / kMxColumns;
  place->col0 = static_cast<int64_t>(tn) * Cfg::BN;
  place->b_row0 = 0;
  if (kProblem == kMxRows) {
    int expert;
    if (!find_segment_tile<Cfg::BM>(p, tm, &expert, &place->row0, &place->rows)) return false;
    place->zero = expert == p.experts;
    place->b_row0 = static_cast<int64_t>(expert) * p.n;
  } else {
    place->row0 = static_cast<int64_t>(tm) * Cfg::BM;
    place->rows = p.m - place->row0 < Cfg::BM ? p.m - place->row0 : Cfg::BM;
    if (kProblem == kMxOverRows) {
      const int expert = uniform_i32(static_cast<int>(batch));
      place->first_step = uniform_i32(p.padded_offsets[expert]) / kMxColumns;
      place->steps = uniform_i32(p.padded_offsets[expert + 1]) / kMxColumns - place->first_step;
      place->zero = place->steps == 0;
      place->out_offset = expert * p.m * p.n;
    }
  }
  place->a_row0 = place->row0;
  return true;
}

template <int DT, typename Cfg>
__device__ __forceinline__ void zero_tile(const MxGemmParams& p, const MxTilePlace& place) {
  for (int i = threadIdx.x; i < Cfg::BM * Cfg::BN; i += Cfg::kThreads) {
    const int64_t r = i / Cfg::BN, col = place.col0 + i % Cfg::BN;
    if (r < place.rows && col < p.n) store_element<DT>(p.out, place.out_offset + (place.row0 + r) * p.ldo + col, 0.0f);
  }
}

template <typename Cfg, int kProblem, int DT>
__global__ __launch_bounds__(Cfg::kThreads, Cfg::kWaves / 4 < 1 ? 1 : Cfg::kWaves / 4) void mxfp4_gemm_kernel(const MxGemmParams p) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds_bytes[];
  constexpr int TM = Cfg::TM, TN = Cfg::TN, kRequests = Cfg::kRequests, kRequestsA = Cfg::kRequestsA;
  MxTilePlace place;
  if (!place_of_workgroup<Cfg, kProblem>(p, &place)) return;  // whole workgroup
  if (place.zero) {
    zero_tile<DT, Cfg>(p, place);
    return;
  }
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;

  // Row i of the tile's operand A or B.  Rows past the last are read from the
  // last (their products are not stored).
  const auto a_row = [&](int i) -> int64_t {
    int64_t row = place.a_row0 + (i < place.rows ? i : place.rows - 1);
    if (kProblem == kMxRows && p.source) row = p.source[row] / p.top_k;
    return row;
  };
  const auto b_row = [&](int i) -> int64_t {
    const int64_t col = place.col0 + i;
    return place.b_row0 + (col < p.n ? col : p.n - 1);
  };
  // Data: request c of a wave fills rows [kRequestRows c + 8 wave, +8), lane l
  // slot l & 7 of row l >> 3.  Slot s of row r holds the 16-byte chunk 2 g + h
  // where g + 4 h = s ^ ((r >> 1) & 7): lane group g of a fragment read takes
  // chunks 2 g and 2 g + 1, for its two k-halves, from slots that do not meet in
  // the banks.
  const int fill_row = lane >> 3;
  const int fill_slot = (lane & 7) ^ (((8 * wave + fill_row) >> 1) & 7);
  const int fill_chunk = 2 * (fill_slot & 3) + (fill_slot >> 2);
  // Offsets from the operands' first rows of the tile (from the matrix where rows are gathered).
  const bool gathered = kProblem == kMxRows && p.source;
  const int64_t a_first = gathered ? 0 : place.a_row0, b_first = place.b_row0 + place.col0;
  uint32_t voff[kRequests];
#pragma unroll
  for (int c = 0; c < kRequests; ++c) {
    const int r = Cfg::kRequestRows * (c < kRequestsA ? c : c - kRequestsA) + 8 * wave + fill_row;
    voff[c] = static_cast<uint32_t>((c < kRequestsA ? (a_row(r) - a_first) * p.lda : (b_row(r) - b_first) * p.ldb) + fill_chunk * 16);
  }
  const uint8_t* a_data = uniform_ptr(p.a + a_first * p.lda + place.first_step * Cfg::kRowBytes);
  const uint8_t* b_data = uniform_ptr(p.b + b_first * p.ldb + place.first_step * Cfg::kRowBytes);
  // Scales: request q = kScaleRequests wave + i fills plane q & 1 of rows [64 (q >> 1), +64).
  uint32_t scale_voff[Cfg::kScaleRequests];
  const uint8_t* scale_src[Cfg::kScaleRequests];
  int64_t scale_step[Cfg::kScaleRequests];
  uint32_t scale_lds[Cfg::kScaleRequests];
#pragma unroll
  for (int i = 0; i < Cfg::kScaleRequests; ++i) {
    const int q = Cfg::kScaleRequests * wave + i, first = 64 * (q >> 1);
    const bool of_a = first < Cfg::BM;
    scale_step[i] = (of_a ? p.a_rows : p.b_rows) * 8;
    scale_src[i] = uniform_ptr((of_a ? p.as : p.bs) + place.first_step * scale_step[i] + 4 * (q & 1));
    scale_voff[i] = static_cast<uint32_t>((of_a ? a_row(first + lane) : b_row(first - Cfg::BM + lane)) * 8);
    scale_lds[i] = Cfg::kDataBytes + (q & 1) * Cfg::kPlaneBytes + first * 4;
  }
  typedef __attribute__((address_space(3))) uint8_t* lds_address;
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_address)lds_bytes));
  const int steps = static_cast<int>(place.steps);
  const auto request = [&](int step, uint32_t stage) {
#pragma unroll
    for (int c = 0; c < kRequests; ++c)
      dma_load_16(voff[c], (c < kRequestsA ? a_data : b_data) + static_cast<int64_t>(step) * Cfg::kRowBytes,
                  lds_base + stage + wave * 1024, c * Cfg::kRequestRows * Cfg::kRowBytes);
#pragma unroll
    for (int i = 0; i < Cfg::kScaleRequests; ++i)
      dma_touch_4(scale_voff[i], scale_src[i] + step * scale_step[i], lds_base + stage + scale_lds[i]);
  };

  const int frag_row = lane & 15, group = lane >> 4;
  uint32_t frag_off[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    frag_off[h] = static_cast<uint32_t>(frag_row * Cfg::kRowBytes + (((group + 4 * h) ^ ((frag_row >> 1) & 7)) * 16));
  const uint32_t scale_off = static_cast<uint32_t>(Cfg::kDataBytes + (group >> 1) * Cfg::kPlaneBytes + frag_row * 4 + (group & 1) * 2);
  // 16 rows from `row` of the tile (A's rows, then B's) of the stage at `stage`
  const auto read_frag = [&](uint32_t stage, int row, int h) -> v8i32 {
    const u32x4 v = *reinterpret_cast<const u32x4*>(lds_bytes + stage + row * Cfg::kRowBytes + frag_off[h]);
    return v8i32{static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w), 0, 0, 0, 0};
  };
  const auto read_scale = [&](uint32_t stage, int row) -> int {
    return *reinterpret_cast<const uint16_t*>(lds_bytes + stage + scale_off + row * 4);
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  constexpr int kInFlight = kRequests + Cfg::kScaleRequests;  // of a step, per wave
#pragma unroll
  for (int s = 0; s + 1 < Cfg::kDepth; ++s)
    if (s < steps) request(s, s * Cfg::kStageBytes);
  uint32_t stage = 0, free_stage = (Cfg::kDepth - 1) * Cfg::kStageBytes;
  const int a0 = wm * Cfg::kWaveM, b0 = Cfg::BM + wn * Cfg::kWaveN;
  for (int step = 0; step < steps; ++step) {
    // This wave's part of the step has landed, then everybody's; behind the
    // barrier nobody reads the stage of the step before any more.
    if (Cfg::kDepth > 2 && step + 1 < steps) wait_for_dma_loads_but<kInFlight*(Cfg::kDepth > 2 ? Cfg::kDepth - 2 : 0)>();
    else wait_for_dma_loads();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (step + Cfg::kDepth - 1 < steps) request(step + Cfg::kDepth - 1, free_stage);
    int sa[TM], sb[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) sa[i] = read_scale(stage, a0 + 16 * i);
#pragma unroll
    for (int j = 0; j < TN; ++j) sb[j] = read_scale(stage, b0 + 16 * j);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v8i32 af[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) af[i] = read_frag(stage, a0 + 16 * i, h);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const v8i32 bf = read_frag(stage, b0 + 16 * j, h);
#pragma unroll
        for (int i = 0; i < TM; ++i)
          acc[i][j] = h == 0 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf, af[i], acc[i][j], 4, 4, 0, sb[j], 0, sa[i])
                             : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf, af[i], acc[i][j], 4, 4, 1, sb[j], 1, sa[i]);
      }
    }
    free_stage = stage;
    stage = stage + Cfg::kStageBytes == Cfg::kLdsBytes ? 0 : stage + Cfg::kStageBytes;
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stages become the epilogue's

  // Lane (r = lane & 15, g) holds columns 4 g .. 4 g + 3 of row r of each block.
  const int64_t wave_row = static_cast<int64_t>(wm) * Cfg::kWaveM, wave_col = place.col0 + wn * Cfg::kWaveN;
  const int64_t row_end = place.row0 + place.rows;
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t col = wave_col + 16 * j + 4 * group + t;
        const float bias = col < p.n ? load_element<DT>(p.bias, col) : 0.0f;
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j][t] += bias;
      }
  }
  if (DT == FSH_DT_F32) {
    float* out = static_cast<float*>(p.out) + place.out_offset;
    const bool vec = p.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t row = place.row0 + wave_row + 16 * i + frag_row;
      if (row >= row_end) continue;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t col = wave_col + 16 * j + 4 * group;
        if (vec && col + 4 <= p.n) {
          *reinterpret_cast<f32x4*>(out + row * p.ldo + col) = acc[i][j];
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (col + t < p.n) out[row * p.ldo + col + t] = acc[i][j][t];
        }
      }
    }
  } else {
    // 16-bit values go through LDS, 32 rows at a time, to leave as whole row pieces.
    uint8_t* region = lds_bytes + wave * Cfg::kRegion;
    uint16_t* out = static_cast<uint16_t*>(p.out) + place.out_offset;
#pragma unroll
    for (int i = 0; i < TM; i += 2) {
#pragma unroll
      for (int ii = 0; ii < 2; ++ii)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const f32x4 v = acc[i + ii][j];
          u32x2 w;
          if (DT == FSH_DT_BF16) w = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
          else w = u32x2{f32_to_f16_bits(v[0]) | (f32_to_f16_bits(v[1]) << 16), f32_to_f16_bits(v[2]) | (f32_to_f16_bits(v[3]) << 16)};
          *reinterpret_cast<u32x2*>(region + (ii * 16 + frag_row) * Cfg::kPitch + (16 * j + 4 * group) * 2) = w;
        }
      wave_lds_sync();
      store_wave_image<32, Cfg::kWaveN, Cfg::kPitch>(region, out, p.ldo, place.row0 + wave_row + 16 * i, wave_col, row_end, p.n, lane);
      wave_lds_sync();
    }
  }
}

}  // namespace
}  // namespace fsh
