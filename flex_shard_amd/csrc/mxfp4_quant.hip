// Quantization of bf16, fp16 and fp32 matrices to microscaled 4-bit floats, in
// runs of 32 along the rows (the operand of a product over the columns), along
// the columns (the transpose, an operand of a product over the rows), or both
// from one read; and back.
//
//   run of 32: e = exponent field of the largest magnitude, byte = max(e - 2, 0),
//   q = E2M1(x * 2^(127 - byte)), to nearest even, at most 6
//
// Multiplying by a power of two is exact, so the only rounding is E2M1's own.
// Bound by memory: an element is read once (2 or 4 bytes) and leaves as 17/32 of
// a byte per form.  Measured (us, TB/s of these bytes; a large copy reaches 4.9):
//   bf16 8192 x 14336    rows 50.5, 5.9   columns 58.6, 5.1   both 75.7, 4.8   back 45.2, 6.6
//   fp32 14336 x 4096    rows 49.5, 5.4   columns 49.6, 5.4   both 56.7, 5.2   back 38.6, 6.9
#include "mxfp4.hpp"

namespace fsh {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxGrid = (1LL << 32) / kThreads - 1;  // a launch's threads are counted in 32 bits

struct MxQuantParams {
  const uint8_t* x;
  int64_t rows, cols, ldx;  // elements; of one matrix of the stack
  int32_t vec;              // rows are 16-byte aligned
  // Rows: [batch * rows][ld_row] and [..][batch * rows][8]
  uint8_t* q_row;
  uint8_t* s_row;
  int64_t ld_row, table_rows;
  // Columns: [batch * cols][ld_col] and [..][batch * cols][8]
  uint8_t* q_col;
  uint8_t* s_col;
  int64_t ld_col, table_cols;
  float* column_sums;  // [ceil(rows / 128)][cols] or null (one matrix)
  int64_t tiles_c, tiles_r;
  // Rows in segments, one per expert: padded row p of segment e, from
  // padded_offsets[e] on, is row offsets[e] + p - padded_offsets[e] of the sorted
  // ones, or of x the row source[that] / top_k.
  const int32_t* offsets;
  const int32_t* padded_offsets;
  const int32_t* source;
  int32_t experts, top_k;
};

// A lane's eight columns of a row, 16 lanes 128 columns, quantized: the data of
// the lane and, in lane 0 of the 16, the four scale bytes.
template <int DT>
__device__ __forceinline__ uint32_t quantize_row_piece(const Raw8<DT>& raw, uint32_t* scales) {
  uint32_t m = max_magnitude8(raw);
  m = dpp_max_u32<0xB1, 0xF>(m);  // quad_perm [1,0,3,2]
  m = dpp_max_u32<0x4E, 0xF>(m);  // quad_perm [2,3,0,1]: the four lanes of a run
  const uint32_t byte = mx_scale_byte(magnitude_bits_to_f32<DT>(m));
  // lanes 4, 8 and 12 of the 16 to lane 0 (row_shl)
  uint32_t all = byte;
  all |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(byte), 0x104, 0xF, 0xF, true)) << 8;
  all |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(byte), 0x108, 0xF, 0xF, true)) << 16;
  all |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(byte), 0x10C, 0xF, 0xF, true)) << 24;
  *scales = all;
  return mx_quantize8(raw, mx_scale(byte));
}

// Stores what quantize_row_piece gave for columns [col, col + 8) of table row `row`.
__device__ __forceinline__ void store_row_piece4(const MxQuantParams& p, int64_t row, int64_t col, uint32_t data, uint32_t scales) {
  *reinterpret_cast<uint32_t*>(p.q_row + row * p.ld_row + col / 2) = data;
  if ((threadIdx.x & 15) == 0)
    *reinterpret_cast<uint32_t*>(p.s_row + ((col / kMxColumns) * p.table_rows + row) * 8 + (col % kMxColumns) / kMxBlock) = scales;
}

// 16 rows x 512 columns per workgroup, a row's 512 by one wave: a run is four lanes,
// its maximum two steps across lanes, and nothing goes through LDS.
constexpr int kRowTileRows = 16, kRowTileCols = 512;
template <int DT>
__global__ __launch_bounds__(kThreads) void mxfp4_quantize_rows_kernel(const MxQuantParams p) {
  const int64_t tile_r = blockIdx.x / p.tiles_c, tile_c = blockIdx.x % p.tiles_c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = tile_c * kRowTileCols + lane * 8;
  if (col >= p.ld_row * 2) return;
  Raw8<DT> raw[kRowTileRows / 4];
#pragma unroll
  for (int i = 0; i < kRowTileRows / 4; ++i) {
    const int64_t row = tile_r * kRowTileRows + 4 * i + wave;
    raw[i] = load_raw8<DT>(p.x + (row * p.ldx + col) * element_bytes<DT>(), row < p.rows ? p.cols - col : 0, p.vec);
  }
#pragma unroll
  for (int i = 0; i < kRowTileRows / 4; ++i) {
    const int64_t row = tile_r * kRowTileRows + 4 * i + wave;
    uint32_t scales;
    const uint32_t data = quantize_row_piece(raw[i], &scales);
    if (row < p.rows) store_row_piece4(p, row, col, data, scales);
  }
}

// 128 x 128 tiles.  The tile goes through LDS as it was read; a thread then owns
// two columns of 32 rows (a wave reads 64 neighbouring pairs of a row at a time),
// so a column's run lies in one thread.  Its 16 bytes go through LDS once more to
// leave as 64 bytes per column.  With kRows the row runs leave from the registers
// that the tile was loaded into.  Gathered rows (65536 x 7168 of 8192 tokens' rows,
// 234 us) cost what as many rows of a matrix do: a token's choices are in the tiles
// of different experts, so its row crosses into an L2 once for each, out of the
// memory-side cache if not from memory.  By the counters the L2s miss 1.14 GB (1.19
// of a matrix), 4.9 TB/s, the rate of a copy; the 9 vector instructions an element
// (5) would take about half of the time.  Neighbouring tiles on one XCD were slower
// (8192 x 14336 both 77 to 84 us).
constexpr int kTile = 128;
template <int DT, bool kRows>
__global__ __launch_bounds__(kThreads) void mxfp4_quantize_columns_kernel(const MxQuantParams p) {
  constexpr int kElement = element_bytes<DT>(), kPitch = kTile * kElement;
  __shared__ __attribute__((aligned(16))) uint8_t tile[kTile * kPitch];
  const int tid = threadIdx.x;
  const int64_t tile_c = blockIdx.x % p.tiles_c, tile_r = blockIdx.x / p.tiles_c % p.tiles_r, batch = blockIdx.x / p.tiles_c / p.tiles_r;
  const int64_t c0 = tile_c * kTile, out_r0 = tile_r * kTile;
  // the tile's first row and how many of its rows exist
  int64_t r0 = out_r0, rows_left = p.rows - out_r0;
  if (p.experts > 0) {
    const int e = count_not_above(p.padded_offsets + 1, p.experts, out_r0);
    if (e >= p.experts) return;  // behind the last segment (whole workgroup)
    r0 = p.offsets[e] + (out_r0 - p.padded_offsets[e]);
    rows_left = p.offsets[e + 1] - r0;
  }
  const int64_t col = c0 + (tid & 15) * 8;
  const uint8_t* x = p.x + batch * p.rows * p.ldx * kElement;
  Raw8<DT> raw[kTile / 16];
#pragma unroll
  for (int i = 0; i < kTile / 16; ++i) {
    const int r = 16 * i + (tid >> 4);
    int64_t row = r0 + r;
    if (p.source && r < rows_left) row = p.source[row] / p.top_k;
    raw[i] = load_raw8<DT>(x + (row * p.ldx + col) * kElement, r < rows_left ? p.cols - col : 0, p.vec);
  }
#pragma unroll
  for (int i = 0; i < kTile / 16; ++i) {
    uint8_t* at = tile + (16 * i + (tid >> 4)) * kPitch + (tid & 15) * 8 * kElement;
#pragma unroll
    for (int j = 0; j < kElement / 2; ++j) *reinterpret_cast<u32x4*>(at + 16 * j) = raw[i].v[j];
  }
  if (kRows && col < p.ld_row * 2) {
#pragma unroll
    for (int i = 0; i < kTile / 16; ++i) {
      const int r = 16 * i + (tid >> 4);
      uint32_t scales;
      const uint32_t data = quantize_row_piece(raw[i], &scales);
      if (r < rows_left) store_row_piece4(p, batch * p.rows + r0 + r, col, data, scales);
    }
  }
  if (c0 >= p.cols) return;  // columns that only the row runs are padded with (whole workgroup)
  __syncthreads();

  const int pair = tid & 63, block = tid >> 6;
  u32x4 data[2];
  uint32_t bytes[2];
  float sums[2] = {0.0f, 0.0f};
  const uint8_t* const columns = tile + block * 32 * kPitch + pair * 2 * kElement;
  if constexpr (DT == FSH_DT_F32) {
    f32x2 f[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = *reinterpret_cast<const f32x2*>(columns + i * kPitch);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const uint32_t b = f32_as_u32(f[i][c]) & 0x7FFFFFFFu;
        m = b > m ? b : m;
      }
      bytes[c] = mx_scale_byte(m);
      const float scale = mx_scale(bytes[c]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = f[8 * w + i][c];
        data[c][w] = mx_quantize8(g, scale);
      }
      if (p.column_sums) {
#pragma unroll
        for (int i = 0; i < 32; ++i) sums[c] += f[i][c];
      }
    }
  } else {
    uint32_t f[32], m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = *reinterpret_cast<const uint32_t*>(columns + i * kPitch);
#pragma unroll
    for (int i = 0; i < 32; ++i) m = pk_max_u16(m, f[i] & 0x7FFF7FFFu);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bytes[c] = mx_scale_byte(magnitude_bits_to_f32<DT>(c ? m >> 16 : m & 0xFFFFu));
      const float scale = mx_scale(bytes[c]);
      constexpr uint32_t kLow = 0x05040100u, kHigh = 0x07060302u;  // the halves of two rows that are a column's
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t pick = c ? kHigh : kLow;
        uint32_t d = 0;
        d = mx_quantize_pair<DT, 0>(d, __builtin_amdgcn_perm(f[8 * w + 1], f[8 * w], pick), scale);
        d = mx_quantize_pair<DT, 1>(d, __builtin_amdgcn_perm(f[8 * w + 3], f[8 * w + 2], pick), scale);
        d = mx_quantize_pair<DT, 2>(d, __builtin_amdgcn_perm(f[8 * w + 5], f[8 * w + 4], pick), scale);
        d = mx_quantize_pair<DT, 3>(d, __builtin_amdgcn_perm(f[8 * w + 7], f[8 * w + 6], pick), scale);
        data[c][w] = d;
      }
      if (p.column_sums) {
#pragma unroll
        for (int i = 0; i < 32; ++i) sums[c] += half_of_pair<DT>(f[i], c);
      }
    }
  }
  __syncthreads();
  // From here on the tile's LDS holds the results: 128 bytes per pair of columns,
  // 16 by 16 in slots that differ from pair to pair; scales; sums.
  uint8_t* const scale_bytes = tile + kTile * 64;
  float* const partial = reinterpret_cast<float*>(tile + kTile * 64 + kTile * 4);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    *reinterpret_cast<u32x4*>(tile + pair * 128 + (((block + 4 * c) ^ (pair & 7)) * 16)) = data[c];
    scale_bytes[(2 * pair + c) * 4 + block] = static_cast<uint8_t>(bytes[c]);
    if (p.column_sums) partial[block * kTile + 2 * pair + c] = sums[c];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = 64 * i + (tid >> 2), b = tid & 3;
    const u32x4 v = *reinterpret_cast<const u32x4*>(tile + (c >> 1) * 128 + (((b + 4 * (c & 1)) ^ ((c >> 1) & 7)) * 16));
    if (c0 + c < p.cols) *reinterpret_cast<u32x4*>(p.q_col + (batch * p.cols + c0 + c) * p.ld_col + out_r0 / 2 + b * 16) = v;
  }
  if (tid < kTile && c0 + tid < p.cols) {
    const int64_t row = batch * p.cols + c0 + tid;
    *reinterpret_cast<uint32_t*>(p.s_col + ((out_r0 / kMxColumns) * p.table_cols + row) * 8 + (out_r0 % kMxColumns) / kMxBlock) =
        *reinterpret_cast<const uint32_t*>(scale_bytes + tid * 4);
    if (p.column_sums && rows_left > 0)
      p.column_sums[tile_r * p.cols + c0 + tid] =
          partial[tid] + partial[kTile + tid] + partial[2 * kTile + tid] + partial[3 * kTile + tid];
  }
}

struct MxDequantParams {
  const uint8_t* q;
  const uint8_t* s;
  uint8_t* out;
  int64_t rows, cols, ldq, ldo, groups;  // groups of 16 bytes' columns per row
  int32_t vec;
};
// A thread writes 16 bytes, past the caches: 8192 x 14336 to bf16 69 us with plain
// stores, 46 so; with 32 bytes of fp32 in two stores they do harm (14336 x 4096 55 / 91).
template <int DT>
__global__ __launch_bounds__(kThreads) void mxfp4_dequantize_kernel(const MxDequantParams p) {
  constexpr int kColumns = 16 / element_bytes<DT>();
  const int64_t total = p.rows * p.groups;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / p.groups, col = (i - row * p.groups) * kColumns;
    const uint8_t* at = p.q + row * p.ldq + col / 2;
    const uint32_t w = kColumns == 8 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at);
    const float scale = mx_scale(p.s[((col / kMxColumns) * p.rows + row) * 8 + (col % kMxColumns) / kMxBlock]);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    const float f[8] = {a.x * scale, a.y * scale, b.x * scale, b.y * scale, c.x * scale, c.y * scale, d.x * scale, d.y * scale};
    uint8_t* out = p.out + (row * p.ldo + col) * element_bytes<DT>();
    if (p.vec && col + kColumns <= p.cols) {
      if constexpr (DT == FSH_DT_F32) __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4*>(out));
      else __builtin_nontemporal_store(pack8<DT>(f), reinterpret_cast<u32x4*>(out));
    } else {
#pragma unroll
      for (int c2 = 0; c2 < kColumns; ++c2)
        if (col + c2 < p.cols) store_element<DT>(out, c2, f[c2]);
    }
  }
}

// out[c] = sum over runs of sums[run][c].  64 columns per workgroup, four
// quarters of the runs side by side.
template <int DT>
__global__ __launch_bounds__(kThreads) void sum_runs_kernel(const float* sums, void* out, int64_t runs, int64_t cols) {
  __shared__ float part[4][64];
  const int lane = threadIdx.x & 63, quarter = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float sum = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t r = quarter; r < runs; r += 4) sum += sums[r * cols + c];
  }
  part[quarter][lane] = sum;
  __syncthreads();
  if (quarter == 0 && c < cols) store_element<DT>(out, c, part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane]);
}

// Checks that both quantizers share; p.x .. p.column_sums are set.
int quantize_checks(MxQuantParams& p, int32_t dtype, const char* who) {
  if (!known_dtype(dtype)) return fail(FSH_EINVAL, "%s: unknown dtype %d", who, dtype);
  if ((p.q_row == nullptr) != (p.s_row == nullptr) || (p.q_col == nullptr) != (p.s_col == nullptr))
    return fail(FSH_EINVAL, "%s: data and scales of a form go together", who);
  if (!p.q_row && !p.q_col) return fail(FSH_EINVAL, "%s: no output", who);
  if (!p.x) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (p.ldx < p.cols) return fail(FSH_EINVAL, "%s: ldx %lld < cols %lld", who, (long long)p.ldx, (long long)p.cols);
  if (!aligned(p.x, dtype_bytes(dtype)) || !aligned(p.q_row, 16) || !aligned(p.q_col, 16) || !aligned(p.s_row, 8) || !aligned(p.s_col, 8))
    return fail(FSH_ENOTSUP, "%s: data must be 16-byte and scales 8-byte aligned, x to its elements", who);
  p.vec = aligned(p.x, 16) && p.ldx * dtype_bytes(dtype) % 16 == 0;
  return FSH_OK;
}

int launch_columns(MxQuantParams& p, int32_t dtype, int64_t batch, int64_t padded_rows, const char* who, void* stream) {
  p.tiles_c = ceil_div(p.q_row ? 2 * p.ld_row : p.cols, (int64_t)kTile);
  p.tiles_r = padded_rows / kTile;
  const int64_t tiles = p.tiles_c * p.tiles_r * batch;
  if (tiles > kMaxGrid) return fail(FSH_ENOTSUP, "%s: too many tiles", who);
  const dim3 grid(static_cast<uint32_t>(tiles)), block(kThreads);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  by_dtype(dtype, [&](auto dt) {
    if (p.q_row) hipLaunchKernelGGL((mxfp4_quantize_columns_kernel<dt.value, true>), grid, block, 0, on, p);
    else hipLaunchKernelGGL((mxfp4_quantize_columns_kernel<dt.value, false>), grid, block, 0, on, p);
  });
  return check_launch("mxfp4_quantize_columns_kernel");
}

}  // namespace
}  // namespace fsh

FSH_API int fsh_mxfp4_quantize(const void* x_dev, int32_t dtype, int64_t batch, int64_t rows, int64_t cols, int64_t ldx,
                               void* q_rows_dev, void* s_rows_dev, void* q_cols_dev, void* s_cols_dev,
                               float* column_sums_dev, void* stream) {
  using namespace fsh;
  const char* who = "fsh_mxfp4_quantize";
  if (batch < 0 || rows < 0 || cols < 0) return fail(FSH_EINVAL, "%s: negative shape", who);
  if (batch == 0 || rows == 0 || cols == 0) return FSH_OK;
  MxQuantParams p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const uint8_t*>(x_dev);
  p.rows = rows; p.cols = cols; p.ldx = ldx;
  p.q_row = static_cast<uint8_t*>(q_rows_dev); p.s_row = static_cast<uint8_t*>(s_rows_dev);
  p.q_col = static_cast<uint8_t*>(q_cols_dev); p.s_col = static_cast<uint8_t*>(s_cols_dev);
  p.ld_row = ceil_div(cols, (int64_t)kMxColumns) * (kMxColumns / 2);
  const int64_t padded_rows = ceil_div(rows, (int64_t)kMxColumns) * kMxColumns;
  p.ld_col = padded_rows / 2;
  p.table_rows = batch * rows; p.table_cols = batch * cols;
  p.column_sums = column_sums_dev;
  if (int rc = quantize_checks(p, dtype, who)) return rc;
  if (batch > 1 && ldx != cols && p.q_col) return fail(FSH_ENOTSUP, "%s: a stack of matrices must be contiguous", who);
  if (column_sums_dev && (!p.q_col || batch != 1)) return fail(FSH_EINVAL, "%s: column sums come with the column form of one matrix", who);
  if (p.q_col) return launch_columns(p, dtype, batch, padded_rows, who, stream);
  p.rows = batch * rows;  // stacked rows are rows
  p.tiles_c = ceil_div(2 * p.ld_row, (int64_t)kRowTileCols);
  const int64_t tiles = ceil_div(p.rows, (int64_t)kRowTileRows) * p.tiles_c;
  if (tiles > kMaxGrid) return fail(FSH_ENOTSUP, "%s: too many tiles", who);
  by_dtype(dtype, [&](auto dt) {
    hipLaunchKernelGGL(mxfp4_quantize_rows_kernel<dt.value>, dim3(static_cast<uint32_t>(tiles)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
  });
  return check_launch("mxfp4_quantize_rows_kernel");
}

FSH_API int fsh_mxfp4_quantize_segments(const void* x_dev, int32_t dtype, int64_t rows, int64_t cols, int64_t ldx,
                                        const int32_t* offsets_dev, const int32_t* padded_offsets_dev, int32_t experts,
                                        const int32_t* source_dev, int32_t top_k, void* q_rows_dev, void* s_rows_dev,
                                        void* q_cols_dev, void* s_cols_dev, int64_t padded_rows, void* stream) {
  using namespace fsh;
  const char* who = "fsh_mxfp4_quantize_segments";
  if (rows < 0 || cols < 0 || experts <= 0 || top_k <= 0 || padded_rows < 0)
    return fail(FSH_EINVAL, "%s: negative shape, or no expert", who);
  if (rows == 0 || cols == 0) return FSH_OK;
  if (!offsets_dev || !padded_offsets_dev || !q_cols_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (padded_rows % kMxColumns || padded_rows < rows)
    return fail(FSH_EINVAL, "%s: padded_rows %lld is not a multiple of %d that holds %lld rows", who, (long long)padded_rows,
                kMxColumns, (long long)rows);
  if (source_dev && q_rows_dev) return fail(FSH_EINVAL, "%s: the row form of gathered rows is that of x itself", who);
  MxQuantParams p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const uint8_t*>(x_dev);
  p.rows = rows; p.cols = cols; p.ldx = ldx;
  p.q_row = static_cast<uint8_t*>(q_rows_dev); p.s_row = static_cast<uint8_t*>(s_rows_dev);
  p.q_col = static_cast<uint8_t*>(q_cols_dev); p.s_col = static_cast<uint8_t*>(s_cols_dev);
  p.ld_row = ceil_div(cols, (int64_t)kMxColumns) * (kMxColumns / 2);
  p.ld_col = padded_rows / 2;
  p.table_rows = rows; p.table_cols = cols;
  p.offsets = offsets_dev; p.padded_offsets = padded_offsets_dev; p.source = source_dev;
  p.experts = experts; p.top_k = top_k;
  if (int rc = quantize_checks(p, dtype, who)) return rc;
  return launch_columns(p, dtype, 1, padded_rows, who, stream);
}

FSH_API int fsh_mxfp4_dequantize(const void* q_dev, const void* s_dev, int64_t rows, int64_t cols, void* out_dev, int32_t dtype,
                                 int64_t ldo, void* stream) {
  using namespace fsh;
  const char* who = "fsh_mxfp4_dequantize";
  if (rows < 0 || cols < 0) return fail(FSH_EINVAL, "%s: negative shape", who);
  if (rows == 0 || cols == 0) return FSH_OK;
  if (!known_dtype(dtype)) return fail(FSH_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (!q_dev || !s_dev || !out_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (ldo < cols) return fail(FSH_EINVAL, "%s: ldo %lld < cols %lld", who, (long long)ldo, (long long)cols);
  if (!aligned(q_dev, 16) || !aligned(out_dev, dtype_bytes(dtype))) return fail(FSH_ENOTSUP, "%s: misaligned pointer", who);
  MxDequantParams p;
  p.q = static_cast<const uint8_t*>(q_dev);
  p.s = static_cast<const uint8_t*>(s_dev);
  p.out = static_cast<uint8_t*>(out_dev);
  p.rows = rows; p.cols = cols; p.ldo = ldo;
  p.ldq = ceil_div(cols, (int64_t)kMxColumns) * (kMxColumns / 2);
  p.groups = ceil_div(cols, (int64_t)(16 / dtype_bytes(dtype)));
  p.vec = aligned(out_dev, 16) && ldo * dtype_bytes(dtype) % 16 == 0;
  const int64_t blocks = ceil_div(rows * p.groups, (int64_t)kThreads);
  const dim3 grid(static_cast<uint32_t>(blocks < kMaxGrid ? blocks : kMaxGrid)), block(kThreads);
  by_dtype(dtype, [&](auto dt) {
    hipLaunchKernelGGL(mxfp4_dequantize_kernel<dt.value>, grid, block, 0, static_cast<hipStream_t>(stream), p);
  });
  return check_launch("mxfp4_dequantize_kernel");
}

FSH_API int fsh_sum_runs(const float* sums_dev, int64_t runs, int64_t cols, void* out_dev, int32_t dtype, void* stream) {
  using namespace fsh;
  if (runs < 0 || cols < 0) return fail(FSH_EINVAL, "fsh_sum_runs: negative shape");
  if (cols == 0) return FSH_OK;
  if (!known_dtype(dtype)) return fail(FSH_EINVAL, "fsh_sum_runs: unknown dtype %d", dtype);
  if ((runs && !sums_dev) || !out_dev) return fail(FSH_EINVAL, "fsh_sum_runs: null pointer");
  const int64_t blocks = ceil_div(cols, (int64_t)64);
  if (blocks > kMaxGrid) return fail(FSH_ENOTSUP, "fsh_sum_runs: too many columns");
  by_dtype(dtype, [&](auto dt) {
    hipLaunchKernelGGL(sum_runs_kernel<dt.value>, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), sums_dev, out_dev, runs, cols);
  });
  return check_launch("sum_runs_kernel");
}
