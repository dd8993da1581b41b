// Root-mean-square norm of rows, with the residual's addition, and with its
// output in 8 bits with scales.
//
//   h = x + r, rounded to the type of r     (h = x without a residual)
//   s = 1 / sqrt(mean(h^2) + eps)            sums and statistics in fp32
//   y = h s w
//
// The norm is that of the rounded h, which is what the next layer adds to and what
// the backward pass reads: the call gives the bits of an addition followed by a
// norm.  The 8-bit form is what the FP8 linear's quantizer makes of y in bf16:
// per run of 128 columns a = max(max |y|, 1e-12), bytes e4m3(y 448 / a), scale
// 1 / (448 / a).
//
// Bound by memory: x, r and w are read once, h and y written once, the row stays
// in registers in between.  All but w streams, past the caches: with h written through them
// 8192 rows of 4096 (bf16, quantized) take 49 us for 44, of 7168 on an fp32 stream 140 for 120.
// Measured: 8192 x 4096 bf16 with a residual 47 us, 5.7 TB/s; quantized 43, 5.5; 8192 x 7168 quantized, on
// an fp32 stream, 108, 6.0; 262144 x 128 25, 5.3; one row of 4096 3.1 us, a launch's chain of loads.
//
// LANES threads share a row (norm_layout.hpp).
#include "norm_layout.hpp"

namespace fsh {
namespace {

struct NormParams {
  const void* x;
  const void* residual;
  const void* weight;
  void* total;
  void* out;
  float* scales;
  float* rstd;
  int64_t rows, cols, ldx, ldr, ldq;
  int64_t row_blocks;
  int32_t weight_dtype;
  float eps;
};

// s of a row from its sum of squares.
__device__ __forceinline__ float inverse_root(float sum, int64_t cols, float eps) {
  return 1.0f / sqrtf(sum / static_cast<float>(cols) + eps);
}

// A vector of h from the vectors of x and r; rounded, and written where there is an r.
template <int XT, int RT, int VEC>
__device__ __forceinline__ void add_residual(const RawVec<XT, VEC>& x, const RawVec<RT, VEC>& r, float (&h)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) h[j] = element<XT, VEC>(x, j);
  if constexpr (RT != kNoType) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) h[j] += element<RT, VEC>(r, j);
  }
}

// A vector of y in 8 bits: the lane's columns from `col` on are the VEC of y behind
// the first `skip`, and zero from there.  128 / VEC neighbouring lanes have a run.
template <int VEC>
__device__ __forceinline__ void write_quantized(const NormParams& p, int64_t row, int64_t col, int skip, bool live, const float (&y)[VEC]) {
  float b[VEC];
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const uint32_t bits = f32_to_bf16_bits(y[j]);
    b[j] = bf16_bits_to_f32(bits);
    largest = max(largest, j < skip ? 0u : bits & 0x7FFFu);
  }
  largest = VEC == 8 ? row16_max_u32(largest) : max32_u32(largest);
  float scale, recip;
  tile_scale(bf16_bits_to_f32(largest), 1e-12f, scale, recip);
  if (live && col < p.ldq) {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) {
      w[j] = cvt2_fp8(b[4 * j] * scale, b[4 * j + 1] * scale, 0, false);
      w[j] = cvt2_fp8(b[4 * j + 2] * scale, b[4 * j + 3] * scale, w[j], true);
    }
    typename std::conditional<VEC == 8, uint64_t, uint32_t>::type bytes;
    static_assert(sizeof(bytes) == sizeof(w));
    __builtin_memcpy(&bytes, w, sizeof(w));
    bytes >>= 8 * skip;
    __builtin_memcpy(static_cast<uint8_t*>(p.out) + row * p.ldq + col, &bytes, sizeof(bytes));
    if (col % 128 == 0) p.scales[col / 128 * p.rows + row] = recip;
  }
}

template <int XT, int RT, bool kQuant, typename L>
__global__ __launch_bounds__(L::THREADS) void rms_norm_kernel(const NormParams p) {
  constexpr int VEC = L::VEC, ITEMS = L::ITEMS, TURN = L::TURN;
  // (8192 rows of 7161 on an fp32 stream, quantized: 120 us for 163; with one vector 35 for 33)
  constexpr bool kAgain = L::ENDS == kOverlapping && ITEMS > 1;
  __shared__ float lds[L::LANES > 64 ? 2 * L::LANES / 64 : 1];
  const int lane = threadIdx.x % L::LANES, cols = static_cast<int>(p.cols);
  float w[ITEMS][VEC];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) NormVector<L>((i * L::LANES + lane) * VEC, cols).weights(p.weight, p.weight_dtype, w[i]);
  int turn = 0;
  for (int64_t block = blockIdx.x; block < p.row_blocks; block += gridDim.x) {
    RawVec<XT, VEC> x[TURN][ITEMS];
    RawVec<RT, VEC> r[TURN][ITEMS];
#pragma unroll
    for (int k = 0; k < TURN; ++k) {
      const int64_t row = (block * TURN + k) * L::ROWS + threadIdx.x / L::LANES;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const NormVector<L> c((i * L::LANES + lane) * VEC, cols);
        x[k][i] = c.template load<XT>(p.x, row * p.ldx, row < p.rows);
        r[k][i] = c.template load<RT>(p.residual, row * p.ldr, row < p.rows);
      }
    }
#pragma unroll
    for (int k = 0; k < TURN; ++k, ++turn) {
      const int64_t row = (block * TURN + k) * L::ROWS + threadIdx.x / L::LANES;
      const bool live = row < p.rows;
      float h[ITEMS][VEC];
      float sum = 0.0f;
      const int lane_sum = lane_again<kAgain>(lane);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const NormVector<L> c((i * L::LANES + lane_sum) * VEC, cols);
        add_residual<XT, RT, VEC>(x[k][i], r[k][i], h[i]);
        if constexpr (RT != kNoType) {
          const auto rounded = to_vec<RT, VEC>(h[i]);
          if (live && c.inside) c.template store<RT, true>(p.total, row * p.cols, rounded);
#pragma unroll
          for (int j = 0; j < VEC; ++j) h[i][j] = element<RT, VEC>(rounded, j);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum += j < c.skip ? 0.0f : h[i][j] * h[i][j];
      }
      sum = sum_over_row<L::LANES>(sum, lds, turn);
      const float s = inverse_root(sum, p.cols, p.eps);
      if (p.rstd && live && lane == 0) p.rstd[row] = s;
      const int lane_out = lane_again<kAgain>(lane);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int col = (i * L::LANES + lane_out) * VEC;
        const NormVector<L> c(col, cols);
        float y[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = c.inside && j < c.count ? h[i][j] * s * w[i][j] : 0.0f;
        if constexpr (kQuant) write_quantized<VEC>(p, row, col, c.skip, live, y);
        else if (live && c.inside) c.template store<XT, true>(p.out, row * p.cols, to_vec<XT, VEC>(y));
      }
    }
  }
}

// Rows that do not fit the registers: read once for the sum, then, as h, for the output.
template <int XT, int RT, bool kQuant, typename L>
__global__ __launch_bounds__(L::THREADS) void rms_norm_wide_kernel(const NormParams p) {
  constexpr int VEC = L::VEC, STEP = L::THREADS * VEC;
  __shared__ float lds[2 * L::THREADS / 64];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, ++turn) {
    float sum = 0.0f;
    for (int64_t col = threadIdx.x * VEC; col < p.cols; col += STEP) {
      const auto x = load_vec<XT, VEC>(p.x, row * p.ldx + col, p.cols - col);
      const auto r = load_vec<RT, VEC>(p.residual, row * p.ldr + col, p.cols - col);
      float h[VEC];
      add_residual<XT, RT, VEC>(x, r, h);
      if constexpr (RT != kNoType) {
        const auto rounded = to_vec<RT, VEC>(h);
        store_vec<RT, VEC>(p.total, row * p.cols + col, p.cols - col, rounded);
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[j] = element<RT, VEC>(rounded, j);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum += h[j] * h[j];
    }
    sum = sum_over_row<L::THREADS>(sum, lds, turn);
    const float s = inverse_root(sum, p.cols, p.eps);
    if (p.rstd && threadIdx.x == 0) p.rstd[row] = s;
    // (each thread reads back what it wrote itself; whole runs of 128 columns, for the maxima)
    const int64_t end = ceil_div(p.cols, (int64_t)128) * 128;
    for (int64_t col = threadIdx.x * VEC; col < end; col += STEP) {
      float y[VEC], w[VEC];
      if constexpr (RT == kNoType) {
        const auto x = load_vec<XT, VEC>(p.x, row * p.ldx + col, p.cols - col);
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = element<XT, VEC>(x, j);
      } else {
        const auto h = load_vec<RT, VEC>(p.total, row * p.cols + col, p.cols - col);
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = element<RT, VEC>(h, j);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] = 1.0f;
      if (p.weight && col < p.cols) load_floats<VEC>(p.weight, p.weight_dtype, col, p.cols - col, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) y[j] = col + j < p.cols ? y[j] * s * w[j] : 0.0f;
      if constexpr (kQuant) write_quantized<VEC>(p, row, col, 0, true, y);
      else if (col < p.cols) store_vec<XT, VEC, true>(p.out, row * p.cols + col, p.cols - col, to_vec<XT, VEC>(y));
    }
  }
}

// launch(layout) with the layout for rows of `cols` columns.  Threads as few as keep
// two or more workgroups in a compute unit, for the bytes in flight, and as have few idle at
// the row's end: 24576 rows of 1040 bf16 take 41 us by 64 threads, 57 by 256; 8192 of 5120, quantized, 62 by 320 and
// 68 by 256; of 6144 68 by 512, 72 by 256; of 7168 with an fp32 stream, in vectors of four, 108 by 256, and 2 to 4 %
// more by 512; 4096 of 12288 69 by 768, 81 by 1024.  Narrow rows go two a turn (262144 x 128: 30 us
// with one, 26 with four).  Rows of 2049 to 8192 columns get more lanes each where they are few: 48 of 7168, quantized, 5.0 us
// for 6.7; of 2048 the other way round, 33 for 27.  The two cross between 512 and 768 rows (quantized, with the events around
// them: 512 of 8192 10.3 for 11.0, 640 alike, 768 14.2 for 13.5; 512 of 4096 7.4 for 7.8), values earlier (512 of 7168 10.0
// for 8.9).  Values and bytes take the same sums, of an order that this choice changes: kQuant alone picks whole runs of 128.
template <int ENDS, int VEC, bool kQuant, typename Launch>
void by_columns(int64_t cols, int64_t rows, Launch launch) {
  const bool few = rows <= 512;
  if (ENDS == kPieces || (cols <= 64 && !kQuant)) launch(NormLayout<ENDS, (kQuant ? 128 : 64) / VEC, VEC, VEC, 2>{});
  else if constexpr (ENDS == kPieces) return;
  else if (cols <= 128) launch(NormLayout<ENDS, 128 / VEC, VEC, VEC, 2>{});
  else if (cols <= 256) launch(NormLayout<ENDS, 256 / VEC, VEC, VEC, 2>{});
  else if (cols <= 512) launch(NormLayout<ENDS, 64, 8, VEC, 2>{});
  else if (cols <= 1024) launch(NormLayout<ENDS, 64, 16, VEC>{});
  else if (cols <= 1536) launch(NormLayout<ENDS, 64, 24, VEC>{});
  else if (cols <= 2048) launch(NormLayout<ENDS, 256, 8, VEC>{});
  else if (cols <= 4096 && !few) launch(NormLayout<ENDS, 256, 16, VEC>{});
  else if (cols <= 4096) launch(NormLayout<ENDS, 512, 8, VEC>{});
  else if (cols <= 8192 && few) launch(NormLayout<ENDS, 1024, 8, VEC>{});
  else if (cols <= 5120) launch(NormLayout<ENDS, 320, 16, VEC>{});
  else if (cols <= 8192) launch(NormLayout<ENDS, VEC == 8 ? 512 : 256, VEC == 8 ? 16 : 32, VEC>{});
  else if (cols <= 12288 && VEC == 8) launch(NormLayout<ENDS, VEC == 8 ? 768 : 1024, 16, VEC>{});
  else if (cols <= 16384) launch(NormLayout<ENDS, VEC == 8 ? 512 : 1024, VEC == 8 ? 32 : 16, VEC>{});
  else launch(NormLayout<kEven, 1024, 0, VEC>{});  // (any columns)
}

template <int XT, int RT, bool kQuant>
void launch_norm(NormParams& p, hipStream_t stream) {
  constexpr int VEC = XT == FSH_DT_F32 || RT == FSH_DT_F32 ? 4 : 8;  // 16 bytes of the wider type
  by_ends<VEC>(p.cols, [&](auto ends) {
    by_columns<ends.value, VEC, kQuant>(p.cols, p.rows, [&](auto layout) {
      using L = decltype(layout);
      p.row_blocks = ceil_div(p.rows, (int64_t)L::ROWS * L::TURN);
      constexpr int64_t kMaxGrid = (1LL << 32) / L::THREADS - 1;  // a launch's threads are counted in 32 bits
      const dim3 grid(static_cast<uint32_t>(p.row_blocks < kMaxGrid ? p.row_blocks : kMaxGrid)), block(L::THREADS);
      if constexpr (L::PER == 0)
        hipLaunchKernelGGL((rms_norm_wide_kernel<XT, RT, kQuant, L>), grid, block, 0, stream, p);
      else
        hipLaunchKernelGGL((rms_norm_kernel<XT, RT, kQuant, L>), grid, block, 0, stream, p);
    });
  });
}

template <int XT, int RT>
void launch_form(NormParams& p, bool quant, hipStream_t stream) {
  if (quant) launch_norm<XT, RT, true>(p, stream);
  else launch_norm<XT, RT, false>(p, stream);
}

// out = q scale, eight columns a thread and turn.  Bound by memory: 1 byte read and 2
// (or 4) written, past the caches (8192 x 7168 to bf16: 31 us, 37 through them).  Index: the
// unsigned type that counts the matrix's eights of columns (64 bits: 1 us more, for the division).
struct DequantParams {
  const uint8_t* q;
  const float* scales;
  void* out;
  int64_t rows, cols, ldq, chunks;  // chunks of eight columns in a row
};

template <int DT, typename Index>
__global__ __launch_bounds__(256) void act_dequant_kernel(const DequantParams p) {
  const Index chunks = static_cast<Index>(p.chunks), all = static_cast<Index>(p.rows) * chunks;
  for (Index i = static_cast<Index>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<Index>(gridDim.x) * 256) {
    const Index row = i / chunks;
    const int64_t col = static_cast<int64_t>(i - row * chunks) * 8, r = static_cast<int64_t>(row);
    const u32x2 q = *reinterpret_cast<const u32x2*>(p.q + r * p.ldq + col);
    const float scale = p.scales[col / 128 * p.rows + r];
    float f[8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(q[j]), false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(q[j]), true);
      f[4 * j] = lo[0] * scale;
      f[4 * j + 1] = lo[1] * scale;
      f[4 * j + 2] = hi[0] * scale;
      f[4 * j + 3] = hi[1] * scale;
    }
    store_vec<DT, 8, true>(p.out, r * p.cols + col, p.cols - col, to_vec<DT, 8>(f));
  }
}

}  // namespace
}  // namespace fsh

FSH_API int fsh_rms_norm(const fsh_norm* q, void* stream) {
  using namespace fsh;
  const char* who = "fsh_rms_norm";
  if (!q) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (q->rows < 0 || q->cols < 0) return fail(FSH_EINVAL, "%s: negative shape", who);
  const bool residual = q->residual_dev != nullptr, quant = q->form == FSH_NORM_FP8;
  if (!is_dtype(q->x_dtype) || (q->weight_dev && !is_dtype(q->weight_dtype)))
    return fail(FSH_EINVAL, "%s: unknown dtype %d or %d", who, q->x_dtype, q->weight_dtype);
  if (q->form != FSH_NORM_VALUES && !quant) return fail(FSH_EINVAL, "%s: unknown form %d", who, q->form);
  if (residual && q->residual_dtype != q->x_dtype && q->residual_dtype != FSH_DT_F32)
    return fail(FSH_EINVAL, "%s: the residual's dtype %d is neither that of x (%d) nor fp32", who, q->residual_dtype, q->x_dtype);
  if (!(q->eps >= 0.0f)) return fail(FSH_EINVAL, "%s: eps is negative or not a number", who);
  if (q->rows == 0 || q->cols == 0) return FSH_OK;
  if (!q->x_dev || !q->out_dev || (residual && !q->total_dev) || (quant && !q->scales_dev)) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (q->ldx < q->cols || (residual && q->ldr < q->cols))
    return fail(FSH_EINVAL, "%s: a row stride (%lld, %lld) is less than cols %lld", who, (long long)q->ldx, (long long)q->ldr, (long long)q->cols);
  if (!aligned(q->x_dev, bytes_of(q->x_dtype)) || (residual && (!aligned(q->residual_dev, bytes_of(q->residual_dtype)) || !aligned(q->total_dev, bytes_of(q->residual_dtype)))) ||
      (q->weight_dev && !aligned(q->weight_dev, bytes_of(q->weight_dtype))) || !aligned(q->out_dev, quant ? 8 : bytes_of(q->x_dtype)) ||
      !aligned(q->scales_dev, 4) || !aligned(q->rstd_dev, 4))
    return fail(FSH_ENOTSUP, "%s: tensors must be aligned to their elements, bytes to 8", who);
  // (the last columns of a row are written twice, by two lanes that have read them; wide rows read the total back)
  const int64_t n = q->rows, k = q->cols, runs = ceil_div(k, (int64_t)128);
  const RowSpan inputs[] = {{q->x_dev, n, k, q->ldx, bytes_of(q->x_dtype)},
                            {q->residual_dev, n, k, q->ldr, bytes_of(q->residual_dtype)},
                            span_of(q->weight_dev, k, bytes_of(q->weight_dtype))};
  const RowSpan outputs[] = {span_of(residual ? q->total_dev : nullptr, n * k, bytes_of(q->residual_dtype)),
                             span_of(q->out_dev, quant ? n * runs * 128 : n * k, quant ? 1 : bytes_of(q->x_dtype)),
                             span_of(quant ? q->scales_dev : nullptr, n * runs, 4), span_of(q->rstd_dev, n, 4)};
  if (outputs_overlap(inputs, outputs)) return fail(FSH_EINVAL, "%s: an output overlaps an input or another output", who);
  NormParams p = {};
  p.x = q->x_dev;
  p.residual = q->residual_dev;
  p.weight = q->weight_dev;
  p.total = q->total_dev;
  p.out = q->out_dev;
  p.scales = q->scales_dev;
  p.rstd = q->rstd_dev;
  p.rows = q->rows;
  p.cols = q->cols;
  p.ldx = q->ldx;
  p.ldr = q->ldr;
  p.ldq = ceil_div(q->cols, (int64_t)128) * 128;
  p.weight_dtype = q->weight_dtype;
  p.eps = q->eps;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  const int x = q->x_dtype, r = residual ? q->residual_dtype : kNoType;
  if (x == FSH_DT_BF16 && r == kNoType) launch_form<FSH_DT_BF16, kNoType>(p, quant, on);
  else if (x == FSH_DT_BF16 && r == FSH_DT_BF16) launch_form<FSH_DT_BF16, FSH_DT_BF16>(p, quant, on);
  else if (x == FSH_DT_BF16) launch_form<FSH_DT_BF16, FSH_DT_F32>(p, quant, on);
  else if (x == FSH_DT_F16 && r == kNoType) launch_form<FSH_DT_F16, kNoType>(p, quant, on);
  else if (x == FSH_DT_F16 && r == FSH_DT_F16) launch_form<FSH_DT_F16, FSH_DT_F16>(p, quant, on);
  else if (x == FSH_DT_F16) launch_form<FSH_DT_F16, FSH_DT_F32>(p, quant, on);
  else if (r == kNoType) launch_form<FSH_DT_F32, kNoType>(p, quant, on);
  else launch_form<FSH_DT_F32, FSH_DT_F32>(p, quant, on);
  return check_launch("rms_norm_kernel");
}

FSH_API int fsh_act_dequant_1x128(const void* q_dev, const float* scales_dev, int64_t rows, int64_t cols, int64_t ldq, void* out_dev,
                                  int32_t dtype, void* stream) {
  using namespace fsh;
  const char* who = "fsh_act_dequant_1x128";
  if (rows < 0 || cols < 0) return fail(FSH_EINVAL, "%s: negative shape", who);
  if (!is_dtype(dtype)) return fail(FSH_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (rows == 0 || cols == 0) return FSH_OK;
  if (!q_dev || !scales_dev || !out_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (ldq < ceil_div(cols, (int64_t)128) * 128)
    return fail(FSH_EINVAL, "%s: ldq %lld is less than cols %lld rounded up to 128", who, (long long)ldq, (long long)cols);
  if (ldq % 8 || !aligned(q_dev, 8) || !aligned(scales_dev, 4) || !aligned(out_dev, bytes_of(dtype)))
    return fail(FSH_ENOTSUP, "%s: the bytes' rows must be 8-byte aligned, the others to their elements", who);
  const int64_t runs = ceil_div(cols, (int64_t)128);
  const RowSpan inputs[] = {{q_dev, rows, runs * 128, ldq, 1}, span_of(scales_dev, rows * runs, 4)};
  const RowSpan outputs[] = {span_of(out_dev, rows * cols, bytes_of(dtype))};
  if (outputs_overlap(inputs, outputs)) return fail(FSH_EINVAL, "%s: the output overlaps an input", who);
  DequantParams p = {static_cast<const uint8_t*>(q_dev), scales_dev, out_dev, rows, cols, ldq, ceil_div(cols, (int64_t)8)};
  constexpr int64_t kMaxGrid = (1LL << 32) / 256 - 1;
  const int64_t blocks = ceil_div(rows * p.chunks, (int64_t)256);
  const dim3 grid(static_cast<uint32_t>(blocks < kMaxGrid ? blocks : kMaxGrid)), block(256);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  // (32 bits as long as a turn past the end still counts in them)
  const bool small = rows * p.chunks < (1LL << 31);
  const auto go = [&](auto dt) {
    if (small) hipLaunchKernelGGL((act_dequant_kernel<dt.value, uint32_t>), grid, block, 0, on, p);
    else hipLaunchKernelGGL((act_dequant_kernel<dt.value, uint64_t>), grid, block, 0, on, p);
  };
  if (dtype == FSH_DT_BF16) go(std::integral_constant<int, FSH_DT_BF16>{});
  else if (dtype == FSH_DT_F16) go(std::integral_constant<int, FSH_DT_F16>{});
  else go(std::integral_constant<int, FSH_DT_F32>{});
  return check_launch("act_dequant_kernel");
}
