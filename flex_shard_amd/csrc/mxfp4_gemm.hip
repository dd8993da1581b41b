// Products of microscaled 4-bit matrices: a linear layer's forward, its input
// gradient and its weight gradient are all a b^T of operands quantized along the
// contraction; the experts' layers are the same with rows (or the contraction)
// in segments.
#include "mxfp4_few.hpp"

namespace fsh {
namespace {

constexpr int64_t kFewMaxRows = 16;

template <typename Cfg, int kProblem>
int launch_mx_tiles(MxGemmParams& p, int64_t tiles_m, int64_t batch, hipStream_t stream) {
  MxSchedule& s = p.schedule;
  const int64_t tiles_n = ceil_div(p.n, static_cast<int64_t>(Cfg::BN)), tiles = tiles_m * tiles_n;
  if (tiles * batch > 0x3FFFFFLL) return fail(FSH_ENOTSUP, "fsh_mxfp4_gemm: too many tiles");
  s.tiles_m = static_cast<int32_t>(tiles_m);
  s.tiles_n = static_cast<int32_t>(tiles_n);
  s.items = static_cast<int32_t>(tiles * batch);
  s.items_per_xcd = (s.items + kXcds - 1) / kXcds;
  const int32_t eighth = static_cast<int32_t>(ceil_div(tiles, static_cast<int64_t>(kXcds)));
  s.run = eighth < kGroupTilesM ? kGroupTilesM : eighth;
  s.by_span = Divisor::of(static_cast<uint32_t>(kGroupTilesM * tiles_n));
  s.by_run = Divisor::of(static_cast<uint32_t>(s.run));
  s.by_round = Divisor::of(static_cast<uint32_t>(s.run * batch));
  int64_t blocks = static_cast<int64_t>(s.items_per_xcd) * kXcds;
  if (Cfg::kResident) {
    const int64_t units = compute_units(), resident = units >= kXcds ? units / kXcds * kXcds : kXcds;
    blocks = blocks < resident ? blocks : resident;
  }
  const dim3 grid(static_cast<uint32_t>(blocks)), block(Cfg::kThreads);
  int rc = FSH_OK;
  by_dtype(p.out_dtype, [&](auto dt) {
    static LdsReservation reserved;
    const auto kernel = &mxfp4_gemm_kernel<Cfg, kProblem, dt.value>;
    rc = reserve_lds_once(reserved, kernel, Cfg::kLdsBytes);
    if (rc == FSH_OK) hipLaunchKernelGGL(kernel, grid, block, Cfg::kLdsBytes, stream, p);
  });
  return rc != FSH_OK ? rc : check_launch("mxfp4_gemm_kernel");
}

// Tiles of BM rows that the segments of p.m rows take at most: each of the
// experts and the rows behind the last can end inside a tile.
template <typename Cfg>
int64_t segment_tiles(const MxGemmParams& p) { return p.m / Cfg::BM + p.experts + 1; }

// (see mx_tile_kind for what each is good at)
using MxLarge = MxTile<2, 2, 4, 4, 2, 5, true>;     // 256 x 256, one workgroup per compute unit
using MxMid = MxTile<2, 2, 2, 2, 2, 0, false>;      // 128 x 128, two
using MxMidDeep = MxTile<2, 2, 2, 2, 4, 0, false>;  // 128 x 128, one, four steps in flight
using MxSmall = MxTile<2, 2, 1, 1, 4, 0, false>;    // 64 x 64, two

template <typename Cfg>
int launch_mx(MxGemmParams& p, MxProblem problem, hipStream_t stream) {
  const int64_t tiles_m = ceil_div(p.m, static_cast<int64_t>(Cfg::BM));
  if (problem == kMxRows) return launch_mx_tiles<Cfg, kMxRows>(p, segment_tiles<Cfg>(p), 1, stream);
  if (problem == kMxOverRows) return launch_mx_tiles<Cfg, kMxOverRows>(p, tiles_m, p.experts, stream);
  return launch_mx_tiles<Cfg, kMxDense>(p, tiles_m, 1, stream);
}

// Which tiles a product takes: those with the lowest estimated time, from what
// the four measured (us, 64 x 64 / 128 x 128 / 128 x 128 deep / 256 x 256):
//   48 x 14336, k 4096      7.8  14.4  10.6  24.8    128 x 14336, k 4096    10.3  15.0  11.1  24.7
//   256 x 1024, k 4096      6.3  10.0   9.6  24.6    512 x 4096, k 4096     10.7  14.6  11.2  25.3
//   64 x 4096, k 14336     15.3  39.4  24.2  64.1    445 x 3932, k 11071    23.4  36.6  26.4  71.0
//   1000 x 5120, k 2048    14.9  11.5  14.3  17.1    1000 x 2048, k 5120    12.8  18.0  13.1  29.8
//   3000 x 1024, k 1500     8.6   7.9   7.4  15.3    2048 x 2048, k 2048    11.8   9.5   8.9  17.3
//   1024 x 4096, k 8192    36.6  29.6  25.2  41.8    512 x 14336, k 4096    34.1  21.0  26.2  25.9
//   2048 x 4096, k 4096    35.4  22.2  24.9  27.3    4096 x 4096, k 4096    69.2  42.9  47.6  35.7
//   4096 x 14336, k 4096    221   136   155   120    14336 x 4096, k 1000   83.0  50.0  66.1  50.8
// Rows of 32 experts, 7168 to 2048 columns, by rows per expert:
//   4   50.5  50.3  56.8  77.1    64  79.4  53.9  58.6  66.9    128  111  93.8  85.4  72.2    512  288  209  221  174
// Over rows of 32 experts, [2048, 7168] each, by rows per expert:
//   64  421  207  324  207    256  462  243  342  238    1024  731  411  551  364
// Few rows have a kernel of their own (mxfp4_few.hpp); us, it / 64 x 64 tiles, by rows (1, 4, 16):
//   14336, k 4096  8.5 / 9.0  9.0 / 9.1  10.9 / 9.4    4096, k 4096  4.2 / 7.5  4.4 / 7.6  4.9 / 7.6
//   4096, k 14336  9.6 / 17   9.9 / 17   11.5 / 18     1024, k 4096  3.5 / 7.1  3.7 / 7.1  4.3 / 7.2
bool takes_few_rows(int64_t m, int64_t n) { return m <= kFewMaxRows && (m <= kFewQuantize || n <= 8192); }

enum MxTileKind { kMxTiles64, kMxTiles128, kMxTiles128Deep, kMxTiles256, kMxFewRows };
MxTileKind mx_tile_kind(const MxGemmParams& p, MxProblem problem, int64_t units) {
  static constexpr TileShape kShapes[] = {
      {64, 64, 512.0, 0.18, 0.34, 0.49, 1.2},
      {128, 128, 512.0, 0.75, 0.80, 1.20, 2.8},
      {128, 128, 256.0, 0.42, 0.54, 0.60, 2.2},
      {256, 256, 256.0, 1.34, 1.50, 2.05, 5.0},
  };
  const bool segments = problem == kMxRows;
  if (problem == kMxDense && takes_few_rows(p.m, p.n)) return kMxFewRows;
  // Experts that have rows, and their rows: evenly spread for all that is known here.
  const double experts = segments ? static_cast<double>(p.m < p.experts ? p.m : p.experts) : 1.0;
  const double rows = static_cast<double>(p.m) / experts;
  double steps = static_cast<double>(p.k / kMxColumns);
  if (problem == kMxOverRows) steps = steps / p.experts < 1.0 ? 1.0 : steps / p.experts;
  // Every expert's weight comes from memory.
  const double memory_us = segments ? experts * static_cast<double>(p.n) * static_cast<double>(p.k) * (17.0 / 32.0) / 5.2e6 : 0.0;
  MxTileKind best = kMxTiles64;
  double best_us = 0.0;
  for (int i = 0; i < 4; ++i) {
    TileShape shape = kShapes[i];
    shape.round *= static_cast<double>(units) / 256.0;
    double tiles_m = ceil(rows / static_cast<double>(shape.m));
    if (segments && 2.0 * rows > static_cast<double>(shape.m)) tiles_m = rows / static_cast<double>(shape.m) + 0.5;  // (some have more rows)
    double tiles = experts * tiles_m * static_cast<double>(ceil_div(p.n, shape.m));
    if (problem == kMxOverRows) tiles *= p.experts;
    if (segments && i < 3) {  // (two tile rows of an expert do not meet in the L2 as those of one matrix do)
      shape.empty *= 1.4;
      shape.half *= 1.4;
      shape.full *= 1.4;
    }
    double us = rounds_us(shape, tiles, tiles * steps, steps);
    if (us < memory_us) us = memory_us;
    if (i == 0 || us < best_us) {
      best = static_cast<MxTileKind>(i);
      best_us = us;
    }
  }
  return best;
}

// How many waves share a workgroup's contraction: enough to fill the chip.
int few_waves(int64_t workgroups, int64_t steps) {
  int waves = 4;
  while (waves < kFewMaxWaves && workgroups * waves < 2048 && 2 * waves <= steps) waves *= 2;
  return static_cast<int>(waves < steps ? waves : steps);
}
int few_lds_bytes(const MxFewParams& p, int waves, bool quantize) {
  return waves * 16 * 17 * 4 + (quantize ? kFewQuantize * (static_cast<int>(p.ld) + 16 + 8 * p.steps) : 0);
}

template <bool kQuantize>
int launch_few(MxFewParams& p, int32_t dtype, hipStream_t stream) {
  const int64_t blocks = ceil_div(p.n, static_cast<int64_t>(kFewRows));
  if (blocks > 0x3FFFFFLL) return fail(FSH_ENOTSUP, "fsh_mxfp4_gemm: too many tiles");
  p.waves = few_waves(blocks, p.steps);
  const dim3 grid(static_cast<uint32_t>(blocks)), block(64 * p.waves);
  const int lds = few_lds_bytes(p, p.waves, kQuantize);
  by_dtype(dtype, [&](auto dt) {
    hipLaunchKernelGGL((mxfp4_few_rows_kernel<dt.value, kQuantize>), grid, block, lds, stream, p);
  });
  return check_launch("mxfp4_few_rows_kernel");
}

// A product's mode and whether its bias is fp32 (FSH_MXFP4_BIAS_F32 is added to the mode of a dense one).
struct MxMode {
  int32_t mode;
  bool bias_f32;
  explicit MxMode(int32_t m) : mode(m & ~FSH_MXFP4_BIAS_F32), bias_f32((m & FSH_MXFP4_BIAS_F32) != 0) {}
  bool known() const { return mode == FSH_MXFP4_DENSE || (!bias_f32 && (mode == FSH_MXFP4_ROWS || mode == FSH_MXFP4_OVER_ROWS)); }
  bool dense() const { return mode == FSH_MXFP4_DENSE; }
  int bias_bytes(int32_t out_dtype) const { return bias_f32 ? 4 : dtype_bytes(out_dtype); }
};

// A tile of rows in segments holds the first tile of every segment in LDS (kTableBytes).
int check_experts(MxMode mode, int32_t experts, const char* who) {
  if (mode.mode == FSH_MXFP4_ROWS && experts > FSH_MAX_EXPERTS)
    return fail(FSH_ENOTSUP, "%s: rows in segments of at most %d experts, got %d", who, FSH_MAX_EXPERTS, experts);
  return FSH_OK;
}

MxFewParams few_params(const fsh_mxfp4_product& q) {
  MxFewParams p;
  memset(&p, 0, sizeof(p));
  p.a = static_cast<const uint8_t*>(q.a_dev); p.as = static_cast<const uint8_t*>(q.a_scales_dev);
  p.b = static_cast<const uint8_t*>(q.b_dev); p.bs = static_cast<const uint8_t*>(q.b_scales_dev);
  p.out = q.out_dev; p.bias = q.bias_dev;
  p.bias_f32 = MxMode(q.mode).bias_f32;
  p.m = q.m; p.n = q.n; p.a_rows = q.a_rows; p.b_rows = q.b_rows;
  p.ld = q.k / 2; p.ldo = q.ldo;
  p.steps = static_cast<int32_t>(q.k / kMxColumns);
  return p;
}

}  // namespace
}  // namespace fsh

FSH_API int fsh_mxfp4_gemm(const fsh_mxfp4_product* product, void* stream) {
  using namespace fsh;
  const char* who = "fsh_mxfp4_gemm";
  if (!product) return fail(FSH_EINVAL, "%s: null product", who);
  const fsh_mxfp4_product& q = *product;
  if (q.m < 0 || q.n < 0 || q.k < 0) return fail(FSH_EINVAL, "%s: negative size", who);
  const MxMode mode(q.mode);
  if (!mode.known()) return fail(FSH_EINVAL, "%s: unknown mode %d", who, q.mode);
  if (!mode.dense() && q.experts <= 0) return fail(FSH_EINVAL, "%s: no expert", who);
  if (int rc = check_experts(mode, q.experts, who)) return rc;
  if (q.m == 0 || q.n == 0) return FSH_OK;
  if (!known_dtype(q.out_dtype)) return fail(FSH_EINVAL, "%s: unknown dtype %d", who, q.out_dtype);
  if (!q.a_dev || !q.a_scales_dev || !q.b_dev || !q.b_scales_dev || !q.out_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (q.k == 0 || q.k % kMxColumns)
    return fail(FSH_ENOTSUP, "%s: k must be a positive multiple of %d (operands are padded), got %lld", who, kMxColumns, (long long)q.k);
  if (q.k >= (1LL << 31) || q.m >= (1LL << 28) || q.n >= (1LL << 28) || q.a_rows >= (1LL << 28) || q.b_rows >= (1LL << 28))
    return fail(FSH_ENOTSUP, "%s: sizes beyond 2^28 rows or 2^31 columns", who);
  if (q.ldo < q.n) return fail(FSH_EINVAL, "%s: ldo %lld < n %lld", who, (long long)q.ldo, (long long)q.n);
  const bool segments = q.mode == FSH_MXFP4_ROWS;
  if (!mode.dense() && !q.offsets_dev) return fail(FSH_EINVAL, "%s: segments without offsets", who);
  if (segments && q.top_k <= 0) return fail(FSH_EINVAL, "%s: top_k must be positive", who);
  if (q.a_rows < (q.source_dev ? 1 : q.m) || q.b_rows < q.n * (segments ? q.experts : 1))
    return fail(FSH_EINVAL, "%s: operands of %lld and %lld rows are too few", who, (long long)q.a_rows, (long long)q.b_rows);
  if (q.source_dev && !segments) return fail(FSH_EINVAL, "%s: gathered rows belong to segments of rows", who);
  if (q.mode == FSH_MXFP4_OVER_ROWS && (q.bias_dev || q.ldo != q.n))
    return fail(FSH_EINVAL, "%s: products over rows are contiguous and have no bias", who);
  if (segments && q.bias_dev) return fail(FSH_ENOTSUP, "%s: segments have no bias", who);
  if (!aligned(q.a_dev, 16) || !aligned(q.b_dev, 16) || !aligned(q.a_scales_dev, 8) || !aligned(q.b_scales_dev, 8) ||
      !aligned(q.out_dev, dtype_bytes(q.out_dtype)) || !aligned(q.bias_dev, mode.bias_bytes(q.out_dtype)))
    return fail(FSH_ENOTSUP, "%s: data must be 16-byte and scales 8-byte aligned, out and bias to their elements", who);
  // The lanes' offsets are 32 bits from a tile's first row, or from the matrix for gathered rows.
  if (256 * (q.k / 2) >= (1LL << 32) || (q.source_dev && q.a_rows * (q.k / 2) >= (1LL << 32)))
    return fail(FSH_ENOTSUP, "%s: rows that are gathered, or a tile of them, span 4 GiB or more", who);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  MxGemmParams p;
  memset(&p, 0, sizeof(p));
  p.a = static_cast<const uint8_t*>(q.a_dev); p.as = static_cast<const uint8_t*>(q.a_scales_dev);
  p.b = static_cast<const uint8_t*>(q.b_dev); p.bs = static_cast<const uint8_t*>(q.b_scales_dev);
  p.out = q.out_dev; p.bias = q.bias_dev;
  p.bias_f32 = mode.bias_f32;
  p.m = q.m; p.n = q.n; p.k = q.k;
  p.a_rows = q.a_rows; p.b_rows = q.b_rows;
  p.lda = p.ldb = q.k / 2;
  p.ldo = q.ldo;
  p.out_dtype = q.out_dtype;
  p.experts = q.experts; p.top_k = q.top_k;
  p.offsets = p.padded_offsets = q.offsets_dev;
  p.source = q.source_dev;
  if (p.top_k > 0) p.by_top_k = Divisor::of(static_cast<uint32_t>(p.top_k));
  const MxProblem problem = segments ? kMxRows : q.mode == FSH_MXFP4_OVER_ROWS ? kMxOverRows : kMxDense;
  const int64_t units = compute_units();
  switch (mx_tile_kind(p, problem, units > 0 ? units : 256)) {
    case kMxTiles64: return launch_mx<MxSmall>(p, problem, on);
    case kMxTiles128: return launch_mx<MxMid>(p, problem, on);
    case kMxTiles128Deep: return launch_mx<MxMidDeep>(p, problem, on);
    case kMxFewRows: {
      MxFewParams few = few_params(q);
      return launch_few<false>(few, q.out_dtype, on);
    }
    default: return launch_mx<MxLarge>(p, problem, on);
  }
}

FSH_API int fsh_mxfp4_gemm_tiles(int64_t m, int64_t n, int64_t k, int32_t mode, int32_t experts) {
  using namespace fsh;
  if (m <= 0 || n <= 0 || k <= 0 || mode < FSH_MXFP4_DENSE || mode > FSH_MXFP4_OVER_ROWS || (mode != FSH_MXFP4_DENSE && experts <= 0))
    return fail(FSH_EINVAL, "fsh_mxfp4_gemm_tiles: bad sizes");
  if (int rc = check_experts(MxMode(mode), experts, "fsh_mxfp4_gemm_tiles")) return rc;
  MxGemmParams p;
  memset(&p, 0, sizeof(p));
  p.m = m; p.n = n; p.k = ceil_div(k, (int64_t)kMxColumns) * kMxColumns;
  p.experts = experts;
  const int64_t units = compute_units();
  static constexpr int kNames[] = {FSH_TILES_64, FSH_TILES_128, FSH_TILES_128_DEEP, FSH_TILES_256, FSH_TILES_FEW_ROWS};
  return kNames[mx_tile_kind(p, mode == FSH_MXFP4_ROWS ? kMxRows : mode == FSH_MXFP4_OVER_ROWS ? kMxOverRows : kMxDense, units > 0 ? units : 256)];
}

FSH_API int64_t fsh_mxfp4_matrix_bytes(int64_t rows, int64_t cols) {
  using namespace fsh;
  if (rows <= 0 || cols <= 0) return 0;
  return rows * ceil_div(cols, (int64_t)kMxColumns) * (kMxColumns / 2 + 8);
}

FSH_API int fsh_mxfp4_linear(const void* x_dev, int32_t dtype, int64_t rows, int64_t ldx, const fsh_mxfp4_product* product,
                             int64_t in_dim, void* scratch_dev, int64_t scratch_nbytes, void* stream) {
  using namespace fsh;
  const char* who = "fsh_mxfp4_linear";
  if (!product) return fail(FSH_EINVAL, "%s: null product", who);
  fsh_mxfp4_product q = *product;
  if (rows < 0 || in_dim < 0 || q.m < 0 || q.n < 0) return fail(FSH_EINVAL, "%s: negative shape", who);
  if (q.k != ceil_div(in_dim, (int64_t)kMxColumns) * kMxColumns)
    return fail(FSH_EINVAL, "%s: k %lld is not in_dim %lld rounded up to %d", who, (long long)q.k, (long long)in_dim, kMxColumns);
  if (q.out_dtype != dtype) return fail(FSH_EINVAL, "%s: the output has the activation's dtype", who);
  if (q.m == 0 || q.n == 0) return FSH_OK;
  if (q.k == 0) return fail(FSH_ENOTSUP, "%s: in_dim must be positive", who);
  q.a_rows = rows;
  const MxMode mode(q.mode);
  if (int rc = check_experts(mode, q.experts, who)) return rc;
  if (mode.dense() && q.m <= kFewQuantize) {
    MxFewParams p = few_params(q);
    if (few_lds_bytes(p, kFewMaxWaves, true) <= 64 * 1024) {
      if (!known_dtype(dtype)) return fail(FSH_EINVAL, "%s: unknown dtype %d", who, dtype);
      if (rows < q.m || ldx < in_dim || q.ldo < q.n || q.b_rows < q.n)
        return fail(FSH_EINVAL, "%s: rows or leading dimensions too small", who);
      if (!x_dev || !q.b_dev || !q.b_scales_dev || !q.out_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
      const int bytes = dtype_bytes(dtype);
      if (!aligned(x_dev, bytes) || !aligned(q.b_dev, 16) || !aligned(q.b_scales_dev, 8) || !aligned(q.out_dev, bytes) ||
          !aligned(q.bias_dev, mode.bias_bytes(dtype)))
        return fail(FSH_ENOTSUP, "%s: weights must be 16-byte and scales 8-byte aligned, x, out and bias to their elements", who);
      p.a = static_cast<const uint8_t*>(x_dev);
      p.cols = in_dim; p.ldx = ldx;
      p.vec = aligned(x_dev, 16) && ldx * bytes % 16 == 0;
      return launch_few<true>(p, dtype, static_cast<hipStream_t>(stream));
    }
  }
  const int64_t need = fsh_mxfp4_matrix_bytes(rows, in_dim);
  if (!scratch_dev || scratch_nbytes < need)
    return fail(FSH_EINVAL, "%s: scratch of %lld bytes, needs %lld", who, (long long)scratch_nbytes, (long long)need);
  uint8_t* data = static_cast<uint8_t*>(scratch_dev);
  uint8_t* scales = data + rows * (q.k / 2);
  if (int rc = fsh_mxfp4_quantize(x_dev, dtype, 1, rows, in_dim, ldx, data, scales, nullptr, nullptr, nullptr, stream)) return rc;
  q.a_dev = data;
  q.a_scales_dev = scales;
  return fsh_mxfp4_gemm(&q, stream);
}
