// Products of microscaled 4-bit matrices: a linear layer's forward, its input
// gradient and its weight gradient are all a b^T of operands quantized along the
// contraction; the experts' layers are the same with rows (or the contraction)
// in segments.
#include "mxfp4_few.hpp"

namespace fsh {
namespace {

template <typename Cfg, int kProblem>
int launch_mx_tiles(MxGemmParams& p, int64_t tiles_m, int64_t batch, hipStream_t stream) {
  GemmParams& s = p.schedule;
  const int64_t tiles_n = ceil_div(p.n, static_cast<int64_t>(Cfg::BN)), tiles = tiles_m * tiles_n;
  if (tiles * batch > 0x3FFFFFLL) return fail(FSH_ENOTSUP, "fsh_mxfp4_gemm: too many tiles");
  s.tiles_m = static_cast<int32_t>(tiles_m);
  s.tiles_n = static_cast<int32_t>(tiles_n);
  s.tiles_per_matrix = static_cast<int32_t>(tiles);
  s.work_items = tiles * batch;
  s.items_per_xcd = ceil_div(s.work_items, static_cast<int64_t>(kXcds));
  int64_t blocks = s.items_per_xcd * kXcds;
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

using MxLarge = MxTile<2, 2, 4, 4, 2, 5, true>;
using MxSmall = MxTile<2, 2, 1, 1, 4, 0, false>;

template <typename Cfg>
int launch_mx(MxGemmParams& p, MxProblem problem, hipStream_t stream) {
  const int64_t tiles_m = ceil_div(p.m, static_cast<int64_t>(Cfg::BM));
  if (problem == kMxRows) return launch_mx_tiles<Cfg, kMxRows>(p, segment_tiles<Cfg>(p), 1, stream);
  if (problem == kMxOverRows) return launch_mx_tiles<Cfg, kMxOverRows>(p, tiles_m, p.experts, stream);
  return launch_mx_tiles<Cfg, kMxDense>(p, tiles_m, 1, stream);
}

// Few rows: which kernel, and how many waves share a workgroup's contraction.
constexpr int64_t kFewMaxRows = 64;
int few_waves(int64_t workgroups, int64_t steps) {
  int waves = 4;
  while (waves < 16 && workgroups * waves < 2048 && 2 * waves <= steps) waves *= 2;
  return static_cast<int>(waves < steps ? waves : steps);
}
int few_lds_bytes(const MxFewParams& p, int token_blocks, bool quantize) {
  return p.waves * token_blocks * 16 * 17 * 4 + (quantize ? kFewQuantize * (static_cast<int>(p.ld) + 16 + 8 * p.steps) : 0);
}

// kDense: p.m rows at most kFewMaxRows; kExperts: any rows, 16 of an expert at a time.
template <bool kExperts, bool kQuantize>
int launch_few(MxFewParams& p, int32_t dtype, hipStream_t stream) {
  const int64_t tiles_n = ceil_div(p.n, static_cast<int64_t>(kFewRows)), blocks = tiles_n * (kExperts ? p.experts + 1 : 1);
  if (blocks > 0x3FFFFFLL) return fail(FSH_ENOTSUP, "fsh_mxfp4_gemm: too many tiles");
  p.tiles_n = static_cast<int32_t>(tiles_n);
  p.waves = few_waves(blocks, p.steps);
  const dim3 grid(static_cast<uint32_t>(blocks)), block(64 * p.waves);
  const int token_blocks = kExperts || p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4;
  const int lds = few_lds_bytes(p, token_blocks, kQuantize);
  by_dtype(dtype, [&](auto dt) {
    if (token_blocks == 1) hipLaunchKernelGGL((mxfp4_few_rows_kernel<dt.value, 1, kExperts, kQuantize>), grid, block, lds, stream, p);
    else if constexpr (!kExperts && !kQuantize) {
      if (token_blocks == 2) hipLaunchKernelGGL((mxfp4_few_rows_kernel<dt.value, 2, false, false>), grid, block, lds, stream, p);
      else hipLaunchKernelGGL((mxfp4_few_rows_kernel<dt.value, 4, false, false>), grid, block, lds, stream, p);
    }
  });
  return check_launch("mxfp4_few_rows_kernel");
}

MxFewParams few_params(const fsh_mxfp4_product& q) {
  MxFewParams p;
  memset(&p, 0, sizeof(p));
  p.a = static_cast<const uint8_t*>(q.a_dev); p.as = static_cast<const uint8_t*>(q.a_scales_dev);
  p.b = static_cast<const uint8_t*>(q.b_dev); p.bs = static_cast<const uint8_t*>(q.b_scales_dev);
  p.out = q.out_dev; p.bias = q.bias_dev;
  p.m = q.m; p.n = q.n; p.a_rows = q.a_rows; p.b_rows = q.b_rows;
  p.ld = q.k / 2; p.ldo = q.ldo;
  p.steps = static_cast<int32_t>(q.k / kMxColumns);
  p.experts = q.experts; p.top_k = q.top_k;
  p.offsets = q.offsets_dev; p.source = q.source_dev;
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
  if (q.mode != FSH_MXFP4_DENSE && q.mode != FSH_MXFP4_ROWS && q.mode != FSH_MXFP4_OVER_ROWS)
    return fail(FSH_EINVAL, "%s: unknown mode %d", who, q.mode);
  if (q.mode != FSH_MXFP4_DENSE && q.experts <= 0) return fail(FSH_EINVAL, "%s: no expert", who);
  if (q.m == 0 || q.n == 0) return FSH_OK;
  if (!known_dtype(q.out_dtype)) return fail(FSH_EINVAL, "%s: unknown dtype %d", who, q.out_dtype);
  if (!q.a_dev || !q.a_scales_dev || !q.b_dev || !q.b_scales_dev || !q.out_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (q.k == 0 || q.k % kMxColumns)
    return fail(FSH_ENOTSUP, "%s: k must be a positive multiple of %d (operands are padded), got %lld", who, kMxColumns, (long long)q.k);
  if (q.k >= (1LL << 31) || q.m >= (1LL << 28) || q.n >= (1LL << 28) || q.a_rows >= (1LL << 28) || q.b_rows >= (1LL << 28))
    return fail(FSH_ENOTSUP, "%s: sizes beyond 2^28 rows or 2^31 columns", who);
  if (q.ldo < q.n) return fail(FSH_EINVAL, "%s: ldo %lld < n %lld", who, (long long)q.ldo, (long long)q.n);
  const bool segments = q.mode == FSH_MXFP4_ROWS;
  if (q.mode != FSH_MXFP4_DENSE && !q.offsets_dev) return fail(FSH_EINVAL, "%s: segments without offsets", who);
  if (segments && q.top_k <= 0) return fail(FSH_EINVAL, "%s: top_k must be positive", who);
  if (q.a_rows < (q.source_dev ? 1 : q.m) || q.b_rows < q.n * (segments ? q.experts : 1))
    return fail(FSH_EINVAL, "%s: operands of %lld and %lld rows are too few", who, (long long)q.a_rows, (long long)q.b_rows);
  if (q.source_dev && !segments) return fail(FSH_EINVAL, "%s: gathered rows belong to segments of rows", who);
  if (q.mode == FSH_MXFP4_OVER_ROWS && (q.bias_dev || q.ldo != q.n))
    return fail(FSH_EINVAL, "%s: products over rows are contiguous and have no bias", who);
  if (segments && q.bias_dev) return fail(FSH_ENOTSUP, "%s: segments have no bias", who);
  if (!aligned(q.a_dev, 16) || !aligned(q.b_dev, 16) || !aligned(q.a_scales_dev, 8) || !aligned(q.b_scales_dev, 8) ||
      !aligned(q.out_dev, dtype_bytes(q.out_dtype)) || !aligned(q.bias_dev, dtype_bytes(q.out_dtype)))
    return fail(FSH_ENOTSUP, "%s: data must be 16-byte and scales 8-byte aligned, out and bias to their elements", who);
  // The lanes' offsets are 32 bits from a tile's first row, or from the matrix for gathered rows.
  if (256 * (q.k / 2) >= (1LL << 32) || (q.source_dev && q.a_rows * (q.k / 2) >= (1LL << 32)))
    return fail(FSH_ENOTSUP, "%s: rows that are gathered, or a tile of them, span 4 GiB or more", who);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (q.mode == FSH_MXFP4_DENSE && q.m <= kFewMaxRows) {
    MxFewParams few = few_params(q);
    return launch_few<false, false>(few, q.out_dtype, on);
  }
  if (segments && q.m <= 16 * static_cast<int64_t>(q.experts)) {
    MxFewParams few = few_params(q);
    return launch_few<true, false>(few, q.out_dtype, on);
  }
  MxGemmParams p;
  memset(&p, 0, sizeof(p));
  p.a = static_cast<const uint8_t*>(q.a_dev); p.as = static_cast<const uint8_t*>(q.a_scales_dev);
  p.b = static_cast<const uint8_t*>(q.b_dev); p.bs = static_cast<const uint8_t*>(q.b_scales_dev);
  p.out = q.out_dev; p.bias = q.bias_dev;
  p.m = q.m; p.n = q.n; p.k = q.k;
  p.a_rows = q.a_rows; p.b_rows = q.b_rows;
  p.lda = p.ldb = q.k / 2;
  p.ldo = q.ldo;
  p.out_dtype = q.out_dtype;
  p.experts = q.experts; p.top_k = q.top_k;
  p.offsets = p.padded_offsets = q.offsets_dev;
  p.source = q.source_dev;
  const MxProblem problem = segments ? kMxRows : q.mode == FSH_MXFP4_OVER_ROWS ? kMxOverRows : kMxDense;
  const int64_t rows = segments ? q.m / q.experts : q.m;
  if (rows * q.n >= 128 * 128 * 64) return launch_mx<MxLarge>(p, problem, on);
  return launch_mx<MxSmall>(p, problem, on);
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
  if (rows < 0 || in_dim < 0) return fail(FSH_EINVAL, "%s: negative shape", who);
  fsh_mxfp4_product q = *product;
  if (q.k != ceil_div(in_dim, (int64_t)kMxColumns) * kMxColumns)
    return fail(FSH_EINVAL, "%s: k %lld is not in_dim %lld rounded up to %d", who, (long long)q.k, (long long)in_dim, kMxColumns);
  if (q.out_dtype != dtype) return fail(FSH_EINVAL, "%s: the output has the activation's dtype", who);
  if (q.m == 0 || q.n == 0 || rows == 0) return FSH_OK;
  q.a_rows = rows;
  if (q.mode == FSH_MXFP4_DENSE && q.m <= kFewQuantize) {
    MxFewParams p = few_params(q);
    p.waves = 16;
    if (few_lds_bytes(p, 1, true) <= 64 * 1024) {
      if (!known_dtype(dtype)) return fail(FSH_EINVAL, "%s: unknown dtype %d", who, dtype);
      if (rows < q.m || ldx < in_dim || q.ldo < q.n || q.b_rows < q.n)
        return fail(FSH_EINVAL, "%s: rows or leading dimensions too small", who);
      if (!x_dev || !q.b_dev || !q.b_scales_dev || !q.out_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
      const int bytes = dtype_bytes(dtype);
      if (!aligned(x_dev, bytes) || !aligned(q.b_dev, 16) || !aligned(q.b_scales_dev, 8) || !aligned(q.out_dev, bytes) || !aligned(q.bias_dev, bytes))
        return fail(FSH_ENOTSUP, "%s: weights must be 16-byte and scales 8-byte aligned, x, out and bias to their elements", who);
      p.a = static_cast<const uint8_t*>(x_dev);
      p.cols = in_dim; p.ldx = ldx;
      p.vec = aligned(x_dev, 16) && ldx * bytes % 16 == 0;
      return launch_few<false, true>(p, dtype, static_cast<hipStream_t>(stream));
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
