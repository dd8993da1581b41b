// Gradients of the root-mean-square norm (norm_forward.hip):
//
//   n = h s,  a = dy w,  c = mean(a n) over the row
//   dh = s (a - n c) + (the gradient of h from what reads it besides)
//   dx = dr = dh, rounded to their types;  dw = sum over the rows of dy n
//
// Bound by memory: dy, h and the gradient of h are read once, dx is written once.
// A workgroup takes rows in turn and keeps its part of dw in registers, in fp32;
// the parts are added up in a fixed order by a second kernel.  Measured, both: 8192 x 4096 bf16 with a
// residual 46 + 4 us, 5.8 TB/s in the first; 262144 x 128 37 + 4, 5.4; 1000 x 1001 fp32 6.3 + 4.6.
// Requesting the next row ahead of the present one's sum changed nothing up to 8192 columns
// and spilled at 16384.
#include "norm_layout.hpp"

namespace fsh {
namespace {

struct NormGradParams {
  const void* grad;
  const void* h;
  const void* weight;
  const float* rstd;
  const void* grad_total;
  void* grad_x;
  void* grad_residual;
  float* parts;  // [workgroups][cols], or null
  int64_t rows, cols, ldg, ldh, ldt;
  int64_t row_blocks;
  int32_t weight_dtype;
};

// Workgroups that rows are dealt out to, so many that all are resident: of 256
// threads, of up to 512, of 1024.  More leave more parts of dw: 8192 rows of 4096 bf16 take 56 us with 512
// of 512 threads, 58 with 768, 68 with 256; of 7168 93 with 256 of 1024, 99 with 512; 24576 of 1280 51 with 512 of 256
// threads, 61 with 768.
template <typename L>
constexpr int kGradGroups = L::THREADS == 256 ? (L::PER > 16 ? 512 : 1024) : L::THREADS <= 512 ? 512 : 256;

// (two workgroups of 448 in a compute unit: 128 registers)
template <int GT, int HT, int XT, typename L>
__global__ __launch_bounds__(L::THREADS, L::THREADS == 448 ? 4 : 1) void rms_norm_grad_kernel(const NormGradParams p) {
  constexpr int VEC = L::VEC, ITEMS = L::ITEMS;
  // fp32 outputs leave past the caches: 8192 rows of 7168 on an fp32 stream 187 -> 167 us; bf16 ones
  // the layer behind finds there (4096 of bf16: 56 us either way).
  constexpr bool kStreamOut = HT == FSH_DT_F32;
  // Where the registers would not do: 4096 rows of 9001 on an fp32 stream 122 us for 151 (of bf16 82 for 79).
  constexpr bool kAgain = L::ENDS == kOverlapping && VEC == 4 && L::THREADS == 1024 && L::PER == 16;
  __shared__ float lds[L::LANES > 64 ? 2 * L::LANES / 64 : L::ROWS * L::LANES * L::PER];
  const int lane = threadIdx.x % L::LANES, group = threadIdx.x / L::LANES, cols = static_cast<int>(p.cols);
  float w[ITEMS][VEC], part[ITEMS][VEC];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    NormVector<L>((i * L::LANES + lane) * VEC, cols).weights(p.weight, p.weight_dtype, w[i]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) part[i][j] = 0.0f;
  }
  int turn = 0;
  for (int64_t block = blockIdx.x; block < p.row_blocks; block += gridDim.x, ++turn) {
    const int64_t row = block * L::ROWS + group;
    const bool live = row < p.rows;
    RawVec<GT, VEC> g[ITEMS];
    RawVec<HT, VEC> h[ITEMS], t[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const NormVector<L> c((i * L::LANES + lane) * VEC, cols);
      g[i] = c.template load<GT>(p.grad, row * p.ldg, live);
      h[i] = c.template load<HT>(p.h, row * p.ldh, live);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      t[i] = NormVector<L>((i * L::LANES + lane) * VEC, cols).template load<HT>(p.grad_total, row * p.ldt, live && p.grad_total);
    const float s = live ? p.rstd[row] : 0.0f;
    float sum = 0.0f;
    const int lane_sum = lane_again<kAgain>(lane);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const NormVector<L> c((i * L::LANES + lane_sum) * VEC, cols);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float dy = element<GT, VEC>(g[i], j), n = element<HT, VEC>(h[i], j) * s;
        sum += j < c.skip ? 0.0f : dy * w[i][j] * n;
        part[i][j] += dy * n;
      }
    }
    const float c = sum_over_row<L::LANES>(sum, lds, turn) / static_cast<float>(p.cols);
    const int lane_out = lane_again<kAgain>(lane);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const NormVector<L> v((i * L::LANES + lane_out) * VEC, cols);
      if (!live || !v.inside) continue;
      float d[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float dy = element<GT, VEC>(g[i], j), n = element<HT, VEC>(h[i], j) * s;
        d[j] = s * (dy * w[i][j] - n * c) + element<HT, VEC>(t[i], j);
      }
      if (p.grad_x) v.template store<XT, kStreamOut>(p.grad_x, row * p.cols, to_vec<XT, VEC>(d));
      if (HT != XT && p.grad_residual) v.template store<HT, kStreamOut>(p.grad_residual, row * p.cols, to_vec<HT, VEC>(d));
    }
  }
  if (!p.parts) return;
  float* const mine = p.parts + blockIdx.x * p.cols;
  if constexpr (L::ROWS == 1) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const NormVector<L> v((i * L::LANES + lane) * VEC, cols);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (v.inside && j < v.count) mine[v.at + j] = part[i][j];
    }
  } else {
    // (LANES <= 64: no sum over a row goes through LDS)
    constexpr int kWidth = L::LANES * L::PER;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const NormVector<L> v((i * L::LANES + lane) * VEC, cols);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (v.inside) lds[group * kWidth + v.at + j] = part[i][j];
    }
    __syncthreads();
    for (int col = threadIdx.x; col < cols; col += L::THREADS) {
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < L::ROWS; ++k) sum += lds[k * kWidth + col];
      mine[col] = sum;
    }
  }
}

// Rows that do not fit the registers: the sum first, then the gradients, with dw's
// part of a workgroup read and written for every row it takes.  What is read or written
// for the last time streams, so that the parts stay in the caches (2048 rows of 20480 bf16 131 us; with the
// parts read and written by elements 200, and nothing streamed 213).
template <int GT, int HT, int XT, typename L>
__global__ __launch_bounds__(L::THREADS) void rms_norm_grad_wide_kernel(const NormGradParams p) {
  constexpr int VEC = L::VEC, STEP = L::THREADS * VEC;
  __shared__ float lds[2 * L::THREADS / 64];
  int turn = 0;
  float* const mine = p.parts ? p.parts + blockIdx.x * p.cols : nullptr;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, ++turn) {
    const float s = p.rstd[row];
    float sum = 0.0f;
    for (int64_t col = threadIdx.x * VEC; col < p.cols; col += STEP) {
      const auto g = load_vec<GT, VEC>(p.grad, row * p.ldg + col, p.cols - col);
      const auto h = load_vec<HT, VEC>(p.h, row * p.ldh + col, p.cols - col);
      float w[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] = 1.0f;
      if (p.weight) load_floats<VEC>(p.weight, p.weight_dtype, col, p.cols - col, w);
      const auto before = load_vec<FSH_DT_F32, VEC>(mine, col, mine && turn ? p.cols - col : 0);
      float part[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float dy = element<GT, VEC>(g, j), n = element<HT, VEC>(h, j) * s;
        sum += dy * w[j] * n;
        part[j] = element<FSH_DT_F32, VEC>(before, j) + dy * n;
      }
      if (mine) store_vec<FSH_DT_F32, VEC>(mine, col, p.cols - col, to_vec<FSH_DT_F32, VEC>(part));
    }
    const float c = sum_over_row<L::THREADS>(sum, lds, turn) / static_cast<float>(p.cols);
    for (int64_t col = threadIdx.x * VEC; col < p.cols; col += STEP) {
      const auto g = load_vec<GT, VEC, true>(p.grad, row * p.ldg + col, p.cols - col);
      const auto h = load_vec<HT, VEC, true>(p.h, row * p.ldh + col, p.cols - col);
      const auto t = load_vec<HT, VEC, true>(p.grad_total, row * p.ldt + col, p.grad_total ? p.cols - col : 0);
      float w[VEC], d[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] = 1.0f;
      if (p.weight) load_floats<VEC>(p.weight, p.weight_dtype, col, p.cols - col, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float dy = element<GT, VEC>(g, j), n = element<HT, VEC>(h, j) * s;
        d[j] = s * (dy * w[j] - n * c) + element<HT, VEC>(t, j);
      }
      if (p.grad_x) store_vec<XT, VEC, true>(p.grad_x, row * p.cols + col, p.cols - col, to_vec<XT, VEC>(d));
      if (HT != XT && p.grad_residual) store_vec<HT, VEC, true>(p.grad_residual, row * p.cols + col, p.cols - col, to_vec<HT, VEC>(d));
    }
  }
}

// dw[c] = the sum of the workgroups' parts: 32 columns a workgroup, 32 threads a
// column, always in the same order.
template <int DT>
__global__ __launch_bounds__(1024) void norm_weight_grad_kernel(const float* parts, void* out, int64_t groups, int64_t cols) {
  __shared__ float lds[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.0f;
  if (c < cols) {
#pragma unroll 16
    for (int64_t r = slice; r < groups; r += 32) sum += parts[r * cols + c];
  }
  lds[slice][lane] = sum;
  __syncthreads();
  // (a slice's threads now share a column, a half-wave)
  sum = sum32(lds[lane][slice]);
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * 32 + slice;
  if (lane != 0 || mine >= cols) return;
  if (DT == FSH_DT_F32) static_cast<float*>(out)[mine] = sum;
  else static_cast<uint16_t*>(out)[mine] = static_cast<uint16_t>(bits_of<DT>(sum));
}

// launch(layout) with the layout for rows of `cols` columns.  Two workgroups or more to a
// compute unit: 8192 rows of 5120 bf16 take 63 us by 448 threads, 78 by 1024 (but with
// an fp32 stream 178 for 166).  With few rows the parts of dw count for more: 512 of 7168 take 19.0 us for 17.6, of 5120 16.1 for 15.4; the
// two are alike at 1000 and at 768, and at the border 1024 threads take 1.7 and 2.4 us longer.  24576 of 1040 47 by 64 and 56 by 256; 16384 of 2048 51 and 54.
template <int ENDS, int VEC, typename Launch>
void by_columns(int64_t rows, int64_t cols, Launch launch) {
  if (ENDS == kPieces || cols <= 64) launch(NormLayout<ENDS, 64 / VEC, VEC, VEC>{});
  else if constexpr (ENDS == kPieces) return;
  else if (cols <= 128) launch(NormLayout<ENDS, 128 / VEC, VEC, VEC>{});
  else if (cols <= 256) launch(NormLayout<ENDS, 256 / VEC, VEC, VEC>{});
  else if (cols <= 512) launch(NormLayout<ENDS, 64, 8, VEC>{});
  else if (cols <= 1024) launch(NormLayout<ENDS, 64, 16, VEC>{});
  else if (cols <= 1536) launch(NormLayout<ENDS, 64, 24, VEC>{});
  else if (cols <= 2048) launch(NormLayout<ENDS, 64, 32, VEC>{});
  else if (cols <= 4096) launch(NormLayout<ENDS, 512, 8, VEC>{});
  else if (cols <= 7168 && VEC == 8 && rows > 2048) launch(NormLayout<ENDS, VEC == 8 ? 448 : 1024, VEC == 8 ? 16 : 8, VEC>{});
  else if (cols <= 8192) launch(NormLayout<ENDS, 1024, 8, VEC>{});
  else if (cols <= 16384) launch(NormLayout<ENDS, 1024, 16, VEC>{});
  else launch(NormLayout<kEven, 1024, 0, VEC>{});  // (any columns)
}

// Workgroups that a gradient's rows are dealt out to: as many parts of dw.
template <typename L>
int64_t groups_of(int64_t rows) {
  const int64_t blocks = ceil_div(rows, (int64_t)L::ROWS);
  return blocks < kGradGroups<L> ? blocks : kGradGroups<L>;
}
template <int VEC>
int64_t groups_of(int64_t rows, int64_t cols) {
  int64_t groups = 0;
  by_ends<VEC>(cols, [&](auto ends) { by_columns<ends.value, VEC>(rows, cols, [&](auto layout) { groups = groups_of<decltype(layout)>(rows); }); });
  return groups;
}

// Launches the gradients; returns how many parts of dw they leave, or -1 without
// room for them.
template <int GT, int HT, int XT>
int64_t launch_grad(NormGradParams& p, int64_t room, hipStream_t stream) {
  constexpr int VEC = GT == FSH_DT_F32 || HT == FSH_DT_F32 || XT == FSH_DT_F32 ? 4 : 8;
  int64_t groups = 0;
  by_ends<VEC>(p.cols, [&](auto ends) {
    by_columns<ends.value, VEC>(p.rows, p.cols, [&](auto layout) {
      using L = decltype(layout);
      p.row_blocks = ceil_div(p.rows, (int64_t)L::ROWS);
      groups = groups_of<L>(p.rows);
      if (p.parts && groups * p.cols > room) {
        groups = -1;
        return;
      }
      const dim3 grid(static_cast<uint32_t>(groups)), block(L::THREADS);
      if constexpr (L::PER == 0)
        hipLaunchKernelGGL((rms_norm_grad_wide_kernel<GT, HT, XT, L>), grid, block, 0, stream, p);
      else
        hipLaunchKernelGGL((rms_norm_grad_kernel<GT, HT, XT, L>), grid, block, 0, stream, p);
    });
  });
  return groups;
}

}  // namespace
}  // namespace fsh

FSH_API int64_t fsh_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  using namespace fsh;
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t four = groups_of<4>(rows, cols), eight = groups_of<8>(rows, cols), groups = four > eight ? four : eight;
  return groups * cols * static_cast<int64_t>(sizeof(float));
}

FSH_API int fsh_rms_norm_backward(const fsh_norm_gradient* q, void* stream) {
  using namespace fsh;
  const char* who = "fsh_rms_norm_backward";
  if (!q) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (q->rows < 0 || q->cols < 0) return fail(FSH_EINVAL, "%s: negative shape", who);
  const int g = q->grad_dtype, h = q->total_dtype, x = q->x_dtype;
  if (!is_dtype(g) || !is_dtype(h) || !is_dtype(x) || (q->weight_dev && !is_dtype(q->weight_dtype)))
    return fail(FSH_EINVAL, "%s: unknown dtype (%d, %d, %d, %d)", who, g, h, x, q->weight_dtype);
  if ((g != x && g != FSH_DT_BF16) || (h != x && h != FSH_DT_F32))
    return fail(FSH_EINVAL, "%s: a gradient of dtype %d (that of x, %d, or bf16) of a sum of dtype %d (that of x, or fp32)", who, g, x, h);
  if (q->grad_weight_dev && !q->weight_dev) return fail(FSH_EINVAL, "%s: a weight's gradient without a weight", who);
  if (q->rows == 0 || q->cols == 0) {
    if (q->grad_weight_dev && q->cols) return fail(FSH_ENOTSUP, "%s: a weight's gradient needs rows", who);
    return FSH_OK;
  }
  if (!q->grad_dev || !q->total_dev || !q->rstd_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (q->ldg < q->cols || q->ldh < q->cols || (q->grad_total_dev && q->ldt < q->cols))
    return fail(FSH_EINVAL, "%s: a row stride (%lld, %lld, %lld) is less than cols %lld", who, (long long)q->ldg, (long long)q->ldh, (long long)q->ldt,
                (long long)q->cols);
  if (!aligned(q->grad_dev, bytes_of(g)) || !aligned(q->total_dev, bytes_of(h)) || !aligned(q->rstd_dev, 4) || !aligned(q->grad_total_dev, bytes_of(h)) ||
      !aligned(q->grad_x_dev, bytes_of(x)) || !aligned(q->grad_residual_dev, bytes_of(h)) || !aligned(q->workspace_dev, 4) ||
      (q->weight_dev && (!aligned(q->weight_dev, bytes_of(q->weight_dtype)) || !aligned(q->grad_weight_dev, bytes_of(q->weight_dtype)))))
    return fail(FSH_ENOTSUP, "%s: tensors must be aligned to their elements", who);
  if (q->grad_weight_dev && (!q->workspace_dev || q->workspace_nbytes < fsh_rms_norm_backward_workspace_bytes(q->rows, q->cols)))
    return fail(FSH_EINVAL, "%s: workspace of %lld bytes, %lld needed", who, (long long)q->workspace_nbytes,
                (long long)fsh_rms_norm_backward_workspace_bytes(q->rows, q->cols));
  if (ceil_div(q->cols, (int64_t)32) > (1LL << 22) - 1) return fail(FSH_ENOTSUP, "%s: too many columns", who);
  // (the last columns of a row are written twice, by two lanes that have read them)
  const int64_t n = q->rows, k = q->cols;
  const RowSpan inputs[] = {{q->grad_dev, n, k, q->ldg, bytes_of(g)},
                            {q->total_dev, n, k, q->ldh, bytes_of(h)},
                            {q->grad_total_dev, n, k, q->ldt, bytes_of(h)},
                            span_of(q->weight_dev, k, bytes_of(q->weight_dtype)),
                            span_of(q->rstd_dev, n, 4)};
  const RowSpan outputs[] = {span_of(q->grad_x_dev, n * k, bytes_of(x)),
                             span_of(h == x ? nullptr : q->grad_residual_dev, n * k, bytes_of(h)),
                             span_of(q->grad_weight_dev, k, bytes_of(q->weight_dtype)),
                             span_of(q->grad_weight_dev ? q->workspace_dev : nullptr, fsh_rms_norm_backward_workspace_bytes(n, k), 1)};
  if (outputs_overlap(inputs, outputs)) return fail(FSH_EINVAL, "%s: an output or the workspace overlaps an input or another output", who);
  NormGradParams p = {};
  p.grad = q->grad_dev;
  p.h = q->total_dev;
  p.weight = q->weight_dev;
  p.rstd = q->rstd_dev;
  p.grad_total = q->grad_total_dev;
  p.grad_x = q->grad_x_dev;
  p.grad_residual = q->grad_residual_dev;
  p.parts = q->grad_weight_dev ? static_cast<float*>(q->workspace_dev) : nullptr;
  p.rows = q->rows;
  p.cols = q->cols;
  p.ldg = q->ldg;
  p.ldh = q->ldh;
  p.ldt = q->ldt;
  p.weight_dtype = q->weight_dtype;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  const int64_t room = q->workspace_nbytes / static_cast<int64_t>(sizeof(float));
  int64_t groups;
  if (x == FSH_DT_BF16) groups = h == x ? launch_grad<FSH_DT_BF16, FSH_DT_BF16, FSH_DT_BF16>(p, room, on) : launch_grad<FSH_DT_BF16, FSH_DT_F32, FSH_DT_BF16>(p, room, on);
  else if (x == FSH_DT_F16 && g == x) groups = h == x ? launch_grad<FSH_DT_F16, FSH_DT_F16, FSH_DT_F16>(p, room, on) : launch_grad<FSH_DT_F16, FSH_DT_F32, FSH_DT_F16>(p, room, on);
  else if (x == FSH_DT_F16) groups = h == x ? launch_grad<FSH_DT_BF16, FSH_DT_F16, FSH_DT_F16>(p, room, on) : launch_grad<FSH_DT_BF16, FSH_DT_F32, FSH_DT_F16>(p, room, on);
  else if (g == x) groups = launch_grad<FSH_DT_F32, FSH_DT_F32, FSH_DT_F32>(p, room, on);
  else groups = launch_grad<FSH_DT_BF16, FSH_DT_F32, FSH_DT_F32>(p, room, on);
  if (groups < 0) return fail(FSH_EINVAL, "%s: workspace of %lld bytes", who, (long long)q->workspace_nbytes);
  if (int rc = check_launch("rms_norm_grad_kernel")) return rc;
  if (!q->grad_weight_dev) return FSH_OK;
  const dim3 grid(static_cast<uint32_t>(ceil_div(q->cols, (int64_t)32))), block(1024);
  if (q->weight_dtype == FSH_DT_BF16) hipLaunchKernelGGL(norm_weight_grad_kernel<FSH_DT_BF16>, grid, block, 0, on, p.parts, q->grad_weight_dev, groups, q->cols);
  else if (q->weight_dtype == FSH_DT_F16) hipLaunchKernelGGL(norm_weight_grad_kernel<FSH_DT_F16>, grid, block, 0, on, p.parts, q->grad_weight_dev, groups, q->cols);
  else hipLaunchKernelGGL(norm_weight_grad_kernel<FSH_DT_F32>, grid, block, 0, on, p.parts, q->grad_weight_dev, groups, q->cols);
  return check_launch("norm_weight_grad_kernel");
}
