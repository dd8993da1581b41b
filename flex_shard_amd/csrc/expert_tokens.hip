// Tokens sorted by expert, gathered, and brought back with the router's weights;
// and the gradients.
//
//   route     a stable counting sort of the choices by expert: a choice's row is
//             the expert's first row + the earlier choices of that expert
//   dispatch  out[position[t, j]] = x[t]
//   combine   out[t] = sum_j w[t, j] rows[position[t, j]]
//   combine's gradient: grad_rows[position[t, j]] = w[t, j] grad[t],
//             grad_w[t, j] = <grad[t], rows[position[t, j]]>
//
// The sort is bound by latency; the others by memory: every row of the experts
// is read or written once, the tokens' rows once.  Measured, 8192 tokens of 7168
// bf16, 8 of 32 experts each: sort 13 us; dispatch 187 us, 5.7 TB/s; combine 212 us,
// 5.0; its gradient 393 us, 5.1.  4096 tokens' fp32 rows combined to bf16: 205 us,
// 4.9.  16 tokens: 3.6, 4.2 and 4.8 us, a launch's chain of loads each.
#include "mxfp4.hpp"

namespace fsh {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMaxGrid = (1LL << 32) / kThreads - 1;
constexpr int kMaxExperts = FSH_MAX_EXPERTS;
constexpr int kSegmentPad = kMxColumns;

// ------------------------------------------------------------------- the sort
constexpr int kChoicesPerBlock = 2048;

struct RouteParams {
  const void* ids;
  int64_t choices;
  int32_t id_bytes, experts, blocks;
  int32_t* position;
  int32_t* offsets;
  int32_t* source;
  int32_t* padded_offsets;
  int32_t* counts;  // [blocks][experts]
};

// Lanes of a wave hand LDS values to one another in program order; the compiler is kept to it.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The expert of choice i: p.experts for none.
__device__ __forceinline__ int expert_of(const RouteParams& p, int64_t i) {
  const int64_t id = p.id_bytes == 8 ? static_cast<const int64_t*>(p.ids)[i] : static_cast<const int32_t*>(p.ids)[i];
  return id < 0 || id >= p.experts ? p.experts : static_cast<int>(id);
}

// How many choices of each expert every block of choices has.
__global__ __launch_bounds__(kThreads) void expert_count_kernel(const RouteParams p) {
  __shared__ int32_t count[kMaxExperts];
  for (int e = threadIdx.x; e < p.experts; e += kThreads) count[e] = 0;
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kChoicesPerBlock;
#pragma unroll
  for (int i = 0; i < kChoicesPerBlock / kThreads; ++i) {
    const int64_t at = first + i * kThreads + threadIdx.x;
    const int e = at < p.choices ? expert_of(p, at) : p.experts;
    if (e < p.experts) atomicAdd(&count[e], 1);  // whole numbers: any order gives the same
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kThreads) p.counts[static_cast<int64_t>(blockIdx.x) * p.experts + e] = count[e];
}

// Each wave places a quarter of the block's choices, 64 at a time: a choice's
// rank among the 64 is the number of earlier lanes with its expert.  Every block
// reads all blocks' counts, which in all is quadratic in the choices: 32 blocks of
// 32 counts for 8192 tokens of 8 choices, 4 KB a block.
__global__ __launch_bounds__(kThreads) void expert_place_kernel(const RouteParams p) {
  __shared__ int32_t next[kWaves][kMaxExperts];  // first the waves' counts, then the next row of each expert
  __shared__ int32_t total[kMaxExperts + 1], before[kMaxExperts];  // of all blocks, of those before this one
  __shared__ int32_t wave_sum[2][kWaves];
  constexpr int kPerWave = kChoicesPerBlock / kWaves, kRounds = kPerWave / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kChoicesPerBlock + wave * kPerWave;
  int mine[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int64_t at = first + 64 * i + lane;
    mine[i] = at < p.choices ? expert_of(p, at) : p.experts;
  }
  for (int e = tid; e < p.experts; e += kThreads) {
    total[e] = before[e] = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) next[w][e] = 0;
  }
  __syncthreads();
  // (whole numbers: the order of the additions does not matter)
#pragma unroll
  for (int i = 0; i < kRounds; ++i)
    if (mine[i] < p.experts) atomicAdd(&next[wave][mine[i]], 1);
  if (p.blocks > 1) {
    const int own = static_cast<int>(blockIdx.x) * p.experts, counts = p.blocks * p.experts;
#pragma unroll 4
    for (int i = tid; i < counts; i += kThreads) {
      const int32_t c = p.counts[i];
      const int e = i % p.experts;
      if (c) atomicAdd(&total[e], c);
      if (c && i < own) atomicAdd(&before[e], c);
    }
  }
  __syncthreads();
  // A thread has neighbouring experts, for the scan over them.
  constexpr int kPerThread = kMaxExperts / kThreads;
  const int used = (p.experts + kThreads - 1) / kThreads;  // experts per thread
  int32_t all[kPerThread];
  int32_t sum = 0, padded_sum = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int e = tid * used + i;
    all[i] = 0;
    if (i >= used || e >= p.experts) continue;
    if (p.blocks > 1) {
      all[i] = total[e];
    } else {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all[i] += next[w][e];
    }
    sum += all[i];
    padded_sum += (all[i] + kSegmentPad - 1) / kSegmentPad * kSegmentPad;
  }
  int32_t scan = sum, padded_scan = padded_sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int32_t a = __shfl_up(scan, off, kWave), b = __shfl_up(padded_scan, off, kWave);
    if (lane >= off) {
      scan += a;
      padded_scan += b;
    }
  }
  if (lane == 63) {
    wave_sum[0][wave] = scan;
    wave_sum[1][wave] = padded_scan;
  }
  __syncthreads();
  int32_t row = scan - sum, padded = padded_scan - padded_sum;
  for (int w = 0; w < wave; ++w) {
    row += wave_sum[0][w];
    padded += wave_sum[1][w];
  }
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int e = tid * used + i;
    if (i >= used || e >= p.experts) continue;
    int32_t at = row + before[e];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int32_t c = next[w][e];
      next[w][e] = at;
      at += c;
    }
    row += all[i];
    padded += (all[i] + kSegmentPad - 1) / kSegmentPad * kSegmentPad;
    if (e + 1 == p.experts) total[p.experts] = row;
    if (blockIdx.x == 0) {
      p.offsets[e + 1] = row;
      p.padded_offsets[e + 1] = padded;
    }
  }
  if (blockIdx.x == 0 && tid == 0) p.offsets[0] = p.padded_offsets[0] = 0;
  __syncthreads();
  int bits = 0;
  while ((1 << bits) <= p.experts) ++bits;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (first + 64 * i >= p.choices) break;  // (the whole wave)
    const int e = mine[i];
    uint64_t same = ~0ull;
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const int64_t at = first + 64 * i + lane;
    int32_t place = -1;
    if (e < p.experts) place = next[wave][e] + rank;
    wave_fence();
    if (e < p.experts && rank == 0) next[wave][e] += __popcll(same);
    wave_fence();
    if (at < p.choices) {
      p.position[at] = place;
      if (place >= 0) p.source[place] = static_cast<int32_t>(at);
    }
  }
  // The rows behind the last expert's: this block's share of them.
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kThreads + tid; r < p.choices; r += static_cast<int64_t>(p.blocks) * kThreads)
    if (r >= total[p.experts]) p.source[r] = -1;
}

// ------------------------------------------------------------------ the rows
// A thread has neighbouring elements: where all rows are 16-byte aligned 16 bytes'
// worth (kCount: as many as 16 bytes of another type hold), one otherwise.
template <int DT, bool kVec, int kCount = 16 / element_bytes<DT>()>
struct Piece {
  static constexpr int kElements = kVec ? kCount : 1;
  // kStream: a row that is read once
  template <bool kStream>
  static __device__ __forceinline__ void load(const uint8_t* row, int64_t piece, float (&f)[kElements]) {
    if constexpr (kVec) {
      constexpr int kLoads = kElements * element_bytes<DT>() / 16, kPerLoad = kElements / kLoads;
      const u32x4* at = reinterpret_cast<const u32x4*>(row) + piece * kLoads;
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const u32x4 v = kStream ? __builtin_nontemporal_load(at + l) : at[l];
#pragma unroll
        for (int i = 0; i < kPerLoad; ++i)
          f[l * kPerLoad + i] = DT == FSH_DT_F32 ? u32_as_f32(v[i % 4]) : half_of_pair<DT>(v[i / 2 % 4], i % 2);
      }
    } else {
      f[0] = load_element<DT>(row, piece);
    }
  }
  static __device__ __forceinline__ void store(uint8_t* row, int64_t piece, const float (&f)[kElements]) {
    static_assert(!kVec || kCount * element_bytes<DT>() == 16, "one store");
    if constexpr (!kVec) {
      store_element<DT>(row, piece, f[0]);
    } else if constexpr (DT == FSH_DT_F32) {
      __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4*>(row + piece * 16));
    } else {
      __builtin_nontemporal_store(pack8<DT>(f), reinterpret_cast<u32x4*>(row + piece * 16));
    }
  }
};

struct RowsParams {
  const uint8_t* x;     // dispatch: the tokens' rows; backward: their gradients
  const uint8_t* rows;  // the experts' rows
  uint8_t* out;
  const int32_t* position;
  const int32_t* offsets;
  const void* weights;  // or null
  void* grad_weights;
  int32_t weights_dtype, experts, top_k;
  int64_t tokens, pieces, row_bytes, slabs;
  int64_t out_row_bytes;  // combine: of its output's rows, whose type may differ
};

__device__ __forceinline__ float weight_of(const RowsParams& p, int64_t choice) {
  if (!p.weights) return 1.0f;
  if (p.weights_dtype == FSH_DT_F32) return load_element<FSH_DT_F32>(p.weights, choice);
  if (p.weights_dtype == FSH_DT_F16) return load_element<FSH_DT_F16>(p.weights, choice);
  return load_element<FSH_DT_BF16>(p.weights, choice);
}

// Zeros to the rows behind offsets[experts], by blocks past the tokens' own.
template <int DT, bool kVec>
__device__ __forceinline__ void zero_unused_rows(const RowsParams& p, int64_t block, int64_t blocks) {
  const int64_t rows = p.tokens * p.top_k;
  const float zero[Piece<DT, kVec>::kElements] = {};
  for (int64_t r = p.offsets[p.experts] + block; r < rows; r += blocks)
    for (int64_t i = threadIdx.x; i < p.pieces; i += kThreads) Piece<DT, kVec>::store(p.out + r * p.row_bytes, i, zero);
}
constexpr int kZeroBlocks = 64;

// One token, kThreads pieces of its row: read once, written for every choice.
template <int DT, bool kVec>
__global__ __launch_bounds__(kThreads) void expert_dispatch_kernel(const RowsParams p) {
  using P = Piece<DT, kVec>;
  const int64_t token = blockIdx.x / p.slabs, piece = blockIdx.x % p.slabs * kThreads + threadIdx.x;
  if (token >= p.tokens) {
    zero_unused_rows<DT, kVec>(p, blockIdx.x - p.tokens * p.slabs, kZeroBlocks);
    return;
  }
  if (piece >= p.pieces) return;
  float f[P::kElements];
  P::template load<false>(p.x + token * p.row_bytes, piece, f);
  for (int j = 0; j < p.top_k; ++j) {
    const int64_t row = p.position[token * p.top_k + j];
    if (row >= 0) P::store(p.out + row * p.row_bytes, piece, f);
  }
}

// One token, kThreads pieces of its row.  Eight rows are in flight at a time.  OUT:
// the output's type; fp32 rows can leave as 16 bits, rounded after their sum.
template <int DT, int OUT, bool kVec>
__global__ __launch_bounds__(kThreads) void expert_combine_kernel(const RowsParams p) {
  using P = Piece<DT, kVec, 16 / element_bytes<OUT>()>;
  const int64_t token = blockIdx.x / p.slabs, piece = blockIdx.x % p.slabs * kThreads + threadIdx.x;
  if (piece >= p.pieces) return;
  float sum[P::kElements] = {};
  for (int j0 = 0; j0 < p.top_k; j0 += 8) {
    float f[8][P::kElements], w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t choice = token * p.top_k + j0 + j, row = j0 + j < p.top_k ? p.position[choice] : -1;
      w[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < P::kElements; ++i) f[j][i] = 0.0f;
      if (row >= 0) {
        w[j] = weight_of(p, choice);
        P::template load<true>(p.rows + row * p.row_bytes, piece, f[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j0 + j < p.top_k)
#pragma unroll
        for (int i = 0; i < P::kElements; ++i) sum[i] = __builtin_fmaf(w[j], f[j][i], sum[i]);
  }
  Piece<OUT, kVec>::store(p.out + token * p.out_row_bytes, piece, sum);
}

// One token: a piece of its gradient is read once for eight choices, whose rows are
// in flight together; the dot products are joined over the workgroup in a fixed order.
constexpr int kMaxTopK = FSH_MAX_CHOICES;
template <int DT, bool kVec>
__global__ __launch_bounds__(kThreads) void expert_combine_backward_kernel(const RowsParams p) {
  using P = Piece<DT, kVec>;
  __shared__ float dots[kWaves][kMaxTopK];
  const int64_t token = blockIdx.x;
  if (token >= p.tokens) {
    zero_unused_rows<DT, kVec>(p, token - p.tokens, kZeroBlocks);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int j0 = 0; j0 < p.top_k; j0 += 8) {
    int64_t row[8];
    float w[8], dot[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t choice = token * p.top_k + j0 + j;
      row[j] = j0 + j < p.top_k ? p.position[choice] : -1;
      w[j] = row[j] >= 0 ? weight_of(p, choice) : 0.0f;
      dot[j] = 0.0f;
    }
    for (int64_t piece = threadIdx.x; piece < p.pieces; piece += kThreads) {
      float g[P::kElements], f[8][P::kElements];
      P::template load<false>(p.x + token * p.row_bytes, piece, g);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (row[j] >= 0) P::template load<true>(p.rows + row[j] * p.row_bytes, piece, f[j]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (row[j] >= 0) {
          float out[P::kElements];
#pragma unroll
          for (int i = 0; i < P::kElements; ++i) {
            dot[j] = __builtin_fmaf(g[i], f[j][i], dot[j]);
            out[i] = g[i] * w[j];
          }
          P::store(p.out + row[j] * p.row_bytes, piece, out);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float sum = wave_sum_f32(dot[j]);
      if (lane == 0 && j0 + j < p.top_k) dots[wave][j0 + j] = sum;
    }
  }
  __syncthreads();
  const int j = threadIdx.x;
  if (j < p.top_k) {
    const float dot = dots[0][j] + dots[1][j] + dots[2][j] + dots[3][j];
    const int64_t choice = token * p.top_k + j;
    if (p.weights_dtype == FSH_DT_F32) store_element<FSH_DT_F32>(p.grad_weights, choice, dot);
    else if (p.weights_dtype == FSH_DT_F16) store_element<FSH_DT_F16>(p.grad_weights, choice, dot);
    else store_element<FSH_DT_BF16>(p.grad_weights, choice, dot);
  }
}

// Checks that the row kernels share, and the sizes that follow from the dtype and the pointers.
int rows_checks(RowsParams& p, int64_t tokens, int32_t top_k, int64_t width, int32_t dtype, int32_t out_dtype, bool* vec, const char* who) {
  if (tokens < 0 || width < 0 || top_k <= 0) return fail(FSH_EINVAL, "%s: negative shape, or top_k not positive", who);
  if (!known_dtype(dtype) || !known_dtype(out_dtype) || (p.weights && !known_dtype(p.weights_dtype))) return fail(FSH_EINVAL, "%s: unknown dtype", who);
  if (top_k > kMaxTopK) return fail(FSH_ENOTSUP, "%s: at most %d choices per token, got %d", who, kMaxTopK, top_k);
  if (tokens * top_k >= (1LL << 31)) return fail(FSH_ENOTSUP, "%s: 2^31 choices or more", who);
  if (tokens == 0 || width == 0) return FSH_OK;
  if (!p.position || !p.out) return fail(FSH_EINVAL, "%s: null pointer", who);
  const int bytes = dtype_bytes(dtype), out_bytes = dtype_bytes(out_dtype);
  if (!aligned(p.x, bytes) || !aligned(p.rows, bytes) || !aligned(p.out, out_bytes)) return fail(FSH_ENOTSUP, "%s: misaligned pointer", who);
  p.tokens = tokens; p.top_k = top_k;
  p.row_bytes = width * bytes;
  p.out_row_bytes = width * out_bytes;
  *vec = p.row_bytes % 16 == 0 && p.out_row_bytes % 16 == 0 && aligned(p.x, 16) && aligned(p.rows, 16) && aligned(p.out, 16);
  p.pieces = *vec ? p.out_row_bytes / 16 : width;
  p.slabs = ceil_div(p.pieces, static_cast<int64_t>(kThreads));
  if (tokens * p.slabs + kZeroBlocks > kMaxGrid) return fail(FSH_ENOTSUP, "%s: too many rows", who);
  return FSH_OK;
}

}  // namespace
}  // namespace fsh

FSH_API int64_t fsh_expert_route_workspace_bytes(int64_t choices, int32_t experts) {
  using namespace fsh;
  if (choices <= 0 || experts <= 0) return 0;
  const int64_t blocks = ceil_div(choices, static_cast<int64_t>(kChoicesPerBlock));
  return blocks > 1 ? blocks * experts * 4 : 0;
}

FSH_API int fsh_expert_route(const void* expert_ids_dev, int32_t id_bytes, int64_t choices, int32_t experts, int32_t* position_dev,
                             int32_t* offsets_dev, int32_t* source_dev, int32_t* padded_offsets_dev, void* workspace_dev,
                             int64_t workspace_nbytes, void* stream) {
  using namespace fsh;
  const char* who = "fsh_expert_route";
  if (choices < 0 || experts <= 0) return fail(FSH_EINVAL, "%s: negative size, or no expert", who);
  if (id_bytes != 4 && id_bytes != 8) return fail(FSH_EINVAL, "%s: ids of 4 or 8 bytes, got %d", who, id_bytes);
  if (experts > kMaxExperts) return fail(FSH_ENOTSUP, "%s: at most %d experts, got %d", who, kMaxExperts, experts);
  // (padded segments are counted in 32 bits too)
  if (choices + static_cast<int64_t>(experts) * kSegmentPad >= (1LL << 31)) return fail(FSH_ENOTSUP, "%s: 2^31 rows or more", who);
  if (!offsets_dev || !padded_offsets_dev || (choices && (!expert_ids_dev || !position_dev || !source_dev)))
    return fail(FSH_EINVAL, "%s: null pointer", who);
  if (!aligned(expert_ids_dev, id_bytes)) return fail(FSH_ENOTSUP, "%s: misaligned ids", who);
  const int64_t need = fsh_expert_route_workspace_bytes(choices, experts);
  if (need && (!workspace_dev || workspace_nbytes < need))
    return fail(FSH_EINVAL, "%s: workspace of %lld bytes, needs %lld", who, (long long)workspace_nbytes, (long long)need);
  RouteParams p;
  p.ids = expert_ids_dev;
  p.choices = choices; p.id_bytes = id_bytes; p.experts = experts;
  const int64_t blocks = ceil_div(choices, static_cast<int64_t>(kChoicesPerBlock));
  p.blocks = static_cast<int32_t>(blocks > 0 ? blocks : 1);
  p.position = position_dev; p.offsets = offsets_dev; p.source = source_dev; p.padded_offsets = padded_offsets_dev;
  p.counts = static_cast<int32_t*>(workspace_dev);
  const dim3 grid(static_cast<uint32_t>(p.blocks)), block(kThreads);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (p.blocks > 1) {
    hipLaunchKernelGGL(expert_count_kernel, grid, block, 0, on, p);
    if (int rc = check_launch("expert_count_kernel")) return rc;
  }
  hipLaunchKernelGGL(expert_place_kernel, grid, block, 0, on, p);
  return check_launch("expert_place_kernel");
}

FSH_API int fsh_expert_dispatch(const void* x_dev, const int32_t* position_dev, const int32_t* offsets_dev, int32_t experts,
                                int64_t tokens, int32_t top_k, int64_t width, int32_t dtype, void* out_dev, void* stream) {
  using namespace fsh;
  const char* who = "fsh_expert_dispatch";
  RowsParams p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const uint8_t*>(x_dev);
  p.out = static_cast<uint8_t*>(out_dev);
  p.position = position_dev; p.offsets = offsets_dev; p.experts = experts;
  bool vec = false;
  if (int rc = rows_checks(p, tokens, top_k, width, dtype, dtype, &vec, who)) return rc;
  if (tokens == 0 || width == 0) return FSH_OK;
  if (!x_dev || !offsets_dev || experts <= 0) return fail(FSH_EINVAL, "%s: null pointer, or no expert", who);
  const dim3 grid(static_cast<uint32_t>(tokens * p.slabs + kZeroBlocks)), block(kThreads);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  by_dtype(dtype, [&](auto dt) {
    if (vec) hipLaunchKernelGGL((expert_dispatch_kernel<dt.value, true>), grid, block, 0, on, p);
    else hipLaunchKernelGGL((expert_dispatch_kernel<dt.value, false>), grid, block, 0, on, p);
  });
  return check_launch("expert_dispatch_kernel");
}

namespace fsh {
namespace {

int combine(const void* rows_dev, int32_t dtype, const int32_t* position_dev, const void* weights_dev, int32_t weights_dtype, int64_t tokens,
            int32_t top_k, int64_t width, int32_t out_dtype, void* out_dev, void* stream, const char* who) {
  RowsParams p;
  memset(&p, 0, sizeof(p));
  p.rows = static_cast<const uint8_t*>(rows_dev);
  p.out = static_cast<uint8_t*>(out_dev);
  p.position = position_dev;
  p.weights = weights_dev; p.weights_dtype = weights_dtype;
  bool vec = false;
  if (int rc = rows_checks(p, tokens, top_k, width, dtype, out_dtype, &vec, who)) return rc;
  if (tokens == 0 || width == 0) return FSH_OK;
  if (!rows_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  const dim3 grid(static_cast<uint32_t>(tokens * p.slabs)), block(kThreads);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  by_dtype(out_dtype, [&](auto out) {
    const auto launch = [&](auto rows) {
      if (vec) hipLaunchKernelGGL((expert_combine_kernel<rows.value, out.value, true>), grid, block, 0, on, p);
      else hipLaunchKernelGGL((expert_combine_kernel<rows.value, out.value, false>), grid, block, 0, on, p);
    };
    if (dtype == FSH_DT_F32) launch(std::integral_constant<int, FSH_DT_F32>{});
    else launch(out);
  });
  return check_launch("expert_combine_kernel");
}

}  // namespace
}  // namespace fsh

FSH_API int fsh_expert_combine(const void* rows_dev, const int32_t* position_dev, const void* weights_dev, int32_t weights_dtype,
                               int64_t tokens, int32_t top_k, int64_t width, int32_t dtype, void* out_dev, void* stream) {
  return fsh::combine(rows_dev, dtype, position_dev, weights_dev, weights_dtype, tokens, top_k, width, dtype, out_dev, stream,
                      "fsh_expert_combine");
}

FSH_API int fsh_expert_combine_f32(const float* rows_dev, const int32_t* position_dev, const void* weights_dev, int32_t weights_dtype,
                                   int64_t tokens, int32_t top_k, int64_t width, int32_t out_dtype, void* out_dev, void* stream) {
  return fsh::combine(rows_dev, FSH_DT_F32, position_dev, weights_dev, weights_dtype, tokens, top_k, width, out_dtype, out_dev, stream,
                      "fsh_expert_combine_f32");
}

FSH_API int fsh_expert_combine_backward(const void* grad_dev, const void* rows_dev, const int32_t* position_dev,
                                        const int32_t* offsets_dev, int32_t experts, const void* weights_dev,
                                        int32_t weights_dtype, int64_t tokens, int32_t top_k, int64_t width, int32_t dtype,
                                        void* grad_rows_dev, void* grad_weights_dev, void* stream) {
  using namespace fsh;
  const char* who = "fsh_expert_combine_backward";
  RowsParams p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const uint8_t*>(grad_dev);
  p.rows = static_cast<const uint8_t*>(rows_dev);
  p.out = static_cast<uint8_t*>(grad_rows_dev);
  p.position = position_dev; p.offsets = offsets_dev; p.experts = experts;
  p.weights = weights_dev; p.weights_dtype = weights_dtype;
  p.grad_weights = grad_weights_dev;
  bool vec = false;
  if (int rc = rows_checks(p, tokens, top_k, width, dtype, dtype, &vec, who)) return rc;
  if (tokens == 0 || width == 0) return FSH_OK;
  if (!grad_dev || !rows_dev || !offsets_dev || experts <= 0 || !weights_dev || !grad_weights_dev)
    return fail(FSH_EINVAL, "%s: null pointer, or no expert", who);
  const dim3 grid(static_cast<uint32_t>(tokens + kZeroBlocks)), block(kThreads);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  by_dtype(dtype, [&](auto dt) {
    if (vec) hipLaunchKernelGGL((expert_combine_backward_kernel<dt.value, true>), grid, block, 0, on, p);
    else hipLaunchKernelGGL((expert_combine_backward_kernel<dt.value, false>), grid, block, 0, on, p);
  });
  return check_launch("expert_combine_backward_kernel");
}
