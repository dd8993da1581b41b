// One AdamW step of many tensors, with states in 32 or in 8 bits, and the sum of
// the squares of many gradients, by which they are clipped.
//
//   c = min(1, max_norm / (sqrt(S) + 1e-6))            S: the sum of squares, or c = 1
//   g = c g;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32, the parameter rounded to its type once.  S that is an infinity or not a
// number leaves parameters, states and step counts as they are.
//
// Bound by memory: everything is read once and written once, 22 bytes an element
// (bf16 parameters and gradients, 32-bit states), 10 1/8 with 8-bit states.  218 M
// parameters: 756 us, 6.3 TB/s, and fp32 with 8-bit states 550 to 595, 5.9 to 6.4; bf16 with those
// 405, 5.4, half of it instructions.  The tensors of a launch come with its arguments, so that nothing is uploaded and a
// captured launch keeps its own table; what a step's number and learning rate make of the
// hyperparameters is worked out once for each tensor, by a launch of a single workgroup ahead (4.6 us).
//
// Eight-bit states.  128 consecutive elements share a scale, their largest
// magnitude (at least 2^-100).  A value over its scale is at most 1; of its fp32 bits
// the exponent and 3 bits of the mantissa are kept, counted from those of 1.0 (1016)
// down: the first moment has a sign and codes 1 to 127, 16 octaves; the second, never
// negative, codes 1 to 255, 32 octaves, which are 16 of the gradient's.  Code 0 is
// zero.  Rounding is dithered: a number from [0, 1), which every element has anew in
// every step, is added to the bits below, and the carry decides.  To nearest, a second
// moment that changes by 1 - b2 of itself, less than half a step, would never leave its code; this
// way it moves at the right rate on average, and the bits are the same every time.  (Multiples of an irrational
// number modulo 1 do not do: the rounding's own past goes along with them, and a moment that is to fall to 0.049
// in 300 steps falls to 0.038.)  A first moment below the smallest code becomes that or zero, evenly
// too; a second one never becomes zero, for the first is divided by its root.
// What is an infinity or not a number makes the whole block not a number.
#include "rows.hpp"

#include <algorithm>
#include <memory>
#include <new>

namespace fsh {
namespace {

constexpr int kThreads = 256;
constexpr int kStateBlock = FSH_ADAMW_BLOCK;
constexpr int64_t kMaxGrid = (1LL << 32) / kThreads - 1;

// -------------------------------------------------- per-tensor factors of a step
struct alignas(16) StepFactors {
  float b1, one_b1, b2, one_b2;
  float eps, decay, step_size, root_factor;  // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  float clip;
  uint32_t t;
  int32_t skip, unused;
};

constexpr int kFactorTensors = 240;  // of one launch: 12 bytes each beside the groups
struct FactorParams {
  fsh_adamw_group groups[FSH_ADAMW_GROUPS];
  int32_t* step[kFactorTensors];
  uint8_t group[kFactorTensors];
  StepFactors* factors;
  const double* square_sum;
  double max_norm;
  int32_t count;
};
static_assert(sizeof(FactorParams) <= 4096, "kernel arguments");

// b^t by squaring, in 64 bits: 1 - b^t loses ten bits at b = 0.999 and t = 1.
__device__ double power(double b, uint32_t t) {
  double r = 1.0;
  for (; t; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}

__global__ __launch_bounds__(kThreads) void adamw_factors_kernel(const FactorParams p) {
  const int i = threadIdx.x;
  if (i >= p.count) return;
  float clip = 1.0f;
  bool skip = false;
  if (p.square_sum) {
    const double sum = *p.square_sum;
    skip = !(fabs(sum) <= 1.7976931348623157e308);
    if (p.max_norm > 0.0) {
      const double factor = p.max_norm / (sqrt(sum) + 1e-6);
      clip = static_cast<float>(factor < 1.0 ? factor : 1.0);
    }
  }
  const fsh_adamw_group g = p.groups[p.group[i]];
  const double lr = g.lr_dev ? static_cast<double>(*g.lr_dev) : g.lr;
  const uint32_t t = static_cast<uint32_t>(*p.step[i]) + (skip ? 0u : 1u);
  if (!skip) *p.step[i] = static_cast<int32_t>(t);
  StepFactors f;
  f.b1 = static_cast<float>(g.beta1);
  f.one_b1 = static_cast<float>(1.0 - g.beta1);
  f.b2 = static_cast<float>(g.beta2);
  f.one_b2 = static_cast<float>(1.0 - g.beta2);
  f.eps = static_cast<float>(g.eps);
  f.decay = static_cast<float>(1.0 - lr * g.weight_decay);
  f.step_size = static_cast<float>(lr / (1.0 - power(g.beta1, t)));
  f.root_factor = static_cast<float>(1.0 / sqrt(1.0 - power(g.beta2, t)));
  f.clip = clip;
  f.t = t;
  f.skip = skip;
  f.unused = 0;
  p.factors[i] = f;
}

// ------------------------------------------------------------- the tensors' table
// Tensors of one launch, cut into chunks that are numbered through.
constexpr int kTensors = 60;
struct AdamTable {
  void* param[kTensors];
  const void* grad[kTensors];
  void* m[kTensors];
  void* v[kTensors];
  float* m_scale[kTensors];
  float* v_scale[kTensors];
  int64_t numel[kTensors];
  uint32_t factors[kTensors];
  uint32_t first_chunk[kTensors];  // 0xFFFFFFFF behind the last
  const StepFactors* all_factors;
  int64_t chunks;
};
static_assert(sizeof(AdamTable) <= 4096, "kernel arguments");

// The tensor that a chunk belongs to: the last that begins at or before it (a lane each).
template <int N>
__device__ __forceinline__ int tensor_of(const uint32_t (&first)[N], uint32_t chunk) {
  const int lane = threadIdx.x & 63;
  int at = -1;
#pragma unroll
  for (int base = 0; base < N; base += 64)
    at += __popcll(__ballot(base + lane < N && first[base + lane < N ? base + lane : 0] <= chunk));
  return __builtin_amdgcn_readfirstlane(at);
}

// ------------------------------------------------------------------ 8-bit codes
constexpr uint32_t kFirstBase = 1016 - 127, kSecondBase = 1016 - 255;  // 1016: the upper 12 bits of 1.0f
__device__ __forceinline__ float first_value(uint32_t code) {
  const uint32_t size = code & 127u;
  return u32_as_f32((size ? (size + kFirstBase) << 20 : 0u) | ((code & 128u) << 24));
}
__device__ __forceinline__ float second_value(uint32_t code) { return u32_as_f32(code ? (code + kSecondBase) << 20 : 0u); }
// The codes of a value over its block's scale, of at most 1 and a few units in the last
// place, which the dither cannot carry further (of a block that is not a number: any bits).
// half: the dither in units of 2^-16.  kSmall: the value may be below the smallest code.
constexpr float kFirstSmallest = 1.25f / 65536.0f, kSecondSmallest = kFirstSmallest / 65536.0f;
template <bool kSmall>
__device__ __forceinline__ uint32_t first_code(float value, uint32_t half) {
  const uint32_t bits = f32_as_u32(value) & 0x7FFFFFFFu, sign = (f32_as_u32(value) >> 24) & 128u;
  const uint32_t up = ((bits + (half << 4)) >> 20) - kFirstBase;
  if constexpr (!kSmall) return up | sign;
  const float size = u32_as_f32(bits);
  // (the product with 1 / kFirstSmallest, rounded as such, against half / 65536)
  const uint32_t few = size * (1.0f / kFirstSmallest * 65536.0f) > static_cast<float>(half) ? 1u : 0u;
  return (size < kFirstSmallest ? few : up) | sign;
}
template <bool kSmall>
__device__ __forceinline__ uint32_t second_code(float size, uint32_t half) {
  const int up = static_cast<int>((f32_as_u32(size) + (half << 4)) >> 20) - static_cast<int>(kSecondBase);
  if constexpr (!kSmall) return static_cast<uint32_t>(up);
  const int least = static_cast<int>(min(f32_as_u32(size), 1u));  // 1 of what is not zero
  return static_cast<uint32_t>(max(up, least));
}
// The dither of an element in a step, 16 bits for each moment (the first's below):
// multiples of the golden ratio and of the square root of 2, modulo 2^32, mixed by one
// product with the square root of 3 between two shifts, which leaves no correlation beyond
// chance between neighbours, steps or the halves (2^20 elements).
constexpr uint32_t kOverElements = 0x9E3779B9u, kOverSteps = 0x6A09E667u;
__device__ __forceinline__ uint32_t dither(uint32_t multiple) {
  const uint32_t z = (multiple ^ (multiple >> 16)) * 0xBB67AE85u;
  return z ^ (z >> 15);
}

template <bool kSmall, int VEC>
__device__ __forceinline__ void codes_of(const float (&m)[VEC], const float (&v)[VEC], uint32_t multiple, uint32_t (&mc)[VEC / 4], uint32_t (&vc)[VEC / 4]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const uint32_t u = dither(multiple + static_cast<uint32_t>(j) * kOverElements);
    const uint32_t first = first_code<kSmall>(m[j], u & 0xFFFFu) << (8 * (j % 4)), second = second_code<kSmall>(v[j], u >> 16) << (8 * (j % 4));
    mc[j / 4] = j % 4 ? mc[j / 4] | first : first;
    vc[j / 4] = j % 4 ? vc[j / 4] | second : second;
  }
}

// The scale of a block from its largest magnitude's bits, and 1 over it.
__device__ __forceinline__ float block_scale(uint32_t largest, float& inverse) {
  const float least = u32_as_f32(0x0D800000u);  // 2^-100
  const float amax = u32_as_f32(largest >= 0x7F800000u ? 0x7FC00000u : largest);
  const float scale = amax < least ? least : amax;  // (not a number stays)
  inverse = 1.0f / scale;
  return scale;
}

// --------------------------------------------------------------------- the step
// A workgroup takes a chunk: vectors of four neighbours a thread, the loads of all
// of them requested first.  With 32-bit states one vector, with 8-bit ones, where instructions
// count and what is done once per chunk is spread, 16 elements (218 M parameters, us: bf16 and 32
// bits with 4, 8 and 16 elements 768, 855, 820; 8 bits with 8, 16 and 32 bf16 420, 405, 420, fp32 590, 595, 615).
// Everything streams: through the caches the 32-bit step takes 919 us, and workgroups that stay for more chunks than
// one are slower still (2048 of them: 1049).
constexpr int chunk_of(bool eight) { return (eight ? 4 : 1) * 4 * kThreads; }

// Neighbours in a vector: eight of bf16 parameters with 8-bit states, which makes a block a
// row of 16 lanes and halves what is done once a block (405 us; with four 428).  Of fp32 parameters, where
// eight are two loads of lanes apart, four (595 us; with eight 720).
constexpr int vector_of(int param_dtype, bool eight) { return eight && param_dtype == FSH_DT_BF16 ? 8 : 4; }

// What a vector's step reads.
template <int PT, int GT, bool kEight, int VEC>
struct StepInput {
  RawVec<PT, VEC> p;
  RawVec<GT, VEC> g;
  RawVec<FSH_DT_F32, VEC> m, v;
  uint32_t mc[VEC / 4], vc[VEC / 4];
  float ms, vs;
};

// Where a chunk's part of a tensor lies.
struct ChunkOf {
  uint8_t* param;
  const uint8_t* grad;
  uint8_t* m;
  uint8_t* v;
  float* m_scale;
  float* v_scale;
};

// Up to VEC codes, the others zero.
template <bool kFull, int WORDS>
__device__ __forceinline__ void load_codes(const uint8_t* src, int count, uint32_t (&c)[WORDS]) {
  if (kFull || count >= 4 * WORDS) {
    __builtin_memcpy(c, src, sizeof(c));
  } else {
#pragma unroll
    for (int j = 0; j < 4 * WORDS; ++j) {
      const uint32_t code = j < count ? src[j] : 0u;
      c[j / 4] = j % 4 ? c[j / 4] | code << (8 * (j % 4)) : code;
    }
  }
}
template <bool kFull, int WORDS>
__device__ __forceinline__ void store_codes(uint8_t* dst, int count, const uint32_t (&c)[WORDS]) {
  if (kFull || count >= 4 * WORDS) {
    __builtin_memcpy(dst, c, sizeof(c));
  } else {
#pragma unroll
    for (int j = 0; j < 4 * WORDS; ++j)
      if (j < count) dst[j] = static_cast<uint8_t>(c[j / 4] >> (8 * (j % 4)));
  }
}

// kFull: the chunk ends inside the tensor; `left`: elements from the chunk's first on.
template <int PT, int GT, bool kEight, bool kFull>
__device__ __forceinline__ void step_chunk(const ChunkOf& c, const StepFactors& f, uint32_t first_index, int left) {
  constexpr int VEC = vector_of(PT, kEight), kVectors = chunk_of(kEight) / (VEC * kThreads);
  StepInput<PT, GT, kEight, VEC> in[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int at = (i * kThreads + static_cast<int>(threadIdx.x)) * VEC;
    const int count = kFull ? VEC : left - at;
    in[i].p = load_vec<PT, VEC, true>(c.param, at, count);
    in[i].g = load_vec<GT, VEC, true>(c.grad, at, count);
    if constexpr (kEight) {
      load_codes<kFull>(c.m + at, count, in[i].mc);
      load_codes<kFull>(c.v + at, count, in[i].vc);
      in[i].ms = count > 0 ? c.m_scale[at / kStateBlock] : 0.0f;
      in[i].vs = count > 0 ? c.v_scale[at / kStateBlock] : 0.0f;
    } else {
      in[i].m = load_vec<FSH_DT_F32, VEC, true>(c.m, at, count);
      in[i].v = load_vec<FSH_DT_F32, VEC, true>(c.v, at, count);
    }
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int at = (i * kThreads + static_cast<int>(threadIdx.x)) * VEC;
    const int count = kFull ? VEC : left - at;
    float m[VEC], v[VEC], p[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if constexpr (kEight) {
        m[j] = first_value((in[i].mc[j / 4] >> (8 * (j % 4))) & 255u) * in[i].ms;
        v[j] = second_value((in[i].vc[j / 4] >> (8 * (j % 4))) & 255u) * in[i].vs;
      } else {
        m[j] = element<FSH_DT_F32, VEC>(in[i].m, j);
        v[j] = element<FSH_DT_F32, VEC>(in[i].v, j);
      }
      const float g = element<GT, VEC>(in[i].g, j) * f.clip;
      m[j] = m[j] * f.b1 + g * f.one_b1;
      v[j] = v[j] * f.b2 + (g * g) * f.one_b2;
      float update;
      if constexpr (kEight) {
        // (root and quotient to one unit in the last place: this form is bound by instructions
        // otherwise.  A v below 2^-126 may count as zero.)
        update = m[j] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[j]) * f.root_factor + f.eps);
      } else {
        update = m[j] / (sqrtf(v[j]) * f.root_factor + f.eps);
      }
      p[j] = element<PT, VEC>(in[i].p, j) * f.decay - f.step_size * update;
    }
    if (kFull || count > 0) store_vec<PT, VEC, true>(c.param, at, count, to_vec<PT, VEC>(p));
    if constexpr (kEight) {
      // A block is half a wave's, or a row's of 16 lanes; elements behind the tensor's last are zero.
      uint32_t m_max = 0, v_max = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (!kFull && j >= count) m[j] = v[j] = 0.0f;
        m_max = max(m_max, f32_as_u32(m[j]) & 0x7FFFFFFFu);
        v_max = max(v_max, f32_as_u32(v[j]) & 0x7FFFFFFFu);
      }
      // Both moments' maxima over each row of 16 lanes.  One division does for both: the
      // first's in even rows and the second's in odd ones, which a swap of the first's odd rows with
      // the second's even ones gives (and joins the two rows of a block); with a block in a
      // row, in even and odd lanes.
      m_max = row16_max_u32(m_max);
      v_max = row16_max_u32(v_max);
      float inverse, m_inverse, v_inverse, scale;
      if constexpr (VEC == 4) {
        const auto pair = __builtin_amdgcn_permlane16_swap(m_max, v_max, false, false);
        scale = block_scale(max(pair[0], pair[1]), inverse);
        const auto inverses = __builtin_amdgcn_permlane16_swap(f32_as_u32(inverse), f32_as_u32(inverse), false, false);
        m_inverse = u32_as_f32(inverses[0]);
        v_inverse = u32_as_f32(inverses[1]);
      } else {
        scale = block_scale(threadIdx.x & 1 ? v_max : m_max, inverse);
        const int both = static_cast<int>(f32_as_u32(inverse));
        m_inverse = u32_as_f32(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, both, 0xA0, 0xF, 0xF, true)));  // quad_perm [0,0,2,2]
        v_inverse = u32_as_f32(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, both, 0xF5, 0xF, 0xF, true)));  // quad_perm [1,1,3,3]
      }
      float m_least = 1.0f, v_least = 1.0f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        m[j] *= m_inverse;
        v[j] *= v_inverse;
        m_least = fminf(m_least, fabsf(m[j]));
        v_least = fminf(v_least, v[j]);
      }
      const uint32_t multiple = (first_index + static_cast<uint32_t>(at)) * kOverElements + f.t * kOverSteps;
      uint32_t mc[VEC / 4], vc[VEC / 4];
      // (a wave rarely has a value below the smallest code; with this and the one division, in
      // vectors of four, bf16 parameters took 430 us for 485)
      if (__ballot(m_least < kFirstSmallest || v_least < kSecondSmallest)) codes_of<true>(m, v, multiple, mc, vc);
      else codes_of<false>(m, v, multiple, mc, vc);
      store_codes<kFull>(c.m + at, count, mc);
      store_codes<kFull>(c.v + at, count, vc);
      // (a block's first lane has its first moment's scale, the sixteenth behind it, or the next, the second's)
      constexpr int kSecond = VEC == 4 ? 16 : 1;
      if ((threadIdx.x & (kStateBlock / VEC - 1) & ~kSecond) == 0) {
        const int of = at - (threadIdx.x & kSecond) * VEC;  // the block's first element
        if (kFull || left > of) (threadIdx.x & kSecond ? c.v_scale : c.m_scale)[of / kStateBlock] = scale;
      }
    } else if (kFull || count > 0) {
      store_vec<FSH_DT_F32, VEC, true>(c.m, at, count, to_vec<FSH_DT_F32, VEC>(m));
      store_vec<FSH_DT_F32, VEC, true>(c.v, at, count, to_vec<FSH_DT_F32, VEC>(v));
    }
  }
}

template <int PT, int GT, bool kEight>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const AdamTable a) {
  constexpr int kChunk = chunk_of(kEight);
  for (int64_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    const int k = tensor_of(a.first_chunk, static_cast<uint32_t>(chunk));
    const StepFactors f = a.all_factors[a.factors[k]];
    if (f.skip) continue;
    const int64_t at = (chunk - a.first_chunk[k]) * kChunk, left = a.numel[k] - at;
    constexpr int kStateBytes = kEight ? 1 : 4;
    const ChunkOf c = {static_cast<uint8_t*>(a.param[k]) + at * bytes_of(PT), static_cast<const uint8_t*>(a.grad[k]) + at * bytes_of(GT),
                       static_cast<uint8_t*>(a.m[k]) + at * kStateBytes, static_cast<uint8_t*>(a.v[k]) + at * kStateBytes,
                       a.m_scale[k] + at / kStateBlock, a.v_scale[k] + at / kStateBlock};
    if (left >= kChunk) step_chunk<PT, GT, kEight, true>(c, f, static_cast<uint32_t>(at), kChunk);
    else step_chunk<PT, GT, kEight, false>(c, f, static_cast<uint32_t>(at), static_cast<int>(left));
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void adamw_values_kernel(const uint8_t* m, const float* m_scale, const uint8_t* v, const float* v_scale,
                                                                void* m_out, void* v_out, int64_t numel) {
  for (int64_t at = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 8; at < numel; at += static_cast<int64_t>(gridDim.x) * kThreads * 8) {
    const int64_t count = numel - at;
    uint8_t mc[8] = {}, vc[8] = {};
    if (count >= 8) {
      __builtin_memcpy(mc, m + at, 8);
      __builtin_memcpy(vc, v + at, 8);
    } else {
      for (int j = 0; j < count; ++j) {
        mc[j] = m[at + j];
        vc[j] = v[at + j];
      }
    }
    const float ms = m_scale[at / kStateBlock], vs = v_scale[at / kStateBlock];
    float mf[8], vf[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mf[j] = first_value(mc[j]) * ms;
      vf[j] = second_value(vc[j]) * vs;
    }
    store_vec<DT, 8, true>(m_out, at, count, to_vec<DT, 8>(mf));
    store_vec<DT, 8, true>(v_out, at, count, to_vec<DT, 8>(vf));
  }
}

// --------------------------------------------------------------- sum of squares
// In 64 bits, where the squares of bf16, fp16 and fp32 values are exact or nearly: a
// workgroup adds up its chunks, its threads' sums are joined in a fixed order, and
// one workgroup joins the workgroups'.  Bound by memory.  Gradients that the last-level cache
// cannot hold for the step behind (256 MB) are read past the caches: 218 M, us without and with, bf16 77 and
// 70, fp32 152 and 130; of 55 M the step then takes 10 more.  Fewer workgroups leave the memory idle
// between their chunks (2048: 83 and 178).
constexpr int kSquareTensors = 160;
constexpr int kSquareChunk = 8 * kThreads * 4;  // elements: four vectors of eight a thread
constexpr int kSquareGroups = 4096;
constexpr int64_t kSquareStream = 256LL << 20;  // bytes
struct SquareTable {
  const void* grad[kSquareTensors];
  int64_t numel[kSquareTensors];
  uint32_t first_chunk[kSquareTensors];
  uint8_t dtype[kSquareTensors];
  double* parts;
  int64_t chunks;
};
static_assert(sizeof(SquareTable) <= 4096, "kernel arguments");

// A thread's vectors of elements [at, at + kSquareChunk), `thread` of kThreads, and
// the sum of their squares.
template <int DT>
struct SquareVectors {
  static constexpr int VEC = DT == FSH_DT_F32 ? 4 : 8, N = kSquareChunk / kThreads / VEC;
  RawVec<DT, VEC> r[N];
  template <bool kStream>
  __device__ __forceinline__ void load(const void* g, int64_t at, int64_t numel, int thread) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t here = at + (static_cast<int64_t>(i) * kThreads + thread) * VEC;
      r[i] = load_vec<DT, VEC, kStream>(g, here, numel - here);
    }
  }
  __device__ __forceinline__ double sum() const {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const double x = static_cast<double>(element<DT, VEC>(r[i], j));
        sum = __builtin_fma(x, x, sum);
      }
    return sum;
  }
};
template <int DT, bool kStream>
__device__ __forceinline__ double squares_of(const SquareTable& a, int k, int64_t at) {
  SquareVectors<DT> v;
  v.template load<kStream>(a.grad[k], at, a.numel[k], threadIdx.x);
  return v.sum();
}

template <int THREADS>
__device__ __forceinline__ double workgroup_sum(double v, double* lds) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, kWave);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) sum += lds[w];
  return sum;
}

template <bool kStream>
__global__ __launch_bounds__(kThreads) void square_sum_kernel(const SquareTable a) {
  __shared__ double lds[kThreads / 64];
  double sum = 0.0;
  for (int64_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    const int k = tensor_of(a.first_chunk, static_cast<uint32_t>(chunk));
    const int64_t at = (chunk - a.first_chunk[k]) * kSquareChunk;
    const int dtype = a.dtype[k];
    if (dtype == FSH_DT_F32) sum += squares_of<FSH_DT_F32, kStream>(a, k, at);
    else if (dtype == FSH_DT_BF16) sum += squares_of<FSH_DT_BF16, kStream>(a, k, at);
    else sum += squares_of<FSH_DT_F16, kStream>(a, k, at);
  }
  sum = workgroup_sum<kThreads>(sum, lds);
  if (threadIdx.x == 0) a.parts[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kThreads) void square_join_kernel(const double* parts, int64_t count, double* out) {
  __shared__ double lds[kThreads / 64];
  double sum = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < count; i += kThreads) sum += parts[i];
  sum = workgroup_sum<kThreads>(sum, lds);
  if (threadIdx.x == 0) *out = sum;
}

// A few chunks of one type in one workgroup, two at a time for each quarter of it,
// which writes the sum itself: norm weights and biases, where a second launch would be the
// longer part.  Bound by latency and by what one compute unit reads; the table is fetched once, into
// LDS.  20 vectors of 4096 fp32: 10.4 us; as two launches 7.6, but 20 of the host's instead of 16.  (A
// replayed graph of the call on 262144 elements, 32 whole chunks: 21 us this way, 12.5 as two.)
constexpr int kFewChunks = 32, kFewThreads = 1024;
constexpr int64_t kFewElements = 16 * kSquareChunk;
template <int DT>
__global__ __launch_bounds__(kFewThreads) void square_sum_few_kernel(const SquareTable a) {
  __shared__ double lds[kFewThreads / 64];
  __shared__ const void* grad[kSquareTensors];
  __shared__ int64_t numel[kSquareTensors];
  __shared__ uint32_t first_chunk[kSquareTensors];
  constexpr int kParts = kFewThreads / kThreads;
  if (threadIdx.x < kSquareTensors) {
    grad[threadIdx.x] = a.grad[threadIdx.x];
    numel[threadIdx.x] = a.numel[threadIdx.x];
    first_chunk[threadIdx.x] = a.first_chunk[threadIdx.x];
  }
  __syncthreads();
  const int part = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kThreads), thread = threadIdx.x % kThreads;
  const int chunks = static_cast<int>(a.chunks);
  double sum = 0.0;
  for (int chunk = part; chunk < chunks; chunk += 2 * kParts) {
    SquareVectors<DT> v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int mine = min(chunk + i * kParts, chunks - 1);
      const int k = tensor_of(first_chunk, static_cast<uint32_t>(mine));
      const int64_t at = static_cast<int64_t>(mine - static_cast<int>(first_chunk[k])) * kSquareChunk;
      v[i].template load<false>(grad[k], at, chunk + i * kParts < chunks ? numel[k] : 0, thread);
    }
    sum += v[0].sum() + v[1].sum();
  }
  sum = workgroup_sum<kFewThreads>(sum, lds);
  if (threadIdx.x == 0) a.parts[0] = sum;
}

// Chunks of one launch are numbered in 32 bits.
constexpr int64_t kMaxChunks = 0xFFFFFFFELL;

// Workgroups of each of the launches that the tensors take; their number.  One of a
// single workgroup where one can do it all.
template <typename Each>
int square_launches(const int64_t* tensors, int32_t count, Each each) {
  int32_t begin = 0;
  int launches = 0;
  while (begin < count) {
    int64_t chunks = 0;
    int32_t end = begin;
    while (end < count && end - begin < kSquareTensors) {
      const int64_t more = ceil_div(tensors[3 * end + 1], (int64_t)kSquareChunk);
      if (chunks + more > kMaxChunks) break;
      chunks += more;
      ++end;
    }
    if (end == begin) return -1;  // a tensor of more than 2^44 elements
    bool few = begin == 0 && end == count && chunks <= kFewChunks;
    int64_t elements = 0;
    for (int32_t i = 0; few && i < count; ++i) {
      elements += tensors[3 * i + 1];
      few = tensors[3 * i + 2] == tensors[2] && elements <= kFewElements;  // (of one type)
    }
    if (chunks) each(begin, end, chunks, few ? 0 : chunks < kSquareGroups ? chunks : static_cast<int64_t>(kSquareGroups));
    ++launches;
    begin = end;
  }
  return launches;
}

// Whether a step writes memory that it also reads or writes elsewhere (a parameter that is listed
// twice, say): parameters, states, scales, step counts and the workspace, each once, and no gradient
// over them, but for one that is its own parameter, which every thread reads before it writes there. -1 without
// memory for the list.
int tensors_overlap(const fsh_adamw_tensor* tensors, int32_t count, const void* workspace) {
  struct Span {
    uintptr_t begin, end;
    bool written;
  };
  std::unique_ptr<Span[]> spans(new (std::nothrow) Span[7 * static_cast<size_t>(count) + 1]);
  if (!spans) return -1;
  size_t n = 0;
  const auto add = [&](const void* base, int64_t nbytes, bool written) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(base);
    if (base) spans[n++] = {begin, begin + static_cast<uintptr_t>(nbytes), written};
  };
  add(workspace, fsh_adamw_step_workspace_bytes(count), true);
  for (int32_t i = 0; i < count; ++i) {
    const fsh_adamw_tensor& t = tensors[i];
    add(t.step_dev, sizeof(int32_t), true);
    if (t.numel == 0) continue;
    const int64_t state = t.state_bits == 8 ? 1 : 4;
    add(t.param_dev, t.numel * bytes_of(static_cast<int>(t.param_dtype)), true);
    if (t.grad_dev != t.param_dev || t.grad_dtype != t.param_dtype) add(t.grad_dev, t.numel * bytes_of(static_cast<int>(t.grad_dtype)), false);
    add(t.exp_avg_dev, t.numel * state, true);
    add(t.exp_avg_sq_dev, t.numel * state, true);
    if (t.state_bits != 8) continue;
    add(t.exp_avg_scale_dev, 4 * ceil_div(t.numel, (int64_t)kStateBlock), true);
    add(t.exp_avg_sq_scale_dev, 4 * ceil_div(t.numel, (int64_t)kStateBlock), true);
  }
  std::sort(spans.get(), spans.get() + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t written = 0, touched = 0;  // ends of those before
  for (size_t i = 0; i < n; ++i) {
    const Span& s = spans[i];
    if (s.begin < (s.written ? touched : written)) return 1;
    touched = std::max(touched, s.end);
    if (s.written) written = std::max(written, s.end);
  }
  return 0;
}

// What a step refuses of its tensors and groups.
int check_step(const fsh_adamw_tensor* tensors, int32_t count, const fsh_adamw_group* groups, int32_t group_count, const void* workspace, const char* who) {
  for (int32_t i = 0; i < group_count; ++i) {
    const fsh_adamw_group& g = groups[i];
    if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0)) return fail(FSH_EINVAL, "%s: group %d: betas in [0, 1), eps not negative", who, i);
    if (!aligned(g.lr_dev, 4)) return fail(FSH_ENOTSUP, "%s: group %d: the learning rate must be 4-byte aligned", who, i);
  }
  for (int32_t i = 0; i < count; ++i) {
    const fsh_adamw_tensor& t = tensors[i];
    if (t.numel < 0 || t.group < 0 || t.group >= group_count) return fail(FSH_EINVAL, "%s: tensor %d: negative size, or group %lld of %d", who, i, (long long)t.group, group_count);
    if ((t.param_dtype != FSH_DT_BF16 && t.param_dtype != FSH_DT_F32) || (t.grad_dtype != FSH_DT_BF16 && t.grad_dtype != FSH_DT_F32) || (t.state_bits != 8 && t.state_bits != 32))
      return fail(FSH_EINVAL, "%s: tensor %d: bf16 or fp32 parameters and gradients, states of 8 or 32 bits", who, i);
    if (!t.step_dev || (t.numel && (!t.param_dev || !t.grad_dev || !t.exp_avg_dev || !t.exp_avg_sq_dev || (t.state_bits == 8 && (!t.exp_avg_scale_dev || !t.exp_avg_sq_scale_dev)))))
      return fail(FSH_EINVAL, "%s: tensor %d: null pointer", who, i);
    if (!aligned(t.param_dev, bytes_of(t.param_dtype)) || !aligned(t.grad_dev, bytes_of(t.grad_dtype)) || !aligned(t.exp_avg_dev, t.state_bits == 8 ? 1 : 4) ||
        !aligned(t.exp_avg_sq_dev, t.state_bits == 8 ? 1 : 4) || !aligned(t.exp_avg_scale_dev, 4) || !aligned(t.exp_avg_sq_scale_dev, 4) || !aligned(t.step_dev, 4))
      return fail(FSH_ENOTSUP, "%s: tensor %d is not aligned to its elements", who, i);
    if (ceil_div(t.numel, (int64_t)chunk_of(t.state_bits == 8)) > kMaxChunks) return fail(FSH_ENOTSUP, "%s: tensor %d is too long", who, i);
  }
  if (const int overlap = tensors_overlap(tensors, count, workspace))
    return overlap < 0 ? fail(FSH_ENOTSUP, "%s: no host memory for %d tensors", who, count)
                       : fail(FSH_EINVAL, "%s: parameters, gradients, states, step counts or the workspace overlap", who);
  return FSH_OK;
}

template <int PT, int GT>
void launch_step(const AdamTable& a, bool eight, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(a.chunks < kMaxGrid ? a.chunks : kMaxGrid)), block(kThreads);
  if (eight) hipLaunchKernelGGL((adamw_kernel<PT, GT, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((adamw_kernel<PT, GT, false>), grid, block, 0, stream, a);
}

}  // namespace
}  // namespace fsh

FSH_API int64_t fsh_grad_square_sum_workspace_bytes(const int64_t* tensors, int32_t count) {
  using namespace fsh;
  if (!tensors || count < 0) return 0;
  int64_t groups = 0;
  square_launches(tensors, count, [&](int32_t, int32_t, int64_t, int64_t mine) { groups += mine; });
  return groups * static_cast<int64_t>(sizeof(double));
}

FSH_API int fsh_grad_square_sum(const int64_t* tensors, int32_t count, double* out_dev, void* workspace_dev, int64_t workspace_nbytes, void* stream) {
  using namespace fsh;
  const char* who = "fsh_grad_square_sum";
  if (count < 0) return fail(FSH_EINVAL, "%s: negative count", who);
  if (!out_dev || (count && !tensors)) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (!aligned(out_dev, 8) || !aligned(workspace_dev, 8)) return fail(FSH_ENOTSUP, "%s: the sum and the workspace must be 8-byte aligned", who);
  for (int32_t i = 0; i < count; ++i) {
    const int64_t address = tensors[3 * i], numel = tensors[3 * i + 1], dtype = tensors[3 * i + 2];
    if (numel < 0) return fail(FSH_EINVAL, "%s: tensor %d has a negative size", who, i);
    if (dtype < 0 || !is_dtype(static_cast<int32_t>(dtype < 99 ? dtype : 99))) return fail(FSH_EINVAL, "%s: tensor %d has an unknown dtype %lld", who, i, (long long)dtype);
    if (numel && !address) return fail(FSH_EINVAL, "%s: null pointer", who);
    if (address % bytes_of(static_cast<int>(dtype))) return fail(FSH_ENOTSUP, "%s: tensor %d is not aligned to its elements", who, i);
  }
  const int64_t need = fsh_grad_square_sum_workspace_bytes(tensors, count);
  if (need && (!workspace_dev || workspace_nbytes < need)) return fail(FSH_EINVAL, "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_nbytes, (long long)need);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  double* const parts = static_cast<double*>(workspace_dev);
  int64_t used = 0, nbytes = 0;
  for (int32_t i = 0; i < count; ++i) nbytes += tensors[3 * i + 1] * bytes_of(static_cast<int>(tensors[3 * i + 2]));
  bool done = false;
  int rc = FSH_OK;
  const int launches = square_launches(tensors, count, [&](int32_t begin, int32_t end, int64_t chunks, int64_t groups) {
    SquareTable a;
    uint32_t first = 0;
    for (int k = 0; k < kSquareTensors; ++k) {
      const bool here = begin + k < end;
      const int64_t* t = tensors + 3 * (here ? begin + k : begin);
      a.grad[k] = reinterpret_cast<const void*>(t[0]);
      a.numel[k] = t[1];
      a.dtype[k] = static_cast<uint8_t>(t[2]);
      a.first_chunk[k] = here ? first : 0xFFFFFFFFu;
      if (here) first += static_cast<uint32_t>(ceil_div(t[1], (int64_t)kSquareChunk));
    }
    a.parts = groups ? parts + used : out_dev;
    a.chunks = chunks;
    done = groups == 0;
    if (rc == FSH_OK) {
      if (done && a.dtype[0] == FSH_DT_F32) hipLaunchKernelGGL(square_sum_few_kernel<FSH_DT_F32>, dim3(1), dim3(kFewThreads), 0, on, a);
      else if (done && a.dtype[0] == FSH_DT_BF16) hipLaunchKernelGGL(square_sum_few_kernel<FSH_DT_BF16>, dim3(1), dim3(kFewThreads), 0, on, a);
      else if (done) hipLaunchKernelGGL(square_sum_few_kernel<FSH_DT_F16>, dim3(1), dim3(kFewThreads), 0, on, a);
      else if (nbytes > kSquareStream) hipLaunchKernelGGL(square_sum_kernel<true>, dim3(static_cast<uint32_t>(groups)), dim3(kThreads), 0, on, a);
      else hipLaunchKernelGGL(square_sum_kernel<false>, dim3(static_cast<uint32_t>(groups)), dim3(kThreads), 0, on, a);
      rc = check_launch("square_sum_kernel");
    }
    used += groups;
  });
  if (launches < 0) return fail(FSH_ENOTSUP, "%s: a tensor is too long", who);
  if (rc || done) return rc;
  hipLaunchKernelGGL(square_join_kernel, dim3(1), dim3(kThreads), 0, on, parts, used, out_dev);
  return check_launch("square_join_kernel");
}

FSH_API int64_t fsh_adamw_step_workspace_bytes(int32_t count) {
  return count < 0 ? 0 : static_cast<int64_t>(count) * static_cast<int64_t>(sizeof(fsh::StepFactors));
}

FSH_API int fsh_adamw_check(const fsh_adamw_tensor* tensors, int32_t count, const fsh_adamw_group* groups, int32_t group_count) {
  using namespace fsh;
  const char* who = "fsh_adamw_check";
  if (count < 0 || group_count < 0) return fail(FSH_EINVAL, "%s: negative count", who);
  if (count == 0) return FSH_OK;
  if (!tensors || !groups) return fail(FSH_EINVAL, "%s: null pointer", who);
  return check_step(tensors, count, groups, group_count, nullptr, who);
}

FSH_API int fsh_adamw_step(const fsh_adamw_tensor* tensors, int32_t count, const fsh_adamw_group* groups, int32_t group_count, const double* square_sum_dev,
                           double max_norm, void* workspace_dev, int64_t workspace_nbytes, void* stream) {
  using namespace fsh;
  const char* who = "fsh_adamw_step";
  if (count < 0) return fail(FSH_EINVAL, "%s: negative count", who);
  if (count == 0) return FSH_OK;
  if (!tensors || !groups || !workspace_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (group_count < 1 || group_count > FSH_ADAMW_GROUPS) return fail(FSH_ENOTSUP, "%s: 1 to %d groups, got %d", who, FSH_ADAMW_GROUPS, group_count);
  if (workspace_nbytes < fsh_adamw_step_workspace_bytes(count) || !aligned(workspace_dev, 16))
    return fail(FSH_EINVAL, "%s: workspace of %lld bytes, %lld needed, 16-byte aligned", who, (long long)workspace_nbytes, (long long)fsh_adamw_step_workspace_bytes(count));
  if (!aligned(square_sum_dev, 8)) return fail(FSH_ENOTSUP, "%s: the sum of squares must be 8-byte aligned", who);
  if (max_norm != max_norm) return fail(FSH_EINVAL, "%s: max_norm is not a number", who);
  if (int rc = check_step(tensors, count, groups, group_count, workspace_dev, who)) return rc;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  StepFactors* const factors = static_cast<StepFactors*>(workspace_dev);
  for (int32_t begin = 0; begin < count; begin += kFactorTensors) {
    FactorParams p = {};
    for (int32_t i = 0; i < group_count; ++i) p.groups[i] = groups[i];
    p.count = count - begin < kFactorTensors ? count - begin : kFactorTensors;
    for (int32_t i = 0; i < p.count; ++i) {
      p.step[i] = tensors[begin + i].step_dev;
      p.group[i] = static_cast<uint8_t>(tensors[begin + i].group);
    }
    p.factors = factors + begin;
    p.square_sum = square_sum_dev;
    p.max_norm = max_norm;
    hipLaunchKernelGGL(adamw_factors_kernel, dim3(1), dim3(kThreads), 0, on, p);
    if (int rc = check_launch("adamw_factors_kernel")) return rc;
  }
  // Tensors of the same types share launches.
  for (int kind = 0; kind < 8; ++kind) {
    const int pt = kind & 1 ? FSH_DT_F32 : FSH_DT_BF16, gt = kind & 2 ? FSH_DT_F32 : FSH_DT_BF16;
    const bool eight = (kind & 4) != 0;
    for (int32_t next = 0; next < count;) {
      AdamTable a;
      int32_t n = 0;
      a.chunks = 0;
      for (; next < count && n < kTensors; ++next) {
        const fsh_adamw_tensor& t = tensors[next];
        if (t.param_dtype != pt || t.grad_dtype != gt || (t.state_bits == 8) != eight || t.numel == 0) continue;
        const int64_t more = ceil_div(t.numel, (int64_t)chunk_of(eight));
        if (a.chunks + more > kMaxChunks) break;
        a.param[n] = t.param_dev;
        a.grad[n] = t.grad_dev;
        a.m[n] = t.exp_avg_dev;
        a.v[n] = t.exp_avg_sq_dev;
        a.m_scale[n] = t.exp_avg_scale_dev;
        a.v_scale[n] = t.exp_avg_sq_scale_dev;
        a.numel[n] = t.numel;
        a.factors[n] = static_cast<uint32_t>(next);
        a.first_chunk[n] = static_cast<uint32_t>(a.chunks);
        a.chunks += more;
        ++n;
      }
      if (n == 0) break;  // (no more of this kind)
      for (int32_t i = n; i < kTensors; ++i) a.first_chunk[i] = 0xFFFFFFFFu;
      a.all_factors = factors;
      if (pt == FSH_DT_BF16 && gt == FSH_DT_BF16) launch_step<FSH_DT_BF16, FSH_DT_BF16>(a, eight, on);
      else if (pt == FSH_DT_BF16) launch_step<FSH_DT_BF16, FSH_DT_F32>(a, eight, on);
      else if (gt == FSH_DT_BF16) launch_step<FSH_DT_F32, FSH_DT_BF16>(a, eight, on);
      else launch_step<FSH_DT_F32, FSH_DT_F32>(a, eight, on);
      if (int rc = check_launch("adamw_kernel")) return rc;
    }
  }
  return FSH_OK;
}

FSH_API int fsh_adamw_state_values(const void* exp_avg_dev, const float* exp_avg_scale_dev, const void* exp_avg_sq_dev, const float* exp_avg_sq_scale_dev,
                                   int64_t numel, void* exp_avg_out_dev, void* exp_avg_sq_out_dev, int32_t dtype, void* stream) {
  using namespace fsh;
  const char* who = "fsh_adamw_state_values";
  if (numel < 0) return fail(FSH_EINVAL, "%s: negative size", who);
  if (!is_dtype(dtype)) return fail(FSH_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (numel == 0) return FSH_OK;
  if (!exp_avg_dev || !exp_avg_scale_dev || !exp_avg_sq_dev || !exp_avg_sq_scale_dev || !exp_avg_out_dev || !exp_avg_sq_out_dev) return fail(FSH_EINVAL, "%s: null pointer", who);
  if (!aligned(exp_avg_scale_dev, 4) || !aligned(exp_avg_sq_scale_dev, 4) || !aligned(exp_avg_out_dev, bytes_of(dtype)) || !aligned(exp_avg_sq_out_dev, bytes_of(dtype)))
    return fail(FSH_ENOTSUP, "%s: tensors must be aligned to their elements", who);
  const int64_t scales = ceil_div(numel, (int64_t)kStateBlock);
  const RowSpan inputs[] = {span_of(exp_avg_dev, numel, 1), span_of(exp_avg_sq_dev, numel, 1), span_of(exp_avg_scale_dev, scales, 4), span_of(exp_avg_sq_scale_dev, scales, 4)};
  const RowSpan outputs[] = {span_of(exp_avg_out_dev, numel, bytes_of(dtype)), span_of(exp_avg_sq_out_dev, numel, bytes_of(dtype))};
  if (outputs_overlap(inputs, outputs)) return fail(FSH_EINVAL, "%s: an output overlaps an input or the other output", who);
  const int64_t blocks = ceil_div(numel, (int64_t)kThreads * 8);
  const dim3 grid(static_cast<uint32_t>(blocks < kMaxGrid ? blocks : kMaxGrid)), block(kThreads);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, block, 0, on, static_cast<const uint8_t*>(exp_avg_dev), exp_avg_scale_dev, static_cast<const uint8_t*>(exp_avg_sq_dev),
                       exp_avg_sq_scale_dev, exp_avg_out_dev, exp_avg_sq_out_dev, numel);
  };
  if (dtype == FSH_DT_BF16) go(adamw_values_kernel<FSH_DT_BF16>);
  else if (dtype == FSH_DT_F16) go(adamw_values_kernel<FSH_DT_F16>);
  else go(adamw_values_kernel<FSH_DT_F32>);
  return check_launch("adamw_values_kernel");
}
