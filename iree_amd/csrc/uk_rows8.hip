// Rows of 8 bits with a scale for each token: the residual's addition with RMS norm, and rows
// or silu(gate) * up as they are (include/iree_amd_uk.h has the formulas).
//
// A row's codes are rne(127 y / max|y|): the norm's own factor cancels and goes into the scale
// alone. So y is the product of a kept sum and a weight, both of 16 bits, which f32 holds exactly between 2^-126 and
// 2^128, and the codes need neither the sum of squares nor its root: largest value and sum of
// squares come out of one reduction, and a row is read once. (Rows of bf16 with products past these ends can be worked on in
// 64 bits behind the loop; what that takes of its registers costs all other rows of bf16 2 to 3 %, and is left out.)
//
// A row stays in the registers of the threads that share it: 16 lanes have up to 128 elements, a wave up to 1024, 256 threads
// up to 4096, 512 up to 8192, 1024 the longer ones (4096 elements, 4099 rows of bf16: a wave 47 us, two 35, four 28,
// eight 27, before the weight was held and the next row on its way). Norms of 4099 x 4096 bf16, 117 MB, take 25.1 us, 22.8 on
// the device (5.1 TB/s, 11 of them vector instructions), eight weighted addends of 2048 x 4096, 176 MB, 36.1 and
// 34.6 (16 of them vector instructions: the sums in 64 bits), one row 3.2; the gate of 2048 x 14336,
// 147 MB, 36.0: 20 of them vector instructions, which the one workgroup of a compute unit does not hide behind its
// barriers (two of 512 threads with twice the elements each: 50 us, more registers than two have room for). Rows above
// 16384 spill: norms of 512 x 32768 37.7 us, of 256 x 65536 94, the gate of 1024 x 28672 42.0, all of 117 or 147 MB.
#include "uk_common.h"
#include "uk_kv4.h"

#include <type_traits>

namespace uk {
namespace {
using namespace kv4;

// 8 elements of 16 bits or 8 codes, wherever they lie.
typedef uint32_t row_bits_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t code_bits_t __attribute__((ext_vector_type(2), aligned(1)));

constexpr int kWidth = 8;      // elements a thread holds side by side

// Elements [at, at + 8) of a row of `dim`, zeros past its end.
__device__ inline u32x4 load8(const uint16_t* row, int at, int dim) {
  u32x4 w = {0, 0, 0, 0};
  if (at + kWidth <= dim) {
    w = *(const row_bits_t*)(row + at);
  } else {
#pragma unroll
    for (int i = 0; i < kWidth; ++i)
      if (at + i < dim) w[i / 2] |= (uint32_t)row[at + i] << (i % 2 * 16);
  }
  return w;
}
__device__ inline void store8(uint16_t* row, int at, int dim, u32x4 w) {
  if (at + kWidth <= dim) {
    *(row_bits_t*)(row + at) = w;
  } else {
#pragma unroll
    for (int i = 0; i < kWidth; ++i)
      if (at + i < dim) row[at + i] = (uint16_t)(w[i / 2] >> (i % 2 * 16));
  }
}
template <typename T>
__device__ inline void widen8(u32x4 w, float* x) {
  widen4<T>(u32x2{w.x, w.y}, x);
  widen4<T>(u32x2{w.z, w.w}, x + 4);
}

// The larger size; NaN where one is NaN.
__device__ inline float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
struct Larger {
  __device__ float operator()(float a, float b) const { return larger(a, b); }
  __device__ double operator()(double a, double b) const { return a > b ? a : b; }
};
struct Sum {
  __device__ double operator()(double a, double b) const { return a + b; }
};
constexpr float kMostFloat = 3.4028234663852886e38f;

// The values of a lane and its partner in one step of a reduction over a wave, in an order that both
// have (of the last two steps).
template <int kStep>
__device__ inline void partners(uint32_t v, uint32_t* a, uint32_t* b) {
  if constexpr (kStep < 4) {
    constexpr int control = kStep == 0 ? 0xB1 : kStep == 1 ? 0x4E : kStep == 2 ? 0x141 : 0x140;
    *a = v;
    *b = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, control, 0xF, 0xF, true);
  } else if constexpr (kStep == 4) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    *a = (uint32_t)p[0], *b = (uint32_t)p[1];
  } else {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    *a = (uint32_t)p[0], *b = (uint32_t)p[1];
  }
}
template <int kStep, typename F>
__device__ inline float joined(float v, F f) {
  uint32_t a, b;
  partners<kStep>(__builtin_bit_cast(uint32_t, v), &a, &b);
  return f(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
template <int kStep, typename F>
__device__ inline double joined(double v, F f) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  uint32_t a, b, c, d;
  partners<kStep>((uint32_t)u, &a, &b);
  partners<kStep>((uint32_t)(u >> 32), &c, &d);
  return f(__builtin_bit_cast(double, (uint64_t)c << 32 | a), __builtin_bit_cast(double, (uint64_t)d << 32 | b));
}
// Over the lanes of a wave, or its groups of 16 lanes.
template <int kLanes, typename V, typename F>
__device__ inline V over_lanes(V v, F f) {
  static_assert(kLanes == 16 || kLanes == 64, "a group of lanes");
  v = joined<0>(v, f);
  v = joined<1>(v, f);
  v = joined<2>(v, f);
  v = joined<3>(v, f);
  if constexpr (kLanes == 64) {
    v = joined<4>(v, f);
    v = joined<5>(v, f);
  }
  return v;
}

// The joint value of the kWaves (2, 4, 8 or 16) waves of a row, each of which has left its own in LDS.
template <int kWaves, typename V, typename F>
__device__ inline V over_waves(const V* shared, F f) {
  V v = shared[threadIdx.x & (kWaves - 1)];
  v = joined<0>(v, f);
  if constexpr (kWaves > 2) v = joined<1>(v, f);
  if constexpr (kWaves > 4) v = joined<2>(v, f);
  if constexpr (kWaves > 8) v = joined<3>(v, f);
  return v;
}

// 127 y / top of 8 values as codes: t times `inverse` is added to 1.5 * 2^23 with one rounding, which
// leaves the code in the last byte; `far` grows to the largest distance from a code.
__device__ inline u32x2 codes8(const float* t, float inverse, float* far) {
  constexpr float kShift = 12582912.f;
  uint32_t b[kWidth];
#pragma unroll
  for (int i = 0; i < kWidth; ++i) {
    const float moved = __builtin_fmaf(t[i], inverse, kShift), q = moved - kShift;
    *far = fmaxf(*far, fabsf(__builtin_fmaf(t[i], inverse, -q)));
    b[i] = __builtin_bit_cast(uint32_t, moved);
  }
  u32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0C0C0400);
    const uint32_t hi = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x04000C0C);
    w[h] = lo | hi;
  }
  return w;
}

__device__ inline void store_codes8(int8_t* row, int at, int dim, u32x2 w) {
  if (at + kWidth <= dim) {
    *(code_bits_t*)(row + at) = w;
  } else {
#pragma unroll
    for (int i = 0; i < kWidth; ++i)
      if (at + i < dim) row[at + i] = (int8_t)(w[i / 4] >> (i % 4 * 8));
  }
}

// The code of a value in 64 bits, which lies between a and a + 1 in size: of a product of two values of 16 bits,
// over another, both sides are exact.
__device__ inline uint32_t code_between(double y, double top, float a) {
  const double size = fabs(y) * 127.0, border = ((double)a + 0.5) * top;
  const int q = (int)a + (size > border || (size == border && ((int)a & 1)));
  return (uint32_t)(y < 0.0 ? -q : q) & 0xFF;
}

// f32 gives 127 t / top with an error below this (127 / top and its product with t are each rounded
// once, below 127 * 2^-23 together): where a value lies nearer than that to the border between two
// codes, 64 bits decide.
constexpr float kSlack = 1.f / 32768;

// Codes of 8 exact values.
__device__ inline u32x2 exact_codes8(const float* t, float inverse, float top) {
  float far = 0.f;
  u32x2 w = codes8(t, inverse, &far);
  if (far >= 0.5f - kSlack) {
#pragma unroll
    for (int i = 0; i < kWidth; ++i) {
      const float v = fabsf(t[i] * inverse), a = floorf(v);
      if (fabsf(v - a - 0.5f) <= 2 * kSlack) {
        asm volatile("");      // (a branch of its own: worked out for all 8, it takes 30 registers more)
        w[i / 4] = (w[i / 4] & ~(0xFFu << (i % 4 * 8))) | code_between(t[i], top, a) << (i % 4 * 8);
      }
    }
  }
  return w;
}

// Rows whose largest value lies below this are worked on 2^100 times as large: 127 / top would overflow.
constexpr float kTiny = 1e-30f, kTinyScale = 1.2676506002282294e30f;

template <int kReps>
__device__ inline float scaled_if_tiny(float (&t)[kReps][kWidth], float top) {
  if (!(top < kTiny)) return top;
#pragma unroll
  for (int r = 0; r < kReps; ++r)
#pragma unroll
    for (int i = 0; i < kWidth; ++i) t[r][i] *= kTinyScale;
  return top * kTinyScale;
}

template <int kThreads>
constexpr int kBlockOf = kThreads < 256 ? 256 : kThreads;

// ---------------------------------------------------------------------------
// rms_norm_quantize
// ---------------------------------------------------------------------------

// Which row of its workgroup's a wave has a part of.
template <int kThreads>
__device__ inline int row_of_wave() {
  if constexpr (kThreads >= 256) return 0;
  else if constexpr (kThreads >= 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  else return threadIdx.x / kThreads;
}

// Rows of a launch are dealt to its workgroups in turn, kRows at a time; while a row is worked on, the next
// one of its threads is on its way.

// kOne: one addend without a weight.
template <typename T, bool kOne, int kThreads, int kReps>
__global__ __launch_bounds__(kBlockOf<kThreads>) void rms_norm_quantize_kernel(RmsNormQuantizeArgs a) {
  constexpr int kRows = kBlockOf<kThreads> / kThreads, kLanes = kThreads < 64 ? kThreads : 64, kWaves = kThreads / kLanes;
  __shared__ double shared_squares[kWaves];
  __shared__ float shared_top[kWaves];
  const int thread = threadIdx.x % kThreads, dim = a.dim;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t token = (int64_t)blockIdx.x * kRows + row_of_wave<kThreads>();
  u32x4 next_added[kOne ? kReps : 1], next_bits[kReps];
  auto load_row = [&](int64_t of) {
    const uint16_t* x = (const uint16_t*)a.x + of * a.x_stride0;
    const uint16_t* residual = a.residual ? (const uint16_t*)a.residual + of * a.residual_stride : nullptr;
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
      if constexpr (kOne) next_added[r] = at < dim ? load8(x, at, dim) : u32x4{0, 0, 0, 0};
      next_bits[r] = residual && at < dim ? load8(residual, at, dim) : u32x4{0, 0, 0, 0};
    }
  };
  // (rows above 16384, of 32 or 64 elements a thread, spill registers without a second row as well: 34 to 36 and 234 to 258
  // with one addend, 74 to 76 and more with several)
  constexpr bool kAhead = kReps <= 2;
  if (kAhead && token < a.tokens) load_row(token);
  // (the weight, too, is on its way before it is needed, and for all rows of a workgroup, where there is room for it)
  constexpr bool kHeld = kReps <= 2;
  u32x4 weight[kHeld ? kReps : 1];
  auto load_weight = [&](int r) {
    const int at = (r * kThreads + thread) * kWidth;
    return at < dim ? load8((const uint16_t*)a.weight, at, dim) : u32x4{0, 0, 0, 0};
  };
  if constexpr (kHeld) {
    if (a.weight) {
#pragma unroll
      for (int r = 0; r < kReps; ++r) weight[r] = load_weight(r);
    }
  }
  for (; token < a.tokens; token += step) {
    if constexpr (!kAhead) load_row(token);
    u32x4 added[kOne ? kReps : 1], bits[kReps];
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      if constexpr (kOne) added[r] = next_added[r];
      bits[r] = next_bits[r];
    }
    if (kAhead && token + step < a.tokens) load_row(token + step);
    // The sum, rounded to its type.
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
      float h[kWidth];
      __builtin_amdgcn_sched_barrier(0);      // (one after the other, in the same registers)
      widen8<T>(bits[r], h);
      if constexpr (kOne) {
        float v[kWidth];
        widen8<T>(added[r], v);
#pragma unroll
        for (int i = 0; i < kWidth; ++i) h[i] += v[i];
      } else if (at < dim) {
        // (several addends in 64 bits: f32 would round at every one of them. The sum is then rounded twice, to f32 and to its
        // type, as the sum of one addend is and as torch's own conversions do: of random sums of f16 one in 16000 goes to the
        // farther of two neighbours that f32 cannot tell apart, by at most 2^-24 of itself)
        const uint16_t* x = (const uint16_t*)a.x + token * a.x_stride0;
        const float* factors = a.factors ? a.factors + token * a.factors_stride : nullptr;
        double wide[kWidth];
#pragma unroll
        for (int i = 0; i < kWidth; ++i) wide[i] = h[i];
#pragma unroll 8
        for (int j = 0; j < a.addends; ++j) {
          const float factor = factors ? factors[j] : 1.f;
          float v[kWidth];
          widen8<T>(load8(x + j * a.x_stride1, at, dim), v);
          // (what a slot without an expert holds, NaN too, changes nothing)
#pragma unroll
          for (int i = 0; i < kWidth; ++i) wide[i] = fma((double)factor, (double)(factor == 0.f ? 0.f : v[i]), wide[i]);
        }
#pragma unroll
        for (int i = 0; i < kWidth; ++i) h[i] = (float)wide[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) bits[r][i] = T::narrow2(h[2 * i], h[2 * i + 1]);
    }
    if (a.sum_out) {
      uint16_t* sum_out = (uint16_t*)a.sum_out + token * a.sum_out_stride;
#pragma unroll
      for (int r = 0; r < kReps; ++r) {
        const int at = (r * kThreads + thread) * kWidth;
        if (at < dim) store8(sum_out, at, dim, bits[r]);
      }
    }
    float t[kReps][kWidth], top = 0.f;
    double squares = 0.0;
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      __builtin_amdgcn_sched_barrier(0);
      widen8<T>(bits[r], t[r]);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) squares = fma((double)t[r][i], (double)t[r][i], squares);
      if (a.weight) {
        float w[kWidth];
        if constexpr (kHeld) widen8<T>(weight[r], w);
        else widen8<T>(load_weight(r), w);
#pragma unroll
        for (int i = 0; i < kWidth; ++i) t[r][i] *= w[i];
      }
#pragma unroll
      for (int i = 0; i < kWidth; ++i) top = larger(top, fabsf(t[r][i]));
    }
    squares = over_lanes<kLanes>(squares, Sum());
    top = over_lanes<kLanes>(top, Larger());
    if constexpr (kWaves > 1) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) shared_squares[threadIdx.x >> 6] = squares, shared_top[threadIdx.x >> 6] = top;
      __syncthreads();
      squares = over_waves<kWaves>(shared_squares, Sum());
      top = over_waves<kWaves>(shared_top, Larger());
    }
    const bool finite = top <= kMostFloat;
    const float its_top = scaled_if_tiny<kReps>(t, top), inverse = 127.f / its_top;
    int8_t* q = (int8_t*)a.q + token * a.q_stride;
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
      if (at >= dim) continue;
      u32x2 w = {0, 0};
      __builtin_amdgcn_sched_barrier(0);
      if (finite && top > 0.f) w = exact_codes8(t[r], inverse, its_top);
      store_codes8(q, at, dim, w);
    }
    if (thread == 0) {
      const double rate = 1.0 / sqrt(squares / dim + (double)a.eps);
      a.scale[token] = !finite ? __builtin_nanf("") : top > 0.f ? (float)(top * rate / 127.0) : 0.f;
    }
  }
}

// ---------------------------------------------------------------------------
// quantize_rows
// ---------------------------------------------------------------------------

template <typename T, int kThreads, int kReps>
__global__ __launch_bounds__(kBlockOf<kThreads>) void quantize_rows_kernel(QuantizeRowsArgs a) {
  constexpr int kRows = kBlockOf<kThreads> / kThreads, kLanes = kThreads < 64 ? kThreads : 64, kWaves = kThreads / kLanes;
  __shared__ float shared_top[kWaves];
  const int thread = threadIdx.x % kThreads, cols = a.cols;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + row_of_wave<kThreads>();
  u32x4 next[kReps];
  auto load_row = [&](int64_t of) {
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
      next[r] = at < cols ? load8((const uint16_t*)a.x + of * a.x_stride, at, cols) : u32x4{0, 0, 0, 0};
    }
  };
  if (row < a.rows) load_row(row);
  for (; row < a.rows; row += step) {
    float t[kReps][kWidth], top = 0.f;
#pragma unroll
    for (int r = 0; r < kReps; ++r) widen8<T>(next[r], t[r]);
    if (row + step < a.rows) load_row(row + step);
#pragma unroll
    for (int r = 0; r < kReps; ++r)
#pragma unroll
      for (int i = 0; i < kWidth; ++i) top = larger(top, fabsf(t[r][i]));
    top = over_lanes<kLanes>(top, Larger());
    if constexpr (kWaves > 1) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) shared_top[threadIdx.x >> 6] = top;
      __syncthreads();
      top = over_waves<kWaves>(shared_top, Larger());
    }
    const bool finite = top <= kMostFloat;
    const float its_top = scaled_if_tiny<kReps>(t, top), inverse = 127.f / its_top;
    int8_t* q = (int8_t*)a.q + row * a.q_stride;
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
      if (at >= cols) continue;
      u32x2 w = {0, 0};
      __builtin_amdgcn_sched_barrier(0);      // (one after the other, in the same registers)
      if (finite && top > 0.f) w = exact_codes8(t[r], inverse, its_top);
      store_codes8(q, at, cols, w);
    }
    if (thread == 0) a.scale[row] = finite ? (float)(top / 127.0) : __builtin_nanf("");
  }
}

__device__ inline uint32_t code_of(double y, double top) { return (uint32_t)(int)__builtin_rint(y * 127.0 / top) & 0xFF; }

// silu(g) u, within 2^-19.1 of itself where an exponential of up to 88 closes the gate (past that
// nothing is left of it next to sizes up to 2^40):
//   2^p with p = g * -log2(e), and what p's rounding left out as a factor.
__device__ inline float silu_mul_near(float g, float u) {
  constexpr float kLog2e = 1.44269502162933349609375f;
  const float p = g * -kLog2e, rest = __builtin_fmaf(g, -kLog2e, -p);
  const float e = __builtin_amdgcn_exp2f(p) * __builtin_fmaf(rest, 0.693147180559945f, 1.f);
  return g * __builtin_amdgcn_rcpf(1.f + e) * u;
}
__device__ inline double silu_mul_wide(float g, float u) { return (double)g / (1.0 + exp(-(double)g)) * (double)u; }
// 127 times the error of such a value and of the largest of the row.
constexpr float kGatedSlack = 1.f / 2048;
constexpr float kLarge = 1.0995116e12f;      // 2^40
// Eights of a row with a code (or the largest value) that f32 leaves open: about one in 130, whose elements
// the threads then look at side by side. A row with more of them is worked out in 64 bits as a whole.
constexpr int kMostOpen = 512;

// All of a row in 64 bits: rows of sizes that f32 does not hold, or with too many open codes.
template <typename T, int kThreads>
__device__ inline void gated_row_wide(const uint16_t* x, const uint16_t* up, int8_t* q, float* scale, int cols,
                                      double* shared) {
  const int thread = threadIdx.x;
  double top = 0.0;
#pragma unroll 1
  for (int i = thread; i < cols; i += kThreads) {
    const float g = T::widen(x[i]), u = T::widen(up[i]);
    const double y = fabs(silu_mul_wide(g, u));
    const bool finite = fabsf(g) <= kMostFloat && fabsf(u) <= kMostFloat && y <= kMostFloat;
    top = Larger()(top, finite ? y : (double)__builtin_inff());
  }
  top = over_lanes<64>(top, Larger());
  __syncthreads();
  if ((thread & 63) == 0) shared[thread >> 6] = top;
  __syncthreads();
  top = shared[0];
  for (int w = 1; w < kThreads / 64; ++w) top = Larger()(top, shared[w]);
  const bool finite = top <= kMostFloat;
#pragma unroll 1
  for (int i = thread; i < cols; i += kThreads)
    q[i] = finite && top > 0.0 ? (int8_t)code_of(silu_mul_wide(T::widen(x[i]), T::widen(up[i])), top) : 0;
  if (thread == 0) *scale = finite ? (float)(top / 127.0) : __builtin_nanf("");
}

template <typename T, int kThreads, int kReps>
__global__ __launch_bounds__(kThreads) void quantize_gated_rows_kernel(QuantizeRowsArgs a) {
  constexpr int kWaves = kThreads / 64;
  constexpr bool kAnySize = std::is_same<T, BF16>::value;      // (f16 has none above 2^40)
  __shared__ float shared_top[kWaves];
  __shared__ double shared_wide[kWaves];
  __shared__ int open_count[2], open[2][kMostOpen];      // candidates for the largest, open codes
  const int thread = threadIdx.x, first_thread = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63), cols = a.cols;
  u32x4 gates[kReps], ups[kReps];
  auto load_row = [&](int64_t of) {
    const uint16_t* x = (const uint16_t*)a.x + of * a.x_stride;
    const uint16_t* up = (const uint16_t*)a.up + of * a.up_stride;
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
      gates[r] = at < cols ? load8(x, at, cols) : u32x4{0, 0, 0, 0};
      ups[r] = at < cols ? load8(up, at, cols) : u32x4{0, 0, 0, 0};
    }
  };
  constexpr bool kAhead = kReps <= 2;
  if (kAhead && (int64_t)blockIdx.x < a.rows) load_row(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if constexpr (!kAhead) load_row(row);
    const uint16_t* x = (const uint16_t*)a.x + row * a.x_stride;
    const uint16_t* up = (const uint16_t*)a.up + row * a.up_stride;
    int8_t* q = (int8_t*)a.q + row * a.q_stride;
    float t[kReps][kWidth], mine[kReps], top = 0.f, large = 0.f;
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      mine[r] = 0.f;
#pragma unroll
      for (int i = 0; i < kWidth; ++i) t[r][i] = 0.f;
      if ((r * kThreads + first_thread) * kWidth >= cols) continue;      // (a wave behind the row's end)
      float g[kWidth], u[kWidth];
      __builtin_amdgcn_sched_barrier(0);      // (one after the other, in the same registers)
      widen8<T>(gates[r], g);
      widen8<T>(ups[r], u);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) {
        t[r][i] = silu_mul_near(g[i], u[i]);
        if constexpr (kAnySize) large = fmaxf(fmaxf(large, fabsf(g[i])), fabsf(u[i]));
      }
      // (a gate or factor that is not finite gives a product that is not either)
#pragma unroll
      for (int i = 0; i < kWidth; ++i) mine[r] = larger(mine[r], fabsf(t[r][i]));
      top = larger(top, mine[r]);
    }
    if (kAhead && row + gridDim.x < a.rows) load_row(row + gridDim.x);
    // (sizes that f32 does not see through count as not finite here)
    if (kAnySize && !(large <= kLarge)) top = __builtin_nanf("");
    top = over_lanes<64>(top, Larger());
    if ((thread & 63) == 0) shared_top[thread >> 6] = top;
    if (thread < 2) open_count[thread] = 0;
    __syncthreads();
    if constexpr (kWaves > 1) top = over_waves<kWaves>(shared_top, Larger());
    bool wide = !(top <= kLarge * kLarge) || top < 1.f / kLarge;
    const float from = top * (1.f - 1.f / 131072), inverse = 127.f / top;
    if (!wide) {
#pragma unroll
      for (int r = 0; r < kReps; ++r) {
        const int at = (r * kThreads + thread) * kWidth;
        if ((r * kThreads + first_thread) * kWidth >= cols) continue;
        float far = 0.f;
        __builtin_amdgcn_sched_barrier(0);
        const u32x2 w = codes8(t[r], inverse, &far);
        if (at < cols) store_codes8(q, at, cols, w);
        if (mine[r] >= from) {
          const int n = atomicAdd(&open_count[0], 1);
          if (n < kMostOpen) open[0][n] = at;
        }
        if (far >= 0.5f - kGatedSlack) {
          const int n = atomicAdd(&open_count[1], 1);
          if (n < kMostOpen) open[1][n] = at;
        }
      }
      __syncthreads();           // (the codes are stored, the lists are complete)
      wide = open_count[0] > kMostOpen || open_count[1] > kMostOpen;
    }
    if (wide) {
      gated_row_wide<T, kThreads>(x, up, q, &a.scale[row], cols, shared_wide);
    } else {
      // One wave has the largest in 64 bits, which is among those near the largest in 32; the others meanwhile
      // work out the first values with an open code, and then all the codes.
      const int items = open_count[1] * kWidth;
      auto item = [&](int n, int* i, double* y) {
        *i = open[1][n / kWidth] + n % kWidth;
        if (*i >= cols) return false;
        const float g = T::widen(x[*i]), u = T::widen(up[*i]), v = silu_mul_near(g, u) * inverse;
        if (fabsf(v - __builtin_rintf(v)) < 0.5f - 1.02f * kGatedSlack) return false;
        *y = silu_mul_wide(g, u);
        return true;
      };
      int first_i = 0;
      double first_y = 0.0;
      bool first_is_open = false;
      if (thread < 64) {
        double exact = 0.0;
        for (int n = thread; n < open_count[0] * kWidth; n += 64) {
          const int i = open[0][n / kWidth] + n % kWidth;
          if (i >= cols) continue;
          const float g = T::widen(x[i]), u = T::widen(up[i]);
          if (fabsf(silu_mul_near(g, u)) >= from) exact = Larger()(exact, fabs(silu_mul_wide(g, u)));
        }
        exact = over_lanes<64>(exact, Larger());
        if (thread == 0) shared_wide[0] = exact, a.scale[row] = (float)(exact / 127.0);
      } else if (thread - 64 < items) {
        first_is_open = item(thread - 64, &first_i, &first_y);
      }
      __syncthreads();
      const double exact = shared_wide[0];
      if (first_is_open) q[first_i] = (int8_t)code_of(first_y, exact);
      for (int n = kThreads - 64 + thread; n < items; n += kThreads) {
        int i;
        double y;
        if (item(n, &i, &y)) q[i] = (int8_t)code_of(y, exact);
      }
    }
    __syncthreads();             // (the lists are used up)
  }
}

// Workgroups of `block` threads for so many rows, `rows_of_block` in each at a time: at most `waves` of them on
// a vector unit, whether resident or not; they take the rows in turn.
unsigned grid_of(int64_t rows, int rows_of_block, int block, int waves) {
  const int64_t blocks = ceil_div(rows, (int64_t)rows_of_block), most = (int64_t)device_cu_count() * waves * 256 / block;
  return (unsigned)(blocks < most ? blocks : most);
}

// Calls launch(threads, reps) with the first of the shapes (threads that share a row, times 8 elements of
// each) that holds a row of `dim` elements.
#define UK_ROW_SHAPE(threads, reps) \
  if (dim <= (threads) * (reps) * kWidth) return launch(std::integral_constant<int, threads>(), std::integral_constant<int, reps>())
constexpr const char* kTooLong = "rows of more than 65536 elements";
// (norms of 2^24 elements of bf16: rows of 64 with 16 threads 37 us, with a wave 118)
template <typename Launch>
int with_row_shape(int64_t dim, Launch launch) {
  UK_ROW_SHAPE(16, 1);
  UK_ROW_SHAPE(64, 1);
  UK_ROW_SHAPE(64, 2);
  UK_ROW_SHAPE(256, 1);
  UK_ROW_SHAPE(256, 2);
  UK_ROW_SHAPE(512, 2);
  UK_ROW_SHAPE(1024, 2);
  UK_ROW_SHAPE(1024, 4);
  UK_ROW_SHAPE(1024, 8);
  return fail(IREE_AMD_UK_STATUS_UNIMPLEMENTED, kTooLong);
}
// (more waves where each row needs more loads: four addends of 2048 x 8192 28.9 us, with 512 threads 37.7)
template <typename Launch>
int with_row_shape_of_addends(int64_t dim, Launch launch) {
  UK_ROW_SHAPE(16, 1);
  UK_ROW_SHAPE(64, 1);
  UK_ROW_SHAPE(64, 2);
  UK_ROW_SHAPE(256, 1);
  UK_ROW_SHAPE(256, 2);
  UK_ROW_SHAPE(1024, 1);
  UK_ROW_SHAPE(1024, 2);
  UK_ROW_SHAPE(1024, 4);
  UK_ROW_SHAPE(1024, 8);
  return fail(IREE_AMD_UK_STATUS_UNIMPLEMENTED, kTooLong);
}
// (gated rows have a workgroup each: 2^24 elements in rows of 64 with one wave 181 us, with four 460)
template <typename Launch>
int with_gated_row_shape(int64_t dim, Launch launch) {
  UK_ROW_SHAPE(64, 1);
  UK_ROW_SHAPE(64, 2);
  UK_ROW_SHAPE(128, 2);
  UK_ROW_SHAPE(256, 2);
  UK_ROW_SHAPE(512, 2);
  UK_ROW_SHAPE(1024, 2);
  UK_ROW_SHAPE(1024, 4);
  UK_ROW_SHAPE(1024, 8);
  return fail(IREE_AMD_UK_STATUS_UNIMPLEMENTED, kTooLong);
}
#undef UK_ROW_SHAPE

}  // namespace

template <bool kOne>
static int launch_norm(const RmsNormQuantizeArgs& a, hipStream_t s) {
  auto launch = [&](auto threads, auto reps) {
    constexpr int kThreads = decltype(threads)::value, kReps = decltype(reps)::value, kBlock = kBlockOf<kThreads>;
    const dim3 grid(grid_of(a.tokens, kBlock / kThreads, kBlock, 8));
    if (a.bf16) hipLaunchKernelGGL((rms_norm_quantize_kernel<BF16, kOne, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    else hipLaunchKernelGGL((rms_norm_quantize_kernel<F16, kOne, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    return check_hip(hipGetLastError(), "rms_norm_quantize launch");
  };
  if constexpr (kOne) return with_row_shape(a.dim, launch);
  else return with_row_shape_of_addends(a.dim, launch);
}
int launch_rms_norm_quantize(const RmsNormQuantizeArgs& a, hipStream_t s) {
  return a.addends == 1 && !a.factors ? launch_norm<true>(a, s) : launch_norm<false>(a, s);
}

int launch_quantize_rows(const QuantizeRowsArgs& a, hipStream_t s) {
  if (a.up)
    return with_gated_row_shape(a.cols, [&](auto threads, auto reps) {
      constexpr int kThreads = decltype(threads)::value, kReps = decltype(reps)::value;
      const dim3 grid(grid_of(a.rows, 1, kThreads, 4)), block(kThreads);
      if (a.bf16) hipLaunchKernelGGL((quantize_gated_rows_kernel<BF16, kThreads, kReps>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((quantize_gated_rows_kernel<F16, kThreads, kReps>), grid, block, 0, s, a);
      return check_hip(hipGetLastError(), "quantize_rows launch");
    });
  return with_row_shape(a.cols, [&](auto threads, auto reps) {
    constexpr int kThreads = decltype(threads)::value, kReps = decltype(reps)::value, kBlock = kBlockOf<kThreads>;
    const dim3 grid(grid_of(a.rows, kBlock / kThreads, kBlock, 8));
    if (a.bf16) hipLaunchKernelGGL((quantize_rows_kernel<BF16, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    else hipLaunchKernelGGL((quantize_rows_kernel<F16, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    return check_hip(hipGetLastError(), "quantize_rows launch");
  });
}

}  // namespace uk
