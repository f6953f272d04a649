// Rows of 8 bits with a scale for each token: the residual's addition with RMS norm, and rows
// or silu(gate) * up as they are (include/iree_amd_uk.h has the formulas).
//
// A row's codes are rne(127 y / max|y|): the norm's own factor cancels and goes into the scale
// alone. So y is the product of a kept sum and a weight, both of 16 bits, which f32 holds exactly,
// and the codes need neither the sum of squares nor its root: largest value and sum of
// squares come out of one reduction, and a row is read once.
//
// A row stays in the registers of the threads that share it: one wave up to 1024 elements, 256
// threads up to 8192, 1024 threads up to 65536. What bounds them is memory.
#include "uk_common.h"
#include "uk_kv4.h"

namespace uk {
namespace {
using namespace kv4;

// 8 elements of 16 bits or 8 codes, wherever they lie.
typedef uint32_t row_bits_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t code_bits_t __attribute__((ext_vector_type(2), aligned(1)));

constexpr int kWidth = 8;      // elements a thread holds side by side

// Elements [at, at + 8) of a row of `dim`, zeros past its end.
template <typename T>
__device__ inline void load8(const uint16_t* row, int at, int dim, float* x) {
  u32x4 w = {0, 0, 0, 0};
  if (at + kWidth <= dim) {
    w = *(const row_bits_t*)(row + at);
  } else {
#pragma unroll
    for (int i = 0; i < kWidth; ++i)
      if (at + i < dim) w[i / 2] |= (uint32_t)row[at + i] << (i % 2 * 16);
  }
  widen4<T>(u32x2{w.x, w.y}, x);
  widen4<T>(u32x2{w.z, w.w}, x + 4);
}

// What a row's reductions give.
struct RowSums {
  double squares;
  float top;             // largest size
  float bad;             // 0, or NaN where a value is not finite
};

__device__ inline RowSums join(RowSums a, RowSums b) {
  return {a.squares + b.squares, fmaxf(a.top, b.top), a.bad + b.bad};
}
struct RowSizes {
  float top, large;      // largest size, and that of what it is made of
  float bad;
};
__device__ inline RowSizes join(RowSizes a, RowSizes b) {
  return {fmaxf(a.top, b.top), fmaxf(a.large, b.large), a.bad + b.bad};
}
__device__ inline double join(double a, double b) { return fmax(a, b); }

__device__ inline RowSums other(RowSums v, int mask) {
  return {__shfl_xor(v.squares, mask), __shfl_xor(v.top, mask), __shfl_xor(v.bad, mask)};
}
__device__ inline RowSizes other(RowSizes v, int mask) {
  return {__shfl_xor(v.top, mask), __shfl_xor(v.large, mask), __shfl_xor(v.bad, mask)};
}
__device__ inline double other(double v, int mask) { return __shfl_xor(v, mask); }

// The joint value of the kThreads threads of a row, the same in all of them, added in a fixed
// order. `shared`: one value for each wave of the row; a barrier on entry for those of a
// workgroup, so that it may be used again.
template <int kThreads, typename V>
__device__ inline V over_row(V v, V* shared) {
#pragma unroll
  for (int mask = 1; mask < 64; mask *= 2) v = join(v, other(v, mask));
  if constexpr (kThreads > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) v = join(v, shared[w]);
  }
  return v;
}

// The codes of 8 values t that stand for `exact(i)`, whose largest size in the row is `top`.
// f32 gives 127 t / top with an error below kSlack; where that leaves open which side of the border
// between two codes a value lies on, the 64-bit quotient decides: a product of two values of 16 bits
// over another that is not on a border lies 2^-26 of itself away from it at least.
template <typename Exact>
__device__ inline u32x2 codes8(const float* t, float inverse, double top, float slack, Exact exact) {
  int q[kWidth];
  float nearest = 1.f;
#pragma unroll
  for (int i = 0; i < kWidth; ++i) {
    const float v = t[i] * inverse, r = __builtin_rintf(v);
    nearest = fminf(nearest, 0.5f - fabsf(v - r));
    q[i] = (int)r;
  }
  if (nearest <= slack) {
#pragma unroll
    for (int i = 0; i < kWidth; ++i) {
      const float v = t[i] * inverse;
      // (a value that f32 does not hold may be NaN here)
      if (!(0.5f - fabsf(v - __builtin_rintf(v)) > slack)) q[i] = (int)__builtin_rint(exact(i) * 127.0 / top);
    }
  }
  u32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = (uint32_t)(q[4 * h] & 0xFF) | (uint32_t)(q[4 * h + 1] & 0xFF) << 8 | (uint32_t)(q[4 * h + 2] & 0xFF) << 16 |
           (uint32_t)q[4 * h + 3] << 24;
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

// A product of two values of 16 bits is exact in f32, 127 / top and its product with t are each
// rounded once: below 127 * 2^-23 together, and the subtraction's rounding.
constexpr float kSlack = 1.f / 32768;
// Below this a quotient by the largest value could overflow f32: all of the row in 64 bits.
constexpr float kTiny = 1e-30f;

// ---------------------------------------------------------------------------
// rms_norm_quantize
// ---------------------------------------------------------------------------

template <typename T, int kThreads, int kReps>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void rms_norm_quantize_kernel(RmsNormQuantizeArgs a) {
  constexpr int kBlock = kThreads < 256 ? 256 : kThreads, kRows = kBlock / kThreads;
  __shared__ RowSums shared[kBlock / 64];
  const int thread = threadIdx.x % kThreads, dim = a.dim;
  for (int64_t token = (int64_t)blockIdx.x * kRows + threadIdx.x / kThreads; token < a.tokens;
       token += (int64_t)gridDim.x * kRows) {
    const uint16_t* x = (const uint16_t*)a.x + token * a.x_stride0;
    const uint16_t* residual = a.residual ? (const uint16_t*)a.residual + token * a.residual_stride : nullptr;
    uint16_t* sum_out = a.sum_out ? (uint16_t*)a.sum_out + token * a.sum_out_stride : nullptr;
    const float* factors = a.factors ? a.factors + token * a.factors_stride : nullptr;
    float t[kReps][kWidth];
    RowSums sums = {0.0, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
#pragma unroll
      for (int i = 0; i < kWidth; ++i) t[r][i] = 0.f;
      if (at >= dim) continue;
      float h[kWidth] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (residual) load8<T>(residual, at, dim, h);
      if (a.addends == 1 && !factors) {
        float v[kWidth];
        load8<T>(x, at, dim, v);
#pragma unroll
        for (int i = 0; i < kWidth; ++i) h[i] += v[i];
      } else {
        // (several addends in 64 bits, so that their order cannot show in the sum's rounding)
        double wide[kWidth];
#pragma unroll
        for (int i = 0; i < kWidth; ++i) wide[i] = h[i];
#pragma unroll 4
        for (int j = 0; j < a.addends; ++j) {
          const float factor = factors ? factors[j] : 1.f;
          float v[kWidth];
          load8<T>(x + j * a.x_stride1, at, dim, v);
          // (what a slot without an expert holds, NaN too, changes nothing)
#pragma unroll
          for (int i = 0; i < kWidth; ++i)
            wide[i] = fma((double)factor, factor == 0.f ? 0.0 : (double)v[i], wide[i]);
        }
#pragma unroll
        for (int i = 0; i < kWidth; ++i) h[i] = (float)wide[i];
      }
      // The sum as it is kept.
      u32x4 bits;
#pragma unroll
      for (int i = 0; i < 4; ++i) bits[i] = T::narrow2(h[2 * i], h[2 * i + 1]);
      if (sum_out) {
        if (at + kWidth <= dim) {
          *(row_bits_t*)(sum_out + at) = bits;
        } else {
#pragma unroll
          for (int i = 0; i < kWidth; ++i)
            if (at + i < dim) sum_out[at + i] = (uint16_t)(bits[i / 2] >> (i % 2 * 16));
        }
      }
      widen4<T>(u32x2{bits.x, bits.y}, h);
      widen4<T>(u32x2{bits.z, bits.w}, h + 4);
      float w[kWidth] = {1, 1, 1, 1, 1, 1, 1, 1};
      if (a.weight) load8<T>((const uint16_t*)a.weight, at, dim, w);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) {
        t[r][i] = h[i] * w[i];
        sums.squares = fma((double)h[i], (double)h[i], sums.squares);
        sums.top = fmaxf(sums.top, fabsf(t[r][i]));
        sums.bad = fmaf(t[r][i], 0.f, sums.bad);
      }
      // (a sum that is not finite next to a weight of 0)
      if (a.weight) {
#pragma unroll
        for (int i = 0; i < kWidth; ++i) sums.bad = fmaf(h[i], 0.f, sums.bad);
      }
    }
    sums = over_row<kThreads>(sums, shared + threadIdx.x / kThreads * (kThreads / 64));
    const bool finite = sums.bad == 0.f;
    const bool tiny = sums.top < kTiny;
    const float inverse = finite && !tiny ? 127.f / sums.top : 0.f;
    int8_t* q = (int8_t*)a.q + token * a.q_stride;
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
      if (at >= dim) continue;
      u32x2 w = {0, 0};
      if (finite && sums.top > 0.f)
        w = codes8(t[r], inverse, sums.top, tiny ? 1.f : kSlack, [&](int i) { return (double)t[r][i]; });
      store_codes8(q, at, dim, w);
    }
    if (thread == 0) {
      const double rate = 1.0 / sqrt(sums.squares / dim + (double)a.eps);
      a.scale[token] = !finite ? __builtin_nanf("") : sums.top > 0.f ? (float)(sums.top * rate / 127.0) : 0.f;
    }
  }
}

// ---------------------------------------------------------------------------
// quantize_rows
// ---------------------------------------------------------------------------

// silu(g) u, within 2^-21 of itself for sizes up to 2^40 and an exponential that f32 holds (past it: 0).
__device__ inline float silu_mul_near(float g, float u) {
  constexpr float kLog2e = 1.44269502162933349609375f, kRest = 1.92596299112661746887e-8f;
  const float p = -g * kLog2e;
  const float rest = fmaf(-g, kLog2e, -p) - g * kRest;       // -g log2(e) - p
  const float e = __builtin_amdgcn_exp2f(p);
  const float sum = 1.f + (p > 126.f ? __builtin_inff() : fmaf(e, rest * 0.693147180559945f, e));
  return g * __builtin_amdgcn_rcpf(sum) * u;
}
__device__ inline double silu_mul_wide(float g, float u) { return (double)g / (1.0 + exp(-(double)g)) * (double)u; }
constexpr float kGatedSlack = 1.f / 8192;
constexpr float kLarge = 1.0995116e12f;      // 2^40

template <typename T, bool kGated, int kThreads, int kReps>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void quantize_rows_kernel(QuantizeRowsArgs a) {
  constexpr int kBlock = kThreads < 256 ? 256 : kThreads, kRows = kBlock / kThreads;
  __shared__ RowSizes shared[kBlock / 64];
  __shared__ double shared_top[kBlock / 64];
  const int thread = threadIdx.x % kThreads, cols = a.cols, first_wave = threadIdx.x / kThreads * (kThreads / 64);
  for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kThreads; row < a.rows;
       row += (int64_t)gridDim.x * kRows) {
    const uint16_t* x = (const uint16_t*)a.x + row * a.x_stride;
    const uint16_t* up = kGated ? (const uint16_t*)a.up + row * a.up_stride : nullptr;
    float t[kReps][kWidth];
    RowSizes sizes = {0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
#pragma unroll
      for (int i = 0; i < kWidth; ++i) t[r][i] = 0.f;
      if (at >= cols) continue;
      load8<T>(x, at, cols, t[r]);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) sizes.bad = fmaf(t[r][i], 0.f, sizes.bad);
      if constexpr (kGated) {
        float u[kWidth];
        load8<T>(up, at, cols, u);
#pragma unroll
        for (int i = 0; i < kWidth; ++i) {
          sizes.bad = fmaf(u[i], 0.f, sizes.bad);
          sizes.large = fmaxf(sizes.large, fmaxf(fabsf(t[r][i]), fabsf(u[i])));
          t[r][i] = silu_mul_near(t[r][i], u[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < kWidth; ++i) sizes.top = fmaxf(sizes.top, fabsf(t[r][i]));
    }
    const float mine = sizes.top;
    sizes = over_row<kThreads>(sizes, shared + first_wave);
    const bool finite = sizes.bad == 0.f;
    // Values so large or small that f32 does not hold what the codes are made of: all in 64 bits.
    const bool wide = sizes.top < kTiny || (kGated && (sizes.large > kLarge || sizes.top < 1.f / kLarge));
    double top = sizes.top;
    auto exact = [&](int r, int i) -> double {
      if constexpr (kGated) {
        const int at = (r * kThreads + thread) * kWidth + i;
        return at < cols ? silu_mul_wide(T::widen(x[at]), T::widen(up[at])) : 0.0;
      } else {
        return (double)t[r][i];
      }
    };
    if constexpr (kGated) {
      // The largest in 64 bits is among those that are near the largest in 32.
      top = 0.0;
      const float from = wide ? -1.f : sizes.top * (1.f - 1.f / 262144);
      if (finite && mine >= from) {
#pragma unroll 1
        for (int at = thread * kWidth; at < cols; at += kThreads * kWidth)
          for (int i = 0; i < kWidth && at + i < cols; ++i) {
            const float g = T::widen(x[at + i]), u = T::widen(up[at + i]);
            if (fabsf(silu_mul_near(g, u)) >= from || wide) top = fmax(top, fabs(silu_mul_wide(g, u)));
          }
      }
      top = over_row<kThreads>(top, shared_top + first_wave);
    }
    const bool fits = finite && top <= 3.4028234663852886e38;
    const float inverse = fits && !wide ? 127.f / (float)top : 0.f;
    int8_t* q = (int8_t*)a.q + row * a.q_stride;
#pragma unroll
    for (int r = 0; r < kReps; ++r) {
      const int at = (r * kThreads + thread) * kWidth;
      if (at >= cols) continue;
      u32x2 w = {0, 0};
      if (fits && top > 0.0)
        w = codes8(t[r], inverse, top, wide ? 1.f : kGated ? kGatedSlack : kSlack, [&](int i) { return exact(r, i); });
      store_codes8(q, at, cols, w);
    }
    if (thread == 0) a.scale[row] = fits ? (float)(top / 127.0) : __builtin_nanf("");
  }
}

// Rows of a launch in workgroups of `block` threads, `rows` of them in each. (A grid's threads are
// counted in 32 bits.)
unsigned grid_of(int64_t rows, int rows_of_block, int block) {
  const int64_t blocks = ceil_div(rows, rows_of_block), most = 0xFFFFFFFFll / block;
  return (unsigned)(blocks < most ? blocks : most);
}

// Calls launch(threads, reps) with the shape that holds a row of `dim` elements.
template <typename Launch>
int with_row_shape(int64_t dim, Launch launch) {
#define UK_ROW_SHAPE(threads, reps) \
  if (dim <= (threads) * (reps) * kWidth) return launch(std::integral_constant<int, threads>(), std::integral_constant<int, reps>())
  UK_ROW_SHAPE(64, 1);
  UK_ROW_SHAPE(64, 2);
  UK_ROW_SHAPE(256, 1);
  UK_ROW_SHAPE(256, 2);
  UK_ROW_SHAPE(256, 4);
  UK_ROW_SHAPE(1024, 2);
  UK_ROW_SHAPE(1024, 4);
  UK_ROW_SHAPE(1024, 8);
#undef UK_ROW_SHAPE
  return fail(IREE_AMD_UK_STATUS_UNIMPLEMENTED, "rows of more than 65536 elements");
}

}  // namespace

int launch_rms_norm_quantize(const RmsNormQuantizeArgs& a, hipStream_t s) {
  return with_row_shape(a.dim, [&](auto threads, auto reps) {
    constexpr int kThreads = decltype(threads)::value, kReps = decltype(reps)::value;
    constexpr int kBlock = kThreads < 256 ? 256 : kThreads;
    const dim3 grid(grid_of(a.tokens, kBlock / kThreads, kBlock));
    if (a.bf16)
      hipLaunchKernelGGL((rms_norm_quantize_kernel<BF16, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    else
      hipLaunchKernelGGL((rms_norm_quantize_kernel<F16, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    return check_hip(hipGetLastError(), "rms_norm_quantize launch");
  });
}

int launch_quantize_rows(const QuantizeRowsArgs& a, hipStream_t s) {
  return with_row_shape(a.cols, [&](auto threads, auto reps) {
    constexpr int kThreads = decltype(threads)::value, kReps = decltype(reps)::value;
    constexpr int kBlock = kThreads < 256 ? 256 : kThreads;
    const dim3 grid(grid_of(a.rows, kBlock / kThreads, kBlock));
    if (a.bf16 && a.up)
      hipLaunchKernelGGL((quantize_rows_kernel<BF16, true, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    else if (a.bf16)
      hipLaunchKernelGGL((quantize_rows_kernel<BF16, false, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    else if (a.up)
      hipLaunchKernelGGL((quantize_rows_kernel<F16, true, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    else
      hipLaunchKernelGGL((quantize_rows_kernel<F16, false, kThreads, kReps>), grid, dim3(kBlock), 0, s, a);
    return check_hip(hipGetLastError(), "quantize_rows launch");
  });
}

}  // namespace uk
