// Head norms with position rotation, rows into and out of the 4-bit cache, and copies of
// its pages (include/iree_amd_uk.h has the formulas and the layout).
//
// All four are bound by memory, or for a few tokens by the launch.
#include "uk_common.h"
#include "uk_kv4.h"

namespace uk {
namespace {
using namespace kv4;

constexpr int kBlock = 256;

// ---------------------------------------------------------------------------
// qk_norm_rope
// ---------------------------------------------------------------------------

// Sums and extrema over the L = D / 8 lanes that hold a row.
template <int L>
__device__ inline double row_sum(double v) {
  for (int m = 1; m < L; m *= 2) v += __shfl_xor(v, m);
  return v;
}
template <int L>
__device__ inline float row_min(float v) {
  for (int m = 1; m < L; m *= 2) v = fminf(v, __shfl_xor(v, m));
  return v;
}
template <int L>
__device__ inline float row_max(float v) {
  for (int m = 1; m < L; m *= 2) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

struct Params {
  uint32_t bits;     // scale and offset, f16 each
  uint32_t code[8];
};

// Codes of a row, 8 values a lane. A code is decided on x - offset against (code +- 1/2)
// scale, both exact in 64 bits, so that ties go to the even code and a value next to a
// border falls on its own side, whatever the estimate in 32 bits said.
template <int L>
__device__ inline Params quantise(const float* x) {
  float lo = x[0], hi = x[0];
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    finite = finite && fabsf(x[i]) < INFINITY;
  }
  lo = row_min<L>(lo);
  hi = row_max<L>(hi);
  const float bad = row_max<L>(finite ? 0.f : 1.f);
  const _Float16 offset = (_Float16)fminf(fmaxf(lo, -65504.f), 65504.f);
  const double range = (double)hi - (double)lo;
  const _Float16 step = (_Float16)fminf((float)(range / 15.0), 65504.f);
  Params p;
  const float s = (float)step, m = (float)offset, inv = s > 0.f ? 1.f / s : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float c = fminf(fmaxf(rintf((x[i] - m) * inv), 0.f), 15.f);
    const double rest = fma(-(double)c, (double)s, (double)x[i] - (double)m), half = 0.5 * (double)s;
    const bool odd = ((int)c & 1) != 0;
    if (rest > half || (rest == half && odd)) c += 1.f;
    if (rest < -half || (rest == -half && odd)) c -= 1.f;
    p.code[i] = s > 0.f && bad == 0.f ? (uint32_t)fminf(fmaxf(c, 0.f), 15.f) : 0u;
  }
  p.bits = bad == 0.f ? (uint32_t)__builtin_bit_cast(uint16_t, step) |
                            ((uint32_t)__builtin_bit_cast(uint16_t, offset) << 16)
                      : 0x00007E00u;   // scale NaN, offset 0
  return p;
}

// A group of L lanes takes `kRows` consecutive head rows of one token (query heads, then
// key heads, then value heads), so that it reads the token's cosines once. A lane holds two
// runs of four values: of a rotated row d = 4 i .. and rotary / 2 + 4 i .., the two halves
// of its pairs, so that the rotation needs no exchange between lanes; else d = 8 i .. + 8.
// Norm and rotation run in 64 bits: with a cache, the key is about to be compared with the
// borders between its codes, and the vector unit has the time (the launch is bound by
// memory either way).
template <int D, typename T, int kRows>
__global__ __launch_bounds__(kBlock) void qk_norm_rope_kernel(QkNormRopeArgs a, int q_rows, int k_rows, int rows,
                                                              int chunks) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x % L;
  const int64_t group = (int64_t)blockIdx.x * (kBlock / L) + threadIdx.x / L;
  const int64_t token = group / chunks;
  if (token >= a.tokens) return;
  const int first = (int)(group % chunks) * kRows;
  float cs[8];
  if (a.cos_sin) {
    const int64_t position = a.positions[token];
    if (position < 0 || position >= a.table_rows) return;
    if (lane < a.rotary / 8) {
      const float* at = a.cos_sin + position * a.rotary + lane * 4;
      *(float4*)cs = *(const float4*)at;
      const float* sin_at = at + a.rotary / 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) cs[4 + i] = sin_at[i];
    }
  }
  const bool turns = a.cos_sin && lane < a.rotary / 8;
  const bool halves = turns && !a.interleaved;
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int row = first + j;
    if (row >= rows) return;
    const bool is_q = row < q_rows, is_k = !is_q && row < q_rows + k_rows;
    const int head = is_q ? row : is_k ? row - q_rows : row - q_rows - k_rows;
    const uint16_t* src = is_q  ? (const uint16_t*)a.q + token * a.q_stride
                          : is_k ? (const uint16_t*)a.k + token * a.k_stride
                                 : (const uint16_t*)a.v + token * a.v_stride;
    src += (int64_t)head * D;
    const int d0 = halves && (is_q || is_k) ? lane * 4 : lane * 8;
    const int d1 = halves && (is_q || is_k) ? a.rotary / 2 + lane * 4 : lane * 8 + 4;
    float x[8];
    widen4<T>(*(const uint2*)(src + d0), x);
    widen4<T>(*(const uint2*)(src + d1), x + 4);
    if (is_q || is_k) {
      double y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i];
      const uint16_t* weight = (const uint16_t*)(is_q ? a.q_weight : a.k_weight);
      if (weight) {
        double sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fma(y[i], y[i], sum);
        sum = row_sum<L>(sum);
        const double r = 1.0 / sqrt(sum / D + (double)a.eps);
        float w[8];
        widen4<T>(*(const uint2*)(weight + d0), w);
        widen4<T>(*(const uint2*)(weight + d1), w + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * r * (double)w[i];
      }
      if (turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = a.interleaved ? 2 * i : i, q = a.interleaved ? 2 * i + 1 : i + 4;
          const double c = cs[i], s = cs[4 + i], u = y[p], v = y[q];
          y[p] = u * c - v * s;
          y[q] = v * c + u * s;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)y[i];
      const uint2 r0 = narrow4<T>(x), r1 = narrow4<T>(x + 4);
      uint16_t* dst = is_q     ? (uint16_t*)a.q_out + token * a.q_out_stride
                      : a.k_out ? (uint16_t*)a.k_out + token * a.k_out_stride
                                : nullptr;
      if (dst) {
        *(uint2*)(dst + (int64_t)head * D + d0) = r0;
        *(uint2*)(dst + (int64_t)head * D + d1) = r1;
      }
      widen4<T>(r0, x);
      widen4<T>(r1, x + 4);
    }
    if (is_q || !a.pool.base) continue;
    const int64_t slot = a.slots[token];
    const int page = 1 << a.pool.page_shift, at = (int)(slot & (page - 1));
    const Params p = quantise<L>(x);
    if (slot < 0 || (slot >> a.pool.page_shift) >= a.pool.pages) continue;
    char* block = a.pool.base + (slot >> a.pool.page_shift) * a.pool.page_stride + head * Block<D>::bytes(page);
    uint32_t low = 0, high = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      low |= p.code[i] << (4 * i);
      high |= p.code[4 + i] << (4 * i);
    }
    if (is_k) {
      *(uint16_t*)(block + Block<D>::k_row(at) + d0 / 2) = (uint16_t)low;
      *(uint16_t*)(block + Block<D>::k_row(at) + d1 / 2) = (uint16_t)high;
      if (lane == 0) *(uint32_t*)(block + Block<D>::k_params(page, at)) = p.bits;
    } else {
      *(uint32_t*)(block + Block<D>::v_dword(page, at, lane)) = low | (high << 16);
      if (lane == 0) *(uint32_t*)(block + Block<D>::v_params(page, at)) = p.bits;
    }
  }
}

template <int D, typename T, int kRows>
int launch_rows(const QkNormRopeArgs& a, hipStream_t s) {
  const int q_rows = a.q ? a.heads : 0, k_rows = a.k ? a.kv_heads : 0;
  const int rows = q_rows + k_rows + (a.pool.base ? a.kv_heads : 0);
  const int chunks = (int)ceil_div(rows, kRows);
  const int64_t blocks = ceil_div(a.tokens * chunks, kBlock / (D / 8));
  if (blocks > 0x7FFFFFFF) return fail(IREE_AMD_UK_STATUS_INVALID_ARGUMENT, "qk_norm_rope: too many rows for one call");
  hipLaunchKernelGGL((qk_norm_rope_kernel<D, T, kRows>), dim3((unsigned)blocks), dim3(kBlock), 0, s, a, q_rows, k_rows,
                     rows, chunks);
  return check_hip(hipGetLastError(), "qk_norm_rope");
}

template <int D, typename T>
int launch_dim(const QkNormRopeArgs& a, hipStream_t s) {
  // Few tokens want every row in flight at once; many want the cosines read once.
  return a.tokens >= 512 ? launch_rows<D, T, 4>(a, s) : launch_rows<D, T, 1>(a, s);
}

// ---------------------------------------------------------------------------
// kv4_read
// ---------------------------------------------------------------------------

// A group of D / 8 lanes reads one K row and the V row of the same head.
template <int D, typename T>
__global__ __launch_bounds__(kBlock) void kv4_read_kernel(Kv4ReadArgs a) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x % L;
  const int64_t group = (int64_t)blockIdx.x * (kBlock / L) + threadIdx.x / L;
  const int64_t row = group / a.kv_heads;
  if (row >= a.rows) return;
  const int head = (int)(group % a.kv_heads);
  const int64_t slot = a.slots[row];
  if (slot < 0 || (slot >> a.pool.page_shift) >= a.pool.pages) return;
  const int page = 1 << a.pool.page_shift, at = (int)(slot & (page - 1));
  const char* block = a.pool.base + (slot >> a.pool.page_shift) * a.pool.page_stride + head * Block<D>::bytes(page);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    uint16_t* out = (uint16_t*)(which ? a.v_out : a.k_out);
    if (!out) continue;
    const uint32_t codes = *(const uint32_t*)(block + (which ? Block<D>::v_dword(page, at, lane)
                                                             : Block<D>::k_row(at) + lane * 4));
    const uint32_t bits = *(const uint32_t*)(block + (which ? Block<D>::v_params(page, at)
                                                            : Block<D>::k_params(page, at)));
    const float s = F16::widen(bits & 0xFFFFu), m = F16::widen(bits >> 16);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((codes >> (4 * i)) & 15u), s, m);
    const uint2 r0 = narrow4<T>(x), r1 = narrow4<T>(x + 4);
    out += row * (which ? a.v_out_stride : a.k_out_stride) + (int64_t)head * D + lane * 8;
    *(uint4*)out = make_uint4(r0.x, r0.y, r1.x, r1.y);
  }
}

template <int D, typename T>
int launch_read(const Kv4ReadArgs& a, hipStream_t s) {
  const int64_t blocks = ceil_div(a.rows * a.kv_heads, kBlock / (D / 8));
  if (blocks > 0x7FFFFFFF) return fail(IREE_AMD_UK_STATUS_INVALID_ARGUMENT, "kv4_read: too many rows for one call");
  hipLaunchKernelGGL((kv4_read_kernel<D, T>), dim3((unsigned)blocks), dim3(kBlock), 0, s, a);
  return check_hip(hipGetLastError(), "kv4_read");
}

// ---------------------------------------------------------------------------
// copy_pages
// ---------------------------------------------------------------------------

// The page numbers travel as kernel arguments: nothing has to be copied to the device
// first, and a captured launch keeps them.
constexpr int kPairs = 384;
struct PagePairs {
  int32_t src[kPairs], dst[kPairs];
};

// A workgroup copies kBlock * kCopies * 16 bytes of one page.
constexpr int kCopies = 4;
__global__ __launch_bounds__(kBlock) void copy_pages_kernel(char* pool, int64_t chunks, int64_t stride, PagePairs pairs) {
  const uint4* src = (const uint4*)(pool + pairs.src[blockIdx.y] * stride);
  uint4* dst = (uint4*)(pool + pairs.dst[blockIdx.y] * stride);
  const int64_t at = (int64_t)blockIdx.x * (kBlock * kCopies) + threadIdx.x;
  uint4 v[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i)
    if (at + i * kBlock < chunks) v[i] = src[at + i * kBlock];
#pragma unroll
  for (int i = 0; i < kCopies; ++i)
    if (at + i * kBlock < chunks) dst[at + i * kBlock] = v[i];
}

}  // namespace

int launch_qk_norm_rope(const QkNormRopeArgs& a, hipStream_t s) {
  switch (a.dim) {
    case 64: return a.bf16 ? launch_dim<64, BF16>(a, s) : launch_dim<64, F16>(a, s);
    case 128: return a.bf16 ? launch_dim<128, BF16>(a, s) : launch_dim<128, F16>(a, s);
    default: return a.bf16 ? launch_dim<256, BF16>(a, s) : launch_dim<256, F16>(a, s);
  }
}

int launch_kv4_read(const Kv4ReadArgs& a, hipStream_t s) {
  switch (a.dim) {
    case 64: return a.bf16 ? launch_read<64, BF16>(a, s) : launch_read<64, F16>(a, s);
    case 128: return a.bf16 ? launch_read<128, BF16>(a, s) : launch_read<128, F16>(a, s);
    default: return a.bf16 ? launch_read<256, BF16>(a, s) : launch_read<256, F16>(a, s);
  }
}

int launch_copy_pages(void* pool, int64_t page_bytes, int64_t page_stride, const int32_t* src, const int32_t* dst,
                      int64_t count, hipStream_t s) {
  const int64_t chunks = page_bytes / 16;
  const int64_t blocks = ceil_div(chunks, kBlock * kCopies);
  if (blocks > 0x7FFFFFFF) return fail(IREE_AMD_UK_STATUS_INVALID_ARGUMENT, "copy_pages: a page too large for one launch");
  for (int64_t at = 0; at < count; at += kPairs) {
    PagePairs pairs;
    const int n = (int)(count - at < kPairs ? count - at : kPairs);
    for (int i = 0; i < kPairs; ++i) {
      pairs.src[i] = i < n ? src[at + i] : 0;
      pairs.dst[i] = i < n ? dst[at + i] : 0;
    }
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)blocks, (unsigned)n), dim3(kBlock), 0, s, (char*)pool, chunks,
                       page_stride, pairs);
    UK_RETURN_IF_HIP(hipGetLastError());
  }
  return 0;
}

}  // namespace uk
