// Head norms with position rotation, rows into and out of the 4-bit cache, and copies of
// its pages (include/iree_amd_uk.h has the formulas and the layout).
//
// Norms and rotation, rows back out and copies are bound by memory, or for a few tokens by the launch:
// 4099 tokens with 32 + 8 heads of 128, 85 MB, in 17.5 us (4.8 TB/s), one token in 2.5; 8191 tokens back
// out of the cache, 42 MB, in 10, of which 6.5 are HBM at a copy's rate and 2.4 what a launch of a few rows
// takes. Norms with values and the cache are bound by memory and by the vector unit: 8191 tokens, 181 MB
// (written to the byte what is kept: 76 MB), in 46 us, of HBM 28 and of 16300 vector instructions a
// vector unit 27, 56 % of which are the stored third of the rows: keys in 64 bits, codes.
#include "uk_common.h"
#include "uk_kv4.h"

#include <type_traits>

namespace uk {
namespace {
using namespace kv4;

constexpr int kBlock = 256;
constexpr int64_t kMostBlocks = 0xFFFFFFFFll / kBlock;      // a grid's threads are counted in 32 bits

// ---------------------------------------------------------------------------
// qk_norm_rope
// ---------------------------------------------------------------------------

// A value of the lane at the other end of one step of a reduction over L lanes: within 16 lanes
// through the vector unit's own exchange (lane ^ 1, lane ^ 2, the mirrors of 8 and of 16), the
// last step of 32 lanes through LDS.
template <int kStep>
__device__ inline float other_lane(float v) {
  if constexpr (kStep == 4) {
    return __shfl_xor(v, 16);
  } else {
    constexpr int control = kStep == 0 ? 0xB1 : kStep == 1 ? 0x4E : kStep == 2 ? 0x141 : 0x140;
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), control, 0xF, 0xF, true));
  }
}
template <int kStep>
__device__ inline double other_lane(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const float lo = other_lane<kStep>(__builtin_bit_cast(float, (uint32_t)u));
  const float hi = other_lane<kStep>(__builtin_bit_cast(float, (uint32_t)(u >> 32)));
  return __builtin_bit_cast(double, (uint64_t)__builtin_bit_cast(uint32_t, lo) |
                                        ((uint64_t)__builtin_bit_cast(uint32_t, hi) << 32));
}
// f over the L = 8, 16 or 32 lanes of a row, the same in all of them.
template <int L, typename V, typename F>
__device__ inline V over_row(V v, F f) {
  v = f(v, other_lane<0>(v));
  v = f(v, other_lane<1>(v));
  v = f(v, other_lane<2>(v));
  if constexpr (L > 8) v = f(v, other_lane<3>(v));
  if constexpr (L > 16) v = f(v, other_lane<4>(v));
  return v;
}

struct Params {
  uint32_t bits;         // scale and offset, f16 each
  uint32_t low, high;    // codes of a lane's first and last four values
};

// Codes of a row, 8 values a lane. An estimate in f32 is off by less than 2^-17 of a code; where a
// value lies within 2^-15 of a border between two codes (one wave in fifty has one, if values
// are not on a lattice), all are decided by comparing x - offset with (code +- 1/2) scale in 64
// bits, which is exact, ties to the even code.
template <int L>
__device__ inline Params quantise(const float* x) {
  float lo = x[0], hi = x[0], size = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    size = fmaf(x[i], 0.f, size);            // 0, or NaN where a value is not finite
  }
  lo = over_row<L>(lo, [](float a, float b) { return fminf(a, b); });
  hi = over_row<L>(hi, [](float a, float b) { return fmaxf(a, b); });
  const float bad = over_row<L>(size == 0.f ? 0.f : 1.f, [](float a, float b) { return fmaxf(a, b); });
  const _Float16 offset = (_Float16)fminf(fmaxf(lo, -65504.f), 65504.f);
  // (the quotient by 15, correctly rounded: a product with the reciprocal and one correction)
  const double range = (double)hi - (double)lo, q = range * (1.0 / 15.0);
  const _Float16 step = (_Float16)fminf((float)fma(fma(-15.0, q, range), 1.0 / 15.0, q), 65504.f);
  Params p;
  const float s = (float)step, m = (float)offset, inv = s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;
  float c[8], gap = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = (x[i] - m) * inv;
    c[i] = rintf(t);
    gap = fmaxf(gap, fabsf(t - c[i]));
    c[i] = __builtin_amdgcn_fmed3f(c[i], 0.f, 15.f);
  }
  if (gap > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double rest = fma(-(double)c[i], (double)s, (double)x[i] - (double)m), half = 0.5 * (double)s;
      const bool odd = ((int)c[i] & 1) != 0;
      const float up = rest > half || (rest == half && odd) ? 1.f : 0.f;
      const float down = rest < -half || (rest == -half && odd) ? 1.f : 0.f;
      c[i] = __builtin_amdgcn_fmed3f(c[i] + up - down, 0.f, 15.f);
    }
  }
  const bool stored = s > 0.f && bad == 0.f;
  p.low = p.high = 0;
  if (stored) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p.low |= (uint32_t)c[i] << (4 * i);
      p.high |= (uint32_t)c[4 + i] << (4 * i);
    }
  }
  p.bits = bad == 0.f ? (uint32_t)__builtin_bit_cast(uint16_t, step) |
                            ((uint32_t)__builtin_bit_cast(uint16_t, offset) << 16)
                      : 0x00007E00u;   // scale NaN, offset 0
  return p;
}

__device__ inline float inverse_root(float v) { return rsqrtf(v); }
__device__ inline double inverse_root(double v) { return 1.0 / sqrt(v); }

// Rows of many tokens leave past the caches, which they would fill (67 MB of queries 26 us,
// through them 34); those of a few stay for the attention that reads them next.
template <bool kPast>
__device__ inline void store(u32x2* to, u32x2 v) {
  if constexpr (kPast) __builtin_nontemporal_store(v, to);
  else *to = v;
}

enum RowKind { kQuery, kKey, kCachedKey, kValue };

// A group of L lanes takes kRows consecutive head rows of one token, so that it reads the token's
// cosines once, and has all of their loads in flight. A lane holds two runs of four values: of a
// rotated row d = 4 i .. and rotary / 2 + 4 i .., the two halves of its pairs, so that the rotation
// needs no exchange between lanes; else d = 8 i .. + 8. Norm and rotation run in f32, in 64 bits for
// a key that goes into the cache: it is about to be compared with the borders between its codes, and
// which side of one it falls on should not depend on an order of additions.
template <int D, typename T, RowKind kKind, int kRows>
__device__ inline void rows_body(const QkNormRopeArgs& a, int64_t block) {
  constexpr int L = D / 8;
  typedef typename std::conditional<kKind == kCachedKey, double, float>::type Wide;
  constexpr bool kTurned = kKind != kValue, kStored = kKind == kCachedKey || kKind == kValue;
  const int heads = kKind == kQuery ? a.heads : a.kv_heads;
  const int chunks = (heads + kRows - 1) / kRows;
  const int lane = threadIdx.x % L;
  const int64_t group = block * (kBlock / L) + threadIdx.x / L;
  const int64_t token = group / chunks;
  if (token >= a.tokens) return;
  const int first = (int)(group - token * chunks) * kRows;
  const bool lane_turns = kTurned && a.cos_sin && lane < a.rotary / 8;
  const bool halves = lane_turns && !a.interleaved;
  const int d0 = halves ? lane * 4 : lane * 8, d1 = halves ? a.rotary / 2 + lane * 4 : lane * 8 + 4;
  const uint16_t* src = kKind == kQuery   ? (const uint16_t*)a.q + token * a.q_stride
                        : kKind == kValue ? (const uint16_t*)a.v + token * a.v_stride
                                          : (const uint16_t*)a.k + token * a.k_stride;
  u32x2 raw[kRows][2];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int head = first + j < heads ? first + j : heads - 1;
    raw[j][0] = *(const u32x2*)(src + (int64_t)head * D + d0);
    raw[j][1] = *(const u32x2*)(src + (int64_t)head * D + d1);
  }
  float cs[8];
  if (a.cos_sin) {
    const int64_t position = a.positions[token];
    if (position < 0 || position >= a.table_rows) return;
    if (lane_turns) {
      const float* at = a.cos_sin + position * a.rotary + lane * 4;
      *(float4*)cs = *(const float4*)at;
      const float* sin_at = at + a.rotary / 2;
      *(float4*)(cs + 4) = *(const float4*)sin_at;
    }
  }
  const uint16_t* weight = kTurned ? (const uint16_t*)(kKind == kQuery ? a.q_weight : a.k_weight) : nullptr;
  float w[8];
  if (weight) {
    widen4<T>(*(const u32x2*)(weight + d0), w);
    widen4<T>(*(const u32x2*)(weight + d1), w + 4);
  }
  int64_t slot = 0;
  if (kStored) slot = a.slots[token];
  const int page = 1 << a.pool.page_shift, at = (int)(slot & (page - 1));
  const bool exists = slot >= 0 && (slot >> a.pool.page_shift) < a.pool.pages;
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int head = first + j;
    if (head >= heads) return;
    float x[8];
    widen4<T>(raw[j][0], x);
    widen4<T>(raw[j][1], x + 4);
    if constexpr (kTurned) {
      Wide y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i];
      if (weight) {
        Wide sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = y[i] * y[i] + sum;
        sum = over_row<L>(sum, [](Wide u, Wide v) { return u + v; });
        const Wide r = inverse_root(sum * (Wide)(1.0 / D) + (Wide)a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * r * (Wide)w[i];
      }
      if (lane_turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Wide c = cs[i], s = cs[4 + i];
          if (a.interleaved) {
            const Wide u = y[2 * i], v = y[2 * i + 1];
            y[2 * i] = u * c - v * s;
            y[2 * i + 1] = v * c + u * s;
          } else {
            const Wide u = y[i], v = y[i + 4];
            y[i] = u * c - v * s;
            y[i + 4] = v * c + u * s;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)y[i];
      const u32x2 r0 = narrow4<T>(x), r1 = narrow4<T>(x + 4);
      uint16_t* dst = kKind == kQuery ? (uint16_t*)a.q_out + token * a.q_out_stride
                      : a.k_out       ? (uint16_t*)a.k_out + token * a.k_out_stride
                                      : nullptr;
      if (dst) {
        store<(kRows > 1)>((u32x2*)(dst + (int64_t)head * D + d0), r0);
        store<(kRows > 1)>((u32x2*)(dst + (int64_t)head * D + d1), r1);
      }
      widen4<T>(r0, x);
      widen4<T>(r1, x + 4);
    }
    if constexpr (kStored) {
      const Params p = quantise<L>(x);
      if (!exists) continue;
      char* to = a.pool.base + (slot >> a.pool.page_shift) * a.pool.page_stride + head * Block<D>::bytes(page);
      if (kKind == kCachedKey) {
        *(uint16_t*)(to + Block<D>::k_row(at) + d0 / 2) = (uint16_t)p.low;
        *(uint16_t*)(to + Block<D>::k_row(at) + d1 / 2) = (uint16_t)p.high;
        if (lane == 0) *(uint32_t*)(to + Block<D>::k_params(page, at)) = p.bits;
      } else {
        *(uint32_t*)(to + Block<D>::v_dword(page, at, lane)) = p.low | (p.high << 16);
        if (lane == 0) *(uint32_t*)(to + Block<D>::v_params(page, at)) = p.bits;
      }
    }
  }
}

// The first q_blocks workgroups take queries, the next k_blocks keys, the others values.
template <int D, typename T, int kRows>
__global__ __launch_bounds__(kBlock) void qk_norm_rope_kernel(QkNormRopeArgs a, int64_t q_blocks, int64_t k_blocks) {
  const int64_t block = blockIdx.x;
  if (block < q_blocks) rows_body<D, T, kQuery, kRows>(a, block);
  else if (block >= q_blocks + k_blocks) rows_body<D, T, kValue, kRows>(a, block - q_blocks - k_blocks);
  else if (a.pool.base) rows_body<D, T, kCachedKey, kRows>(a, block - q_blocks);
  else rows_body<D, T, kKey, kRows>(a, block - q_blocks);
}

template <int D, typename T, int kRows>
int launch_rows(const QkNormRopeArgs& a, hipStream_t s) {
  constexpr int kGroups = kBlock / (D / 8);
  const int64_t q_blocks = a.q ? ceil_div(a.tokens * ceil_div(a.heads, kRows), kGroups) : 0;
  const int64_t kv_blocks = ceil_div(a.tokens * ceil_div(a.kv_heads, kRows), kGroups);
  const int64_t blocks = q_blocks + (a.k ? kv_blocks : 0) + (a.pool.base ? kv_blocks : 0);
  if (blocks > kMostBlocks) return fail(IREE_AMD_UK_STATUS_INVALID_ARGUMENT, "qk_norm_rope: too many rows for one call");
  hipLaunchKernelGGL((qk_norm_rope_kernel<D, T, kRows>), dim3((unsigned)blocks), dim3(kBlock), 0, s, a, q_blocks,
                     a.k ? kv_blocks : 0);
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
    const u32x2 r0 = narrow4<T>(x), r1 = narrow4<T>(x + 4);
    out += row * (which ? a.v_out_stride : a.k_out_stride) + (int64_t)head * D + lane * 8;
    *(u32x4*)out = u32x4{r0.x, r0.y, r1.x, r1.y};
  }
}

template <int D, typename T>
int launch_read(const Kv4ReadArgs& a, hipStream_t s) {
  const int64_t blocks = ceil_div(a.rows * a.kv_heads, kBlock / (D / 8));
  if (blocks > kMostBlocks) return fail(IREE_AMD_UK_STATUS_INVALID_ARGUMENT, "kv4_read: too many rows for one call");
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

// A workgroup copies kBlock * kCopies * 16 bytes of one page, past the caches: 600 pages of 544 KiB
// in 125 us (5.3 TB/s), through them 135, with four pieces to a thread 131.
constexpr int kCopies = 2;
__global__ __launch_bounds__(kBlock) void copy_pages_kernel(char* pool, int64_t chunks, int64_t stride, PagePairs pairs) {
  const u32x4* src = (const u32x4*)(pool + pairs.src[blockIdx.y] * stride);
  u32x4* dst = (u32x4*)(pool + pairs.dst[blockIdx.y] * stride);
  const int64_t at = (int64_t)blockIdx.x * (kBlock * kCopies) + threadIdx.x;
  u32x4 v[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i)
    if (at + i * kBlock < chunks) v[i] = __builtin_nontemporal_load(src + at + i * kBlock);
#pragma unroll
  for (int i = 0; i < kCopies; ++i)
    if (at + i * kBlock < chunks) __builtin_nontemporal_store(v[i], dst + at + i * kBlock);
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
  if (blocks > kMostBlocks) return fail(IREE_AMD_UK_STATUS_INVALID_ARGUMENT, "copy_pages: a page too large for one launch");
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
