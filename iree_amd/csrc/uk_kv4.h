// Layout of a block of the 4-bit cache (one kv head of one page, include/iree_amd_uk.h),
// and conversions between the rows' types and f32. Device code and sizes only.
#ifndef IREE_AMD_CSRC_UK_KV4_H_
#define IREE_AMD_CSRC_UK_KV4_H_

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace uk {
namespace kv4 {

// Byte offsets inside a block of `page` tokens of D values.
template <int D>
struct Block {
  __host__ __device__ static constexpr int64_t bytes(int page) { return (int64_t)page * (D + 8); }
  __device__ static int k_row(int row) { return row * (D / 2); }
  // The dword of V that holds d = 8 * i .. 8 * i + 7 of a row.
  __device__ static int v_dword(int page, int row, int i) {
    return page * (D / 2) + (((row >> 2) * (D / 8) + i) * 4 + (row & 3)) * 4;
  }
  __device__ static int k_params(int page, int row) { return page * D + row * 4; }
  __device__ static int v_params(int page, int row) { return page * (D + 4) + row * 4; }
};

// (Not HIP's structs of the same sizes: arrays of those do not stay in registers, and the
// compiler takes reads of them from LDS for possible readers of every load into LDS on its way.)
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

typedef float floatx2 __attribute__((ext_vector_type(2)));

// Row values as bits. (A value that comes from 64 bits is rounded from its 32: contracted, the
// two roundings would become one for f16 and not for bf16.)
struct F16 {
  __device__ static float widen(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }
  __device__ static uint32_t narrow2(float a, float b) {
#pragma clang fp contract(off)
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{a, b}), pair));
  }
};
struct BF16 {
  __device__ static float widen(uint32_t b) { return __builtin_bit_cast(float, b << 16); }
  __device__ static uint32_t narrow2(float a, float b) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{a, b}), pair));
  }
};

template <typename T>
__device__ inline void widen4(u32x2 w, float* x) {
  x[0] = T::widen(w.x & 0xFFFFu);
  x[1] = T::widen(w.x >> 16);
  x[2] = T::widen(w.y & 0xFFFFu);
  x[3] = T::widen(w.y >> 16);
}
template <typename T>
__device__ inline u32x2 narrow4(const float* x) {
  return u32x2{T::narrow2(x[0], x[1]), T::narrow2(x[2], x[3])};
}

}  // namespace kv4
}  // namespace uk

#endif  // IREE_AMD_CSRC_UK_KV4_H_
