// The products of rows of 8 bits with scales for each row and channel, over one matrix or over
// ragged groups of rows (uk_w8a8.hip, uk_w8a8_mfma.hip): arguments and what the kernels share.
#ifndef IREE_AMD_UK_W8A8_H_
#define IREE_AMD_UK_W8A8_H_

#include "uk_common.h"
#include "uk_mfma_cfg.h"

namespace uk {

struct W8A8Args {
  const char* lhs;
  int64_t lhs_stride, lhs_rows;        // bytes between rows
  const float* lhs_scale;
  const char* rhs;
  int64_t rhs_stride, rhs_expert;      // bytes between outer columns, between experts
  const float* rhs_scale;              // [experts][N]
  const float* bias;                   // [N] or null (one matrix only)
  char* out;
  int64_t out_stride, out_rows;        // elements between rows
  int64_t positions;                   // rows of one matrix; entries of the list of rows
  const int32_t* offsets;              // null: one matrix
  const int32_t* rows;
  int32_t rows_per_token;
  bool gather, scatter;
  int experts, N, K;
  int type;                            // of the result: 1 f16, 2 bf16, 3 f32
};

int launch_w8a8(const W8A8Args& a, hipStream_t s);
// Macro tiles (uk_w8a8_mfma.hip), by number.
constexpr int kW8A8Shapes = 5;
constexpr int kW8A8MfmaThreads = 256;
int launch_w8a8_mfma(const W8A8Args& a, int shape, hipStream_t s);
// Tiles of rows that there can be at most: of every expert that has any, the last is not full.
inline int64_t w8a8_row_tiles(const W8A8Args& a, int height) {
  if (!a.offsets) return ceil_div(a.positions, (int64_t)height);
  return a.positions / height + (a.experts < a.positions ? a.experts : a.positions);
}
// Workgroups of a call on tiles of that size.
inline int64_t w8a8_workgroups(const W8A8Args& a, int height, int width) {
  return w8a8_row_tiles(a, height) * ceil_div((int64_t)a.N, (int64_t)width);
}

namespace w8a8 {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A tile of rows: the positions [first, end) of `expert`, at most a tile's height of them used;
// expert < 0: there is no such tile.
struct RowTile { int expert; int64_t first, end; };

// Tile number `tile` of the rows of all experts, each expert's rows in tiles of `height`: the
// wave looks at 64 experts at a time.
__device__ __forceinline__ RowTile find_row_tile(const W8A8Args& a, int64_t tile, int height) {
  if (!a.offsets) {
    RowTile t = {0, tile * height, a.positions};
    if (t.first >= t.end) t.expert = -1;
    return t;
  }
  const int lane = threadIdx.x & 63, most = (int)a.positions;
  int before = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    const int e = e0 + lane;
    int begin = 0, end = 0;
    if (e < a.experts) {
      begin = a.offsets[e], end = a.offsets[e + 1];
      // (whatever the list holds, no place outside it is used)
      begin = begin < 0 ? 0 : begin;
      end = end > most ? most : end;
    }
    const int tiles = end > begin ? (int)(((uint32_t)(end - begin) + height - 1) / (uint32_t)height) : 0;
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    const uint64_t past = __ballot(before + sum > tile);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int first = __builtin_amdgcn_readlane(begin, l), its_end = __builtin_amdgcn_readlane(end, l);
      const int skipped = before + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l);
      const int64_t at = first + (tile - skipped) * height;
      // (counts of a list that falls may have wrapped around)
      if (at < first || at >= its_end) return {-1, 0, 0};
      return {e0 + l, at, its_end};
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return {-1, 0, 0};
}

// Row of the left-hand side at a position of the list, row of the result; -1: none.
__device__ __forceinline__ int64_t lhs_row(const W8A8Args& a, int64_t position) {
  if (!a.gather) return position < a.lhs_rows ? position : -1;
  const int32_t row = a.rows[position];
  return row >= 0 && row / a.rows_per_token < a.lhs_rows ? row / a.rows_per_token : -1;
}
__device__ __forceinline__ int64_t out_row(const W8A8Args& a, int64_t position) {
  const int64_t row = a.scatter ? a.rows[position] : position;
  return row >= 0 && row < a.out_rows ? row : -1;
}

// Four consecutive results of a row, in the type of the result, rounded once.
template <typename out_t>
__device__ __forceinline__ void store4(const W8A8Args& a, int64_t row, int col, const float* v) {
  typedef out_t out4_t __attribute__((ext_vector_type(4), aligned(sizeof(out_t))));
  out_t* dst = (out_t*)a.out + row * a.out_stride + col;
  out4_t x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (out_t)v[e];
  if (col + 4 <= a.N) {
    *(out4_t*)dst = x;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < a.N) dst[e] = x[e];
  }
}

// Scales (and what is added) of four consecutive channels, zeros past the last.
__device__ __forceinline__ floatx4 channels4(const float* of, int col, int N) {
  typedef float any4_t __attribute__((ext_vector_type(4), aligned(4)));
  if (col + 4 <= N) return *(const any4_t*)(of + col);
  floatx4 v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < N) v[e] = of[col + e];
  return v;
}

}  // namespace w8a8
}  // namespace uk

#endif  // IREE_AMD_UK_W8A8_H_
