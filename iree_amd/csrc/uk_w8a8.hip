// Products of rows of 8 bits with a scale for each row and each channel: few rows, and the choice
// between the kernels (include/iree_amd_uk.h has the formulas).
//
// A workgroup owns 16 to 64 rows by 16 to 64 channels; its eight waves deal K among them in pairs of
// 64-byte steps and their sums meet in LDS. Weights go from memory straight into the registers that
// feed the matrix cores (packed tiles are in operand order); rows, which lie one after the other,
// come through the wave's own part of LDS, a quad of lanes fetching the 64 bytes of one row. The sums
// are integers, so the order of their additions cannot show.
//
// One row against 4096 -> 14336 is a stream of 58.7 MB of weights: 11.0 us, 5.4 TB/s (a pass that only reads 117 MB
// reaches 6.7).
#include "uk_w8a8.h"

#include <cmath>
#include <type_traits>

namespace uk {
namespace {
using namespace w8a8;

constexpr int kWaves = 8;
constexpr uint32_t kNowhere = 0xFFFFFFFFu;     // past the end of every descriptor: the load gives zeros

template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// MB x NB blocks of 16 x 16 results per workgroup; D steps of 64 bytes of K in flight per wave.
template <int MB, int NB, int D>
__device__ __forceinline__ void w8a8_few_rows_body(const W8A8Args& a, int tiles_n) {
  constexpr int F = MB * NB;
  static_assert(D % 2 == 0, "steps come in pairs");
  constexpr int kRingBytes = D * MB * 1024;                 // of a wave
  constexpr int kSharedBytes = kWaves * (kRingBytes > F * 1024 ? kRingBytes : F * 1024);
  __shared__ __attribute__((aligned(1024))) char shared[kSharedBytes];
  intx4 (*const sums)[F][64] = (intx4 (*)[F][64])shared;
  const int lane = threadIdx.x & 63, l16 = lane & 15, kc = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (the row tiles of one column tile lie tiles_n workgroups apart: on the same XCD where that is whole 8s)
  const int64_t row_tile = blockIdx.x / tiles_n;
  const int tn = blockIdx.x % tiles_n;
  const RowTile tile = find_row_tile(a, row_tile, MB * 16);
  if (tile.expert < 0) return;
  const int k_chunks = (a.K + 15) / 16;
  // ---- where this lane's pieces of the operands lie --------------------------
  const int64_t first_row = a.gather ? 0 : tile.first;
  const int64_t rows_left = a.lhs_rows - first_row;
  int64_t lhs_bytes = rows_left > 0 ? (rows_left - 1) * a.lhs_stride + k_chunks * 16 : 0;
  lhs_bytes = lhs_bytes < 0xFFFFFFF0ll ? lhs_bytes : 0xFFFFFFF0ll;
  const __amdgpu_buffer_rsrc_t lhs_src = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.lhs + first_row * a.lhs_stride), 0, (int)(uint32_t)lhs_bytes, 0x00020000);
  const int first_col = tn * NB / 2, outer_cols = (a.N + 31) / 32;           // (outer ones)
  const int64_t rhs_bytes = (int64_t)(outer_cols - 1 - first_col) * a.rhs_stride + k_chunks * 512;
  const __amdgpu_buffer_rsrc_t rhs_src = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.rhs + tile.expert * a.rhs_expert + first_col * a.rhs_stride), 0,
      (int)(uint32_t)(rhs_bytes < 0xFFFFFFF0ll ? rhs_bytes : 0xFFFFFFF0ll), 0x00020000);
  const int lhs_r = lane >> 2, lhs_c = ((lane & 3) - (lane >> 4)) & 3;
  uint32_t lhs_at[MB], rhs_at[NB];
#pragma unroll
  for (int x = 0; x < MB; ++x) {
    const int64_t position = tile.first + x * 16 + lhs_r;
    const int64_t row = position < tile.end ? lhs_row(a, position) : -1;
    lhs_at[x] = row >= 0 ? (uint32_t)((row - first_row) * a.lhs_stride) + lhs_c * 16 : kNowhere;
  }
#pragma unroll
  for (int y = 0; y < NB; ++y) {
    const int block = tn * NB + y, col = block / 2;
    rhs_at[y] = col < outer_cols ? (uint32_t)((col - first_col) * a.rhs_stride) + block % 2 * 256 + l16 * 16 + kc * 512
                                 : kNowhere;
  }
  // ---- the products ----------------------------------------------------------
  const int groups = (k_chunks + 4 * kWaves * D - 1) / (4 * kWaves * D);
  intx4 acc[MB][NB];
#pragma unroll
  for (int x = 0; x < MB; ++x)
#pragma unroll
    for (int y = 0; y < NB; ++y) acc[x][y] = intx4{0, 0, 0, 0};
  u32x4 fa[2][MB], fb[D][NB];
  char* const ring = shared + wave * kRingBytes;
  auto load = [&](int group, int d) {
    const int step = ((group * (D / 2) + d / 2) * kWaves + wave) * 2 + d % 2;
    const bool lhs_exists = step * 4 + lhs_c < k_chunks, rhs_exists = step * 4 + kc < k_chunks;
#pragma unroll
    for (int x = 0; x < MB; ++x)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          lhs_src, (__attribute__((address_space(3))) void*)(ring + (d * MB + x) * 1024), 16,
          lhs_exists && lhs_at[x] != kNowhere ? lhs_at[x] + step * 64 : kNowhere, 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);     // (the order that `read` counts on)
#pragma unroll
    for (int y = 0; y < NB; ++y)
      fb[d][y] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                     rhs_src, rhs_exists && rhs_at[y] != kNowhere ? rhs_at[y] + step * 2048 : kNowhere, 0, 0));
    __builtin_amdgcn_sched_barrier(0);
  };
  // the blocks of step d from LDS; `behind`: loads issued after theirs
  auto read = [&](int d, auto behind) {
    wait_loads<decltype(behind)::value>();
#pragma unroll
    for (int x = 0; x < MB; ++x)
      fa[d % 2][x] = *(const u32x4*)(ring + (d * MB + x) * 1024 + l16 * 64 + ((kc + (l16 >> 2)) & 3) * 16);
  };
  auto multiply = [&](int d) {
#pragma unroll
    for (int x = 0; x < MB; ++x)
#pragma unroll
      for (int y = 0; y < NB; ++y)
        acc[x][y] = S8Cfg16::mfma(__builtin_bit_cast(int4v, fb[d][y]), __builtin_bit_cast(int4v, fa[d % 2][x]), acc[x][y]);
  };
  typedef std::integral_constant<int, NB + (D - 1) * (MB + NB)> AllButOne;
  typedef std::integral_constant<int, NB + (D - 2) * (MB + NB)> AllButTwo;
#pragma unroll
  for (int d = 0; d < D; ++d) load(0, d);
  __builtin_amdgcn_sched_barrier(0);
  read(0, AllButOne());
#pragma unroll 1
  for (int g = 1; g < groups; ++g) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      // (the next step's blocks leave LDS while this one's are multiplied)
      __builtin_amdgcn_sched_barrier(0);
      read((d + 1) % D, AllButTwo());
      multiply(d);
      __builtin_amdgcn_sched_barrier(0);
      load(g, d);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int d = 0; d < D; ++d) {
    if (d + 1 < D) read(d + 1, std::integral_constant<int, 0>());
    multiply(d);
  }
  __syncthreads();     // (the sums take the place of the rings)
  // ---- the waves' sums, and the results ---------------------------------------
#pragma unroll
  for (int x = 0; x < MB; ++x)
#pragma unroll
    for (int y = 0; y < NB; ++y) sums[wave][x * NB + y][lane] = acc[x][y];
  __syncthreads();
  // Element e of lane l: row l % 16 of the block, channel 4 (l / 16) + e.
#pragma unroll
  for (int f0 = 0; f0 < F; f0 += kWaves) {
    const int f = f0 + wave;
    if (f >= F) break;
    const int x = f / NB, y = f % NB;
    const int64_t position = tile.first + x * 16 + l16;
    const int col = (tn * NB + y) * 16 + kc * 4;
    if (position >= tile.end || col >= a.N) continue;
    const int64_t from = lhs_row(a, position), to = out_row(a, position);
    if (from < 0 || to < 0) continue;
    intx4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += sums[w][f][lane];
    const float scale = a.lhs_scale[from];
    const floatx4 channel = channels4(a.rhs_scale + (int64_t)tile.expert * a.N, col, a.N);
    const floatx4 added = a.bias ? channels4(a.bias, col, a.N) : floatx4{0, 0, 0, 0};
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf((float)sum[e] * scale, channel[e], added[e]);
    if (a.type == 1) store4<_Float16>(a, to, col, v);
    else if (a.type == 2) store4<__bf16>(a, to, col, v);
    else store4<float>(a, to, col, v);
  }
}

template <int MB, int NB, int D, int kOcc>
__global__ __launch_bounds__(kWaves * 64, kOcc) void w8a8_few_rows_kernel(W8A8Args a, int tiles_n) {
  w8a8_few_rows_body<MB, NB, D>(a, tiles_n);
}

// Tiles of both kernels: rows, channels, workgroups that a compute unit holds, and the estimated time in us of a
// call on them (estimate_us below).
struct Tile {
  int rows, cols, resident;
  float call, round, round_k, last, last_k, last_busy, last_more, last_two, weights, results, grouped, empty;
};
constexpr int kFewRowsTiles = 4;
constexpr Tile kTile[] = {
    {16, 16, 2, 4.143f, 1.805f, 0.7211f, 0.f, 0.1075f, 0.2474f, 0.5751f, 0.1138f, 0.0083f, 0.8617f, 0.1784f, 1.735f},
    {16, 32, 3, 4.036f, 1.694f, 1.679f, 0.f, 0.2252f, 0.3195f, 2.144f, 0.2949f, 0.0336f, 2.011f, 0.2491f, 2.421f},
    {32, 32, 2, 0.f, 1.126f, 1.907f, 4.011f, 0.3567f, 0.6245f, 0.5663f, 0.5877f, 0.0024f, 0.8203f, 0.1823f, 2.864f},
    {64, 64, 1, 1.141f, 1.179f, 2.323f, 3.293f, 0.9435f, 1.231f, 0.f, 0.f, 0.0064f, 1.174f, 0.2325f, 6.05f},
    {256, 256, 1, 9.399f, 1.559f, 11.91f, 0.f, 9.164f, 0.9042f, 0.f, 0.f, 0.0165f, 0.3693f, 0.f, 15.56f},
    {128, 256, 2, 7.456f, 0.2931f, 13.33f, 0.f, 4.775f, 0.845f, 3.996f, 4.356f, 0.0598f, 0.231f, 0.f, 5.972f},
    {128, 128, 2, 5.658f, 0.0885f, 8.541f, 0.f, 3.24f, 0.4588f, 2.626f, 2.666f, 0.0372f, 0.2887f, 0.f, 4.465f},
    {64, 256, 2, 0.f, 1.831f, 8.642f, 6.502f, 2.956f, 0.7383f, 2.982f, 3.023f, 0.0813f, 0.1775f, 0.f, 3.544f},
    {64, 128, 2, 0.f, 1.266f, 5.003f, 4.913f, 2.127f, 0.0007f, 1.69f, 2.067f, 0.0717f, 0.2717f, 0.109f, 2.562f}};
constexpr int kTiles = sizeof(kTile) / sizeof(kTile[0]);
static_assert(kTiles == kFewRowsTiles + kW8A8Shapes, "a tile for each kernel");

// Workgroups run in rounds of as many as are resident, each `round` plus round_k per KB of K. The last round
// takes `last`, and per KB of K last_k, last_busy times the share of compute units that have a workgroup, and where
// some have more last_two and last_more times how many more. `weights` and `results` are per MB; groups add `grouped` for finding a
// tile and `empty` per 1000 workgroups of the grid. How the rows are dealt to the experts only the device knows:
// as if each position's expert were drawn at random, an expert with rows has a tile that is half full.
// Fitted (non-negative least squares, errors relative to the time) to the times of every tile on 1305 problems: 1 to 16384
// rows or tokens, 64 to 16384 channels and K, matrices and groups of 8 to 256 experts. On the 1340 others of
// profiles/w8a8_tiles.txt what it picks is 1.0 % from the best tile on average for one matrix and 1.9 % for groups, in the 95th
// percentile 8 and 11 %. (Of the floor the best tile itself may be far: 1.3 to 4 times, by the same record.)
double estimate_us(const W8A8Args& a, const Tile& t, int cus) {
  const double P = (double)a.positions, width = (double)ceil_div((int64_t)a.N, (int64_t)t.cols);
  double experts = 1.0, row_tiles = (double)ceil_div(a.positions, (int64_t)t.rows), us = t.call;
  if (a.offsets) {
    experts = a.experts * (1.0 - std::exp(-P / a.experts));
    const double tiles = P / experts / t.rows + 0.45;
    row_tiles = experts * (tiles > 1.0 ? tiles : 1.0);
    us += t.grouped + t.empty * 1e-3 * width * w8a8_row_tiles(a, t.rows);
  }
  const double slots = (double)cus * t.resident, kb = ceil_div(a.K, 64) / 16.0, workgroups = row_tiles * width;
  const double rounds = std::floor(workgroups / slots), rest = (workgroups - rounds * slots) / cus;
  us += rounds * (t.round + t.round_k * kb);
  if (rest > 0)
    us += t.last + kb * (t.last_k + t.last_busy * (rest < 1.0 ? rest : 1.0) +
                         (rest > 1.0 ? t.last_two + t.last_more * (rest - 1.0) / t.resident : 0.0));
  return us + t.weights * 1e-6 * experts * a.N * a.K + t.results * 1e-6 * P * a.N * (a.type == 3 ? 4 : 2);
}

int launch_few_rows(const W8A8Args& a, int v, hipStream_t s) {
  void (*kernel)(W8A8Args, int) = nullptr;
  switch (v) {
    case 0: kernel = w8a8_few_rows_kernel<1, 1, 8, 4>; break;
    case 1: kernel = w8a8_few_rows_kernel<1, 2, 6, 4>; break;
    case 2: kernel = w8a8_few_rows_kernel<2, 2, 4, 4>; break;
    default: kernel = w8a8_few_rows_kernel<4, 4, 2, 2>; break;
  }
  const int64_t tiles_n = ceil_div((int64_t)a.N, (int64_t)kTile[v].cols);
  note_kernel_path("w8a8:few-rows");
  note_macro_tile(kTile[v].rows, kTile[v].cols, 1);
  hipLaunchKernelGGL(kernel, dim3((unsigned)w8a8_workgroups(a, kTile[v].rows, kTile[v].cols)), dim3(kWaves * 64), 0,
                     s, a, (int)tiles_n);
  return check_hip(hipGetLastError(), "w8a8 launch");
}

}  // namespace

int launch_w8a8(const W8A8Args& a, hipStream_t s) {
  const int cus = device_cu_count();
  int best = -1;
  double least = INFINITY;
  for (int v = 0; v < kTiles; ++v) {
    // (a grid's threads are counted in 32 bits)
    const int64_t most = 0xFFFFFFFFll / (v < kFewRowsTiles ? kWaves * 64 : kW8A8MfmaThreads);
    if (w8a8_workgroups(a, kTile[v].rows, kTile[v].cols) > most) continue;
    const double us = estimate_us(a, kTile[v], cus);
    if (us < least) least = us, best = v;
  }
  if (best < 0) return fail(IREE_AMD_UK_STATUS_UNIMPLEMENTED, "w8a8: too many tiles for one call");
  return best < kFewRowsTiles ? launch_few_rows(a, best, s) : launch_w8a8_mfma(a, best - kFewRowsTiles, s);
}

}  // namespace uk
