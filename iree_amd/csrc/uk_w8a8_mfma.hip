// Products of rows of 8 bits with scales, many rows: macro tiles on v_mfma_i32_16x16x64_i8.
//
// A workgroup of four waves (2 x 2) owns a tile of 64 to 256 rows by 128 or 256 channels, a wave a
// quarter of it in registers, WM x WN blocks of 16 x 16. Steps of 64 bytes of K go from memory straight
// into a ring of slots in LDS, several steps ahead; a step's operands leave LDS while the step before
// is multiplied; one barrier a step, behind the first products of it, frees the slot that was read and
// publishes the next. A slot holds blocks of 16 rows or channels by 64 bytes, 1 KiB each. Of packed
// weights the lanes of a load fetch a block in the order in which the matrix cores take it. Of the
// row-major rows four lanes fetch the 64 bytes of one row, and the pieces of a row are turned by row /
// 4, so that the reads of 16 rows touch every bank alike.
//
// The weights are the instruction's first operand: a lane then holds four consecutive channels of one
// row. What lies past the end of K is zeros of the weights, whose descriptors end there.
//
// The rows of all experts are cut into tiles expert by expert; a workgroup finds its own from the offsets,
// 64 experts at a time. Consecutive workgroups go to the eight XCDs in turn; each XCD takes a contiguous part of
// the tiles, in panels of a few tiles of rows, so that the operands its tiles share are in its L2.
//
// 4096^3 with bf16 results 58.7 us (2.34 POP/s, one round of 128 x 256, two to a compute unit; 59.6 on 256 x 256), by
// expert 4096 tokens x 8 of 64 experts, 4096 -> 3584, 544 to 555 us: 1.75 POP/s, 2.0 with the rows that fill the last
// tile of each expert, which is what several rounds sustain (2048 x 14336 x 4096 116 us, 2.07 POP/s). A last tile of
// 256 rows worked on at half its height where that suffices took 550 us and is not kept. 500 x 4096 x
// 14336 takes 38.8 us on 256 workgroups of 64 x 128, whose 2.75 MB of operands each come in at 71 GB/s.
#include "uk_w8a8.h"

#include <type_traits>

namespace uk {
namespace {
using namespace w8a8;

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Share of `n` items that falls to slot `i` of `slots` when they are spread evenly.
constexpr int share(int n, int slots, int i) { return (i + 1) * n / slots - i * n / slots; }

// Pins the order of issue of one basic block: kMfma matrix instructions, the kReads LDS reads behind the
// first kReadMfma of them, the kLoads loads spread over all.
template <int kMfma, int kReadMfma, int kReads, int kLoads, int I = 0>
__device__ __forceinline__ void spread_issue() {
  if constexpr (I < kMfma) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (I < kReadMfma) {
      constexpr int d = share(kReads, kReadMfma, I);
      if constexpr (d > 0) __builtin_amdgcn_sched_group_barrier(0x100, d, 0);
    }
    constexpr int v = share(kLoads, kMfma, I);
    if constexpr (v > 0) __builtin_amdgcn_sched_group_barrier(0x020, v, 0);
    spread_issue<kMfma, kReadMfma, kReads, kLoads, I + 1>();
  }
}

struct MfmaTileArgs {
  W8A8Args a;
  int tiles_n, panel_rows;
};

// The tile of a workgroup: positions [first, end) of an expert, tile tn of the channels.
struct MacroTile { int expert, tn; int64_t first, end; };

__device__ __forceinline__ MacroTile find_macro_tile(const MfmaTileArgs& args, int height) {
  const W8A8Args& a = args.a;
  const int tiles_n = args.tiles_n, lane = threadIdx.x & 63;
  auto bounds = [&](int e, int* begin, int* end) {
    *begin = *end = 0;
    if (e < a.experts) {
      if (a.offsets) {
        // (whatever the list holds, no place outside it is used)
        *begin = a.offsets[e] < 0 ? 0 : a.offsets[e];
        *end = a.offsets[e + 1] > (int)a.positions ? (int)a.positions : a.offsets[e + 1];
      } else {
        *end = (int)a.positions;
      }
    }
  };
  auto row_tiles = [&](int begin, int end) {
    return end > begin ? (int)(((uint32_t)(end - begin) + height - 1) / (uint32_t)height) : 0;
  };
  // How many there are, and which of them is this workgroup's.
  int total = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    int begin, end;
    bounds(e0 + lane, &begin, &end);
    total += row_tiles(begin, end);
  }
#pragma unroll
  for (int mask = 1; mask < 64; mask *= 2) total += __shfl_xor(total, mask);
  const int64_t tiles = (int64_t)__builtin_amdgcn_readfirstlane(total) * tiles_n;
  const int xcd = (int)(blockIdx.x % 8), index = (int)(blockIdx.x / 8);
  const int64_t per = tiles / 8, rest = tiles % 8;
  if (index >= per + (xcd < rest ? 1 : 0)) return {-1, 0, 0, 0};
  const int64_t logical = xcd * per + (xcd < rest ? xcd : rest) + index;
  const int row_tile = (int)(logical / tiles_n);        // (the expert's panels reorder the rest below)
  int before = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    int begin, end;
    bounds(e0 + lane, &begin, &end);
    const int count = row_tiles(begin, end);
    int sum = count;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    const uint64_t past = __ballot(before + sum > row_tile);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int its_begin = __builtin_amdgcn_readlane(begin, l), its_end = __builtin_amdgcn_readlane(end, l);
      const int its_count = __builtin_amdgcn_readlane(count, l);
      const int skipped = before + __builtin_amdgcn_readlane(sum, l) - its_count;
      const int in_expert = (int)(logical - (int64_t)skipped * tiles_n);
      const int panel = in_expert / (args.panel_rows * tiles_n), first_row = panel * args.panel_rows;
      const int rows = its_count - first_row < args.panel_rows ? its_count - first_row : args.panel_rows;
      const int in_panel = in_expert - first_row * tiles_n;
      if (rows < 1 || in_panel < 0) return {-1, 0, 0, 0};
      const int64_t first = its_begin + (int64_t)(first_row + in_panel % rows) * height;
      // (counts of a list that falls may have wrapped around)
      if (first < its_begin || first >= its_end) return {-1, 0, 0, 0};
      return {e0 + l, in_panel / rows, first, its_end};
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return {-1, 0, 0, 0};
}

template <int WM, int WN, int kRing>
__device__ __forceinline__ void w8a8_mfma_body(const MfmaTileArgs& args) {
  const W8A8Args& a = args.a;
  constexpr int TM = 2 * WM, TN = 2 * WN;                    // blocks of 16 of the workgroup
  constexpr int kHeight = TM * 16;
  constexpr int kLhsLoads = TM / 4, kRhsLoads = TN / 4;      // blocks a wave brings in a step
  constexpr int kLoads = kLhsLoads + kRhsLoads, kFrags = WM + WN;
  constexpr int kLhsBytes = TM * 1024, kSlotBytes = (TM + TN) * 1024;
  // Matrix instructions of a step, of the part behind its barrier, and how many of these have reads
  // behind them: the last reads have to be back when the step ends.
  constexpr int kRest = (WN - 1) * WM;
  constexpr int kReadRest = kRest - (kRest >= 32 ? 16 : kRest / 2);
  static_assert(TM % 4 == 0 && TN % 4 == 0, "every wave brings in whole blocks");
  static_assert((kRing - 1) * kLoads < 64, "too many loads in flight for vmcnt");
  extern __shared__ __attribute__((aligned(1024))) char lds[];

  const int lane = threadIdx.x & 63, l16 = lane & 15, kc = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / 2, wn = wave % 2;
  const MacroTile tile = find_macro_tile(args, kHeight);
  if (tile.expert < 0) return;
  const int k_chunks = (a.K + 15) / 16;
  const int T = (k_chunks + 3) / 4;

  // ---- what this wave brings in ------------------------------------------------
  const int64_t base_row = a.gather ? 0 : tile.first;
  const int64_t rows_left = a.lhs_rows - base_row;
  const int64_t lhs_bytes = rows_left > 0 ? (rows_left - 1) * a.lhs_stride + k_chunks * 16 : 0;
  const __amdgpu_buffer_rsrc_t lhs_src = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.lhs + base_row * a.lhs_stride), 0, (int)(uint32_t)(lhs_bytes < 0xFFFFFFF0ll ? lhs_bytes : 0xFFFFFFF0ll),
      0x00020000);
  const int quad_row = lane >> 2, quad_chunk = ((lane & 3) - (lane >> 4)) & 3;
  uint32_t lhs_at[kLhsLoads], rhs_at[kRhsLoads];
#pragma unroll
  for (int r = 0; r < kLhsLoads; ++r) {
    // (rows that are not there are read from one that is, and not stored)
    const int64_t position = tile.first + (wave * kLhsLoads + r) * 16 + quad_row;
    int64_t row = position < tile.end ? lhs_row(a, position) : -1;
    row = row >= 0 ? row : base_row;
    lhs_at[r] = (uint32_t)((row - base_row) * a.lhs_stride) + quad_chunk * 16;
  }
  const int outer_cols = (a.N + 31) / 32;
  __amdgpu_buffer_rsrc_t rhs_src[kRhsLoads];
#pragma unroll
  for (int r = 0; r < kRhsLoads; ++r) {
    const int block = tile.tn * TN + wave * kRhsLoads + r, col = block / 2;
    rhs_src[r] = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(a.rhs + tile.expert * a.rhs_expert + (int64_t)(col < outer_cols ? col : 0) * a.rhs_stride), 0,
        col < outer_cols ? k_chunks * 512 : 0, 0x00020000);
    rhs_at[r] = block % 2 * 256 + l16 * 16 + kc * 512;
  }
  auto issue_one = [&](int step, int slot, int d) {
    char* base = lds + slot * kSlotBytes;
    if (d < kLhsLoads)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          lhs_src, (__attribute__((address_space(3))) void*)(base + (wave * kLhsLoads + d) * 1024), 16,
          lhs_at[d] + step * 64, 0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rhs_src[d - kLhsLoads],
          (__attribute__((address_space(3))) void*)(base + kLhsBytes + (wave * kRhsLoads + d - kLhsLoads) * 1024), 16,
          rhs_at[d - kLhsLoads] + step * 2048, 0, 0, 0);
  };
  // ---- the products ----------------------------------------------------------------
  intx4 acc[WM][WN];
  int4v fa[2][WM], fb[2][WN];
  const uint32_t lhs_read = l16 * 64 + ((kc + (l16 >> 2)) & 3) * 16;
  // (the rows first: the first products need all of them and one block of channels)
  auto read_one = [&](int slot, int r, int4v (&na)[WM], int4v (&nb)[WN]) {
    const char* base = lds + slot * kSlotBytes;
    if (r < WM) na[r] = *(const int4v*)(base + (wm * WM + r) * 1024 + lhs_read);
    else nb[r - WM] = *(const int4v*)(base + kLhsBytes + (wn * WN + r - WM) * 1024 + lane * 16);
  };
  auto multiply = [&](const int4v (&na)[WM], const int4v (&nb)[WN], int from, int to) {
#pragma unroll
    for (int y = 0; y < WN; ++y)
      if (y >= from && y < to) {
#pragma unroll
        for (int x = 0; x < WM; ++x) acc[x][y] = S8Cfg16::mfma(nb[y], na[x], acc[x][y]);
      }
  };
  auto clear = [&]() {
#pragma unroll
    for (int x = 0; x < WM; ++x)
#pragma unroll
      for (int y = 0; y < WN; ++y) {
        acc[x][y] = intx4{0, 0, 0, 0};
        // (The sums of the largest tile fill the accumulator half of the registers. The compiler, which knows
        // that they begin as zeros, mixes them with the operands' half and moves them to and fro in
        // the loop, 155 us instead of 55 at 4096^3; pinned here, they stay.)
        if constexpr (WM * WN == 64) asm volatile("" : "+a"(acc[x][y]));
      }
  };
  auto issue_step = [&](int s) {
#pragma unroll
    for (int d = 0; d < kLoads; ++d) issue_one(s, s, d);
  };
  auto rest_of_steps = [&](int done, int slot) {
#pragma unroll 1
    for (; done < T; ++done) {
#pragma unroll
      for (int r = 0; r < kFrags; ++r) read_one(slot, r, fa[0], fb[0]);
      multiply(fa[0], fb[0], 0, WN);
      slot = slot + 1 == kRing ? 0 : slot + 1;
    }
  };
  if (T > kRing) {
    int done = 0, slot = 0;                  // steps multiplied; slot of step `done`
    int next = kRing, next_slot = 0;         // step to load and its slot
#pragma unroll 1
    for (int s = 0; s < kRing; ++s) issue_step(s);
    clear();
    wait_vmcnt<(kRing - 1) * kLoads>();
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int r = 0; r < kFrags; ++r) read_one(0, r, fa[0], fb[0]);
    // Two steps a round, so that the registers of the operands return to their places.
    while (done + 2 <= T) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int read_slot = slot + 1 == kRing ? 0 : slot + 1;
        // (past the end the last step again, into a slot that nobody reads any more: as many loads in
        // flight as ever)
        const int load = next < T ? next : T - 1;
        __builtin_amdgcn_sched_barrier(0);
        multiply(fa[p], fb[p], 0, 1);
        __builtin_amdgcn_sched_barrier(0);
        // This step's operands are in registers, the next step's loads have landed: its slot is free, and
        // the next is readable by all. (A bare barrier: __syncthreads() would wait for every load.)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_vmcnt<(kRing - 2) * kLoads>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kRest; ++i) {
          if (i < kReadRest) {
#pragma unroll
            for (int r = i * kFrags / kReadRest; r < (i + 1) * kFrags / kReadRest; ++r)
              read_one(read_slot, r, fa[p ^ 1], fb[p ^ 1]);
          }
#pragma unroll
          for (int d = i * kLoads / kRest; d < (i + 1) * kLoads / kRest; ++d) issue_one(load, next_slot, d);
        }
        multiply(fa[p], fb[p], 1, WN);
        spread_issue<kRest, kReadRest, kFrags, kLoads>();
        __builtin_amdgcn_sched_barrier(0);
        ++next;
        next_slot = next_slot + 1 == kRing ? 0 : next_slot + 1;
        slot = read_slot;
      }
      done += 2;
    }
    // What is left is in its slots.
    wait_vmcnt<0>();
    __syncthreads();
    rest_of_steps(done, slot);
  } else {
#pragma unroll 1
    for (int s = 0; s < T; ++s) issue_step(s);
    clear();
    wait_vmcnt<0>();
    __syncthreads();
    rest_of_steps(0, 0);
  }

  // ---- the results: element e of block (x, y) is row l % 16, channel 4 (l / 16) + e ------
  const float* channels = a.rhs_scale + (int64_t)tile.expert * a.N;
  auto store = [&](auto zero) {
    typedef decltype(zero) out_t;
    const int col0 = (tile.tn * TN + wn * WN) * 16;
    floatx4 scale[WN], added[WN];
#pragma unroll
    for (int y = 0; y < WN; ++y) {
      scale[y] = channels4(channels, col0 + y * 16 + kc * 4, a.N);
      added[y] = a.bias ? channels4(a.bias, col0 + y * 16 + kc * 4, a.N) : floatx4{0, 0, 0, 0};
    }
#pragma unroll
    for (int x = 0; x < WM; ++x) {
      const int64_t position = tile.first + (wm * WM + x) * 16 + l16;
      int64_t from = -1, to = -1;
      if (position < tile.end) from = lhs_row(a, position), to = out_row(a, position);
      const bool exists = from >= 0 && to >= 0;
      const float row_scale = exists ? a.lhs_scale[from] : 0.f;
      out_t* dst = (out_t*)a.out + to * a.out_stride;
      if constexpr (sizeof(out_t) == 2) {
        // Two blocks side by side exchange lane rows, after which lane group g (of 16) has channels 8 (g
        // / 2) .. + 8 of block g % 2: one store of 16 bytes a lane for both.
        typedef out_t out2_t __attribute__((ext_vector_type(2)));
        typedef out_t out8_t __attribute__((ext_vector_type(8), aligned(2)));
#pragma unroll
        for (int y = 0; y < WN; y += 2) {
          uint32_t w[2][2];
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float v[2];
#pragma unroll
              for (int e = 0; e < 2; ++e)
                v[e] = fmaf((float)acc[x][y + b][2 * h + e] * row_scale, scale[y + b][2 * h + e], added[y + b][2 * h + e]);
              w[b][h] = __builtin_bit_cast(uint32_t, out2_t{(out_t)v[0], (out_t)v[1]});
            }
          const auto p = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
          const auto q = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
          const out8_t v8 = __builtin_bit_cast(out8_t, u32x4{(uint32_t)p[0], (uint32_t)q[0], (uint32_t)p[1], (uint32_t)q[1]});
          const int col = col0 + y * 16 + (lane >> 4 & 1) * 16 + (lane >> 5) * 8;
          if (exists) {
            if (col + 8 <= a.N) {
              *(out8_t*)(dst + col) = v8;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (col + e < a.N) dst[col + e] = v8[e];
            }
          }
        }
      } else {
#pragma unroll
        for (int y = 0; y < WN; ++y) {
          const int col = col0 + y * 16 + kc * 4;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf((float)acc[x][y][e] * row_scale, scale[y][e], added[y][e]);
          if (exists && col < a.N) store4<float>(a, to, col, v);
        }
      }
    }
  };
  if (a.type == 1) store((_Float16)0);
  else if (a.type == 2) store((__bf16)0);
  else store(0.f);
}

template <int WM, int WN, int kRing, int kOcc>
__global__ __launch_bounds__(kW8A8MfmaThreads, kOcc) void w8a8_mfma_kernel(MfmaTileArgs args) {
  w8a8_mfma_body<WM, WN, kRing>(args);
}

template <int WM, int WN, int kRing, int kOcc>
int launch_tile(const W8A8Args& a, hipStream_t s) {
  constexpr int lds_bytes = kRing * 2 * (WM + WN) * 1024;
  static_assert(lds_bytes * kOcc <= 160 * 1024, "the rings exceed a compute unit's LDS");
  auto kernel = w8a8_mfma_kernel<WM, WN, kRing, kOcc>;
  static PerDeviceOnce set_on;
  int dev = 0;
  UK_RETURN_IF_HIP(hipGetDevice(&dev));
  if (!set_on.done(dev)) {
    UK_RETURN_IF_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes));
    set_on.mark(dev);
  }
  const MfmaTileArgs args{a, (int)ceil_div((int64_t)a.N, (int64_t)WN * 32), WM < WN ? 8 : 4};
  note_kernel_path("w8a8:mfma");
  note_macro_tile(WM * 32, WN * 32, 1);
  hipLaunchKernelGGL(kernel, dim3((unsigned)w8a8_workgroups(a, WM * 32, WN * 32)), dim3(kW8A8MfmaThreads), lds_bytes, s, args);
  return check_hip(hipGetLastError(), "w8a8 launch");
}

}  // namespace

int launch_w8a8_mfma(const W8A8Args& a, int shape, hipStream_t s) {
  switch (shape) {
    case 0: return launch_tile<8, 8, 5, 1>(a, s);
    case 1: return launch_tile<4, 8, 3, 2>(a, s);
    case 2: return launch_tile<4, 4, 4, 2>(a, s);
    case 3: return launch_tile<2, 8, 4, 2>(a, s);
    default: return launch_tile<2, 4, 6, 2>(a, s);
  }
}

}  // namespace uk
