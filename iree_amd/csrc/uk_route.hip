// Each token's experts and their weights from its logits, and the tokens' slots in the order of
// their experts (include/iree_amd_uk.h).
//
// A wave chooses for a token: its lanes hold the logits as integers of the same order, and top_k times the
// largest is taken from the lowest expert that has it. The slots are then sorted by expert the way one digit of
// a radix sort is: blocks of consecutive tokens count their slots of every expert, and a slot's place
// is its expert's first place, plus the counts of the blocks and waves before, plus the lanes before it
// with the same expert. The order of no addition decides anything: the lists are the same on every call.
//
// Up to 128 tokens one workgroup does all; more take two launches, the counts of the blocks in the
// workspace between them. 32 tokens of 64 experts take 7.8 us in one launch, 8191 of 128 10.4 and 7.2 in two: top_k
// reductions one after the other and the barriers between the steps, and of 8191 tokens' 10.4 us 4.4, of their 7.2 2.8
// are vector instructions (617 a wave for two tokens and their counts). (A wave that chooses for one token at a time takes 14.5
// us instead of 10.4.)
//
// Both sides of the lines, calls of 8 experts a token, in us. One workgroup against two launches: 64 experts, 32 tokens 8.1 and 9.9,
// 64 12.5 and 9.9, 128 21.6 and 10.1; 256 experts, 32 tokens 13.9 and 15.4, 64 22.8 and 15.4, 128 40.7 and 16.0: two
// launches win from somewhere between 32 and 64 tokens on, so that calls of 64 to 128 cost more than need be, and more than
// one of 1000 (11.1 and 17.0). Blocks of 16 tokens at least: with 32 0.3 to 1 more (512 tokens of 64 experts 10.9 and 10.6), with 8
// 0.7 to 3 less up to 1024 tokens (512 of 64 experts 9.9 and 10.6, of 256 14.2 and 16.4) and 1.5 more for 16 tokens of 64,
// which are then two blocks. 256 blocks at most: 8191 tokens of 256 experts 22.1, with 128 28.7, with 512, whose counts every
// block reads, 42.6; 65536 of 64 experts 47.4, 85.0 and 43.8.
#include "uk_common.h"
#include "uk_kv4.h"

#include <type_traits>

namespace uk {
namespace {
using namespace kv4;

constexpr int kMostExperts = 512;
constexpr int kMostBlocks = 256;           // blocks of tokens
constexpr int kBlockTokens = 16;           // of one, at least
constexpr int kWaves = 16;                 // of a workgroup
constexpr int kHeldSlots = 8192;           // of a block whose choices stay in LDS
constexpr int kOneBlockTokens = 128;       // up to which one workgroup does all

struct RouteArgs {
  MoeRouteArgs r;
  int block_tokens, blocks;
  int32_t* counts;                         // [blocks][experts]
};

// Order of floats as that of integers; 0 for what is not chosen.
__device__ inline uint32_t order_of(float v) {
  if (!(v > -__builtin_inff())) return 0;                   // (-inf and NaN)
  v = fminf(v, 3.4028234663852886e38f) + 0.f;               // (+inf counts as the largest; -0 is 0)
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float value_of(uint32_t order) {
  return __builtin_bit_cast(float, order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

template <typename T>
__device__ inline float logit(const void* row, int e) {
  if constexpr (std::is_same<T, float>::value) return ((const float*)row)[e];
  else return T::widen(((const uint16_t*)row)[e]);
}

__device__ inline uint32_t largest_of_wave(uint32_t v) {
  auto with = [&](uint32_t o) { v = o > v ? o : v; };
  with((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));       // lane ^ 1, ^ 2, mirrors of 8 and 16
  with((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
  with((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));
  with((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));
  const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = p[0] > p[1] ? p[0] : p[1];
  const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = q[0] > q[1] ? q[0] : q[1];
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

// The experts and weights of two tokens, by a wave, whose steps wait for nothing of each other; the second may be
// past the last. kLogits: of a token, a lane's. `ids` (or null): the choices of the block's tokens from `first` on, in LDS.
template <typename T, int kLogits>
__device__ inline void choose(const MoeRouteArgs& a, const int64_t (&token)[2], int64_t last, int64_t first, int16_t* ids) {
  const int lane = threadIdx.x & 63;
  uint32_t order[2][kLogits];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const char* row = (const char*)a.logits + token[t] * a.logits_stride * (int64_t)(std::is_same<T, float>::value ? 4 : 2);
#pragma unroll
    for (int i = 0; i < kLogits; ++i) {
      const int e = i * 64 + lane;
      order[t][i] = e < a.experts && token[t] < last ? order_of(logit<T>(row, e)) : 0;
    }
  }
  float total[2] = {0.f, 0.f}, top[2] = {0.f, 0.f}, mine_logit[2] = {0.f, 0.f};
  int mine[2] = {-1, -1};
  if (!a.renormalize) {
    // (the sum's exponentials before any is taken)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t best = order[t][0];
#pragma unroll
      for (int i = 1; i < kLogits; ++i) best = order[t][i] > best ? order[t][i] : best;
      top[t] = value_of(largest_of_wave(best));
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kLogits; ++i)
        if (order[t][i]) sum += expf(value_of(order[t][i]) - top[t]);
#pragma unroll
      for (int mask = 32; mask; mask >>= 1) sum += __shfl_xor(sum, mask);
      total[t] = sum;
    }
  }
  for (int k = 0; k < a.top_k; ++k) {
    uint32_t best[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      best[t] = order[t][0];
#pragma unroll
      for (int i = 1; i < kLogits; ++i) best[t] = order[t][i] > best[t] ? order[t][i] : best[t];
    }
    best[0] = largest_of_wave(best[0]);
    best[1] = largest_of_wave(best[1]);
    if (!(best[0] | best[1])) break;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float its_logit = value_of(best[t]);
      if (k == 0) top[t] = its_logit;
      int e = best[t] ? -1 : -2;            // (-2: none is left)
#pragma unroll
      for (int i = 0; i < kLogits; ++i) {
        const uint64_t has = __ballot(order[t][i] == best[t]);
        if (e == -1 && has) {
          const int l = __builtin_ctzll(has);
          e = i * 64 + l;
          if (lane == l) order[t][i] = 0;
        }
      }
      if (lane == k && e >= 0) mine[t] = e, mine_logit[t] = its_logit;
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (token[t] >= last) continue;
    const float p = lane < a.top_k && mine[t] >= 0 ? expf(mine_logit[t] - top[t]) : 0.f;
    if (a.renormalize) {
      float sum = p;
#pragma unroll
      for (int mask = 32; mask; mask >>= 1) sum += __shfl_xor(sum, mask);
      total[t] = sum;
    }
    if (lane < a.top_k) {
      a.expert_ids[token[t] * a.top_k + lane] = mine[t];
      a.expert_weights[token[t] * a.top_k + lane] = mine[t] >= 0 ? p / total[t] : 0.f;
      if (ids) ids[(token[t] - first) * a.top_k + lane] = (int16_t)mine[t];
    }
  }
}

// Lanes that hold the same expert as this one.
__device__ inline uint64_t same_expert(int e, int bits) {
  uint64_t same = __ballot(e >= 0);
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot(e >> b & 1);
    same &= e >> b & 1 ? set : ~set;
  }
  return same;
}

// Slots of a block in the waves' shares of it, one after the other.
struct Share { uint32_t begin, end; };
template <int kWaves>
__device__ inline Share share_of_wave(uint32_t slots) {
  const uint32_t share = (uint32_t)ceil_div(ceil_div(slots, kWaves), 64) * 64;
  const uint32_t begin = min((threadIdx.x >> 6) * share, slots);
  return {begin, min(begin + share, slots)};
}

// Counts of the waves' shares, [waves][experts] in LDS, which is zeros. id(i): the expert of slot i of the block.
template <int kWaves, typename Id>
__device__ inline void count_shares(Share share, int experts, int* counts, Id id) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (uint32_t i = share.begin + lane; i < share.end; i += 64) {
    const int e = id(i);
    if (e >= 0) atomicAdd(&counts[wave * experts + e], 1);
  }
}

// Places of a block's slots: counts become the places of the waves' first slots, of which the block's begin at
// first[e].
template <int kWaves, typename Id>
__device__ inline void place(const MoeRouteArgs& a, int64_t first_slot, Share share, int* places, const int* first, Id id) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, experts = a.experts;
  for (int e = threadIdx.x; e < experts; e += kWaves * 64) {
    int at = first[e];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int n = places[w * experts + e];
      places[w * experts + e] = at;
      at += n;
    }
  }
  __syncthreads();
  const int bits = 32 - __builtin_clz(experts | 1);
  for (uint32_t i = share.begin; i < share.end; i += 64) {
    const int e = i + lane < share.end ? id(i + lane) : -1;
    const uint64_t same = same_expert(e, bits);
    const int before = __popcll(same & ((1ull << lane) - 1));
    int at = 0;
    if (e >= 0) at = places[wave * experts + e] + before;
    __builtin_amdgcn_wave_barrier();
    if (e >= 0) {
      if (before == 0) places[wave * experts + e] = at + __popcll(same);
      a.rows[at] = (int32_t)(first_slot + i + lane);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Turns the counts of all experts into the place of the first slot of each, in LDS, by one wave, 64
// experts at a time; returns how many slots there are (in that wave).
__device__ inline int first_places(int* count, int experts) {
  const int lane = threadIdx.x & 63;
  int at = 0;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = e0 + lane, n = e < experts ? count[e] : 0;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    if (e < experts) count[e] = at + sum - n;
    at += __shfl(sum, 63);
  }
  return at;
}

// kAll: one workgroup does all. Else only the choices and the counts of a block.
template <typename T, int kLogits, bool kAll>
__global__ __launch_bounds__(kWaves * 64) void moe_route_kernel(RouteArgs args) {
  constexpr int kThreads = kWaves * 64;
  const MoeRouteArgs& a = args.r;
  extern __shared__ int memory[];            // counts [waves][experts], (kAll) of all [experts]
  __shared__ int16_t ids[kHeldSlots];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), experts = a.experts;
  const int64_t first = (int64_t)blockIdx.x * args.block_tokens;
  const int64_t last = min(first + args.block_tokens, a.tokens);
  const int64_t first_slot = first * a.top_k;
  const uint32_t slots = (uint32_t)((last - first) * a.top_k);      // (below 2^31)
  const bool held = slots <= kHeldSlots;     // (without its workspace one block may have any number of tokens)
  for (int i = threadIdx.x; i < kWaves * experts; i += kThreads) memory[i] = 0;
  for (int64_t token = first + wave; token < last; token += 2 * kWaves)
    choose<T, kLogits>(a, {token, token + kWaves}, last, first, held ? ids : nullptr);
  __syncthreads();                           // (the choices are read below, by other waves of the workgroup)
  const Share share = share_of_wave<kWaves>(slots);
  auto id = [&](uint32_t i) { return held ? (int)ids[i] : a.expert_ids[first_slot + i]; };
  count_shares<kWaves>(share, experts, memory, id);
  __syncthreads();
  int* const count = memory + kWaves * experts;
  for (int e = threadIdx.x; e < experts; e += kThreads) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += memory[w * experts + e];
    if constexpr (kAll) count[e] = sum;
    else args.counts[(int64_t)blockIdx.x * experts + e] = sum;
  }
  if constexpr (kAll) {
    __shared__ int all;
    __syncthreads();
    if (wave == 0) {
      const int n = first_places(count, experts);
      if (threadIdx.x == 0) all = n;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kThreads) a.offsets[e] = count[e];
    if (threadIdx.x == 0) a.offsets[experts] = all;
    for (int64_t i = all + threadIdx.x; i < slots; i += kThreads) a.rows[i] = -1;
    place<kWaves>(a, 0, share, memory, count, id);
  }
}

// Second launch: a block's slots to their places.
__global__ __launch_bounds__(kWaves * 64) void moe_route_place_kernel(RouteArgs args) {
  constexpr int kThreads = kWaves * 64;
  const MoeRouteArgs& a = args.r;
  extern __shared__ int memory[];            // counts [waves][experts], then of all and of the blocks before
  const int experts = a.experts;
  int* const first = memory + kWaves * experts;
  int* const before = first + experts;
  __shared__ int all;
  for (int i = threadIdx.x; i < (kWaves + 2) * experts; i += kThreads) memory[i] = 0;
  const int64_t first_token = (int64_t)blockIdx.x * args.block_tokens, first_slot = first_token * a.top_k;
  const uint32_t slots = (uint32_t)(min((int64_t)args.block_tokens, a.tokens - first_token) * a.top_k);
  const Share share = share_of_wave<kWaves>(slots);
  auto id = [&](uint32_t i) { return a.expert_ids[first_slot + i]; };
  __syncthreads();
  count_shares<kWaves>(share, experts, memory, id);
  // (experts side by side, and as many parts of the blocks as there are threads for)
  const int width = experts <= 64 ? 64 : experts <= 128 ? 128 : experts <= 256 ? 256 : 512;
  const int parts = kThreads / width, e = threadIdx.x % width;
  if (e < experts) {
    int mine = 0, total = 0;
#pragma unroll 8
    for (int b = threadIdx.x / width; b < args.blocks; b += parts) {
      const int n = args.counts[(int64_t)b * experts + e];
      mine += b < (int)blockIdx.x ? n : 0;
      total += n;
    }
    atomicAdd(&first[e], total);
    atomicAdd(&before[e], mine);
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int n = first_places(first, experts);
    if (threadIdx.x == 0) all = n;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < experts; i += kThreads) a.offsets[i] = first[i];
    if (threadIdx.x == 0) a.offsets[experts] = all;
  }
  for (int64_t i = all + (int64_t)blockIdx.x * kThreads + threadIdx.x; i < a.tokens * a.top_k;
       i += (int64_t)args.blocks * kThreads)
    a.rows[i] = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < experts; i += kThreads) first[i] += before[i];
  __syncthreads();
  place<kWaves>(a, first_slot, share, memory, first, id);
}

template <typename T, int kLogits>
int launch_choose(const RouteArgs& args, hipStream_t s) {
  const int experts = args.r.experts;
  if (args.blocks == 1)
    hipLaunchKernelGGL((moe_route_kernel<T, kLogits, true>), dim3(1), dim3(kWaves * 64), (kWaves + 1) * experts * 4, s, args);
  else
    hipLaunchKernelGGL((moe_route_kernel<T, kLogits, false>), dim3((unsigned)args.blocks), dim3(kWaves * 64),
                       kWaves * experts * 4, s, args);
  return check_hip(hipGetLastError(), "moe_route launch");
}

template <typename T>
int launch_type(const RouteArgs& args, hipStream_t s) {
  const int experts = args.r.experts;
  if (experts <= 64) return launch_choose<T, 1>(args, s);
  if (experts <= 128) return launch_choose<T, 2>(args, s);
  if (experts <= 256) return launch_choose<T, 4>(args, s);
  return launch_choose<T, kMostExperts / 64>(args, s);
}

// Blocks of tokens of a call that has the workspace.
int64_t route_blocks(int64_t tokens, int64_t* block_tokens) {
  *block_tokens = tokens;
  if (tokens <= kOneBlockTokens) return 1;
  *block_tokens = ceil_div(ceil_div(tokens, kMostBlocks), kBlockTokens) * kBlockTokens;
  return ceil_div(tokens, *block_tokens);
}

}  // namespace

uint64_t moe_route_workspace(int64_t tokens, int experts) {
  int64_t block_tokens;
  const int64_t blocks = route_blocks(tokens, &block_tokens);
  return blocks > 1 ? (uint64_t)blocks * experts * 4 : 0;
}

int launch_moe_route(const MoeRouteArgs& a, hipStream_t s) {
  RouteArgs args{a, 0, 1, (int32_t*)a.workspace};
  int64_t block_tokens, blocks = route_blocks(a.tokens, &block_tokens);
  if (blocks > 1 && a.workspace_bytes < moe_route_workspace(a.tokens, a.experts)) blocks = 1, block_tokens = a.tokens;
  args.block_tokens = (int)block_tokens;
  args.blocks = (int)blocks;
  int st = a.type == 3 ? launch_type<float>(args, s) : a.type == 2 ? launch_type<BF16>(args, s) : launch_type<F16>(args, s);
  if (st || blocks == 1) return st;
  hipLaunchKernelGGL(moe_route_place_kernel, dim3((unsigned)blocks), dim3(kWaves * 64), (kWaves + 2) * a.experts * 4, s, args);
  return check_hip(hipGetLastError(), "moe_route launch");
}

}  // namespace uk
