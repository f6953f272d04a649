// Attention over the paged 4-bit cache (include/iree_amd_uk.h has the formula and the
// layout of a block).
//
// With codes c, scale s and offset m of a key's rows, a query q and G query heads to a kv
// head:
//   q . k = s_k (q . c_k) + m_k sum(q)
//   sum_j p_j v_j = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (m_j + 8 s_j)
// so the matrix cores multiply the codes themselves, which f16 holds exactly, and each
// key costs two multiply-adds for its scale and offset instead of a dequantised row. The
// codes of V are centred, because the sum over a long sequence is small next to its parts
// and the matrix cores cut off what does not fit the sum: 131072 keys, 6.4e-4 of the result
// with codes from 0, 2.1e-4 (the result's own rounding) with these.
#include "uk_common.h"
#include "uk_kv4.h"
#include "uk_mfma_cfg.h"

#include <type_traits>

namespace uk {
namespace {
using namespace kv4;

constexpr float kLog2e = 1.4426950408889634f;

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
__device__ inline half2v as_half2(uint32_t u) { return __builtin_bit_cast(half2v, u); }

// Where a workgroup's rows stand. Rows r of a sequence are its query tokens times the G
// heads of one kv head, token by token. Tiles of R rows are numbered over the batch: number b
// < batch is the first tile of sequence b (a decode step has no others), the numbers from
// batch on are the sequences' further tiles.
struct Rows {
  int b;             // sequence, -1: none
  int first;         // first row of the tile
  int count;         // rows of the sequence
  int tokens;        // its query tokens
  int token0;        // its first token
  int kv_len;
  int64_t slot;
};

// Of up to 64 sequences the further tiles stand one after the other, as a sum over 64 lanes
// finds them. Of more, sequence b's begin at floor(q_starts[b] G / R), which leaves room for
// all before it, and the last sequence that begins at or before a number is the one to have it:
// 64 lanes look for it at 64 sequences at a time. (Numbers without rows cost more than their own
// start: workgroups go to the parts of the device in turn, and with every second number empty half of it
// stays idle: 16 sequences of 128 rows on 16384 keys in four splits, with one f16 a weight, 414 us, so 241.)
__device__ inline Rows find_rows(const AttentionKv4Args& a, int64_t slot, int G, int R) {
  const int lane = threadIdx.x & 63;
  const int64_t further = slot - a.batch;
  int64_t b = slot, tile = 0;
  if (further >= 0) {
    int64_t lo = 0, n = a.batch;                    // candidates [lo, lo + n)
    while (n > 64) {
      const int64_t step = (n + 63) / 64;
      const int64_t at = lo + lane * step;
      const uint64_t yes = __ballot(at < lo + n && (int64_t)a.q_starts[at < lo + n ? at : lo] * G / R <= further);
      const int64_t from = lo + (yes ? 63 - __builtin_clzll(yes) : 0) * step;
      n = from + step < lo + n ? step : lo + n - from;
      lo = from;
    }
    const int64_t at = lo + (lane < n ? lane : n - 1);
    const int64_t start = a.q_starts[at];
    int64_t before = start * G / R;
    if (a.batch <= 64) {
      const int64_t rows = (a.q_starts[at + 1] - start) * G;
      const int mine = lane < n && rows > 0 ? (int)((rows - 1) / R) : 0;
      int sum = mine;
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const int other = __shfl_up(sum, m);
        sum += lane >= m ? other : 0;
      }
      before = sum - mine;
    }
    const uint64_t yes = __ballot(lane < n && before <= further);
    const int last = yes ? 63 - __builtin_clzll(yes) : 0;
    b = lo + last;
    tile = further - __builtin_amdgcn_readlane((int)before, last) + 1;
  }
  b = __builtin_amdgcn_readfirstlane((int)b);
  const int from = a.q_starts[b], to = a.q_starts[b + 1];
  const int64_t first = tile * R, rows = ((int64_t)to - from) * G;
  const bool mine = from >= 0 && to <= a.tokens && first >= 0 && first < rows;
  // (the same in all lanes, which the compiler is told: all addresses follow from them)
  Rows r;
  r.b = __builtin_amdgcn_readfirstlane(mine ? (int)b : -1);
  r.first = __builtin_amdgcn_readfirstlane((int)first);
  r.count = __builtin_amdgcn_readfirstlane((int)rows);
  r.tokens = __builtin_amdgcn_readfirstlane(to - from);
  r.token0 = __builtin_amdgcn_readfirstlane(from);
  r.kv_len = __builtin_amdgcn_readfirstlane(a.kv_lens[b]);
  r.slot = slot;
  return r;
}

// Position of a query token: below 0 where it sees nothing.
__device__ inline int position(const Rows& r, int token) {
  const int64_t p = (int64_t)r.kv_len - r.tokens + token;
  return p < 0 ? -1 : (int)p;
}

// The keys that rows at positions lo_pos..hi_pos see, in tiles of kKeys: the sinks, then
// the window (or everything).
template <int kKeys>
struct Keys {
  int sink_tiles, first, total;
  __device__ Keys(const AttentionKv4Args& a, int lo_pos, int hi_pos) {
    const int64_t capacity = a.max_pages << a.pool.page_shift;
    const int64_t end = hi_pos + 1 < capacity ? hi_pos + 1 : capacity;
    const int64_t begin = a.window && lo_pos + 1 > a.window ? lo_pos + 1 - a.window : 0;
    const int64_t last = (end + kKeys - 1) / kKeys;
    const int64_t sinks = a.sinks < end ? a.sinks : end;
    first = (int)(begin / kKeys);
    const int64_t st = (sinks + kKeys - 1) / kKeys;
    sink_tiles = (int)(st < first ? st : first);
    total = end <= 0 || a.pool.pages == 0 ? 0 : sink_tiles + (int)(last > first ? last - first : 0);
  }
  __device__ int key(int tile) const { return (tile < sink_tiles ? tile : first + tile - sink_tiles) * kKeys; }
};

__device__ inline float max4(float a, float b, float c, float d) { return fmaxf(fmaxf(a, b), fmaxf(c, d)); }
// Over 16 lanes next to each other.
template <int kControl>
__device__ inline float dpp_max(float v) {
  const int other = __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), kControl, 0xF, 0xF, true);
  return fmaxf(v, __builtin_bit_cast(float, other));
}
__device__ inline float row16_max(float v) {
  v = dpp_max<0xB1>(v);            // lane ^ 1
  v = dpp_max<0x4E>(v);            // lane ^ 2
  v = dpp_max<0x141>(v);           // the other half of 8, mirrored
  return dpp_max<0x140>(v);        // the other half of 16, mirrored
}
// Over the four lanes that share lane % 16.
__device__ inline float across_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float across_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// ---------------------------------------------------------------------------
// Few rows: decode steps
// ---------------------------------------------------------------------------

constexpr int kTile = 32;      // keys a wave takes at a time
constexpr int kWaves = 4;      // of a workgroup; they take the tiles of its range in turn
constexpr int kRows = 16;
constexpr int kMaxSplits = 1024;

// A row's weights p = 2^(score - ref) are carried against a reference that is only moved
// when p s leaves the range of f16: it is set so that the largest p s of the keys that the row sees
// is 2^kTarget, and looked at again when a p s comes to 2^kMost (few rows), or when the tile's largest
// score and its largest scale of V would together (prompts). What is dropped at the other end lies
// 2^-31 below the largest p s. A scale counts as at least 2^-24; where it is 0, the sum of the p shows
// that they grow.
// p s goes to the matrix cores as f16, for rows of f16 with a second f16 for the rest. One f16, at most
// 2^-11 of each weight off, next to a result of f16 would show: 2.9e-4 of it in all, 2.1e-4 with two, which is
// the result's own rounding (two caches of 131072 keys 53 us, with two 58; a prompt of 4096 tokens 207 and
// 248). Next to one of bf16 it does not: 1.67e-3, with two 1.66e-3. The sums of p and of p (m + 8 s)
// stay in f32.
constexpr int kTarget = 7, kMost = 13;
template <typename T>
constexpr bool kTwo = std::is_same<T, F16>::value;
constexpr float kMostWeight = 1 << kMost, kMostSum = 0x1p60f;

// Of a key's scale and offset.
__device__ inline float log2_scale(half2v sm) { return __builtin_amdgcn_logf(fmaxf((float)sm[0], 0x1p-24f)); }

// Partial results of a split: per (tile of the launch, kv head, split) O [R][D], reference [R], sum [R].
template <int D, int R>
__host__ __device__ constexpr int64_t part_floats() { return R * (D + 2); }

struct SplitArgs {
  AttentionKv4Args a;
  int group;           // G
  int splits, chunk;   // key tiles of a split
  int64_t slot0;       // number of the launch's first tile of rows
};

__device__ inline int active_splits(const SplitArgs& s, int total) {
  const int n = (total + s.chunk - 1) / s.chunk;
  return n < 1 ? 1 : n < s.splits ? n : s.splits;
}

// A key tile on its way through LDS, in the order in which the lanes read it: for each of
// its two halves of 16 keys the K codes [D / 128][64 lanes][16 bytes] (D = 64: [64][8]), the
// V codes likewise, then K and V parameters [2][16 keys].
template <int D>
struct TileLds {
  static constexpr int kCodes = 8 * D;              // bytes of 16 keys' K (V) codes
  static constexpr int kHalf = 2 * kCodes + 128;
  static constexpr int kBytes = 2 * kHalf;
  static constexpr int kLoads = 2 * (D == 64 ? 2 : 2 * (D / 128) + 1);
};

// One half straight into LDS: per instruction 64 (params: 8) lanes of 16 bytes, past the
// caches (kPast) where nobody else will ask for them.
template <int D, bool kPast>
__device__ inline void request_half(char* lds, const char* block, int page, int row, const uint32_t (&k_at)[2],
                                    uint32_t p_at, int lane) {
  typedef __attribute__((address_space(3))) void lds_t;
  constexpr int kPolicy = kPast ? 2 : 0;            // bit 1: not kept
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)block, 0, 0x7FFFFFFF, 0x00020000);
  const int codes = row * (D / 2), v_codes = codes + page * (D / 2);
  if constexpr (D == 64) {
    // (a wave's worth holds K in its first half, V in the second)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t*)lds, 16, k_at[0], codes, 0, kPolicy);
  } else {
#pragma unroll
    for (int i = 0; i < D / 128; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t*)(lds + 1024 * i), 16, k_at[0], codes + 16 * i, 0, kPolicy);
#pragma unroll
    for (int i = 0; i < D / 128; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t*)(lds + TileLds<D>::kCodes + 1024 * i), 16, k_at[1],
                                               v_codes + 256 * i, 0, kPolicy);
  }
  if (lane < 8)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t*)(lds + 2 * TileLds<D>::kCodes), 16, p_at, row * 4, 0, kPolicy);
}

template <int N>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ inline void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

union Frag {
  uint32_t u[4];
  half2v h[4];
  half8 f;
};

// A dword of K codes as 8 f16 subnormals, 2^-24 of their values (products and sums are exact
// all the same): nibbles 0, 4, 1, 5, 2, 6, 3, 7, the odd ones 16 times too large, which the
// queries take back.
__device__ inline half8 k_frag(uint32_t w) {
  Frag f;
  f.u[0] = w & 0x000F000Fu;
  f.u[1] = w & 0x00F000F0u;
  f.u[2] = (w >> 8) & 0x000F000Fu;
  f.u[3] = (w >> 8) & 0x00F000F0u;
  return f.f;
}

// Byte b of two tokens' dwords in the halves of a dword.
template <int b>
__device__ inline uint32_t pair_bytes(uint32_t first, uint32_t second) {
  return __builtin_amdgcn_perm(second, first, 0x0C040C00u | b | (b << 16));
}
// Tiles of a wave in LDS: the one in use and the one on its way. (Three, which leave room for
// three workgroups on a compute unit instead of four: two caches of 131072 keys, with one f16 a
// weight, 51.2 us, with two tiles 50.4.)
constexpr int kRing = 2;

// LDS of a workgroup: the waves' rings, later their results; behind them the waves'
// references and sums.
template <int D>
constexpr int split_lds_bytes() {
  constexpr int ring = kWaves * kRing * TileLds<D>::kBytes, join = kWaves * kRows * (D + 4) * 4;
  return (ring > join ? ring : join) + 2 * kWaves * kRows * 4;
}

// The low (high) nibbles of both halves as f16 c - 8: 1024 + c (64 + c) by or-ing c into the
// mantissa, exactly. The or's constant comes in a register, or the and before it could not
// be the same instruction.
__device__ inline half2v low_codes(uint32_t x, uint32_t bias) {
  return as_half2((x & 0x000F000Fu) | bias) - (half2v)(_Float16)1032.f;
}
__device__ inline half2v high_codes(uint32_t x, uint32_t bias) {
  return as_half2((x & 0x00F000F0u) | bias) - (half2v)(_Float16)72.f;
}

// One kv head, 16 rows, the key tiles of one split. v_mfma_f32_16x16x32_f16 with the keys
// as rows of the scores: a lane holds one query row and 8 of the 32 keys, its weights are
// then already the operand of the second product (whose k index may be any order of the
// keys), and everything that belongs to a row (its reference, its sums, the factor of its
// result) is one value of the lane. The waves of a workgroup take key tiles in turn, each
// with a running softmax of its own; they join through LDS at the end. The next tile is
// requested before the current one is used. Bound by HBM, with the vector instructions (about 200 a
// tile of 32 keys and D = 128) not far behind: two caches of 131072 keys, 251 MB, in 50 us (5.0
// TB/s), 32 of 1000 to 8192 keys, 160 MB, in 38 us (4.2 TB/s), without the join (rows of bf16 45 and 36).
template <int D, typename T, bool kPast>
__global__ __launch_bounds__(64 * kWaves, 2) void attention_kv4_split_kernel(SplitArgs args) {
  const AttentionKv4Args& a = args.a;
  constexpr int S = D / 32;                        // matrix-core steps of a score
  constexpr int C = D >= 128 ? D / 128 : 1;        // dwords of a V row in a lane
  constexpr int NI = D / 16;                       // accumulators of O
  extern __shared__ __attribute__((aligned(1024))) char memory[];
  float (*ref_s)[kRows] = (float (*)[kRows])(memory + split_lds_bytes<D>()) - 2 * kWaves;
  float (*sum_s)[kRows] = ref_s + kWaves;
  float (*o_s)[kRows][D + 4] = (float (*)[kRows][D + 4])memory;      // (once all tiles are used)
  const int G = args.group;
  const int head = blockIdx.x % a.kv_heads;
  const Rows rows = find_rows(a, args.slot0 + blockIdx.x / a.kv_heads, G, kRows);
  if (rows.b < 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int last_row = rows.count - 1 < rows.first + kRows - 1 ? rows.count - 1 : rows.first + kRows - 1;
  const int lo_pos = position(rows, rows.first / G), hi_pos = position(rows, last_row / G);
  const Keys<kTile> keys(a, lo_pos, hi_pos);
  const int parts = active_splits(args, keys.total);
  const int split = blockIdx.y;
  if (split >= parts) return;
  const int begin = split * args.chunk;
  const int end = split == parts - 1 ? keys.total : begin + args.chunk;

  // The lane's query row (rows past the sequence's last repeat it; they are not written).
  const int row = rows.first + n < last_row ? rows.first + n : last_row;
  const int pos = position(rows, row / G);
  const uint16_t* q = (const uint16_t*)a.q + (int64_t)(rows.token0 + row / G) * a.q_stride + (int64_t)(head * G + row % G) * D +
                      g * (D / 4);
  Frag qf[S];
  float f, qsum;
  {
    float x[D / 4], top = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < D / 4; i += 8) {
      const u32x4 w = *(const u32x4*)(q + i);
      widen4<T>(u32x2{w.x, w.y}, x + i);
      widen4<T>(u32x2{w.z, w.w}, x + i + 4);
    }
    const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      x[i] *= sign;
      top = fmaxf(top, fabsf(x[i]));
      sum += x[i];
    }
    top = across_max(top);
    sum = across_sum(sum);
    // Queries in f16 with their largest value near 2^8: exact but for what lies 2^-18 and
    // more below it.
    const int e = top > 0.f && top < INFINITY ? 8 - ilogbf(top) : 0;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int nibble = (j >> 1) + 4 * (j & 1);
        qf[s].f[j] = (_Float16)ldexpf(x[8 * s + nibble], nibble & 1 ? e - 4 : e);
      }
    // score log2(e) scale = s_k f S + m_k qsum, S the product with codes of 2^-24
    f = ldexpf(fabsf(a.scale) * kLog2e, 24 - e);
    qsum = sum * (fabsf(a.scale) * kLog2e);
  }

  floatx4 o[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float ref = -1e30f, l = 0.f, bias = 0.f;
  const int32_t* table = a.page_table + rows.b * a.page_table_stride;
  const int shift = a.pool.page_shift;

  const int page_size = 1 << shift, pages = (int)a.pool.pages, wide = (int)a.max_pages;
  const char* base = a.pool.base + head * Block<D>::bytes(page_size);
  // What the lane's row sees: keys up to pos, of them those past `below` and the sinks.
  const int below = a.window ? pos - (int)a.window : -1, sinks = a.window ? (int)a.sinks : 0;
  // Pages of the wave's next 32 tiles, a lane per half of a tile; -1 and others outside the
  // pool: no keys. (An entry that is fetched when it is needed costs every tile its latency.)
  int tile = begin + wave;
  int pages_from = tile, page_ids = -1;
  auto fetch_pages = [&](int from) {
    const int t = from + (lane >> 1) * kWaves;
    const int i = t < end ? (keys.key(t) + 16 * (lane & 1)) >> shift : wide;
    pages_from = from;
    page_ids = i < wide ? table[i] : -1;
    asm volatile("" : "+v"(page_ids));     // (waited for here, not at each use)
  };
  auto page_at = [&](int t, int half) {
    return __builtin_amdgcn_readlane(page_ids, (t - pages_from) / kWaves * 2 + half);
  };
  // Where a lane fetches from, so that what it reads from LDS is its own operand: K row n,
  // bytes of group g; V dword n of the 4 keys of group g.
  char* ring = memory + wave * kRing * TileLds<D>::kBytes;
  uint32_t k_at[2], p_at;
  if constexpr (D == 64) {
    // (lanes 0..31 fetch K: chunk c of 16 bytes of row lane / 2; lanes 32.. V: 8 dwords of 4 keys a group)
    k_at[0] = lane < 32 ? lane * 16 : (lane - 32) * 16 + page_size * (D / 2);
    k_at[1] = 0;
  } else {
    k_at[0] = n * (D / 2) + g * (D / 8);
    k_at[1] = g * (D / 8) * 16 + n * 16;
  }
  p_at = page_size * D + (lane & 3) * 16 + (lane >> 2) * page_size * 4;      // lanes 0..3 the K parameters, 4..7 those of V
  // What has been requested: its first key, and whether the pages of its halves exist.
  struct Tile {
    int key, exist;
  };
  auto request = [&](int slot, int t) {
    char* to = ring + slot * TileLds<D>::kBytes;
    Tile w{keys.key(t), 0};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int p = page_at(t, half);
      const bool ok = (unsigned)p < (unsigned)pages;
      w.exist |= ok ? 1 << half : 0;
      request_half<D, kPast>(to + half * TileLds<D>::kHalf, base + (ok ? p : 0) * a.pool.page_stride, page_size,
                      (w.key + 16 * half) & (page_size - 1), k_at, p_at, lane);
    }
    return w;
  };
  uint32_t bias_low, bias_high;
  asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(bias_low));
  asm volatile("v_mov_b32 %0, 0x54005400" : "=v"(bias_high));

  // The next tile of the wave is on its way while one is used. (No other wave reads them, so
  // the wave's own counter of loads is all there is to wait for.)
  Tile now{}, next{};
  if (tile < end) {
    fetch_pages(tile);
    next = request(0, tile);
  }
  int slot = 0;
  for (; tile < end; tile += kWaves, slot ^= 1) {
    now = next;
    const int ahead = tile + kWaves;
    if (ahead < end) {
      if (ahead >= pages_from + 32 * kWaves) fetch_pages(ahead);
      wait_reads();                     // (its place was read from a tile ago)
      next = request(slot ^ 1, ahead);
      wait_loads<TileLds<D>::kLoads>();
    } else {
      wait_loads<0>();
    }
    const int key = now.key;
    const bool exist0 = now.exist & 1, exist1 = now.exist >> 1 & 1;
    const char* mine = ring + slot * TileLds<D>::kBytes;
    uint32_t kc[2][S], kp[8], vp[8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const char* at = mine + half * TileLds<D>::kHalf;
      if constexpr (D == 64) {
        const u32x2 v = *(const u32x2*)(at + n * 32 + g * 8);
        kc[half][0] = v[0], kc[half][1] = v[1];
      } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
          const u32x4 v = *(const u32x4*)(at + 1024 * i + lane * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) kc[half][4 * i + j] = v[j];
        }
      }
      const u32x4 kv = *(const u32x4*)(at + 2 * TileLds<D>::kCodes + g * 16);
      const u32x4 vv = *(const u32x4*)(at + 2 * TileLds<D>::kCodes + 64 + g * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) kp[4 * half + j] = kv[j], vp[4 * half + j] = vv[j];
    }
    floatx4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      s0 = F16Cfg16::mfma(k_frag(kc[0][i]), qf[i].f, s0);
      s1 = F16Cfg16::mfma(k_frag(kc[1][i]), qf[i].f, s1);
    }
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const half2v sm = as_half2(kp[j]);
      (j < 4 ? s0 : s1)[j & 3] *= f;
      x[j] = fmaf((float)sm[0], (j < 4 ? s0 : s1)[j & 3], fmaf((float)sm[1], qsum, -ref));
    }
    // Every row sees the whole tile, or each looks at each key: one it does not see has no
    // weight, and no scale or offset, which may be NaN there.
    const bool whole = exist0 && exist1 && key + kTile <= lo_pos + 1 &&
                       (!a.window || key > hi_pos - (int)a.window || key + kTile <= sinks);
    uint32_t seen = 0xFF;
    if (!whole) {
      seen = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = key + 16 * (j >> 2) + 4 * g + (j & 3);
        const bool yes = (j < 4 ? exist0 : exist1) & (k <= pos) & ((k > below) | (k < sinks));
        seen |= yes ? 1u << j : 0u;
        x[j] = yes ? x[j] : -INFINITY;
        vp[j] = yes ? vp[j] : 0u;
      }
    }
    // The weights, and in the rare tile in which one is too large for f16 all again, against a
    // reference that holds for its largest score and scale.
    Frag w, rest;
    float l_next, bias_next;
    auto weigh = [&]() {
      l_next = l, bias_next = bias;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const half2v sm = as_half2(vp[j]);
        const float p = __builtin_amdgcn_exp2f(x[j]);
        l_next += p;
        bias_next = fmaf(p, fmaf((float)sm[0], 8.f, (float)sm[1]), bias_next);
        w.f[j] = (_Float16)fmaf(p, (float)sm[0], 0.f);
        if constexpr (kTwo<T>) rest.f[j] = (_Float16)fmaf(p, (float)sm[0], -(float)w.f[j]);
      }
    };
    weigh();
    half2v most_w = __builtin_elementwise_max(__builtin_elementwise_max(w.h[0], w.h[1]),
                                              __builtin_elementwise_max(w.h[2], w.h[3]));
    most_w = __builtin_elementwise_max(most_w, __builtin_shufflevector(most_w, most_w, 1, 0));
    if (__ballot(most_w[0] > (_Float16)kMostWeight || l_next > kMostSum)) {
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const half2v sm = as_half2(kp[j]);
        x[j] = fmaf((float)sm[0], (j < 4 ? s0 : s1)[j & 3], (float)sm[1] * qsum);
        x[j] = seen >> j & 1 ? x[j] : -INFINITY;
        most = fmaxf(most, x[j] + log2_scale(as_half2(vp[j])));
      }
      const float raised = fmaxf(ref, across_max(most) - kTarget);
      const float factor = __builtin_amdgcn_exp2f(ref - raised);
      l *= factor;
      bias *= factor;
      ref = raised;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] -= ref;
#pragma unroll
      for (int i = 0; i < NI; ++i) o[i] *= factor;
      weigh();
    }
    l = l_next, bias = bias_next;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint32_t d[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char* at = mine + half * TileLds<D>::kHalf + TileLds<D>::kCodes;
        const u32x4 v = *(const u32x4*)(at + (D == 64 ? g * 128 + (n & 7) * 16 : 1024 * c + lane * 16));
#pragma unroll
        for (int j = 0; j < 4; ++j) d[4 * half + j] = v[j];
      }
      auto add = [&](int i, const Frag& v) {
        o[i] = F16Cfg16::mfma(v.f, w.f, o[i]);
        if constexpr (kTwo<T>) o[i] = F16Cfg16::mfma(v.f, rest.f, o[i]);
      };
      auto byte = [&](auto which) {
        constexpr int b = decltype(which)::value;
        Frag even, odd;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          uint32_t both = pair_bytes<b>(d[2 * p], d[2 * p + 1]);
          if constexpr (D == 64) both >>= (n >> 3) * 4;    // lanes 8.. of 16 take the odd d
          even.h[p] = low_codes(both, bias_low);
          if constexpr (D != 64) odd.h[p] = high_codes(both, bias_high);
        }
        if constexpr (D == 64) {
          add(b, even);
        } else {
          add(c * 8 + 2 * b, even);
          add(c * 8 + 2 * b + 1, odd);
        }
      };
      byte(std::integral_constant<int, 0>{});
      byte(std::integral_constant<int, 1>{});
      byte(std::integral_constant<int, 2>{});
      byte(std::integral_constant<int, 3>{});
    }
  }
  __syncthreads();           // (the join's memory is the rings')

  // Join the waves: everything relative to the largest reference.
  l = across_sum(l);
  bias = across_sum(bias);
  if (g == 0) {
    ref_s[wave][n] = ref;
    sum_s[wave][n] = l;
  }
  __syncthreads();
  float top = ref_s[0][n];
  for (int i = 1; i < kWaves; ++i) top = fmaxf(top, ref_s[i][n]);
  const float factor = exp2f(ref - top);
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = 4 * g + r;
      const int d = D == 64 ? 8 * (m & 7) + 2 * i + (m >> 3) : 8 * (m + 16 * (i >> 3)) + (i & 7);
      o_s[wave][n][d] = (o[i][r] + bias) * factor;
    }
  __syncthreads();
  float* part = (float*)a.workspace + ((int64_t)blockIdx.x * args.splits + split) * part_floats<D, kRows>();
  for (int at = threadIdx.x; at < kRows * D / 8; at += 64 * kWaves) {
    const int r = at / (D / 8), d = at % (D / 8) * 8;
    const int mine = rows.first + r;
    if (mine > last_row) continue;
    float v[8] = {}, total = 0.f, most = ref_s[0][r];
    for (int i = 1; i < kWaves; ++i) most = fmaxf(most, ref_s[i][r]);
    for (int i = 0; i < kWaves; ++i) {
      total += sum_s[i][r] * exp2f(ref_s[i][r] - most);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += o_s[i][r][d + j];
    }
    if (parts > 1) {
      *(float4*)(part + r * D + d) = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)(part + r * D + d + 4) = make_float4(v[4], v[5], v[6], v[7]);
      if (d == 0) {
        part[kRows * D + r] = most;
        part[kRows * (D + 1) + r] = total;
      }
      continue;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = total != 0.f ? v[j] / total : 0.f;
    const u32x2 r0 = narrow4<T>(v), r1 = narrow4<T>(v + 4);
    uint16_t* out = (uint16_t*)a.out + (int64_t)(rows.token0 + mine / G) * a.out_stride + (int64_t)(head * G + mine % G) * D + d;
    *(u32x4*)out = u32x4{r0.x, r0.y, r1.x, r1.y};
  }
}

// Adds the partial results of the splits. A workgroup takes every gridDim.y-th row of a tile:
// groups of D / 4 threads a row each, or where there are fewer rows than groups a share of a
// row's splits, joined in a fixed order.
constexpr int kJoinThreads = 256;
template <int D, typename T, int R, int kKeys>
__global__ __launch_bounds__(kJoinThreads) void attention_kv4_join_kernel(SplitArgs args) {
  const AttentionKv4Args& a = args.a;
  constexpr int L = D / 4, kGroups = kJoinThreads / L;
  __shared__ float sum_s[kGroups][D], total_s[kGroups];
  const int head = blockIdx.x % a.kv_heads, G = args.group;
  const Rows rows = find_rows(a, args.slot0 + blockIdx.x / a.kv_heads, G, R);
  if (rows.b < 0) return;
  const int last_row = rows.count - 1 < rows.first + R - 1 ? rows.count - 1 : rows.first + R - 1;
  const Keys<kKeys> keys(a, position(rows, rows.first / G), position(rows, last_row / G));
  const int parts = active_splits(args, keys.total);
  if (parts == 1) return;
  const float* part = (const float*)a.workspace + (int64_t)blockIdx.x * args.splits * part_floats<D, R>();
  const int Y = gridDim.y, y = blockIdx.y;
  const int count = (last_row - rows.first - y + Y) / Y;        // rows y, y + Y, ... of the tile
  if (count <= 0) return;
  const int share = count < kGroups ? kGroups / count : 1;      // groups of a row
  const int group = threadIdx.x / L, lane = threadIdx.x % L, d = lane * 4;
  for (int first = 0; first < count; first += kGroups / share) {
    const int nth = first + group / share, r = y + nth * Y;
    if (nth < count && group < kGroups / share * share) {
      float most = -1e30f;
      for (int i = lane; i < parts; i += L) most = fmaxf(most, part[i * part_floats<D, R>() + R * D + r]);
      for (int m = 1; m < L; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float total = 0.f;
#pragma unroll 8
      for (int i = group % share; i < parts; i += share) {
        const float* p = part + i * part_floats<D, R>();
        const float factor = __builtin_amdgcn_exp2f(p[R * D + r] - most);
        const float4 v = *(const float4*)(p + r * D + d);
        total = fmaf(p[R * (D + 1) + r], factor, total);
        sum.x = fmaf(v.x, factor, sum.x), sum.y = fmaf(v.y, factor, sum.y);
        sum.z = fmaf(v.z, factor, sum.z), sum.w = fmaf(v.w, factor, sum.w);
      }
      *(float4*)&sum_s[group][d] = sum;
      if (lane == 0) total_s[group] = total;
    }
    __syncthreads();
    if (nth < count && group % share == 0 && group < kGroups / share * share) {
      float v[4] = {}, total = 0.f;
      for (int i = 0; i < share; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += sum_s[group + i][d + j];
        total += total_s[group + i];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = total != 0.f ? v[j] / total : 0.f;
      const int row = rows.first + r;
      uint16_t* out = (uint16_t*)a.out + (int64_t)(rows.token0 + row / G) * a.out_stride + (int64_t)(head * G + row % G) * D + d;
      *(u32x2*)out = narrow4<T>(v);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Many rows: prompts
// ---------------------------------------------------------------------------

constexpr int kPromptRows = 128;      // of a workgroup, 32 of each of its four waves
constexpr int kPromptKeys = 64;

// One of the two buffers of key tiles in LDS: K and V codes as f16 in the order in which the
// lanes read them, then the keys' parameters, scale and offset. (Offset + 8 scales of V is formed where
// it is used, in f32: f16 ends at 65504, which either of the two may come to. From LDS as f32
// it costs more than the multiply-add: a prompt of 8192 tokens 720 us, so 678.)
template <int D>
struct PromptLds {
  static constexpr int N = kPromptKeys;
  static constexpr int kV = N * D * 2;                  // K before it: [N / 32][D / 16][64 lanes] of 16 bytes
  static constexpr int kParams = 2 * kV;                // V: [N / 16][D / 32][64 lanes]
  static constexpr int kBytes = kParams + N * 8;
};
template <int D>
constexpr int prompt_lds_bytes() { return 2 * PromptLds<D>::kBytes + 64; }

// 128 rows of one kv head against its key tiles. The workgroup turns each tile's codes into f16
// once, in LDS (centred for V, see above; subnormals for K), while its waves multiply the tile
// before it: v_mfma_f32_32x32x16_f16 with the keys as rows of the scores, as in the kernel for
// few rows, 32 rows a wave. Two waves fit a vector unit (three with D = 64), and one's softmax (eleven
// instructions to a score: three for scale and offset, one each for the largest, the sum and the operand, two
// for the offsets of V, an exponential at a quarter of the rate; one more for the rest of a weight) has only the
// other's products beside it: a prompt of 4096 tokens, 32 heads of 128, 137 GFLOP, in 240 us (0.57 PFLOP/s; vector
// unit 59 % of the time, matrix cores 35 %), one of 8192 in 867 (0.63), rows of bf16 in 202 and 678.
template <int D, typename T>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attention_kv4_prompt_kernel(SplitArgs args) {
  const AttentionKv4Args& a = args.a;
  constexpr int N = kPromptKeys, KB = N / 32, KK = N / 16;     // keys; blocks of 32; steps of 16
  constexpr int S = D / 16, DB = D / 32;                            // steps of a score; blocks of d
  extern __shared__ __attribute__((aligned(1024))) char memory[];
  const int G = args.group;
  const int head = blockIdx.x % a.kv_heads;
  // (the last tiles of a prompt see most keys: they start first)
  const Rows rows = find_rows(a, args.slot0 + gridDim.x / a.kv_heads - 1 - blockIdx.x / a.kv_heads, G, kPromptRows);
  if (rows.b < 0) return;
  const int last_row = rows.count - 1 < rows.first + kPromptRows - 1 ? rows.count - 1 : rows.first + kPromptRows - 1;
  const int wg_lo = position(rows, rows.first / G), wg_hi = position(rows, last_row / G);
  const Keys<N> keys(a, wg_lo, wg_hi);
  const int parts = active_splits(args, keys.total);
  const int split = blockIdx.y;
  if (split >= parts) return;
  const int begin = split * args.chunk, end = split == parts - 1 ? keys.total : begin + args.chunk;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;

  // The lane's query row; the rows of its wave.
  const int wave_first = rows.first + wave * 32 < last_row ? rows.first + wave * 32 : last_row;
  const int wave_last = wave_first + 31 < last_row ? wave_first + 31 : last_row;
  const bool idle = rows.first + wave * 32 > last_row;
  const int row = wave_first + n < wave_last ? wave_first + n : wave_last;
  const int pos = position(rows, row / G), lo_pos = position(rows, wave_first / G), hi_pos = position(rows, wave_last / G);
  const uint16_t* q = (const uint16_t*)a.q + (int64_t)(rows.token0 + row / G) * a.q_stride +
                      (int64_t)(head * G + row % G) * D + h * 8;
  Frag qf[S];
  float f, qsum;
  {
    float top = 0.f, sum = 0.f;
    const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const u32x4 w = *(const u32x4*)(q + 16 * s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        qf[s].u[j] = w[j];
        const float x0 = T::widen(w[j] & 0xFFFFu), x1 = T::widen(w[j] >> 16);
        top = fmaxf(top, fmaxf(fabsf(x0), fabsf(x1)));
        sum += x0 + x1;
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    sum = (sum + __shfl_xor(sum, 32)) * sign;
    const int e = top > 0.f && top < INFINITY ? 8 - ilogbf(top) : 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = T::widen(qf[s].u[j] & 0xFFFFu) * sign;
        x[2 * j + 1] = T::widen(qf[s].u[j] >> 16) * sign;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int nibble = (j >> 1) + 4 * (j & 1);
        qf[s].f[j] = (_Float16)ldexpf(x[nibble], nibble & 1 ? e - 4 : e);
      }
    }
    f = ldexpf(fabsf(a.scale) * kLog2e, 24 - e);
    qsum = sum * (fabsf(a.scale) * kLog2e);
  }

  // Staging. A wave takes a group of 16 keys, so that their page is the same for all its lanes: 16 (D = 64: 8) bytes of K codes a lane, and of V the 8 keys
  // x 8 d of two 16-byte pieces to two (four) lanes, which turn a part of the d each.
  const int shift = a.pool.page_shift, page_size = 1 << shift, pages = (int)a.pool.pages, wide = (int)a.max_pages;
  const char* base = a.pool.base + head * Block<D>::bytes(page_size);
  const int32_t* table = a.page_table + rows.b * a.page_table_stride;
  constexpr int KL = D == 64 ? 2 : 4;                    // dwords of K to a lane
  constexpr int VL = D == 64 ? 4 : 2;                    // lanes to a unit of V
  const int group = wave;
  auto k_turn = [](int step) { return D == 128 ? step & 6 : step * 2 & 6; };
  // Where a lane's pieces lie in a block (behind a group's first key) and where they go in LDS.
  const int v_h = lane / VL / (D / 8), v_w = lane / VL % (D / 8);
  const int k_row = lane / (D / 8 / KL), k_c = lane % (D / 8 / KL) * KL;
  const int k_from = k_row * (D / 2) + k_c * 4, v_from = v_h * (D / 8) * 16 + v_w * 16;
  const int p_from = ((lane & 15) + (lane >> 4) * page_size) * 4;
  const int k_to = ((group >> 1) * S * 64 + k_c / 2 * 64) * 16 + (((group & 1) * 16 + k_row) ^ k_turn(k_c / 2)) * 16;
  const int v_to = PromptLds<D>::kV + ((group * DB + v_w / 4) * 64 + v_h * 32 + v_w % 4 * 8) * 16;
  const int turn = (v_w & 3) + 4 * v_h;
  int pages_from = begin, page_ids = -1;
  auto fetch_pages = [&](int from) {
    const int t = from + lane / KK;
    const int i = t < end ? (keys.key(t) + 16 * (lane % KK)) >> shift : wide;
    pages_from = from;
    page_ids = i < wide ? table[i] : -1;
    asm volatile("" : "+v"(page_ids));
  };
  u32x4 raw_v[2];
  uint32_t raw_k[KL], raw_p;
  int exist_next = 0;           // whether the pages of the fetched tile's groups of 16 keys exist
  auto fetch = [&](int t) {
    exist_next = (int)(__ballot((unsigned)page_ids < (unsigned)pages) >> ((t - pages_from) * KK)) & ((1 << KK) - 1);
    const int key = keys.key(t) + 16 * group;
    // (what does not exist, and parameters that no row of the workgroup sees, count as zeros: what
    // lies there may be NaN)
    raw_v[0] = raw_v[1] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < KL; ++i) raw_k[i] = 0;
    raw_p = 0;
    if (exist_next >> group & 1) {
      const int p = __builtin_amdgcn_readlane(page_ids, (t - pages_from) * KK + group);
      const char* block = base + p * a.pool.page_stride;
      const int r = key & (page_size - 1);
      const char* k_at = block + Block<D>::k_row(r) + k_from;
      if constexpr (D == 64) {
        const u32x2 v = *(const u32x2*)k_at;
        raw_k[0] = v[0], raw_k[1] = v[1];
      } else {
        const u32x4 v = *(const u32x4*)k_at;
#pragma unroll
        for (int i = 0; i < 4; ++i) raw_k[i] = v[i];
      }
      const char* v_at = block + Block<D>::v_dword(page_size, r, 0) + v_from;
      raw_v[0] = *(const u32x4*)v_at;
      raw_v[1] = *(const u32x4*)(v_at + D / 8 * 32);
      // (lanes 0..15: of K, 16..31: of V)
      if (lane < 32 && key + (lane & 15) <= wg_hi)
        raw_p = *(const uint32_t*)(block + Block<D>::k_params(page_size, r) + p_from);
    }
  };
  uint32_t bias_low, bias_high;
  asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(bias_low));
  asm volatile("v_mov_b32 %0, 0x54005400" : "=v"(bias_high));
  float* scales = (float*)(memory + 2 * PromptLds<D>::kBytes);      // per buffer and wave the largest scale of V
  // In LDS the d of a unit of V lie next to each other, turned by the unit, or the lanes that
  // write them would meet in an eighth of the banks; the lanes' places of a step of K likewise.
  auto stage = [&](int buffer) {
    char* to = memory + buffer * PromptLds<D>::kBytes;
    // (the two halves of a step have the same turn, with D = 128 the next step's too)
#pragma unroll
    for (int i = 0; i < KL; ++i) *(half8*)(to + k_to + (i / 2 * 64 + i % 2 * 32) * 16) = k_frag(raw_k[i]);
#pragma unroll
    for (int i = 0; i < 4 / VL; ++i) {
      // Byte b of every token's dword: d = 2 b and 2 b + 1.
      const int b = lane % VL * (4 / VL) + i;
      const uint32_t select = 0x0C040C00u | b | (b << 16);
      Frag even, odd;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t both =
            __builtin_amdgcn_perm(raw_v[p >> 1][2 * (p & 1) + 1], raw_v[p >> 1][2 * (p & 1)], select);
        even.h[p] = low_codes(both, bias_low);
        odd.h[p] = high_codes(both, bias_high);
      }
      *(half8*)(to + v_to + ((2 * b) ^ turn) * 16) = even.f;
      *(half8*)(to + v_to + ((2 * b + 1) ^ turn) * 16) = odd.f;
    }
    // A key whose V row is not finite (in scale or offset) gets a K row that is not, and zeros
    // for V: rows that see it have a NaN for their weight, for all others its weight is 0.
    const bool broken = (raw_p & 0x7C00u) == 0x7C00u || (raw_p & 0x7C000000u) == 0x7C000000u;
    const uint32_t all_broken = (uint32_t)__ballot(broken);
    const half2v sm = as_half2(broken ? 0u : raw_p);
    float most = (float)sm[0];
    most = row16_max(most);
    uint32_t bits = __builtin_bit_cast(uint32_t, sm);
    if (lane < 16) bits = (all_broken | all_broken >> 16) >> lane & 1 ? 0x7E007E00u : raw_p;
    if (lane < 32)
      *(uint32_t*)(to + PromptLds<D>::kParams + (lane >= 16 ? N * 4 : 0) + (16 * group + (lane & 15)) * 4) = bits;
    if (lane == 16) scales[4 * buffer + group] = most;
  };

  floatx16 o[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) o[i] = floatx16{};
  float ref = 0.f, l = 0.f, bias = 0.f;
  bool fresh = true;                   // no score yet
  float limit = -INFINITY;             // what a score and the largest scale may come to
  const int below = a.window ? pos - (int)a.window : -1, sinks = a.window ? (int)a.sinks : 0;
  if (begin < end) {
    fetch_pages(begin);
    fetch(begin);
    stage(0);
  }
  __syncthreads();
  for (int tile = begin; tile < end; ++tile) {
    const int buffer = (tile - begin) & 1, exist = exist_next;
    const bool more = tile + 1 < end;
    if (more) {
      if (tile + 1 >= pages_from + 64 / KK) fetch_pages(tile + 1);
      fetch(tile + 1);
    }
    const int key = keys.key(tile);
    // (rows of this wave that see some of the tile: behind its last row there is nothing)
    const bool works = !idle && key <= hi_pos;
    const bool whole = exist == (1 << KK) - 1 && key + N <= lo_pos + 1 &&
                       (!a.window || key > hi_pos - (int)a.window || key + N <= sinks);
    const char* from = memory + buffer * PromptLds<D>::kBytes;
    if (works) {
      float stop = 0x1p-24f;
#pragma unroll
      for (int i = 0; i < KK; ++i) stop = fmaxf(stop, scales[4 * buffer + i]);
      const int stop_e = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(stop));
      // Scores minus the row's reference. Element j of a lane: key 32 kb + 8 (j / 4) + 4 h + j % 4.
      floatx16 x[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) x[kb] = floatx16{};
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          x[kb] = F16Cfg::mfma(*(const half8*)(from + ((kb * S + i) * 64 + (lane ^ k_turn(i))) * 16), qf[i].f, x[kb]);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const u32x4 kp = *(const u32x4*)(from + PromptLds<D>::kParams + (32 * kb + 2 * j + 4 * h) * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const half2v sm = as_half2(kp[i]);
            x[kb][j + i] = fmaf((float)sm[0], x[kb][j + i] * f, fmaf((float)sm[1], qsum, -ref));
          }
        }
      if (!whole) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int from_lane = key + 32 * kb + 4 * h;
          const int up_to = pos - from_lane, past = below - from_lane, sink = sinks - from_lane;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int k = 8 * (j >> 2) + (j & 3);
            const bool yes = (k <= up_to) & ((k > past) | (k < sink)) & ((exist >> (2 * kb + j / 8) & 1) != 0);
            x[kb][j] = yes ? x[kb][j] : -INFINITY;
          }
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, x[kb][j]);
      if (__ballot(top > limit - (float)stop_e)) {
        float most = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const u32x4 vp = *(const u32x4*)(from + PromptLds<D>::kParams + (N + 32 * kb + 2 * j + 4 * h) * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, x[kb][j + i] + log2_scale(as_half2(vp[i])));
          }
        const float over = fmaxf(most, __shfl_xor(most, 32)) - kTarget;
        // (a row's first scores set its reference, wherever they lie; later ones only raise it)
        const float by = fresh ? (over > -INFINITY ? over : 0.f) : fmaxf(over, 0.f);
        const float factor = fresh ? 1.f : __builtin_amdgcn_exp2f(-by);
        if (over > -INFINITY) fresh = false, limit = (float)(kMost + 1);
        l *= factor;
        bias *= factor;
        ref += by;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 16; ++j) x[kb][j] -= by;
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] *= factor;
      }
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        Frag p, rest;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const u32x4 vp = *(const u32x4*)(from + PromptLds<D>::kParams + (N + 16 * kk + 2 * j + 4 * h) * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const half2v sm = as_half2(vp[i]);
            const float w = __builtin_amdgcn_exp2f(x[kk / 2][kk % 2 * 8 + j + i]);
            l += w;
            bias = fmaf(w, fmaf((float)sm[0], 8.f, (float)sm[1]), bias);
            p.f[j + i] = (_Float16)fmaf(w, (float)sm[0], 0.f);
            if constexpr (kTwo<T>) rest.f[j + i] = (_Float16)fmaf(w, (float)sm[0], -(float)p.f[j + i]);
          }
        }
        half8 v[DB];
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          const int at = (kk * DB + i) * 64 + h * 32 + (n & 24) + ((n & 7) ^ ((n >> 3) + 4 * h));
          v[i] = *(const half8*)(from + PromptLds<D>::kV + at * 16);
          o[i] = F16Cfg::mfma(v[i], p.f, o[i]);
        }
        // (after all of the first products, or each would wait for the one before it)
        if constexpr (kTwo<T>) {
#pragma unroll
          for (int i = 0; i < DB; ++i) o[i] = F16Cfg::mfma(v[i], rest.f, o[i]);
        }
      }
    }
    if (more) stage(buffer ^ 1);
    __syncthreads();
  }

  if (idle) return;
  l += __shfl_xor(l, 32);
  bias += __shfl_xor(bias, 32);
  if (wave_first + n > wave_last) return;
  if (parts > 1) {
    const int64_t unit = (rows.slot - args.slot0) * a.kv_heads + head;
    float* part = (float*)a.workspace + (unit * args.splits + split) * part_floats<D, kPromptRows>();
    const int r = wave * 32 + n;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *(float4*)(part + r * D + 32 * i + 2 * j + 4 * h) =
            make_float4(o[i][j] + bias, o[i][j + 1] + bias, o[i][j + 2] + bias, o[i][j + 3] + bias);
    if (h == 0) {
      part[kPromptRows * D + r] = fresh ? -1e30f : ref;
      part[kPromptRows * (D + 1) + r] = l;
    }
    return;
  }
  const float inverse = l != 0.f ? 1.f / l : 0.f;
  uint16_t* out = (uint16_t*)a.out + (int64_t)(rows.token0 + row / G) * a.out_stride + (int64_t)(head * G + row % G) * D;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = (o[i][j + k] + bias) * inverse;
      *(u32x2*)(out + 32 * i + 2 * j + 4 * h) = narrow4<T>(v);
    }
}

// Which kernel, and how many splits of how many of its key tiles. Of all the tiles of rows the
// grid can hold, and of the keys the longest sequence shows them.
struct Split {
  bool prompt;
  int64_t tiles;       // numbers of tiles of rows
  int splits, chunk;
  bool past;           // few rows: keys past the caches
  int64_t slice;       // tiles of rows to a launch
  uint64_t bytes;      // of partial results of a launch
};
// Partial results that a long prompt may ask for: more of them come from more work than fills the
// device many times over (4096 workgroups of the prompt kernel), in launches one after the other that
// use the same memory. (All at once, a prompt of 131072 tokens of 32 + 8 heads of 128 takes 17.5 GB.)
constexpr uint64_t kMostPartBytes = 256ull << 20;

// Splits of the prompt kernel: `units` workgroups with `tiles` key tiles each at most. In half
// microseconds, a key tile costs 7.2 for each two workgroups that share a compute unit and 6 for a
// last one alone, a workgroup's start about four tiles, the join a little and more with each
// partial result. (8 sequences of 8192 keys with 128 rows each, 64 units: 8 splits 86 us, 4 splits 125, 16
// splits 98; with 512 rows, 256 units: 2 splits 245 us, 4 splits 247, none 274.)
int64_t prompt_splits(int64_t units, int64_t tiles, int64_t cus) {
  int64_t best = 1;
  double least = INFINITY;
  for (int64_t s = 1; s == 1 || (s <= tiles / 8 && s <= 64); ++s) {
    const int64_t load = ceil_div(units * s, cus);         // workgroups of the busiest compute unit
    const double tile = 7.2 * (load / 2) + 6 * (load % 2);
    const double cost = (ceil_div(tiles, s) + 4) * tile + (s > 1 ? 8 + 0.02 * units * s : 0);
    if (cost < 0.95 * least) best = s, least = cost;      // (more of them only where it shows)
  }
  return best;
}

Split plan(int64_t tokens, int64_t batch, int heads, int kv_heads, int dim, int64_t window, int64_t sinks,
           int64_t max_kv_len) {
  const int64_t G = heads / kv_heads, rows = tokens * G, cus = device_cu_count();
  auto seen = [&](int64_t R, int64_t tile) {           // keys that a tile of R rows sees
    int64_t keys = max_kv_len;
    const int64_t reach = window + sinks + R / G + 2 * tile;
    if (window && reach < keys) keys = reach;
    return keys < 1 ? 1 : keys > 0x7FFFFFFF ? 0x7FFFFFFF : keys;
  };
  auto units_of = [&](int64_t R) { return batch * ceil_div(ceil_div(rows, batch), R) * kv_heads; };
  // Prompts where sequences have a tile's rows on average and there is work for the whole device
  // (8 sequences of 8192 keys with 128 rows each 87 us, as few rows 97; 4 of 1024 keys with 384 rows
  // 34, as few rows 24, with 2048 rows 64 and 87; 4 of 512 with 1024 rows 26 and 33). The device is full
  // by tiles of the longest, and of one whole prompt half as many work: one of 1024 tokens, which is at the
  // line, 50 us, as few rows 37, of 1024 on 2048 keys 79 and 70, of 1536 on 2048 keys 82 and 90. Never with heads
  // of 256, whose tiles leave room for one wave on a vector unit (2048 tokens with 16 + 4 heads on
  // 4096 keys, with one f16 a weight, 349 us, as few rows 235).
  Split p;
  int64_t units = units_of(kPromptRows), keys = seen(kPromptRows, kPromptKeys);
  p.prompt = dim <= 128 && rows >= kPromptRows * batch &&
             (units >= cus || units * ceil_div(keys, kPromptKeys) >= 32 * cus);
  if (!p.prompt) units = units_of(kRows), keys = seen(kRows, kTile);
  p.tiles = rows / (p.prompt ? kPromptRows : kRows) + batch;
  // Keys that one tile of rows reads once, and that are too many for the caches to hold until the
  // next step, go past them: two sequences of 131072 keys 58.8 us through them, 54.4 past them, 32 of 1000 to
  // 8192 keys 48.6 and 44.5; 72 MB of windows 20.5 and 20.2, which a repeated call still finds there.
  p.past = !p.prompt && tokens <= batch && G <= kRows && (double)batch * keys * kv_heads * (dim + 8) > 128e6;
  const int64_t key_tiles = ceil_div(keys, p.prompt ? kPromptKeys : kTile);
  int64_t splits;
  if (p.prompt) {
    splits = prompt_splits(units, key_tiles, cus);
  } else {
    // Five workgroups to a compute unit, so that lengths that differ even out (32 sequences of
    // 1000 to 8192 keys: 44.5 us, with four 48.6, with eight 47.8), but no more than 32 splits where
    // fewer fill the device: the join reads them all (two of 131072 keys, rows of bf16: 52.1 us, with 48 splits
    // 54.9, with 64 54.3; of f16 all 57). A split has enough tiles to be worth its start and the join, fewer where
    // most of the device is idle.
    splits = ceil_div(5 * cus, units);
    if (splits > 32) splits = ceil_div(2 * cus, units) > 32 ? ceil_div(2 * cus, units) : 32;
    const int64_t most = 2 * units <= cus ? ceil_div(key_tiles, 16) : key_tiles / 32;
    splits = splits < most ? splits : most;
  }
  // Past 16384 keys the f32 sums of a wave, which the matrix cores cut off, would begin to show in the
  // result: f16 of a prompt on 65536 keys in one split 2.14e-4 off, on 131072 2.3e-4, on 524288 4.3e-4, next to
  // 2.08e-4; of few rows on 524288 2.2e-4.
  if (splits < ceil_div(keys, 16384)) splits = ceil_div(keys, 16384);
  splits = splits < 1 ? 1 : splits > kMaxSplits ? kMaxSplits : splits;
  p.chunk = (int)ceil_div(key_tiles, splits);
  if (!p.prompt) p.chunk = (int)(ceil_div(p.chunk, kWaves) * kWaves);
  p.splits = (int)ceil_div(key_tiles, p.chunk);
  p.slice = p.tiles;
  p.bytes = 0;
  if (p.splits > 1) {
    const uint64_t one = (uint64_t)kv_heads * p.splits * (p.prompt ? kPromptRows : kRows) * (dim + 2) * 4;
    const int64_t most = kMostPartBytes > one ? (int64_t)(kMostPartBytes / one) : 1;
    p.slice = ceil_div(p.tiles, ceil_div(p.tiles, most));
    p.bytes = p.slice * one;
  }
  return p;
}

template <typename Kernel>
int allow_lds(Kernel kernel, int bytes, PerDeviceOnce& once) {
  if (bytes <= 65536) return 0;
  int dev = 0;
  UK_RETURN_IF_HIP(hipGetDevice(&dev));
  if (once.done(dev)) return 0;
  UK_RETURN_IF_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  once.mark(dev);
  return 0;
}

template <int D, typename T>
int launch_split(const AttentionKv4Args& a, hipStream_t s) {
  Split p = plan(a.tokens, a.batch, a.heads, a.kv_heads, D, a.window, a.sinks, a.max_kv_len);
  // (a grid's threads are counted in 32 bits)
  if (p.tiles * a.kv_heads > 0xFFFFFFFFll / 256)
    return fail(IREE_AMD_UK_STATUS_INVALID_ARGUMENT, "attention_kv4: too many rows for one call");
  if (p.splits > 1 && a.workspace_bytes < p.bytes) p.splits = 1, p.slice = p.tiles;
  static PerDeviceOnce once[3];
  // (a prompt's last tiles see most keys: they start first)
  for (int64_t to = p.tiles; to > 0; to -= p.slice) {
    const int64_t from = to > p.slice ? to - p.slice : 0, blocks = (to - from) * a.kv_heads;
    SplitArgs args{a, a.heads / a.kv_heads, p.splits, p.chunk, from};
    const dim3 grid((unsigned)blocks, (unsigned)p.splits);
    auto run = [&](auto kernel, int bytes, PerDeviceOnce& set) {
      UK_RETURN_IF_ERROR(allow_lds(kernel, bytes, set));
      hipLaunchKernelGGL(kernel, grid, dim3(256), bytes, s, args);
      return 0;
    };
    if (!p.prompt && p.past) {
      UK_RETURN_IF_ERROR(run(attention_kv4_split_kernel<D, T, true>, split_lds_bytes<D>(), once[0]));
    } else if (!p.prompt) {
      UK_RETURN_IF_ERROR(run(attention_kv4_split_kernel<D, T, false>, split_lds_bytes<D>(), once[1]));
    } else if constexpr (D <= 128) {
      UK_RETURN_IF_ERROR(run(attention_kv4_prompt_kernel<D, T>, prompt_lds_bytes<D>(), once[2]));
    }
    UK_RETURN_IF_HIP(hipGetLastError());
    if (p.splits == 1) continue;
    // A row a workgroup where the tiles are few, one workgroup a tile where they fill the device
    // (most rows of a tile are not there in a decode step, and each workgroup has to find that out).
    const int64_t R = p.prompt ? kPromptRows : kRows;
    int64_t shares = 2ll * device_cu_count() / blocks;
    shares = shares < 1 ? 1 : shares > R ? R : shares;
    if (p.prompt && shares < 8) shares = 8;
    const dim3 join((unsigned)blocks, (unsigned)shares);
    if (!p.prompt)
      hipLaunchKernelGGL((attention_kv4_join_kernel<D, T, kRows, kTile>), join, dim3(kJoinThreads), 0, s, args);
    else if constexpr (D <= 128)
      hipLaunchKernelGGL((attention_kv4_join_kernel<D, T, kPromptRows, kPromptKeys>), join, dim3(kJoinThreads), 0, s, args);
    UK_RETURN_IF_HIP(hipGetLastError());
  }
  note_kernel_path(p.prompt ? (p.splits > 1 ? "attention_kv4:prompt-split" : "attention_kv4:prompt")
                            : (p.splits > 1 ? "attention_kv4:few-rows-split" : "attention_kv4:few-rows"));
  return 0;
}

}  // namespace

uint64_t attention_kv4_workspace(int64_t tokens, int64_t batch, int heads, int kv_heads, int dim, int64_t window,
                                 int64_t sinks, int64_t max_kv_len) {
  return plan(tokens, batch, heads, kv_heads, dim, window, sinks, max_kv_len).bytes;
}

int launch_attention_kv4(const AttentionKv4Args& a, hipStream_t s) {
  switch (a.dim) {
    case 64: return a.bf16 ? launch_split<64, BF16>(a, s) : launch_split<64, F16>(a, s);
    case 128: return a.bf16 ? launch_split<128, BF16>(a, s) : launch_split<128, F16>(a, s);
    default: return a.bf16 ? launch_split<256, BF16>(a, s) : launch_split<256, F16>(a, s);
  }
}

}  // namespace uk
