// Attention over the paged 4-bit cache (include/iree_amd_uk.h has the formula and the
// layout of a block).
//
// With codes c, scale s and offset m of a key's rows, a query q and G query heads to a kv
// head:
//   q . k = s_k (q . c_k) + m_k sum(q)
//   sum_j p_j v_j = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (m_j + 8 s_j)
// so the matrix cores multiply the codes themselves, which f16 holds exactly, and each
// key costs two multiply-adds for its scale and offset instead of a dequantised row. The
// codes of V are centred because the sum over a long sequence is small next to its parts:
// of uncentred codes and offsets the f32 sums would cancel (measured at 131072 keys in one
// chain: 1.9e-3 of the result).
#include "uk_common.h"
#include "uk_kv4.h"
#include "uk_mfma_cfg.h"

#include <type_traits>

namespace uk {
namespace {
using namespace kv4;

constexpr float kLog2e = 1.4426950408889634f;

// Where a workgroup's rows stand. Rows r of a sequence are its query tokens times the G
// heads of one kv head, token by token; tiles of R rows are numbered over the batch with
// gaps: sequence b has the tiles from floor(q_starts[b] G / R) + b on, which leaves room
// for its own and needs no sums over the batch.
struct Rows {
  int b;             // sequence, -1: none
  int first;         // first row of the tile
  int count;         // rows of the sequence
  int tokens;        // its query tokens
  int64_t token0;    // its first token
  int64_t kv_len;
};

// The sequence of tile `slot`: the last b whose first tile is at most it. 64 lanes look at
// 64 sequences at a time, so a batch of up to 64 costs one load.
__device__ inline Rows find_rows(const AttentionKv4Args& a, int64_t slot, int G, int R) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, n = a.batch;                      // candidates [lo, lo + n)
  while (n > 1) {
    const int64_t step = (n + 63) / 64;
    const int64_t b = lo + lane * step;
    const bool mine = b < lo + n && (int64_t)a.q_starts[b] * G / R + b <= slot;
    const uint64_t yes = __ballot(mine);
    const int last = yes ? 63 - __builtin_clzll(yes) : 0;
    const int64_t from = lo + last * step;
    n = from + step < lo + n ? step : lo + n - from;
    lo = from;
  }
  Rows r;
  const int64_t start = a.q_starts[lo], next = a.q_starts[lo + 1];
  const int64_t first = (slot - (start * G / R + lo)) * R;
  const int64_t rows = (next - start) * G;
  r.b = start >= 0 && next <= a.tokens && first >= 0 && first < rows ? (int)lo : -1;
  r.first = (int)first;
  r.count = (int)rows;
  r.tokens = (int)(next - start);
  r.token0 = start;
  r.kv_len = a.kv_lens[lo];
  return r;
}

// Position of a query token: below 0 where it sees nothing.
__device__ inline int position(const Rows& r, int token) {
  const int64_t p = r.kv_len - r.tokens + token;
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
#ifndef WPE
#define WPE 2
#endif
#ifndef NWV
#define NWV 4
#endif
#ifndef WANT
#define WANT 4
#endif
#ifndef MINC
#define MINC 16
#endif
constexpr int kWaves = NWV;      // of a workgroup; they take the tiles of its range in turn
constexpr int kRows = 16;

// Exponents: weights p = 2^(t) with t <= kLazy above the row's reference, which is only
// moved when a score passes that; p s is carried in f16 times 2^-E, E moved when a scale
// passes 2^kScaleMost of it: p s 2^-E stays below 2^15, and what is dropped at the other end
// lies 2^-32 below the largest scale.
constexpr float kLazy = 4.f;
constexpr float kScaleMost = 2048.f;

// Partial results of a split: per (tile, kv head, split) O [16][D], reference [16], sum [16].
template <int D>
__host__ __device__ constexpr int64_t part_floats() { return kRows * (D + 2); }

struct SplitArgs {
  AttentionKv4Args a;
  int group;           // G
  int splits, chunk;   // key tiles of a split
};

__device__ inline int active_splits(const SplitArgs& s, int total) {
  const int n = (total + s.chunk - 1) / s.chunk;
  return n < 1 ? 1 : n < s.splits ? n : s.splits;
}

template <int D>
struct KvTile {
  static constexpr int S = D / 32;              // dwords of a K row in a lane: MFMA steps
  static constexpr int C = D >= 128 ? D / 128 : 1;
  uint32_t k[2][S];
  uint4 v[2][C];
  uint4 kp[2], vp[2];
};

// A lane's places in the 16 rows that one half of a tile reads; everything else of an
// address is the same for the wave.
template <int D>
struct LaneAt {
  uint32_t k, v, p;
  __device__ LaneAt(int n, int g) {
    k = n * (D / 2) + g * (D / 8);
    v = g * (D / 8) * 16 + (D >= 128 ? n : n & 7) * 16;
    p = g * 16;
  }
};

// A tile's keys and where its halves, 16 keys apart, lie; pages clamped into the pool.
struct TileAt {
  int key;
  int page[2];           // -1 and others outside the pool: no keys
  const char* block[2];  // the kv head's block
  int row[2];
};

template <int D>
__device__ inline void load_k(KvTile<D>& t, const TileAt& w, const LaneAt<D>& at) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const char* k = w.block[half] + Block<D>::k_row(w.row[half]) + at.k;
    if constexpr (D == 64) {
      const uint2 v = *(const uint2*)k;
      t.k[half][0] = v.x, t.k[half][1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < D / 128; ++i) {
        const uint4 v = *(const uint4*)(k + 16 * i);
        t.k[half][4 * i] = v.x, t.k[half][4 * i + 1] = v.y, t.k[half][4 * i + 2] = v.z, t.k[half][4 * i + 3] = v.w;
      }
    }
  }
}
template <int D>
__device__ inline void load_kp(KvTile<D>& t, const TileAt& w, const LaneAt<D>& at, int page) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
    t.kp[half] = *(const uint4*)(w.block[half] + Block<D>::k_params(page, w.row[half]) + at.p);
}
template <int D>
__device__ inline void load_vp(KvTile<D>& t, const TileAt& w, const LaneAt<D>& at, int page) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
    t.vp[half] = *(const uint4*)(w.block[half] + Block<D>::v_params(page, w.row[half]) + at.p);
}
template <int D>
__device__ inline void load_v(KvTile<D>& t, const TileAt& w, const LaneAt<D>& at, int page) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int c = 0; c < KvTile<D>::C; ++c)
      t.v[half][c] = *(const uint4*)(w.block[half] + Block<D>::v_dword(page, w.row[half], 0) + at.v + 256 * c);
}

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
union Frag {
  uint32_t u[4];
  half2v h[4];
  half8 f;
};

__device__ inline half2v as_half2(uint32_t u) { return __builtin_bit_cast(half2v, u); }

// A dword of K codes as 8 f16 subnormals (products and sums are exact all the same): nibbles
// 0, 4, 1, 5, 2, 6, 3, 7, the odd ones 16 times too large, which the queries take back.
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
// Both low (high) nibbles as centred f16 codes c - 8: 1024 + c (64 + c) by or-ing c into the
// mantissa, exactly.
__device__ inline half2v low_codes(uint32_t x) {
  const uint32_t u = (x & 0x000F000Fu) | 0x64006400u;
  return as_half2(u) - (half2v)(_Float16)1032.f;
}
__device__ inline half2v high_codes(uint32_t x) {
  const uint32_t u = (x & 0x00F000F0u) | 0x54005400u;
  return as_half2(u) - (half2v)(_Float16)72.f;
}

__device__ inline uint32_t dword(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// One kv head, 16 rows, the key tiles of one split. v_mfma_f32_16x16x32_f16 with the keys
// as rows of the scores: a lane holds one query row and 8 of the 32 keys, its weights are
// then already the operand of the second product (whose k index may be any order of the
// keys), and everything that belongs to a row (its reference, its sums, the factor of its
// result) is one value of the lane. The waves of a workgroup take key tiles in turn, each
// with a running softmax of its own; they join through LDS at the end. The next tile is
// requested before the current one is used.
template <int D, typename T>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(WPE))) void attention_kv4_split_kernel(SplitArgs args) {
  const AttentionKv4Args& a = args.a;
  constexpr int S = KvTile<D>::S, C = KvTile<D>::C;
  constexpr int NI = D / 16;                       // accumulators of O
  constexpr bool kExact = __is_same(T, F16);
  __shared__ float ref_s[kWaves][kRows], sum_s[kWaves][kRows];
  __shared__ float o_s[kWaves][kRows][D + 4];
  const int G = args.group;
  const int head = blockIdx.x % a.kv_heads;
  const int64_t slot = blockIdx.x / a.kv_heads;
  const Rows rows = find_rows(a, slot, G, kRows);
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
  const uint16_t* q = (const uint16_t*)a.q + (rows.token0 + row / G) * a.q_stride + (int64_t)(head * G + row % G) * D +
                      g * (D / 4);
  Frag qf[S];
  float f, qsum;
  {
    float x[D / 4], top = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < D / 4; i += 8) {
      const uint4 w = *(const uint4*)(q + i);
      widen4<T>(make_uint2(w.x, w.y), x + i);
      widen4<T>(make_uint2(w.z, w.w), x + i + 4);
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
    // score log2(e) scale = f (s_k S + m_k qsum), S the product with codes of 2^-24
    f = ldexpf(fabsf(a.scale) * kLog2e, 24 - e);
    qsum = ldexpf(sum, e - 24);
  }

  floatx4 o[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float ref = -1e30f, l = 0.f, bias = 0.f;
  float vscale = 0.f;             // 2^-E; 0 before the first scale
  const int32_t* table = a.page_table + rows.b * a.page_table_stride;
  const int shift = a.pool.page_shift;

  const int page_size = 1 << shift, pages = (int)a.pool.pages, wide = (int)a.max_pages;
  const char* base = a.pool.base + head * Block<D>::bytes(page_size);
  // What the lane's row sees: keys up to pos, of them those past `below` and the sinks.
  const int below = a.window ? pos - (int)a.window : -1, sinks = a.window ? (int)a.sinks : 0;
  auto locate = [&](int tile) {
    TileAt w;
    w.key = keys.key(tile);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int key = w.key + 16 * half, i = key >> shift;
      w.page[half] = i < wide ? table[i] : -1;
      w.row[half] = key & (page_size - 1);
    }
    return w;
  };
  // (once the page numbers are needed: they have had a tile's time to arrive)
  auto resolve = [&](TileAt& w) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int p = (unsigned)w.page[half] < (unsigned)pages ? w.page[half] : 0;
      w.block[half] = base + p * a.pool.page_stride;
    }
  };

  const LaneAt<D> at(n, g);
  KvTile<D> t;
  TileAt now, next;
  int tile = begin + wave;
  if (tile < end) {
    now = locate(tile);
    resolve(now);
    load_k<D>(t, now, at);
    load_kp<D>(t, now, at, page_size);
    load_vp<D>(t, now, at, page_size);
    load_v<D>(t, now, at, page_size);
    next = locate(tile + kWaves < end ? tile + kWaves : tile);
  }
  // Each part of a tile is requested again, for the wave's next tile, as soon as it has been
  // used: one tile is in flight at any time, in the registers of one. (The last tile requests
  // itself once more.)
  for (; tile < end; tile += kWaves) {
    const int key = now.key;
    const bool exist0 = (unsigned)now.page[0] < (unsigned)pages, exist1 = (unsigned)now.page[1] < (unsigned)pages;
    resolve(next);
    floatx4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      s0 = F16Cfg16::mfma(k_frag(t.k[0][i]), qf[i].f, s0);
      s1 = F16Cfg16::mfma(k_frag(t.k[1][i]), qf[i].f, s1);
    }
    load_k<D>(t, next, at);
    __builtin_amdgcn_sched_barrier(0);
    float w[8], x[8];
    uint32_t vp[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t kp = dword(t.kp[j >> 2], j & 3);
      w[j] = fmaf(F16::widen(kp & 0xFFFFu), j < 4 ? s0[j & 3] : s1[j & 3], F16::widen(kp >> 16) * qsum);
      x[j] = fmaf(w[j], f, -ref);
      vp[j] = dword(t.vp[j >> 2], j & 3);
    }
    load_kp<D>(t, next, at, page_size);
    load_vp<D>(t, next, at, page_size);
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
    const float top = fmaxf(max4(x[0], x[1], x[2], x[3]), max4(x[4], x[5], x[6], x[7]));
    half2v smost = as_half2(vp[0]);                 // (scales are not negative, and the low halves)
#pragma unroll
    for (int j = 1; j < 8; ++j) smost = __builtin_elementwise_max(smost, as_half2(vp[j]));
    const float stop = (float)smost[0];
    if (__ballot(top > kLazy || stop * vscale >= kScaleMost || vscale == 0.f)) {
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, seen >> j & 1 ? w[j] * f : -INFINITY);
      const float raised = fmaxf(ref, across_max(most));
      float factor = exp2f(ref - raised);
      l *= factor;
      bias *= factor;
      ref = raised;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = seen >> j & 1 ? fmaf(w[j], f, -ref) : -INFINITY;
      float smax = stop;
      for (int m = 1; m < 64; m *= 2) smax = fmaxf(smax, __shfl_xor(smax, m));
      if (smax * vscale >= kScaleMost || (vscale == 0.f && smax > 0.f)) {
        const float to = ldexpf(1.f, 7 - ilogbf(smax));
        factor *= vscale == 0.f ? 0.f : to / vscale;
        vscale = to;
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) o[i] *= factor;
    }
    Frag hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const half2v sm = as_half2(vp[j]);
      const float p = __builtin_amdgcn_exp2f(x[j]);
      l += p;
      bias = fmaf(p, fmaf((float)sm[0], 8.f, (float)sm[1]), bias);
      const float weight = p * ((float)sm[0] * vscale);
      hi.f[j] = (_Float16)weight;
      if constexpr (kExact) lo.f[j] = (_Float16)(weight - (float)hi.f[j]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint32_t d[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = dword(t.v[j >> 2][c], j & 3);
      auto add = [&](int i, const Frag& v) {
        o[i] = F16Cfg16::mfma(v.f, hi.f, o[i]);
        if constexpr (kExact) o[i] = F16Cfg16::mfma(v.f, lo.f, o[i]);
      };
      auto byte = [&](auto which) {
        constexpr int b = decltype(which)::value;
        Frag even, odd;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          uint32_t both = pair_bytes<b>(d[2 * p], d[2 * p + 1]);
          if constexpr (D == 64) both >>= (n >> 3) * 4;    // lanes 8.. of 16 take the odd d
          even.h[p] = low_codes(both);
          if constexpr (D != 64) odd.h[p] = high_codes(both);
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
    load_v<D>(t, next, at, page_size);
    now = next;
    next = locate(tile + 2 * kWaves < end ? tile + 2 * kWaves : tile);
  }

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
  const float vfactor = vscale == 0.f ? 0.f : factor / vscale;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = 4 * g + r;
      const int d = D == 64 ? 8 * (m & 7) + 2 * i + (m >> 3) : 8 * (m + 16 * (i >> 3)) + (i & 7);
      o_s[wave][n][d] = fmaf(o[i][r], vfactor, bias * factor);
    }
  __syncthreads();
  float* part = (float*)a.workspace + ((int64_t)blockIdx.x * args.splits + split) * part_floats<D>();
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
    const uint2 r0 = narrow4<T>(v), r1 = narrow4<T>(v + 4);
    uint16_t* out = (uint16_t*)a.out + (rows.token0 + mine / G) * a.out_stride + (int64_t)(head * G + mine % G) * D + d;
    *(uint4*)out = make_uint4(r0.x, r0.y, r1.x, r1.y);
  }
}

// Adds the partial results of a tile's splits in order, one workgroup per row.
template <int D, typename T>
__global__ __launch_bounds__(D / 2) void attention_kv4_join_kernel(SplitArgs args) {
  const AttentionKv4Args& a = args.a;
  const int head = blockIdx.x % a.kv_heads, G = args.group;
  const Rows rows = find_rows(a, blockIdx.x / a.kv_heads, G, kRows);
  if (rows.b < 0) return;
  const int row = rows.first + blockIdx.y;
  if (row >= rows.count) return;
  const int last_row = rows.count - 1 < rows.first + kRows - 1 ? rows.count - 1 : rows.first + kRows - 1;
  const Keys<kTile> keys(a, position(rows, rows.first / G), position(rows, last_row / G));
  const int parts = active_splits(args, keys.total);
  if (parts == 1) return;
  const float* part = (const float*)a.workspace + (int64_t)blockIdx.x * args.splits * part_floats<D>();
  const int r = blockIdx.y, d = threadIdx.x * 2;
  float most = -1e30f;
  for (int i = 0; i < parts; ++i) most = fmaxf(most, part[i * part_floats<D>() + kRows * D + r]);
  float total = 0.f, x = 0.f, y = 0.f;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float* p = part + i * part_floats<D>();
    const float factor = exp2f(p[kRows * D + r] - most);
    const float2 v = *(const float2*)(p + r * D + d);
    total = fmaf(p[kRows * (D + 1) + r], factor, total);
    x = fmaf(v.x, factor, x);
    y = fmaf(v.y, factor, y);
  }
  x = total != 0.f ? x / total : 0.f;
  y = total != 0.f ? y / total : 0.f;
  uint16_t* out = (uint16_t*)a.out + (rows.token0 + row / G) * a.out_stride + (int64_t)(head * G + row % G) * D + d;
  *(uint32_t*)out = T::narrow(x) | (T::narrow(y) << 16);
}

// How many splits of how many key tiles. Of all the tiles of rows the grid can hold, and of
// the keys the longest sequence shows them.
struct Split {
  int64_t tiles;       // of rows, with the gaps of their numbering
  int splits, chunk;
};

Split plan(int64_t tokens, int64_t batch, int heads, int kv_heads, int64_t window, int64_t sinks, int64_t max_kv_len) {
  const int64_t G = heads / kv_heads;
  Split p;
  p.tiles = tokens * G / kRows + batch;
  int64_t keys = max_kv_len;
  if (window && window + sinks < keys) keys = window + sinks + 2 * kTile;
  if (keys > 0x7FFFFFFF) keys = 0x7FFFFFFF;
  const int64_t key_tiles = ceil_div(keys, kTile);
  const int64_t units = (tokens * G / kRows < batch ? batch : tokens * G / kRows) * kv_heads;
  const int64_t wanted = 1ll * WANT * device_cu_count();
  int64_t chunk = ceil_div(key_tiles * units, wanted);
  chunk = ceil_div(chunk < MINC ? MINC : chunk, kWaves) * kWaves;
  p.chunk = (int)chunk;
  p.splits = (int)ceil_div(key_tiles < 1 ? 1 : key_tiles, chunk);
  if (p.splits > 1024) {
    p.splits = 1024;
    p.chunk = (int)ceil_div(key_tiles, 1024);
  }
  return p;
}

template <int D, typename T>
int launch_split(const AttentionKv4Args& a, hipStream_t s) {
  Split p = plan(a.tokens, a.batch, a.heads, a.kv_heads, a.window, a.sinks, a.max_kv_len);
  const int64_t blocks = p.tiles * a.kv_heads;
  if (blocks > 0x7FFFFFFF) return fail(IREE_AMD_UK_STATUS_INVALID_ARGUMENT, "attention_kv4: too many rows for one call");
  const uint64_t one = (uint64_t)blocks * part_floats<D>() * 4;
  if (p.splits > 1 && a.workspace_bytes < one * p.splits) p.splits = 1;
  SplitArgs args{a, a.heads / a.kv_heads, p.splits, p.chunk};
  hipLaunchKernelGGL((attention_kv4_split_kernel<D, T>), dim3((unsigned)blocks, (unsigned)p.splits), dim3(64 * kWaves), 0,
                     s, args);
  UK_RETURN_IF_HIP(hipGetLastError());
  if (p.splits == 1) return 0;
  const int64_t rows = a.tokens * args.group < kRows ? a.tokens * args.group : kRows;
  hipLaunchKernelGGL((attention_kv4_join_kernel<D, T>), dim3((unsigned)blocks, (unsigned)rows), dim3(D / 2), 0, s, args);
  return check_hip(hipGetLastError(), "attention_kv4");
}

}  // namespace

uint64_t attention_kv4_workspace(int64_t tokens, int64_t batch, int heads, int kv_heads, int dim, int64_t window,
                                 int64_t sinks, int64_t max_kv_len) {
  const Split p = plan(tokens, batch, heads, kv_heads, window, sinks, max_kv_len);
  if (p.splits == 1) return 0;
  const int64_t part = dim == 64 ? part_floats<64>() : dim == 128 ? part_floats<128>() : part_floats<256>();
  return (uint64_t)p.tiles * kv_heads * p.splits * part * 4;
}

int launch_attention_kv4(const AttentionKv4Args& a, hipStream_t s) {
  switch (a.dim) {
    case 64: return a.bf16 ? launch_split<64, BF16>(a, s) : launch_split<64, F16>(a, s);
    case 128: return a.bf16 ? launch_split<128, BF16>(a, s) : launch_split<128, F16>(a, s);
    default: return a.bf16 ? launch_split<256, BF16>(a, s) : launch_split<256, F16>(a, s);
  }
}

}  // namespace uk
