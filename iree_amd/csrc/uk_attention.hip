// Attention over the paged 4-bit cache (include/iree_amd_uk.h has the formula).
#include "uk_common.h"
#include "uk_kv4.h"

namespace uk {
namespace {
using namespace kv4;

// One wave per query row: a lane takes one key of 64 at a time for the scores, then D / 64
// values of d for the sum over those keys. Running maximum m and sum l of the softmax, f32.
template <int D, typename T>
__global__ __launch_bounds__(64) void attention_kv4_rows_kernel(AttentionKv4Args a) {
  __shared__ float q[D], weight[64], offset[64];
  __shared__ const char* where[64];
  const int64_t token = blockIdx.x;
  const int head = blockIdx.y, lane = threadIdx.x;
  if (token < a.q_starts[0] || token >= a.q_starts[a.batch]) return;
  int64_t lo = 0, hi = a.batch;                 // q_starts[lo] <= token < q_starts[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (a.q_starts[mid] <= token) lo = mid; else hi = mid;
  }
  const int64_t kv_len = a.kv_lens[lo], position = kv_len - a.q_starts[lo + 1] + token;
  const int32_t* table = a.page_table + lo * a.page_table_stride;
  const int shift = a.pool.page_shift, page = 1 << shift, kv_head = head / (a.heads / a.kv_heads);
  const int64_t end = position + 1 < a.max_pages << shift ? position + 1 : a.max_pages << shift;
  float sum_q = 0.f;
  for (int d = lane; d < D; d += 64) q[d] = T::widen(((const uint16_t*)a.q)[token * a.q_stride + (int64_t)head * D + d]) * a.scale;
  __syncthreads();
  for (int d = 0; d < D; ++d) sum_q += q[d];
  float m = -3e38f, l = 0.f, bias = 0.f, o[D / 64] = {};
  for (int64_t base = 0; base < end; base += 64) {
    if (a.window && base >= a.sinks && base + 64 <= position - a.window + 1) continue;
    const int64_t j = base + lane;
    float score = -INFINITY;
    const char* block = nullptr;
    if (j < end && (!a.window || j > position - a.window || j < a.sinks)) {
      const int64_t p = table[j >> shift];
      if (p >= 0 && p < a.pool.pages) block = a.pool.base + p * a.pool.page_stride + kv_head * Block<D>::bytes(page);
    }
    const int at = (int)(j & (page - 1));
    if (block) {
      const uint32_t* codes = (const uint32_t*)(block + Block<D>::k_row(at));
      float dot = 0.f;
      for (int i = 0; i < D / 8; ++i)
        for (int n = 0; n < 8; ++n) dot = fmaf(q[8 * i + n], (float)((codes[i] >> (4 * n)) & 15u), dot);
      const uint32_t bits = *(const uint32_t*)(block + Block<D>::k_params(page, at));
      score = dot * F16::widen(bits & 0xFFFFu) + sum_q * F16::widen(bits >> 16);
    }
    float top = score;
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    top = fmaxf(top, m);
    const float again = expf(m - top), e = block ? expf(score - top) : 0.f;
    m = top;
    float s = 0.f, b = 0.f;
    if (block) {
      const uint32_t bits = *(const uint32_t*)(block + Block<D>::v_params(page, at));
      s = e * F16::widen(bits & 0xFFFFu);
      b = e * F16::widen(bits >> 16);
    }
    float total = e;
    for (int x = 1; x < 64; x *= 2) { total += __shfl_xor(total, x); b += __shfl_xor(b, x); }
    l = l * again + total;
    bias = bias * again + b;
    __syncthreads();
    weight[lane] = s;
    where[lane] = block ? block + page * (D / 2) : nullptr;
    __syncthreads();
    for (int i = 0; i < D / 64; ++i) o[i] *= again;
    for (int k = 0; k < 64; ++k) {
      if (!where[k]) continue;
      const int row = (int)((base + k) & (page - 1));
      for (int i = 0; i < D / 64; ++i) {
        const int d = lane + 64 * i;
        const uint32_t w = *(const uint32_t*)(where[k] + (((row >> 2) * (D / 8) + d / 8) * 4 + (row & 3)) * 4);
        o[i] = fmaf(weight[k], (float)((w >> (4 * (d & 7))) & 15u), o[i]);
      }
    }
  }
  for (int i = 0; i < D / 64; ++i)
    ((uint16_t*)a.out)[token * a.out_stride + (int64_t)head * D + lane + 64 * i] =
        (uint16_t)T::narrow(l != 0.f ? (o[i] + bias) / l : 0.f);
}

template <int D, typename T>
int launch_rows(const AttentionKv4Args& a, hipStream_t s) {
  hipLaunchKernelGGL((attention_kv4_rows_kernel<D, T>), dim3((unsigned)a.tokens, (unsigned)a.heads), dim3(64), 0, s, a);
  return check_hip(hipGetLastError(), "attention_kv4");
}

}  // namespace

uint64_t attention_kv4_workspace(int64_t, int64_t, int, int, int, int64_t, int64_t, int64_t) { return 0; }

int launch_attention_kv4(const AttentionKv4Args& a, hipStream_t s) {
  switch (a.dim) {
    case 64: return a.bf16 ? launch_rows<64, BF16>(a, s) : launch_rows<64, F16>(a, s);
    case 128: return a.bf16 ? launch_rows<128, BF16>(a, s) : launch_rows<128, F16>(a, s);
    default: return a.bf16 ? launch_rows<256, BF16>(a, s) : launch_rows<256, F16>(a, s);
  }
}

}  // namespace uk
