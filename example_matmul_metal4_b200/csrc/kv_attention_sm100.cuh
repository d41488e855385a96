// Attention over the key / value cache: O = softmax(scale * Q K^T) V with K
// and V read from the cache's codes.
#pragma once

#include "kv_cache_sm100.cuh"

namespace mm4 {

struct KvAttnArgs {
  KvBatch kb;
  const __half* Q;
  __half* O;
  float* lse;            // optional [tokens][heads_q]
  long long q_stride, o_stride;
  const uint8_t* cache;
  int heads_q, group;    // group = heads_q / heads_kv
  int causal;
  float scale_log2;      // scale * log2(e)
};

__device__ __forceinline__ float kv_warp_sum(float x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
  return x;
}

// One warp per row of Q: lanes share the head dimension, keys one at a time,
// online softmax in fp32.
template <int D, int BITS>
__global__ void __launch_bounds__(128) kv_attention_row_kernel(const KvAttnArgs a) {
  using Row = KvRow<D, BITS>;
  constexpr int E = D / 32;
  const KvBatch& kb = a.kb;
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= static_cast<long long>(kb.tokens) * a.heads_q) return;
  const int t = static_cast<int>(w / a.heads_q), h = static_cast<int>(w % a.heads_q);
  const int b = kv_find_sequence(kb, t, lane);
  if (b < 0) return;
  const KvSequence s = kv_sequence(kb, b);
  if (s.n == 0 || t < s.first || t >= s.first + s.n) return;
  if (s.n > kb.max_new) kv_note(KV_DATA_NEW);
  const int limit = a.causal ? min(s.len, max(0, s.len - (s.n - 1 - (t - s.first)))) : s.len;
  float q[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __half2float(a.Q[t * a.q_stride + static_cast<long long>(h) * D + lane * E + e]);
    acc[e] = 0.f;
  }
  const int hk = h / a.group;
  float m = -INFINITY, l = 0.f;
  auto value = [&](const uint8_t* row, int d) {
    const uint32_t c = BITS == 8 ? row[d] : (row[d / 2] >> (4 * (d % 2))) & 15u;
    const __half* par = reinterpret_cast<const __half*>(row + Row::CODES + d / KV_GROUP * 4);
    return __half2float(__hfma(__uint2half_rn(c), par[0], par[1]));
  };
  for (int p = 0; p < limit; ++p) {
    const int page = kb.table[static_cast<long long>(b) * kb.pages_per_seq + (p >> kb.page_shift)];
    if (page < 0 || page >= kb.pages) {
      kv_note(KV_DATA_PAGE);
      continue;
    }
    const uint8_t* krow = a.cache + page * kb.page_bytes +
                          ((static_cast<long long>(hk * 2) << kb.page_shift) + (p & ((1 << kb.page_shift) - 1))) *
                              Row::BYTES;
    const uint8_t* vrow = krow + (static_cast<long long>(Row::BYTES) << kb.page_shift);
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) dot += q[e] * value(krow, lane * E + e);
    const float x = kv_warp_sum(dot) * a.scale_log2;
    const float m_new = fmaxf(m, x);
    const float f = exp2f(m - m_new), pr = exp2f(x - m_new);
    m = m_new;
    l = l * f + pr;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + pr * value(vrow, lane * E + e);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.O[t * a.o_stride + static_cast<long long>(h) * D + lane * E + e] = __float2half_rn(acc[e] * inv);
  if (a.lse != nullptr && lane == 0)
    a.lse[static_cast<long long>(t) * a.heads_q + h] = (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace mm4
