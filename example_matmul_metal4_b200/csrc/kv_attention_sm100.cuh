// Attention over the key / value cache: O = softmax(scale * Q K^T) V with K
// and V read from the cache's codes. This file has what the two kernels share,
// the one for few rows (kv_attention_few_sm100.cuh) and the one for many
// (kv_attention_many_sm100.cuh).
//
// The work. A unit is one key / value head of one sequence with up to ROWS rows
// (a row is one query head of one token; the heads of a group share a unit,
// so their keys are read once). A unit's keys are walked in tiles, and all
// tiles of the call, unit after unit, form one line that is cut into equal
// ranges, one for each worker. The lengths lie on the device and may change
// between replays of a captured call, so every worker finds its range itself
// from two scans over the lengths. A unit that spans several workers leaves
// one partial result (m, l and unscaled O) per worker in the workspace, and a
// second kernel joins them in worker order, so results do not depend on
// timing.
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
  float* partials;       // workspace
  int workers;           // of the launch
  int join_rows;         // few rows: rows of a unit to a block of the join
  uint32_t k1024;        // KV_1024
  unsigned long long timeout_ns;
};

// A run of partials is found by arithmetic alone: worker w takes tiles
// [w T / A, (w + 1) T / A) of the T on the line, A workers being active, so
// tile x belongs to worker floor(((x + 1) A - 1) / T).
__device__ __forceinline__ long long kv_range_begin(long long w, long long T, long long A) { return w * T / A; }
__device__ __forceinline__ long long kv_worker_of(long long x, long long T, long long A) {
  return ((x + 1) * A - 1) / T;
}

// Partials of worker w: slot 2 w is a segment that began in another worker's
// range, slot 2 w + 1 one that begins a unit here and goes on elsewhere.
// Each holds ROWS x D floats, then (m, l) of ROWS rows; m is a score.
template <int D, int ROWS>
struct KvPartial {
  static constexpr int FLOATS = ROWS * (D + 2);
};

// Exponentials are 2^((s - m) scale log2 e) with m, the running maximum, a score
// like s: the maximum gives exactly 1 however large it is. (2^(s scale log2 e - m)
// with m in the log2 domain would be off by m's rounding, which passes 2^16 for
// scores that fp16 inputs reach.)
//
// P is 2^7 times that: at most 2^15, as maxima may be stale by 8 in the log2 domain.
// fp16 has steps of 2^-24 at the least, so P is off by 2^-32 of a row's largest and
// not by 2^-25, which would drop the many small P of a long cache from O that l
// counts: 2^17 keys of 2^-25.5 each are 0.3 % of a row.
constexpr float KV_LOG2_P = 7.0f;
constexpr float KV_NO_MAX = -1e30f;  // of a row that has seen no key: below all scores (2^39) of fp16 rows

// Tiles of TK keys of a sequence (at least one: a row block with no key still
// takes a tile, which writes its zeros), and its row blocks of ROWS rows (none if
// it has no rows in this call). Blocks of few rows walk all tiles alike.
template <int TK>
__device__ __forceinline__ int kv_tiles(const KvSequence& s) {
  return max(1, (s.len + TK - 1) / TK);
}
template <int ROWS>
__device__ __forceinline__ int kv_blocks(const KvBatch& kb, const KvSequence& s, int group) {
  return (min(s.n, kb.max_new) * group + ROWS - 1) / ROWS;
}
template <int TK, int ROWS>
__device__ __forceinline__ int kv_sequence_tiles(const KvBatch& kb, int b, int group) {
  const KvSequence s = kv_sequence(kb, b);
  return kv_tiles<TK>(s) * kv_blocks<ROWS>(kb, s, group);
}

// Sum of kv_sequence_tiles over all sequences, by one warp.
template <int TK, int ROWS>
__device__ __forceinline__ long long kv_total_tiles(const KvBatch& kb, int group, int lane) {
  long long sum = 0;
  for (int b = lane; b < kb.sequences; b += 32) sum += kv_sequence_tiles<TK, ROWS>(kb, b, group);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  return sum;
}

// Sequence b whose tiles hold x (x < the total), and the tiles before it.
template <int TK, int ROWS>
__device__ __forceinline__ int kv_find_tile(const KvBatch& kb, long long x, int group, int lane, long long* before) {
  long long done = 0;
  for (int b0 = 0; b0 < kb.sequences; b0 += 32) {
    const int b = b0 + lane;
    const int t = b < kb.sequences ? kv_sequence_tiles<TK, ROWS>(kb, b, group) : 0;
    long long inc = t;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, s);
      if (lane >= s) inc += up;
    }
    const unsigned over = __ballot_sync(0xffffffffu, done + inc > x);
    if (over != 0) {
      const int k = __ffs(over) - 1;
      *before = done + __shfl_sync(0xffffffffu, inc - t, k);
      return b0 + k;
    }
    done += __shfl_sync(0xffffffffu, inc, 31);
  }
  *before = done;
  return kb.sequences;  // not reached for x < the total
}

// Keys that row r of a unit sees: those before limit (<= 0: none).
__device__ __forceinline__ int kv_limit(const KvSequence& s, int token, int causal) {
  return causal ? s.len - (s.n - 1 - token) : s.len;
}

__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Natural-log sum of exp(scale * S) from the maximum and the sum of P.
__device__ __forceinline__ float kv_lse(float m, float l, float scale_log2) {
  return fmaf(m, scale_log2, log2f(l) - KV_LOG2_P) * 0.6931471805599453f;
}

// Lets the next kernel of the stream start its blocks, and waits in it until
// the kernel before it has finished and its writes are visible.
__device__ __forceinline__ void kv_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void kv_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float kv_warp_sum(float x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
  return x;
}

}  // namespace mm4
