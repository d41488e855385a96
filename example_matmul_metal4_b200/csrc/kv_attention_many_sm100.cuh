// Attention over the key / value cache for many rows (prompts, chunks of them,
// and tokens times query heads beyond 48 rows).
//
// Bound by the tensor cores and the exponentials, as attention over fp16 K and
// V is (4 D FLOP and one exponential per row and key); what the cache adds is
// turning its codes into fp16 operands. That is done once per 64 keys for all
// 256 rows of a CTA by warps of its own, into the 128-byte-swizzled layout
// that tcgen05.mma reads, and overlaps the products of earlier keys.
//
// A row is one query head of one token, rows of a unit ordered by token and
// then head, so grouped heads fill the 128-row tiles and share the unpacked
// keys. A unit is one key / value head of one sequence and 256 rows, two tiles of
// 128. 16 warps:
//   warp 0        copies pages as they lie in the cache into a ring (untiled bulk
//                 copies).
//   warp 1        TMEM allocation; one lane issues S_i(g) = Q_i K(g)^T (M = 128,
//                 N = 64) into slot g % 2 of row tile i.
//   warp 2        one lane issues O_i += P_i(g) V(g) (P from TMEM).
//   warp 3        finds the CTA's range (and warp 2, before its products, the unit
//                 that the range leaves to others).
//   warps 4-11    softmax, one row a thread: P = 2^((S - max) scale log2 e) with fp32
//                 maxima and sums, P rounded to fp16 for the product (2^-11 of
//                 itself, like the result, or 2^-32 of the row's largest); O is
//                 rescaled only when the maximum grew by more than 8 in the log2
//                 domain. Results out; a warp also copies its rows of the next
//                 unit's Q, as soon as it has the last scores of the unit.
//   warps 12-15   codes to fp16: a lane takes 32 elements (one scale and zero).
// TMEM: two 64-column S slots for each row tile, then O_i (D columns each). Steps
// of 64 keys are counted across a CTA's units (g), which fixes slots and
// mbarrier phases; S runs two steps ahead of the softmax.
//
// Four prompts of 4096 tokens, 16 heads of 128, causal, 4 bits, on one B200: 297 us,
// 926 TFLOP/s (floor 163 us of measured peak); 344 us in long runs, under the power
// cap. A step of 64 keys takes about 2000 clocks, of which the products need 1280
// (S of N = 64 is bound by the 6 KB an instruction reads from shared memory);
// unpacking alone costs 11 %, its 42 KB a step through shared memory among them.
#pragma once

#include "attention_sm100.cuh"
#include "kv_attention_sm100.cuh"

namespace mm4 {

constexpr int KVM_TK = 64;        // keys of a step
constexpr int KVM_THREADS = 512;
// What a unit costs beyond its steps (its Q, its masked steps, its results, the
// pipeline run empty and filled), in steps: a CTA's range is cut by steps
// plus this for each unit, or the first blocks of causal prompts, 4 steps
// each, would take twice the time of the last ones.
constexpr int KVM_UNIT = 4;

template <int D, int BITS>
struct KvMany {
  static constexpr int QT = 2;                         // row tiles of 128
  static constexpr int ROWS = 128 * QT;
  static constexpr int Q_BYTES = 128 * D * 2;          // a row tile of Q
  static constexpr int TILE_BYTES = KVM_TK * D * 2;    // unpacked K or V of a step
  static constexpr int RAW_BYTES = 2 * KVM_TK * KvRow<D, BITS>::BYTES;
  static constexpr int KS = 3, VS = 3;
  static constexpr int RS = RAW_BYTES <= 10240 ? 3 : 2;
  static constexpr int OUT_ROW = 64 + 16;              // a row of 32 results, on banks of its own
  static constexpr int OUT_BYTES = 32 * OUT_ROW;       // a softmax warp's results on their way out
  static constexpr int OUT_OFFSET = QT * Q_BYTES + (KS + VS) * TILE_BYTES + RS * RAW_BYTES;
  static constexpr int MAX_OFFSET = OUT_OFFSET + 4 * QT * OUT_BYTES;  // each row's largest score
  static constexpr int BAR_OFFSET = MAX_OFFSET + ROWS * 4;
  static constexpr int SMEM_BYTES = BAR_OFFSET + 512 + 1024;
  // Registers: 128 threads each of warps 0-3, the softmax warps and the
  // unpacking warps; the sum must not exceed what the block is launched with.
  static constexpr int REGS_LOW = 88;
  static constexpr int REGS_SOFTMAX = 160;
  static constexpr int REGS_UNPACK = 104;
  static constexpr int REGS_NEEDED = (REGS_LOW + 2 * REGS_SOFTMAX + REGS_UNPACK) / 4;
  static_assert(REGS_NEEDED <= 128, "register split");
  static_assert(SMEM_BYTES <= 232448, "shared memory");
};

enum : int {
  SITE_KVM_RAW = 120,
  SITE_KVM_S = 122,
  SITE_KVM_PV = 123,
  SITE_KVM_SOFTMAX = 124,
  SITE_KVM_UNPACK = 125,
  SITE_KVM_DRAIN = 126,
};

// Row blocks of a sequence, and the steps of one: the keys its last row sees.
__device__ __forceinline__ int kvm_blocks(const KvSequence& s, int group, int rows) {
  return (s.n * group + rows - 1) / rows;
}
__device__ __forceinline__ int kvm_steps(const KvSequence& s, int rb, const KvAttnArgs& a, int rows) {
  int limit = s.len;
  if (a.causal) {
    const int last = min((rb + 1) * rows - 1, s.n * a.group - 1) / a.group;
    limit = min(s.len, kv_limit(s, last, 1));
  }
  return max(1, (limit + KVM_TK - 1) / KVM_TK);
}
// A sequence with more rows than max_new is left out (and reported).
__device__ __forceinline__ KvSequence kvm_sequence(const KvAttnArgs& a, int b) {
  KvSequence s = kv_sequence(a.kb, b);
  if (s.n > a.kb.max_new) {
    kv_note(KV_DATA_NEW);
    s.n = 0;
  }
  return s;
}
// Cost of a sequence for one head. The lanes of a warp share either the
// sequences or, where those are fewer than the row blocks that a sequence may
// have, the blocks of one sequence after the other.
__device__ __forceinline__ bool kvm_by_block(const KvAttnArgs& a, int rows) {
  return a.kb.sequences < kvm_blocks(KvSequence{0, 0, a.kb.max_new}, a.group, rows);
}
__device__ __forceinline__ long long kvm_warp_sum(long long x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
  return x;
}
__device__ __forceinline__ long long kvm_lane_cost(const KvAttnArgs& a, int b, int rows) {  // lanes: sequences
  if (b >= a.kb.sequences) return 0;
  const KvSequence s = kvm_sequence(a, b);
  const int blocks = kvm_blocks(s, a.group, rows);
  long long sum = 0;
  for (int rb = 0; rb < blocks; ++rb) sum += KVM_UNIT + kvm_steps(s, rb, a, rows);
  return sum;
}
__device__ __forceinline__ long long kvm_block_cost(const KvAttnArgs& a, const KvSequence& s, int rows,
                                                     int lane) {  // lanes: blocks
  const int blocks = kvm_blocks(s, a.group, rows);
  long long sum = 0;
  for (int rb = lane; rb < blocks; rb += 32) sum += KVM_UNIT + kvm_steps(s, rb, a, rows);
  return kvm_warp_sum(sum);
}

// A place on the line of all units: sequences, their row blocks, heads, and
// the offset in the unit: KVM_UNIT before its first step.
struct KvmPlace {
  int b, rb, h, off;
};
__device__ __forceinline__ long long kvm_total(const KvAttnArgs& a, int rows, int lane) {
  long long sum = 0;
  if (kvm_by_block(a, rows)) {
    for (int b = 0; b < a.kb.sequences; ++b) {
      const KvSequence s = kvm_sequence(a, b);
      const int blocks = kvm_blocks(s, a.group, rows);
      for (int rb = lane; rb < blocks; rb += 32) sum += KVM_UNIT + kvm_steps(s, rb, a, rows);
    }
  } else {
    for (int b = lane; b < a.kb.sequences; b += 32) sum += kvm_lane_cost(a, b, rows);
  }
  return kvm_warp_sum(sum) * a.kb.heads_kv;
}
// Place x (by one warp); also where its unit begins and what it costs.
__device__ __forceinline__ KvmPlace kvm_find(const KvAttnArgs& a, int rows, long long x, int lane,
                                             long long* unit_begin, int* unit_cost) {
  const int heads = a.kb.heads_kv;
  KvmPlace p{0, 0, 0, 0};
  long long at = 0;  // where sequence p.b begins
  if (kvm_by_block(a, rows)) {
    for (; p.b < a.kb.sequences; ++p.b) {
      const long long all = kvm_block_cost(a, kvm_sequence(a, p.b), rows, lane) * heads;
      if (at + all > x) break;
      at += all;
    }
  } else {
    for (; p.b < a.kb.sequences; p.b += 32) {
      const long long t = kvm_lane_cost(a, p.b + lane, rows);
      long long inc = t;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, s);
        if (lane >= s) inc += up;
      }
      const unsigned over = __ballot_sync(0xffffffffu, at + inc * heads > x);
      if (over != 0) {
        const int k = __ffs(over) - 1;
        at += __shfl_sync(0xffffffffu, inc - t, k) * heads;
        p.b += k;
        break;
      }
      at += __shfl_sync(0xffffffffu, inc, 31) * heads;
    }
  }
  *unit_begin = x;
  *unit_cost = 1;
  if (p.b >= a.kb.sequences) return KvmPlace{a.kb.sequences, 0, 0, 0};
  // The row block: a scan over 32 blocks at a time.
  const KvSequence s = kvm_sequence(a, p.b);
  const int blocks = kvm_blocks(s, a.group, rows);
  for (; p.rb < blocks; p.rb += 32) {
    const int t = p.rb + lane < blocks ? KVM_UNIT + kvm_steps(s, p.rb + lane, a, rows) : 0;
    int inc = t;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, k);
      if (lane >= k) inc += up;
    }
    const unsigned over = __ballot_sync(0xffffffffu, at + static_cast<long long>(inc) * heads > x);
    if (over != 0) {
      const int k = __ffs(over) - 1;
      const int cost = __shfl_sync(0xffffffffu, t, k);
      at += static_cast<long long>(__shfl_sync(0xffffffffu, inc - t, k)) * heads;
      p.rb += k;
      p.h = static_cast<int>((x - at) / cost);
      p.off = static_cast<int>((x - at) % cost);
      *unit_begin = x - p.off;
      *unit_cost = cost;
      return p;
    }
    at += static_cast<long long>(__shfl_sync(0xffffffffu, inc, 31)) * heads;
  }
  return KvmPlace{a.kb.sequences, 0, 0, 0};
}

// Segments of a CTA's range: steps [n0, n1) of one unit.
struct KvmSegment {
  KvSequence s;
  int b, rb, h, n0, n1, steps;
};
struct KvmWalk {
  KvmPlace p;
  long long left;
};
__device__ __forceinline__ bool kvm_next(const KvAttnArgs& a, int rows, KvmWalk& w, KvmSegment& g) {
  while (w.left > 0 && w.p.b < a.kb.sequences) {
    if (g.b != w.p.b) {
      g.s = kvm_sequence(a, w.p.b);
      g.b = w.p.b;
    }
    const int blocks = kvm_blocks(g.s, a.group, rows);
    if (w.p.rb >= blocks) {
      w.p = KvmPlace{w.p.b + 1, 0, 0, 0};
      continue;
    }
    g.rb = w.p.rb;
    g.h = w.p.h;
    g.steps = kvm_steps(g.s, g.rb, a, rows);
    const int cost = KVM_UNIT + g.steps;
    const int end = static_cast<int>(min(static_cast<long long>(cost), w.p.off + w.left));
    g.n0 = max(0, w.p.off - KVM_UNIT);
    g.n1 = end - KVM_UNIT;
    w.left -= end - w.p.off;
    w.p.off = end;
    if (end == cost) {
      w.p.off = 0;
      if (++w.p.h == a.kb.heads_kv) {
        w.p.h = 0;
        ++w.p.rb;
      }
    }
    if (g.n1 <= g.n0) continue;  // the range ends before the unit's first step
    return true;
  }
  return false;
}

// A partial of ROWS rows: O in groups of 4 elements, [D / 4][ROWS][4] floats, so
// that a warp of rows writes and reads whole lines; then m [ROWS], l [ROWS].
template <int D, int ROWS>
__device__ __forceinline__ long long kvm_slot(long long slot) {
  return slot * KvPartial<D, ROWS>::FLOATS;
}
// Behind the partials, for each worker: the unit that it begins and leaves to
// others, and the last of them (last = -1: none).
struct KvmShared {
  int b, rb, h, last;
};
template <int D, int ROWS>
__device__ __forceinline__ KvmShared* kvm_shared(const KvAttnArgs& a) {
  return reinterpret_cast<KvmShared*>(a.partials + kvm_slot<D, ROWS>(2ll * a.workers));
}

// P = 2^(x sl2 - m) of a row's 64 scores as fp16 pairs into the TMEM columns at
// tP; returns their fp32 sum. Calls between() behind the first half. All
// exponentials on MUFU (2^-22): the sum is a softmax statistic, and a cubic on the
// FMA pipe, good enough for fp16 P, would leave 7e-5 of a row's largest key in it.
// At head_dim 64, 3 chunks of 1000 tokens on 12,000 in 8 bits: 177 us; with 2 of 8 by
// the cubic 183, by a polynomial of degree 5 (2^-23) 187.
template <typename F>
__device__ __forceinline__ float kvm_exp_store64(const float (&x)[64], float sl2, float m, uint32_t tP, F&& between) {
  const float2 sc = make_float2(sl2, sl2);
  const float2 nm = make_float2(-m, -m);
  float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t pk[16];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int idx = half * 32 + c * 8 + 2 * e;
        const float2 y = ffma2(make_float2(x[idx], x[idx + 1]), sc, nm);
        const float2 p = make_float2(ex2_approx(y.x), ex2_approx(y.y));
        acc[e] = fadd2(acc[e], p);
        pk[c * 4 + e] = pack_half2(p.x, p.y);
      }
    }
    tmem_st_32x32b_x16(tP + half * 16, pk);
    if (half == 0) between();
  }
  const float2 sum = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
  return sum.x + sum.y;
}

// P = 2^((s - top) sl2 + KV_LOG2_P) of a row's 64 scores, read again from the TMEM
// columns at tP, of which the first `valid` count. kvm_exp_store64 subtracts m =
// fl(top sl2 - KV_LOG2_P) from the product, so its P are off by the rounding: a factor
// that a row's P share, but one that passes fp16's range for scores that fp16 inputs
// reach (2^474). From 2^20 on, where it passes 2^(1/16), m is a NaN, which takes the
// row's warp to this function. Subtracting top from every score instead costs 5 %
// (prompts, head_dim 128); this way, with no instruction and no register on the common
// path, nothing.
__device__ __forceinline__ float kvm_exp_store64_far(float sl2, float top, int valid, uint32_t tP) {
  float sum = 0.f;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    uint32_t v[32], pk[16];
    __syncwarp();
    tmem_ld_32x32b_x32(tP + half * 32, v);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const int key = half * 32 + i;
      const float p0 = key < valid ? ex2_approx(fmaf(__uint_as_float(v[i]) - top, sl2, KV_LOG2_P)) : 0.f;
      const float p1 = key + 1 < valid ? ex2_approx(fmaf(__uint_as_float(v[i + 1]) - top, sl2, KV_LOG2_P)) : 0.f;
      sum += p0 + p1;
      pk[i / 2] = pack_half2(p0, p1);
    }
    tmem_st_32x32b_x16(tP + half * 16, pk);
  }
  return sum;
}

// log2 of the factor by which kvm_exp_store64's P are too small.
__device__ __forceinline__ float kvm_rest(float top, float sl2, bool far) {
  return far || top == KV_NO_MAX ? 0.f : fmaf(-top, sl2, fmaf(top, sl2, -KV_LOG2_P)) + KV_LOG2_P;
}

template <int D, int BITS>
__global__ void __launch_bounds__(KVM_THREADS, 1) kv_attention_many_kernel(const __grid_constant__ KvAttnArgs a) {
  using Cfg = KvMany<D, BITS>;
  using Row = KvRow<D, BITS>;
  constexpr int QT = Cfg::QT, ROWS = Cfg::ROWS, KS = Cfg::KS, VS = Cfg::VS, RS = Cfg::RS, RB = Row::BYTES;
  constexpr int TB = Cfg::TILE_BYTES, QB = Cfg::Q_BYTES;
  constexpr uint32_t IDESC_S = idesc_f16_f32(128, KVM_TK, false, false);
  constexpr uint32_t IDESC_O = idesc_f16_f32(128, D, false, true);

  extern __shared__ uint8_t kvm_smem_raw[];
  const uint32_t raw_addr = smem_u32(kvm_smem_raw);
  uint8_t* smem = kvm_smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  uint8_t* sQ = smem;                       // [QT]
  uint8_t* sK = smem + QT * QB;             // [KS]
  uint8_t* sV = sK + KS * TB;               // [VS]
  uint8_t* sR = sV + VS * TB;               // [RS] pages as they lie in the cache: K rows, V rows
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFFSET);
  uint64_t* q_full = bars;                  // [tile] the unit's Q_i in place
  uint64_t* s_full = bars + 4;              // [tile][slot] S_i(g) in TMEM
  uint64_t* p_full = bars + 8;              // [tile][slot] P_i(g) in TMEM, O_i rescaled
  uint64_t* pv_done = bars + 12;            // [tile][slot] O_i += P_i(g) V(g) complete
  uint64_t* o_full = bars + 16;             // [tile] the segment's last P V complete
  uint64_t* o_empty = bars + 18;            // [tile] O_i read from TMEM
  uint64_t* drain = bars + 20;
  uint64_t* k_full = bars + 21;             // [KS] unpacked
  uint64_t* k_empty = k_full + KS;          // [KS] read by the last S
  uint64_t* v_full = k_empty + KS;          // [VS]
  uint64_t* v_empty = v_full + VS;          // [VS]
  uint64_t* r_full = v_empty + VS;          // [RS] copied
  uint64_t* r_empty = r_full + RS;          // [RS] unpacked
  uint64_t* turn = r_empty + RS;            // [tile][quadrant] exponentials of this tile's warp done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(turn + 8);
  KvmWalk* start = reinterpret_cast<KvmWalk*>(smem + Cfg::BAR_OFFSET + 448);

  const KvBatch& kb = a.kb;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Watchdog wd{&g_kv_wait, a.timeout_ns};
  kv_launch_dependents();

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 128);
      for (int sl = 0; sl < 2; ++sl) {
        mbar_init(&s_full[2 * i + sl], 1);
        mbar_init(&p_full[2 * i + sl], 128);
        mbar_init(&pv_done[2 * i + sl], 1);
      }
    }
    mbar_init(drain, 2);
    for (int i = 0; i < 8; ++i) mbar_init(&turn[i], 1);
    for (int i = 0; i < KS; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < VS; ++i) {
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < RS; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], 4);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 2) {
    // For the join: the unit that this CTA begins and leaves to others.
    const long long total = kvm_total(a, ROWS, lane);
    const long long active = min(static_cast<long long>(a.workers), total);
    const int w = blockIdx.x;
    KvmShared shared{0, 0, 0, -1};
    if (w + 1 < active) {
      long long begin;
      int cost;
      const KvmPlace f = kvm_find(a, ROWS, kv_range_begin(w + 1, total, active), lane, &begin, &cost);
      // Behind the unit's first step, and the first border that is.
      if (f.off > KVM_UNIT && begin + KVM_UNIT >= kv_range_begin(w, total, active) && f.b < kb.sequences)
        shared = KvmShared{f.b, f.rb, f.h, static_cast<int>(kv_worker_of(begin + cost - 1, total, active))};
    }
    if (lane == 0) kvm_shared<D, ROWS>(a)[w] = shared;
  }
  if (warp == 3) {
    const long long total = kvm_total(a, ROWS, lane);
    const long long active = min(static_cast<long long>(a.workers), total);
    KvmWalk w{KvmPlace{0, 0, 0, 0}, 0};
    if (blockIdx.x < active) {
      const long long x = kv_range_begin(blockIdx.x, total, active);
      long long begin;
      int cost;
      w.p = kvm_find(a, ROWS, x, lane, &begin, &cost);
      w.left = kv_range_begin(blockIdx.x + 1, total, active) - x;
    }
    if (lane == 0) *start = w;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  KvmWalk walk = *start;
  KvmSegment sg;
  sg.b = -1;

  if (warp < 4) {
    regs_dec<Cfg::REGS_LOW>();
    if (warp == 0) {
      // ---------------------------------------------------------- pages
      const int ps = 1 << kb.page_shift;
      const int chunk = min(KVM_TK, ps);  // keys of a copy
      const uint32_t bytes = static_cast<uint32_t>(chunk * RB);
      int cnt = 0, ids = 0, ids_base = 0;
      bool ok = true;
      while (ok && kvm_next(a, ROWS, walk, sg)) {
        ids_base = -64;  // page numbers of another sequence
        for (int n = sg.n0; n < sg.n1; ++n, ++cnt) {
          const int rs = cnt % RS;
          const int key0 = n * KVM_TK;
          const int valid = min(KVM_TK, sg.s.len - key0);
          const int copies = valid <= 0 ? 0 : (valid + chunk - 1) / chunk;
          const int first = key0 >> kb.page_shift;
          if (copies > 0 && first + copies > ids_base + 32) {
            ids_base = first;
            const int i = first + lane;
            ids = 0;
            if (i < kb.pages_per_seq && (i << kb.page_shift) < sg.s.len) {
              ids = __ldg(kb.table + static_cast<long long>(sg.b) * kb.pages_per_seq + i);
              if (ids < 0 || ids >= kb.pages) {
                kv_note(KV_DATA_PAGE);
                ids = 0;  // read in place of the page outside the pool
              }
            }
          }
          const int mine = lane >> 1, kv = lane & 1;  // lanes 0 .. 2 copies - 1 issue one copy each
          const int page = __shfl_sync(0xffffffffu, ids, (first - ids_base + min(mine, max(0, copies - 1))) & 31);
          ok = cnt < RS || mbar_wait(&r_empty[rs], (cnt / RS - 1) & 1, wd, SITE_KVM_RAW);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) {
            if (copies > 0)
              mbar_arrive_expect_tx(&r_full[rs], bytes * 2 * copies);
            else
              mbar_arrive(&r_full[rs]);
          }
          __syncwarp();
          if (mine < copies) {
            const uint8_t* src = a.cache + page * kb.page_bytes +
                                 (static_cast<long long>((sg.h * 2 + kv) << kb.page_shift) + (key0 & (ps - 1))) * RB;
            bulk_load(sR + rs * Cfg::RAW_BYTES + (kv * KVM_TK + mine * chunk) * RB, src, bytes, &r_full[rs]);
          }
        }
      }
      // The last copies land before the CTA ends.
      for (int t = max(0, cnt - RS); t < cnt; ++t) mbar_wait(&r_full[t % RS], (t / RS) & 1, wd, SITE_KVM_DRAIN);
    } else if (warp != 3 && elect_one()) {
      // ---------------------------------------------------------- MMA issuers
      const uint64_t q_desc0 = sw128_desc(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc0 = sw128_desc(smem_u32(sK), 16, 1024);
      const uint64_t v_desc0 = sw128_desc(smem_u32(sV), KVM_TK * 128, 1024);
      bool ok = true;
      int g = 0;  // steps across segments
      bool more = kvm_next(a, ROWS, walk, sg);
      for (int ul = 0; ok && more; ++ul) {
        const int n0 = sg.n0, n1 = sg.n1;
        more = kvm_next(a, ROWS, walk, sg);  // while this segment's first steps are on their way
        for (int n = n0; n < n1 && ok; ++n, ++g) {
          const int sl = g & 1;
          if (warp == 1) {
            const int ks = g % KS;
            ok = mbar_wait(&k_full[ks], (g / KS) & 1, wd, SITE_KVM_S);
            for (int i = 0; i < QT && ok; ++i) {
              if (n == n0) ok = mbar_wait(&q_full[i], ul & 1, wd, SITE_KVM_S);
              if (ok && g >= 2) ok = mbar_wait(&pv_done[2 * i + sl], ((g - 2) >> 1) & 1, wd, SITE_KVM_S);
              if (!ok) break;
              tc_fence_after();
              const uint64_t qd = q_desc0 + static_cast<uint32_t>(i * (QB >> 4));
              const uint64_t kd = k_desc0 + static_cast<uint32_t>((ks * TB) >> 4);
              const uint32_t d_tmem = tmem_base + i * 128 + sl * KVM_TK;
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                umma_f16_ss(d_tmem, qd + (((kk >> 2) * 16384 + (kk & 3) * 32) >> 4),
                            kd + (((kk >> 2) * (KVM_TK * 128) + (kk & 3) * 32) >> 4), IDESC_S, kk > 0 ? 1u : 0u);
              umma_commit(&s_full[2 * i + sl]);
              if (i == QT - 1) umma_commit(&k_empty[ks]);
            }
          } else {
            const int vs = g % VS;
            for (int i = 0; i < QT && ok; ++i) {
              ok = mbar_wait(&p_full[2 * i + sl], (g >> 1) & 1, wd, SITE_KVM_PV);
              if (ok && i == 0) ok = mbar_wait(&v_full[vs], (g / VS) & 1, wd, SITE_KVM_PV);
              if (ok && n == n0 && ul > 0) ok = mbar_wait(&o_empty[i], (ul - 1) & 1, wd, SITE_KVM_PV);
              if (!ok) break;
              tc_fence_after();
              const uint64_t vd = v_desc0 + static_cast<uint32_t>((vs * TB) >> 4);
              const uint32_t d_tmem = tmem_base + 256 + i * D;
              const uint32_t p_tmem = tmem_base + i * 128 + sl * KVM_TK;
#pragma unroll
              for (int kk = 0; kk < KVM_TK / 16; ++kk)
                umma_f16_ts(d_tmem, p_tmem + kk * 8, vd + static_cast<uint32_t>(kk * (2048 >> 4)), IDESC_O,
                            (n > n0 || kk > 0) ? 1u : 0u);
              umma_commit(&pv_done[2 * i + sl]);
              if (n == n1 - 1) umma_commit(&o_full[i]);
              if (i == QT - 1) umma_commit(&v_empty[vs]);
            }
          }
        }
      }
      umma_commit(drain);
      mbar_wait(drain, 0, wd, SITE_KVM_DRAIN);
    }
  } else if (warp < 4 + 4 * QT) {
    // ---------------------------------------------------------- softmax
    regs_inc<Cfg::REGS_SOFTMAX>();
    const int ti = (warp - 4) >> 2;
    const int q = warp & 3;  // TMEM lane quadrant
    const int r = q * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tS = tmem_base + ti * 128 + lane_off;
    const uint32_t tO = tmem_base + 256 + ti * D + lane_off;
    const float sl2 = a.scale_log2;
    // This row's running maximum, a score (possibly stale by 8 in the log2 domain).
    // Needed where it is raised, for large ones and for partials, so it takes no register.
    auto top = [&] { return reinterpret_cast<volatile float*>(smem + Cfg::MAX_OFFSET) + (threadIdx.x - 128); };
    bool ok = true;
    int g = 0;
    // This thread's row of a segment, and its copy of it into Q_i.
    struct RowOf {
      bool have;
      int tok, head, limit;
    };
    auto row_of = [&](const KvmSegment& u) {
      const int row = u.rb * ROWS + ti * 128 + r;
      RowOf x;
      x.have = row < u.s.n * a.group;
      const int tok = x.have ? row / a.group : 0;
      x.tok = u.s.first + tok;
      x.head = u.h * a.group + (x.have ? row - tok * a.group : 0);
      x.limit = x.have ? kv_limit(u.s, tok, a.causal) : u.s.len;
      return x;
    };
    // The warp's 32 rows of Q: D / 8 lanes a row, so that a copy instruction
    // touches few lines (a thread copying its own row: 32 of them; 4 us a unit).
    auto copy_q = [&](const RowOf& x) {
      constexpr int CH = D / 8, RPI = 32 / CH;
      const long long mine = x.tok * a.q_stride + static_cast<long long>(x.head) * D;
      const int ch = lane % CH;
      const uint32_t dst = smem_u32(sQ + ti * QB) + (ch >> 3) * 16384 + q * 32 * 128;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int rr = i * RPI + lane / CH;
        const long long off = __shfl_sync(0xffffffffu, mine, rr);
        const bool have = __shfl_sync(0xffffffffu, static_cast<int>(x.have), rr) != 0;
        const uint32_t n = have ? 16u : 0u;  // 0: filled with zeros
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + rr * 128 +
                                                                           (((ch & 7) ^ (rr & 7)) * 16)),
                     "l"(a.Q + off + ch * 8), "r"(n)
                     : "memory");
      }
    };
    auto q_in_place = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      mbar_arrive(&q_full[ti]);
    };
    bool more = kvm_next(a, ROWS, walk, sg);
    RowOf me = row_of(sg);
    if (more) {
      copy_q(me);
      q_in_place();
    }
    for (int ul = 0; ok && more; ++ul) {
      struct {
        int n0, n1, steps;
      } const cur{sg.n0, sg.n1, sg.steps};
      RowOf next{};
      const int limit = me.limit;
      float m = KV_NO_MAX;  // its product with sl2, less KV_LOG2_P; NaN for large ones
      float l = 0.f;
      *top() = KV_NO_MAX;
      for (int n = cur.n0; n < cur.n1; ++n, ++g) {
        const int sl = g & 1;
        const uint32_t tSl = tS + sl * KVM_TK;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * ti + sl], (g >> 1) & 1, wd, SITE_KVM_SOFTMAX));
        if (!ok) break;
        tc_fence_after();
        float x[64];
        {
          uint32_t v0[32], v1[32];
          tmem_ld_32x32b_x32(tSl + 0, v0);
          tmem_ld_32x32b_x32(tSl + 32, v1);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            x[i] = __uint_as_float(v0[i]);
            x[32 + i] = __uint_as_float(v1[i]);
          }
        }
        const int valid = limit - n * KVM_TK;
        if (__any_sync(0xffffffffu, valid < KVM_TK)) {
          const uint64_t seen = valid <= 0 ? 0ull : valid >= 64 ? ~0ull : (1ull << valid) - 1;
          const uint32_t lo = static_cast<uint32_t>(seen), hi = static_cast<uint32_t>(seen >> 32);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if ((lo & (1u << i)) == 0) x[i] = -INFINITY;
            if ((hi & (1u << i)) == 0) x[32 + i] = -INFINITY;
          }
        }
        const float raw = att_row_max64(x);
        const float mx = raw * sl2;
        if (__any_sync(0xffffffffu, !(mx <= m + (8.0f + KV_LOG2_P)))) {
          const bool was = __any_sync(0xffffffffu, isnan(m));
          const float old = *top();
          float y = kvm_rest(old, sl2, was);
          if (was ? raw > old : mx > m + (8.0f + KV_LOG2_P)) {
            m = fabsf(mx) < 0x1p20f ? fmaf(raw, sl2, -KV_LOG2_P) : NAN;
            *top() = raw;
            y += (old - raw) * sl2;
          }
          const bool far = __any_sync(0xffffffffu, isnan(m));
          const float factor = ex2_approx(y - kvm_rest(*top(), sl2, far));
          l *= factor;
          if (n > cur.n0 && __any_sync(0xffffffffu, factor != 1.0f)) {
            // Rescale this warp's O rows once the previous step's P V (the only
            // MMA that may still write them) is done.
            ok = __all_sync(0xffffffffu,
                            mbar_wait(&pv_done[2 * ti + (sl ^ 1)], ((g - 1) >> 1) & 1, wd, SITE_KVM_SOFTMAX));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t v[16];
              tmem_ld_32x32b_x16(tO + c * 16, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * factor);
              tmem_st_32x32b_x16(tO + c * 16, v);
            }
            tmem_st_wait();
          }
          if (far) {
            // The turns are taken as below.
            if (ti == 1 || g > 0)
              ok = mbar_wait(&turn[(1 - ti) * 4 + q], (ti == 1 ? g : g - 1) & 1, wd, SITE_KVM_SOFTMAX);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            l += kvm_exp_store64_far(sl2, *top(), valid, tSl);
            if (lane == 0) mbar_arrive(&turn[ti * 4 + q]);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&p_full[2 * ti + sl]);
            continue;
          }
        }
        // The two row tiles' warps of an SM quarter take turns at the
        // exponentials: at the same time each would take twice as long, and
        // neither would load scores or find maxima meanwhile.
        if (ti == 1 || g > 0)
          ok = mbar_wait(&turn[(1 - ti) * 4 + q], (ti == 1 ? g : g - 1) & 1, wd, SITE_KVM_SOFTMAX);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const float part = kvm_exp_store64(x, sl2, m, tSl, [&] {
          if (lane == 0) mbar_arrive(&turn[ti * 4 + q]);
        });
        l += part;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[2 * ti + sl]);
      }
      if (!ok) break;
      // The unit's last S_i is complete: Q_i takes the next unit's rows.
      more = kvm_next(a, ROWS, walk, sg);
      if (more) {
        next = row_of(sg);
        copy_q(next);
      }
      // The segment's O: out, or into a partial if the unit goes on elsewhere.
      ok = __all_sync(0xffffffffu, mbar_wait(&o_full[ti], ul & 1, wd, SITE_KVM_SOFTMAX));
      if (!ok) break;
      tc_fence_after();
      const bool whole = cur.n0 == 0 && cur.n1 == cur.steps;
      // 4-bit values lie as elements 0 4 1 5 2 6 3 7 in each 8 columns.
      auto column = [](int k) { return BITS == 4 ? (k < 4 ? 2 * k : 2 * (k - 4) + 1) : k; };
      if (whole) {
        const float inv_l = l > 0.f ? 1.0f / l : 0.f;
        uint32_t out[D / 2];  // the row in fp16: O's columns are free before it is stored
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tO + c * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            out[c * 16 + i / 2] = pack_half2(__uint_as_float(o[(i & ~7) + column(i & 7)]) * inv_l,
                                             __uint_as_float(o[(i & ~7) + column((i & 7) + 1)]) * inv_l);
        }
        tc_fence_before();
        mbar_arrive(&o_empty[ti]);
        if (more) q_in_place();
        // Rows go out through shared memory, 32 elements at a time, four lanes to
        // a row.
        uint8_t* stage = smem + Cfg::OUT_OFFSET + (warp - 4) * Cfg::OUT_BYTES;
        const long long mine = me.tok * a.o_stride + static_cast<long long>(me.head) * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stage + lane * Cfg::OUT_ROW + i * 16) =
                make_uint4(out[c * 16 + 4 * i], out[c * 16 + 4 * i + 1], out[c * 16 + 4 * i + 2],
                           out[c * 16 + 4 * i + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rr = i * 8 + (lane >> 2);
            const long long off = __shfl_sync(0xffffffffu, mine, rr);
            const bool have = __shfl_sync(0xffffffffu, static_cast<int>(me.have), rr) != 0;
            if (have)
              *reinterpret_cast<uint4*>(a.O + off + c * 32 + (lane & 3) * 8) =
                  *reinterpret_cast<const uint4*>(stage + rr * Cfg::OUT_ROW + (lane & 3) * 16);
          }
        }
        if (a.lse != nullptr) {
          const float fix = ex2_approx(kvm_rest(*top(), sl2, __any_sync(0xffffffffu, isnan(m))));
          if (me.have) a.lse[static_cast<long long>(me.tok) * a.heads_q + me.head] = kv_lse(*top(), l * fix, sl2);
        }
      } else {
        float* part = a.partials + kvm_slot<D, ROWS>(2ll * blockIdx.x + (cur.n0 == 0 ? 1 : 0));
        float4* dst = reinterpret_cast<float4*>(part) + ti * 128 + r;
        // Partials of a row then differ by their maxima alone.
        const float fix = ex2_approx(kvm_rest(*top(), sl2, __any_sync(0xffffffffu, isnan(m))));
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld_32x32b_x32(tO + c * 32, o);
          tmem_ld_wait();
          if (me.have) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              dst[(c * 8 + i / 4) * ROWS] = make_float4(
                  __uint_as_float(o[(i & ~7) + column(i & 7)]) * fix,
                  __uint_as_float(o[(i & ~7) + column((i & 7) + 1)]) * fix,
                  __uint_as_float(o[(i & ~7) + column((i & 7) + 2)]) * fix,
                  __uint_as_float(o[(i & ~7) + column((i & 7) + 3)]) * fix);
          }
        }
        __syncwarp();
        tc_fence_before();
        mbar_arrive(&o_empty[ti]);
        if (more) q_in_place();
        if (me.have) {
          part[ROWS * D + ti * 128 + r] = *top();
          part[ROWS * D + ROWS + ti * 128 + r] = l * fix;
        }
      }
      me = next;
    }
  } else {
    // ---------------------------------------------------------- codes to fp16
    regs_dec<Cfg::REGS_UNPACK>();
    constexpr int GR = D / KV_GROUP;          // groups of a row
    constexpr int RW = 32 / GR;               // rows of a warp at a time
    constexpr int PASSES = KVM_TK / (RW * 4);
    const int uw = warp - 12;
    // Eight lanes take eight rows and one group: the row pitches (80, 144, 40,
    // 72 bytes) and the swizzle then put their accesses on different banks.
    const int sub = (lane & 7) + 8 * (lane / (8 * GR));
    const int gr = (lane >> 3) % GR;
    const uint32_t k1024 = __shfl_sync(0xffffffffu, a.k1024, 0);
    // Places of this thread's first row in a raw stage and of its four chunks in
    // a tile; later passes and V lie at constant distances (rows go up by a
    // multiple of 8, so the swizzle stays).
    constexpr int PASS_ROWS = 4 * RW;
    const int row0 = uw * RW + sub;
    const uint32_t raw0 = smem_u32(sR) + row0 * RB, codes0 = raw0 + gr * (KV_GROUP * BITS / 8),
                   par0 = raw0 + Row::CODES + gr * 4;
    uint32_t chunk0[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int ch = gr * 4 + c;
      chunk0[c] = smem_u32(sK) + (ch >> 3) * (KVM_TK * 128) + row0 * 128 + (((ch & 7) ^ (row0 & 7)) * 16);
    }
    int g = 0, rs = 0, ks = 0, vs = 0;  // step, and its place in each ring
    bool ok = true;
    while (ok && kvm_next(a, ROWS, walk, sg)) {
      for (int n = sg.n0; n < sg.n1 && ok; ++n, ++g) {
        ok = mbar_wait(&r_full[rs], (g / RS) & 1, wd, SITE_KVM_UNPACK);
        const int valid = sg.s.len - n * KVM_TK;
        const bool tail = valid < KVM_TK;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int depth = kv == 0 ? KS : VS;
          if (ok && g >= depth)
            ok = mbar_wait(kv == 0 ? &k_empty[ks] : &v_empty[vs], (g / depth - 1) & 1, wd, SITE_KVM_UNPACK);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t to = kv == 0 ? ks * TB : KS * TB + vs * TB;
          const uint32_t from = rs * Cfg::RAW_BYTES;
#pragma unroll
          for (int p = 0; p < PASSES; ++p) {
            const int skip = (kv * KVM_TK + p * PASS_ROWS) * RB;
            uint32_t par;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(par) : "r"(par0 + from + skip));
            // Rows behind the sequence hold anything; their values count as 0.
            if (tail && row0 + p * PASS_ROWS >= valid) par = 0u;
            const __half2 s2 = __low2half2(as_half2(par)), z2 = __high2half2(as_half2(par));
            constexpr int WORDS = KV_GROUP * BITS / 32;
            uint32_t w[WORDS];
            if constexpr (RB % 16 == 0) {
#pragma unroll
              for (int i = 0; i < WORDS; i += 4)
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                             : "r"(codes0 + from + skip + 4 * i));
            } else {
#pragma unroll
              for (int i = 0; i < WORDS; i += 2)
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                             : "=r"(w[i]), "=r"(w[i + 1])
                             : "r"(codes0 + from + skip + 4 * i));
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // 8 elements, 16 bytes
              uint4 out;
              if constexpr (BITS == 4) {
                __half2 h[4];
                kv_codes4(w[c], h, k1024);
                const uint32_t p0 = as_u32(__hfma2(h[0], s2, z2)), p1 = as_u32(__hfma2(h[1], s2, z2)),
                               p2 = as_u32(__hfma2(h[2], s2, z2)), p3 = as_u32(__hfma2(h[3], s2, z2));
                // K in the order of Q's elements; V as it comes (columns of O).
                if (kv == 0)
                  out = make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410),
                                   __byte_perm(p0, p1, 0x7632), __byte_perm(p2, p3, 0x7632));
                else
                  out = make_uint4(p0, p1, p2, p3);
              } else {
                out.x = as_u32(__hfma2(kv_codes8(w[2 * c], 0x4140), s2, z2));
                out.y = as_u32(__hfma2(kv_codes8(w[2 * c], 0x4342), s2, z2));
                out.z = as_u32(__hfma2(kv_codes8(w[2 * c + 1], 0x4140), s2, z2));
                out.w = as_u32(__hfma2(kv_codes8(w[2 * c + 1], 0x4342), s2, z2));
              }
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk0[c] + to + p * PASS_ROWS * 128),
                           "r"(out.x), "r"(out.y), "r"(out.z), "r"(out.w)
                           : "memory");
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(kv == 0 ? &k_full[ks] : &v_full[vs]);
        }
        if (ok && lane == 0) mbar_arrive(&r_empty[rs]);
        rs = rs + 1 == RS ? 0 : rs + 1;
        ks = ks + 1 == KS ? 0 : ks + 1;
        vs = vs + 1 == VS ? 0 : vs + 1;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the partials of units that several CTAs share: block (w, c) 32 rows of
// the unit that worker w began and left to others. Lane = row; a warp takes D / 8
// elements of them.
template <int D, int ROWS>
__global__ void __launch_bounds__(256) kv_attention_many_join_kernel(const __grid_constant__ KvAttnArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int G4 = D / 32;  // groups of 4 elements a warp
  const int w = blockIdx.x;
  kv_wait_for_previous();  // in every block: what follows this kernel also follows the one before it
  const int4 left = __ldcg(reinterpret_cast<const int4*>(kvm_shared<D, ROWS>(a) + w));
  const KvmShared p{left.x, left.y, left.z, left.w};
  const int last = p.last;
  if (last < 0) return;
  const KvSequence s = kvm_sequence(a, p.b);
  const int local = blockIdx.y * 32 + lane;
  const int row = p.rb * ROWS + local;
  if (row >= s.n * a.group) return;
  float m = KV_NO_MAX, l = 0.f, acc[G4][4];
#pragma unroll
  for (int i = 0; i < G4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
  for (int k = w; k <= last; ++k) {
    const float* part = a.partials + kvm_slot<D, ROWS>(2ll * k + (k == w ? 1 : 0));
    const float pm = __ldcg(part + ROWS * D + local), pl = __ldcg(part + ROWS * D + ROWS + local);
    const float m_new = fmaxf(m, pm), f = kv_ex2((m - m_new) * a.scale_log2), fp = kv_ex2((pm - m_new) * a.scale_log2);
    m = m_new;
    l = l * f + pl * fp;
#pragma unroll
    for (int i = 0; i < G4; ++i) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(part) + (warp * G4 + i) * ROWS + local);
      acc[i][0] = acc[i][0] * f + v.x * fp;
      acc[i][1] = acc[i][1] * f + v.y * fp;
      acc[i][2] = acc[i][2] * f + v.z * fp;
      acc[i][3] = acc[i][3] * f + v.w * fp;
    }
  }
  const long long token = s.first + row / a.group;
  const int head = p.h * a.group + row % a.group;
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  __half* out = a.O + token * a.o_stride + static_cast<long long>(head) * D + warp * (D / 8);
#pragma unroll
  for (int i = 0; i < G4; ++i)
    *reinterpret_cast<uint2*>(out + 4 * i) = make_uint2(pack_half2(acc[i][0] * inv, acc[i][1] * inv),
                                                        pack_half2(acc[i][2] * inv, acc[i][3] * inv));
  if (a.lse != nullptr && warp == 0) a.lse[token * a.heads_q + head] = kv_lse(m, l, a.scale_log2);
}

}  // namespace mm4
