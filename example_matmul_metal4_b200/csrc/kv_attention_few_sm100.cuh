// Attention over the key / value cache for few rows: up to 16 rows of a unit
// (a token or a few, times the query heads that share a key / value head).
//
// Bound by the cache's bytes: each is read once, 160 a token and head at
// D = 128 in 4 bits, and the arithmetic has to hide behind them: at 6.4 TB/s
// an SM has about 40 elements of K or V a clock to unpack, scale and multiply.
//  - Every warp works alone: it copies its tiles of 32 keys into its own ring in
//    shared memory (untiled bulk copies, a page is contiguous) and needs no
//    barrier with other warps.
//  - S^T = K Q^T and O^T += V^T P^T on m16n8k16 tensor instructions, with the
//    cache as the 16-row operand and the rows of Q as the 8 columns: half
//    the tensor work of a form with 16 padded rows of Q.
//  - A lane takes the elements of one word for its share of the contraction
//    (Q's fragments are built in the same order), so codes go from a word to
//    operand registers by logic instructions and one fp16 fused multiply-add a
//    pair; no shuffles. For V the pairs are two keys of one element: one byte
//    permute per two words.
//  - The running maximum is raised only when a score exceeds it by 2^8 (log2
//    domain), which one vote per tile decides; the stale maximum cancels in
//    O / l.
#pragma once

#include "kv_attention_sm100.cuh"

namespace mm4 {

constexpr int KVF_TK = 32;  // keys of a tile

template <int D, int BITS, int NT>
struct KvFew {
  static constexpr int ROWS = 8 * NT;
  static constexpr int ROW_BYTES = KvRow<D, BITS>::BYTES;
  static constexpr int STAGE_BYTES = 2 * KVF_TK * ROW_BYTES;  // K rows, then V rows
  // Warps a CTA and tiles in flight a warp: up to 164 KB of copies in flight.
  static constexpr int WARPS = NT == 1 && STAGE_BYTES <= 5120 ? 16 : 8;
  static constexpr int STAGES = STAGE_BYTES * WARPS * 4 <= 168 * 1024 ? 4 : 2;
  static constexpr int SLOTS = WARPS / 2;                     // of the join inside a CTA
  static constexpr int RING_BYTES = WARPS * STAGES * STAGE_BYTES;
  static constexpr int SMEM_BYTES = RING_BYTES + SLOTS * KvPartial<D, ROWS>::FLOATS * 4 + WARPS * STAGES * 8;
};

__device__ __forceinline__ void kv_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t kv_transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// N consecutive 32-bit words from shared memory in the widest loads that the
// rows' pitch allows (72 and 40 bytes: 8).
template <int N, bool WIDE>
__device__ __forceinline__ void kv_load_words(const uint8_t* p, uint32_t (&w)[N]) {
  static_assert(N == 1 || N % 2 == 0, "word count");
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2 || !WIDE) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p + 4 * i);
      w[i] = v.x;
      w[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x;
      w[i + 1] = v.y;
      w[i + 2] = v.z;
      w[i + 3] = v.w;
    }
  }
}

// Pairs of K's operand from one word of codes, in the order of kv_query_pairs:
// 4 bits (0,4) (1,5) (2,6) (3,7); 8 bits (0,1) (2,3).
template <int BITS>
__device__ __forceinline__ void kv_key_pairs(uint32_t w, __half2 s2, __half2 z2, uint32_t (&out)[16 / BITS]) {
  if constexpr (BITS == 4) {
    __half2 c[4];
    kv_codes4(w, c);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = as_u32(__hfma2(c[j], s2, z2));
  } else {
    out[0] = as_u32(__hfma2(kv_codes8(w, 0x4140), s2, z2));
    out[1] = as_u32(__hfma2(kv_codes8(w, 0x4342), s2, z2));
  }
}

// V's operand for one word of two keys: out[e] = (element e of key a, of key b).
template <int BITS>
__device__ __forceinline__ void kv_value_pairs(uint32_t wa, uint32_t wb, __half2 s2, __half2 z2,
                                               uint32_t (&out)[32 / BITS]) {
  const uint32_t lo = __byte_perm(wa, wb, 0x5410), hi = __byte_perm(wa, wb, 0x7632);
  if constexpr (BITS == 4) {
    __half2 c[4];
    kv_codes4(lo, c);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = as_u32(__hfma2(c[j], s2, z2));
    kv_codes4(hi, c);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[4 + j] = as_u32(__hfma2(c[j], s2, z2));
  } else {
    const __half2 m1024 = __float2half2_rn(-1024.0f);
    out[0] = as_u32(__hfma2(__hadd2(kv_bits_1024(lo, 0x00FF00FFu), m1024), s2, z2));
    out[1] = as_u32(__hfma2(__hadd2(kv_bits_1024(lo >> 8, 0x00FF00FFu), m1024), s2, z2));
    out[2] = as_u32(__hfma2(__hadd2(kv_bits_1024(hi, 0x00FF00FFu), m1024), s2, z2));
    out[3] = as_u32(__hfma2(__hadd2(kv_bits_1024(hi >> 8, 0x00FF00FFu), m1024), s2, z2));
  }
}

// One warp walks its range. Lane = 4 g + c: in K Q^T it has keys g and g + 8 of
// each 16, the c-th quarter of the head dimension, and rows 2 c and 2 c + 1
// of the result; in V^T P^T the g-th eighth of the head dimension and keys 2 c,
// 2 c + 1, 2 c + 8, 2 c + 9.
//
// TEAM: a CTA takes whole units, its warps every WARPS-th tile of each, and
// joins them in shared memory: one launch and no workspace, for caches that
// hold few keys a sequence. Otherwise a worker is a warp (worker index =
// warp * CTAs + CTA, so few workers spread over the SMs).
template <int D, int BITS, int NT, bool TEAM>
__global__ void __launch_bounds__(KvFew<D, BITS, NT>::WARPS * 32, 1) kv_attention_few_kernel(const KvAttnArgs a) {
  using Cfg = KvFew<D, BITS, NT>;
  using Row = KvRow<D, BITS>;
  constexpr int W = Cfg::WARPS, ST = Cfg::STAGES, RB = Cfg::ROW_BYTES;
  constexpr int KC = D / 4;               // elements of a lane's share of a key row
  constexpr int KW = KC * BITS / 32;      // words of it
  constexpr int VC = D / 8;               // elements of a lane's share of a value row
  constexpr int VW = VC * BITS / 32;
  constexpr int MT = D / 16;              // 16-element tiles of O^T

  extern __shared__ __align__(128) uint8_t kvf_smem[];
  const KvBatch& kb = a.kb;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  uint8_t* ring = kvf_smem + warp * ST * Cfg::STAGE_BYTES;
  float* join = reinterpret_cast<float*>(kvf_smem + Cfg::RING_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(kvf_smem + Cfg::SMEM_BYTES) - W * ST + warp * ST;
  const Watchdog wd{&g_kv_wait, a.timeout_ns};
  if (lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  if (!TEAM) kv_launch_dependents();

  // The range: tiles left of the loader and of the consumer, and their places.
  struct Place {
    int b, h, n, tiles;
    KvSequence s;
  };
  long long todo = 0;  // tiles of this warp (TEAM: units of this CTA)
  Place at{};
  if constexpr (TEAM) {
    const long long units = static_cast<long long>(kb.sequences) * kb.heads_kv;
    todo = (units - blockIdx.x + gridDim.x - 1) / gridDim.x;
    if (todo <= 0) return;
    at.b = static_cast<int>(blockIdx.x / kb.heads_kv);
    at.h = static_cast<int>(blockIdx.x % kb.heads_kv);
    at.n = warp;
  } else {
    const long long total = kv_total_tiles<KVF_TK>(kb, lane) * kb.heads_kv;
    const long long active = min(static_cast<long long>(a.workers), total);
    const long long w = static_cast<long long>(warp) * gridDim.x + blockIdx.x;
    if (w >= active) return;
    const long long x = kv_range_begin(w, total, active);
    todo = kv_range_begin(w + 1, total, active) - x;
    long long before;
    at.b = kv_find_tile<KVF_TK>(kb, x / kb.heads_kv, lane, &before);
    // x / heads lies in this sequence: its tiles start at heads * before.
    at.s = kv_sequence(kb, at.b);
    at.tiles = kv_tiles<KVF_TK>(at.s);
    const long long in = x - before * kb.heads_kv;
    at.h = static_cast<int>(in / at.tiles);
    at.n = static_cast<int>(in % at.tiles);
  }

  // Moves to the next unit.
  auto next_unit = [&](Place& p) {
    if constexpr (TEAM) {
      const long long u = static_cast<long long>(p.b) * kb.heads_kv + p.h + gridDim.x;
      p.b = static_cast<int>(u / kb.heads_kv);
      p.h = static_cast<int>(u % kb.heads_kv);
      p.n = warp;
    } else {
      p.n = 0;
      if (++p.h == kb.heads_kv) {
        p.h = 0;
        ++p.b;
      }
    }
  };
  auto read_sequence = [&](Place& p) {
    p.s = kv_sequence(kb, p.b);
    p.tiles = kv_tiles<KVF_TK>(p.s);
  };

  // ------------------------------------------------------------ loader
  Place ld = at;
  long long ld_todo = todo;   // TEAM: units, else tiles
  int ids_b = -1, ids_base = 0, ids = 0;  // 32 page numbers of sequence ids_b from ids_base, one a lane
  int loaded = 0;             // tiles issued
  // Skips sequences without rows (and, in TEAM, units whose tiles end before
  // this warp's first); false when the range is done.
  auto settle = [&](Place& p, long long& left) -> bool {
    while (left > 0 && p.b < kb.sequences) {
      read_sequence(p);
      if (p.n < p.tiles) return true;
      next_unit(p);
      if (TEAM) --left;
    }
    return false;
  };
  bool ld_have = settle(ld, ld_todo);
  auto load_next = [&]() {
    if (!ld_have) return;
    const int st = loaded % ST;
    uint8_t* dst = ring + st * Cfg::STAGE_BYTES;
    const int key0 = ld.n * KVF_TK;
    const int valid = ld.s.len - key0;  // <= 0 only for a sequence of length 0
    const int ps = 1 << kb.page_shift;
    const int chunk = min(KVF_TK, ps);  // keys of a copy
    const int copies = valid <= 0 ? 0 : (valid > chunk && chunk < KVF_TK) ? 2 : 1;
    if (copies > 0) {
      const int first = key0 >> kb.page_shift;
      if (ids_b != ld.b || first < ids_base || first + copies > ids_base + 32) {
        ids_b = ld.b;
        ids_base = first;
        const int i = first + lane;
        ids = 0;
        if (i < kb.pages_per_seq && (i << kb.page_shift) < ld.s.len) {
          ids = __ldg(kb.table + static_cast<long long>(ld.b) * kb.pages_per_seq + i);
          if (ids < 0 || ids >= kb.pages) {
            kv_note(KV_DATA_PAGE);
            ids = 0;  // read in place of the page outside the pool
          }
        }
      }
      const int mine = lane >> 1, kv = lane & 1;  // lanes 0 .. 2 copies - 1 issue one copy each
      const int page = __shfl_sync(0xffffffffu, ids, min(31, first - ids_base + min(mine, copies - 1)));
      const uint32_t bytes = static_cast<uint32_t>(chunk * RB);
      if (lane == 0) mbar_arrive_expect_tx(&bars[st], bytes * 2 * copies);
      __syncwarp();
      if (mine < copies) {
        const uint8_t* src = a.cache + page * kb.page_bytes +
                             (static_cast<long long>((ld.h * 2 + kv) << kb.page_shift) + (key0 & (ps - 1))) * RB;
        bulk_load(dst + (kv * KVF_TK + mine * chunk) * RB, src, bytes, &bars[st]);
      }
    } else if (lane == 0) {
      mbar_arrive(&bars[st]);
    }
    ++loaded;
    if constexpr (TEAM) {
      ld.n += W;
      if (ld.n >= ld.tiles) {
        next_unit(ld);
        --ld_todo;
        ld_have = settle(ld, ld_todo);
      }
    } else {
      --ld_todo;
      if (++ld.n == ld.tiles) {
        next_unit(ld);
        ld_have = settle(ld, ld_todo);
      } else {
        ld_have = ld_todo > 0;
      }
    }
  };
  for (int i = 0; i < ST; ++i) load_next();

  // ------------------------------------------------------------ consumer
  uint32_t q[NT][D / 16][2];
  float acc[NT][MT][4];
  float m[NT][2], l[NT][2];
  int limit[NT][2];
  int used = 0;  // tiles consumed
  bool ok = true;
  const float sl2 = a.scale_log2;

  auto start_unit = [&](const Place& p) {
    const int rows = min(p.s.n * a.group, Cfg::ROWS);
    if (static_cast<long long>(p.s.n) * a.group > Cfg::ROWS || p.s.n > kb.max_new) kv_note(KV_DATA_NEW);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const bool have = r < rows;
      const int tok = have ? r / a.group : 0, hd = have ? r % a.group : 0;
      const uint4* src = reinterpret_cast<const uint4*>(
          a.Q + (p.s.first + tok) * a.q_stride + static_cast<long long>(p.h * a.group + hd) * D + c * KC);
      uint4 v[KC / 8];
#pragma unroll
      for (int i = 0; i < KC / 8; ++i) v[i] = have ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < KC / 8; ++i) {
        if constexpr (BITS == 4) {
          q[nt][2 * i][0] = __byte_perm(v[i].x, v[i].z, 0x5410);      // (0, 4)
          q[nt][2 * i][1] = __byte_perm(v[i].x, v[i].z, 0x7632);      // (1, 5)
          q[nt][2 * i + 1][0] = __byte_perm(v[i].y, v[i].w, 0x5410);  // (2, 6)
          q[nt][2 * i + 1][1] = __byte_perm(v[i].y, v[i].w, 0x7632);  // (3, 7)
        } else {
          q[nt][2 * i][0] = v[i].x;
          q[nt][2 * i][1] = v[i].y;
          q[nt][2 * i + 1][0] = v[i].z;
          q[nt][2 * i + 1][1] = v[i].w;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nt * 8 + 2 * c + e;
        limit[nt][e] = row < rows ? kv_limit(p.s, row / a.group, a.causal) : p.s.len;
        m[nt][e] = KV_NO_MAX;
        l[nt][e] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][t][e] = 0.f;
    }
  };

  auto tile = [&](const Place& p) {
    const uint8_t* sk = ring + (used % ST) * Cfg::STAGE_BYTES;
    const uint8_t* sv = sk + KVF_TK * RB;
    const int key0 = p.n * KVF_TK;
    // S^T for 2 x 16 keys.
    float s[2][NT][4];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint8_t* ka = sk + (hf * 16 + g) * RB;
      const uint8_t* kb8 = ka + 8 * RB;
      uint32_t wa[KW], wb[KW];
      kv_load_words<KW, RB % 16 == 0>(ka + c * (KC * BITS / 8), wa);
      kv_load_words<KW, RB % 16 == 0>(kb8 + c * (KC * BITS / 8), wb);
      const __half2 pa = *reinterpret_cast<const __half2*>(ka + Row::CODES + (c * KC / KV_GROUP) * 4);
      const __half2 pb = *reinterpret_cast<const __half2*>(kb8 + Row::CODES + (c * KC / KV_GROUP) * 4);
      const __half2 sa = __low2half2(pa), za = __high2half2(pa), sb = __low2half2(pb), zb = __high2half2(pb);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[hf][nt][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        uint32_t xa[16 / BITS], xb[16 / BITS];
        kv_key_pairs<BITS>(wa[i], sa, za, xa);
        kv_key_pairs<BITS>(wb[i], sb, zb, xb);
#pragma unroll
        for (int j = 0; j < 8 / BITS; ++j) {
          const int step = i * (8 / BITS) + j;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            kv_mma(s[hf][nt], xa[2 * j], xb[2 * j], xa[2 * j + 1], xb[2 * j + 1], q[nt][step][0], q[nt][step][1]);
        }
      }
    }
    // Masks: keys at and behind a row's limit.
    bool inside = true;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) inside = inside && key0 + KVF_TK <= limit[nt][0] && key0 + KVF_TK <= limit[nt][1];
    inside = __all_sync(0xffffffffu, inside);
    if (!inside) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + hf * 16 + g + (e >> 1) * 8 >= limit[nt][e & 1]) s[hf][nt][e] = -INFINITY;
    }
    // The running maximum, raised when a score is over it by more than 8.
    bool grow = false;
    float mx[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[nt][e] = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2])) * sl2;
        grow = grow || mx[nt][e] > m[nt][e] + 8.0f;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = mx[nt][e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float m_new = fmaxf(m[nt][e], x);
          const float f = kv_ex2(m[nt][e] - m_new);
          m[nt][e] = m_new;
          l[nt][e] *= f;
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            acc[nt][t][e] *= f;
            acc[nt][t][e + 2] *= f;
          }
        }
    }
    // P, its sums, and P^T as an operand.
    uint32_t pt[2][NT][2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p4[e] = kv_ex2(fmaf(s[hf][nt][e], sl2, -m[nt][e & 1]));
          l[nt][e & 1] += p4[e];
        }
        pt[hf][nt][0] = kv_transpose(pack_half2(p4[0], p4[1]));
        pt[hf][nt][1] = kv_transpose(pack_half2(p4[2], p4[3]));
      }
    // O^T += V^T P^T. Rows behind the sequence hold anything: their scale and
    // zero count as 0, so the product with P = 0 is 0.
    const int valid = p.s.len - key0;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      uint32_t w4[4][VW];
      __half2 par[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = hf * 16 + 2 * c + (i & 1) + (i >> 1) * 8;
        const uint8_t* row = sv + key * RB;
        kv_load_words<VW, RB % 16 == 0>(row + g * (VC * BITS / 8), w4[i]);
        par[i] = *reinterpret_cast<const __half2*>(row + Row::CODES + (g * VC / KV_GROUP) * 4);
        if (key >= valid) par[i] = __float2half2_rn(0.f);
      }
      const __half2 s01 = __lows2half2(par[0], par[1]), z01 = __highs2half2(par[0], par[1]);
      const __half2 s23 = __lows2half2(par[2], par[3]), z23 = __highs2half2(par[2], par[3]);
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        uint32_t x[32 / BITS], y[32 / BITS];
        kv_value_pairs<BITS>(w4[0][i], w4[1][i], s01, z01, x);
        kv_value_pairs<BITS>(w4[2][i], w4[3][i], s23, z23, y);
#pragma unroll
        for (int j = 0; j < 16 / BITS; ++j) {
          const int t = i * (16 / BITS) + j;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            kv_mma(acc[nt][t], x[2 * j], x[2 * j + 1], y[2 * j], y[2 * j + 1], pt[hf][nt][0], pt[hf][nt][1]);
        }
      }
    }
  };

  // Sums l over the lanes that share a row.
  auto sum_l = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      }
  };
  // Stores the rows of a partial: this lane's VC elements of rows 2 c, 2 c + 1.
  auto store_partial = [&](float* dst, int rows) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nt * 8 + 2 * c + e;
        if (row >= rows) continue;
        float4* out = reinterpret_cast<float4*>(dst + row * D + g * VC);
#pragma unroll
        for (int t = 0; t < MT; t += 2)
          out[t / 2] = make_float4(acc[nt][t][e], acc[nt][t][e + 2], acc[nt][t + 1][e], acc[nt][t + 1][e + 2]);
        if (g == 0) {
          dst[Cfg::ROWS * D + 2 * row] = m[nt][e];
          dst[Cfg::ROWS * D + 2 * row + 1] = l[nt][e];
        }
      }
  };
  auto output_row = [&](const Place& p, int row, __half** o, float** lse) {
    const long long tok = p.s.first + row / a.group;
    const int head = p.h * a.group + row % a.group;
    *o = a.O + tok * a.o_stride + static_cast<long long>(head) * D;
    *lse = a.lse ? a.lse + tok * a.heads_q + head : nullptr;
  };

  if constexpr (!TEAM) {
    float* slots = a.partials + 2 * (static_cast<long long>(warp) * gridDim.x + blockIdx.x) * KvPartial<D, Cfg::ROWS>::FLOATS;
    while (todo > 0 && ok) {
      if (!settle(at, todo)) break;
      start_unit(at);
      const int n0 = at.n;
      const int n1 = static_cast<int>(min(static_cast<long long>(at.tiles), at.n + todo));
      for (; at.n < n1; ++at.n) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars[used % ST], (used / ST) & 1, wd, 110));
        if (!ok) break;
        tile(at);
        __syncwarp();
        ++used;
        load_next();
      }
      todo -= n1 - n0;
      sum_l();
      const int rows = min(at.s.n * a.group, Cfg::ROWS);
      if (n0 == 0 && n1 == at.tiles) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = nt * 8 + 2 * c + e;
            if (row >= rows) continue;
            __half* o;
            float* lse;
            output_row(at, row, &o, &lse);
            const float inv = l[nt][e] > 0.f ? 1.0f / l[nt][e] : 0.f;
            uint4* out = reinterpret_cast<uint4*>(o + g * VC);
#pragma unroll
            for (int t = 0; t < MT; t += 4)
              out[t / 4] = make_uint4(pack_half2(acc[nt][t][e] * inv, acc[nt][t][e + 2] * inv),
                                      pack_half2(acc[nt][t + 1][e] * inv, acc[nt][t + 1][e + 2] * inv),
                                      pack_half2(acc[nt][t + 2][e] * inv, acc[nt][t + 2][e + 2] * inv),
                                      pack_half2(acc[nt][t + 3][e] * inv, acc[nt][t + 3][e + 2] * inv));
            if (lse != nullptr && g == 0) *lse = (m[nt][e] + log2f(l[nt][e])) * 0.6931471805599453f;
          }
      } else {
        store_partial(slots + (n0 == 0 ? KvPartial<D, Cfg::ROWS>::FLOATS : 0), rows);
      }
      if (n1 == at.tiles) next_unit(at);
    }
  } else {
    while (todo > 0) {  // every warp of the CTA walks the same units
      read_sequence(at);
      if (at.tiles > 0) {
        start_unit(at);
        const int rows = min(at.s.n * a.group, Cfg::ROWS);
        for (; at.n < at.tiles && ok; at.n += W) {
          ok = __all_sync(0xffffffffu, mbar_wait(&bars[used % ST], (used / ST) & 1, wd, 111));
          if (!ok) break;
          tile(at);
          __syncwarp();
          ++used;
          load_next();
        }
        sum_l();
        // Two rounds: the upper half of the warps hands over to the lower, then
        // all threads sum the lower half's slots.
        constexpr int F = KvPartial<D, Cfg::ROWS>::FLOATS;
        if (warp >= Cfg::SLOTS) store_partial(join + (warp - Cfg::SLOTS) * F, rows);
        __syncthreads();
        if (warp < Cfg::SLOTS) {
          const float* other = join + warp * F;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = nt * 8 + 2 * c + e;
              if (row >= rows) continue;
              const float m2 = other[Cfg::ROWS * D + 2 * row], l2 = other[Cfg::ROWS * D + 2 * row + 1];
              const float mm = fmaxf(m[nt][e], m2), f1 = kv_ex2(m[nt][e] - mm), f2 = kv_ex2(m2 - mm);
              m[nt][e] = mm;
              l[nt][e] = l[nt][e] * f1 + l2 * f2;
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                acc[nt][t][e] = acc[nt][t][e] * f1 + other[row * D + g * VC + 2 * t] * f2;
                acc[nt][t][e + 2] = acc[nt][t][e + 2] * f1 + other[row * D + g * VC + 2 * t + 1] * f2;
              }
            }
        }
        __syncwarp();
        if (warp < Cfg::SLOTS) store_partial(join + warp * F, rows);
        __syncthreads();
        for (int i = threadIdx.x; i < rows * (D / 2); i += W * 32) {
          const int row = i / (D / 2), d = (i % (D / 2)) * 2;
          float mm = KV_NO_MAX;
#pragma unroll
          for (int k = 0; k < Cfg::SLOTS; ++k) mm = fmaxf(mm, join[k * F + Cfg::ROWS * D + 2 * row]);
          float ls = 0.f, x = 0.f, y = 0.f;
#pragma unroll
          for (int k = 0; k < Cfg::SLOTS; ++k) {
            const float f = kv_ex2(join[k * F + Cfg::ROWS * D + 2 * row] - mm);
            ls += f * join[k * F + Cfg::ROWS * D + 2 * row + 1];
            x += f * join[k * F + row * D + d];
            y += f * join[k * F + row * D + d + 1];
          }
          __half* o;
          float* lse;
          output_row(at, row, &o, &lse);
          const float inv = ls > 0.f ? 1.0f / ls : 0.f;
          *reinterpret_cast<__half2*>(o + d) = __floats2half2_rn(x * inv, y * inv);
          if (lse != nullptr && d == 0) *lse = (mm + log2f(ls)) * 0.6931471805599453f;
        }
        __syncthreads();  // the slots are free for the next unit
      }
      next_unit(at);
      --todo;
    }
  }
  // Copies still in flight after a run-out wait land before the CTA ends.
  for (; used < loaded; ++used) mbar_wait(&bars[used % ST], (used / ST) & 1, wd, 112);
}

// Joins the partials of the units that several workers share: a block of 8
// warps per unit and 8 rows, (row, part of the partials) to a warp, parts
// joined in shared memory in order. Launched to overlap the tail of the
// kernel before it, which it waits for before it reads a partial.
template <int D, int ROWS, int TK>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(const KvAttnArgs a) {
  constexpr int F = KvPartial<D, ROWS>::FLOATS;
  constexpr int V = D / 32;  // floats of a lane
  __shared__ float part[8][D + 2];
  const KvBatch& kb = a.kb;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = static_cast<int>(blockIdx.x / kb.heads_kv), h = static_cast<int>(blockIdx.x % kb.heads_kv);
  const KvSequence s = kv_sequence(kb, b);
  const int row0 = blockIdx.y * 8;
  const int rows = min(min(s.n * a.group, ROWS) - row0, 8);
  const long long total = kv_total_tiles<TK>(kb, lane) * kb.heads_kv;
  const long long active = min(static_cast<long long>(a.workers), total);
  const int tiles = kv_tiles<TK>(s);
  long long first = 0, last = 0;
  if (rows > 0) {
    const long long x0 = kv_tiles_before<TK>(kb, b, lane) * kb.heads_kv + static_cast<long long>(h) * tiles;
    first = kv_worker_of(x0, total, active);
    last = kv_worker_of(x0 + tiles - 1, total, active);
  }
  kv_wait_for_previous();  // in every block: what follows this kernel also follows the one before it
  if (rows <= 0 || first == last) return;
  int per = 1;  // rows rounded up to a power of two, so that parts are whole
  while (per < rows) per *= 2;
  const int parts = 8 / per, row = warp % per, mine = warp / per;
  const int count = static_cast<int>(last - first + 1);
  const int c0 = static_cast<int>(static_cast<long long>(mine) * count / parts),
            c1 = static_cast<int>(static_cast<long long>(mine + 1) * count / parts);
  float mm = KV_NO_MAX, ls = 0.f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  if (row < rows) {
    auto slot = [&](int i) { return a.partials + (2 * (first + i) + (i == 0 ? 1 : 0)) * F; };
    for (int i0 = c0; i0 < c1; i0 += 32) {
      const int n = min(32, c1 - i0);
      float pm = KV_NO_MAX, pl = 0.f;
      if (lane < n) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(slot(i0 + lane) + ROWS * D + 2 * (row0 + row)));
        pm = ml.x;
        pl = ml.y;
      }
      float top = pm;
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
      const float m_new = fmaxf(mm, top), f = kv_ex2(mm - m_new), w = kv_ex2(pm - m_new);
      mm = m_new;
      ls *= f;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= f;
      ls += kv_warp_sum(w * pl);
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const float* src = slot(i0 + i) + (row0 + row) * D + lane * V;
        if constexpr (V == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          acc[0] += wi * v.x;
          acc[1] += wi * v.y;
          acc[2] += wi * v.z;
          acc[3] += wi * v.w;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          acc[0] += wi * v.x;
          acc[1] += wi * v.y;
        }
      }
    }
  }
  if (parts > 1) {
    if (row < rows) {
#pragma unroll
      for (int i = 0; i < V; ++i) part[warp][lane * V + i] = acc[i];
      if (lane == 0) {
        part[warp][D] = mm;
        part[warp][D + 1] = ls;
      }
    }
    __syncthreads();
    if (mine == 0 && row < rows) {
      for (int k = 1; k < parts; ++k) {
        const float* o = part[k * per + row];
        const float m2 = o[D], m_new = fmaxf(mm, m2), f1 = kv_ex2(mm - m_new), f2 = kv_ex2(m2 - m_new);
        mm = m_new;
        ls = ls * f1 + o[D + 1] * f2;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = acc[i] * f1 + o[lane * V + i] * f2;
      }
    }
  }
  if (mine == 0 && row < rows) {
    const int r = row0 + row;
    const long long tok = s.first + r / a.group;
    const int head = h * a.group + r % a.group;
    const float inv = ls > 0.f ? 1.0f / ls : 0.f;
    __half* o = a.O + tok * a.o_stride + static_cast<long long>(head) * D + lane * V;
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(o) = make_uint2(pack_half2(acc[0] * inv, acc[1] * inv),
                                                pack_half2(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(o) = pack_half2(acc[0] * inv, acc[1] * inv);
    if (a.lse != nullptr && lane == 0) a.lse[tok * a.heads_q + head] = (mm + log2f(ls)) * 0.6931471805599453f;
  }
}

}  // namespace mm4
