// Attention over the key / value cache for few rows (a token or a few, times the
// query heads that share a key / value head): units of 8, 16 or 24 rows, and
// two units of 24 for up to 48 rows.
//
// Bound by the cache's bytes: each is read once, 160 a token and head at
// D = 128 in 4 bits, and the arithmetic has to hide behind them: at 6.4 TB/s
// an SM has about 40 elements of K or V a clock to unpack, scale and multiply.
//  - Every warp works alone on tiles of 32 keys that land in its own ring in
//    shared memory (untiled bulk copies, a page is contiguous), without a barrier
//    with other warps. One more warp does all the copying: lane i walks the
//    range of warp i, so finding places and page numbers costs one instruction
//    stream for all of them.
//  - S^T = K Q^T and O^T += V^T P^T on m16n8k16 tensor instructions, with the
//    cache as the 16-row operand and the rows of Q as 8 columns, or 2 or 3
//    times 8: unpacking the cache costs the same for any number of rows.
//  - A lane takes the elements of one word for its share of the contraction
//    (Q's fragments are built in the same order), so codes go from a word to
//    operand registers by logic instructions and one fp16 fused multiply-add a
//    pair; no shuffles. For V the pairs are two keys of one element: one byte
//    permute per two words.
//  - P is rounded to fp16 for its product (2^-11 of itself, like the result, or
//    2^-32 of the row's largest); sums, maxima and O stay fp32. O's error is then
//    about 1.4 times that of its own rounding. A second product with what the
//    rounding of P leaves over makes it 1.0 times and costs 7 % (105 us where this
//    takes 98, 82 for 76, 45 for 39 with 24 rows): not taken.
//  - The running maximum is raised only when a score exceeds it by 8 in the log2
//    domain (P up to 2^15), which one vote per tile decides; the stale maximum
//    cancels in O / l.
//
// 64 sequences of up to 8192 tokens, heads 32 / 8 of 128, 4 bits, on one B200: 98 us,
// 4.5 TB/s (floor 68 us; copying the tiles without computing takes 73 us); 106 us in
// long runs.
// Logic and fp16 instructions share a half-rate port here and fill 91 % of
// it: 244 and 256 a tile and lane, of which unpacking needs 176 and 256.
#pragma once

#include "kv_attention_sm100.cuh"

namespace mm4 {

constexpr int KVF_TK = 32;  // keys of a tile

template <int D, int BITS, int NT, bool TEAM>
struct KvFew {
  static constexpr int ROWS = 8 * NT;
  static constexpr int ROW_BYTES = KvRow<D, BITS>::BYTES;
  static constexpr int STAGE_BYTES = 2 * KVF_TK * ROW_BYTES;  // K rows of a tile, then V rows
  // Warps that compute: 15 with 128 registers a thread, or 7 with more (9 to 12
  // warps get 168). 14 with three tiles each in flight: 99 us where 15 with two
  // take 97. At head_dim 128 in 8 bits, whose tiles are larger and whose 8 rows need
  // 146 registers, 7 warps with three tiles, 9 and 11 with two: 64 sequences of 6000
  // tokens 142, 145, 144 us, 2 of 100,000 78, 80, 80, 1 of 3000 9.7, 11.3, 11.3.
  static constexpr int WARPS = NT == 1 && STAGE_BYTES <= 5120 ? 15 : 7;
  static constexpr int THREADS = 32 * (WARPS + 1);
  static constexpr int PARTS = (WARPS + 1) / 2;               // of the join inside a CTA (TEAM)
  static constexpr int JOIN_BYTES = TEAM ? PARTS * KvPartial<D, ROWS>::FLOATS * 4 : 0;
  // Tiles of a warp's ring: what shared memory holds, at most 5.
  static constexpr int FIT = (225 * 1024 - JOIN_BYTES - WARPS * (32 + 2 * 5 * 8)) / (WARPS * STAGE_BYTES);
  static constexpr int STAGES = FIT < 5 ? FIT : 5;
  static constexpr int RING_BYTES = WARPS * STAGES * STAGE_BYTES;
  static constexpr int BAR_BYTES = 2 * WARPS * STAGES * 8;
  static constexpr int SMEM_BYTES = RING_BYTES + JOIN_BYTES + BAR_BYTES + WARPS * 32;
  static_assert(STAGES >= 2 && SMEM_BYTES <= 232448 && BAR_BYTES % 16 == 0, "shared memory");
};

// Where a warp's range begins: unit u (head, then row block) of sequence b,
// tile n, and how much there is (tiles, or units where a CTA takes whole units).
struct alignas(16) KvStart {
  int b, u, n, pad;
  long long todo;
};

// d = a b + (FIRST ? 0 : d).
template <bool FIRST>
__device__ __forceinline__ void kv_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  const float c0 = FIRST ? 0.f : d[0], c1 = FIRST ? 0.f : d[1], c2 = FIRST ? 0.f : d[2], c3 = FIRST ? 0.f : d[3];
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
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
__device__ __forceinline__ void kv_key_pairs(uint32_t w, __half2 s2, __half2 z2, uint32_t (&out)[16 / BITS],
                                             uint32_t k1024) {
  if constexpr (BITS == 4) {
    __half2 c[4];
    kv_codes4(w, c, k1024);
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
                                               uint32_t (&out)[32 / BITS], uint32_t k1024) {
  const uint32_t lo = __byte_perm(wa, wb, 0x5410), hi = __byte_perm(wa, wb, 0x7632);
  if constexpr (BITS == 4) {
    __half2 c[4];
    kv_codes4(lo, c, k1024);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = as_u32(__hfma2(c[j], s2, z2));
    kv_codes4(hi, c, k1024);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[4 + j] = as_u32(__hfma2(c[j], s2, z2));
  } else {
    const __half2 m1024 = __float2half2_rn(-1024.0f);
    out[0] = as_u32(__hfma2(__hadd2(kv_bits_1024(lo, 0x00FF00FFu, k1024), m1024), s2, z2));
    out[1] = as_u32(__hfma2(__hadd2(kv_bits_1024(lo >> 8, 0x00FF00FFu, k1024), m1024), s2, z2));
    out[2] = as_u32(__hfma2(__hadd2(kv_bits_1024(hi, 0x00FF00FFu, k1024), m1024), s2, z2));
    out[3] = as_u32(__hfma2(__hadd2(kv_bits_1024(hi >> 8, 0x00FF00FFu, k1024), m1024), s2, z2));
  }
}

// A computing warp walks its range. Lane = 4 g + c: in K Q^T it has keys g and
// g + 8 of each 16, the c-th quarter of the head dimension, and rows 2 c and
// 2 c + 1 of the result; in V^T P^T the g-th eighth of the head dimension and
// keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9.
//
// TEAM: a CTA takes whole units, its warps every WARPS-th tile of each, and
// joins them in shared memory: one launch and no workspace, for caches that
// hold few keys a sequence. Otherwise a worker is a warp (worker index =
// warp * CTAs + CTA, so few workers spread over the SMs).
template <int D, int BITS, int NT, bool TEAM>
__global__ void __launch_bounds__(KvFew<D, BITS, NT, TEAM>::THREADS, 1) kv_attention_few_kernel(const KvAttnArgs a) {
  using Cfg = KvFew<D, BITS, NT, TEAM>;
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
  float* join = reinterpret_cast<float*>(kvf_smem + Cfg::RING_BYTES);
  uint64_t* full = reinterpret_cast<uint64_t*>(kvf_smem + Cfg::RING_BYTES + Cfg::JOIN_BYTES);  // [W][ST] landed
  uint64_t* empty = full + W * ST;                                                              // [W][ST] read
  KvStart* starts = reinterpret_cast<KvStart*>(kvf_smem + Cfg::RING_BYTES + Cfg::JOIN_BYTES + Cfg::BAR_BYTES);
  const Watchdog wd{&g_kv_wait, a.timeout_ns};
  if (!TEAM) kv_launch_dependents();

  if (warp < W) {
    KvStart s{};
    if constexpr (TEAM) {
      const long long units = static_cast<long long>(kb.sequences) * kb.heads_kv;
      s.todo = (units - blockIdx.x + gridDim.x - 1) / gridDim.x;
      s.b = static_cast<int>(blockIdx.x / kb.heads_kv);
      s.u = static_cast<int>(blockIdx.x % kb.heads_kv);
      s.n = warp;
    } else {
      constexpr int R = Cfg::ROWS;
      const long long total = kv_total_tiles<KVF_TK, R>(kb, a.group, lane) * kb.heads_kv;
      const long long active = min(static_cast<long long>(a.workers), total);
      const long long w = static_cast<long long>(warp) * gridDim.x + blockIdx.x;
      if (w < active) {
        const long long x = kv_range_begin(w, total, active);
        s.todo = kv_range_begin(w + 1, total, active) - x;
        long long before;
        // Sequence b has heads * blocks * tiles places on the line, from heads *
        // (those before it, for one head).
        s.b = kv_find_tile<KVF_TK, R>(kb, x / kb.heads_kv, a.group, lane, &before);
        const int tiles = s.b < kb.sequences ? kv_tiles<KVF_TK>(kv_sequence(kb, s.b)) : 1;
        const long long in = x - before * kb.heads_kv;
        s.u = static_cast<int>(in / tiles);
        s.n = static_cast<int>(in % tiles);
      }
    }
    if (lane == 0) {
      starts[warp] = s;
      for (int i = 0; i < ST; ++i) {
        mbar_init(&full[warp * ST + i], 1);
        mbar_init(&empty[warp * ST + i], 1);
      }
      fence_mbar_init();
    }
  }
  __syncthreads();

  // A place on the line, and the walk over units.
  struct Place {
    int b, u, n, tiles, blocks;
    KvSequence s;
    long long todo;  // tiles left (TEAM: units)
  };
  auto place_of = [&](int w) {
    const KvStart s = starts[w];
    Place p{};
    p.b = s.b;
    p.u = s.u;
    p.n = s.n;
    p.todo = s.todo;
    return p;
  };
  auto read_sequence = [&](Place& p) {
    p.s = kv_sequence(kb, p.b);
    p.tiles = kv_tiles<KVF_TK>(p.s);
    p.blocks = kv_blocks<Cfg::ROWS>(kb, p.s, a.group);
  };
  auto next_unit = [&](Place& p, int w) {
    if constexpr (TEAM) {
      const long long u = static_cast<long long>(p.b) * kb.heads_kv + p.u + gridDim.x;
      p.b = static_cast<int>(u / kb.heads_kv);
      p.u = static_cast<int>(u % kb.heads_kv);
      p.n = w;
      --p.todo;
    } else {
      p.n = 0;
      if (++p.u >= kb.heads_kv * p.blocks) {
        p.u = 0;
        ++p.b;
      }
    }
  };
  // Goes on to the next tile there is (sequences without rows have none, and in
  // TEAM a unit may end before this warp's first); false at the range's end.
  auto settle = [&](Place& p, int w) -> bool {
    while (p.todo > 0 && p.b < kb.sequences) {
      read_sequence(p);
      if (p.blocks > 0 && p.n < p.tiles) return true;
      next_unit(p, w);
    }
    return false;
  };
  // Head and first row of a unit.
  auto head_of = [&](const Place& p) { return NT < 3 ? p.u : p.u / p.blocks; };
  auto row_of = [&](const Place& p) { return NT < 3 ? 0 : (p.u % p.blocks) * Cfg::ROWS; };

  if (warp == W) {
    // ------------------------------------------------------------ copies
    const int w = min(lane, W - 1);
    uint8_t* ring = kvf_smem + w * ST * Cfg::STAGE_BYTES;
    uint64_t* my_full = full + w * ST;
    uint64_t* my_empty = empty + w * ST;
    const int ps = 1 << kb.page_shift;
    const int chunk = min(KVF_TK, ps);  // keys of a copy: a tile lies in one page, or in two of 16
    Place p = place_of(w);
    if (lane >= W) p.todo = 0;
    bool have = settle(p, w);
    int page[2] = {0, 0};               // of the next tile
    int copies = 0, head = 0;
    // Reads the page numbers of the next tile; they are looked at when it is
    // copied, so their latency is not waited for here.
    auto look_up = [&]() {
      const int key0 = p.n * KVF_TK;
      const int valid = p.s.len - key0;  // <= 0 only for a sequence of length 0
      copies = valid <= 0 ? 0 : (valid > chunk && chunk < KVF_TK) ? 2 : 1;
      head = head_of(p);
      const int* t = kb.table + static_cast<long long>(p.b) * kb.pages_per_seq + (key0 >> kb.page_shift);
      if (copies > 0) page[0] = __ldg(t);
      if (copies > 1) page[1] = __ldg(t + 1);
    };
    if (have) look_up();
    int issued = 0, st = 0, phase = 1;  // copies; the next one's slot and the parity of its last use
    uint64_t since = globaltimer_ns();
    while (__any_sync(0xffffffffu, have)) {
      const bool go = have && (issued < ST || mbar_test_wait(&my_empty[st], phase));
      if (go) {
        uint8_t* dst = ring + st * Cfg::STAGE_BYTES;
        const uint32_t bytes = static_cast<uint32_t>(chunk * RB);
        if (copies == 0) {
          mbar_arrive(&my_full[st]);
        } else {
          mbar_arrive_expect_tx(&my_full[st], bytes * 2 * copies);
          for (int i = 0; i < copies; ++i) {
            int id = page[i];
            if (id < 0 || id >= kb.pages) {
              kv_note(KV_DATA_PAGE);
              id = 0;  // read in place of the page outside the pool
            }
            const uint8_t* src = a.cache + id * kb.page_bytes +
                                 (static_cast<long long>(head * 2 << kb.page_shift) + (p.n * KVF_TK & (ps - 1))) * RB;
            bulk_load(dst + i * chunk * RB, src, bytes, &my_full[st]);
            bulk_load(dst + (KVF_TK + i * chunk) * RB, src + (static_cast<long long>(RB) << kb.page_shift), bytes,
                      &my_full[st]);
          }
        }
        ++issued;
        if (++st == ST) {
          st = 0;
          phase ^= 1;
        }
        if constexpr (TEAM) {
          p.n += W;
          if (p.n >= p.tiles) {
            next_unit(p, w);
            have = settle(p, w);
          }
        } else {
          --p.todo;
          if (++p.n == p.tiles) {
            next_unit(p, w);
            have = settle(p, w);
          } else {
            have = p.todo > 0;
          }
        }
        if (have) look_up();
      }
      if (__any_sync(0xffffffffu, go)) {
        since = globaltimer_ns();
      } else {
        __nanosleep(40);
        const bool late = globaltimer_ns() - since > wd.limit_ns;
        if (late) record_error(wd.status, MM4_ERR_TIMEOUT, 113);
        if (__any_sync(0xffffffffu, late || aborted(wd.status))) break;
      }
    }
    // Copies still in flight after a run-out wait land before the CTA ends.
    for (int i = max(0, issued - ST); i < issued; ++i) mbar_wait(&my_full[i % ST], (i / ST) & 1, wd, 112);
    return;
  }

  // ------------------------------------------------------------ computation
  const int g = lane >> 2, c = lane & 3;
  const uint8_t* ring = kvf_smem + warp * ST * Cfg::STAGE_BYTES;
  uint64_t* my_full = full + warp * ST;
  uint64_t* my_empty = empty + warp * ST;
  Place at = place_of(warp);
  uint32_t q[NT][D / 16][2];
  float acc[NT][MT][4];
  float m[NT][2], l[NT][2];  // running maximum (a score) and sum of rows 2 c, 2 c + 1
  float raise[NT][2];        // the score above which the maximum is raised
  int limit[NT][2];
  int clear = 0;             // keys before this one are masked in no row
  int st = 0, phase = 0;     // the ring's next tile and its parity
  bool ok = true;
  const float sl2 = a.scale_log2, margin = 8.0f / sl2;
  const uint32_t k1024 = __shfl_sync(0xffffffffu, a.k1024, 0);

  // Rows of the unit at p: at most ROWS, and none behind max_new tokens.
  auto rows_of = [&](const Place& p) { return min(min(p.s.n, kb.max_new) * a.group - row_of(p), Cfg::ROWS); };
  auto start_unit = [&](const Place& p) {
    const int row0 = row_of(p), rows = rows_of(p);
    if (p.s.n > kb.max_new) kv_note(KV_DATA_NEW);
    const int head0 = head_of(p) * a.group;
    clear = p.s.len;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const bool have = r < rows;
      const int tok = have ? (row0 + r) / a.group : 0, hd = have ? (row0 + r) % a.group : 0;
      const uint4* src = reinterpret_cast<const uint4*>(
          a.Q + (p.s.first + tok) * a.q_stride + static_cast<long long>(head0 + hd) * D + c * KC);
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
        limit[nt][e] = row < rows ? kv_limit(p.s, (row0 + row) / a.group, a.causal) : p.s.len;
        clear = min(clear, limit[nt][e]);
        m[nt][e] = KV_NO_MAX;
        raise[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][t][e] = 0.f;
    }
    clear = min(clear, __shfl_xor_sync(0xffffffffu, clear, 1));
    clear = min(clear, __shfl_xor_sync(0xffffffffu, clear, 2));
  };

  auto tile = [&](const Place& p) {
    const uint8_t* sk = ring + st * Cfg::STAGE_BYTES;
    const uint8_t* sv = sk + KVF_TK * RB;
    const int key0 = p.n * KVF_TK;
    const bool masked = key0 + KVF_TK > clear;
    if (masked && key0 + lane >= p.s.len) {
      // Rows behind the sequence hold anything: with a scale and zero of 0 their
      // values are 0, and so is their product with P = 0.
      for (int i = 0; i < D / KV_GROUP; ++i)
        *reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(sv) + lane * RB + Row::CODES + 4 * i) = 0u;
      fence_proxy_async_smem();  // before the next copy into this stage
    }
    __syncwarp();
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
      for (int i = 0; i < KW; ++i) {
        uint32_t xa[16 / BITS], xb[16 / BITS];
        kv_key_pairs<BITS>(wa[i], sa, za, xa, k1024);
        kv_key_pairs<BITS>(wb[i], sb, zb, xb, k1024);
#pragma unroll
        for (int j = 0; j < 8 / BITS; ++j) {
          const int step = i * (8 / BITS) + j;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (step == 0)
              kv_mma<true>(s[hf][nt], xa[0], xb[0], xa[1], xb[1], q[nt][0][0], q[nt][0][1]);
            else
              kv_mma<false>(s[hf][nt], xa[2 * j], xb[2 * j], xa[2 * j + 1], xb[2 * j + 1], q[nt][step][0],
                            q[nt][step][1]);
          }
        }
      }
    }
    if (masked) {
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
        mx[nt][e] = fmaxf(fmax3(s[0][nt][e], s[0][nt][e + 2], s[1][nt][e]), s[1][nt][e + 2]);
        grow = grow || mx[nt][e] > raise[nt][e];
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
          const float f = kv_ex2((m[nt][e] - m_new) * sl2);
          m[nt][e] = m_new;
          raise[nt][e] = __fadd_rd(m_new, margin);  // down, so that no P passes 2^15 where scores lie far apart
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
          p4[e] = kv_ex2(fmaf(s[hf][nt][e] - m[nt][e & 1], sl2, KV_LOG2_P));
          l[nt][e & 1] += p4[e];
        }
        pt[hf][nt][0] = kv_transpose(pack_half2(p4[0], p4[1]));
        pt[hf][nt][1] = kv_transpose(pack_half2(p4[2], p4[3]));
      }
    // O^T += V^T P^T.
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      uint32_t w4[4][VW];
      __half2 par[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* row = sv + (hf * 16 + 2 * c + (i & 1) + (i >> 1) * 8) * RB;
        kv_load_words<VW, RB % 16 == 0>(row + g * (VC * BITS / 8), w4[i]);
        par[i] = *reinterpret_cast<const __half2*>(row + Row::CODES + (g * VC / KV_GROUP) * 4);
      }
      // Scales and zeros of the two keys of a pair. The shuffle (of a lane with
      // itself) keeps the compiler from merging them again for each of their
      // uses, which costs more than the unpacking (106 -> 96 us).
      auto keep = [&](__half2 v) { return as_half2(__shfl_sync(0xffffffffu, as_u32(v), lane)); };
      const __half2 s01 = keep(__lows2half2(par[0], par[1])), z01 = keep(__highs2half2(par[0], par[1]));
      const __half2 s23 = keep(__lows2half2(par[2], par[3])), z23 = keep(__highs2half2(par[2], par[3]));
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        uint32_t x[32 / BITS], y[32 / BITS];
        kv_value_pairs<BITS>(w4[0][i], w4[1][i], s01, z01, x, k1024);
        kv_value_pairs<BITS>(w4[2][i], w4[3][i], s23, z23, y, k1024);
#pragma unroll
        for (int j = 0; j < 16 / BITS; ++j) {
          const int t = i * (16 / BITS) + j;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            kv_mma<false>(acc[nt][t], x[2 * j], x[2 * j + 1], y[2 * j], y[2 * j + 1], pt[hf][nt][0], pt[hf][nt][1]);
        }
      }
    }
  };
  // Waits for the next tile, computes it and gives its stage back.
  auto take = [&](const Place& p) -> bool {
    if (!mbar_try_wait(&my_full[st], phase) && !mbar_wait(&my_full[st], phase, wd, 110)) ok = false;
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) return false;
    tile(p);
    __syncwarp();
    if (lane == 0) mbar_arrive(&my_empty[st]);
    if (++st == ST) {
      st = 0;
      phase ^= 1;
    }
    return true;
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
    row += row_of(p);
    const long long tok = p.s.first + row / a.group;
    const int head = head_of(p) * a.group + row % a.group;
    *o = a.O + tok * a.o_stride + static_cast<long long>(head) * D;
    *lse = a.lse ? a.lse + tok * a.heads_q + head : nullptr;
  };

  if constexpr (!TEAM) {
    float* slots = a.partials + 2 * (static_cast<long long>(warp) * gridDim.x + blockIdx.x) * KvPartial<D, Cfg::ROWS>::FLOATS;
    while (ok && settle(at, warp)) {
      start_unit(at);
      const int n0 = at.n;
      const int n1 = static_cast<int>(min(static_cast<long long>(at.tiles), at.n + at.todo));
      for (; at.n < n1; ++at.n)
        if (!take(at)) break;
      at.todo -= n1 - n0;
      sum_l();
      const int rows = rows_of(at);
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
            if (lse != nullptr && g == 0) *lse = kv_lse(m[nt][e], l[nt][e], sl2);
          }
      } else {
        store_partial(slots + (n0 == 0 ? KvPartial<D, Cfg::ROWS>::FLOATS : 0), rows);
      }
      if (n1 == at.tiles) next_unit(at, warp);
    }
  } else {
    while (at.todo > 0) {  // every computing warp of the CTA walks the same units
      read_sequence(at);
      if (at.blocks > 0) {
        const int rows = rows_of(at);
        start_unit(at);
        for (; ok && at.n < at.tiles; at.n += W)
          if (!take(at)) break;
        sum_l();
        // Two rounds: the upper half of the warps hands over to the lower, then
        // all threads sum the lower half's parts.
        constexpr int F = KvPartial<D, Cfg::ROWS>::FLOATS;
        if (warp >= Cfg::PARTS) store_partial(join + (warp - Cfg::PARTS) * F, rows);
        named_barrier(1, W * 32);
        if (warp + Cfg::PARTS < W) {
          const float* other = join + warp * F;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = nt * 8 + 2 * c + e;
              if (row >= rows) continue;
              const float m2 = other[Cfg::ROWS * D + 2 * row], l2 = other[Cfg::ROWS * D + 2 * row + 1];
              const float mm = fmaxf(m[nt][e], m2), f1 = kv_ex2((m[nt][e] - mm) * sl2), f2 = kv_ex2((m2 - mm) * sl2);
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
        if (warp < Cfg::PARTS) store_partial(join + warp * F, rows);
        named_barrier(1, W * 32);
        for (int i = threadIdx.x; i < rows * (D / 2); i += W * 32) {
          const int row = i / (D / 2), d = (i % (D / 2)) * 2;
          float mm = KV_NO_MAX;
#pragma unroll
          for (int k = 0; k < Cfg::PARTS; ++k) mm = fmaxf(mm, join[k * F + Cfg::ROWS * D + 2 * row]);
          float ls = 0.f, x = 0.f, y = 0.f;
#pragma unroll
          for (int k = 0; k < Cfg::PARTS; ++k) {
            const float f = kv_ex2((join[k * F + Cfg::ROWS * D + 2 * row] - mm) * sl2);
            ls += f * join[k * F + Cfg::ROWS * D + 2 * row + 1];
            x += f * join[k * F + row * D + d];
            y += f * join[k * F + row * D + d + 1];
          }
          __half* o;
          float* lse;
          output_row(at, row, &o, &lse);
          const float inv = ls > 0.f ? 1.0f / ls : 0.f;
          *reinterpret_cast<__half2*>(o + d) = __floats2half2_rn(x * inv, y * inv);
          if (lse != nullptr && d == 0) *lse = kv_lse(mm, ls, sl2);
        }
        named_barrier(1, W * 32);  // the parts are free for the next unit
      }
      next_unit(at, warp);
    }
  }
}

// Joins the partials of the units that several workers share: a block of 8
// warps per unit and join_rows rows, (row, part of the partials) to a warp, parts
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
  const int chunks = (min(ROWS, kb.max_new * a.group) + a.join_rows - 1) / a.join_rows;  // of a row block
  const int blocks = kv_blocks<ROWS>(kb, s, a.group), block = blockIdx.y / chunks;
  const int row0 = blockIdx.y % chunks * a.join_rows;  // in the unit
  const int rows = min(min(min(s.n, kb.max_new) * a.group - block * ROWS, ROWS) - row0, a.join_rows);
  // Tiles of all sequences and of those before this one, by the whole block.
  __shared__ long long sums[2][8];
  long long all = 0, ahead = 0;
  for (int i = threadIdx.x; i < kb.sequences; i += 256) {
    const int t = kv_sequence_tiles<TK, ROWS>(kb, i, a.group);
    all += t;
    if (i < b) ahead += t;
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, k);
    ahead += __shfl_xor_sync(0xffffffffu, ahead, k);
  }
  if (lane == 0) {
    sums[0][warp] = all;
    sums[1][warp] = ahead;
  }
  __syncthreads();
  all = ahead = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    all += sums[0][k];
    ahead += sums[1][k];
  }
  const long long total = all * kb.heads_kv;
  const long long active = min(static_cast<long long>(a.workers), total);
  const int tiles = kv_tiles<TK>(s);
  long long first = 0, last = 0;
  if (rows > 0) {
    const long long x0 = ahead * kb.heads_kv + (static_cast<long long>(h) * blocks + block) * tiles;
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
  const float sl2 = a.scale_log2;
  float mm = KV_NO_MAX, ls = 0.f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  if (row < rows) {
    auto slot = [&](int i) { return a.partials + (2 * (first + i) + (i == 0 ? 1 : 0)) * F; };
    auto load = [&](int i, float (&v)[V]) {
      const float* src = slot(i) + (row0 + row) * D + lane * V;
      if constexpr (V == 4) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
        v[0] = x.x;
        v[1] = x.y;
        v[2] = x.z;
        v[3] = x.w;
      } else {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
        v[0] = x.x;
        v[1] = x.y;
      }
    };
    for (int i0 = c0; i0 < c1; i0 += 32) {
      const int n = min(32, c1 - i0);
      // The first O rows are on their way while weights are formed.
      float early[8][V];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) load(i0 + i, early[i]);
      float pm = KV_NO_MAX, pl = 0.f;
      if (lane < n) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(slot(i0 + lane) + ROWS * D + 2 * (row0 + row)));
        pm = ml.x;
        pl = ml.y;
      }
      float top = pm;
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
      const float m_new = fmaxf(mm, top), f = kv_ex2((mm - m_new) * sl2), w = kv_ex2((pm - m_new) * sl2);
      mm = m_new;
      ls *= f;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= f;
      ls += kv_warp_sum(w * pl);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        if (i < n)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += wi * early[i][e];
      }
#pragma unroll 8
      for (int i = 8; i < n; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        float v[V];
        load(i0 + i, v);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += wi * v[e];
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
        const float m2 = o[D], m_new = fmaxf(mm, m2), f1 = kv_ex2((mm - m_new) * sl2), f2 = kv_ex2((m2 - m_new) * sl2);
        mm = m_new;
        ls = ls * f1 + o[D + 1] * f2;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = acc[i] * f1 + o[lane * V + i] * f2;
      }
    }
  }
  if (mine == 0 && row < rows) {
    const int r = block * ROWS + row0 + row;
    const long long tok = s.first + r / a.group;
    const int head = h * a.group + r % a.group;
    const float inv = ls > 0.f ? 1.0f / ls : 0.f;
    __half* o = a.O + tok * a.o_stride + static_cast<long long>(head) * D + lane * V;
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(o) = make_uint2(pack_half2(acc[0] * inv, acc[1] * inv),
                                                pack_half2(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(o) = pack_half2(acc[0] * inv, acc[1] * inv);
    if (a.lse != nullptr && lane == 0) a.lse[tok * a.heads_q + head] = kv_lse(mm, ls, sl2);
  }
}

}  // namespace mm4
