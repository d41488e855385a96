// The key / value cache in 4 or 8 bits: its layout, the batch it is used
// with, and the kernels that write it and read it back.
//
// Layout: pages of [heads_kv][2: K, V][page_size] rows; a row is one head's
// vector of one token, D codes of BITS bits and then, for each 32 elements, an
// fp16 scale and an fp16 zero. A code c stands for fp16(c * scale + zero),
// one rounding (a half-precision fused multiply-add), and every kernel that
// reads the cache forms exactly that value. A group of 32 with an fp16 pair
// costs one bit an element: a row of 128 is 80 bytes in 4 bits and 144 in 8.
#pragma once

#include "mm4_ptx.cuh"

namespace mm4 {

constexpr int KV_GROUP = 32;  // elements that share a scale and a zero

// Status words of these kernels, apart from the library's own: a wrong page
// number in one call's batch must not make the bounded waits of later kernels
// give up. g_kv_wait takes run-out waits, g_kv_data what is wrong in a batch.
static __device__ int g_kv_wait;
static __device__ int g_kv_data;

enum : int {
  KV_DATA_PAGE = 1,     // page number outside the pool
  KV_DATA_LENGTH = 2,   // length negative or beyond the page table
  KV_DATA_OFFSETS = 3,  // offsets out of order or beyond the rows
  KV_DATA_NEW = 4,      // more rows of a sequence than max_new
};

struct KvBatch {
  const int* table;
  const int* lengths;
  const int* offsets;
  int sequences, tokens, max_new, pages_per_seq;
  int page_shift;        // log2(page_size)
  long long pages;
  int heads_kv;
  long long page_bytes;
};

template <int D, int BITS>
struct KvRow {
  static_assert((D == 64 || D == 128) && (BITS == 4 || BITS == 8), "head_dim 64 or 128, 4 or 8 bits");
  static constexpr int CODES = D * BITS / 8;
  static constexpr int BYTES = CODES + D / KV_GROUP * 4;
};

__device__ __forceinline__ void kv_note(int site) { record_error(&g_kv_data, MM4_ERR_INVALID, site); }

// Rows of sequence b in this call and its length, made safe: first .. first + n
// lies in the tokens and len in the page table.
struct KvSequence {
  int len, first, n;
};
__device__ __forceinline__ KvSequence kv_sequence(const KvBatch& kb, int b) {
  KvSequence s;
  s.len = kb.lengths[b];
  s.first = kb.offsets[b];
  const int end = kb.offsets[b + 1];
  const int room = kb.pages_per_seq << kb.page_shift;
  if (s.len < 0 || s.len > room) {
    kv_note(KV_DATA_LENGTH);
    s.len = s.len < 0 ? 0 : room;
  }
  if (s.first < 0 || end < s.first || end > kb.tokens) {
    kv_note(KV_DATA_OFFSETS);
    s.first = s.n = 0;
  } else {
    s.n = end - s.first;
  }
  return s;
}

// The sequence whose rows hold row t: a search of the ascending offsets, then a
// check, so where offsets are out of order a row finds a sequence whose own
// offsets hold it, or none. -1 for padding rows, and for sequences whose offsets
// leave the rows: kv_sequence gives them no rows either. Lanes with tokens of their
// own search binary; a warp with one token searches 32-way, two steps for up to
// 1024 sequences.
template <bool WARP>
__device__ __forceinline__ int kv_find_sequence(const KvBatch& kb, int t, int lane) {
  int lo = 0, n = kb.sequences;
  while (n > 1) {
    if constexpr (WARP) {
      const int step = (n + 31) / 32, probe = lane * step;
      const unsigned hit = __ballot_sync(0xffffffffu, probe < n && __ldg(kb.offsets + lo + probe) <= t);
      if (hit == 0) return -1;
      const int k = (31 - __clz(hit)) * step;
      lo += k;
      n = min(step, n - k);
    } else {
      const int half = n >> 1;
      const bool right = __ldg(kb.offsets + lo + half) <= t;
      lo = right ? lo + half : lo;
      n = right ? n - half : half;
    }
  }
  const int first = __ldg(kb.offsets + lo), end = __ldg(kb.offsets + lo + 1);
  return first >= 0 && first <= t && t < end && end <= kb.tokens ? lo : -1;
}

// Where the K row of token t lies for head 0, as an offset into the cache; -1 if
// the row has no place (padding, a sequence with a wrong length, before position
// 0, a page outside the pool). Wrong offsets and lengths are reported by
// kv_check_batch.
template <bool WARP>
__device__ __forceinline__ long long kv_place(const KvBatch& kb, int t, int row_bytes, int lane) {
  const int b = kv_find_sequence<WARP>(kb, t, lane);
  if (b < 0) return -1;
  const int end = __ldg(kb.offsets + b + 1);
  const int len = __ldg(kb.lengths + b);
  const long long pos = static_cast<long long>(len) - (end - t);
  const int room = kb.pages_per_seq << kb.page_shift;
  if (pos < 0 || len > room) return -1;  // pos < 0 for a negative length too
  const int p = static_cast<int>(pos);
  const int page = __ldg(kb.table + static_cast<long long>(b) * kb.pages_per_seq + (p >> kb.page_shift));
  if (page < 0 || page >= kb.pages) {
    kv_note(KV_DATA_PAGE);
    return -1;
  }
  return page * kb.page_bytes + static_cast<long long>(p & ((1 << kb.page_shift) - 1)) * row_bytes;
}

// Reports what is wrong in the lengths and offsets of a batch, whether a row's
// search meets it or not: threads `first`, `first + step`, ... of a call take a
// sequence each. Offsets are in order if every sequence's are, and the last ends
// in the rows.
__device__ __forceinline__ void kv_check_batch(const KvBatch& kb, int first, int step) {
  for (long long b = first; b < kb.sequences; b += step) kv_sequence(kb, static_cast<int>(b));
}

// ---------------------------------------------------------------------------
// codes to values
// ---------------------------------------------------------------------------

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

constexpr uint32_t KV_1024 = 0x64006400u;  // fp16 1024 in both halves

// (x & mask) | KV_1024: fp16 1024 + the masked bits, exactly. The kernels that
// unpack in their inner loops get KV_1024 as an argument: as a literal it would be
// moved into a register again for each use, since the mask takes the one
// immediate operand of the instruction.
__device__ __forceinline__ __half2 kv_bits_1024(uint32_t x, uint32_t mask, uint32_t k1024) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(k1024));
  return as_half2(r);
}

// The codes of a word whose 16-bit halves hold four 4-bit codes each: out[j] =
// (code j of the low half, code j of the high half) as exact integers. Codes under the
// exponent of 1024, which is then taken off, are a published way to halves (Kim et al.,
// "Who Says Elephants Can't Run", 2022).
__device__ __forceinline__ void kv_codes4(uint32_t w, __half2 (&out)[4], uint32_t k1024) {
  const __half2 m1024 = __float2half2_rn(-1024.0f), m64 = __float2half2_rn(-64.0f),
                sixteenth = __float2half2_rn(0.0625f);
  const uint32_t v = w >> 8;
  out[0] = __hadd2(kv_bits_1024(w, 0x000F000Fu, k1024), m1024);
  out[1] = __hfma2(kv_bits_1024(w, 0x00F000F0u, k1024), sixteenth, m64);  // (1024 + 16 c) / 16 - 64
  out[2] = __hadd2(kv_bits_1024(v, 0x000F000Fu, k1024), m1024);
  out[3] = __hfma2(kv_bits_1024(v, 0x00F000F0u, k1024), sixteenth, m64);
}

// Two of a word's four 8-bit codes, picked by a byte-permute selector whose
// odd bytes take 0x64 (selector digits 4), as exact integers.
__device__ __forceinline__ __half2 kv_codes8(uint32_t w, uint32_t selector) {
  return __hadd2(as_half2(__byte_perm(w, 0x64646464u, selector)), __float2half2_rn(-1024.0f));
}

// ---------------------------------------------------------------------------
// write and read back
// ---------------------------------------------------------------------------

constexpr int KV_IO_WARPS = 4;                // warps of a block
constexpr int KV_IO_VECS = 4;                 // 8-element vectors of a lane and token, all in flight
constexpr int KV_IO_PART = 32 * KV_IO_VECS;   // vectors of a warp and token

struct KvIoArgs {
  KvBatch kb;
  const __half* in_k;   // append
  const __half* in_v;
  __half* out_k;        // read
  __half* out_v;
  long long k_stride, v_stride;
  uint8_t* cache;
  int blocks;           // that move rows; those behind them check the batch
  int parts;            // warps that share a token
  int tokens_per_warp;  // 1 .. 32: looked up by a lane each, so that their places cost one latency
};

// The work of a warp: tokens t0 .. t0 + n - 1 (lane i has the place of token
// t0 + i), vectors vec0 + 32 i. False if it has none.
struct KvIoWork {
  int t0, n, vec0;
  long long place;
};
template <int ROW_BYTES>
__device__ __forceinline__ bool kv_io_work(const KvIoArgs& a, int lane, KvIoWork* w) {
  if (blockIdx.x >= a.blocks) {
    kv_check_batch(a.kb, static_cast<int>((blockIdx.x - a.blocks) * blockDim.x + threadIdx.x),
                   static_cast<int>((gridDim.x - a.blocks) * blockDim.x));
    return false;
  }
  const long long id = static_cast<long long>(blockIdx.x) * KV_IO_WARPS + (threadIdx.x >> 5);
  const long long t0 = id / a.parts * a.tokens_per_warp;
  if (t0 >= a.kb.tokens) return false;
  w->t0 = static_cast<int>(t0);
  w->n = min(a.tokens_per_warp, a.kb.tokens - w->t0);
  w->vec0 = static_cast<int>(id % a.parts) * KV_IO_PART + lane;
  if (a.tokens_per_warp == 1)
    w->place = kv_place<true>(a.kb, w->t0, ROW_BYTES, lane);
  else
    w->place = lane < w->n ? kv_place<false>(a.kb, w->t0 + lane, ROW_BYTES, lane) : -1;
  return true;
}

// Where vector v of a token (8 elements; K's, then as many of V) lies: head and
// K or V in the page, element in the row.
template <int D, int BITS>
__device__ __forceinline__ int kv_vector_row(const KvBatch& kb, int v, int half_vecs, int* d) {
  const int kv = v >= half_vecs ? 1 : 0;
  const int e = (v - kv * half_vecs) * 8;
  *d = e % D;
  return ((e / D * 2 + kv) << kb.page_shift) * KvRow<D, BITS>::BYTES;
}

// The smallest and the largest of a group's fp16 values, as (min, -max) in one
// register, from the 8 in `w` and those of the three lanes beside.
__device__ __forceinline__ __half2 kv_group_range(const uint32_t (&w)[4]) {
  __half2 lo = __hmin2(__hmin2(as_half2(w[0]), as_half2(w[1])), __hmin2(as_half2(w[2]), as_half2(w[3])));
  __half2 hi = __hmax2(__hmax2(as_half2(w[0]), as_half2(w[1])), __hmax2(as_half2(w[2]), as_half2(w[3])));
  // (lo.x, -hi.x) and (lo.y, -hi.y)
  hi = __hneg2(hi);
  __half2 r = __hmin2(__lows2half2(lo, hi), __highs2half2(lo, hi));
  r = __hmin2(r, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(r), 1)));
  return __hmin2(r, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(r), 2)));
}

// Codes of 8 values: min(top, round_half_even((x - lo) / s)). The quotient is
// first formed with an approximate reciprocal (off by 2^-23) and a product (2^-24),
// so it is off by less than 2^-14.3 below 260. Where that could decide between
// two codes (closer than 2^-14 to a half), the division itself decides; so it does
// for subnormal scales, the only ones whose quotients pass top + 1/2 (a scale is cut
// by up to 2^-10 of itself otherwise). out[j] holds KV_CODE + code.
constexpr uint32_t KV_CODE = 0x4B400000u;  // fp32 1.5 * 2^23: adding it rounds to an integer, half to even
__device__ __forceinline__ void kv_quantise8(const uint32_t (&w)[4], float lo, float s, float top,
                                             uint32_t (&out)[8]) {
  const float round = __uint_as_float(KV_CODE);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  bool exact = s < 6.103515625e-5f;
  if (exact) inv = 0.f;
  float2 d[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    d[j] = fadd2(__half22float2(as_half2(w[j])), make_float2(-lo, -lo));
    const float2 q = ffma2(d[j], make_float2(inv, inv), make_float2(0.f, 0.f));
    const float2 r = fadd2(q, make_float2(round, round));
    const float2 n = fadd2(r, make_float2(-round, -round));
    const float2 off = fadd2(q, make_float2(-n.x, -n.y));
    exact = exact || fmaxf(fabsf(off.x), fabsf(off.y)) > 0.5f - 6.103515625e-5f;
    out[2 * j] = __float_as_uint(r.x);
    out[2 * j + 1] = __float_as_uint(r.y);
  }
  if (exact) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = (j & 1) ? d[j / 2].y : d[j / 2].x;
      out[j] = s > 0.f ? __float_as_uint(__fadd_rn(fminf(__fdiv_rn(x, s), top), round)) : KV_CODE;
    }
  }
}

// x / top rounded to fp32 as a division would: a product with the rounded
// reciprocal is off by less than a unit in the last place, its remainder is exact
// in a fused multiply-add, and adding remainder * reciprocal rounds correctly
// (Markstein, IBM J. Res. Dev. 34, 1990). x is 0 or at least 2^-24.
template <int TOP>
__device__ __forceinline__ float kv_divide_by_top(float x) {
  constexpr float INV = 1.0f / TOP;
  const float q = __fmul_rn(x, INV);
  return __fmaf_rn(__fmaf_rn(-q, static_cast<float>(TOP), x), INV, q);
}

// Quantises K and V of the batch's rows. A warp takes 128 vectors of 8 elements of
// each of its tokens; the four lanes of a group of 32 find its range by two
// shuffles of one register. Its floor are the bytes it moves: 512 in and 160 out
// per token and head at D = 128 in 4 bits, 25 us for four prompts of up to 4096
// tokens and 16 heads; it takes 50 us, and as much in 8 bits (30 us of bytes). No unit
// is full (issue slots 64 %, logic 45 %): 142 instructions for 8 elements a lane, and a
// token's loads wait for the codes of the one before it.
template <int D, int BITS>
__global__ void __launch_bounds__(KV_IO_WARPS * 32, 6) kv_append_kernel(const KvIoArgs a) {
  constexpr int TOP = (1 << BITS) - 1;
  using Row = KvRow<D, BITS>;
  const int lane = threadIdx.x & 31;
  const int half_vecs = a.kb.heads_kv * (D / 8);  // vectors of K; as many of V
  KvIoWork work;
  if (!kv_io_work<Row::BYTES>(a, lane, &work)) return;
  // What does not change from token to token: where this lane's vectors come
  // from, and where their codes and parameters go in a page (-1: no vector).
  const __half* src[KV_IO_VECS];
  int to[KV_IO_VECS], par[KV_IO_VECS];
#pragma unroll
  for (int k = 0; k < KV_IO_VECS; ++k) {
    const int v = work.vec0 + 32 * k;
    const bool is_v = v >= half_vecs;
    const __half* rows = is_v ? a.in_v + (v - half_vecs) * 8 : a.in_k + v * 8;
    src[k] = rows + work.t0 * (is_v ? a.v_stride : a.k_stride);
    int d;
    const int row = kv_vector_row<D, BITS>(a.kb, v, half_vecs, &d);
    to[k] = v < 2 * half_vecs ? row + d * BITS / 8 : -1;
    par[k] = row + Row::CODES + d / KV_GROUP * 4;
  }
#pragma unroll 1
  for (int i = 0; i < work.n; ++i) {
    uint32_t w[KV_IO_VECS][4];
    uint32_t odd = 0;
#pragma unroll
    for (int k = 0; k < KV_IO_VECS; ++k) {
      uint4 in = make_uint4(0u, 0u, 0u, 0u);
      if (to[k] >= 0) in = __ldg(reinterpret_cast<const uint4*>(src[k]));
      src[k] += work.vec0 + 32 * k >= half_vecs ? a.v_stride : a.k_stride;
      w[k][0] = in.x;
      w[k][1] = in.y;
      w[k][2] = in.z;
      w[k][3] = in.w;
    }
    const long long place = __shfl_sync(0xffffffffu, work.place, i);
    if (place < 0) continue;
    uint8_t* page = a.cache + place;
    // NaN counts as 0 and infinities as the largest finite value: exponents of
    // all ones carry into the sign bit here.
#pragma unroll
    for (int k = 0; k < KV_IO_VECS; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) odd |= (w[k][j] & 0x7FFF7FFFu) + 0x04000400u;
    if ((odd & 0x80008000u) != 0) {
#pragma unroll
      for (int k = 0; k < KV_IO_VECS; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t fixed = 0;
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            uint32_t x = (w[k][j] >> h) & 0xFFFFu;
            if ((x & 0x7FFFu) > 0x7C00u) x = 0;                         // NaN
            if ((x & 0x7FFFu) == 0x7C00u) x = (x & 0x8000u) | 0x7BFFu;  // infinity
            fixed |= x << h;
          }
          w[k][j] = fixed;
        }
    }
#pragma unroll
    for (int k = 0; k < KV_IO_VECS; ++k) {
      const __half2 range = kv_group_range(w[k]);
      const __half zero = __low2half(range);
      const float lo = __half2float(zero), hi = -__half2float(__high2half(range));
      const __half scale = __float2half_rz(kv_divide_by_top<TOP>(__fsub_rn(hi, lo)));
      uint32_t code[8];
      kv_quantise8(w[k], lo, __half2float(scale), static_cast<float>(TOP), code);
      if (to[k] < 0) continue;
      // Codes are packed by multiplication and addition modulo 2^32, KV_CODE with
      // them, and what that adds up to is taken off.
      if constexpr (BITS == 4) {
        constexpr uint32_t TAKE = KV_CODE * 0x11111111u;
        uint32_t packed = code[7];
#pragma unroll
        for (int j = 6; j >= 0; --j) packed = packed * 16u + code[j];
        *reinterpret_cast<uint32_t*>(page + to[k]) = packed - TAKE;
      } else {
        constexpr uint32_t TAKE = KV_CODE * 0x01010101u;
        uint32_t packed[2] = {code[3], code[7]};
#pragma unroll
        for (int j = 2; j >= 0; --j) {
          packed[0] = packed[0] * 256u + code[j];
          packed[1] = packed[1] * 256u + code[4 + j];
        }
        *reinterpret_cast<uint2*>(page + to[k]) = make_uint2(packed[0] - TAKE, packed[1] - TAKE);
      }
      if ((lane & 3) == 0) *reinterpret_cast<__half2*>(page + par[k]) = __halves2half2(scale, zero);
    }
  }
}

// Reads the rows of a batch back as fp16 values; the mapping of kv_append_kernel.
// Bound by memory: 8 sequences of up to 8192 tokens and 8 heads of 128 in 4 bits, 306 MB,
// in 59 us (5.2 TB/s), in 8 bits, 364 MB, in 72 us (5.1).
template <int D, int BITS>
__global__ void __launch_bounds__(KV_IO_WARPS * 32) kv_read_kernel(const KvIoArgs a) {
  using Row = KvRow<D, BITS>;
  const int lane = threadIdx.x & 31;
  const int half_vecs = a.kb.heads_kv * (D / 8);
  KvIoWork work;
  if (!kv_io_work<Row::BYTES>(a, lane, &work)) return;
#pragma unroll 2
  for (int i = 0; i < work.n; ++i) {
    const long long t = work.t0 + i;
    const long long place = __shfl_sync(0xffffffffu, work.place, i);
    if (place < 0) continue;
    const uint8_t* page = a.cache + place;
    uint2 codes[KV_IO_VECS];
    __half2 par[KV_IO_VECS];
#pragma unroll
    for (int k = 0; k < KV_IO_VECS; ++k) {
      const int v = work.vec0 + 32 * k;
      if (v >= 2 * half_vecs) continue;
      int d;
      const uint8_t* src = page + kv_vector_row<D, BITS>(a.kb, v, half_vecs, &d);
      if constexpr (BITS == 4)
        codes[k] = make_uint2(__ldg(reinterpret_cast<const uint32_t*>(src + d / 2)), 0u);
      else
        codes[k] = __ldg(reinterpret_cast<const uint2*>(src + d));
      par[k] = as_half2(__ldg(reinterpret_cast<const uint32_t*>(src + Row::CODES + d / KV_GROUP * 4)));
    }
#pragma unroll
    for (int k = 0; k < KV_IO_VECS; ++k) {
      const int v = work.vec0 + 32 * k;
      if (v >= 2 * half_vecs) continue;
      const __half2 s2 = __low2half2(par[k]), z2 = __high2half2(par[k]);
      uint4 out;
      if constexpr (BITS == 4) {
        __half2 c[4];
        kv_codes4(codes[k].x, c, KV_1024);  // pairs (0,4) (1,5) (2,6) (3,7)
        const uint32_t p0 = as_u32(__hfma2(c[0], s2, z2)), p1 = as_u32(__hfma2(c[1], s2, z2)),
                       p2 = as_u32(__hfma2(c[2], s2, z2)), p3 = as_u32(__hfma2(c[3], s2, z2));
        out = make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632),
                         __byte_perm(p2, p3, 0x7632));
      } else {
        out.x = as_u32(__hfma2(kv_codes8(codes[k].x, 0x4140), s2, z2));
        out.y = as_u32(__hfma2(kv_codes8(codes[k].x, 0x4342), s2, z2));
        out.z = as_u32(__hfma2(kv_codes8(codes[k].y, 0x4140), s2, z2));
        out.w = as_u32(__hfma2(kv_codes8(codes[k].y, 0x4342), s2, z2));
      }
      __half* dst = v < half_vecs ? a.out_k + t * a.k_stride + v * 8 : a.out_v + t * a.v_stride + (v - half_vecs) * 8;
      *reinterpret_cast<uint4*>(dst) = out;
    }
  }
}

}  // namespace mm4
