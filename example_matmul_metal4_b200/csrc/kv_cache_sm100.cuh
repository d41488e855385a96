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

// The sequence whose rows hold row t (all lanes of the warp call it with the
// same t): a 32-way search of the ascending offsets, two steps for up to 1024
// sequences, then a check, so offsets that are out of order find nothing
// rather than something wrong. -1 for padding rows.
__device__ __forceinline__ int kv_find_sequence(const KvBatch& kb, int t, int lane) {
  int lo = 0, n = kb.sequences;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int probe = lane * step;
    const unsigned hit = __ballot_sync(0xffffffffu, probe < n && __ldg(kb.offsets + lo + probe) <= t);
    if (hit == 0) return -1;
    const int k = (31 - __clz(hit)) * step;
    lo += k;
    n = min(step, n - k);
  }
  const int first = __ldg(kb.offsets + lo), end = __ldg(kb.offsets + lo + 1);
  if (end < first) kv_note(KV_DATA_OFFSETS);
  return first <= t && t < end ? lo : -1;
}

// Address of the K rows of one token's page and head 0, plus its row number;
// nullptr if the row has no place (padding, before position 0, beyond the page
// table, a page outside the pool).
__device__ __forceinline__ uint8_t* kv_place(const KvBatch& kb, uint8_t* cache, int t, int lane, int* row) {
  const int b = kv_find_sequence(kb, t, lane);
  if (b < 0) return nullptr;
  const int end = __ldg(kb.offsets + b + 1);
  const int len = __ldg(kb.lengths + b);
  const long long pos = static_cast<long long>(len) - (end - t);
  const int room = kb.pages_per_seq << kb.page_shift;
  if (len < 0 || len > room) kv_note(KV_DATA_LENGTH);
  if (pos < 0 || pos >= room) return nullptr;
  const int p = static_cast<int>(pos);
  const int page = __ldg(kb.table + static_cast<long long>(b) * kb.pages_per_seq + (p >> kb.page_shift));
  if (page < 0 || page >= kb.pages) {
    kv_note(KV_DATA_PAGE);
    return nullptr;
  }
  *row = p & ((1 << kb.page_shift) - 1);
  return cache + page * kb.page_bytes;
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
// (code j of the low half, code j of the high half) as exact integers.
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
constexpr int KV_IO_VECS = 4;                 // 8-element vectors of a lane, all in flight
constexpr int KV_IO_PART = 32 * KV_IO_VECS;   // vectors of a warp

struct KvIoArgs {
  KvBatch kb;
  const __half* in_k;   // append
  const __half* in_v;
  __half* out_k;        // read
  __half* out_v;
  long long k_stride, v_stride;
  uint8_t* cache;
  int parts;            // warps of one token
};

// Quantises one token's K and V. A warp takes 128 vectors of 8 elements (of the
// 2 * heads_kv * D / 8 that a token has, K first), four to a lane; the four
// lanes of a group of 32 elements find its minimum and maximum by two
// shuffles. Bound by the bytes it moves: 512 in and 160 out per token and head
// at D = 128 in 4 bits.
template <int D, int BITS>
__global__ void __launch_bounds__(KV_IO_WARPS * 32) kv_append_kernel(const KvIoArgs a) {
  constexpr float TOP = static_cast<float>((1 << BITS) - 1);
  using Row = KvRow<D, BITS>;
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * KV_IO_WARPS + (threadIdx.x >> 5);
  const long long t64 = w / a.parts;
  if (t64 >= a.kb.tokens) return;
  const int t = static_cast<int>(t64);
  const int vec0 = static_cast<int>(w % a.parts) * KV_IO_PART + lane;
  const int half_vecs = a.kb.heads_kv * (D / 8);  // vectors of K; as many of V
  // The inputs do not wait for the page number.
  uint4 in[KV_IO_VECS];
#pragma unroll
  for (int i = 0; i < KV_IO_VECS; ++i) {
    const int v = vec0 + 32 * i;
    if (v >= 2 * half_vecs) continue;
    const __half* src = v < half_vecs ? a.in_k + t * a.k_stride + v * 8 : a.in_v + t * a.v_stride + (v - half_vecs) * 8;
    in[i] = __ldg(reinterpret_cast<const uint4*>(src));
  }
  int row = 0;
  uint8_t* page = kv_place(a.kb, a.cache, t, lane, &row);
  if (page == nullptr) return;
#pragma unroll
  for (int i = 0; i < KV_IO_VECS; ++i) {
    const int v = vec0 + 32 * i;
    const bool have = v < 2 * half_vecs;
    float x[8];
    if (have) {
      const uint32_t words[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(as_half2(words[j]));
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
    }
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = x[j] != x[j] ? 0.f : fminf(fmaxf(x[j], -65504.f), 65504.f);
      lo = fminf(lo, x[j]);
      hi = fmaxf(hi, x[j]);
    }
#pragma unroll
    for (int s = 1; s <= 2; s <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
    }
    const __half scale = __float2half_rz(__fdiv_rn(__fsub_rn(hi, lo), TOP));
    const float s = __half2float(scale);
    uint32_t code[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      code[j] = s > 0.f ? static_cast<uint32_t>(fminf(rintf(__fdiv_rn(__fsub_rn(x[j], lo), s)), TOP)) : 0u;
    if (!have) continue;
    const int kv = v >= half_vecs ? 1 : 0;
    const int e = (v - kv * half_vecs) * 8;
    const int head = e / D, d = e % D;
    uint8_t* dst = page + (static_cast<long long>((head * 2 + kv) << a.kb.page_shift) + row) * Row::BYTES;
    if constexpr (BITS == 4) {
      uint32_t packed = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) packed |= code[j] << (4 * j);
      *reinterpret_cast<uint32_t*>(dst + d / 2) = packed;
    } else {
      *reinterpret_cast<uint2*>(dst + d) =
          make_uint2(code[0] | (code[1] << 8) | (code[2] << 16) | (code[3] << 24),
                     code[4] | (code[5] << 8) | (code[6] << 16) | (code[7] << 24));
    }
    if ((lane & 3) == 0)
      *reinterpret_cast<__half2*>(dst + Row::CODES + d / KV_GROUP * 4) = __halves2half2(scale, __float2half_rn(lo));
  }
}

// Reads the rows of a batch back as fp16 values; the mapping of kv_append_kernel.
template <int D, int BITS>
__global__ void __launch_bounds__(KV_IO_WARPS * 32) kv_read_kernel(const KvIoArgs a) {
  using Row = KvRow<D, BITS>;
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * KV_IO_WARPS + (threadIdx.x >> 5);
  const long long t64 = w / a.parts;
  if (t64 >= a.kb.tokens) return;
  const int t = static_cast<int>(t64);
  const int vec0 = static_cast<int>(w % a.parts) * KV_IO_PART + lane;
  const int half_vecs = a.kb.heads_kv * (D / 8);
  int row = 0;
  const uint8_t* page = kv_place(a.kb, a.cache, t, lane, &row);
  if (page == nullptr) return;
  uint2 codes[KV_IO_VECS];
  __half2 par[KV_IO_VECS];
#pragma unroll
  for (int i = 0; i < KV_IO_VECS; ++i) {
    const int v = vec0 + 32 * i;
    if (v >= 2 * half_vecs) continue;
    const int kv = v >= half_vecs ? 1 : 0;
    const int e = (v - kv * half_vecs) * 8;
    const int head = e / D, d = e % D;
    const uint8_t* src = page + (static_cast<long long>((head * 2 + kv) << a.kb.page_shift) + row) * Row::BYTES;
    if constexpr (BITS == 4)
      codes[i] = make_uint2(*reinterpret_cast<const uint32_t*>(src + d / 2), 0u);
    else
      codes[i] = *reinterpret_cast<const uint2*>(src + d);
    par[i] = *reinterpret_cast<const __half2*>(src + Row::CODES + d / KV_GROUP * 4);
  }
#pragma unroll
  for (int i = 0; i < KV_IO_VECS; ++i) {
    const int v = vec0 + 32 * i;
    if (v >= 2 * half_vecs) continue;
    const __half2 s2 = __low2half2(par[i]), z2 = __high2half2(par[i]);
    uint4 out;
    if constexpr (BITS == 4) {
      __half2 c[4];
      kv_codes4(codes[i].x, c, KV_1024);  // pairs (0,4) (1,5) (2,6) (3,7)
      const uint32_t p0 = as_u32(__hfma2(c[0], s2, z2)), p1 = as_u32(__hfma2(c[1], s2, z2)),
                     p2 = as_u32(__hfma2(c[2], s2, z2)), p3 = as_u32(__hfma2(c[3], s2, z2));
      out = make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632),
                       __byte_perm(p2, p3, 0x7632));
    } else {
      out.x = as_u32(__hfma2(kv_codes8(codes[i].x, 0x4140), s2, z2));
      out.y = as_u32(__hfma2(kv_codes8(codes[i].x, 0x4342), s2, z2));
      out.z = as_u32(__hfma2(kv_codes8(codes[i].y, 0x4140), s2, z2));
      out.w = as_u32(__hfma2(kv_codes8(codes[i].y, 0x4342), s2, z2));
    }
    __half* dst = v < half_vecs ? a.out_k + t * a.k_stride + v * 8 : a.out_v + t * a.v_stride + (v - half_vecs) * 8;
    *reinterpret_cast<uint4*>(dst) = out;
  }
}

}  // namespace mm4
