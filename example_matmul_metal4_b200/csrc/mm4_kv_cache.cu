// Key / value cache plans and dispatch: argument checks, launches and the
// status words of the mm4_kv_cache_* entry points.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <new>

#include "kv_attention_few_sm100.cuh"
#include "kv_attention_many_sm100.cuh"
#include "kv_cache_sm100.cuh"
#include "mm4_internal.h"

using namespace mm4;

struct mm4_kv_cache_plan {
  mm4_kv_cache_desc d;
  float scale;
  int page_shift;
  long long page_bytes;
};

namespace {

constexpr int kMaxDevices = 64;
constexpr float LOG2E = 1.4426950408889634f;
// Set once a kernel that can write the status words was launched on a device;
// before that mm4_check has nothing to read there.
std::atomic<bool> g_used[kMaxDevices];

int row_bytes(const mm4_kv_cache_desc& d) { return d.head_dim * d.bits / 8 + d.head_dim / KV_GROUP * 4; }

mm4_status check_batch(const mm4_kv_cache_plan* p, const mm4_kv_cache_batch* b) {
  if (!p) return fail(MM4_ERR_INVALID, "null plan");
  if (!b) return fail(MM4_ERR_INVALID, "null batch");
  if (b->sequences < 0 || b->tokens < 0 || b->max_new < 0 || b->pages_per_sequence < 0)
    return fail(MM4_ERR_INVALID, "batch sizes must not be negative");
  if (b->sequences == 0 || b->tokens == 0) return MM4_OK;
  if (!b->page_table && b->pages_per_sequence > 0) return fail(MM4_ERR_INVALID, "null page table");
  if (!b->lengths || !b->offsets) return fail(MM4_ERR_INVALID, "null lengths or offsets");
  const void* ptrs[] = {b->page_table, b->lengths, b->offsets};
  for (const void* q : ptrs)
    if ((reinterpret_cast<uintptr_t>(q) & 3u) != 0)
      return fail(MM4_ERR_INVALID, "page_table, lengths and offsets must be 4-byte aligned");
  if ((static_cast<long long>(b->pages_per_sequence) << p->page_shift) > (1ll << 30))
    return fail(MM4_ERR_UNSUPPORTED, "a sequence of more than 2^30 tokens");
  return MM4_OK;
}

mm4_status check_rows(const char* name, const void* ptr, int64_t stride, int64_t width) {
  if (!ptr) return fail(MM4_ERR_INVALID, "null %s pointer", name);
  if (!aligned16(ptr)) return fail(MM4_ERR_INVALID, "%s must be 16-byte aligned", name);
  if (stride % 8 != 0 || stride < width)
    return fail(MM4_ERR_INVALID, "the rows of %s must be a multiple of 8 elements and at least %lld apart", name,
                static_cast<long long>(width));
  return MM4_OK;
}

mm4_status check_cache(const void* cache) {
  if (!cache) return fail(MM4_ERR_INVALID, "null cache pointer");
  if (!aligned16(cache)) return fail(MM4_ERR_INVALID, "the cache must be 16-byte aligned");
  return MM4_OK;
}

KvBatch batch_args(const mm4_kv_cache_plan* p, const mm4_kv_cache_batch* b) {
  KvBatch kb{};
  kb.table = b->page_table;
  kb.lengths = b->lengths;
  kb.offsets = b->offsets;
  kb.sequences = b->sequences;
  kb.tokens = b->tokens;
  kb.max_new = b->max_new;
  kb.pages_per_seq = b->pages_per_sequence;
  kb.page_shift = p->page_shift;
  kb.pages = p->d.pages;
  kb.heads_kv = p->d.heads_kv;
  kb.page_bytes = p->page_bytes;
  return kb;
}

mm4_status use_device(DeviceInfo* info) {
  mm4_status rc = current_device(info);
  if (rc != MM4_OK) return rc;
  if (info->device < 0 || info->device >= kMaxDevices)
    return fail(MM4_ERR_CUDA, "device id %d out of range", info->device);
  g_used[info->device].store(true);
  return MM4_OK;
}

// Calls f<D, BITS>() for the plan's head_dim and bits.
template <typename F>
mm4_status by_row(const mm4_kv_cache_desc& d, F&& f) {
  if (d.head_dim == 128)
    return d.bits == 4 ? f(KvRow<128, 4>{}, std::integral_constant<int, 128>{}, std::integral_constant<int, 4>{})
                       : f(KvRow<128, 8>{}, std::integral_constant<int, 128>{}, std::integral_constant<int, 8>{});
  return d.bits == 4 ? f(KvRow<64, 4>{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{})
                     : f(KvRow<64, 8>{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
}

mm4_status launch_io(const mm4_kv_cache_plan* p, KvIoArgs& a, bool write, cudaStream_t st) {
  DeviceInfo info;
  mm4_status rc = use_device(&info);
  if (rc != MM4_OK) return rc;
  const int vecs = 2 * p->d.heads_kv * p->d.head_dim / 8;
  a.parts = (vecs + KV_IO_PART - 1) / KV_IO_PART;
  // One token a warp until every SM has its 64 warps, then up to 8.
  const long long warps = static_cast<long long>(a.kb.tokens) * a.parts;
  a.tokens_per_warp = static_cast<int>(std::max(1ll, std::min(8ll, warps / (64ll * info.sm_count))));
  const long long groups = (a.kb.tokens + a.tokens_per_warp - 1) / a.tokens_per_warp;
  const long long blocks = (groups * a.parts + KV_IO_WARPS - 1) / KV_IO_WARPS;
  // Blocks of their own check the batch, beside the others and at no cost to them.
  const int checks = std::min(info.sm_count, (a.kb.sequences - 1) / (KV_IO_WARPS * 32) + 1);
  if (blocks + checks > 0x7fffffffLL) return fail(MM4_ERR_UNSUPPORTED, "too many tokens for one launch");
  a.blocks = static_cast<int>(blocks);
  const unsigned grid = static_cast<unsigned>(blocks + checks);
  return by_row(p->d, [&](auto, auto D, auto B) -> mm4_status {
    if (write)
      kv_append_kernel<D.value, B.value><<<grid, KV_IO_WARPS * 32, 0, st>>>(a);
    else
      kv_read_kernel<D.value, B.value><<<grid, KV_IO_WARPS * 32, 0, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, write ? "kv_append_kernel launch" : "kv_read_kernel launch");
    return MM4_OK;
  });
}

// Which kernel attention over a batch runs, from its sizes alone (the lengths
// lie on the device). Rows are the most that one key / value head has in one
// sequence: max_new tokens times the query heads that share it.
//   FEW    up to 8, 16 or 24 rows of a unit, and two units of 24: its time grows
//          with the units. MANY for more: 256 rows cost little more than one.
//          16 sequences of 4096 tokens, heads 32 / 8 of 128, 4 bits, one B200:
//          rows      24     48     72     96    256
//          FEW       42     72    100    128    327 us
//          MANY      75     76     77     77     84 us
//          (heads of 64, 8 bits: FEW 31, 50, 68, 86, 215, MANY 70, 73, 73, 75, 81).
//          The most rows of any sequence decide for all: 63 single tokens over up to
//          8192 take 102 us, a chunk of 1000 on 4000 takes 79, both in one call 365.
//   TEAM   FEW of at most 16 rows where no sequence can hold more than 2048 tokens
//          and there are no more units than the 148 SMs of a B200 (the workspace is
//          asked for without a device): a whole unit to a CTA, one launch, no
//          workspace. 8 heads, TEAM against split ranges, us:
//                                    64 tokens     512          1024         2048
//          128, 4 bits, 8 rows
//             1 sequence             6.2,  7.5   8.1,  8.3   9.9,  9.5  14.1,  9.9
//             4                      6.4,  8.0   8.3, 10.0  10.2, 10.7  14.0, 13.0
//             18                     6.6, 12.5   8.6, 16.1  10.6, 19.2  14.4, 23.1
//             64                    20.8, 13.4  27.8, 21.7  37.6, 30.1
//          128, 4 bits, 16 rows
//             1 sequence             6.9,  8.3   9.7, 10.0  12.5, 10.3  19.0, 11.1
//             18                     7.5, 13.1   9.9, 18.4  13.0, 20.5  20.0, 26.4
//             64                    23.0, 18.7  33.7, 28.6  45.4, 39.5
//          128, 8 bits, 8 rows
//             1 sequence             5.2,  7.5   7.7,  7.8  10.1,  8.1  15.8,  8.5
//             18                     5.4, 12.2   8.3, 15.8  10.6, 18.3  16.7, 23.1
//             64                    15.6, 13.1  25.7, 21.9  39.3, 37.2
//          64, 8 bits, 8 rows (4 bits alike)
//             1 sequence             4.6,  7.3   6.5,  8.5   8.1, 10.5  11.9, 10.8
//             18                     4.8, 10.3   6.6, 12.8   8.5, 14.6  12.2, 18.2
//             64                    14.0, 11.8  19.4, 18.7  25.7, 25.6
//          The room of a table is known here, the lengths in it are not: one or a few
//          sequences that nearly fill 2048 tokens are the ones that lose.
struct Form {
  enum Kind { FEW8, FEW16, FEW24, MANY } kind;
  bool team;
  size_t workspace;
  const char* name;
};

constexpr int kMaxCtas = 160;    // workspaces are sized for this many SMs
constexpr int kFewRows = 48;     // the most rows that FEW takes
constexpr int kTeamTokens = 2048;         // the most tokens of a sequence for TEAM
constexpr long long kTeamUnits = 148;     // and the most units (heads of sequences): one for each SM

Form attention_form(const mm4_kv_cache_plan* p, const mm4_kv_cache_batch* b) {
  const int group = p->d.heads_q / p->d.heads_kv;
  const long long rows = static_cast<long long>(b->max_new) * group;
  const long long room = static_cast<long long>(b->pages_per_sequence) << p->page_shift;
  Form f{};
  if (rows > kFewRows) {
    f.kind = Form::MANY;
    f.workspace = sizeof(float) * 2 * kMaxCtas * 256 * (p->d.head_dim + 2) + sizeof(KvmShared) * kMaxCtas;
    f.name = "kv_attention_many";
    return f;
  }
  f.kind = rows <= 8 ? Form::FEW8 : rows <= 16 ? Form::FEW16 : Form::FEW24;
  f.team = rows <= 16 && room <= kTeamTokens && static_cast<long long>(b->sequences) * p->d.heads_kv <= kTeamUnits;
  const int nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 3;
  const int warps = nt == 1 ? 15 : 7;  // at most
  if (!f.team) f.workspace = sizeof(float) * 2 * kMaxCtas * warps * 8 * nt * (p->d.head_dim + 2);
  static const char* const names[3][2] = {{"kv_attention_few<8 rows, split>", "kv_attention_few<8 rows, team>"},
                                          {"kv_attention_few<16 rows, split>", "kv_attention_few<16 rows, team>"},
                                          {"kv_attention_few<24 rows, split>", ""}};
  f.name = names[nt - 1][f.team ? 1 : 0];
  return f;
}

// Launches a join of partials, allowed to start while the kernel before it ends.
mm4_status launch_join(void (*kernel)(KvAttnArgs), dim3 grid, const KvAttnArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) return cuda_fail(e, "launch of the join of partials");
  return MM4_OK;
}

template <int D, int BITS, int NT, bool TEAM>
mm4_status launch_few(KvAttnArgs& a, int sms, cudaStream_t st) {
  const int blocks = (a.kb.max_new * a.group + 8 * NT - 1) / (8 * NT);
  using Cfg = KvFew<D, BITS, NT, TEAM>;
  mm4_status rc = ensure_smem_attr(reinterpret_cast<const void*>(kv_attention_few_kernel<D, BITS, NT, TEAM>),
                                   Cfg::SMEM_BYTES);
  if (rc != MM4_OK) return rc;
  const long long units = static_cast<long long>(a.kb.sequences) * a.kb.heads_kv;
  const unsigned grid = static_cast<unsigned>(TEAM ? std::min<long long>(units, sms) : sms);
  static_assert(Cfg::WARPS <= (NT == 1 ? 15 : 7), "attention_form sizes the workspace for this many");
  a.workers = sms * Cfg::WARPS;
  kv_attention_few_kernel<D, BITS, NT, TEAM><<<grid, Cfg::THREADS, Cfg::SMEM_BYTES, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "kv_attention_few_kernel launch");
  if (TEAM) return MM4_OK;
  // Up to 8 rows of a unit to a block of the join, one where that leaves SMs idle.
  const long long rows = std::min(8 * NT, a.kb.max_new * a.group);
  a.join_rows = 8;
  while (a.join_rows > 1 && units * blocks * ((rows + a.join_rows - 1) / a.join_rows) < 2 * sms) a.join_rows /= 2;
  const unsigned chunks = static_cast<unsigned>(blocks * ((rows + a.join_rows - 1) / a.join_rows));
  return launch_join(kv_attention_join_kernel<D, Cfg::ROWS, KVF_TK>, dim3(static_cast<unsigned>(units), chunks), a, st);
}

template <int D, int BITS>
mm4_status launch_many(KvAttnArgs& a, int sms, cudaStream_t st) {
  using Cfg = KvMany<D, BITS>;
  const void* kern = reinterpret_cast<const void*>(kv_attention_many_kernel<D, BITS>);
  mm4_status rc = ensure_smem_attr(kern, Cfg::SMEM_BYTES);
  if (rc != MM4_OK) return rc;
  {
    // The kernel moves registers between warpgroups (setmaxnreg); that only
    // completes if the launch allocates enough of them.
    static std::atomic<int> regs{0};
    int launch_regs = regs.load();
    if (launch_regs == 0) {
      cudaFuncAttributes fa;
      cudaError_t e = cudaFuncGetAttributes(&fa, kern);
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes(kv_attention_many_kernel)");
      regs.store(launch_regs = fa.numRegs);
    }
    if (launch_regs < Cfg::REGS_NEEDED)
      return fail(MM4_ERR_UNSUPPORTED, "attention kernel built with %d registers per thread, needs %d", launch_regs,
                  Cfg::REGS_NEEDED);
  }
  a.workers = sms;
  kv_attention_many_kernel<D, BITS><<<sms, KVM_THREADS, Cfg::SMEM_BYTES, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "kv_attention_many_kernel launch");
  if (sms < 2) return MM4_OK;
  return launch_join(kv_attention_many_join_kernel<D, Cfg::ROWS>, dim3(sms - 1, Cfg::ROWS / 32), a, st);
}

}  // namespace

namespace mm4 {

mm4_status kv_cache_take_status(int dev, int* wait, int* data) {
  if (dev < 0 || dev >= kMaxDevices || !g_used[dev].load()) return MM4_OK;
  const int zero = 0;
  MM4_CUDA_TRY(cudaMemcpyFromSymbol(wait, g_kv_wait, sizeof(int)));
  if (*wait != 0) MM4_CUDA_TRY(cudaMemcpyToSymbol(g_kv_wait, &zero, sizeof(int)));
  if (*wait != 0 || !data) return MM4_OK;
  MM4_CUDA_TRY(cudaMemcpyFromSymbol(data, g_kv_data, sizeof(int)));
  if (*data != 0) MM4_CUDA_TRY(cudaMemcpyToSymbol(g_kv_data, &zero, sizeof(int)));
  return MM4_OK;
}

const char* kv_cache_site_text(int site) {
  switch (site) {
    case KV_DATA_PAGE: return "a page number lies outside the pool";
    case KV_DATA_LENGTH: return "a length is negative or beyond the page table";
    case KV_DATA_OFFSETS: return "offsets are out of order or beyond the rows";
    case KV_DATA_NEW: return "a sequence has more rows than max_new";
    default: return "unknown";
  }
}

}  // namespace mm4

extern "C" {

mm4_status mm4_kv_cache_plan_create(mm4_kv_cache_plan** out, const mm4_kv_cache_desc* d) {
  if (!out) return fail(MM4_ERR_INVALID, "null plan pointer");
  *out = nullptr;
  if (!d) return fail(MM4_ERR_INVALID, "null key / value cache descriptor");
  if (d->pages <= 0 || d->heads_q <= 0 || d->heads_kv <= 0 || d->head_dim <= 0)
    return fail(MM4_ERR_INVALID, "pages, heads and head_dim must be positive");
  if (d->heads_q % d->heads_kv != 0)
    return fail(MM4_ERR_INVALID, "heads_kv (%d) must divide heads_q (%d)", d->heads_kv, d->heads_q);
  if (d->page_size < 16 || d->page_size > 256 || (d->page_size & (d->page_size - 1)) != 0)
    return fail(MM4_ERR_INVALID, "page_size %d: 16, 32, 64, 128 or 256", d->page_size);
  if (d->bits != 4 && d->bits != 8) return fail(MM4_ERR_INVALID, "bits %d: 4 or 8", d->bits);
  if (d->causal != 0 && d->causal != 1) return fail(MM4_ERR_INVALID, "causal must be 0 or 1");
  if (d->head_dim != 128 && d->head_dim != 64)
    return fail(MM4_ERR_UNSUPPORTED, "head_dim %d: this build implements head_dim 128 and 64", d->head_dim);
  if (std::isnan(d->scale) || std::isinf(d->scale)) return fail(MM4_ERR_INVALID, "scale must be finite");
  if (d->scale > 0.f && std::isinf(d->scale * LOG2E)) return fail(MM4_ERR_UNSUPPORTED, "scale %g: at most 2^127", d->scale);
  if (d->heads_q > 4096) return fail(MM4_ERR_UNSUPPORTED, "heads_q %d: at most 4096", d->heads_q);
  if (d->pages > 0x7fffffffLL) return fail(MM4_ERR_UNSUPPORTED, "more than 2^31 - 1 pages");
  mm4_kv_cache_plan* p = new (std::nothrow) mm4_kv_cache_plan();
  if (!p) return fail(MM4_ERR_INVALID, "out of host memory");
  p->d = *d;
  p->scale = d->scale > 0.f ? d->scale : 1.0f / std::sqrt(static_cast<float>(d->head_dim));
  p->page_shift = 0;
  while ((1 << p->page_shift) < d->page_size) ++p->page_shift;
  p->page_bytes = 2ll * d->heads_kv * d->page_size * row_bytes(*d);
  *out = p;
  return MM4_OK;
}

void mm4_kv_cache_plan_destroy(mm4_kv_cache_plan* plan) { delete plan; }

size_t mm4_kv_cache_page_bytes(const mm4_kv_cache_plan* p) { return p ? static_cast<size_t>(p->page_bytes) : 0; }

size_t mm4_kv_cache_bytes(const mm4_kv_cache_plan* p) {
  return p ? static_cast<size_t>(p->page_bytes) * static_cast<size_t>(p->d.pages) : 0;
}

mm4_status mm4_kv_cache_append(const mm4_kv_cache_plan* p, const mm4_kv_cache_batch* b, const void* K,
                               int64_t k_stride, const void* V, int64_t v_stride, void* cache, mm4_stream_t stream) {
  mm4_status rc = check_batch(p, b);
  if (rc != MM4_OK) return rc;
  if (b->sequences == 0 || b->tokens == 0) return MM4_OK;
  const int64_t width = static_cast<int64_t>(p->d.heads_kv) * p->d.head_dim;
  if ((rc = check_rows("K", K, k_stride, width)) != MM4_OK) return rc;
  if ((rc = check_rows("V", V, v_stride, width)) != MM4_OK) return rc;
  if ((rc = check_cache(cache)) != MM4_OK) return rc;
  KvIoArgs a{};
  a.kb = batch_args(p, b);
  a.in_k = static_cast<const __half*>(K);
  a.in_v = static_cast<const __half*>(V);
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.cache = static_cast<uint8_t*>(cache);
  return launch_io(p, a, true, static_cast<cudaStream_t>(stream));
}

mm4_status mm4_kv_cache_read(const mm4_kv_cache_plan* p, const mm4_kv_cache_batch* b, const void* cache, void* K,
                             int64_t k_stride, void* V, int64_t v_stride, mm4_stream_t stream) {
  mm4_status rc = check_batch(p, b);
  if (rc != MM4_OK) return rc;
  if (b->sequences == 0 || b->tokens == 0) return MM4_OK;
  const int64_t width = static_cast<int64_t>(p->d.heads_kv) * p->d.head_dim;
  if ((rc = check_rows("K", K, k_stride, width)) != MM4_OK) return rc;
  if ((rc = check_rows("V", V, v_stride, width)) != MM4_OK) return rc;
  if ((rc = check_cache(cache)) != MM4_OK) return rc;
  KvIoArgs a{};
  a.kb = batch_args(p, b);
  a.out_k = static_cast<__half*>(K);
  a.out_v = static_cast<__half*>(V);
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.cache = static_cast<uint8_t*>(const_cast<void*>(cache));
  return launch_io(p, a, false, static_cast<cudaStream_t>(stream));
}

size_t mm4_kv_cache_attention_workspace_size(const mm4_kv_cache_plan* p, const mm4_kv_cache_batch* b) {
  if (!p || !b || b->sequences <= 0 || b->tokens <= 0 || b->max_new <= 0) return 0;
  return attention_form(p, b).workspace;
}

const char* mm4_kv_cache_attention_kernel_name(const mm4_kv_cache_plan* p, const mm4_kv_cache_batch* b) {
  if (!p || !b) return "";
  return attention_form(p, b).name;
}

mm4_status mm4_kv_cache_attention(const mm4_kv_cache_plan* p, const mm4_kv_cache_batch* b, const void* Q,
                                  int64_t q_stride, const void* cache, void* O, int64_t o_stride, float* lse,
                                  void* workspace, size_t workspace_bytes, mm4_stream_t stream) {
  mm4_status rc = check_batch(p, b);
  if (rc != MM4_OK) return rc;
  if (b->sequences == 0 || b->tokens == 0) return MM4_OK;
  if (b->max_new < 1) return fail(MM4_ERR_INVALID, "max_new must be at least 1");
  const int64_t width = static_cast<int64_t>(p->d.heads_q) * p->d.head_dim;
  if ((rc = check_rows("Q", Q, q_stride, width)) != MM4_OK) return rc;
  if ((rc = check_rows("O", O, o_stride, width)) != MM4_OK) return rc;
  if ((rc = check_cache(cache)) != MM4_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(lse) & 3u) != 0) return fail(MM4_ERR_INVALID, "lse must be 4-byte aligned");
  if (static_cast<long long>(b->max_new) * (p->d.heads_q / p->d.heads_kv) > (1 << 28) ||
      static_cast<long long>(b->sequences) * p->d.heads_kv > 0x7fffffffLL)
    return fail(MM4_ERR_UNSUPPORTED, "too many rows or sequences for one launch");
  const Form form = attention_form(p, b);
  if (form.workspace > 0) {
    if (!workspace || workspace_bytes < form.workspace)
      return fail(MM4_ERR_WORKSPACE, "attention over this batch needs a %zu-byte workspace", form.workspace);
    if (!aligned16(workspace)) return fail(MM4_ERR_INVALID, "workspace must be 16-byte aligned");
  }
  // Workers read the Q of a unit when others have written their rows of O.
  if (O == Q) return fail(MM4_ERR_INVALID, "O must not be Q");
  DeviceInfo info;
  if ((rc = use_device(&info)) != MM4_OK) return rc;
  KvAttnArgs a{};
  a.kb = batch_args(p, b);
  a.Q = static_cast<const __half*>(Q);
  a.O = static_cast<__half*>(O);
  a.lse = lse;
  a.q_stride = q_stride;
  a.o_stride = o_stride;
  a.cache = static_cast<const uint8_t*>(cache);
  a.heads_q = p->d.heads_q;
  a.group = p->d.heads_q / p->d.heads_kv;
  a.causal = p->d.causal;
  a.scale_log2 = p->scale * LOG2E;
  a.partials = static_cast<float*>(workspace);
  a.k1024 = KV_1024;
  a.timeout_ns = wait_timeout_ns();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = std::min(info.sm_count, kMaxCtas);
  return by_row(p->d, [&](auto, auto D, auto B) -> mm4_status {
    if (form.kind == Form::FEW8)
      return form.team ? launch_few<D.value, B.value, 1, true>(a, sms, st)
                       : launch_few<D.value, B.value, 1, false>(a, sms, st);
    if (form.kind == Form::FEW16)
      return form.team ? launch_few<D.value, B.value, 2, true>(a, sms, st)
                       : launch_few<D.value, B.value, 2, false>(a, sms, st);
    if (form.kind == Form::FEW24) return launch_few<D.value, B.value, 3, false>(a, sms, st);
    return launch_many<D.value, B.value>(a, sms, st);
  });
}

}  // extern "C"
