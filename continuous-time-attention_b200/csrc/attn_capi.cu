// C ABI of the attention and key/value-cache operators: argument checks, the
// choice of kernel, launches.  Declarations and contracts live in
// include/cta_stencil.h.
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <mutex>

#include "attn_tc.cuh"
#include "cta_stencil.h"

namespace cta {
void set_last_error(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
}

using namespace cta;

namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

}  // namespace

bool cta::attn_map(CUtensorMap* m, const void* base, int dtype, int64_t nb, int64_t tokens, int64_t heads, int64_t d,
                   const AttnStrides& s, int box_heads, int box_tokens) {
  const auto fn = encode_fn();
  if (fn == nullptr || reinterpret_cast<uintptr_t>(base) % 16 != 0 || d % 8 != 0) return false;
  // the stride of an axis of one entry means nothing: any valid one
  const int64_t row = 2 * d;
  const int64_t st[3] = {heads == 1 ? row : 2 * s.h, tokens == 1 ? row : 2 * s.t, nb == 1 ? row : 2 * s.b};
  for (int64_t x : st)
    if (x <= 0 || x % 16 != 0 || x >= (1LL << 40)) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(nb)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(st[0]), static_cast<cuuint64_t>(st[1]),
                                 static_cast<cuuint64_t>(st[2])};
  const cuuint32_t box[4] = {64u, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens), 1u};
  const cuuint32_t step[4] = {1u, 1u, 1u, 1u};
  return fn(m, dtype == CTA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr int kMaxHeadDim = 256;

#define fail(code, ...) (set_last_error(__VA_ARGS__), (code))

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return CTA_OK;
  return fail(CTA_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

AttnStrides strides(const int64_t s[3]) { return AttnStrides{s[0], s[1], s[2]}; }

// argument checks shared by both directions; kNothing = an empty call
constexpr int kNothing = -1;
int prompt_args(const cta_attention_args* p, AttnArgs& a) {
  if (p == nullptr) return fail(CTA_EINVAL, "null arguments");
  if (p->dtype != CTA_F32 && p->dtype != CTA_BF16 && p->dtype != CTA_F16)
    return fail(CTA_EINVAL, "unsupported dtype code %d", p->dtype);
  if (p->batch < 0 || p->length < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0)
    return fail(CTA_EINVAL, "bad shape: batch %lld, length %lld, heads %lld, kv_heads %lld", (long long)p->batch,
                (long long)p->length, (long long)p->heads, (long long)p->kv_heads);
  if (p->dim < 1 || p->dim > kMaxHeadDim)
    return fail(CTA_EINVAL, "head dim must be in 1..%d, got %lld", kMaxHeadDim, (long long)p->dim);
  if (p->length >= (1LL << 30) || p->batch >= (1LL << 30) || p->heads >= (1LL << 20))
    return fail(CTA_EUNSUPPORTED, "batch, length and heads must be below 2^30, 2^30 and 2^20");
  if (p->cu_seqlens != nullptr && p->mask_words != nullptr)
    return fail(CTA_EINVAL, "a key mask takes padded sequences, not packed ones");
  // packed rows without sequences all lie behind the last one and may have to be cleared
  if ((p->batch == 0 && p->cu_seqlens == nullptr) || p->length == 0) return kNothing;
  if (p->q == nullptr || p->k == nullptr || p->v == nullptr || p->out == nullptr)
    return fail(CTA_EINVAL, "null tensor pointer");
  std::memset(&a, 0, sizeof(a));
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.o = p->out;
  a.low = p->dtype == CTA_F32 ? nullptr : p->out_low;
  a.lse = p->lse;
  a.g = p->grad_out;
  a.delta = p->delta;
  a.dq = p->dq;
  a.dk = p->dk;
  a.dv = p->dv;
  a.qs = strides(p->q_stride);
  a.ks = strides(p->k_stride);
  a.vs = strides(p->v_stride);
  a.os = strides(p->out_stride);
  a.gs = strides(p->grad_stride);
  a.dqs = strides(p->dq_stride);
  a.dks = strides(p->dk_stride);
  a.dvs = strides(p->dv_stride);
  a.cu = p->cu_seqlens;
  a.mask = p->mask_words;
  a.mask_words = cta_attention_mask_words_per_row(p->length);
  a.L = p->length;
  a.nseq = static_cast<int>(p->batch);
  a.H = static_cast<int>(p->heads);
  a.Hk = static_cast<int>(p->kv_heads);
  a.d = static_cast<int>(p->dim);
  a.causal = p->causal != 0;
  a.zero_tail = p->zero_tail != 0;
  a.scale = p->scale;
  return CTA_OK;
}

int cache_args(const cta_kv_cache_args* p, bool write, CacheArgs& a) {
  if (p == nullptr) return fail(CTA_EINVAL, "null arguments");
  if (p->dtype != CTA_BF16 && p->dtype != CTA_F16)
    return fail(CTA_EINVAL, "the cache takes bf16 or fp16 rows, got dtype code %d", p->dtype);
  if (p->tokens < 0 || p->kv_heads < 1 || p->pages < 0 || p->page_size < 1)
    return fail(CTA_EINVAL, "bad cache shape");
  if (p->dim < 16 || p->dim > kMaxHeadDim || p->dim % 16 != 0)
    return fail(CTA_EINVAL, "the cache's head dim must be a multiple of 16 in 16..%d, got %lld", kMaxHeadDim,
                (long long)p->dim);
  // the kernels number up to 32 lanes per token and four heads in 32 bits
  if (p->pages >= (1LL << 31) || p->page_size >= (1LL << 31) || p->pages * p->page_size >= (1LL << 31) ||
      p->tokens >= (1LL << 27) || p->kv_heads >= (1LL << 20) || p->tokens * ((p->kv_heads + 3) / 4) >= (1LL << 27))
    return fail(CTA_EUNSUPPORTED, "slots must be below 2^31, tokens * ceil(heads / 4) below 2^27, heads below 2^20");
  if (p->quantized && p->pages > 0 && (p->k_scale == nullptr || p->v_scale == nullptr))
    return fail(CTA_EINVAL, "an e4m3 cache needs its scales");
  if (p->tokens == 0) return kNothing;
  // a pool without pages has no address
  if (p->k == nullptr || p->v == nullptr || p->slots == nullptr ||
      (p->pages > 0 && (p->k_cache == nullptr || p->v_cache == nullptr)))
    return fail(CTA_EINVAL, "null tensor pointer");
  const int64_t rows = 8, cells = p->quantized ? 16 : 8;  // elements in 16 bytes
  for (int64_t s : {p->k_stride[0], p->k_stride[1], p->v_stride[0], p->v_stride[1]})
    if (s % rows != 0) return fail(CTA_EINVAL, "rows must start on 16 bytes");
  for (int64_t s : {p->k_cache_stride[0], p->k_cache_stride[1], p->k_cache_stride[2], p->v_cache_stride[0],
                    p->v_cache_stride[1], p->v_cache_stride[2]})
    if (s % cells != 0) return fail(CTA_EINVAL, "the cache's rows must start on 16 bytes");
  for (const void* x : {p->k, p->v, (const void*)p->k_cache, (const void*)p->v_cache})
    if (reinterpret_cast<uintptr_t>(x) % 16 != 0) return fail(CTA_EINVAL, "tensors must start on 16 bytes");
  std::memset(&a, 0, sizeof(a));
  if (write) {
    a.k_in = p->k;
    a.v_in = p->v;
  } else {
    a.k_out = const_cast<void*>(p->k);
    a.v_out = const_cast<void*>(p->v);
  }
  a.k_sT = p->k_stride[0];
  a.k_sH = p->k_stride[1];
  a.v_sT = p->v_stride[0];
  a.v_sH = p->v_stride[1];
  a.k_cache = p->k_cache;
  a.v_cache = p->v_cache;
  a.kc_sP = p->k_cache_stride[0];
  a.kc_sS = p->k_cache_stride[1];
  a.kc_sH = p->k_cache_stride[2];
  a.vc_sP = p->v_cache_stride[0];
  a.vc_sS = p->v_cache_stride[1];
  a.vc_sH = p->v_cache_stride[2];
  a.k_scale = p->k_scale;
  a.v_scale = p->v_scale;
  a.slots = p->slots;
  a.T = p->tokens;
  a.n_slots = p->pages * p->page_size;
  a.page = static_cast<int>(p->page_size);
  a.Hk = static_cast<int>(p->kv_heads);
  a.d = static_cast<int>(p->dim);
  a.quantized = p->quantized != 0;
  return CTA_OK;
}

// A sliding window and the first keys that stay visible, as the kernels take them.  A window that reaches over all of
// `length` keys, whatever the sinks, is none.
int window_args(int64_t window, int64_t sinks, int64_t length, int& w, int& s) {
  if (window < 0 || sinks < 0) return fail(CTA_EINVAL, "window and sinks must not be negative");
  if (window == 0 && sinks != 0) return fail(CTA_EINVAL, "sinks go with a window");
  w = s = 0;
  if (window == 0 || window >= length || sinks >= length - window) return CTA_OK;
  w = static_cast<int>(window);  // both below `length`
  s = static_cast<int>(sinks);
  return CTA_OK;
}
int prompt_window(const cta_attention_args* p, int64_t window, int64_t sinks, AttnArgs& a) {
  if (p != nullptr && window > 0 && !p->causal) return fail(CTA_EINVAL, "a window needs the causal mask");
  const int rc = prompt_args(p, a);
  if (rc != CTA_OK && rc != kNothing) return rc;
  const int wrc = window_args(window, sinks, p->length, a.window, a.sinks);
  return wrc != CTA_OK ? wrc : rc;
}

int paged_args(const cta_paged_attention_args* p, PagedArgs& a) {
  if (p == nullptr) return fail(CTA_EINVAL, "null arguments");
  if (p->dtype != CTA_BF16 && p->dtype != CTA_F16)
    return fail(CTA_EINVAL, "paged attention takes bf16 or fp16, got dtype code %d", p->dtype);
  if (p->rows < 0 || p->batch < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0)
    return fail(CTA_EINVAL, "bad shape: rows %lld, batch %lld, heads %lld, kv_heads %lld", (long long)p->rows,
                (long long)p->batch, (long long)p->heads, (long long)p->kv_heads);
  if (p->dim < 16 || p->dim > 128 || p->dim % 16 != 0)
    return fail(CTA_EINVAL, "paged attention's head dim must be a multiple of 16 in 16..128, got %lld",
                (long long)p->dim);
  if (p->page_size < 16 || p->page_size % 16 != 0)
    return fail(CTA_EINVAL, "the page size must be a multiple of 16, got %lld", (long long)p->page_size);
  // key numbers, a tile past the last one included, and (row, head) pairs are 32-bit
  constexpr int64_t most = (1LL << 31) - 256;
  if (p->pages < 0 || p->pages >= most || p->page_size >= most || p->pages * p->page_size >= most ||
      p->table_width < 0 || p->table_width >= most || p->table_width * p->page_size >= most || p->rows >= (1LL << 28) ||
      p->batch >= (1LL << 28) || p->heads >= (1LL << 20) || p->rows * p->heads >= most)
    return fail(CTA_EUNSUPPORTED,
                "slots, table_width * page_size and rows * heads must be below 2^31 - 256, rows and batch below 2^28, "
                "heads below 2^20");
  if (p->max_rows < 1) return fail(CTA_EINVAL, "max_rows must be at least 1");
  if (p->cu_seqlens == nullptr && p->rows != p->batch)
    return fail(CTA_EINVAL, "without offsets there is one row per sequence: %lld rows, %lld sequences",
                (long long)p->rows, (long long)p->batch);
  if (p->quantized && p->pages > 0 && (p->k_scale == nullptr || p->v_scale == nullptr))
    return fail(CTA_EINVAL, "an e4m3 cache needs its scales");
  std::memset(&a, 0, sizeof(a));
  a.q = p->q;
  a.o = p->out;
  a.q_sT = p->q_stride[0];
  a.q_sH = p->q_stride[1];
  a.o_sT = p->out_stride[0];
  a.o_sH = p->out_stride[1];
  a.k_cache = p->k_cache;
  a.v_cache = p->v_cache;
  a.kc_sP = p->k_cache_stride[0];
  a.kc_sS = p->k_cache_stride[1];
  a.kc_sH = p->k_cache_stride[2];
  a.vc_sP = p->v_cache_stride[0];
  a.vc_sS = p->v_cache_stride[1];
  a.vc_sH = p->v_cache_stride[2];
  a.k_scale = p->quantized ? p->k_scale : nullptr;
  a.v_scale = p->quantized ? p->v_scale : nullptr;
  a.table = p->block_table;
  a.table_sB = p->table_stride;
  a.seq_lens = p->seq_lens;
  a.cu = p->cu_seqlens;
  a.T = p->rows;
  a.B = static_cast<int>(p->batch);
  a.H = static_cast<int>(p->heads);
  a.Hk = static_cast<int>(p->kv_heads);
  a.d = static_cast<int>(p->dim);
  a.page = static_cast<int>(p->page_size);
  a.table_width = static_cast<int>(p->table_width);
  a.n_pages = static_cast<int>(p->pages);
  a.max_rows = static_cast<int>(p->max_rows < p->rows ? p->max_rows : p->rows);
  a.scale = p->scale;
  return CTA_OK;
}

int paged_window(const cta_paged_attention_args* p, int64_t window, int64_t sinks, PagedArgs& a) {
  const int rc = paged_args(p, a);
  if (rc != CTA_OK) return rc;
  const int64_t keys = p->table_width * p->page_size;
  const int wrc = window_args(window, sinks, keys, a.window, a.sinks);
  if (wrc != CTA_OK) return wrc;
  if (a.window > 0 && keys >= (1LL << 30))  // the split kernel counts groups past the last key
    return fail(CTA_EUNSUPPORTED, "table_width * page_size must be below 2^30 with a window");
  return CTA_OK;
}

// The tensor-core kernel takes 128 (row, head) pairs at once but has a CTA per pair of such tiles only;
// the split kernel takes 16, reads the keys again for each 16, and fills the GPU whatever the shape.
// Measured (32/8 heads of 128, B200): a 16-row tile costs the split kernel 0.11 ns per key, a pass of
// the other kernel over one wave of its CTAs 15 ns per key, i.e. as much as 137 such tiles.  One
// sequence of 8192 keys: 64 rows 96 us split, 142 us on tensor cores; 128 rows 179 and 144 us.  8
// sequences of 4096: 8 rows 65 and 69 us, 16 rows 112 and 70 us.  Over an e4m3 cache the pages have to
// be expanded first: 32 sequences of 2048, 8 rows 119 and 198 us, 16 rows 225 and 199 us (fp16 232); one of
// 8192 keys, 512 rows: 675 and 299 us (fp16 408).
//
// What TMA cannot address, a pool without pages among it, is for the split kernel.
bool tma_strides(std::initializer_list<int64_t> elements) {
  for (int64_t s : elements)
    if (s <= 0 || s >= (1LL << 39)) return false;
  return true;
}
bool tma_can_address(const PagedArgs& a) {
  // an axis of one entry has no stride
  const auto axis = [](int64_t entries, int64_t stride) { return entries == 1 ? int64_t{8} : stride; };
  if (!tma_strides({axis(a.T, a.q_sT), axis(a.H, a.q_sH)})) return false;
  if (a.k_scale != nullptr) return true;  // the expanded copy is what TMA reads
  return a.n_pages > 0 && tma_strides({axis(a.n_pages, a.kc_sP), axis(a.page, a.kc_sS), axis(a.Hk, a.kc_sH),
                                       axis(a.n_pages, a.vc_sP), axis(a.page, a.vc_sS), axis(a.Hk, a.vc_sH)});
}
bool tensor_cores_pay(const PagedArgs& a) {
  if (!tma_can_address(a)) return false;
  const int64_t group = a.H / a.Hk, pack = attn_pack(static_cast<int>(group));
  if (a.cu == nullptr || a.max_rows * group <= 16 || !(a.scale > 0.f)) return false;
  const int64_t b = a.B;
  const int64_t tiles = std::max(b, (a.T * group + 15) / 16) * a.Hk;
  const int64_t ctas = std::max(b, (a.T * pack + 255) / 256) * (a.H / pack);
  return tiles > (a.k_scale != nullptr ? 256 : 128) * ((ctas + 147) / 148);
}

// 16-bit copy of the pages that the table can name, k then v, and what goes beside them; 0 where that is too much to
// ask for
constexpr int64_t kMostExpanded = 1LL << 31;
int64_t copy_bytes(int64_t slots, int64_t beside, int64_t hk, int64_t d) {
  if (slots >= (1LL << 24) || slots * hk >= (1LL << 26)) return 0;
  const int64_t bytes = slots * hk * d * 4 + beside * hk * 8;
  return bytes > 0 && bytes <= kMostExpanded ? bytes + 32 : 0;  // and what puts its start on 32 bytes
}
int64_t expanded_bytes(int64_t b, int64_t width, int64_t page, int64_t hk, int64_t d) {
  return copy_bytes(b * width * page, b * residue_row(width * page), hk, d);
}
// of chunks, and where their keys go under a window
int64_t chunk_bytes(PagedArgs& a) {
  if (a.window == 0) return expanded_bytes(a.B, a.table_width, a.page, a.Hk, a.d);
  plan_copy_slots(a);
  return copy_bytes(a.copy_slots, a.copy_slots, a.Hk, a.d);
}

int64_t split_bytes(int workers, int d) {
  return 2LL * workers * 16 * ((d <= 64 ? 64 : 128) + 4) * static_cast<int64_t>(sizeof(float));
}

// The arguments' pointers and the workspace.
int paged_pointers(const PagedArgs& a, int quantized, const void* workspace, int64_t workspace_bytes, int64_t need) {
  // a pool without pages and a table without entries have no address
  if (a.q == nullptr || a.o == nullptr || (a.n_pages > 0 && (a.k_cache == nullptr || a.v_cache == nullptr)) ||
      (a.table == nullptr && a.table_width > 0) || a.seq_lens == nullptr)
    return fail(CTA_EINVAL, "null tensor pointer");
  const int64_t cells = quantized ? 16 : 8;
  for (int64_t s : {a.q_sT, a.q_sH, a.o_sT, a.o_sH})
    if (s % 8 != 0) return fail(CTA_EINVAL, "rows must start on 16 bytes");
  for (int64_t s : {a.kc_sP, a.kc_sS, a.kc_sH, a.vc_sP, a.vc_sS, a.vc_sH})
    if (s % cells != 0) return fail(CTA_EINVAL, "the cache's rows must start on 16 bytes");
  for (const void* x : {a.q, static_cast<const void*>(a.o), a.k_cache, a.v_cache, workspace})
    if (reinterpret_cast<uintptr_t>(x) % 16 != 0) return fail(CTA_EINVAL, "tensors must start on 16 bytes");
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(CTA_EINVAL, "workspace of %lld bytes needed, got %lld", (long long)need, (long long)workspace_bytes);
  return CTA_OK;
}

// Expands the pages of an e4m3 cache that p's table names into `ws`, and points x at them.
cudaError_t expand_pages(const PagedArgs& p, int dtype, char* ws, PagedArgs& x, cudaStream_t st) {
  const int64_t pages = static_cast<int64_t>(p.B) * p.table_width;
  const int64_t part = (p.window > 0 ? p.copy_slots : pages * p.page) * p.Hk * p.d * 2;
  ws += -reinterpret_cast<intptr_t>(ws) & 31;
  float* k_res = reinterpret_cast<float*>(ws + 2 * part);
  float* v_res = k_res + (p.window > 0 ? p.copy_slots : p.B * residue_row(static_cast<int64_t>(p.table_width) * p.page)) * p.Hk;
  PagedArgs fold = p;
  fold.fold_scale = p.window > 0 || p.seq_lens == nullptr;  // windows, and the whole table of a prefix
  const cudaError_t e = launch_cache_expand(fold, dtype, ws, ws + part, k_res, v_res, st);
  x.k_cache = ws;
  x.v_cache = ws + part;
  x.k_res = k_res;
  x.v_res = v_res;
  x.expanded_pages = pages;
  return e;
}

// The plan of a batch with a shared prefix: the prefix in parts on the tensor cores, 256 (row, head) pairs at once, then
// the sequences' own keys in the split kernel, whose join takes the parts in.  Not of chunks for the tensor cores, whose
// kernel goes through each sequence's pages.
struct PrefixPlan {
  int keys = 0;  // 0: the prefix is not used
  int splits = 0, chunk = 0;
  int64_t sums = 0, expanded = 0, bytes = 0;  // workspace: the parts, the expanded pages, all with the split kernel's
};

std::atomic<int> g_prefix_always{0};

PrefixPlan prefix_plan(const PagedArgs& a, int dtype, int quantized, int64_t shared) {
  PrefixPlan p;
  const int64_t width = a.table_width, keys = std::min(shared / a.page, width) * a.page;
  // the split kernel counts groups past the last key, hence 2^30
  if (a.T < 2 || keys < 1 || width * a.page >= (1LL << 30) || !(a.scale > 0.f) || !tma_can_address(a) || tensor_cores_pay(a) ||
      a.n_pages < 1)
    return p;
  // It costs a launch, two over e4m3, the sums' way through memory, and a split kernel whose last workers start when the
  // parts are done; and what is read again comes from L2 in part.  So it is for calls that spare 120 MB, over e4m3, where
  // reading is bound by the codes' conversion, 450,000 rows of k and of v (fp16, whose parts take longer, 900,000).  How
  // many keys of their own the sequences have is not known here (a block table is as wide as its owner's longest
  // sequence may ever be), so it has to do for few and for many.  GPU time with and without it, 32/8 heads of 128: 16
  // sequences of 16 to 64, 16 to 1024, 2048 to 4096 own keys behind 2048, 126 MB, 16, 25, 55 and 27, 31, 54 us; 4 behind
  // 8192, 100 MB, 25, 26, 40 and 30, 30, 36.  e4m3, few and many: 64 behind 1024, 516,000 rows, 22, 127 and 39, 125, in
  // fp16 24, 129 and 39, 117; 16 behind 2048, 246,000 rows, 21, 55 and 25, 51.  The worst found: 128 of 2048 to 4096 own
  // keys behind 2048, 8/1 heads, whose prefix L2 holds, 61 and 55.
  const int64_t rows = (std::max<int64_t>(a.B, (a.T * (a.H / a.Hk) + 15) / 16) - 1) * keys * a.Hk;  // of k and of v, read again
  const double bytes = static_cast<double>(rows) * 2 * (quantized ? a.d + 4 : 2 * a.d);
  const bool pays = !quantized ? bytes >= 120e6 : rows >= (dtype == CTA_F16 ? 900000 : 450000);
  if (!pays && g_prefix_always.load(std::memory_order_relaxed) == 0) return p;
  const int64_t tiles = (keys + 127) / 128, ctas = prefix_tiles(a);
  // Both kernels run at once, a part on an SM of its own; the workers that find no room start when a part ends.  Few long
  // parts keep the call waiting where the own keys are few, many short ones keep their SMs from them where they are many.
  // A part takes 12 us and 3.5 for each key tile (e4m3 3.8, in fp16 5.5), measured; it is to end within a seventh of what
  // reading the prefix again would take, and within 16 tiles, on 64 to 112 SMs.  Own keys as above, 64 sequences behind
  // 8192: 8 parts (64 SMs), the rule's, 41, 63, 165 us, 13 parts 34, 68, 163, 5 parts 55, 60, 174; without 218, 233, 307.
  // 16 behind 8192: 13 parts, the rule's, 26, 35, 62, 8 parts 33, 36, 69.  4 behind 16384: 13 parts, the rule's, 39, 40, 48, 8
  // parts 55, 56, 59; without 43, 44, 51.  128 behind 16384, e4m3 in fp16, up to 512 own keys: 7 parts (112 SMs), the rule's,
  // 134, 8 parts 148, 6 parts 147.
  const double tile_us = !quantized ? 3.5 : dtype == CTA_F16 ? 5.5 : 3.8, again_us = bytes / 6.5e6;
  const double longest = std::min(16., std::max(1., (again_us / 7. - 12.) / tile_us));  // key tiles of a part
  const int64_t few = std::max<int64_t>(1, 64 / ctas), many = std::max<int64_t>(1, 112 / ctas);
  const int64_t most = std::max(few, std::min(many, static_cast<int64_t>(std::ceil(tiles / longest))));
  const int64_t per = (tiles + most - 1) / most, splits = (tiles + per - 1) / per;
  const int dp = a.d <= 64 ? 64 : 128;
  // the values' rows start on 32 bytes, the workspace on 16
  const int64_t sums = 32 + (splits + 1) * a.T * a.H * (dp + 4) * static_cast<int64_t>(sizeof(float));
  int64_t expanded = 0;
  if (quantized) {
    expanded = expanded_bytes(1, keys / a.page, a.page, a.Hk, a.d);
    if (expanded == 0) return p;
  }
  if (sums > (1LL << 30)) return p;
  PagedArgs x = a;
  x.skip = static_cast<int>(keys);
  p.keys = x.skip;
  p.splits = static_cast<int>(splits);
  p.chunk = static_cast<int>(per * 128);
  p.sums = sums;
  p.expanded = expanded;
  p.bytes = sums + expanded + split_bytes(paged_split_workers(x, dtype, quantized), a.d);
  return p;
}

}  // namespace

int cta::set_prefix_always(int value) { return g_prefix_always.exchange(value != 0 ? 1 : 0); }

extern "C" {

int64_t cta_attention_mask_words_per_row(int64_t length) { return kMaskHead + (length + 127) / 128 * 4; }

int cta_attention_mask_words(const void* mask, int mask_dtype, int64_t mask_sB, int64_t mask_sL, int64_t B, int64_t L,
                             uint32_t* words, void* stream) {
  if (B < 0 || L < 0 || L >= (1LL << 30) || B >= (1LL << 30)) return fail(CTA_EINVAL, "bad mask shape");
  if (mask_dtype < CTA_MASK_U8 || mask_dtype > CTA_MASK_F16) return fail(CTA_EINVAL, "bad mask dtype %d", mask_dtype);
  if (B == 0) return CTA_OK;
  if (mask == nullptr || words == nullptr) return fail(CTA_EINVAL, "null mask pointer");
  return launched(launch_attn_mask_words(mask, mask_dtype, mask_sB, mask_sL, B, L, words,
                                         cta_attention_mask_words_per_row(L), static_cast<cudaStream_t>(stream)),
                  "attention mask launch");
}

int cta_attention_forward(const cta_attention_args* args, void* stream) {
  return cta_window_attention_forward(args, 0, 0, stream);
}

int cta_window_attention_forward(const cta_attention_args* args, int64_t window, int64_t sinks, void* stream) {
  AttnArgs a;
  const int rc = prompt_window(args, window, sinks, a);
  if (rc != CTA_OK) return rc == kNothing ? CTA_OK : rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (!launch_attn_tc_fwd(a, args->dtype, st, &e)) e = launch_attn_simt_fwd(a, args->dtype, st);
  return launched(e, "attention forward launch");
}

int cta_attention_backward(const cta_attention_args* args, void* stream) {
  return cta_window_attention_backward(args, 0, 0, nullptr, 0, stream);
}

// for either kernel
static int64_t backward_bytes(const AttnArgs& a, int dtype) {
  return a.dk != nullptr ? std::max(far_bytes(a, dtype), simt_far_bytes(a)) : 0;
}

// The tensor cores need weights and score gradients in 16 bits, which leaves dQ and dK 1.45 times as far off as the rounding
// of their own, and 1.5 to 1.8 times where a row sees up to 8 keys, since there are few terms to average over; the FP32
// pipe 1.05 to 1.2 (1.4 for two keys).  That is a trade of time for it, for calls that a training step does not notice: a CTA
// walks the heads of its group and two row tiles, or with first keys up to four, so within these limits the backward takes
// 19 to 105 us against 11 to 28, and a training call in PyTorch takes 130 to make; a captured graph pays the difference.
// 32/8 heads of 128, past them: 256 tokens, window 4, 208 and 23 us, with 4 first keys 369 and 27; 2048 tokens of 8 heads of 64,
// with first keys, 104 and 29.  A window that reaches over a short sequence counts as one.
static bool few_keys(const AttnArgs& a, int64_t window) {
  const int64_t tokens = a.cu != nullptr ? a.L : a.L * a.nseq, keys = a.window > 0 ? a.window + a.sinks : a.L;
  const int chain = a.H / a.Hk * (a.d <= 64 ? 64 : 128) * (a.sinks > 0 ? 2 : 1);
  return window > 0 && keys <= 8 && chain <= 256 && tokens * a.H * a.d <= (1 << 19);
}

int64_t cta_window_attention_workspace_bytes(const cta_attention_args* args, int64_t window, int64_t sinks) {
  AttnArgs a;
  const int rc = prompt_window(args, window, sinks, a);
  if (rc != CTA_OK) return rc == kNothing ? 0 : -rc;
  return backward_bytes(a, args->dtype);
}

int cta_window_attention_backward(const cta_attention_args* args, int64_t window, int64_t sinks, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  AttnArgs a;
  const int rc = prompt_window(args, window, sinks, a);
  if (rc != CTA_OK) return rc == kNothing ? CTA_OK : rc;
  if (a.g == nullptr || a.lse == nullptr || a.delta == nullptr)
    return fail(CTA_EINVAL, "the backward needs grad_out, lse and the delta scratch");
  if ((a.dk == nullptr) != (a.dv == nullptr)) return fail(CTA_EINVAL, "dk and dv come together");
  if (args->delta_planes < 0) return fail(CTA_EINVAL, "delta_planes must not be negative");
  if (args->dtype == CTA_F16 && args->delta_planes >= 3 && a.d <= 128) {
    const int64_t plane = (a.cu != nullptr ? 1 : a.nseq) * static_cast<int64_t>(a.H) * a.L;
    a.g_norm = a.delta + plane;
    a.v_norm = a.g_norm + plane;
  }
  const int64_t need = backward_bytes(a, args->dtype);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(CTA_EINVAL, "workspace of %lld bytes needed, got %lld", (long long)need, (long long)workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(CTA_EINVAL, "the workspace must start on 16 bytes");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_attn_delta(a, args->dtype, st);
  if (e == cudaSuccess && (few_keys(a, window) || !launch_attn_tc_bwd(a, args->dtype, workspace, st, &e)))
    e = launch_attn_simt_bwd(a, args->dtype, workspace, st);
  return launched(e, "attention backward launch");
}

int cta_kv_cache_write(const cta_kv_cache_args* args, void* stream) {
  CacheArgs a;
  const int rc = cache_args(args, true, a);
  if (rc != CTA_OK) return rc == kNothing ? CTA_OK : rc;
  return launched(launch_cache_write(a, args->dtype, static_cast<cudaStream_t>(stream)), "cache write launch");
}

int cta_kv_cache_read(const cta_kv_cache_args* args, void* stream) {
  CacheArgs a;
  const int rc = cache_args(args, false, a);
  if (rc != CTA_OK) return rc == kNothing ? CTA_OK : rc;
  return launched(launch_cache_read(a, args->dtype, static_cast<cudaStream_t>(stream)), "cache read launch");
}

int cta_rotary_cache_write(const cta_kv_cache_args* args, const cta_rotary_args* rotary, void* stream) {
  RotaryArgs r;
  std::memset(&r, 0, sizeof(r));
  const int rc = cache_args(args, true, r.cache);
  if (rc != CTA_OK && rc != kNothing) return rc;
  const cta_rotary_args* p = rotary;
  if (p == nullptr) return fail(CTA_EINVAL, "null arguments");
  if (p->heads < 1 || p->heads >= (1LL << 20)) return fail(CTA_EINVAL, "heads must be in 1..2^20 - 1");
  if (p->rotary_dim < 16 || p->rotary_dim % 16 != 0 || p->rotary_dim > args->dim)
    return fail(CTA_EINVAL, "rotary_dim must be a multiple of 16 in 16..%lld, got %lld", (long long)args->dim,
                (long long)p->rotary_dim);
  if (p->table_dtype != CTA_F32 && p->table_dtype != args->dtype)
    return fail(CTA_EINVAL, "the table is fp32 or of the rows' type, got dtype code %d", p->table_dtype);
  if (p->positions_end < 0) return fail(CTA_EINVAL, "bad table shape");
  const int64_t blocks = (p->heads + 3) / 4 + 2 * ((args->kv_heads + 3) / 4);
  if (args->tokens * blocks >= (1LL << 27))
    return fail(CTA_EUNSUPPORTED, "tokens * ceil(heads / 4), of q, k and v, must be below 2^27");
  if (rc == kNothing) return CTA_OK;
  if (p->q == nullptr || p->q_out == nullptr || p->positions == nullptr || (p->table == nullptr && p->positions_end > 0))
    return fail(CTA_EINVAL, "null tensor pointer");
  for (int64_t s : {p->q_stride[0], p->q_stride[1], p->q_out_stride[0], p->q_out_stride[1]})
    if (s % 8 != 0) return fail(CTA_EINVAL, "rows must start on 16 bytes");
  if (p->table_stride % (p->table_dtype == CTA_F32 ? 4 : 8) != 0) return fail(CTA_EINVAL, "the table's rows must start on 16 bytes");
  for (const void* x : {p->q, static_cast<const void*>(p->q_out), p->table})
    if (reinterpret_cast<uintptr_t>(x) % 16 != 0) return fail(CTA_EINVAL, "tensors must start on 16 bytes");
  r.q = p->q;
  r.q_out = p->q_out;
  r.q_sT = p->q_stride[0];
  r.q_sH = p->q_stride[1];
  r.o_sT = p->q_out_stride[0];
  r.o_sH = p->q_out_stride[1];
  r.positions = p->positions;
  r.table = p->table;
  r.table_sP = p->table_stride;
  r.positions_end = p->positions_end;
  r.H = static_cast<int>(p->heads);
  r.pairs = static_cast<int>(p->rotary_dim / 2);
  r.interleaved = p->interleaved != 0;
  return launched(launch_rotary_write(r, args->dtype, p->table_dtype != CTA_F32, static_cast<cudaStream_t>(stream)),
                  "rotary cache write launch");
}

int64_t cta_paged_attention_workspace_bytes(const cta_paged_attention_args* args) {
  return cta_window_paged_attention_workspace_bytes(args, 0, 0);
}

int cta_paged_attention(const cta_paged_attention_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
  return cta_window_paged_attention(args, 0, 0, workspace, workspace_bytes, stream);
}

int64_t cta_window_paged_attention_workspace_bytes(const cta_paged_attention_args* args, int64_t window, int64_t sinks) {
  PagedArgs a;
  const int rc = paged_window(args, window, sinks, a);
  if (rc != CTA_OK) return -rc;
  if (a.T == 0 || a.B == 0) return 0;
  if (tensor_cores_pay(a)) {
    if (!args->quantized) return 0;
    const int64_t bytes = chunk_bytes(a);
    if (bytes > 0) return bytes;
  }
  return split_bytes(paged_split_workers(a, args->dtype, args->quantized), a.d);
}

int cta_window_paged_attention(const cta_paged_attention_args* args, int64_t window, int64_t sinks, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  PagedArgs a;
  const int rc = paged_window(args, window, sinks, a);
  if (rc != CTA_OK) return rc;
  if (a.T == 0 || a.B == 0) return CTA_OK;
  const int64_t need = cta_window_paged_attention_workspace_bytes(args, window, sinks);
  const int prc = paged_pointers(a, args->quantized, workspace, workspace_bytes, need);
  if (prc != CTA_OK) return prc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (tensor_cores_pay(a)) {
    const int64_t bytes = chunk_bytes(a);
    if (!args->quantized) {
      if (launch_paged_tc(a, args->dtype, st, &e)) return launched(e, "paged attention launch");
      return fail(CTA_EUNSUPPORTED, "paged attention of chunks: the tensors cannot be addressed by TMA");
    }
    if (bytes > 0) {
      PagedArgs x = a;
      e = expand_pages(a, args->dtype, static_cast<char*>(workspace), x, st);
      if (e != cudaSuccess) return launched(e, "paged attention launch");
      if (launch_paged_tc(x, args->dtype, st, &e)) return launched(e, "paged attention launch");
      return fail(CTA_EUNSUPPORTED, "paged attention of chunks: the tensors cannot be addressed by TMA");
    }
  }
  a.workers = paged_split_workers(a, args->dtype, args->quantized);
  a.part_ml = static_cast<float*>(workspace);
  a.part_o = a.part_ml + 2LL * a.workers * 16 * 4;
  return launched(launch_paged_split(a, args->dtype, args->quantized, st), "paged attention launch");
}

int64_t cta_prefix_paged_attention_workspace_bytes(const cta_paged_attention_args* args, int64_t shared_prefix) {
  if (shared_prefix < 0) return -fail(CTA_EINVAL, "shared_prefix must not be negative");
  PagedArgs a;
  const int rc = paged_window(args, 0, 0, a);
  if (rc != CTA_OK) return -rc;
  const PrefixPlan p = prefix_plan(a, args->dtype, args->quantized, shared_prefix);
  return p.keys > 0 ? p.bytes : cta_window_paged_attention_workspace_bytes(args, 0, 0);
}

int cta_prefix_paged_attention(const cta_paged_attention_args* args, int64_t shared_prefix, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  if (shared_prefix < 0) return fail(CTA_EINVAL, "shared_prefix must not be negative");
  PagedArgs a;
  const int rc = paged_window(args, 0, 0, a);
  if (rc != CTA_OK) return rc;
  const PrefixPlan p = prefix_plan(a, args->dtype, args->quantized, shared_prefix);
  if (p.keys == 0) return cta_window_paged_attention(args, 0, 0, workspace, workspace_bytes, stream);
  if (a.T == 0 || a.B == 0) return CTA_OK;
  const int prc = paged_pointers(a, args->quantized, workspace, workspace_bytes, p.bytes);
  if (prc != CTA_OK) return prc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const int64_t pairs = (p.splits + 1LL) * a.T * a.H;
  a.skip = p.keys;
  a.prefix_splits = p.splits;
  a.prefix_chunk = p.chunk;
  a.prefix_o = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(ws) + 31) & ~static_cast<uintptr_t>(31));
  a.prefix_ml = a.prefix_o + pairs * (a.d <= 64 ? 64 : 128);
  cudaError_t e = cudaSuccess;
  PagedArgs x = a;
  x.k_scale = x.v_scale = nullptr;
  if (args->quantized) {
    // the first row's pages, all of them
    PagedArgs one = a;
    one.B = 1;
    one.table_width = p.keys / a.page;
    one.seq_lens = nullptr;
    one.skip = 0;
    e = expand_pages(one, args->dtype, ws + p.sums, x, st);
    if (e != cudaSuccess) return launched(e, "paged attention launch");
  }
  if (!launch_prefix_tc(x, args->dtype, st, &e))
    return fail(CTA_EUNSUPPORTED, "paged attention behind a shared prefix: the tensors cannot be addressed by TMA");
  if (e != cudaSuccess) return launched(e, "paged attention launch");
  a.workers = paged_split_workers(a, args->dtype, args->quantized);
  a.part_ml = reinterpret_cast<float*>(ws + p.sums + p.expanded);
  a.part_o = a.part_ml + 2LL * a.workers * 16 * 4;
  return launched(launch_paged_split(a, args->dtype, args->quantized, st), "paged attention launch");
}

}  // extern "C"
