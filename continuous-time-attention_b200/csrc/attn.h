// Launch descriptors of the attention and key/value-cache kernels, shared by
// the C ABI (attn_capi.cu) and the kernel units.  Not part of the public ABI.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace cta {

// Element strides of a [batch, token, head, dim] tensor; the dim axis is contiguous.
struct AttnStrides {
  int64_t b, t, h;
};

// Softmax attention of prompts.  Dense: `nseq` sequences of L tokens each.
// Packed (cu != nullptr): one batch of L rows holding nseq sequences, the i-th
// in rows [cu[i], cu[i+1]).
struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* low;         // 16-bit: what rounding o lost, times low_scale<T>(), rows {L * H * d, H * d, d}; or nullptr
  void* o;           // forward: output.  backward: the forward's output (read)
  float* lse;        // [nseq, H, L] dense, [H, L] packed; natural logarithm, -inf for a row without keys
  const void* g;     // backward: gradient of the output
  float* delta;      // backward scratch, laid out as lse: sum_d g * o
  float* g_norm;     // fp16 on tensor cores, else nullptr: |g| of each row, laid out as lse
  float* v_norm;     // and |v| of each key, [nseq, Hk, L] dense, [Hk, L] packed, 0 for a masked one
  void* dq;
  void* dk;
  void* dv;
  AttnStrides qs, ks, vs, os, gs, dqs, dks, dvs;
  const int32_t* cu;
  const uint32_t* mask;  // key mask words (kMaskHead + ...), nullptr = every key valid
  int64_t mask_words;    // words per batch entry
  int64_t L;
  int nseq;
  int H, Hk, d;
  int causal;
  int zero_tail;  // packed: rows behind the last sequence are set to zero (else left as they are)
  float scale;
  int tiles;  // tiles of the launch per (packed) row or per sequence (dense)
};

// Key mask words of one batch entry: {first valid key, one past the last valid
// key, 0, 0} and then one bit per key, 128-bit aligned per 128 keys.
constexpr int kMaskHead = 4;

// dtype codes as in common.cuh
cudaError_t launch_attn_simt_fwd(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_attn_simt_bwd(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_attn_delta(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_attn_mask_words(const void* mask, int mask_dtype, int64_t sB, int64_t sL, int64_t B, int64_t L,
                                   uint32_t* words, int64_t words_per_batch, cudaStream_t st);

// rows per tile of the plain kernels
constexpr int kSimtRows = 64;

// ---------------------------------------------------------------------------
// paged key/value cache
// ---------------------------------------------------------------------------
struct CacheArgs {
  const void* k_in;  // write: new rows [T, Hk, d]; read: unused
  const void* v_in;
  void* k_out;       // read: destination rows
  void* v_out;
  int64_t k_sT, k_sH, v_sT, v_sH;  // strides of the rows
  void* k_cache;
  void* v_cache;
  int64_t kc_sP, kc_sS, kc_sH, vc_sP, vc_sS, vc_sH;  // page, slot in page, head
  float* k_scale;  // e4m3 caches: [pages, Hk, page] contiguous
  float* v_scale;
  const int64_t* slots;
  int64_t T, n_slots;
  int page, Hk, d;
  int quantized;
};
cudaError_t launch_cache_write(const CacheArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_cache_read(const CacheArgs& a, int dtype, cudaStream_t st);

struct PagedArgs {
  const void* q;  // [T, H, d]
  void* o;
  int64_t q_sT, q_sH, o_sT, o_sH;
  const void* k_cache;
  const void* v_cache;
  int64_t kc_sP, kc_sS, kc_sH, vc_sP, vc_sS, vc_sH;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;  // [B, table_width]
  int64_t table_sB;
  const int32_t* seq_lens;
  const int32_t* cu;  // packed rows of q, nullptr: one row per sequence
  int64_t T;
  int B, H, Hk, d;
  int page, table_width, n_pages;
  int max_rows;  // longest chunk (host)
  float scale;
  // split over the keys: one worker per warp
  int workers;
  float* part_o;   // [2 * workers, 16, dim rounded up to 64 or 128] fp32
  float* part_ml;  // [2 * workers, 16, 4] maximum, sum, maximum of the weighted values
  // tensor-core kernel: k_cache and v_cache hold launch_cache_expand's pages, and these what it left out of their
  // elements [B, Hk, residue_row(table_width * page)]: the fractions of the scales in bf16, the key's scale and the
  // logarithm (base 2) of the value's in fp16; else nullptr
  const float* k_res;
  const float* v_res;
};

// workers (warps) of the split kernel on the current device, and its launch
int paged_split_workers(const PagedArgs& a, int dtype, int quantized);
cudaError_t launch_paged_split(const PagedArgs& a, int dtype, int quantized, cudaStream_t st);

// tensor-core forms; false = not for these types, sizes or strides (nothing was launched)
bool launch_attn_tc_fwd(const AttnArgs& a, int dtype, cudaStream_t st, cudaError_t* e);
bool launch_attn_tc_bwd(const AttnArgs& a, int dtype, cudaStream_t st, cudaError_t* e);
int attn_pack(int group);  // heads of a group that one row tile holds: its largest power of two
bool launch_paged_tc(const PagedArgs& p, int dtype, cudaStream_t st, cudaError_t* e);
// e4m3 caches: the pages that the table names, as 16-bit rows in page order (page i of sequence b is page
// b * table_width + i), for the tensor-core kernel
cudaError_t launch_cache_expand(const PagedArgs& p, int dtype, void* k, void* v, float* k_res, float* v_res,
                                cudaStream_t st);
// entries of k_res and v_res for a sequence and head, in whole key tiles
__host__ __device__ constexpr int64_t residue_row(int64_t slots) { return (slots + 127) / 128 * 128; }

int read_device_error_paged(int clear);
int read_device_error_tc_fwd(int clear);
int read_device_error_tc_bwd(int clear);
int read_device_error_cache(int clear);

}  // namespace cta
