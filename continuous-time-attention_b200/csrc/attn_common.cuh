// Device helpers shared by the attention kernels: which sequence a tile belongs
// to, the key mask, base-2 exponentials.
#pragma once

#include <atomic>

#include "attn.h"
#include "common.cuh"

namespace cta {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// device-side error code: a page, slot or length outside the cache
enum : int { kDevBadIndex = 2 };

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// A tile of one sequence: rows [row0, row0 + n) of the batch entry / packed row
// `batch`, the tile's first row at `first` within the sequence.  n == 0: the
// tile lies behind the last sequence; then tail_index of tail_count such tiles,
// and row0 is the first row behind the last sequence.
struct SeqTile {
  int seq;
  int batch;
  int64_t row0;
  int n;      // length of the sequence
  int first;  // first row of the tile within it
  int tail_index, tail_count;
};

__device__ __forceinline__ void clamp_range(const int32_t* cu, int i, int64_t total, int64_t& begin, int& n) {
  const int64_t b = min(max(static_cast<int64_t>(__ldg(cu + i)), static_cast<int64_t>(0)), total);
  const int64_t e = min(max(static_cast<int64_t>(__ldg(cu + i + 1)), b), total);
  begin = b;
  n = static_cast<int>(e - b);
}

// The tile-th tile of `rows` rows.  Called by one whole warp; every lane gets
// the result.  Packed: the lanes walk the offsets 32 sequences at a time with a
// prefix sum of the tile counts, so that the host never reads the offsets.
// Tiles of a sequence are numbered from its end when `backwards` (the last
// tiles of a causal sequence have the most keys and start first).  Otherwise
// one sequence follows the other, unless `across`: not packed, the same tile of all
// sequences comes before the next; packed, up to 32 sequences come by descending
// `weight` (their rows if that is null), so that the longest pieces of work do not
// come last.
__device__ __forceinline__ SeqTile find_tile(const int32_t* cu, int nseq, int64_t L, int tiles, int tile, int rows,
                                             bool backwards, bool across, const int32_t* weight = nullptr) {
  SeqTile t;
  t.tail_index = t.tail_count = 0;
  if (cu == nullptr) {
    const int i = across ? tile / nseq : tile % tiles;
    t.seq = t.batch = across ? tile % nseq : tile / tiles;
    t.row0 = 0;
    t.n = static_cast<int>(L);
    t.first = (backwards ? tiles - 1 - i : i) * rows;
    return t;
  }
  const int lane = threadIdx.x & 31;
  t.batch = 0;
  int before = 0;
  int64_t end = 0;
  const bool ranked = across && nseq > 1 && nseq <= 32;
  for (int s0 = 0; s0 < nseq; s0 += 32) {
    int64_t begin = 0;
    int n = 0;
    if (s0 + lane < nseq) clamp_range(cu, s0 + lane, L, begin, n);
    const int count = (n + rows - 1) / rows;
    int upto = count, total;
    if (ranked) {
      const int w = lane < nseq && weight != nullptr ? __ldg(weight + lane) : n;
      total = __reduce_add_sync(0xffffffffu, count);
      for (int i = 0; i < nseq; ++i) {
        const int wi = __shfl_sync(0xffffffffu, w, i), ci = __shfl_sync(0xffffffffu, count, i);
        if (wi > w || (wi == w && i < lane)) upto += ci;
      }
    } else {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      total = __shfl_sync(0xffffffffu, upto, 31);
    }
    if (tile < before + total) {
      const unsigned hit = __ballot_sync(0xffffffffu, tile < before + upto && tile >= before + upto - count);
      const int src = __ffs(hit) - 1;
      t.seq = s0 + src;
      t.row0 = __shfl_sync(0xffffffffu, begin, src);
      t.n = __shfl_sync(0xffffffffu, n, src);
      const int c = __shfl_sync(0xffffffffu, count, src);
      const int i = tile - before - (__shfl_sync(0xffffffffu, upto, src) - c);
      t.first = (backwards ? c - 1 - i : i) * rows;
      return t;
    }
    before += total;
    int64_t e = begin + n;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) e = max(e, __shfl_xor_sync(0xffffffffu, e, o));
    end = max(end, e);
  }
  t.seq = nseq;
  t.row0 = end;
  t.n = 0;
  t.first = 0;
  t.tail_index = tile - before;
  t.tail_count = tiles - before;
  return t;
}

// Upper bound on the tiles of a packed row plus one tile that is always behind
// the last sequence (it clears the rows there when asked to).
inline int64_t packed_tiles(int64_t L, int nseq, int rows) { return L / rows + nseq + 1; }

// Dynamic shared memory above 48 KB has to be allowed, once per kernel and device.
template <auto Kernel>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit != 0 && (done.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// A kernel without shared memory that starts beside one that fills it would find that one's division of each SM, with
// next to no L1, and keep it to its end; asked for, its own comes with the SMs that are idle.  Once per kernel and device.
template <auto Kernel>
cudaError_t prefer_l1() {
  static std::atomic<uint64_t> done{0};  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit != 0 && (done.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxL1);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

inline int num_sms_here() {
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) return 148;
  return v;
}

// Launches a kernel.  `beside`: its CTAs may start as soon as all of the kernel in
// front of it in the stream have started (that one calls pdl_launch_dependents,
// and this one reads nothing of it), so that they fill the SMs that its last CTAs
// leave idle; every CTA calls pdl_wait before it ends, so that the stream goes on
// only when both are done.  (One that does so is enough: where many end early, all
// of them would hold their SMs until the kernel in front is done.)
template <auto Kernel, typename... Args>
cudaError_t launch_grid(bool beside, int64_t ctas, int threads, int smem, cudaStream_t st, const Args&... args) {
  const cudaError_t e = allow_smem<Kernel>(smem);
  if (e != cudaSuccess) return e;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = beside ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, Kernel, args...);
}

// The backward takes delta = sum_d g * o from an o that rounding has moved.  The
// error, up to 2^-9 |g| |o| in bf16, is the same for all keys of a row; it is small
// beside the rounding of the single P (dP - delta) in long rows, but not where few
// keys make o large: over sequences of 1 to 16 tokens the gradients were 2 to 3 times
// as far off as one rounding of them.  So a training forward keeps o's lost part.
// In fp16 it is scaled, or it would be subnormal for |o| < 2^-3.
template <typename T> __host__ __device__ constexpr float low_scale() { return 1.f; }
template <> __host__ __device__ constexpr float low_scale<__half>() { return 2048.f; }
template <typename T>
__device__ __forceinline__ float lost(float x) {
  return (x - Elem<T>::to_f(Elem<T>::from_f(x))) * low_scale<T>();
}

// Sets rows behind the last sequence to zero, head h, `d` elements each.
template <typename T>
__device__ __forceinline__ void zero_rows(void* base, const AttnStrides& s, int64_t begin, int64_t end, int h, int d,
                                          int index, int count) {
  T* p = static_cast<T*>(base) + h * s.h;
  for (int64_t r = begin + index; r < end; r += count)
    for (int c = threadIdx.x; c < d; c += blockDim.x) p[r * s.t + c] = Elem<T>::from_f(0.f);
}

// First and one past the last valid key of a batch entry.
__device__ __forceinline__ void mask_range(const AttnArgs& a, int batch, int n, int& lo, int& hi) {
  lo = 0;
  hi = n;
  if (a.mask != nullptr) {
    const uint32_t* m = a.mask + batch * a.mask_words;
    lo = static_cast<int>(__ldg(m));
    hi = min(n, static_cast<int>(__ldg(m + 1)));
  }
}
__device__ __forceinline__ bool mask_key(const uint32_t* m, int j) {
  return m == nullptr || ((__ldg(m + kMaskHead + (j >> 5)) >> (j & 31)) & 1u);
}

// Sliding window: the causal row at place i sees the keys j <= i that lie in its
// window, j > i - window, or among the first ones, j < sink_end.
struct Reach {
  int window, sink_end;
  __device__ __forceinline__ int first(int i) const { return i - window + 1; }
  __device__ __forceinline__ bool sees(int i, int j) const { return j > i - window || j < sink_end; }
};
// of a batch entry whose first valid key is `lo`: padding on the left does not count
__device__ __forceinline__ Reach reach_of(const AttnArgs& a, int lo) {
  return Reach{a.window, a.sinks > 0 ? lo + a.sinks : 0};
}

// Where the keys of a sequence lie in the 16-bit copy of an e4m3 cache that a chunk under a window reads.  Dense: whole
// tiles of 128 keys, those of the first keys and those from the first row's window on, so that the copy's size follows
// from the window, the first keys and the rows, not from the block table's width.  A sequence has copy_stride slots
// and one for each of its rows: with tiles of 128 on either side of both, its keys fit.  Where that is no less than the
// table, every key has a slot.
struct CopySlots {
  int base, first, gap;  // key j at base + j, those from `first` on `gap` further down
  __device__ __forceinline__ int at(int key) const { return base + key - (key >= first ? gap : 0); }
};
// of a sequence of n keys (within the table), whose rows begin at `begin`
__device__ __forceinline__ CopySlots copy_slots(int stride, bool dense, int window, int sinks, int seq, int64_t begin, int rows, int n) {
  if (!dense) return CopySlots{seq * stride, 0, 0};
  const int first = static_cast<int>(residue_row(sinks)), low = max(n - rows - window + 1, 0);
  return CopySlots{seq * stride + static_cast<int>(begin) / 128 * 128, first, max(first, low / 128 * 128) - first};
}

// A window's far rows, those behind the window of a key tile of `rows` that holds first keys, go in parts of `chunk`; part c
// of a sequence has the place far_place + c of far_places.  Packed: a sequence has far rows only if it is at least window +
// rows long, so its place among those, or among all if they are fewer, tells them apart.
__host__ __device__ __forceinline__ bool far_by_sequence(const AttnArgs& a, int rows) { return a.nseq <= a.L / (a.window + rows); }
__device__ __forceinline__ int64_t far_place(const AttnArgs& a, const SeqTile& t, int rows, int chunk) {
  if (a.cu == nullptr) return static_cast<int64_t>(t.batch) * ((a.L + chunk - 1) / chunk);
  return t.row0 / chunk + (far_by_sequence(a, rows) ? t.seq : t.row0 / (a.window + rows));
}
inline int64_t far_places(const AttnArgs& a, int rows, int64_t chunk) {
  if (a.cu == nullptr) return a.nseq * ((a.L + chunk - 1) / chunk);
  return a.L / chunk + 1 + (far_by_sequence(a, rows) ? a.nseq : a.L / (a.window + rows) + 1);
}

__device__ __forceinline__ int64_t lse_index(const AttnArgs& a, const SeqTile& t, int h, int row) {
  return (static_cast<int64_t>(t.batch) * a.H + h) * a.L + t.row0 + row;
}

}  // namespace cta
