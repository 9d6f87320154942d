// tcgen05 building blocks of the attention kernels: tensor memory, matrix
// descriptors, 4-D TMA boxes, bounded barrier waits.
#pragma once

#include "attn_common.cuh"

namespace cta {
namespace tc {

__device__ __forceinline__ void alloc(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void dealloc(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Waits for this thread's tensor-memory loads.  The registers they fill pass
// through an empty statement behind the wait, so that no use of them can be
// scheduled before it: to the compiler a load's result is there at once.
__device__ __forceinline__ void arrived(uint32_t (&r)[16]) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
               "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void arrived(uint32_t (&r)[32]) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
               "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
               "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
               "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]));
  asm volatile("" : "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
template <typename... R>
__device__ __forceinline__ void wait_ld(R&... r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  (arrived(r), ...);
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// the barrier completes one arrival when all MMAs issued so far by this thread are done
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

// 32 columns of this warp's 32 tensor-memory lanes, one lane per thread
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Shared-memory operand with the 128-byte swizzle: rows of 128 bytes (64 16-bit
// elements), groups of 8 rows 1024 bytes apart.
//   K-major (the contraction index runs along the 128 bytes): the 1024 is the
//     stride offset, the leading offset is unused;
//   MN-major (the contraction index counts rows): the 1024 separates groups of 8
//     rows along the contraction, the leading offset separates the 64-element
//     blocks of the other index.
// The address and the leading offset make up the low word, the rest is constant:
// a product's descriptors differ by additions to the low word (address / 16).
// Built from 64-bit values instead, each MMA took about 80 cycles to issue.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lead_bytes) {
  return ((addr & 0x3ffffu) >> 4) | ((lead_bytes >> 4) << 16);
}

// kind::f16 instruction descriptor: fp32 accumulator, A and B of type T, M = 128
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool b_mn_major, bool a_mn_major = false) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (static_cast<uint32_t>(a_mn_major) << 15) |
         (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}

// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(static_cast<uint32_t>(accumulate)), "n"(kDescHigh)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(static_cast<uint32_t>(accumulate)), "n"(kDescHigh)
      : "memory");
}

// C[128 x N] = A[128 x DP] B[N x DP]^T, both K-major in shared memory; the
// 64-column halves of A and B lie HALF bytes apart.  One thread.
template <int DP, int HALF = 16384>
__device__ __forceinline__ void product_nt(uint32_t d, uint32_t a, uint32_t b, uint32_t id) {
  const uint32_t al = desc_low(a, 16), bl = desc_low(b, 16);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const uint32_t off = ((k >> 2) * HALF + (k & 3) * 32) >> 4;
    mma_ss(d, al + off, bl + off, id, k > 0);
  }
}
// C[128 x N] (+)= A[tmem, 128 x 128] B[128 x N], B MN-major (rows are the
// contraction index), its 64-column blocks 16 KB apart.  A lies where the warps
// that made it left it: GROUP indices at a time at the start of the GROUP columns
// their fp32 sources took.  One thread.
template <int GROUP>
__device__ __forceinline__ void product_tn(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool accumulate) {
  const uint32_t bl = desc_low(b, 16384);
  constexpr int kPer = GROUP / 16;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    mma_ts(d, a + GROUP * (k / kPer) + 8 * (k % kPer), bl + k * (2048 >> 4), id, accumulate || k > 0);
}

// zero the 128-byte rows of a 128-row tile (HALVES blocks of 64 columns, 16 KB
// apart) whose bit in w is clear, before an MMA reads them: what lies there may
// be NaN, and a zero weight times NaN is NaN.  Whole warp.
template <int HALVES>
__device__ __forceinline__ void clear_rows(uint32_t tile, const uint32_t (&w)[4]) {
  const int lane = threadIdx.x & 31;
  for (int r = lane >> 3; r < 128; r += 4)
    if (!((w[r >> 5] >> (r & 31)) & 1u))
#pragma unroll
      for (int c = 0; c < HALVES; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + c * 16384 + r * 128 + (lane & 7) * 16), "r"(0u)
                     : "memory");
  fence_proxy_async_smem();
  __syncwarp();
}
__device__ __forceinline__ bool all_set(const uint32_t (&w)[4]) { return (w[0] & w[1] & w[2] & w[3]) == 0xffffffffu; }
// bit c of word i: c + 32 i < count
__device__ __forceinline__ void first_bits(int count, uint32_t (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = count - 32 * i;
    w[i] = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
  }
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// Bounded wait on an mbarrier phase, false after about a second.  The timer is
// read only when some tries have failed: reading it costs a few hundred cycles,
// which a wait that is on the critical path would pay after every failed try.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 256; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_bounded(bar, parity);
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Asks for the index of a CTA of this grid that has not started yet, which then
// never starts: a running CTA goes on with its work instead of leaving the SM.
// 16 bytes arrive at `resp` on the barrier.
__device__ __forceinline__ void steal(void* resp, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_addr(resp)),
               "r"(smem_addr(bar))
               : "memory");
}
// the index, or -1 when every CTA has started
__device__ __forceinline__ int stolen(const void* resp) {
  uint32_t ok, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\tld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(ok), "=r"(x)
      : "r"(smem_addr(resp))
      : "memory");
  fence_proxy_async_smem();  // the next answer overwrites it
  return ok ? static_cast<int>(x) : -1;
}

// named barrier of `threads` threads, and the same with an OR of their votes
__device__ __forceinline__ void sync_of(int id, int threads) {
  asm volatile("barrier.cta.sync.aligned %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool any_of(int id, int threads, bool vote) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred.aligned q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(vote))
      : "memory");
  return r != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const typename Elem<T>::Pair p = Elem<T>::pack(make_float2(lo, hi));
  return *reinterpret_cast<const uint32_t*>(&p);
}

// Writes N columns, from `col` on, of the rows that a warp's lanes have in tensor
// memory (one row per lane), times `scale`; `any` false: zeros.  `wide` is the
// alignment of the output's rows in bytes, 32 or 16, or 0 for neither.  LOW
// writes what rounding loses instead (see lost()).
//
// With one row per lane a store touches 32 rows, and the SM takes the rows one
// after another.  So up to four lanes exchange their 32-byte pieces first, and a
// store writes 64 or 128 bytes each of 16 or 8 rows: prompts of 1024 tokens, 32/8
// heads of 128, causal, take 281 us instead of 328 with 16 bytes per lane and 302 with 32.
template <typename T, int N, bool LOW = false>
__device__ __forceinline__ void store_rows(uint32_t taddr, T* out, int col, int d, float scale, bool live, int wide,
                                           bool any) {
  constexpr int NC = N / 16;  // pieces of a lane
  static_assert(NC == 1 || NC == 2 || NC == 4, "");
  const int lane = threadIdx.x & 31;
  uint32_t v[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t o[16];
    if (any) {
      ld16(taddr + 16 * c, o);
      wait_ld(o);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = 0u;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
      const float x = __uint_as_float(o[2 * e]) * scale, y = __uint_as_float(o[2 * e + 1]) * scale;
      v[c][e] = LOW ? pack2<T>(lost<T>(x), lost<T>(y)) : pack2<T>(x, y);
    }
  }
  if (wide == 0) {
    if (!live) return;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const T* x = reinterpret_cast<const T*>(&v[c][e]);
        const int at = col + 16 * c + 2 * e;
        if (at < d) out[at] = x[0];
        if (at + 1 < d) out[at + 1] = x[1];
      }
    return;
  }
  // piece c of lane l goes to lane c of l's group, as its piece l
#pragma unroll
  for (int step = 1; step < NC; step *= 2)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c & step) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool high = lane & step;
        const uint32_t got = __shfl_xor_sync(0xffffffffu, high ? v[c][e] : v[c | step][e], step);
        if (high) v[c][e] = got;
        else v[c | step][e] = got;
      }
    }
  const unsigned long long mine = live ? reinterpret_cast<unsigned long long>(out) : 0ull;
  const int at = col + 16 * (lane & (NC - 1));
#pragma unroll
  for (int r = 0; r < NC; ++r) {
    const unsigned long long row = __shfl_sync(0xffffffffu, mine, (lane & ~(NC - 1)) + r);
    if (row == 0 || at >= d) continue;
    T* to = reinterpret_cast<T*>(row) + at;
    if (wide == 32 && at + 8 < d) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[r][0]), "r"(v[r][1]),
                   "r"(v[r][2]), "r"(v[r][3]), "r"(v[r][4]), "r"(v[r][5]), "r"(v[r][6]), "r"(v[r][7])
                   : "memory");
    } else {
      *reinterpret_cast<uint4*>(to) = make_uint4(v[r][0], v[r][1], v[r][2], v[r][3]);
      if (at + 8 < d) *reinterpret_cast<uint4*>(to + 8) = make_uint4(v[r][4], v[r][5], v[r][6], v[r][7]);
    }
  }
}

}  // namespace tc

// Host: the alignment in bytes of a 16-bit tensor's rows that store_rows can use.
inline int row_alignment(const void* p, const AttnStrides& s, int64_t nb, int64_t heads) {
  auto on = [&](int64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && s.t * 2 % bytes == 0 &&
           (heads == 1 || s.h * 2 % bytes == 0) && (nb == 1 || s.b * 2 % bytes == 0);
  };
  return p == nullptr ? 0 : on(32) ? 32 : on(16) ? 16 : 0;
}

// Host: a 4-D map over a [batch, token, head, dim] tensor of 16-bit elements with
// a box of 64 x box_heads x box_tokens x 1.  False when TMA cannot address it.
bool attn_map(CUtensorMap* m, const void* base, int dtype, int64_t nb, int64_t tokens, int64_t heads, int64_t d,
              const AttnStrides& s, int box_heads, int box_tokens);

}  // namespace cta
