// Attention of the newest rows of each sequence over a paged key/value cache:
// the form for one or a few rows per sequence, where reading the cache once is
// all the work there is.
//
//   O_r = sum_j w_rj V_j / sum_j w_rj,   w_rj = exp(c q_r.k_j),   j <= n - rows + r
//
// What bounds it: HBM, 2 Hk (2 d) bytes per key (e4m3: 2 Hk (d + 4)).  So the
// design keeps loads in flight and does nothing else:
//
// * The products are transposed: K Q^T and V^T P^T, keys (dims) along the 16 of
//   mma.m16n8k16 and the rows of all query heads that share a key/value head
//   along the 8, so that 8 rows fill the instruction.  The lanes load the A
//   fragments straight from the pages, 16 bytes each, without shared memory: a
//   contraction may take its index in any order, so the lane that holds a key
//   takes the eight (e4m3: sixteen) elements that one load brings as its share
//   of two (four) k16 steps, and Q is laid out to match; in V^T P^T the m index
//   is permuted so that a lane ends with the consecutive elements it loaded.
//   The weights change sides by a transposing move.  tcgen05 would need 128 rows
//   where there are 1 to 16.
// * Every warp is a worker.  The 16-key groups of all (sequence, row tile)
//   segments form one list, cut into equal runs, one per worker of a key/value
//   head, whatever the lengths are; the host never reads them.  The workers of
//   all heads walk the list side by side, so that the rows of a token, which lie
//   next to each other, are read at about the same time.  A worker that holds only a part
//   of a segment leaves (maximum, sum, weighted values) in 32 bits, and a second
//   kernel, launched as a programmatic dependent, joins the parts of a segment
//   in worker order.  Nothing is atomic, so results do not depend on timing.
// * The next group's keys load while this group's softmax runs, the next
//   values while the next scores run.
//
// Measured, 32/8 heads of 128, 64 sequences of 512 to 8192 keys: 16-bit 178 us, 6.2
// TB/s, 95 % of what a copy reaches; e4m3 135 us, 4.2 TB/s (a code is converted before
// it is multiplied, and 15 warps an SM do not hide that behind the loads: HBM is busy
// half the time, and instructions issue in 41 % of the cycles).  One sequence of 777 keys: 11 us, the
// latency of two launches and of a chain of loads.
//
// CUT: a segment is two runs of groups, those of the first keys and those that the rows' windows reach, or what lies behind
// a shared prefix, whose sums another kernel leaves for the join.  64 sequences of 512 to 8192 keys in windows of 1024, 4
// first keys, 16 bits: 57 us a call, 53 of them this kernel's, 270 MB at 5.1 TB/s; a worker has 27 groups there, and the
// ramp up and the rest of the workers' ends weigh more than over whole sequences.
// Over e4m3 48 us a call, at three CTAs an SM; with four, as over whole sequences, 72 bytes a thread are spilled and it takes 52.
// Beside the prefix's parts, which fill their SMs' shared memory, it asks for its L1 (prefer_l1): without, 64 sequences of 2048
// to 4096 own keys take 209 us instead of 132.
//
// e4m3: the codes are exact in fp16, so both products run in fp16 whatever the
// type of q.  A bf16 row is first divided by the power of two at its largest
// element, which loses only what is below 2^-24 of that element.  The key's
// scale multiplies the score in 32 bits.  The value's scale joins the weight,
// whose own running maximum keeps weight * scale within fp16 for any scales.
#include <algorithm>

#include "attn_common.cuh"

namespace cta {

__device__ int g_paged_error;

namespace {

constexpr int kThreads = 128;
constexpr int kGroup = 16;      // keys per step of a warp
constexpr int kMinGroups = 2;   // groups a worker gets at least
constexpr int kPartRows = 16;
// the references that weights are relative to move when a weight would pass 2^kLazy
constexpr float kLazy = 8.f;
// fp16 weights carry 2^7, and so stay below 2^15; what is lost to subnormals is below 2^-32 of the reference
constexpr float kHalfShift = 7.f;

template <typename M> struct Mma;
template <> struct Mma<__half> {
  __device__ __forceinline__ static void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ __forceinline__ static uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Mma<__nv_bfloat16> {
  __device__ __forceinline__ static void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ __forceinline__ static uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(v)));
  return h;
}

// rows of a segment: `tile` consecutive (row, head of the group) pairs
struct Seg {
  int b, tile;
  int n, rows;         // keys and rows of the sequence
  int64_t row0;        // its first row in q
  int group, groups;   // first group of this call and groups of the segment
  int64_t start;       // first unit of the segment
};

struct SeqInfo {
  int n, rows, tiles, groups;
  int64_t row0, units;
};

// CUT: a segment takes only some of the sequence's groups: those of the first `sinks` keys, and from the one on that
// holds the first key in the window of the tile's first row (or from `skip` on) as many as its rows' windows can touch.
// A page between the two is not read, nor is its entry in the table.
constexpr int kNoWindow = 1 << 30;
__device__ __forceinline__ int cut_window(const PagedArgs& a) { return a.window > 0 ? a.window : kNoWindow; }
__device__ __forceinline__ int sink_groups(const PagedArgs& a, int n) { return (min(a.sinks, n) + kGroup - 1) / kGroup; }
// groups that the windows of one tile's rows touch at most
__device__ __forceinline__ int window_groups(const PagedArgs& a, int rows, int tile_rows) {
  const int group = a.H / a.Hk;
  const int tokens = min(rows, (tile_rows + group - 2) / group + 1);
  return (cut_window(a) + tokens - 1 + 2 * (kGroup - 1)) / kGroup;
}
// the first group behind those of the first keys, for the tile whose first row is `tok`
__device__ __forceinline__ int first_window_group(const PagedArgs& a, int n, int rows, int tok) {
  const int low = n - rows + tok - cut_window(a) + 1;
  return max(max(low, 0) / kGroup, max(sink_groups(a, n), a.skip / kGroup));
}

template <bool CUT>
__device__ __forceinline__ SeqInfo seq_info(const PagedArgs& a, int b, int tile_rows) {
  SeqInfo s{0, 0, 0, 0, 0, 0};
  if (b >= a.B) return s;
  int n = __ldg(a.seq_lens + b);
  const int64_t most = static_cast<int64_t>(a.table_width) * a.page;
  if (n < 0 || n > most) {
    atomicExch(&g_paged_error, kDevBadIndex);
    n = n < 0 ? 0 : static_cast<int>(most);
  }
  s.n = n;
  if (a.cu != nullptr) {
    clamp_range(a.cu, b, a.T, s.row0, s.rows);
  } else {
    s.row0 = b;
    s.rows = 1;
  }
  s.tiles = (s.rows * (a.H / a.Hk) + tile_rows - 1) / tile_rows;
  s.groups = (n + kGroup - 1) / kGroup;
  if constexpr (CUT) s.groups = min(s.groups - a.skip / kGroup, sink_groups(a, n) + window_groups(a, s.rows, tile_rows));
  s.groups = max(1, s.groups);  // a sequence without keys still writes its zeros
  s.units = static_cast<int64_t>(s.tiles) * s.groups;
  return s;
}

__device__ __forceinline__ int64_t warp_sum(int64_t x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <bool CUT>
__device__ __forceinline__ int64_t total_units(const PagedArgs& a, int tile_rows) {
  int64_t u = 0;
  for (int b = threadIdx.x & 31; b < a.B; b += 32) u += seq_info<CUT>(a, b, tile_rows).units;
  return warp_sum(u);
}

// workers per key/value head, of a.workers / Hk
__device__ __forceinline__ int active_shares(const PagedArgs& a, int64_t units) {
  return static_cast<int>(min(static_cast<int64_t>(a.workers / a.Hk), max(static_cast<int64_t>(1), units / kMinGroups)));
}

// the segment that holds unit u (u < total); whole warp
template <bool CUT>
__device__ __forceinline__ Seg find_segment(const PagedArgs& a, int64_t u, int tile_rows) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int b0 = 0;; b0 += 32) {
    const SeqInfo s = seq_info<CUT>(a, b0 + lane, tile_rows);
    int64_t upto = s.units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
    if (u < before + total || b0 + 32 >= a.B) {
      const unsigned hit = __ballot_sync(0xffffffffu, u < before + upto);
      const int src = max(0, __ffs(hit) - 1);
      Seg g;
      g.b = b0 + src;
      g.n = __shfl_sync(0xffffffffu, s.n, src);
      g.rows = __shfl_sync(0xffffffffu, s.rows, src);
      g.row0 = __shfl_sync(0xffffffffu, s.row0, src);
      g.groups = __shfl_sync(0xffffffffu, s.groups, src);
      const int64_t first = before + __shfl_sync(0xffffffffu, upto - s.units, src);
      const int64_t seg = (u - first) / g.groups;
      g.group = static_cast<int>((u - first) - seg * g.groups);
      g.tile = static_cast<int>(seg);
      g.start = first + seg * g.groups;
      return g;
    }
    before += total;
  }
}

// 8 x 8 of 16-bit values across the warp, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ROWS: 8 or 16 rows per segment
template <typename T, bool FP8, int DP, int ROWS, bool CUT>
__global__ void __launch_bounds__(kThreads, ROWS == 8 ? ((FP8 && !CUT) || DP == 64 ? 4 : 3) : (DP == 64 ? 3 : 2))
    paged_split_kernel(const __grid_constant__ PagedArgs a) {
  using M = typename std::conditional<FP8, __half, T>::type;
  constexpr bool kHalf = std::is_same<M, __half>::value;
  constexpr float kShift = kHalf ? kHalfShift : 0.f;
  constexpr int NR = ROWS / 8;                // n8 tiles of rows
  constexpr int KS = DP / 16;                 // k16 steps of K Q^T
  constexpr int KE = FP8 ? 16 : 8;            // elements of one key load
  constexpr int KL = DP / (4 * KE);           // key loads per lane and key
  constexpr int VE = FP8 && DP == 128 ? 16 : 8;  // elements of one value load
  constexpr int VL = DP / (8 * VE);           // value loads per lane and key
  constexpr int VW = FP8 ? VE / 4 : VE / 2;   // 32-bit words of one value load
  constexpr int MT = DP / 16;                 // m16 tiles of the output

  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, quad = lane & 3, oct = lane >> 2;
  const int worker = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t units = total_units<CUT>(a, ROWS);
  const int shares = active_shares(a, units);
  const int hk = worker % a.Hk, share = worker / a.Hk;
  if (!CUT && (units == 0 || share >= shares)) return;
  int64_t u = units * share / shares;
  const int64_t u_end = share < shares ? units * (share + 1) / shares : u;  // none for the workers left over
  bool first = true;
  const int group = a.H / a.Hk;

  while (u < u_end) {
    const Seg g = find_segment<CUT>(a, u, ROWS);
    const int count = static_cast<int>(min(u_end - u, static_cast<int64_t>(g.groups - g.group)));

    // Q as the B operand: row oct of each n8 tile
    uint32_t qf[KS][NR][2];
    float c2[NR][2];
    int last[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int i = g.tile * ROWS + oct + 8 * r;
      const int tok = i / group;
      const bool live = tok < g.rows;
      const T* q = static_cast<const T*>(a.q) + (g.row0 + tok) * a.q_sT + (hk * group + i - tok * group) * a.q_sH;
      float top = 0.f, mul = a.scale * kLog2e;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int c = FP8 ? 64 * (k / 4) + 16 * quad + 4 * (k % 4) : 32 * (k / 2) + 8 * quad + 4 * (k % 2);
        uint2 w = make_uint2(0u, 0u);
        if (live && c < a.d) w = __ldg(reinterpret_cast<const uint2*>(q + c));
        qf[k][r][0] = w.x;
        qf[k][r][1] = w.y;
        if constexpr (FP8 && !std::is_same<T, __half>::value) {
          const float2 x = Elem<T>::unpack(*reinterpret_cast<const typename Elem<T>::Pair*>(&w.x));
          const float2 y = Elem<T>::unpack(*reinterpret_cast<const typename Elem<T>::Pair*>(&w.y));
          top = fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))), top);
        }
      }
      if constexpr (FP8 && !std::is_same<T, __half>::value) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the power of two at the row's largest element, kept where it and its reciprocal are normal
        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 2), 252);
        const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
        mul *= __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            const float2 x = Elem<T>::unpack(*reinterpret_cast<const typename Elem<T>::Pair*>(&qf[k][r][i2]));
            qf[k][r][i2] = Mma<__half>::pack(x.x * down, x.y * down);
          }
      }
      const int see = live ? g.n - g.rows + tok : -1;
      // scores and weights hold rows 2 quad, 2 quad + 1
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        c2[r][e] = __shfl_sync(0xffffffffu, mul, 4 * (2 * quad + e));
        last[r][e] = __shfl_sync(0xffffffffu, see, 4 * (2 * quad + e));
      }
    }

    // Last key that every row of the tile sees, -1 if one of them sees none.  Rows behind the sequence's last do not
    // count: theirs are not written.
    int least = 0x7fffffff, most = -1;
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool counts = (g.tile * ROWS + 2 * quad + e + 8 * r) / group < g.rows;
        if (counts) least = min(least, max(last[r][e], -1));
        if (CUT && counts) most = max(most, last[r][e]);
      }
    least = __reduce_min_sync(0xffffffffu, least);
    // CUT: the first key that every row's window holds, and the groups as they are numbered here
    const int window = CUT ? cut_window(a) : 0, sinks = CUT ? sink_groups(a, g.n) : 0;
    if constexpr (CUT) most = __reduce_max_sync(0xffffffffu, most) - window + 1;
    const int from = CUT ? first_window_group(a, g.n, g.rows, g.tile * ROWS / group) : 0;
    auto group_at = [&](int i) { return CUT ? (i < sinks ? i : from + i - sinks) : i; };
    float o[MT][NR][4];
    float m[NR][2], l[NR][2], mv[NR][2];  // reference of the weights, their sum, reference of the weighted values
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < NR; ++r) o[t][r][0] = o[t][r][1] = o[t][r][2] = o[t][r][3] = 0.f;
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) m[r][e] = mv[r][e] = neg_inf(), l[r][e] = 0.f;

    const int32_t* table = a.table + g.b * a.table_sB;
    const int per_page = a.page / kGroup;
    auto page_at = [&](int index) -> int {
      // the index-th page of the sequence, -1 if the table's entry lies outside the cache
      if (index * a.page >= g.n) return -1;
      const int p = __ldg(table + index);
      if (p < 0 || p >= a.n_pages) {
        if (lane == 0) atomicExch(&g_paged_error, kDevBadIndex);
        return -1;
      }
      return p;
    };
    using C = typename std::conditional<FP8, uint8_t, T>::type;
    const C* k_base = static_cast<const C*>(a.k_cache) + hk * a.kc_sH + KE * quad;
    const C* v_base = static_cast<const C*>(a.v_cache) + hk * a.vc_sH + VE * oct;
    uint4 kf[2][KL];
    float ks[2], vs[2];
    uint32_t vf[4][VL][VW];
    // A group that lies in the cache and the sequence whole, of full rows, loads without conditions
    const bool full_rows = a.d == DP;
    auto load_keys = [&](int grp, int p, int slot) {
      const C* at = k_base + p * a.kc_sP + (slot + oct) * a.kc_sS;
      const int64_t x = FP8 ? (static_cast<int64_t>(p) * a.Hk + hk) * a.page + slot + oct : 0;
      if (full_rows && p >= 0 && (grp + 1) * kGroup <= g.n) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int i = 0; i < KL; ++i) kf[t][i] = __ldg(reinterpret_cast<const uint4*>(at + 4 * KE * i));
          if constexpr (FP8) {
            ks[t] = __ldg(a.k_scale + x + 8 * t);
            vs[t] = __ldg(a.v_scale + x + 8 * t);
          }
          at += 8 * a.kc_sS;
        }
        return;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool ok = p >= 0 && grp * kGroup + 8 * t + oct < g.n;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          kf[t][i] = make_uint4(0u, 0u, 0u, 0u);
          if (ok && 4 * KE * i + KE * quad < a.d)
            kf[t][i] = __ldg(reinterpret_cast<const uint4*>(at + 8 * t * a.kc_sS + 4 * KE * i));
        }
        if constexpr (FP8) {
          ks[t] = ok ? __ldg(a.k_scale + x + 8 * t) : 1.f;
          vs[t] = ok ? __ldg(a.v_scale + x + 8 * t) : 1.f;
        }
      }
    };
    auto load_row = [&](uint32_t (&w)[VW], const C* q) {
      if constexpr (VW == 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(q));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(q));
        w[0] = v.x, w[1] = v.y;
      }
    };
    auto load_values = [&](int grp, int p, int slot) {
      const C* at = v_base + p * a.vc_sP + (slot + 2 * quad) * a.vc_sS;
      if (full_rows && p >= 0 && (grp + 1) * kGroup <= g.n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int x = 0; x < VL; ++x) load_row(vf[i][x], at + 8 * VE * x);
          at += (i == 1 ? 7 : 1) * a.vc_sS;  // keys 2 quad + {0, 1, 8, 9}
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = (i & 1) + 8 * (i >> 1);
        const bool ok = p >= 0 && grp * kGroup + 2 * quad + k < g.n;
#pragma unroll
        for (int x = 0; x < VL; ++x) {
#pragma unroll
          for (int w = 0; w < VW; ++w) vf[i][x][w] = 0u;
          if (ok && 8 * VE * x + VE * oct < a.d) load_row(vf[i][x], at + k * a.vc_sS + 8 * VE * x);
        }
      }
    };

    // the group's page and its first slot there, now and one group on; the page after that is on its way
    int index = group_at(g.group) / per_page;
    int slot = (group_at(g.group) - index * per_page) * kGroup;
    // CUT: the page after this one, if the groups that follow reach it
    auto page_after = [&](int i) -> int {
      if (CUT && (index + 1) * per_page > (i < sinks ? sinks - 1 : from + g.groups - 1 - sinks)) return -1;
      return page_at(index + 1);
    };
    int page = page_at(index), page_on = page_after(g.group);
    load_keys(group_at(g.group), page, slot);
    load_values(group_at(g.group), page, slot);
    for (int it = 0; it < count; ++it) {
      const int grp = group_at(g.group + it), grp_next = group_at(g.group + it + 1);
      const bool here = page >= 0;
      // where the next group lies
      int slot_next = slot + kGroup, page_next = page;
      if (CUT && g.group + it + 1 == sinks) {
        if (it + 1 < count) {
          index = from / per_page;
          slot_next = (from - index * per_page) * kGroup;
          page_next = page_at(index);
          page_on = page_after(sinks);
        }
      } else if (slot_next == a.page) {
        slot_next = 0;
        page_next = page_on;
        ++index;
        if (it + 1 < count) page_on = page_after(g.group + it + 1);
      }
      // scores: 16 keys x ROWS
      float s[NR][4];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t ka[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if constexpr (FP8) {
            const uint4 w = kf[t][k / 4];
            const uint32_t x = k % 4 == 0 ? w.x : k % 4 == 1 ? w.y : k % 4 == 2 ? w.z : w.w;
            ka[t] = e4m3x2_to_half2(x);
            ka[2 + t] = e4m3x2_to_half2(x >> 16);
          } else {
            const uint4 w = kf[t][k / 2];
            ka[t] = k % 2 == 0 ? w.x : w.z;
            ka[2 + t] = k % 2 == 0 ? w.y : w.w;
          }
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) Mma<M>::run(s[r], ka, qf[k][r][0], qf[k][r][1]);
      }
      float ksc[2], vl2[2];
      if constexpr (FP8) {
#pragma unroll
        for (int t = 0; t < 2; ++t) ksc[t] = ks[t], vl2[t] = __log2f(vs[t]);
      }
      if (it + 1 < count) load_keys(grp_next, page_next, slot_next);

      const bool all_see = here && grp * kGroup + kGroup - 1 <= least &&
                           (!CUT || grp * kGroup >= most || (grp + 1) * kGroup <= a.sinks);
      // weights of keys oct, oct + 8 in rows 2 quad, 2 quad + 1
      uint32_t pf[NR][2];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float y[2][2], z[2][2], top[2], topv[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[e] = m[r][e];
          topv[e] = mv[r][e];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            float x = s[r][2 * t + e] * c2[r][e];
            if constexpr (FP8) x *= ksc[t];
            const int key = grp * kGroup + 8 * t + oct;
            const bool see = all_see || (here && key <= last[r][e] && (!CUT || key > last[r][e] - window || key < a.sinks));
            y[t][e] = see ? x : neg_inf();
            top[e] = fmaxf(top[e], y[t][e]);
            if constexpr (FP8) {
              z[t][e] = see ? x + vl2[t] : neg_inf();
              topv[e] = fmaxf(topv[e], z[t][e]);
            }
          }
          if constexpr (!FP8) topv[e] = top[e];
        }
        // the references move for the whole warp, when some weight would pass 2^kLazy (or there was none)
        bool move = false;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          move |= (top[e] > m[r][e] && !(top[e] - m[r][e] <= kLazy)) || (topv[e] > mv[r][e] && !(topv[e] - mv[r][e] <= kLazy));
        if (__any_sync(0xffffffffu, move)) {
          float shrink[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], x));
              if constexpr (FP8) topv[e] = fmaxf(topv[e], __shfl_xor_sync(0xffffffffu, topv[e], x));
            }
            if constexpr (!FP8) topv[e] = top[e];
            // a reference of -inf moves with weights and sums that are all zero
            l[r][e] *= m[r][e] == top[e] ? 1.f : ex2(m[r][e] - top[e]);
            shrink[e] = mv[r][e] == topv[e] ? 1.f : ex2(mv[r][e] - topv[e]);
            m[r][e] = top[e];
            mv[r][e] = topv[e];
          }
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][r][e] *= shrink[e & 1];
        }
        float w[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float base = m[r][e] == neg_inf() ? 0.f : m[r][e];
          const float basev = mv[r][e] == neg_inf() ? 0.f : mv[r][e] - kShift;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float p = ex2(y[t][e] - base);
            l[r][e] += p;
            if constexpr (FP8) w[t][e] = ex2(z[t][e] - basev);
            else if constexpr (kHalf) w[t][e] = ex2(y[t][e] - basev);
            else w[t][e] = p;
          }
        }
        pf[r][0] = transpose8(Mma<M>::pack(w[0][0], w[0][1]));
        pf[r][1] = transpose8(Mma<M>::pack(w[1][0], w[1][1]));
      }
      // V^T P^T: m16 tile t holds elements 2 t, 2 t + 1 of each lane's load
#pragma unroll
      for (int x = 0; x < VL; ++x) {
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          if constexpr (FP8) {
            // four elements per word: bytes of the two keys of a fragment side by side
            const uint32_t lo0 = __byte_perm(vf[0][x][w], vf[1][x][w], 0x5140), hi0 = __byte_perm(vf[0][x][w], vf[1][x][w], 0x7362);
            const uint32_t lo1 = __byte_perm(vf[2][x][w], vf[3][x][w], 0x5140), hi1 = __byte_perm(vf[2][x][w], vf[3][x][w], 0x7362);
            const int t = x * VE / 2 + 2 * w;
            const uint32_t v0[4] = {e4m3x2_to_half2(lo0), e4m3x2_to_half2(lo0 >> 16), e4m3x2_to_half2(lo1), e4m3x2_to_half2(lo1 >> 16)};
            const uint32_t v1[4] = {e4m3x2_to_half2(hi0), e4m3x2_to_half2(hi0 >> 16), e4m3x2_to_half2(hi1), e4m3x2_to_half2(hi1 >> 16)};
#pragma unroll
            for (int r = 0; r < NR; ++r) {
              Mma<M>::run(o[t][r], v0, pf[r][0], pf[r][1]);
              Mma<M>::run(o[t + 1][r], v1, pf[r][0], pf[r][1]);
            }
          } else {
            const int t = x * VE / 2 + w;
            const uint32_t v0[4] = {__byte_perm(vf[0][x][w], vf[1][x][w], 0x5410), __byte_perm(vf[0][x][w], vf[1][x][w], 0x7632),
                                    __byte_perm(vf[2][x][w], vf[3][x][w], 0x5410), __byte_perm(vf[2][x][w], vf[3][x][w], 0x7632)};
#pragma unroll
            for (int r = 0; r < NR; ++r) Mma<M>::run(o[t][r], v0, pf[r][0], pf[r][1]);
          }
        }
      }
      if (it + 1 < count) load_values(grp_next, page_next, slot_next);
      page = page_next;
      slot = slot_next;
    }

    // this run's share of the segment
    const bool whole = count == g.groups;
    const bool prefix = CUT && a.prefix_splits > 0;  // the join has more to add, to whole segments too
    const int64_t part = 2 * static_cast<int64_t>(worker) + (first ? 0 : 1);
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[r][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int row = 8 * r + 2 * quad + e;
        const int i = g.tile * ROWS + row, tok = i / group;
        if (tok >= g.rows) continue;
        if (whole && !prefix) {
          float mul = 0.f;
          if (sum > 0.f || sum != sum) mul = __fdividef(ex2((FP8 ? mv[r][e] - m[r][e] : 0.f) - kShift), sum);
          T* out = static_cast<T*>(a.o) + (g.row0 + tok) * a.o_sT + (hk * group + i - tok * group) * a.o_sH;
#pragma unroll
          for (int x = 0; x < VL; ++x) {
            const int c = 8 * VE * x + VE * oct;
            if (c < a.d) {
#pragma unroll
              for (int j = 0; j < VE / 2; j += 4) {
                uint4 w;
                uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  wp[y] = Mma<T>::pack(o[x * VE / 2 + j + y][r][e] * mul, o[x * VE / 2 + j + y][r][2 + e] * mul);
                *reinterpret_cast<uint4*>(out + c + 2 * j) = w;
              }
            }
          }
        } else {
          // a worker has two segments in part, and any number whole: those lie behind the prefix's parts
          const int64_t pair = (a.prefix_splits * a.T + g.row0 + tok) * a.H + hk * group + i - tok * group;
          float* po = CUT && prefix && whole ? a.prefix_o + pair * DP : a.part_o + (part * kPartRows + row) * DP;
          float* ml = CUT && prefix && whole ? a.prefix_ml + pair * 4 : a.part_ml + (part * kPartRows + row) * 4;
#pragma unroll
          for (int x = 0; x < VL; ++x)
#pragma unroll
            for (int j = 0; j < VE / 2; j += 2) {
              const int t = x * VE / 2 + j;
              *reinterpret_cast<float4*>(po + 8 * VE * x + VE * oct + 2 * j) =
                  make_float4(o[t][r][e], o[t][r][2 + e], o[t + 1][r][e], o[t + 1][r][2 + e]);
            }
          if (oct == 0)
            *reinterpret_cast<float4*>(ml) = make_float4(m[r][e], sum, mv[r][e], 0.f);
        }
      }
    u += count;
    first = false;
  }
  // launched beside the prefix's sums: the join's wait for this kernel's end covers theirs.  By one CTA: the others' SMs
  // are wanted for those that have not started.
  if (CUT && blockIdx.x == gridDim.x - 1) pdl_wait();
}

// Joins the parts of one (row, head): the warps of the CTA take the parts in turn, then join theirs in order.
constexpr int kMaxJoinWarps = 16;

template <typename T, bool HALF, int DP, int ROWS>
__global__ void paged_join_kernel(const __grid_constant__ PagedArgs a) {
  __shared__ float s_ml[kMaxJoinWarps][4];
  __shared__ float s_o[kMaxJoinWarps][DP];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int h = blockIdx.x % a.H;
  const int64_t row = blockIdx.x / a.H;
  // the row's sequence
  int b = static_cast<int>(row), first_row = 0;
  if (a.cu != nullptr) {
    int64_t begin;
    int n;
    clamp_range(a.cu, 0, a.T, begin, n);
    if (row < begin) return;
    const SeqTile t = find_tile(a.cu, a.B, a.T, static_cast<int>(a.T) + 1, static_cast<int>(row - begin), 1, false, false);
    if (t.n == 0) return;  // behind the last sequence
    b = t.seq;
    first_row = t.first;
  }
  const int group = a.H / a.Hk, hk = h / group;
  // its segment: units before the sequence, and all units
  int64_t before = 0, units = 0;
  for (int s = lane; s < a.B; s += 32) {
    const int64_t x = seq_info<false>(a, s, ROWS).units;
    units += x;
    if (s < b) before += x;
  }
  before = warp_sum(before);
  units = warp_sum(units);
  const SeqInfo s = seq_info<false>(a, b, ROWS);
  const int i = first_row * group + (h - hk * group);
  const int tile = i / ROWS, r = i - tile * ROWS;
  const int64_t u0 = before + static_cast<int64_t>(tile) * s.groups, u1 = u0 + s.groups;
  const int64_t workers = active_shares(a, units);
  const int64_t w0 = ((u0 + 1) * workers - 1) / units, w1 = (u1 * workers - 1) / units;
  if (w0 == w1) return;  // one worker held it all and wrote the output
  const int parts = static_cast<int>(w1 - w0 + 1);
  auto slot_of = [&](int x) -> int64_t {
    const int64_t w = w0 + x;
    return 2 * (w * a.Hk + hk) + (x == 0 && units * w / workers < u0 ? 1 : 0);
  };
  constexpr int V = DP / 32;
  float m = neg_inf(), l = 0.f, mv = neg_inf(), o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int x = warp; x < parts; x += warps) {
    const int64_t at = slot_of(x) * kPartRows + r;
    // ordinary loads: the parts are written while this kernel may already be there
    const float4 ml = __ldcg(reinterpret_cast<const float4*>(a.part_ml + at * 4));
    float po[V];
#pragma unroll
    for (int e = 0; e < V; ++e) po[e] = __ldcg(a.part_o + at * DP + lane + 32 * e);
    const float top = fmaxf(m, ml.x), topv = fmaxf(mv, ml.z);
    const float base = top == neg_inf() ? 0.f : top, basev = topv == neg_inf() ? 0.f : topv;
    l = l * ex2(m - base) + ml.y * ex2(ml.x - base);
    const float mine = ex2(mv - basev), theirs = ex2(ml.z - basev);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = o[e] * mine + po[e] * theirs;
    m = top;
    mv = topv;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) s_o[warp][lane + 32 * e] = o[e];
  if (lane == 0) s_ml[warp][0] = m, s_ml[warp][1] = l, s_ml[warp][2] = mv;
  __syncthreads();
  if (warp != 0) return;
  const int used = min(warps, parts);
  float top = neg_inf(), topv = neg_inf();
  for (int w = 0; w < used; ++w) top = fmaxf(top, s_ml[w][0]), topv = fmaxf(topv, s_ml[w][2]);
  const float base = top == neg_inf() ? 0.f : top, basev = topv == neg_inf() ? 0.f : topv;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = 0.f;
  for (int w = 0; w < used; ++w) {
    l += s_ml[w][1] * ex2(s_ml[w][0] - base);
    const float mul = ex2(s_ml[w][2] - basev);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] += s_o[w][lane + 32 * e] * mul;
  }
  float mul = 0.f;
  if (l > 0.f || l != l) mul = __fdividef(ex2(basev - base - (HALF ? kHalfShift : 0.f)), l);
  T* out = static_cast<T*>(a.o) + row * a.o_sT + h * a.o_sH;
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (lane + 32 * e < a.d) out[lane + 32 * e] = Elem<T>::from_f(o[e] * mul);
}

// The same for segments of CUT.  A lane takes one part's maxima and sum, so that the weights of 32 parts are known after
// one load, and then the parts' values are loaded several at a time, a row per load.  The warps take runs of parts and
// join in order; one warp for a (row, head) where those fill the GPU.  With 16 parts of a shared prefix and 64 rows of 32
// heads of 128, 18 MB, it ends 6 us after the split kernel; the join of whole segments took 16 to 20.
template <typename T, bool HALF, int DP, int ROWS>
__global__ void paged_cut_join_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int V = DP / 32, kDeep = 8;
  __shared__ float s_ml[kMaxJoinWarps][4];
  __shared__ float s_o[kMaxJoinWarps][DP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int h = blockIdx.x % a.H;
  const int64_t row = blockIdx.x / a.H;
  const int group = a.H / a.Hk, hk = h / group;
  // the row's sequence and its segment: units before the sequence, and all units
  int b = static_cast<int>(row), first_row = 0;
  bool live = true;
  if (a.cu != nullptr) {
    int64_t begin;
    int n;
    clamp_range(a.cu, 0, a.T, begin, n);
    live = row >= begin;
    if (live) {
      const SeqTile t = find_tile(a.cu, a.B, a.T, static_cast<int>(a.T) + 1, static_cast<int>(row - begin), 1, false, false);
      live = t.n != 0;  // not behind the last sequence
      b = t.seq;
      first_row = t.first;
    }
  }
  int64_t before = 0, units = 0;
  for (int s = lane; s < a.B; s += 32) {
    const int64_t x = seq_info<true>(a, s, ROWS).units;
    units += x;
    if (s < b) before += x;
  }
  before = warp_sum(before);
  units = warp_sum(units);
  int parts = 0, own = 0;
  int64_t w0 = 0, workers = 1, u0 = 0;
  int r = 0;
  if (live) {
    const SeqInfo s = seq_info<true>(a, b, ROWS);
    const int i = first_row * group + (h - hk * group);
    const int tile = i / ROWS;
    r = i - tile * ROWS;
    u0 = before + static_cast<int64_t>(tile) * s.groups;
    workers = active_shares(a, units);
    w0 = ((u0 + 1) * workers - 1) / units;
    own = static_cast<int>(((u0 + s.groups) * workers - 1) / units - w0) + 1;
    if (own == 1) own = 0;  // one worker held it all: it wrote the output, or a part of its own behind the prefix's
    parts = own + (a.prefix_splits > 0 ? a.prefix_splits + (own == 0) : 0);
  }
  pdl_wait();
  if (parts == 0) return;
  // this warp's parts
  const int from = parts * warp / warps, to = parts * (warp + 1) / warps;
  float m = neg_inf(), l = 0.f, mv = neg_inf(), o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = 0.f;
  for (int x0 = from; x0 < to; x0 += 32) {
    const int x = x0 + lane;
    float4 ml = make_float4(neg_inf(), 0.f, neg_inf(), 0.f);
    const float* po = nullptr;
    if (x < to) {
      // ordinary loads: the parts are written while this kernel may already be there
      if (x < own) {
        const int64_t w = w0 + x;
        const int64_t at = (2 * (w * a.Hk + hk) + (x == 0 && units * w / workers < u0 ? 1 : 0)) * kPartRows + r;
        ml = __ldcg(reinterpret_cast<const float4*>(a.part_ml) + at);
        po = a.part_o + at * DP;
      } else {
        const int64_t at = ((x - own) * a.T + row) * a.H + h;
        ml = __ldcg(reinterpret_cast<const float4*>(a.prefix_ml) + at);
        po = a.prefix_o + at * DP;
      }
    }
    float top = ml.x, topv = ml.z;
#pragma unroll
    for (int y = 16; y > 0; y >>= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
      topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, y));
    }
    top = fmaxf(top, m);
    topv = fmaxf(topv, mv);
    const float base = top == neg_inf() ? 0.f : top, basev = topv == neg_inf() ? 0.f : topv;
    float sum = ml.y * ex2(ml.x - base);
#pragma unroll
    for (int y = 16; y > 0; y >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, y);
    l = l * ex2(m - base) + sum;
    const float mine = ex2(mv - basev), weight = ex2(ml.z - basev);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] *= mine;
    m = top;
    mv = topv;
    const int count = min(32, to - x0);
    for (int y0 = 0; y0 < count; y0 += kDeep) {
      float v[kDeep][V];
#pragma unroll
      for (int y = 0; y < kDeep; ++y) {
        const float* p = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(po), (y0 + y) & 31));
#pragma unroll
        for (int e = 0; e < V; ++e) v[y][e] = 0.f;
        if (y0 + y < count) {
          if constexpr (V == 4) {
            const float4 z = __ldcg(reinterpret_cast<const float4*>(p) + lane);
            v[y][0] = z.x, v[y][1] = z.y, v[y][2] = z.z, v[y][3] = z.w;
          } else {
            const float2 z = __ldcg(reinterpret_cast<const float2*>(p) + lane);
            v[y][0] = z.x, v[y][1] = z.y;
          }
        }
      }
#pragma unroll
      for (int y = 0; y < kDeep; ++y) {
        const float w = __shfl_sync(0xffffffffu, weight, (y0 + y) & 31);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(v[y][e], w, o[e]);
      }
    }
  }
  if (warps > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) s_o[warp][V * lane + e] = o[e];
    if (lane == 0) s_ml[warp][0] = m, s_ml[warp][1] = l, s_ml[warp][2] = mv;
    __syncthreads();
    if (warp != 0) return;
    float top = neg_inf(), topv = neg_inf();
    for (int w = 0; w < warps; ++w) top = fmaxf(top, s_ml[w][0]), topv = fmaxf(topv, s_ml[w][2]);
    const float base = top == neg_inf() ? 0.f : top, basev = topv == neg_inf() ? 0.f : topv;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.f;
    for (int w = 0; w < warps; ++w) {
      l += s_ml[w][1] * ex2(s_ml[w][0] - base);
      const float mul = ex2(s_ml[w][2] - basev);
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] += s_o[w][V * lane + e] * mul;
    }
    m = top;
    mv = topv;
  }
  const float base = m == neg_inf() ? 0.f : m, basev = mv == neg_inf() ? 0.f : mv;
  float mul = 0.f;
  if (l > 0.f || l != l) mul = __fdividef(ex2(basev - base - (HALF ? kHalfShift : 0.f)), l);
  if (V * lane >= a.d) return;
  T* out = static_cast<T*>(a.o) + row * a.o_sT + h * a.o_sH + V * lane;
  if constexpr (V == 4)
    *reinterpret_cast<uint2*>(out) = make_uint2(Mma<T>::pack(o[0] * mul, o[1] * mul), Mma<T>::pack(o[2] * mul, o[3] * mul));
  else
    *reinterpret_cast<uint32_t*>(out) = Mma<T>::pack(o[0] * mul, o[1] * mul);
}

template <typename T, bool FP8, int DP, int ROWS, bool CUT>
struct Split {
  static int workers() {
    static std::atomic<int> per_sm{0};  // the same on every device: a property of the code
    int n = per_sm.load(std::memory_order_relaxed);
    if (n == 0) {
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, paged_split_kernel<T, FP8, DP, ROWS, CUT>, kThreads, 0) !=
              cudaSuccess || n <= 0)
        n = 1;
      per_sm.store(n, std::memory_order_relaxed);
    }
    return n * num_sms_here() * (kThreads / 32);  // what the GPU holds at a time
  }
  static cudaError_t run(const PagedArgs& a, cudaStream_t st) {
    constexpr bool kHalf = FP8 || std::is_same<T, __half>::value;
    if (CUT && a.prefix_splits > 0) {
      const cudaError_t l1 = prefer_l1<paged_split_kernel<T, FP8, DP, ROWS, CUT>>();
      if (l1 != cudaSuccess) return l1;
    }
    const cudaError_t e = launch_grid<paged_split_kernel<T, FP8, DP, ROWS, CUT>>(
        CUT && a.prefix_splits > 0, (a.workers + kThreads / 32 - 1) / (kThreads / 32), kThreads, 0, st, a);
    if (e != cudaSuccess) return e;
    // about as many warps as a segment has parts when all are equally long
    const int64_t segments = static_cast<int64_t>(a.B) * a.Hk;
    const int64_t parts = a.workers / (segments > 0 ? segments : 1) + 2 + (CUT ? a.prefix_splits : 0);
    int warps = parts <= 4 ? 2 : parts <= 16 ? 4 : parts <= 64 ? 8 : kMaxJoinWarps;
    // CUT: eight parts to a warp, and no more warps than about 16 an SM
    if (CUT) warps = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(parts + 7) / 8, 2368 / (a.T * a.H), kMaxJoinWarps})));
    if (a.T * a.H > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.T * a.H));
    cfg.blockDim = dim3(static_cast<unsigned>(warps * 32));
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if constexpr (CUT) return cudaLaunchKernelEx(&cfg, paged_cut_join_kernel<T, kHalf, DP, ROWS>, a);
    else return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, kHalf, DP, ROWS>, a);
  }
};

// rows of the operand: 8 when no sequence has more (row, head) pairs per key/value head
template <template <typename, bool, int, int, bool> class F, typename G>
auto with_variant(const PagedArgs& a, int dtype, int quantized, G&& g) {
  const bool few = static_cast<int64_t>(a.max_rows) * (a.H / a.Hk) <= 8;
  auto by_cut = [&](auto t, auto fp8, auto dp, auto rows) {
    using T = decltype(t);
    if (a.window > 0 || a.skip > 0) return g(F<T, decltype(fp8)::value, decltype(dp)::value, decltype(rows)::value, true>());
    return g(F<T, decltype(fp8)::value, decltype(dp)::value, decltype(rows)::value, false>());
  };
  auto by_rows = [&](auto t, auto fp8, auto dp) {
    if (few) return by_cut(t, fp8, dp, std::integral_constant<int, 8>());
    return by_cut(t, fp8, dp, std::integral_constant<int, 16>());
  };
  auto by_dim = [&](auto t, auto fp8) {
    if (a.d <= 64) return by_rows(t, fp8, std::integral_constant<int, 64>());
    return by_rows(t, fp8, std::integral_constant<int, 128>());
  };
  auto by_cache = [&](auto t) {
    if (quantized) return by_dim(t, std::true_type());
    return by_dim(t, std::false_type());
  };
  if (dtype == kBF16) return by_cache(__nv_bfloat16());
  return by_cache(__half());
}

}  // namespace

int paged_split_workers(const PagedArgs& a, int dtype, int quantized) {
  // the same number for every head, one at least
  const int all = with_variant<Split>(a, dtype, quantized, [](auto f) { return f.workers(); });
  return std::max(1, all / a.Hk) * a.Hk;
}

cudaError_t launch_paged_split(const PagedArgs& a, int dtype, int quantized, cudaStream_t st) {
  return with_variant<Split>(a, dtype, quantized, [&](auto f) { return f.run(a, st); });
}

int read_device_error_paged(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_paged_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_paged_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace cta
