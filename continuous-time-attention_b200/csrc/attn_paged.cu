// Attention of the newest rows of each sequence over a paged key/value cache:
// the form for one or a few rows per sequence, where reading the cache once is
// all the work there is.
//
//   O_r = sum_j w_rj V_j / sum_j w_rj,   w_rj = exp(c q_r.k_j),   j <= n - rows + r
//
// What bounds it: HBM, 2 Hk (2 d) bytes per key (e4m3: 2 Hk (d + 4)).  So the
// design keeps loads in flight and does nothing else:
//
// * The rows of all query heads that share a key/value head form one 16-row
//   (8-row, when no more are live) operand of mma.m16n8k16, whose B fragments
//   the lanes load straight from the pages, 16 bytes each, without shared
//   memory.  A contraction may take its index in any order, so the lane that
//   holds key n of a B fragment takes the eight (e4m3: sixteen) elements that
//   one load brings as its share of two (four) k16 steps, and Q is laid out to
//   match; in P V the n index is permuted the same way and undone in the
//   output's address.  tcgen05 would need 128 rows where there are 1 to 16.
// * Every warp is a worker.  The 16-key groups of all (sequence, row tile, head)
//   segments form one list, cut into equal runs, one per worker, whatever the
//   lengths are; the host never reads them.  A worker that holds only a part
//   of a segment leaves (maximum, sum, weighted values) in 32 bits, and a second
//   kernel, launched as a programmatic dependent, joins the parts of a segment
//   in worker order.  Nothing is atomic, so results do not depend on timing.
// * The next group's keys load while this group's softmax runs, the next
//   values while the next scores run.
//
// e4m3: the codes are exact in fp16, so both products run in fp16 whatever the
// type of q.  A bf16 row is first divided by the power of two at its largest
// element, which loses only what is below 2^-24 of that element.  The key's
// scale multiplies the score in 32 bits.  The value's scale joins the weight,
// whose own running maximum keeps weight * scale within fp16 for any scales.
#include "attn_common.cuh"

namespace cta {

__device__ int g_paged_error;

namespace {

constexpr int kThreads = 128;
constexpr int kGroup = 16;      // keys per step of a warp
constexpr int kMinGroups = 2;   // groups a worker gets at least
constexpr int kPartRows = 16;
// fp16 weights carry 2^14: what is lost to subnormals is below 2^-39 of the largest
constexpr float kHalfShift = 14.f;

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
  int b, tile, hk;
  int n, rows;         // keys and rows of the sequence
  int64_t row0;        // its first row in q
  int group, groups;   // first group of this call and groups of the segment
  int64_t start;       // first unit of the segment
};

struct SeqInfo {
  int n, rows, tiles, groups;
  int64_t row0, units;
};
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
  s.groups = max(1, (n + kGroup - 1) / kGroup);  // a sequence without keys still writes its zeros
  s.units = static_cast<int64_t>(s.tiles) * a.Hk * s.groups;
  return s;
}

__device__ __forceinline__ int64_t warp_sum(int64_t x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ int64_t total_units(const PagedArgs& a, int tile_rows) {
  int64_t u = 0;
  for (int b = threadIdx.x & 31; b < a.B; b += 32) u += seq_info(a, b, tile_rows).units;
  return warp_sum(u);
}

__device__ __forceinline__ int active_workers(const PagedArgs& a, int64_t units) {
  return static_cast<int>(min(static_cast<int64_t>(a.workers), max(static_cast<int64_t>(1), units / kMinGroups)));
}

// the segment that holds unit u (u < total); whole warp
__device__ __forceinline__ Seg find_segment(const PagedArgs& a, int64_t u, int tile_rows) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int b0 = 0;; b0 += 32) {
    const SeqInfo s = seq_info(a, b0 + lane, tile_rows);
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
      g.hk = static_cast<int>(seg % a.Hk);
      g.tile = static_cast<int>(seg / a.Hk);
      g.start = first + seg * g.groups;
      return g;
    }
    before += total;
  }
}

template <typename T, bool FP8, int DP, int ROWS>
__global__ void __launch_bounds__(kThreads, DP == 128 ? 2 : ROWS == 8 ? 4 : 3)
    paged_split_kernel(const __grid_constant__ PagedArgs a) {
  using M = typename std::conditional<FP8, __half, T>::type;
  constexpr bool kHalf = std::is_same<M, __half>::value;
  constexpr int R = ROWS / 8;                 // rows per lane
  constexpr int KS = DP / 16;                 // k16 steps of Q K^T
  constexpr int KE = FP8 ? 16 : 8;            // elements of one key load
  constexpr int KL = DP / (4 * KE);           // key loads per lane and key
  constexpr int VE = FP8 && DP == 128 ? 16 : 8;  // elements of one value load
  constexpr int VL = DP / (8 * VE);           // value loads per lane and key
  constexpr int VW = FP8 ? VE / 4 : VE / 2;   // 32-bit words of one value load
  constexpr int NT = DP / 8;                  // n8 tiles of the output

  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, quad = lane & 3, oct = lane >> 2;
  const int worker = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t units = total_units(a, ROWS);
  if (units == 0) return;
  const int workers = active_workers(a, units);
  if (worker >= workers) return;
  int64_t u = units * worker / workers;
  const int64_t u_end = units * (worker + 1) / workers;
  bool first = true;
  const int group = a.H / a.Hk;

  while (u < u_end) {
    const Seg g = find_segment(a, u, ROWS);
    const int count = static_cast<int>(min(u_end - u, static_cast<int64_t>(g.groups - g.group)));

    // Q fragments, and each row's last visible key
    uint32_t qf[KS][R][2];
    float c2[R];
    int last[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = g.tile * ROWS + oct + 8 * r;
      const int tok = i / group;
      const bool live = tok < g.rows;
      last[r] = live ? g.n - g.rows + tok : -1;
      const T* q = static_cast<const T*>(a.q) + (g.row0 + tok) * a.q_sT + (g.hk * group + i - tok * group) * a.q_sH;
      float top = 0.f;
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
      c2[r] = a.scale * kLog2e;
      if constexpr (FP8 && !std::is_same<T, __half>::value) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the power of two at the row's largest element, kept where it and its reciprocal are normal
        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 2), 252);
        const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
        c2[r] *= __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            const float2 x = Elem<T>::unpack(*reinterpret_cast<const typename Elem<T>::Pair*>(&qf[k][r][i2]));
            qf[k][r][i2] = Mma<__half>::pack(x.x * down, x.y * down);
          }
      }
    }

    float o[NT][4];
    float m[R], l[R], mv[R];  // running maximum of the scores, sum of weights, maximum of the weighted values
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = mv[r] = neg_inf(), l[r] = 0.f;

    const int32_t* table = a.table + g.b * a.table_sB;
    auto page_of = [&](int grp) -> int {
      // the page of a group, -1 if the table's entry lies outside the cache
      if (grp >= g.group + count || grp * kGroup >= g.n) return -1;
      const int p = __ldg(table + grp * kGroup / a.page);
      if (p < 0 || p >= a.n_pages) {
        if (lane == 0) atomicExch(&g_paged_error, kDevBadIndex);
        return -1;
      }
      return p;
    };
    uint4 kf[2][KL];
    float ks[2][2], vs[2][2];
    uint32_t vf[4][VL][VW];
    auto load_keys = [&](int grp, int p) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int j = grp * kGroup + 8 * t + oct;
        const bool ok = p >= 0 && j < g.n;
        const int64_t at = p * a.kc_sP + (j % a.page) * a.kc_sS + g.hk * a.kc_sH;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const int c = 4 * KE * i + KE * quad;
          kf[t][i] = make_uint4(0u, 0u, 0u, 0u);
          if (ok && c < a.d) {
            if constexpr (FP8) kf[t][i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.k_cache) + at + c));
            else kf[t][i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.k_cache) + at + c));
          }
        }
      }
    };
    auto load_scales = [&](int grp, int p) {
      if constexpr (FP8) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = grp * kGroup + 8 * t + 2 * quad + e;
            const bool ok = p >= 0 && j < g.n;
            const int64_t at = (static_cast<int64_t>(p) * a.Hk + g.hk) * a.page + j % a.page;
            ks[t][e] = ok ? __ldg(a.k_scale + at) : 1.f;
            vs[t][e] = ok ? __ldg(a.v_scale + at) : 1.f;
          }
      }
    };
    auto load_values = [&](int grp, int p) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = grp * kGroup + 2 * quad + (i & 1) + 8 * (i >> 1);
        const bool ok = p >= 0 && j < g.n;
        const int64_t at = p * a.vc_sP + (j % a.page) * a.vc_sS + g.hk * a.vc_sH;
#pragma unroll
        for (int x = 0; x < VL; ++x) {
          const int c = 8 * VE * x + VE * oct;
#pragma unroll
          for (int w = 0; w < VW; ++w) vf[i][x][w] = 0u;
          if (ok && c < a.d) {
            if constexpr (VW == 4) {
              const uint4 w = FP8 ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.v_cache) + at + c))
                                  : __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.v_cache) + at + c));
              vf[i][x][0] = w.x, vf[i][x][1] = w.y, vf[i][x][2] = w.z, vf[i][x][3] = w.w;
            } else {
              const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v_cache) + at + c));
              vf[i][x][0] = w.x, vf[i][x][1] = w.y;
            }
          }
        }
      }
    };

    int p_now = page_of(g.group), p_next = page_of(g.group + 1);
    load_keys(g.group, p_now);
    load_scales(g.group, p_now);
    load_values(g.group, p_now);
    for (int it = 0; it < count; ++it) {
      const int grp = g.group + it;
      const int p_after = page_of(grp + 2);
      // scores of 16 keys
      float s[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t qa[4];
          qa[0] = qf[k][0][0];
          qa[2] = qf[k][0][1];
          qa[1] = R == 2 ? qf[k][R - 1][0] : 0u;
          qa[3] = R == 2 ? qf[k][R - 1][1] : 0u;
          uint32_t b0, b1;
          if constexpr (FP8) {
            const uint4 w = kf[t][k / 4];
            const uint32_t x = k % 4 == 0 ? w.x : k % 4 == 1 ? w.y : k % 4 == 2 ? w.z : w.w;
            b0 = e4m3x2_to_half2(x);
            b1 = e4m3x2_to_half2(x >> 16);
          } else {
            const uint4 w = kf[t][k / 2];
            b0 = k % 2 == 0 ? w.x : w.z;
            b1 = k % 2 == 0 ? w.y : w.w;
          }
          Mma<M>::run(s[t], qa, b0, b1);
        }
      }
      float ksc[2][2], vsc[2][2];
      if constexpr (FP8) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) ksc[t][e] = ks[t][e], vsc[t][e] = vs[t][e];
      }
      if (it + 1 < count) {
        load_keys(grp + 1, p_next);
        load_scales(grp + 1, p_next);
      }
      // softmax
      uint32_t pf[4];
      pf[1] = pf[3] = 0u;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float y[2][2], z[2][2];
        float top = m[r], topv = mv[r];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = grp * kGroup + 8 * t + 2 * quad + e;
            const bool see = j <= last[r] && p_now >= 0;
            float x = s[t][2 * r + e] * c2[r];
            if constexpr (FP8) x *= ksc[t][e];
            y[t][e] = see ? x : neg_inf();
            top = fmaxf(top, y[t][e]);
            if constexpr (FP8) {
              z[t][e] = see ? x + __log2f(vsc[t][e]) : neg_inf();
              topv = fmaxf(topv, z[t][e]);
            }
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float base = top == neg_inf() ? 0.f : top;
        float basev = base;
        if constexpr (FP8) {
          topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, 1));
          topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, 2));
          basev = topv == neg_inf() ? 0.f : topv;
        } else {
          topv = top;
        }
        float sum = 0.f, w[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = ex2(y[t][e] - base);
            sum += p;
            if constexpr (FP8) w[t][e] = ex2(z[t][e] - basev + kHalfShift);
            else if constexpr (kHalf) w[t][e] = ex2(y[t][e] - base + kHalfShift);
            else w[t][e] = p;
          }
        l[r] = fmaf(l[r], ex2(m[r] - base), sum);
        const float shrink = ex2(mv[r] - basev);
        m[r] = top;
        if (__any_sync(0xffffffffu, topv != mv[r])) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            o[t][2 * r] *= shrink;
            o[t][2 * r + 1] *= shrink;
          }
        }
        mv[r] = topv;
        pf[r] = Mma<M>::pack(w[0][0], w[0][1]);
        pf[2 + r] = Mma<M>::pack(w[1][0], w[1][1]);
      }
      // P V
#pragma unroll
      for (int x = 0; x < VL; ++x) {
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          if constexpr (FP8) {
            // four columns per word: bytes of the two keys of a fragment side by side
            const uint32_t lo0 = __byte_perm(vf[0][x][w], vf[1][x][w], 0x5140), hi0 = __byte_perm(vf[0][x][w], vf[1][x][w], 0x7362);
            const uint32_t lo1 = __byte_perm(vf[2][x][w], vf[3][x][w], 0x5140), hi1 = __byte_perm(vf[2][x][w], vf[3][x][w], 0x7362);
            const int t = x * VE + 4 * w;
            Mma<M>::run(o[t], pf, e4m3x2_to_half2(lo0), e4m3x2_to_half2(lo1));
            Mma<M>::run(o[t + 1], pf, e4m3x2_to_half2(lo0 >> 16), e4m3x2_to_half2(lo1 >> 16));
            Mma<M>::run(o[t + 2], pf, e4m3x2_to_half2(hi0), e4m3x2_to_half2(hi1));
            Mma<M>::run(o[t + 3], pf, e4m3x2_to_half2(hi0 >> 16), e4m3x2_to_half2(hi1 >> 16));
          } else {
            const int t = x * VE + 2 * w;
            Mma<M>::run(o[t], pf, __byte_perm(vf[0][x][w], vf[1][x][w], 0x5410),
                        __byte_perm(vf[2][x][w], vf[3][x][w], 0x5410));
            Mma<M>::run(o[t + 1], pf, __byte_perm(vf[0][x][w], vf[1][x][w], 0x7632),
                        __byte_perm(vf[2][x][w], vf[3][x][w], 0x7632));
          }
        }
      }
      if (it + 1 < count) load_values(grp + 1, p_next);
      p_now = p_next;
      p_next = p_after;
    }

    // this run's share of the segment
    const bool whole = count == g.groups;
    const int64_t slot = 2 * static_cast<int64_t>(worker) + (first ? 0 : 1);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float sum = l[r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int i = g.tile * ROWS + oct + 8 * r;
      const int tok = i / group;
      if (tok >= g.rows) continue;
      // column VE (8 x) + VE (2 quad + e) + j of n8 tile VE x + j
      if (whole) {
        float mul = 0.f;
        if (sum > 0.f || sum != sum) mul = __fdividef(ex2((FP8 ? mv[r] - m[r] : 0.f) - (kHalf ? kHalfShift : 0.f)), sum);
        T* out = static_cast<T*>(a.o) + (g.row0 + tok) * a.o_sT + (g.hk * group + i - tok * group) * a.o_sH;
#pragma unroll
        for (int x = 0; x < VL; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = 8 * VE * x + VE * (2 * quad + e);
            if (c < a.d) {
#pragma unroll
              for (int j = 0; j < VE; j += 8) {
                uint4 w;
                uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  wp[y] = Mma<T>::pack(o[VE * x + j + 2 * y][2 * r + e] * mul, o[VE * x + j + 2 * y + 1][2 * r + e] * mul);
                *reinterpret_cast<uint4*>(out + c + j) = w;
              }
            }
          }
      } else {
        float* po = a.part_o + (slot * kPartRows + oct + 8 * r) * DP;
#pragma unroll
        for (int x = 0; x < VL; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = 8 * VE * x + VE * (2 * quad + e);
#pragma unroll
            for (int j = 0; j < VE; j += 4)
              *reinterpret_cast<float4*>(po + c + j) =
                  make_float4(o[VE * x + j][2 * r + e], o[VE * x + j + 1][2 * r + e], o[VE * x + j + 2][2 * r + e],
                              o[VE * x + j + 3][2 * r + e]);
          }
        if (quad == 0)
          *reinterpret_cast<float4*>(a.part_ml + (slot * kPartRows + oct + 8 * r) * 4) =
              make_float4(m[r], sum, mv[r], 0.f);
      }
    }
    u += count;
    first = false;
  }
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
    const SeqTile t = find_tile(a.cu, a.B, a.T, static_cast<int>(a.T) + 1, static_cast<int>(row - begin), 1, false);
    if (t.n == 0) return;  // behind the last sequence
    b = t.seq;
    first_row = t.first;
  }
  const int group = a.H / a.Hk, hk = h / group;
  // its segment: units before the sequence, and all units
  int64_t before = 0, units = 0;
  for (int s = lane; s < a.B; s += 32) {
    const int64_t x = seq_info(a, s, ROWS).units;
    units += x;
    if (s < b) before += x;
  }
  before = warp_sum(before);
  units = warp_sum(units);
  const SeqInfo s = seq_info(a, b, ROWS);
  const int i = first_row * group + (h - hk * group);
  const int tile = i / ROWS, r = i - tile * ROWS;
  const int64_t u0 = before + (static_cast<int64_t>(tile) * a.Hk + hk) * s.groups, u1 = u0 + s.groups;
  const int64_t workers = active_workers(a, units);
  const int64_t w0 = ((u0 + 1) * workers - 1) / units, w1 = (u1 * workers - 1) / units;
  if (w0 == w1) return;  // one worker held it all and wrote the output
  const int parts = static_cast<int>(w1 - w0 + 1);
  auto slot_of = [&](int x) -> int64_t {
    const int64_t w = w0 + x;
    return 2 * w + (x == 0 && units * w / workers < u0 ? 1 : 0);
  };
  constexpr int V = DP / 32;
  float m = neg_inf(), l = 0.f, mv = neg_inf(), o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int x = warp; x < parts; x += warps) {
    const int64_t at = slot_of(x) * kPartRows + r;
    const float4 ml = __ldg(reinterpret_cast<const float4*>(a.part_ml + at * 4));
    float po[V];
#pragma unroll
    for (int e = 0; e < V; ++e) po[e] = __ldg(a.part_o + at * DP + lane + 32 * e);
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

int num_sms_here() {
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) return 148;
  return v;
}

template <typename T, bool FP8, int DP, int ROWS>
struct Split {
  static int workers() {
    static int per_sm = 0;  // the same on every device: a property of the code
    if (per_sm == 0) {
      int n = 0;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, paged_split_kernel<T, FP8, DP, ROWS>, kThreads, 0) !=
              cudaSuccess || n <= 0)
        n = 1;
      per_sm = n;
    }
    return per_sm * num_sms_here() * (kThreads / 32);
  }
  static cudaError_t run(const PagedArgs& a, cudaStream_t st) {
    constexpr bool kHalf = FP8 || std::is_same<T, __half>::value;
    paged_split_kernel<T, FP8, DP, ROWS>
        <<<static_cast<unsigned>(a.workers / (kThreads / 32)), kThreads, 0, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // about as many warps as a segment has parts when all are equally long
    const int64_t segments = static_cast<int64_t>(a.B) * a.Hk;
    const int64_t parts = a.workers / (segments > 0 ? segments : 1) + 2;
    const int warps = parts <= 4 ? 2 : parts <= 16 ? 4 : parts <= 64 ? 8 : kMaxJoinWarps;
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
    return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, kHalf, DP, ROWS>, a);
  }
};

// rows of the operand: 8 when no sequence has more (row, head) pairs per key/value head
template <template <typename, bool, int, int> class F, typename G>
auto with_variant(const PagedArgs& a, int dtype, int quantized, G&& g) {
  const bool few = static_cast<int64_t>(a.max_rows) * (a.H / a.Hk) <= 8;
  auto by_rows = [&](auto t, auto fp8, auto dp) {
    using T = decltype(t);
    if (few) return g(F<T, decltype(fp8)::value, decltype(dp)::value, 8>());
    return g(F<T, decltype(fp8)::value, decltype(dp)::value, 16>());
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
  return with_variant<Split>(a, dtype, quantized, [](auto f) { return f.workers(); });
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
