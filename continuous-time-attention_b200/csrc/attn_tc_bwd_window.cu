// Attention backward on the tensor cores under a sliding window whose first keys stay visible, 16-bit tensors: the
// mathematics, the two kernels and their warps are those of attn_tc_bwd.cu, whose comments hold here too.  What is
// different:
//
// * A row tile meets the key tiles of its rows' windows and, before them, those of the first keys; a key tile meets the
//   rows whose windows hold one of its keys.
// * The first keys are seen by all rows.  Their tiles would meet many times as many rows as the others, and the last CTA
//   would work alone: 16384 tokens, 8 heads of 64, window 1024: 128 steps where the others have 10.  So the rows
//   behind such a tile's window, the far ones, are another launch of the dK, dV kernel, a CTA per `chunk` rows, which
//   leaves its sums over the first keys in `far` in 32 bits; the tile's own CTA adds them in order (programmatic
//   dependent launch: it waits for them only then).
// * The pieces of work are short, about as long as it takes to set up a CTA, to fetch its first tiles and to write its
//   results.  So a CTA that is nearly through with a piece takes over another that has not started (cluster launch
//   control): its tiles load and its first scores run under the last weights and the results of the one before.
//   Barriers go on from piece to piece.
//
// Bound by the latency of a piece's first and last steps, and like the kernels of whole sequences in between.  Measured,
// bf16, 16384 tokens, window 1024, 4 first keys: 8 heads of 64 dQ 104 us, dK and dV 125 and 21 for the far rows (a CTA per
// piece: 124, 146, 21); 32/8 heads of 128 500, 690 and 97.  Window 128, none: 47 and 45 us (67 and 69), 223 and 187 (337
// and 225).
#include <algorithm>

#include "attn_tc_bwd.cuh"

namespace cta {

__device__ int g_tc_bwd_window_error;

namespace {

using namespace tcbwd;

struct BwdArgs {
  AttnArgs a;
  int pack, tile_tokens;
  int wide_dq, wide_dk, wide_dv;  // alignment of the gradients' rows, see store_rows
  // window: the far rows' share of the first keys, see kFar
  float* far;
  int chunk, sink_tiles, far_keys;
  int warp_span;  // tokens from a warp's first row to its last
};

// kNear: rows up to the end of the tile's window.  kFar: the others, for the first keys.
enum Form : int { kNear = 0, kFar = 1 };

struct Pieces {
  uint64_t full, taken, answer;
  SeqTile tile[2];
  int id[2];
  __align__(16) uint4 response;
};
enum : int { kNoPiece = -1, kTimeout = -2 };
// One warp plans, the others take.
struct Taker {
  Pieces& s;
  // the it-th piece of this CTA: its number among those of the launch
  __device__ __forceinline__ int operator()(int it, SeqTile& t) const {
    if (it > 0 && !tc::wait(&s.full, (it - 1) & 1)) return kTimeout;
    const int id = s.id[it & 1];
    t = s.tile[it & 1];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::arrive(&s.taken);
    return id;
  }
  // Finds the it-th piece, not the first, when all warps have taken the one before: a warp that is behind would miss a
  // phase of `full` otherwise.
  template <typename Find>
  __device__ __forceinline__ int plan(Find&& find, int it, SeqTile& t) const {
    if (!tc::wait(&s.taken, (it - 1) & 1)) return kTimeout;
    const bool lane0 = (threadIdx.x & 31) == 0;
    if (lane0) {
      mbar_arrive_expect_tx(&s.answer, 16);
      tc::steal(&s.response, &s.answer);
    }
    if (!tc::wait(&s.answer, (it - 1) & 1)) return kTimeout;
    const int id = tc::stolen(&s.response);
    if (id >= 0) t = find(id);
    if (lane0) {
      s.tile[it & 1] = t;
      s.id[it & 1] = id;
      tc::arrive(&s.full);
    }
    __syncwarp();
    return id;
  }
};

// ---------------------------------------------------------------------------
// dQ
// ---------------------------------------------------------------------------
struct DqBars {
  uint64_t q_full, q_empty, kv_full[8], kv_empty[8], s_full[2], s_free[2], dp_full, dp_read, ds_full[2], done, sums_free;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_window_dq_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap gmap,
                      const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ BwdArgs f) {
  using L = Layout<DP>;
  constexpr int NS = L::kStages;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  __shared__ DqBars bars;
  __shared__ float s_most[kHalf ? kWeightWarps : 1];
  __shared__ uint32_t s_tmem;
  __shared__ Pieces s_pieces;
  const AttnArgs& a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const int blocks = a.H / f.pack;
  auto find = [&](int id) {
    return find_tile(a.cu, a.nseq, a.L, a.tiles, id / blocks, f.tile_tokens, true, true);
  };

  if (warp == 0) {
    const SeqTile x = find(blockIdx.x);
    if (lane == 0) s_pieces.tile[0] = x, s_pieces.id[0] = blockIdx.x;
  } else if (warp == kWeightWarps) {
    tc::alloc(&s_tmem, 512);
  } else if (warp == kWeightWarps + 1 && lane == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&bars.kv_full[i], 1);
      mbar_init(&bars.kv_empty[i], 1);
    }
    mbar_init(&bars.s_full[0], 1);
    mbar_init(&bars.s_full[1], 1);
    mbar_init(&bars.s_free[0], 1);
    mbar_init(&bars.s_free[1], 1);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.dp_read, kWeightWarps);
    mbar_init(&bars.ds_full[0], kWeightWarps);
    mbar_init(&bars.ds_full[1], kWeightWarps);
    mbar_init(&bars.done, 1);
    mbar_init(&bars.sums_free, kWeightWarps);
    mbar_init(&s_pieces.full, 1);
    mbar_init(&s_pieces.taken, kWeightWarps + 2);
    mbar_init(&s_pieces.answer, 1);
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t t_dp = tmem + 256, t_dq = tmem + 384;  // scores: columns 0 and 128
  const Taker take{s_pieces};

  struct Plan {
    const uint32_t* mask;
    int h0, hk, lo, j_lo, end, steps;
    // window: from step `jump` on, `gap` tiles further; those between the first keys and the rows' windows are passed over
    int sink_end, window_lo, jump, gap;
    __device__ __forceinline__ int first_key(int j) const { return (j_lo + j + (j >= jump ? gap : 0)) * kRows; }
    // a step of first keys alone, up to 32 of them: a quarter of the products
    __device__ __forceinline__ bool narrow(int j) const { return j < jump && jump < (1 << 30) && sink_end - first_key(j) <= 32; }
    __device__ __forceinline__ void key_words(int n, int j, uint32_t (&w)[4]) const {
      const int j0 = first_key(j);
      tc::first_bits(n - j0, w);
      if (mask != nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (w[i] != 0u) w[i] &= __ldg(mask + kMaskHead + (j0 >> 5) + i);
      }
    }
  };
  auto plan = [&](int id, const SeqTile& t) {
    Plan p;
    p.h0 = id % blocks * f.pack;
    p.hk = p.h0 / (a.H / a.Hk);
    int hi = t.n;
    mask_range(a, t.batch, t.n, p.lo, hi);
    p.mask = a.mask != nullptr ? a.mask + t.batch * a.mask_words : nullptr;
    p.j_lo = p.lo / kRows;
    p.end = min(hi, t.first + f.tile_tokens);
    p.sink_end = a.sinks > 0 ? p.lo + a.sinks : 0;
    p.window_lo = max(p.lo, t.first - a.window + 1);  // first key of the first row's window
    p.jump = 1 << 30;
    p.gap = 0;
    const int sink_tiles = (p.sink_end + kRows - 1) / kRows;
    if (a.sinks == 0) p.j_lo = p.window_lo / kRows;
    else if (p.window_lo / kRows > sink_tiles) p.jump = sink_tiles - p.j_lo, p.gap = p.window_lo / kRows - sink_tiles;
    int steps = (p.end + kRows - 1) / kRows - p.j_lo;
    if (steps > p.jump) steps = max(p.jump, steps - p.gap);
    p.steps = t.first < t.n ? max(0, steps) : 0;
    return p;
  };

  // running numbers, over all pieces: jj steps, x tiles of keys and values, nq pieces with steps
  SeqTile t;
  bool ok = true;
  if (warp == kWeightWarps + 1) {
    // and the pieces to come: the next is asked for when this one's loads are on their way
    int issued = 0, nq = 0, id = blockIdx.x;
    t = s_pieces.tile[0];
    for (int it = 0; id >= 0; id = take.plan(find, ++it, t)) {
      const Plan p = plan(id, t);
      auto load_rows = [&] {
        if (nq > 0) ok = tc::wait(&bars.q_empty, (nq - 1) & 1);
        if (!ok) return;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars.q_full, 2 * L::kTile);
          for (int c = 0; c < DP / 64; ++c) {
            tc::tma_load_4d(smem + c * L::kHalf, &qmap, &bars.q_full, 64 * c, p.h0, static_cast<int>(t.row0) + t.first,
                            t.batch);
            tc::tma_load_4d(smem + L::kTile + c * L::kHalf, &gmap, &bars.q_full, 64 * c, p.h0,
                            static_cast<int>(t.row0) + t.first, t.batch);
          }
        }
        ++nq;
      };
      for (int y = 0; y < 2 * p.steps; ++y) {
        const int x = issued, stage = x % NS;
        if (x >= NS) ok = tc::wait(&bars.kv_empty[stage], ((x / NS) - 1) & 1);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars.kv_full[stage], L::kTile);
          for (int c = 0; c < DP / 64; ++c)
            tc::tma_load_4d(smem + (2 + stage) * L::kTile + c * L::kHalf, (y & 1) ? &vmap : &kmap, &bars.kv_full[stage],
                            64 * c, p.hk, static_cast<int>(t.row0) + p.first_key(y >> 1), t.batch);
        }
        issued = x + 1;
        if (y == 1) load_rows();  // the piece before may still need its own
        if (!ok) break;
      }
      if (!ok) break;
    }
    ok = ok && id != kTimeout;
    if (!ok) {
      atomicExch(&g_tc_bwd_window_error, kDevTimeout);
      for (int x = max(0, issued - NS); x < issued; ++x) tc::wait(&bars.kv_full[x % NS], (x / NS) & 1);
      if (nq > 0) tc::wait(&bars.q_full, (nq - 1) & 1);
    }
  } else if (warp == kWeightWarps) {
    // scores and dO V^T; another warp issues dQ: every wait takes a hundred cycles or two, and one warp
    // for all three was what the steps waited for
    constexpr uint32_t id_s = tc::idesc<T>(kRows, false), id_32 = tc::idesc<T>(32, false);
    const bool leader = tc::elect_one();
    int jj = 0, nq = 0;
    for (int it = 0; ok; ++it) {
      const int id = take(it, t);
      ok = id != kTimeout;
      if (id < 0) break;
      const Plan p = plan(id, t);
      if (p.steps == 0) continue;
      ok = tc::wait(&bars.q_full, nq & 1);
      ++nq;
      for (int j = 0; j < p.steps && ok; ++j, ++jj) {
        const int xk = 2 * jj, xv = xk + 1;
        const uint32_t k = smem + (2 + xk % NS) * L::kTile, v = smem + (2 + xv % NS) * L::kTile;
        const uint32_t id = p.narrow(j) ? id_32 : id_s;
        ok = tc::wait(&bars.kv_full[xk % NS], (xk / NS) & 1);
        if (ok && (p.mask != nullptr || p.first_key(j) + kRows > t.n)) {
          uint32_t w[4];
          p.key_words(t.n, j, w);
          if (!tc::all_set(w)) tc::clear_rows<DP / 64>(k, w);
        }
        // the score gradients of step jj - 2 lie in the buffer until they are in dQ
        if (jj >= 2) ok = ok && tc::wait(&bars.s_free[jj & 1], ((jj >> 1) - 1) & 1);
        tc::fence_after();
        if (ok && leader) {
          tc::product_nt<DP>(tmem + (jj & 1) * 128, smem, k, id);
          tc::commit(&bars.s_full[jj & 1]);
        }
        __syncwarp();
        ok = ok && tc::wait(&bars.kv_full[xv % NS], (xv / NS) & 1);
        if (jj >= 1) ok = ok && tc::wait(&bars.dp_read, (jj - 1) & 1);
        tc::fence_after();
        if (ok && leader) {
          tc::product_nt<DP>(t_dp, smem + L::kTile, v, id);
          tc::commit(&bars.dp_full);
          tc::commit(&bars.kv_empty[xv % NS]);
          if (j + 1 == p.steps) tc::commit(&bars.q_empty);
        }
        __syncwarp();
      }
      if (!ok) break;
    }
    if (!ok && lane == 0) atomicExch(&g_tc_bwd_window_error, kDevTimeout);
  } else if (warp == kWeightWarps + 2) {
    constexpr uint32_t id_o = tc::idesc<T>(DP, true);
    const bool leader = tc::elect_one();
    int jj = 0, nq = 0;
    for (int it = 0; ok; ++it) {
      const int id = take(it, t);
      ok = id != kTimeout;
      if (id < 0) break;
      const Plan p = plan(id, t);
      for (int j = 0; j < p.steps && ok; ++j, ++jj) {
        ok = tc::wait(&bars.ds_full[jj & 1], (jj >> 1) & 1);
        // the sums of the piece before have been read
        if (j == 0 && nq > 0) ok = ok && tc::wait(&bars.sums_free, (nq - 1) & 1);
        tc::fence_after();
        if (ok && leader) {
          const uint32_t ds = tmem + (jj & 1) * 128, k = smem + (2 + (2 * jj) % NS) * L::kTile;
          if (p.narrow(j)) tc::product_tn<32, 2>(t_dq, ds, k, id_o, j > 0);
          else tc::product_tn<32>(t_dq, ds, k, id_o, j > 0);
          tc::commit(&bars.s_free[jj & 1]);
          tc::commit(&bars.kv_empty[(2 * jj) % NS]);
          if (j + 1 == p.steps) tc::commit(&bars.done);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (p.steps > 0) ++nq;
    }
    if (!ok && lane == 0) atomicExch(&g_tc_bwd_window_error, kDevTimeout);
  } else if (warp < kWeightWarps) {
    const int part = warp >> 2;  // columns [32 part, 32 part + 32) of each tile
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float c2 = a.scale * kLog2e;
    int jj = 0, nq = 0;
    for (int it = 0;; ++it) {
      const int id = ok ? take(it, t) : kTimeout;
      ok = id != kTimeout;
      // all of them go on or none; and what the piece before left in s_most has been read
      if (kHalf) ok = !tc::any_of(1, 32 * kWeightWarps, !ok);
      if (!ok || id < 0) break;
      const Plan p = plan(id, t);
      const int tok = t.first + row / f.pack, h = p.h0 + row % f.pack;
      const bool live = tok < t.n;
      // all of these loads are on their way before the first is used
      const int64_t at = live ? lse_index(a, t, h, tok) : 0;
      const float lse = live ? a.lse[at] : neg_inf(), delta = live ? a.delta[at] : 0.f;
      float norm = 0.f, most = 0.f;
      if constexpr (kHalf) {
        norm = live ? a.g_norm[at] : 0.f;
        if (p.steps > 0) {
          const float* norms = a.v_norm + (static_cast<int64_t>(t.batch) * a.Hk + p.hk) * a.L + t.row0;
          most = most_of(norms, p.window_lo, p.end);
          if (p.sink_end > p.lo) most = fmaxf(most, most_of(norms, p.lo, min(min(p.sink_end, p.window_lo), p.end)));
        }
      }
      const float nl = neg_lse2_of(lse);
      const bool none = blind(nl);
      const int limit = tok;                                     // last key the row sees
      const int limit_all = t.first + (warp & 3) * 32 / f.pack;  // and that all rows of the warp see
      const bool any_blind = __any_sync(0xffffffffu, none);
      // fp16: the row's power of two
      int unit = 0;
      if constexpr (kHalf) {
        most = warp_max(most);
        if (lane == 0) s_most[warp] = most;
        __syncwarp();
        tc::sync_of(1, 32 * kWeightWarps);
        most = warp_max(s_most[lane % kWeightWarps]);  // by the whole warp, its rows behind the sequence too
        unit = live ? unit_exponent(finite(norm) * most + finite(delta)) : 0;
      }
      const float up = pow2(unit), neg_delta = -delta * up;
      auto less_delta = [&](float2 x) {
        if constexpr (kHalf) return fma2(x, f2(up), f2(neg_delta));
        else return add2(x, f2(-delta));
      };
      // after a wait that ran out a warp goes on without waiting to the end of the piece
      for (int j = 0; j < p.steps; ++j, ++jj) {
        const uint32_t s_addr = tmem + lanes + (jj & 1) * 128 + part * 32;
        ok = ok && tc::wait(&bars.s_full[jj & 1], (jj >> 1) & 1);
        tc::fence_after();
        uint32_t s[32], dp[32];
        tc::ld32(s_addr, s);
        const int j0 = p.first_key(j);
        bool whole = j0 + kRows <= t.n && !any_blind && j0 + kRows - 1 <= limit_all &&
                     (j0 > limit_all + f.warp_span - a.window || j0 + kRows <= p.sink_end);
        uint32_t w[4];
        if (p.mask != nullptr || !whole) {
          p.key_words(t.n, j, w);
          whole = whole && tc::all_set(w);
        }
        tc::wait_ld(s);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), f2(c2), f2(nl));
          s[e] = __float_as_uint(ex2(x.x));
          s[e + 1] = __float_as_uint(ex2(x.y));
        }
        ok = ok && tc::wait(&bars.dp_full, jj & 1);
        tc::fence_after();
        tc::ld32(t_dp + lanes + part * 32, dp);
        tc::wait_ld(dp);
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::arrive(&bars.dp_read);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = mul2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])),
                                less_delta(make_float2(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1]))));
          dp[e] = __float_as_uint(x.x);
          dp[e + 1] = __float_as_uint(x.y);
        }
        if (!whole) {
          const int left = none ? 0 : limit - j0 - 32 * part + 1;
          uint32_t see = (part == 0 ? w[0] : part == 1 ? w[1] : part == 2 ? w[2] : w[3]) &
                         (left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u);
          see &= tc::bits_from(left - a.window) | ~tc::bits_from(p.sink_end - j0 - 32 * part);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((see >> e) & 1u)) dp[e] = 0u;
        }
        uint32_t ds[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] = tc::pack2<T>(__uint_as_float(dp[2 * e]), __uint_as_float(dp[2 * e + 1]));
        tc::st16(s_addr, ds);
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::arrive(&bars.ds_full[jj & 1]);
      }
      if (p.steps > 0) {
        ok = ok && tc::wait(&bars.done, nq & 1);
        ++nq;
      }
      tc::fence_after();
      if (!ok) {
        if (lane == 0) atomicExch(&g_tc_bwd_window_error, kDevTimeout);
      } else if (t.first < t.n) {
        T* out = static_cast<T*>(a.dq) + t.batch * a.dqs.b + (t.row0 + tok) * a.dqs.t + h * a.dqs.h;
        tc::store_rows<T, DP / 4>(t_dq + lanes + part * (DP / 4), out, part * (DP / 4), a.d,
                                  kHalf ? a.scale * pow2(-unit) : a.scale, live, f.wide_dq, p.steps > 0);
      } else if (a.cu != nullptr && t.n == 0 && part == 0) {
        for (int64_t r = t.row0 + t.tail_index; r < a.L; r += t.tail_count)
          for (int x = threadIdx.x; x < a.d * f.pack; x += kRows)
            static_cast<T*>(a.dq)[r * a.dqs.t + (p.h0 + x / a.d) * a.dqs.h + x % a.d] = Elem<T>::from_f(0.f);
      }
      if (p.steps > 0) {
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::arrive(&bars.sums_free);
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kWeightWarps) tc::dealloc(tmem, 512);
  pdl_wait();  // launched beside dK and dV; a CTA ends only when there is no more work
}

// ---------------------------------------------------------------------------
// dK, dV: the tiles are transposed, rows are keys and columns are query rows
// ---------------------------------------------------------------------------
struct DkvBars {
  uint64_t kv_full, kv_empty, q_full[4], q_empty[4], g_full[4], g_empty[4], stat_full[4], s_full[2], s_free[2], p_full[2], dp_full, dp_free, ds_full[2], done, sums_free;
};

template <typename T, int DP, int FORM>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_window_dkv_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap gmap,
                       const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ BwdArgs f) {
  using L = Layout<DP>;
  constexpr int NS = L::kPairs;  // (Q, dO) pairs in flight
  extern __shared__ uint8_t smem_raw[];
  __shared__ DkvBars bars;
  __shared__ uint32_t s_tmem;
  __shared__ Pieces s_pieces;
  __shared__ __align__(16) float s_stat[NS][2][kRows];  // [stage][-lse2, -delta, fp16: + 14, * its unit][row]
  const AttnArgs& a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
  // With two score buffers dS goes beside P, into the columns that P leaves of its scores', and the next dO V^T can
  // start once this one has been read; with one it goes over dO V^T, so that the next scores wait for dV only.
  constexpr bool kBeside = DP == 64;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  __shared__ float s_most[kHalf ? 3 : 1][kHalf ? kWeightWarps : 1];  // |g|, |delta|, |v|
  const int group = a.H / a.Hk;
  pdl_launch_dependents();  // dQ's CTAs may follow
  auto find = [&](int id) {
    // the first keys of a causal sequence meet the most rows: forwards is heaviest first
    return FORM == kFar ? find_tile(a.cu, a.nseq, a.L, a.tiles, id / a.Hk / f.sink_tiles, f.chunk, false, false)
                        : find_tile(a.cu, a.nseq, a.L, a.tiles, id / a.Hk, kRows, false, true);
  };

  if (warp == 0) {
    const SeqTile x = find(blockIdx.x);
    if (lane == 0) s_pieces.tile[0] = x, s_pieces.id[0] = blockIdx.x;
  } else if (warp == kWeightWarps) {
    tc::alloc(&s_tmem, 512);
  } else if (warp == kWeightWarps + 1 && lane == 0) {
    mbar_init(&bars.kv_full, 1);
    mbar_init(&bars.kv_empty, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&bars.q_full[i], 1);
      mbar_init(&bars.q_empty[i], 1);
      mbar_init(&bars.g_full[i], 1);
      mbar_init(&bars.g_empty[i], 1);
      mbar_init(&bars.stat_full[i], 1);
    }
    mbar_init(&bars.s_full[0], 1);
    mbar_init(&bars.s_full[1], 1);
    mbar_init(&bars.s_free[0], 1);
    mbar_init(&bars.s_free[1], 1);
    mbar_init(&bars.dp_free, kBeside ? kWeightWarps : 1);
    mbar_init(&bars.p_full[0], kWeightWarps);
    mbar_init(&bars.p_full[1], kWeightWarps);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.ds_full[0], kWeightWarps);
    mbar_init(&bars.ds_full[1], kWeightWarps);
    mbar_init(&bars.done, 1);
    mbar_init(&bars.sums_free, kWeightWarps);
    mbar_init(&s_pieces.full, 1);
    mbar_init(&s_pieces.taken, kWeightWarps + 3);
    mbar_init(&s_pieces.answer, 1);
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = s_tmem;
  // Scores: one buffer of 128 columns at dim 128, where the four accumulators fill tensor memory, two at 64
  constexpr int NB = DP == 64 ? 2 : 1;
  const uint32_t t_dp = tmem + NB * 128, t_dv = t_dp + 128, t_dk = t_dv + DP;
  const Taker take{s_pieces};

  struct Plan {
    const uint32_t* mask;
    int hk, lo, row_from, row_to, i_lo, per_head, steps, h_first, pack, tile_tokens;
    int sink_end, far_from;  // far_from: the first of the far rows of a tile that holds first keys
    bool scattered;          // a window may lie on masked keys alone: rows that see none are anywhere
    __device__ __forceinline__ int head_of(int s) const { return h_first + s / per_head * pack; }
    __device__ __forceinline__ int first_of(int s) const { return (i_lo + s % per_head) * tile_tokens; }
  };
  // kFar: t, a chunk of rows, becomes the key tile
  auto plan = [&](int id, SeqTile& t) {
    Plan p;
    p.hk = id % a.Hk;
    p.h_first = p.hk * group;
    p.pack = f.pack;
    p.tile_tokens = f.tile_tokens;
    p.mask = a.mask != nullptr ? a.mask + t.batch * a.mask_words : nullptr;
    int hi;
    mask_range(a, t.batch, t.n, p.lo, hi);
    p.sink_end = a.sinks > 0 ? p.lo + a.sinks : 0;
    p.scattered = p.mask != nullptr && a.sinks == 0;
    const int chunk_from = t.first;
    if constexpr (FORM == kFar) t.first = (p.lo / kRows + id / a.Hk % f.sink_tiles) * kRows;
    // row tiles that meet these keys, for each block of heads of the group
    p.far_from = (min(t.n, t.first + kRows - 1 + a.window) + f.tile_tokens - 1) / f.tile_tokens * f.tile_tokens;
    bool some;  // any valid key
    if constexpr (FORM == kFar) {
      p.row_from = max(chunk_from, p.far_from);
      p.row_to = min(chunk_from + f.chunk, t.n);
      some = t.first < min(min(t.n, hi), p.sink_end) && p.row_from < p.row_to;
    } else {
      p.row_from = t.first;
      p.row_to = min(t.n, p.far_from);
      some = t.first < min(t.n, hi) && t.first + kRows > p.lo;
    }
    p.i_lo = p.row_from / f.tile_tokens;
    p.per_head = max(0, (p.row_to + f.tile_tokens - 1) / f.tile_tokens - p.i_lo);
    p.steps = some ? p.per_head * (group / f.pack) : 0;
    return p;
  };
  // the sums of the far rows of chunk c over the first keys of this tile: dV, then dK, [far_keys][2][DP]
  auto far_at = [&](const Plan& p, const SeqTile& t, int chunk) {
    const int64_t slot = far_place(a, t, kRows, f.chunk) + chunk;
    return f.far + ((slot * f.sink_tiles + (t.first / kRows - p.lo / kRows)) * a.Hk + p.hk) * f.far_keys * 2 * DP;
  };

  // fp16: the exponent of the CTA's power of two; the weight warps and the warp of the statistics
  auto unit_of = [&] {
    tc::sync_of(1, 32 * (kWeightWarps + 1));
    const int w = kHalf ? lane % kWeightWarps : 0;
    return unit_exponent(warp_max(s_most[0][w]) * warp_max(s_most[kHalf ? 2 : 0][w]) + warp_max(s_most[kHalf ? 1 : 0][w]));
  };

  // running numbers, over all pieces: ss steps, nk pieces with steps
  SeqTile t;
  bool ok = true;
  int ss = 0, nk = 0;
  if (warp == kWeightWarps + 1) {
    int issued = 0;
    for (int it = 0; ok; ++it) {
      const int id = take(it, t);
      ok = id != kTimeout;
      if (id < 0) break;
      const Plan p = plan(id, t);
      if (p.steps == 0) continue;
      // Q and dO of a step by turns, each given back when its last product is done
      auto load_rows = [&](int y) {
        const int s = issued >> 1, stage = s % NS;  // y: of this piece
        uint64_t* full = (y & 1) ? &bars.g_full[stage] : &bars.q_full[stage];
        if (s >= NS) ok = tc::wait((y & 1) ? &bars.g_empty[stage] : &bars.q_empty[stage], ((s / NS) - 1) & 1);
        if (!ok) return;
        if (lane == 0) {
          mbar_arrive_expect_tx(full, L::kTile);
          for (int c = 0; c < DP / 64; ++c)
            tc::tma_load_4d(smem + (2 + 2 * stage + (y & 1)) * L::kTile + c * L::kHalf, (y & 1) ? &gmap : &qmap, full, 64 * c,
                            p.head_of(y >> 1), static_cast<int>(t.row0) + p.first_of(y >> 1), t.batch);
        }
        ++issued;
      };
      auto load_keys = [&] {
        if (nk > 0) ok = tc::wait(&bars.kv_empty, (nk - 1) & 1);
        if (!ok) return;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars.kv_full, 2 * L::kTile);
          for (int c = 0; c < DP / 64; ++c) {
            tc::tma_load_4d(smem + c * L::kHalf, &kmap, &bars.kv_full, 64 * c, p.hk, static_cast<int>(t.row0) + t.first,
                            t.batch);
            tc::tma_load_4d(smem + L::kTile + c * L::kHalf, &vmap, &bars.kv_full, 64 * c, p.hk,
                            static_cast<int>(t.row0) + t.first, t.batch);
          }
        }
        ++nk;
      };
      for (int y = 0; y < 2 * p.steps && ok; ++y) {
        load_rows(y);
        if (ok && y == 0) load_keys();  // the piece before may still need its own
      }
    }
    if (!ok) {
      atomicExch(&g_tc_bwd_window_error, kDevTimeout);
      for (int x = max(0, issued - 2 * NS); x < issued; ++x)
        tc::wait((x & 1) ? &bars.g_full[(x >> 1) % NS] : &bars.q_full[(x >> 1) % NS], ((x >> 1) / NS) & 1);
      if (nk > 0) tc::wait(&bars.kv_full, (nk - 1) & 1);
    }
  } else if (warp == kWeightWarps + 2) {
    // and the pieces to come: the next is asked for when this one's statistics are all there
    for (int it = 0;; ++it) {
      int id = kTimeout;
      if (it == 0) t = s_pieces.tile[0], id = blockIdx.x;
      else if (ok) id = take.plan(find, it, t);
      ok = id != kTimeout;
      if (kHalf) ok = !tc::any_of(2, 32 * (kWeightWarps + 1), !ok);
      if (!ok || id < 0) break;
      const Plan p = plan(id, t);
      float down = 1.f;
      if constexpr (kHalf) down = pow2(unit_of() - static_cast<int>(kHalfShift));
      for (int s = 0; s < p.steps; ++s, ++ss) {
        const int stage = ss % NS;
        float nl[4], dl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = lane + 32 * i;
          const int tok = p.first_of(s) + r / f.pack, h = p.head_of(s) + r % f.pack;
          nl[i] = tok < t.n ? neg_lse2_of(__ldg(a.lse + lse_index(a, t, h, tok))) : neg_inf();
          dl[i] = tok < t.n ? -__ldg(a.delta + lse_index(a, t, h, tok)) : 0.f;
          if (blind(nl[i])) dl[i] = 0.f;
          if constexpr (kHalf) {
            nl[i] += kHalfShift;
            dl[i] *= down;
          }
        }
        if (ss >= NS) ok = ok && tc::wait(&bars.q_empty[stage], ((ss / NS) - 1) & 1);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s_stat[stage][0][lane + 32 * i] = nl[i];
          s_stat[stage][1][lane + 32 * i] = dl[i];
        }
        __syncwarp();
        if (lane == 0) tc::arrive(&bars.stat_full[stage]);
      }
    }
  } else if (warp == kWeightWarps) {
    // K Q^T and V dO^T; another warp issues the gradients' products
    constexpr uint32_t id_s = tc::idesc<T>(kRows, false);
    const bool leader = tc::elect_one();
    for (int it = 0; ok; ++it) {
      const int id = take(it, t);
      ok = id != kTimeout;
      if (id < 0) break;
      const Plan p = plan(id, t);
      if (p.steps == 0) continue;
      ok = tc::wait(&bars.kv_full, nk & 1);
      ++nk;
      for (int s = 0; s < p.steps && ok; ++s, ++ss) {
        const uint32_t q = smem + (2 + 2 * (ss % NS)) * L::kTile, g = q + L::kTile;
        ok = tc::wait(&bars.q_full[ss % NS], (ss / NS) & 1);
        // Packed: rows of the next sequence in a tile that reaches past this one; causal behind a mask: rows up to the
        // first valid key, which see none and may hold anything.  In both tensors before anything is made of either.
        const int rows = min(t.n - p.first_of(s), kRows) * f.pack;
        const int blind_rows = min(p.lo - p.first_of(s), kRows) * f.pack;
        if ((a.cu != nullptr && rows < kRows) || blind_rows > 0 || p.scattered) {
          ok = ok && tc::wait(&bars.g_full[ss % NS], (ss / NS) & 1);
          uint32_t w[4], x[4];
          tc::first_bits(rows, w);
          tc::first_bits(blind_rows, x);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] &= ~x[i];
          if (p.scattered) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = lane + 32 * i, tok = p.first_of(s) + r / f.pack;
              w[i] &= __ballot_sync(0xffffffffu, tok < t.n && a.lse[lse_index(a, t, p.head_of(s) + r % f.pack, tok)] != neg_inf());
            }
          }
          if (ok && !tc::all_set(w)) {
            tc::clear_rows<DP / 64>(q, w);
            tc::clear_rows<DP / 64>(g, w);
          }
        }
        // the weights of the step before in this buffer lie there until they are in dV
        if (ss >= NB) ok = ok && tc::wait(&bars.s_free[ss % NB], ((ss / NB) - 1) & 1);
        tc::fence_after();
        if (ok && leader) {
          tc::product_nt<DP>(tmem + (ss % NB) * 128, smem, q, id_s);
          tc::commit(&bars.s_full[ss % NB]);
        }
        __syncwarp();
        ok = ok && tc::wait(&bars.g_full[ss % NS], (ss / NS) & 1);
        if (ss >= 1) ok = ok && tc::wait(&bars.dp_free, (ss - 1) & 1);
        tc::fence_after();
        if (ok && leader) {
          tc::product_nt<DP>(t_dp, smem + L::kTile, g, id_s);
          tc::commit(&bars.dp_full);
          if (s + 1 == p.steps) tc::commit(&bars.kv_empty);
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) atomicExch(&g_tc_bwd_window_error, kDevTimeout);
  } else if (warp == kWeightWarps + 3) {
    constexpr uint32_t id_o = tc::idesc<T>(DP, true);
    const bool leader = tc::elect_one();
    for (int it = 0; ok; ++it) {
      const int id = take(it, t);
      ok = id != kTimeout;
      if (id < 0) break;
      const Plan p = plan(id, t);
      for (int s = 0; s < p.steps && ok; ++s, ++ss) {
        const uint32_t q = smem + (2 + 2 * (ss % NS)) * L::kTile, g = q + L::kTile;
        ok = tc::wait(&bars.p_full[ss & 1], (ss >> 1) & 1) && tc::wait(&bars.g_full[ss % NS], (ss / NS) & 1);
        // the sums of the piece before have been read
        if (s == 0 && nk > 0) ok = ok && tc::wait(&bars.sums_free, (nk - 1) & 1);
        tc::fence_after();
        if (ok && leader) {
          tc::product_tn<32>(t_dv, tmem + (ss % NB) * 128, g, id_o, s > 0);
          if (!kBeside) tc::commit(&bars.s_free[ss % NB]);
        }
        __syncwarp();
        ok = ok && tc::wait(&bars.ds_full[ss & 1], (ss >> 1) & 1);
        tc::fence_after();
        if (ok && leader) {
          tc::product_tn<32>(t_dk, kBeside ? tmem + (ss % NB) * 128 + 16 : t_dp, q, id_o, s > 0);
          tc::commit(kBeside ? &bars.s_free[ss % NB] : &bars.dp_free);
          tc::commit(&bars.q_empty[ss % NS]);
          tc::commit(&bars.g_empty[ss % NS]);  // dO V^T was done before the score gradients
          if (s + 1 == p.steps) tc::commit(&bars.done);
        }
        __syncwarp();
      }
      if (p.steps > 0) ++nk;
    }
    if (!ok && lane == 0) atomicExch(&g_tc_bwd_window_error, kDevTimeout);
  } else {
    const int part = warp >> 2;  // columns [32 part, 32 part + 32) of each tile
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float c2 = a.scale * kLog2e;
    for (int it = 0;; ++it) {
      const int id = ok ? take(it, t) : kTimeout;
      ok = id != kTimeout;
      // all of them go on or none, with the statistics' warp; and what the piece before left in s_most has been read
      if (kHalf) ok = !tc::any_of(2, 32 * (kWeightWarps + 1), !ok);
      if (!ok || id < 0) break;
      const Plan p = plan(id, t);
      const int key = t.first + (warp & 3) * 32 + lane;
      const bool valid = key < t.n && (p.mask == nullptr || mask_key(p.mask, key));
      int unit = 0;
      if constexpr (kHalf) {
        float m[3] = {0.f, 0.f, 0.f};
        if (p.steps > 0) {
          const int from = max(p.row_from, p.lo);  // rows that see a key
          // four heads at a time: one after the other, their loads wait for one another (delta, dK and dV of 8 x 1024 tokens,
          // 32/8 heads of 128: 237 us instead of 225)
          for (int h = 0; h < group; h += 4) {
            const int64_t at = lse_index(a, t, p.h_first + h, 0);
            for (int i = from + static_cast<int>(threadIdx.x); i < p.row_to; i += 32 * kWeightWarps) {
              float g[4], d[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                g[x] = h + x < group ? __ldg(a.g_norm + at + x * a.L + i) : 0.f;
                d[x] = h + x < group ? __ldg(a.delta + at + x * a.L + i) : 0.f;
                // what a row that sees no key holds does not count
                if (p.scattered && h + x < group && __ldg(a.lse + at + x * a.L + i) == neg_inf()) g[x] = d[x] = 0.f;
              }
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                m[0] = fmaxf(m[0], finite(g[x]));
                m[1] = fmaxf(m[1], finite(d[x]));
              }
            }
          }
          m[2] = most_of(a.v_norm + (static_cast<int64_t>(t.batch) * a.Hk + p.hk) * a.L + t.row0, t.first, min(t.n, t.first + kRows));
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          m[i] = warp_max(m[i]);
          if (lane == 0) s_most[i][warp] = m[i];
        }
        __syncwarp();
        unit = unit_of();
      }
      const float up = pow2(unit - static_cast<int>(kHalfShift));
      auto less_delta = [&](float2 dp, float2 neg_delta) {
        if constexpr (kHalf) return fma2(dp, f2(up), neg_delta);
        else return add2(dp, neg_delta);
      };
      const bool all_valid = __all_sync(0xffffffffu, valid);
      // after a wait that ran out a warp goes on without waiting to the end of the piece
      for (int s = 0, first = p.i_lo, left = p.per_head; s < p.steps; ++s, ++ss) {
        // first: the first row of the step's tile
        if (s == 0 || --left == 0) first = p.i_lo * f.tile_tokens, left = p.per_head;
        else first += f.tile_tokens;
        const int stage = ss % NS;
        const uint32_t s_addr = tmem + lanes + (ss % NB) * 128 + part * 32, d_addr = t_dp + lanes + part * 32;
        ok = ok && tc::wait(&bars.stat_full[stage], (ss / NS) & 1) && tc::wait(&bars.s_full[ss % NB], (ss / NB) & 1);
        tc::fence_after();
        uint32_t pr[32], w[16];
        tc::ld32(s_addr, pr);
        // the first row of this part that sees the key, 32 = none, and one past the last
        int from = min(max(max(key - first, -1) * f.pack - part * 32, 0), 32), upto = 32;
        if (!valid) from = 32;
        if (key >= p.sink_end) upto = min(max(min(max(key + a.window - first, 0), f.tile_tokens) * f.pack - part * 32, 0), 32);
        const float4* nl = reinterpret_cast<const float4*>(&s_stat[stage][0][part * 32]);
        const float4* dl = reinterpret_cast<const float4*>(&s_stat[stage][1][part * 32]);
        const bool masked = __any_sync(0xffffffffu, from > 0 || upto < 32);
        tc::wait_ld(pr);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 b = nl[e / 4];
          const float2 x = fma2(make_float2(__uint_as_float(pr[e]), __uint_as_float(pr[e + 1])), f2(c2), make_float2(b.x, b.y));
          const float2 y = fma2(make_float2(__uint_as_float(pr[e + 2]), __uint_as_float(pr[e + 3])), f2(c2), make_float2(b.z, b.w));
          pr[e] = __float_as_uint(ex2(x.x));
          pr[e + 1] = __float_as_uint(ex2(x.y));
          pr[e + 2] = __float_as_uint(ex2(y.x));
          pr[e + 3] = __float_as_uint(ex2(y.y));
        }
        if (masked) {
          const uint32_t see = tc::bits_from(from) & ~tc::bits_from(upto);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((see >> e) & 1u)) pr[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = tc::pack2<T>(__uint_as_float(pr[2 * e]), __uint_as_float(pr[2 * e + 1]));
        tc::st16(s_addr, w);
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::arrive(&bars.p_full[ss & 1]);

        ok = ok && tc::wait(&bars.dp_full, ss & 1);
        tc::fence_after();
        uint32_t d[32];
        tc::ld32(d_addr, d);
        tc::wait_ld(d);
        if (kBeside) {
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::arrive(&bars.dp_free);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 b = dl[e / 4];
          const float2 x = mul2(make_float2(__uint_as_float(pr[e]), __uint_as_float(pr[e + 1])),
                                less_delta(make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), make_float2(b.x, b.y)));
          const float2 y = mul2(make_float2(__uint_as_float(pr[e + 2]), __uint_as_float(pr[e + 3])),
                                less_delta(make_float2(__uint_as_float(d[e + 2]), __uint_as_float(d[e + 3])), make_float2(b.z, b.w)));
          w[e / 2] = tc::pack2<T>(x.x, x.y);
          w[e / 2 + 1] = tc::pack2<T>(y.x, y.y);
        }
        // dO V^T of a key that is not there may be NaN
        if (!all_valid && !valid) {
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = 0u;
        }
        tc::st16(kBeside ? s_addr + 16 : d_addr, w);
        tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::arrive(&bars.ds_full[ss & 1]);
      }
      if (p.steps > 0) {
        ok = ok && tc::wait(&bars.done, nk & 1);
        ++nk;
      }
      tc::fence_after();
      if (!ok) {
        if (lane == 0) atomicExch(&g_tc_bwd_window_error, kDevTimeout);
      } else if (t.first < t.n) {
        const bool live = key < t.n;
        const int c0 = (part & 1) * (DP / 2);  // parts 0, 1: dV, parts 2, 3: dK, half of the columns each
        const uint32_t sums = (part < 2 ? t_dv : t_dk) + lanes + c0;
        float mul = part < 2 ? (kHalf ? kHalfUnit : 1.f) : (kHalf ? a.scale * pow2(-unit) : a.scale);
        const bool first_ones = key >= p.lo && key < p.sink_end;
        const int at = (key - max(t.first, p.lo)) * 2 * DP + (part < 2 ? 0 : DP) + c0;  // in far_at's
        if constexpr (FORM == kFar) {
          if (p.steps > 0) {
            float* to = far_at(p, t, p.row_from / f.chunk) + at;
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
              uint32_t o[16];
              tc::ld16(sums + 16 * c, o);
              tc::wait_ld(o);
              if (first_ones) {
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                  *reinterpret_cast<float4*>(to + 16 * c + e) =
                      make_float4(__uint_as_float(o[e]) * mul, __uint_as_float(o[e + 1]) * mul, __uint_as_float(o[e + 2]) * mul,
                                  __uint_as_float(o[e + 3]) * mul);
              }
            }
          }
        } else {
          if (p.steps > 0 && t.first < p.sink_end && p.far_from < t.n) {
            pdl_wait();  // for the far rows' CTAs
            if (__any_sync(0xffffffffu, first_ones)) {
              // In the gradients' own units, not in the near rows': if those have no gradient theirs is 2^100, and a far
              // sum in it would leave fp32.
#pragma unroll 1
              for (int c = 0; c < DP / 32; ++c) {
                uint32_t o[16];
                tc::ld16(sums + 16 * c, o);
                tc::wait_ld(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * mul);
                if (first_ones) {
                  for (int chunk = p.far_from / f.chunk; chunk * f.chunk < t.n; ++chunk) {
                    const float4* x = reinterpret_cast<const float4*>(far_at(p, t, chunk) + at + 16 * c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      const float4 y = __ldcg(x + e);  // written while this kernel may already be there
                      o[4 * e] = __float_as_uint(__uint_as_float(o[4 * e]) + y.x);
                      o[4 * e + 1] = __float_as_uint(__uint_as_float(o[4 * e + 1]) + y.y);
                      o[4 * e + 2] = __float_as_uint(__uint_as_float(o[4 * e + 2]) + y.z);
                      o[4 * e + 3] = __float_as_uint(__uint_as_float(o[4 * e + 3]) + y.w);
                    }
                  }
                }
                __syncwarp();
                tc::st16(sums + 16 * c, o);
              }
              tc::wait_st();
              mul = 1.f;
            }
          }
          if (part < 2) {
            T* out = static_cast<T*>(a.dv) + t.batch * a.dvs.b + (t.row0 + key) * a.dvs.t + p.hk * a.dvs.h;
            tc::store_rows<T, DP / 2>(sums, out, c0, a.d, mul, live, f.wide_dv, p.steps > 0);
          } else {
            T* out = static_cast<T*>(a.dk) + t.batch * a.dks.b + (t.row0 + key) * a.dks.t + p.hk * a.dks.h;
            tc::store_rows<T, DP / 2>(sums, out, c0, a.d, mul, live, f.wide_dk, p.steps > 0);
          }
        }
      } else if (FORM != kFar && a.cu != nullptr && t.n == 0 && part < 2) {
        T* base = static_cast<T*>(part == 0 ? a.dv : a.dk) + p.hk * (part == 0 ? a.dvs.h : a.dks.h);
        const int64_t st = part == 0 ? a.dvs.t : a.dks.t;
        for (int64_t r = t.row0 + t.tail_index; r < a.L; r += t.tail_count)
          for (int x = threadIdx.x & 127; x < a.d; x += kRows) base[r * st + x] = Elem<T>::from_f(0.f);
      }
      if (p.steps > 0) {
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::arrive(&bars.sums_free);
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kWeightWarps) tc::dealloc(tmem, 512);
  if (FORM == kNear) pdl_wait();  // launched beside the far rows; dQ's wait for this kernel's end covers them
}

int64_t count_tiles(AttnArgs& a, int rows) {
  if (a.cu != nullptr) {
    a.tiles = static_cast<int>(packed_tiles(a.L, a.nseq, rows));
    return a.tiles;
  }
  a.tiles = static_cast<int>((a.L + rows - 1) / rows);
  return static_cast<int64_t>(a.tiles) * a.nseq;
}

template <typename T, int DP>
cudaError_t run(const CUtensorMap& q, const CUtensorMap& g, const CUtensorMap& k, const CUtensorMap& v, BwdArgs f,
                cudaStream_t st) {
  if (f.a.dk != nullptr) {
    if (f.far != nullptr) {
      const int64_t tiles = count_tiles(f.a, f.chunk);
      const cudaError_t e = launch_grid<attn_tc_window_dkv_kernel<T, DP, kFar>>(false, tiles * f.sink_tiles * f.a.Hk, kThreads,
                                                                                Layout<DP>::kSmemKv, st, q, g, k, v, f);
      if (e != cudaSuccess) return e;
    }
    const int64_t tiles = count_tiles(f.a, kRows);
    const cudaError_t e = launch_grid<attn_tc_window_dkv_kernel<T, DP, kNear>>(f.far != nullptr, tiles * f.a.Hk, kThreads,
                                                                               Layout<DP>::kSmemKv, st, q, g, k, v, f);
    if (e != cudaSuccess) return e;
  }
  if (f.a.dq == nullptr) return cudaSuccess;
  const int64_t tiles = count_tiles(f.a, f.tile_tokens);
  return launch_grid<attn_tc_window_dq_kernel<T, DP>>(f.a.dk != nullptr, tiles * (f.a.H / f.pack), kThreads,
                                                      Layout<DP>::kSmem, st, q, g, k, v, f);
}

template <typename T>
cudaError_t dispatch(const CUtensorMap& q, const CUtensorMap& g, const CUtensorMap& k, const CUtensorMap& v, const BwdArgs& f,
                     cudaStream_t st) {
  return f.a.d <= 64 ? run<T, 64>(q, g, k, v, f, st) : run<T, 128>(q, g, k, v, f, st);
}

int far_sink_tiles(const AttnArgs& a) { return a.mask != nullptr ? (a.sinks + kRows - 2) / kRows + 1 : (a.sinks + kRows - 1) / kRows; }
int64_t far_bytes_of(const AttnArgs& a, int64_t chunk) {
  return far_places(a, kRows, chunk) * far_sink_tiles(a) * a.Hk * std::min(a.sinks, kRows) * 2 * (a.d <= 64 ? 64 : 128) * static_cast<int64_t>(sizeof(float));
}
// Rows of a far CTA: about as many as the others' windows; more where there would be more than 64 parts in a row, or
// more than 256 MB of them.
int far_chunk(const AttnArgs& a) {
  int64_t rows = std::max<int64_t>(std::max<int64_t>(a.window + kRows, 512), (a.L + 63) / 64);
  rows = (rows + kRows - 1) / kRows * kRows;
  while (rows < a.L && far_bytes_of(a, rows) > (256LL << 20)) rows *= 2;
  return static_cast<int>(rows);
}

}  // namespace

bool launch_attn_tc_bwd_window(const AttnArgs& a, int dtype, void* far, cudaStream_t st, cudaError_t* e) {
  if (dtype == kF32 || a.d % 8 != 0 || a.d > 128 || !(a.scale > 0.f) || (dtype == kF16 && a.g_norm == nullptr)) return false;
  BwdArgs f = {};
  f.a = a;
  f.pack = attn_pack(a.H / a.Hk);
  f.tile_tokens = kRows / f.pack;
  f.warp_span = 31 / f.pack;
  const int64_t nb = a.cu != nullptr ? 1 : a.nseq;
  CUtensorMap q, g, k, v;
  if (!attn_map(&q, a.q, dtype, nb, a.L, a.H, a.d, a.qs, f.pack, f.tile_tokens) ||
      !attn_map(&g, a.g, dtype, nb, a.L, a.H, a.d, a.gs, f.pack, f.tile_tokens) ||
      !attn_map(&k, a.k, dtype, nb, a.L, a.Hk, a.d, a.ks, 1, kRows) ||
      !attn_map(&v, a.v, dtype, nb, a.L, a.Hk, a.d, a.vs, 1, kRows))
    return false;
  f.wide_dq = row_alignment(a.dq, a.dqs, nb, a.H);
  f.wide_dk = row_alignment(a.dk, a.dks, nb, a.Hk);
  f.wide_dv = row_alignment(a.dv, a.dvs, nb, a.Hk);
  if (far_bytes(a, dtype) > 0 && a.dk != nullptr) {
    f.far = static_cast<float*>(far);
    f.chunk = far_chunk(a);
    f.sink_tiles = far_sink_tiles(a);
    f.far_keys = std::min(a.sinks, kRows);
  }
  *e = dtype == kBF16 ? dispatch<__nv_bfloat16>(q, g, k, v, f, st) : dispatch<__half>(q, g, k, v, f, st);
  return true;
}

int64_t far_bytes(const AttnArgs& a, int dtype) {
  // no row lies behind the window of a whole tile
  if (a.window == 0 || a.sinks == 0 || a.L < a.window + kRows || dtype == kF32 || a.d % 8 != 0 || a.d > 128) return 0;
  return far_bytes_of(a, far_chunk(a));
}

int read_device_error_tc_bwd_window(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_tc_bwd_window_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_tc_bwd_window_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace cta
