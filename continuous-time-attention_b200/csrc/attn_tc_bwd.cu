// Attention backward on the tensor cores, 16-bit tensors.
//
//   P = exp(c Q K^T - lse),  dS = P o (dO V^T - delta)
//   dQ = c dS K,   dK = c dS^T Q,   dV = P^T dO
//
// Two kernels, one that owns 128 query rows (dQ) and one that owns 128 keys (dK,
// dV).  Both recompute the scores, so seven products of a tile pair are done
// where five would do; in exchange every gradient has one owner that sums in
// tensor memory in a fixed order: no atomics, no fp32 scratch for dQ, results
// that do not depend on timing, and the heads that share keys are summed in
// place.  Rows are (token, head) pairs as in the forward.
//
//   warps 0-15  weights: four warpgroups take 32 columns each of a 128 x 128 tile
//   warp 16  MMAs of the scores and of dO V^T    warp 17  TMA loads
//   dQ:      warp 18  MMAs of dQ
//   dK, dV:  warp 18  lse and delta              warp 19  MMAs of dV and dK
//
// Weights and score gradients go back to tensor memory as 16-bit A operands over
// the columns their fp32 sources came from, so a tile pair crosses shared memory
// only as Q, K, V and dO.  The next scores run while dS is computed, the next
// dO V^T while the next P is.
//
// Bound by the products at dim 128 (7 x 512 cycles per tile pair against 2 x
// 1024 of exponentials), by the exponentials at dim 64.  Measured, 8192 tokens, 16
// heads, not causal, bf16: dim 128 dQ 658 us, dK and dV 990, 1170 TFLOP/s of the seven
// products; dim 64 406 and 537, 1020.  Both in one call, delta included, take 1655 and
// 941: dQ's CTAs start while the last ones of dK and dV run.  fp16, with its bounds,
// 1678 and 976.
#include <algorithm>

#include "attn_tc.cuh"

namespace cta {

__device__ int g_tc_bwd_error;

namespace {

constexpr int kThreads = 640;  // five warpgroups; the last has a warp or two to spare
constexpr int kWeightWarps = 16;
constexpr int kRows = 128;
// In fp16 the P of dV carries 2^14: of thousands of keys it would lie among the type's subnormal numbers (one of
// 41891 equal weights was 1.2e-3 off), and with 2^14 what is lost is below 2^-39.  P is at most 1, but for the
// rounding of scores and lse.
constexpr float kHalfShift = 14.f, kHalfUnit = 0x1p-14f;

// fp16 holds nothing below 2^-25, and dS of thousands of keys lies there as soon as the output's gradient is small,
// while its sums dQ and dK do not.  So dS is multiplied by the power of two that takes its bound, |g| |v| + |delta|,
// to 2^14..2^15 (dQ: row by row; dK, dV: for all rows that meet the CTA's keys), and the sums are multiplied back: what
// is lost of a dS is below 2^-39 of that bound.  The attn_delta_kernel leaves the norms.
__device__ __forceinline__ int unit_exponent(float bound) {
  return max(-100, min(100, 14 + 127 - static_cast<int>(__float_as_uint(bound) >> 23)));
}
__device__ __forceinline__ float pow2(int n) { return __uint_as_float(static_cast<uint32_t>(127 + n) << 23); }
__device__ __forceinline__ float finite(float x) { return fabsf(x) < __int_as_float(0x7f800000) ? fabsf(x) : 0.f; }
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
// maximum of |x| over [begin, end), by the weight warps; each thread gets its share's
__device__ __forceinline__ float most_of(const float* x, int begin, int end) {
  float m = 0.f;
#pragma unroll 4
  for (int i = begin + static_cast<int>(threadIdx.x); i < end; i += 32 * kWeightWarps) m = fmaxf(m, finite(__ldg(x + i)));
  return m;
}

struct BwdArgs {
  AttnArgs a;
  int pack, tile_tokens;
  int wide_dq, wide_dk, wide_dv;  // alignment of the gradients' rows, see store_rows
};

template <int DP>
struct Layout {
  static constexpr int kHalf = kRows * 128;
  static constexpr int kTile = kHalf * (DP / 64);
  // tiles of the other side in flight: a key tile is held until its dQ is done, and with four of 32 KB
  // the next but one came too late (dQ at 8192 keys, 16 heads of 128: 4090 cycles a step)
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kStages) * kTile + 1024;
  static constexpr int kPairs = DP == 128 ? 2 : 4;  // (Q, dO) pairs of the keys' kernel
  static constexpr int kSmemKv = (2 + 2 * kPairs) * kTile + 1024;
};

// the row's share of the sums: a row that sees no key, or lies outside, has weight zero everywhere
__device__ __forceinline__ bool blind(float neg_lse2) { return neg_lse2 == neg_inf(); }
__device__ __forceinline__ float neg_lse2_of(float lse) { return lse == neg_inf() ? neg_inf() : -lse * kLog2e; }

// ---------------------------------------------------------------------------
// dQ
// ---------------------------------------------------------------------------
struct DqBars {
  uint64_t q_full, kv_full[8], kv_empty[8], s_full[2], s_free[2], dp_full, dp_read, ds_full[2], done;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_dq_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap gmap,
                      const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ BwdArgs f) {
  using L = Layout<DP>;
  constexpr int NS = L::kStages;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  __shared__ DqBars bars;
  __shared__ float s_most[kHalf ? kWeightWarps : 1];
  __shared__ uint32_t s_tmem;
  __shared__ SeqTile s_tile;
  const AttnArgs& a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const int blocks = a.H / f.pack;
  const int h0 = static_cast<int>(blockIdx.x % blocks) * f.pack, hk = h0 / (a.H / a.Hk);

  if (warp == 0) {
    const SeqTile x = find_tile(a.cu, a.nseq, a.L, a.tiles, blockIdx.x / blocks, f.tile_tokens, a.causal,
                                a.causal || a.cu != nullptr);
    if (lane == 0) s_tile = x;
  } else if (warp == kWeightWarps) {
    tc::alloc(&s_tmem, 512);
  } else if (warp == kWeightWarps + 1 && lane == 0) {
    mbar_init(&bars.q_full, 1);
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
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const SeqTile t = s_tile;
  const uint32_t tmem = s_tmem;
  const uint32_t t_dp = tmem + 256, t_dq = tmem + 384;  // scores: columns 0 and 128

  int lo = 0, hi = t.n;
  mask_range(a, t.batch, t.n, lo, hi);
  const uint32_t* mask = a.mask != nullptr ? a.mask + t.batch * a.mask_words : nullptr;
  const int j_lo = lo / kRows;
  int end = hi;
  if (a.causal) end = min(end, t.first + f.tile_tokens);
  const int steps = t.first < t.n ? max(0, (end + kRows - 1) / kRows - j_lo) : 0;

  auto key_words = [&](int j, uint32_t (&w)[4]) {
    const int j0 = (j_lo + j) * kRows;
    tc::first_bits(t.n - j0, w);
    if (mask != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (w[i] != 0u) w[i] &= __ldg(mask + kMaskHead + (j0 >> 5) + i);
    }
  };

  if (warp == kWeightWarps + 1) {
    bool ok = true;
    int issued = 0;
    if (steps > 0 && lane == 0) {
      mbar_arrive_expect_tx(&bars.q_full, 2 * L::kTile);
      for (int c = 0; c < DP / 64; ++c) {
        tc::tma_load_4d(smem + c * L::kHalf, &qmap, &bars.q_full, 64 * c, h0, static_cast<int>(t.row0) + t.first,
                        t.batch);
        tc::tma_load_4d(smem + L::kTile + c * L::kHalf, &gmap, &bars.q_full, 64 * c, h0,
                        static_cast<int>(t.row0) + t.first, t.batch);
      }
    }
    for (int x = 0; x < 2 * steps; ++x) {
      const int stage = x % NS;
      if (x >= NS) ok = tc::wait(&bars.kv_empty[stage], ((x / NS) - 1) & 1);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars.kv_full[stage], L::kTile);
        for (int c = 0; c < DP / 64; ++c)
          tc::tma_load_4d(smem + (2 + stage) * L::kTile + c * L::kHalf, (x & 1) ? &vmap : &kmap, &bars.kv_full[stage],
                          64 * c, hk, static_cast<int>(t.row0) + (j_lo + (x >> 1)) * kRows, t.batch);
      }
      issued = x + 1;
    }
    if (!ok) {
      atomicExch(&g_tc_bwd_error, kDevTimeout);
      for (int x = max(0, issued - NS); x < issued; ++x) tc::wait(&bars.kv_full[x % NS], (x / NS) & 1);
    }
  } else if (warp == kWeightWarps) {
    // scores and dO V^T; another warp issues dQ: every wait takes a hundred cycles or two, and one warp
    // for all three was what the steps waited for
    constexpr uint32_t id_s = tc::idesc<T>(kRows, false);
    const bool leader = tc::elect_one();
    bool ok = steps == 0 || tc::wait(&bars.q_full, 0);
    for (int j = 0; j < steps && ok; ++j) {
      const uint32_t k = smem + (2 + (2 * j) % NS) * L::kTile, v = smem + (2 + (2 * j + 1) % NS) * L::kTile;
      ok = tc::wait(&bars.kv_full[(2 * j) % NS], ((2 * j) / NS) & 1);
      if (ok && (mask != nullptr || (j_lo + j + 1) * kRows > t.n)) {
        uint32_t w[4];
        key_words(j, w);
        if (!tc::all_set(w)) tc::clear_rows<DP / 64>(k, w);
      }
      // the score gradients of step j - 2 lie in the buffer until they are in dQ
      if (j >= 2) ok = ok && tc::wait(&bars.s_free[j & 1], ((j >> 1) - 1) & 1);
      tc::fence_after();
      if (ok && leader) {
        tc::product_nt<DP>(tmem + (j & 1) * 128, smem, k, id_s);
        tc::commit(&bars.s_full[j & 1]);
      }
      __syncwarp();
      ok = ok && tc::wait(&bars.kv_full[(2 * j + 1) % NS], ((2 * j + 1) / NS) & 1);
      if (j >= 1) ok = ok && tc::wait(&bars.dp_read, (j - 1) & 1);
      tc::fence_after();
      if (ok && leader) {
        tc::product_nt<DP>(t_dp, smem + L::kTile, v, id_s);
        tc::commit(&bars.dp_full);
        tc::commit(&bars.kv_empty[(2 * j + 1) % NS]);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicExch(&g_tc_bwd_error, kDevTimeout);
  } else if (warp == kWeightWarps + 2) {
    constexpr uint32_t id_o = tc::idesc<T>(DP, true);
    const bool leader = tc::elect_one();
    bool ok = true;
    for (int j = 0; j < steps && ok; ++j) {
      ok = tc::wait(&bars.ds_full[j & 1], (j >> 1) & 1);
      tc::fence_after();
      if (ok && leader) {
        tc::product_tn<32>(t_dq, tmem + (j & 1) * 128, smem + (2 + (2 * j) % NS) * L::kTile, id_o, j > 0);
        tc::commit(&bars.s_free[j & 1]);
        tc::commit(&bars.kv_empty[(2 * j) % NS]);
        if (j + 1 == steps) tc::commit(&bars.done);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicExch(&g_tc_bwd_error, kDevTimeout);
  } else if (warp < kWeightWarps) {
    const int part = warp >> 2;  // columns [32 part, 32 part + 32) of each tile
    const int row = (warp & 3) * 32 + lane;
    const int tok = t.first + row / f.pack, h = h0 + row % f.pack;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool live = tok < t.n;
    const float c2 = a.scale * kLog2e;
    // all of these loads are on their way before the first is used
    const int64_t at = live ? lse_index(a, t, h, tok) : 0;
    const float lse = live ? a.lse[at] : neg_inf(), delta = live ? a.delta[at] : 0.f;
    float norm = 0.f, most = 0.f;
    if constexpr (kHalf) {
      norm = live ? a.g_norm[at] : 0.f;
      if (steps > 0) most = most_of(a.v_norm + (static_cast<int64_t>(t.batch) * a.Hk + hk) * a.L + t.row0, lo, end);
    }
    const float nl = neg_lse2_of(lse);
    const bool none = blind(nl);
    const int limit = a.causal ? tok : t.n - 1;
    const int limit_all = t.first + (warp & 3) * 32 / f.pack;  // causal: last key all rows of the warp see
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
    bool ok = true;
    for (int j = 0; j < steps && ok; ++j) {
      const uint32_t s_addr = tmem + lanes + (j & 1) * 128 + part * 32;
      ok = tc::wait(&bars.s_full[j & 1], (j >> 1) & 1);
      if (!ok) break;
      tc::fence_after();
      uint32_t s[32], dp[32];
      tc::ld32(s_addr, s);
      const int j0 = (j_lo + j) * kRows;
      bool whole = j0 + kRows <= t.n && !any_blind && (!a.causal || j0 + kRows - 1 <= limit_all);
      uint32_t w[4];
      if (mask != nullptr || !whole) {
        key_words(j, w);
        whole = whole && tc::all_set(w);
      }
      tc::wait_ld(s);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), f2(c2), f2(nl));
        s[e] = __float_as_uint(ex2(x.x));
        s[e + 1] = __float_as_uint(ex2(x.y));
      }
      ok = tc::wait(&bars.dp_full, j & 1);
      if (!ok) break;
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
        const uint32_t see = (part == 0 ? w[0] : part == 1 ? w[1] : part == 2 ? w[2] : w[3]) &
                             (left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u);
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
      if (lane == 0) tc::arrive(&bars.ds_full[j & 1]);
    }
    if (ok && steps > 0) ok = tc::wait(&bars.done, 0);
    tc::fence_after();
    if (!ok) {
      if (lane == 0) atomicExch(&g_tc_bwd_error, kDevTimeout);
    } else if (t.first < t.n) {
      T* out = static_cast<T*>(a.dq) + t.batch * a.dqs.b + (t.row0 + tok) * a.dqs.t + h * a.dqs.h;
      tc::store_rows<T, DP / 4>(t_dq + lanes + part * (DP / 4), out, part * (DP / 4), a.d, kHalf ? a.scale * pow2(-unit) : a.scale, live, f.wide_dq,
                                    steps > 0);
    } else if (a.cu != nullptr && t.n == 0 && part == 0) {
      for (int64_t r = t.row0 + t.tail_index; r < a.L; r += t.tail_count)
        for (int x = threadIdx.x; x < a.d * f.pack; x += kRows)
          static_cast<T*>(a.dq)[r * a.dqs.t + (h0 + x / a.d) * a.dqs.h + x % a.d] = Elem<T>::from_f(0.f);
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kWeightWarps) tc::dealloc(tmem, 512);
  pdl_wait();  // launched beside dK and dV
}

// ---------------------------------------------------------------------------
// dK, dV: the tiles are transposed, rows are keys and columns are query rows
// ---------------------------------------------------------------------------
struct DkvBars {
  uint64_t kv_full, q_full[4], q_empty[4], g_full[4], g_empty[4], stat_full[4], s_full[2], s_free[2], p_full[2], dp_full, dp_free, ds_full[2], done;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_dkv_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap gmap,
                       const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ BwdArgs f) {
  using L = Layout<DP>;
  constexpr int NS = L::kPairs;  // (Q, dO) pairs in flight
  extern __shared__ uint8_t smem_raw[];
  __shared__ DkvBars bars;
  __shared__ uint32_t s_tmem;
  __shared__ SeqTile s_tile;
  __shared__ __align__(16) float s_stat[NS][2][kRows];  // [stage][-lse2, -delta, fp16: + 14, * its unit][row]
  const AttnArgs& a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
  // With two score buffers dS goes beside P, into the columns that P leaves of its scores', and the next dO V^T can
  // start once this one has been read; with one it goes over dO V^T, so that the next scores wait for dV only.
  constexpr bool kBeside = DP == 64;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  __shared__ float s_most[kHalf ? 3 : 1][kHalf ? kWeightWarps : 1];  // |g|, |delta|, |v|
  const int hk = blockIdx.x % a.Hk, group = a.H / a.Hk;
  pdl_launch_dependents();  // dQ's CTAs may follow

  if (warp == 0) {
    // the first keys of a causal sequence meet the most rows: forwards is heaviest first
    const SeqTile x = find_tile(a.cu, a.nseq, a.L, a.tiles, blockIdx.x / a.Hk, kRows, false,
                                a.causal || a.cu != nullptr);
    if (lane == 0) s_tile = x;
  } else if (warp == kWeightWarps) {
    tc::alloc(&s_tmem, 512);
  } else if (warp == kWeightWarps + 1 && lane == 0) {
    mbar_init(&bars.kv_full, 1);
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
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const SeqTile t = s_tile;
  const uint32_t tmem = s_tmem;
  // Scores: one buffer of 128 columns at dim 128, where the four accumulators fill tensor memory, two at 64
  constexpr int NB = DP == 64 ? 2 : 1;
  const uint32_t t_dp = tmem + NB * 128, t_dv = t_dp + 128, t_dk = t_dv + DP;

  const uint32_t* mask = a.mask != nullptr ? a.mask + t.batch * a.mask_words : nullptr;
  int lo, hi;
  mask_range(a, t.batch, t.n, lo, hi);
  // row tiles that meet these keys, for each block of heads of the group
  const int i_lo = a.causal ? t.first / f.tile_tokens : 0;
  const int per_head = max(0, (t.n + f.tile_tokens - 1) / f.tile_tokens - i_lo);
  const bool some = t.first < min(t.n, hi) && t.first + kRows > lo;  // any valid key
  const int steps = some ? per_head * (group / f.pack) : 0;
  auto head_of = [&](int s) { return hk * group + s / per_head * f.pack; };
  auto first_of = [&](int s) { return (i_lo + s % per_head) * f.tile_tokens; };

  // fp16: the exponent of the CTA's power of two; the weight warps and the warp of the statistics
  auto unit_of = [&] {
    tc::sync_of(1, 32 * (kWeightWarps + 1));
    const int w = kHalf ? lane % kWeightWarps : 0;
    return unit_exponent(warp_max(s_most[0][w]) * warp_max(s_most[kHalf ? 2 : 0][w]) + warp_max(s_most[kHalf ? 1 : 0][w]));
  };

  if (warp == kWeightWarps + 1) {
    bool ok = true;
    int issued = 0;
    if (steps > 0 && lane == 0) {
      mbar_arrive_expect_tx(&bars.kv_full, 2 * L::kTile);
      for (int c = 0; c < DP / 64; ++c) {
        tc::tma_load_4d(smem + c * L::kHalf, &kmap, &bars.kv_full, 64 * c, hk, static_cast<int>(t.row0) + t.first,
                        t.batch);
        tc::tma_load_4d(smem + L::kTile + c * L::kHalf, &vmap, &bars.kv_full, 64 * c, hk,
                        static_cast<int>(t.row0) + t.first, t.batch);
      }
    }
    for (int x = 0; x < 2 * steps; ++x) {
      // Q and dO of a step by turns, each given back when its last product is done
      const int s = x >> 1, stage = s % NS;
      uint64_t* full = (x & 1) ? &bars.g_full[stage] : &bars.q_full[stage];
      if (s >= NS) ok = tc::wait((x & 1) ? &bars.g_empty[stage] : &bars.q_empty[stage], ((s / NS) - 1) & 1);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(full, L::kTile);
        for (int c = 0; c < DP / 64; ++c)
          tc::tma_load_4d(smem + (2 + 2 * stage + (x & 1)) * L::kTile + c * L::kHalf, (x & 1) ? &gmap : &qmap, full, 64 * c,
                          head_of(s), static_cast<int>(t.row0) + first_of(s), t.batch);
      }
      issued = x + 1;
    }
    if (!ok) {
      atomicExch(&g_tc_bwd_error, kDevTimeout);
      for (int x = max(0, issued - 2 * NS); x < issued; ++x)
        tc::wait((x & 1) ? &bars.g_full[(x >> 1) % NS] : &bars.q_full[(x >> 1) % NS], ((x >> 1) / NS) & 1);
    }
  } else if (warp == kWeightWarps + 2) {
    bool ok = true;
    float down = 1.f;
    if constexpr (kHalf) down = pow2(unit_of() - static_cast<int>(kHalfShift));
    for (int s = 0; s < steps; ++s) {
      const int stage = s % NS;
      float nl[4], dl[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = lane + 32 * i;
        const int tok = first_of(s) + r / f.pack, h = head_of(s) + r % f.pack;
        nl[i] = tok < t.n ? neg_lse2_of(__ldg(a.lse + lse_index(a, t, h, tok))) : neg_inf();
        dl[i] = tok < t.n ? -__ldg(a.delta + lse_index(a, t, h, tok)) : 0.f;
        if (blind(nl[i])) dl[i] = 0.f;
        if constexpr (kHalf) {
          nl[i] += kHalfShift;
          dl[i] *= down;
        }
      }
      if (s >= NS) ok = tc::wait(&bars.q_empty[stage], ((s / NS) - 1) & 1);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s_stat[stage][0][lane + 32 * i] = nl[i];
        s_stat[stage][1][lane + 32 * i] = dl[i];
      }
      __syncwarp();
      if (lane == 0) tc::arrive(&bars.stat_full[stage]);
    }
  } else if (warp == kWeightWarps) {
    // K Q^T and V dO^T; another warp issues the gradients' products
    constexpr uint32_t id_s = tc::idesc<T>(kRows, false);
    const bool leader = tc::elect_one();
    bool ok = steps == 0 || tc::wait(&bars.kv_full, 0);
    for (int s = 0; s < steps && ok; ++s) {
      const uint32_t q = smem + (2 + 2 * (s % NS)) * L::kTile, g = q + L::kTile;
      ok = tc::wait(&bars.q_full[s % NS], (s / NS) & 1);
      // Packed: rows of the next sequence in a tile that reaches past this one; causal behind a mask: rows up to the
      // first valid key, which see none and may hold anything.  In both tensors before anything is made of either.
      const int rows = min(t.n - first_of(s), kRows) * f.pack;
      const int blind_rows = a.causal ? min(lo - first_of(s), kRows) * f.pack : 0;
      if ((a.cu != nullptr && rows < kRows) || blind_rows > 0) {
        ok = ok && tc::wait(&bars.g_full[s % NS], (s / NS) & 1);
        uint32_t w[4], x[4];
        tc::first_bits(rows, w);
        tc::first_bits(blind_rows, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] &= ~x[i];
        if (ok) {
          tc::clear_rows<DP / 64>(q, w);
          tc::clear_rows<DP / 64>(g, w);
        }
      }
      // the weights of the step before in this buffer lie there until they are in dV
      if (s >= NB) ok = ok && tc::wait(&bars.s_free[s % NB], ((s / NB) - 1) & 1);
      tc::fence_after();
      if (ok && leader) {
        tc::product_nt<DP>(tmem + (s % NB) * 128, smem, q, id_s);
        tc::commit(&bars.s_full[s % NB]);
      }
      __syncwarp();
      ok = ok && tc::wait(&bars.g_full[s % NS], (s / NS) & 1);
      if (s >= 1) ok = ok && tc::wait(&bars.dp_free, (s - 1) & 1);
      tc::fence_after();
      if (ok && leader) {
        tc::product_nt<DP>(t_dp, smem + L::kTile, g, id_s);
        tc::commit(&bars.dp_full);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicExch(&g_tc_bwd_error, kDevTimeout);
  } else if (warp == kWeightWarps + 3) {
    constexpr uint32_t id_o = tc::idesc<T>(DP, true);
    const bool leader = tc::elect_one();
    bool ok = true;
    for (int s = 0; s < steps && ok; ++s) {
      const uint32_t q = smem + (2 + 2 * (s % NS)) * L::kTile, g = q + L::kTile;
      ok = tc::wait(&bars.p_full[s & 1], (s >> 1) & 1) && tc::wait(&bars.g_full[s % NS], (s / NS) & 1);
      tc::fence_after();
      if (ok && leader) {
        tc::product_tn<32>(t_dv, tmem + (s % NB) * 128, g, id_o, s > 0);
        if (!kBeside) tc::commit(&bars.s_free[s % NB]);
      }
      __syncwarp();
      ok = ok && tc::wait(&bars.ds_full[s & 1], (s >> 1) & 1);
      tc::fence_after();
      if (ok && leader) {
        tc::product_tn<32>(t_dk, kBeside ? tmem + (s % NB) * 128 + 16 : t_dp, q, id_o, s > 0);
        tc::commit(kBeside ? &bars.s_free[s % NB] : &bars.dp_free);
        tc::commit(&bars.q_empty[s % NS]);
        tc::commit(&bars.g_empty[s % NS]);  // dO V^T was done before the score gradients
        if (s + 1 == steps) tc::commit(&bars.done);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicExch(&g_tc_bwd_error, kDevTimeout);
  } else if (warp < kWeightWarps) {
    const int part = warp >> 2;  // columns [32 part, 32 part + 32) of each tile
    const int key = t.first + (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool valid = key < t.n && (mask == nullptr || mask_key(mask, key));
    const float c2 = a.scale * kLog2e;
    int unit = 0;
    if constexpr (kHalf) {
      float m[3] = {0.f, 0.f, 0.f};
      if (steps > 0) {
        const int from = a.causal ? max(t.first, lo) : 0;  // rows that see a key
        // four heads at a time: one after the other, their loads wait for one another (delta, dK and dV of 8 x 1024 tokens,
        // 32/8 heads of 128: 237 us instead of 225)
        for (int h = 0; h < group; h += 4) {
          const int64_t at = lse_index(a, t, hk * group + h, 0);
          for (int i = from + static_cast<int>(threadIdx.x); i < t.n; i += 32 * kWeightWarps) {
            float g[4], d[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              g[x] = h + x < group ? __ldg(a.g_norm + at + x * a.L + i) : 0.f;
              d[x] = h + x < group ? __ldg(a.delta + at + x * a.L + i) : 0.f;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              m[0] = fmaxf(m[0], finite(g[x]));
              m[1] = fmaxf(m[1], finite(d[x]));
            }
          }
        }
        m[2] = most_of(a.v_norm + (static_cast<int64_t>(t.batch) * a.Hk + hk) * a.L + t.row0, t.first, min(t.n, t.first + kRows));
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
    bool ok = true;
    for (int s = 0; s < steps && ok; ++s) {
      const int stage = s % NS;
      const uint32_t s_addr = tmem + lanes + (s % NB) * 128 + part * 32, d_addr = t_dp + lanes + part * 32;
      ok = tc::wait(&bars.stat_full[stage], (s / NS) & 1) && tc::wait(&bars.s_full[s % NB], (s / NB) & 1);
      if (!ok) break;
      tc::fence_after();
      uint32_t p[32], w[16];
      tc::ld32(s_addr, p);
      // causal: the first row of this part that sees the key; 32 = none
      int from = 0;
      if (a.causal) from = min(max(max(key - first_of(s), -1) * f.pack - part * 32, 0), 32);
      if (!valid) from = 32;
      const float4* nl = reinterpret_cast<const float4*>(&s_stat[stage][0][part * 32]);
      const float4* dl = reinterpret_cast<const float4*>(&s_stat[stage][1][part * 32]);
      const bool masked = __any_sync(0xffffffffu, from > 0);
      tc::wait_ld(p);
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 b = nl[e / 4];
        const float2 x = fma2(make_float2(__uint_as_float(p[e]), __uint_as_float(p[e + 1])), f2(c2), make_float2(b.x, b.y));
        const float2 y = fma2(make_float2(__uint_as_float(p[e + 2]), __uint_as_float(p[e + 3])), f2(c2), make_float2(b.z, b.w));
        p[e] = __float_as_uint(ex2(x.x));
        p[e + 1] = __float_as_uint(ex2(x.y));
        p[e + 2] = __float_as_uint(ex2(y.x));
        p[e + 3] = __float_as_uint(ex2(y.y));
      }
      if (masked) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (e < from) p[e] = 0u;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) w[e] = tc::pack2<T>(__uint_as_float(p[2 * e]), __uint_as_float(p[2 * e + 1]));
      tc::st16(s_addr, w);
      tc::wait_st();
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::arrive(&bars.p_full[s & 1]);

      ok = tc::wait(&bars.dp_full, s & 1);
      if (!ok) break;
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
        const float2 x = mul2(make_float2(__uint_as_float(p[e]), __uint_as_float(p[e + 1])),
                              less_delta(make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])), make_float2(b.x, b.y)));
        const float2 y = mul2(make_float2(__uint_as_float(p[e + 2]), __uint_as_float(p[e + 3])),
                              less_delta(make_float2(__uint_as_float(d[e + 2]), __uint_as_float(d[e + 3])), make_float2(b.z, b.w)));
        w[e / 2] = tc::pack2<T>(x.x, x.y);
        w[e / 2 + 1] = tc::pack2<T>(y.x, y.y);
      }
      if (masked) {
        // dO V^T of a key that is not there may be NaN
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (2 * e < from) w[e] &= 0xffff0000u;
          if (2 * e + 1 < from) w[e] &= 0x0000ffffu;
        }
      }
      tc::st16(kBeside ? s_addr + 16 : d_addr, w);
      tc::wait_st();
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::arrive(&bars.ds_full[s & 1]);
    }
    if (ok && steps > 0) ok = tc::wait(&bars.done, 0);
    tc::fence_after();
    if (!ok) {
      if (lane == 0) atomicExch(&g_tc_bwd_error, kDevTimeout);
    } else if (t.first < t.n) {
      const bool live = key < t.n;
      const int c0 = (part & 1) * (DP / 2);  // parts 0, 1: dV, parts 2, 3: dK, half of the columns each
      if (part < 2) {
        T* out = static_cast<T*>(a.dv) + t.batch * a.dvs.b + (t.row0 + key) * a.dvs.t + hk * a.dvs.h;
        tc::store_rows<T, DP / 2>(t_dv + lanes + c0, out, c0, a.d, kHalf ? kHalfUnit : 1.f, live, f.wide_dv, steps > 0);
      } else {
        T* out = static_cast<T*>(a.dk) + t.batch * a.dks.b + (t.row0 + key) * a.dks.t + hk * a.dks.h;
        tc::store_rows<T, DP / 2>(t_dk + lanes + c0, out, c0, a.d, kHalf ? a.scale * pow2(-unit) : a.scale, live, f.wide_dk, steps > 0);
      }
    } else if (a.cu != nullptr && t.n == 0 && part < 2) {
      T* base = static_cast<T*>(part == 0 ? a.dv : a.dk) + hk * (part == 0 ? a.dvs.h : a.dks.h);
      const int64_t st = part == 0 ? a.dvs.t : a.dks.t;
      for (int64_t r = t.row0 + t.tail_index; r < a.L; r += t.tail_count)
        for (int x = threadIdx.x & 127; x < a.d; x += kRows) base[r * st + x] = Elem<T>::from_f(0.f);
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kWeightWarps) tc::dealloc(tmem, 512);
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
    const int64_t tiles = count_tiles(f.a, kRows);
    const cudaError_t e =
        launch_grid<attn_tc_dkv_kernel<T, DP>>(false, tiles * f.a.Hk, kThreads, Layout<DP>::kSmemKv, st, q, g, k, v, f);
    if (e != cudaSuccess) return e;
  }
  if (f.a.dq == nullptr) return cudaSuccess;
  const int64_t tiles = count_tiles(f.a, f.tile_tokens);
  return launch_grid<attn_tc_dq_kernel<T, DP>>(f.a.dk != nullptr, tiles * (f.a.H / f.pack), kThreads, Layout<DP>::kSmem,
                                               st, q, g, k, v, f);
}

}  // namespace

bool launch_attn_tc_bwd(const AttnArgs& a, int dtype, cudaStream_t st, cudaError_t* e) {
  if (dtype == kF32 || a.d % 8 != 0 || a.d > 128 || !(a.scale > 0.f) || (dtype == kF16 && a.g_norm == nullptr)) return false;
  BwdArgs f = {};
  f.a = a;
  f.pack = attn_pack(a.H / a.Hk);
  f.tile_tokens = kRows / f.pack;
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
  if (dtype == kBF16)
    *e = a.d <= 64 ? run<__nv_bfloat16, 64>(q, g, k, v, f, st) : run<__nv_bfloat16, 128>(q, g, k, v, f, st);
  else
    *e = a.d <= 64 ? run<__half, 64>(q, g, k, v, f, st) : run<__half, 128>(q, g, k, v, f, st);
  return true;
}

int read_device_error_tc_bwd(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_tc_bwd_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_tc_bwd_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace cta
