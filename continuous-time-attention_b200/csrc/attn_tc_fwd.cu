// Attention forward on the tensor cores: whole prompts, and chunks of rows over
// a 16-bit paged cache.
//
// A CTA owns two 128-row tiles of one block of heads.  A row is a (token, head)
// pair: where query heads share a key/value head, the largest power of two of
// them that divides the group goes into one tile, token by token, so that a tile
// has fewer tokens (less of a causal diagonal is computed in vain) and the keys
// are read for all of them at once.
//
//   warps 0-3, 4-7   softmax of tile 0 and 1: a thread holds one row
//   warp 8           issues the MMAs        warp 9   issues the TMA loads
//
// Per 128 keys and tile:  S = Q K^T into 128 columns of tensor memory; each
// softmax thread reads its row, P = exp2(c S - m) goes back as 16-bit into the
// same columns; O += P V with P read from tensor memory as the A operand.  While
// one tile's softmax runs, the other tile's products do.  The running maximum
// that P is relative to moves only when it has grown by more than 2^8, so O is
// rescaled (tensor memory -> registers -> tensor memory) a few times per row and
// not per tile; P stays below 2^8, the sum and O are fp32, and the quotient is
// exact in which reference was used.
//
// Bound by the exponentials and the products alike: 128 x 128 exponentials take
// 1024 cycles of the SM's 16-per-cycle unit, the two products of a tile 1024
// cycles at dim 128 (512 at dim 64).
#include <algorithm>

#include "attn_tc.cuh"

namespace cta {

__device__ int g_tc_fwd_error;

namespace {

constexpr int kThreads = 384;  // three warpgroups; warps 10 and 11 idle
constexpr int kRows = 128;  // rows of a tile, and keys of a step
constexpr float kLazy = 8.f;

struct FwdArgs {
  AttnArgs a;
  int pack;          // heads per tile row block
  int tile_tokens;   // kRows / pack
  // paged keys
  const int32_t* table;
  int64_t table_sB;
  const int32_t* seq_lens;
  int table_width, page, n_pages, box;  // box: keys per TMA box
  int vec_out;       // rows of the output are on 16 bytes
};

template <int DP>
struct Layout {
  static constexpr int kHalf = kRows * 128;            // one 64-column block of a 128-row tile
  static constexpr int kTile = kHalf * (DP / 64);
  static constexpr int kStages = DP == 128 ? 4 : 6;
  static constexpr int kSmem = 2 * kTile + kStages * kTile + 1024;
};

struct Bars {
  uint64_t q_full, kv_full[8], kv_empty[8], s_full[2], p_full[2], o_full[2];
};

template <typename T, int DP, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_fwd_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const __grid_constant__ FwdArgs f) {
  using L = Layout<DP>;
  constexpr int NS = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ SeqTile s_tile;
  __shared__ uint32_t s_boxes[16];  // paged: which boxes of a key tile were loaded
  const AttnArgs& a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const int blocks = a.H / f.pack;
  const int hb = blockIdx.x % blocks;
  const int h0 = hb * f.pack, hk = h0 / (a.H / a.Hk);

  if (warp == 0) {
    const SeqTile x = find_tile(a.cu, a.nseq, a.L, a.tiles, blockIdx.x / blocks, 2 * f.tile_tokens, a.causal);
    if (lane == 0) s_tile = x;
  } else if (warp == 8) {
    tc::alloc(&s_tmem, 512);
  } else if (warp == 9 && lane == 0) {
    mbar_init(&bars.q_full, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&bars.kv_full[i], 1);
      mbar_init(&bars.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], kRows);
      mbar_init(&bars.o_full[i], 1);
    }
    fence_mbar_init();
    prefetch_tmap(&qmap);
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const SeqTile t = s_tile;
  const uint32_t tmem = s_tmem;

  // keys: [lo, hi) of the sequence, n of them, row i sees j <= i + shift when causal
  int n = t.n, lo = 0, hi = t.n;
  bool bad_length = false;
  if constexpr (PAGED) {
    if (t.first < t.n) {
      n = __ldg(f.seq_lens + t.seq);
      const int64_t most = static_cast<int64_t>(f.table_width) * f.page;
      bad_length = n < 0 || n > most;
      n = n < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(n), most));
    }
    hi = n;
  } else {
    mask_range(a, t.batch, t.n, lo, hi);
  }
  const int shift = PAGED ? n - t.n : 0;
  const uint32_t* mask = !PAGED && a.mask != nullptr ? a.mask + t.batch * a.mask_words : nullptr;
  const int j_lo = lo / kRows;
  int steps[2], first[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    first[i] = t.first + i * f.tile_tokens;
    int end = hi;
    if (a.causal) end = min(end, min(first[i] + f.tile_tokens, t.n) + shift);
    steps[i] = first[i] < t.n ? max(0, (end + kRows - 1) / kRows - j_lo) : 0;
  }
  const int all = max(steps[0], steps[1]);

  // bit c of word w: key 32 w + c of tile j is one of the sequence's and valid
  auto key_words = [&](int j, uint32_t (&w)[4]) {
    const int j0 = (j_lo + j) * kRows;
    tc::first_bits(n - j0, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (mask != nullptr && n - j0 - 32 * i > 0) w[i] &= __ldg(mask + kMaskHead + (j0 >> 5) + i);
      if constexpr (PAGED) {
        const uint32_t boxes = *reinterpret_cast<volatile uint32_t*>(&s_boxes[j & 15]);
#pragma unroll
        for (int b = 0; b < 2; ++b)
          if (!((boxes >> (2 * i + b)) & 1u)) w[i] &= b == 0 ? 0xffff0000u : 0x0000ffffu;
      }
    }
  };

  // 384 threads x 168 registers at launch = 2 x 128 x 208 + 128 x 88
  if (warp >= 8) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
   if (warp == 9) {
    // ---------------- loads ----------------
    bool ok = true;
    int issued = 0;
    if (bad_length && lane == 0) atomicExch(&g_tc_fwd_error, kDevBadIndex);
    if (all > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars.q_full, 2 * L::kTile);
        for (int i = 0; i < 2; ++i)
          for (int c = 0; c < DP / 64; ++c)
            tc::tma_load_4d(smem + i * L::kTile + c * L::kHalf, &qmap, &bars.q_full, 64 * c, h0,
                            static_cast<int>(t.row0) + first[i], t.batch);
      }
      for (int x = 0; x < 2 * all && ok; ++x) {
        const int stage = x % NS;
        if (x >= NS) ok = mbar_wait_bounded(&bars.kv_empty[stage], ((x / NS) - 1) & 1);
        if (!ok) break;
        const CUtensorMap* map = (x & 1) ? &vmap : &kmap;
        const uint32_t dst = smem + (2 + stage) * L::kTile;
        const int j0 = (j_lo + (x >> 1)) * kRows;
        if constexpr (PAGED) {
          // one lane per box; a box outside the sequence or the cache is left out
          const int boxes = kRows / f.box;
          const int key = j0 + lane * f.box;
          int page = -1;
          if (lane < boxes && key < n) {
            page = __ldg(f.table + t.seq * f.table_sB + key / f.page);
            if (page < 0 || page >= f.n_pages) {
              atomicExch(&g_tc_fwd_error, kDevBadIndex);
              page = -1;
            }
          }
          const uint32_t got = __ballot_sync(0xffffffffu, page >= 0);
          if (lane == 0) {
            // one bit per 16 keys
            uint32_t bits = 0;
            const int per = f.box / 16;
            for (int b = 0; b < boxes; ++b)
              if ((got >> b) & 1u) bits |= ((1u << per) - 1u) << (b * per);
            *reinterpret_cast<volatile uint32_t*>(&s_boxes[(x >> 1) & 15]) = bits;
            mbar_arrive_expect_tx(&bars.kv_full[stage], __popc(got) * f.box * 128 * (DP / 64));
          }
          __syncwarp();
          if (page >= 0)
            for (int c = 0; c < DP / 64; ++c)
              tc::tma_load_4d(dst + c * L::kHalf + lane * f.box * 128, map, &bars.kv_full[stage], 64 * c, hk,
                              key % f.page, page);
        } else if (lane == 0) {
          mbar_arrive_expect_tx(&bars.kv_full[stage], L::kTile);
          for (int c = 0; c < DP / 64; ++c)
            tc::tma_load_4d(dst + c * L::kHalf, map, &bars.kv_full[stage], 64 * c, hk,
                            static_cast<int>(t.row0) + j0, t.batch);
        }
        issued = x + 1;
      }
      // nothing may still be in flight when the CTA ends: the MMA warp has waited for all of it unless a wait ran out
      if (!ok) {
        atomicExch(&g_tc_fwd_error, kDevTimeout);
        for (int x = max(0, issued - NS); x < issued; ++x) mbar_wait_bounded(&bars.kv_full[x % NS], (x / NS) & 1);
      }
    }
  } else if (warp == 8) {
    // ---------------- products ----------------
    constexpr uint32_t id_s = tc::idesc<T>(kRows, false), id_o = tc::idesc<T>(DP, true);
    const bool leader = tc::elect_one();
    bool ok = all == 0 || mbar_wait_bounded(&bars.q_full, 0);
    auto kv_wait = [&](int x) { ok = ok && mbar_wait_bounded(&bars.kv_full[x % NS], (x / NS) & 1); };
    auto kv_addr = [&](int x) { return smem + (2 + x % NS) * L::kTile; };
    auto scores = [&](int i, int j) {
      if (leader) {
        tc::product_nt<DP>(tmem + i * kRows, smem + i * L::kTile, L::kHalf, kv_addr(2 * j), L::kHalf, id_s);
        tc::commit(&bars.s_full[i]);
      }
    };
    if (all > 0) {
      kv_wait(0);
      tc::fence_after();
      if (ok) {
        for (int i = 0; i < 2; ++i)
          if (steps[i] > 0) scores(i, 0);
        if (leader) tc::commit(&bars.kv_empty[0]);
      }
    }
    for (int j = 0; j < all && ok; ++j) {
      kv_wait(2 * j + 1);
      if (!ok) break;
      // values of keys that are not there or not valid may hold anything: a zero weight times NaN is NaN
      uint32_t w[4];
      key_words(j, w);
      if (!tc::all_set(w)) tc::clear_rows<DP / 64>(kv_addr(2 * j + 1), w);
      const bool more = j + 1 < all;
      for (int i = 0; i < 2 && ok; ++i) {
        if (j < steps[i]) {
          ok = mbar_wait_bounded(&bars.p_full[i], j & 1);
          tc::fence_after();
          if (ok && leader) {
            tc::product_tn(tmem + 2 * kRows + i * DP, tmem + i * kRows, kv_addr(2 * j + 1), L::kHalf, id_o, j > 0);
            if (j + 1 == steps[i]) tc::commit(&bars.o_full[i]);
          }
        }
        if (j + 1 < steps[i]) {
          kv_wait(2 * j + 2);
          tc::fence_after();
          if (ok) scores(i, j + 1);
        }
      }
      if (ok && leader) {
        tc::commit(&bars.kv_empty[(2 * j + 1) % NS]);
        if (more) tc::commit(&bars.kv_empty[(2 * j + 2) % NS]);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicExch(&g_tc_fwd_error, kDevTimeout);
   }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---------------- softmax ----------------
    const int i = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int tok = first[i] + row / f.pack, h = h0 + row % f.pack;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + i * kRows, o_addr = tmem + lanes + 2 * kRows + i * DP;
    const float c2 = a.scale * kLog2e;
    const int limit = a.causal ? tok + shift : n - 1;  // last key the row sees
    float m = neg_inf(), sum = 0.f;
    bool ok = true;
    for (int j = 0; j < steps[i]; ++j) {
      ok = mbar_wait_bounded(&bars.s_full[i], j & 1);
      if (!ok) break;
      tc::fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tc::ld32(s_addr + 32 * c, s[c]);
      tc::wait_ld();
      const int j0 = (j_lo + j) * kRows;
      uint32_t w[4];
      key_words(j, w);
      // warp-uniform: does every row of the warp see all 128 keys?
      const bool whole = tc::all_set(w) &&
                         (!a.causal || j0 + kRows - 1 <= first[i] + (warp & 3) * 32 / f.pack + shift);
      if (!whole) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int left = limit - j0 - 32 * c + 1;
          const uint32_t see = w[c] & (left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((see >> e) & 1u)) s[c][e] = 0xff800000u;
        }
      }
      float top[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        top[c] = __uint_as_float(s[c][0]);
#pragma unroll
        for (int e = 1; e < 32; ++e) top[c] = fmaxf(top[c], __uint_as_float(s[c][e]));
      }
      const float now = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
      // move the reference when it has grown by more than kLazy (or there was none)
      const bool move = now > m && !((now - m) * c2 <= kLazy);
      if (__any_sync(0xffffffffu, move)) {
        const float shrink = move ? ex2((m - now) * c2) : 1.f;
        if (move) {
          sum *= shrink;
          m = now;
        }
        if (j > 0) {
          // the scores' barrier also covers the previous O += P V
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tc::ld32(o_addr + 32 * c, o);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
            tc::st32(o_addr + 32 * c, o);
          }
        }
      }
      const float base = m == neg_inf() ? 0.f : -m * c2;
      const float2 c2v = f2(c2), bv = f2(base);
      float2 part = f2(0.f), part2 = f2(0.f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float2 x = fma2(make_float2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), c2v, bv);
          x.x = ex2(x.x);
          x.y = ex2(x.y);
          if (e & 1) part2 = add2(part2, x);
          else part = add2(part, x);
          p[e] = tc::pack2<T>(x.x, x.y);
        }
        tc::st16(s_addr + 16 * c, p);
      }
      part = add2(part, part2);
      sum += part.x + part.y;
      tc::wait_st();
      tc::fence_before();
      tc::arrive(&bars.p_full[i]);
    }
    const bool live = tok < t.n && row / f.pack < f.tile_tokens;
    if (ok && steps[i] > 0) ok = mbar_wait_bounded(&bars.o_full[i], 0);
    tc::fence_after();
    if (!ok) {
      if (lane == 0) atomicExch(&g_tc_fwd_error, kDevTimeout);
    } else if (first[i] < t.n) {
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // NaN stays
      T* out = static_cast<T*>(a.o) + t.batch * a.os.b + (t.row0 + tok) * a.os.t + h * a.os.h;
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (steps[i] > 0) {
          tc::ld32(o_addr + 32 * c, o);
          tc::wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (live) {
          if (f.vec_out) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (32 * c + e < a.d) {
                uint4 x;
                uint32_t* xp = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  xp[y] = tc::pack2<T>(__uint_as_float(o[e + 2 * y]) * inv, __uint_as_float(o[e + 2 * y + 1]) * inv);
                *reinterpret_cast<uint4*>(out + 32 * c + e) = x;
              }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * c + e < a.d) out[32 * c + e] = Elem<T>::from_f(__uint_as_float(o[e]) * inv);
          }
        }
      }
      if (live && a.lse != nullptr)
        a.lse[lse_index(a, t, h, tok)] = sum == 0.f ? neg_inf() : (m * c2 + log2f(sum)) * kLn2;
    } else if (!PAGED && a.cu != nullptr && a.zero_tail && i == 0 && t.n == 0) {
      // a tile behind the last sequence clears rows there
      for (int64_t r = t.row0 + t.tail_index; r < a.L; r += t.tail_count)
        for (int x = threadIdx.x; x < a.d * f.pack; x += kRows)
          static_cast<T*>(a.o)[r * a.os.t + (h0 + x / a.d) * a.os.h + x % a.d] = Elem<T>::from_f(0.f);
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::dealloc(tmem, 512);
}

template <typename T, int DP, bool PAGED>
cudaError_t launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FwdArgs& f, int64_t ctas,
                   cudaStream_t st) {
  const cudaError_t e = allow_smem<attn_tc_fwd_kernel<T, DP, PAGED>>(Layout<DP>::kSmem);
  if (e != cudaSuccess) return e;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  attn_tc_fwd_kernel<T, DP, PAGED><<<static_cast<unsigned>(ctas), kThreads, Layout<DP>::kSmem, st>>>(q, k, v, f);
  return cudaGetLastError();
}

template <bool PAGED>
cudaError_t dispatch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FwdArgs& f, int dtype,
                     int64_t ctas, cudaStream_t st) {
  if (dtype == kBF16)
    return f.a.d <= 64 ? launch<__nv_bfloat16, 64, PAGED>(q, k, v, f, ctas, st)
                       : launch<__nv_bfloat16, 128, PAGED>(q, k, v, f, ctas, st);
  return f.a.d <= 64 ? launch<__half, 64, PAGED>(q, k, v, f, ctas, st)
                     : launch<__half, 128, PAGED>(q, k, v, f, ctas, st);
}

bool on16(const void* p, const AttnStrides& s, int64_t nb, int64_t heads) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s.t % 8 == 0 && (heads == 1 || s.h % 8 == 0) &&
         (nb == 1 || s.b % 8 == 0);
}

}  // namespace

int attn_pack(int group) { return std::min(group & -group, kRows); }

bool launch_attn_tc_fwd(const AttnArgs& a, int dtype, cudaStream_t st, cudaError_t* e) {
  if (dtype == kF32 || a.d % 8 != 0 || a.d > 128 || !(a.scale > 0.f)) return false;
  FwdArgs f = {};
  f.a = a;
  f.pack = attn_pack(a.H / a.Hk);
  f.tile_tokens = kRows / f.pack;
  const int64_t nb = a.cu != nullptr ? 1 : a.nseq;
  CUtensorMap q, k, v;
  if (!attn_map(&q, a.q, dtype, nb, a.L, a.H, a.d, a.qs, f.pack, f.tile_tokens) ||
      !attn_map(&k, a.k, dtype, nb, a.L, a.Hk, a.d, a.ks, 1, kRows) ||
      !attn_map(&v, a.v, dtype, nb, a.L, a.Hk, a.d, a.vs, 1, kRows))
    return false;
  f.vec_out = on16(a.o, a.os, nb, a.H);
  int64_t tiles;
  const int rows = 2 * f.tile_tokens;
  if (a.cu != nullptr) {
    tiles = packed_tiles(a.L, a.nseq, rows);
    f.a.tiles = static_cast<int>(tiles);
  } else {
    f.a.tiles = static_cast<int>((a.L + rows - 1) / rows);
    tiles = static_cast<int64_t>(f.a.tiles) * a.nseq;
  }
  *e = dispatch<false>(q, k, v, f, dtype, tiles * (a.H / f.pack), st);
  return true;
}

bool launch_paged_tc(const PagedArgs& p, int dtype, cudaStream_t st, cudaError_t* e) {
  if (!(p.scale > 0.f) || p.cu == nullptr) return false;
  FwdArgs f = {};
  AttnArgs& a = f.a;
  a.q = p.q;
  a.o = p.o;
  a.qs = AttnStrides{0, p.q_sT, p.q_sH};
  a.os = AttnStrides{0, p.o_sT, p.o_sH};
  a.cu = p.cu;
  a.L = p.T;
  a.nseq = p.B;
  a.H = p.H;
  a.Hk = p.Hk;
  a.d = p.d;
  a.causal = 1;
  a.scale = p.scale;
  f.pack = attn_pack(p.H / p.Hk);
  f.tile_tokens = kRows / f.pack;
  f.table = p.table;
  f.table_sB = p.table_sB;
  f.seq_lens = p.seq_lens;
  f.table_width = p.table_width;
  f.page = p.page;
  f.n_pages = p.n_pages;
  f.box = std::min(p.page & -p.page, kRows);  // the largest power of two that divides a page
  f.vec_out = 1;
  CUtensorMap q, k, v;
  if (!attn_map(&q, p.q, dtype, 1, p.T, p.H, p.d, a.qs, f.pack, f.tile_tokens) ||
      !attn_map(&k, p.k_cache, dtype, p.n_pages, p.page, p.Hk, p.d, AttnStrides{p.kc_sP, p.kc_sS, p.kc_sH}, 1, f.box) ||
      !attn_map(&v, p.v_cache, dtype, p.n_pages, p.page, p.Hk, p.d, AttnStrides{p.vc_sP, p.vc_sS, p.vc_sH}, 1, f.box))
    return false;
  const int64_t tiles = packed_tiles(p.T, p.B, 2 * f.tile_tokens);
  a.tiles = static_cast<int>(tiles);
  *e = dispatch<true>(q, k, v, f, dtype, tiles * (p.H / f.pack), st);
  return true;
}

int read_device_error_tc_fwd(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_tc_fwd_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_tc_fwd_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace cta
