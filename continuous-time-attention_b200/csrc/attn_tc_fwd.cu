// Attention forward on the tensor cores: whole prompts, and chunks of rows over
// a 16-bit paged cache.
//
// An e4m3 cache is first expanded to 16-bit pages (kv_cache.cu) whose elements are exact.
// bf16: codes times the power of two below their scale; the rest of the scale, in [1, 2),
// multiplies the key's scores and, after the sum of the weights, its weights.  fp16, which
// does not reach as far as scales do: the codes alone; the key's scale multiplies the scores,
// and the value's joins the weight's exponent, relative to a running maximum of its own, so
// that any scales are right (with powers of two in the elements, as in bf16, scales from 256 on
// were infinite, and codes under scales below 2^-15 rounded).  Both cost the softmax more than a
// 16-bit cache does: 512 rows over 8192 keys, 32/8 heads of 128, take 143 us over 16 bits,
// 299 in bf16 and 408 in fp16 over e4m3; with k and v times their whole scale, rounded to 16
// bits, the call took 157 us, but fp16 outputs were twice as far off as one rounding of them.
//
// A CTA owns two 128-row tiles of one block of heads.  A row is a (token, head)
// pair: where query heads share a key/value head, the largest power of two of
// them that divides the group goes into one tile, token by token, so that a tile
// has fewer tokens (less of a causal diagonal is computed in vain) and the keys
// are read for all of them at once.
//
//   warps 0-7, 8-15   softmax of tile 0 and 1: two threads per row, 64 keys each
//   warps 16, 19   MMAs of tile 0 and 1    warp 17   TMA loads    warp 18   finds the work
//
// The grid has a CTA for each pair of tiles; a CTA that has finished one takes
// over another that has not started (cluster launch control), so that the loads
// and the first scores of the next pair run under the last weights and the
// output of this one, and the setup is paid once per SM.
//
// Per 128 keys and tile:  S = Q K^T into 128 columns of tensor memory; each
// softmax thread reads its half row, P = exp2(c S - m) goes back as 16-bit into
// the same columns; O += P V with P read from tensor memory as the A operand.
// While one tile's softmax runs, the other tile's products do.  The running maximum
// that P is relative to moves only when it has grown by more than 2^8, so O is
// rescaled (tensor memory -> registers -> tensor memory) a few times per row and
// not per tile; P stays below 2^8, the sum and O are fp32, and the quotient is
// exact in which reference was used.
//
// Bound by the exponentials and the products alike: 128 x 128 exponentials take
// 1024 cycles of the SM's 16-per-cycle unit, the two products of a tile 1024
// cycles at dim 128 (512 at dim 64).  Measured, 8192 tokens: 16 heads of 128 514 us,
// 1070 TFLOP/s; 32/8 heads of 128, causal, 457 us, 1203; 16 heads of 64 426 us, 645
// (runs on other boards: 503 to 510, 445, 400).
// 4 chunks of 512 rows over 1500 to 8192 cached keys, 32/8 heads of 128: 162 us.
#include <algorithm>

#include "attn_tc.cuh"

namespace cta {

__device__ int g_tc_fwd_error;

namespace {

constexpr int kThreads = 640;  // five warpgroups
constexpr int kSoftmaxWarps = 16;
constexpr int kRows = 128;  // rows of a tile, and keys of a step
constexpr float kLazy = 8.f;
// fp16 weights carry 2^7, and so stay below 2^15; what is lost to subnormals is below 2^-32 of the reference
constexpr float kHalfShift = 7.f;
static_assert(kHalfShift == 7.f, "lse takes 2^-7 of the sum");

struct FwdArgs {
  AttnArgs a;
  int pack;          // heads per tile row block
  int tile_tokens;   // kRows / pack
  int across;        // order of the work, see find_tile
  // paged keys
  const int32_t* table;
  int64_t table_sB;
  const int32_t* seq_lens;
  int table_width, page, n_pages, box;  // box: keys per TMA box
  // SCALED: page i of sequence b is page b * table_width + i (the table still says which are valid), and these are
  // what the expansion left out of its elements, see launch_cache_expand
  const float* k_res;
  const float* v_res;
  int wide_out, wide_low;  // alignment of the outputs' rows, see store_rows
};

template <int DP>
struct Layout {
  static constexpr int kHalf = kRows * 128;            // one 64-column block of a 128-row tile
  static constexpr int kTile = kHalf * (DP / 64);
  static constexpr int kStages = DP == 128 ? 4 : 6;
  static constexpr int kSmem = 2 * kTile + kStages * kTile + 1024;
};

struct Bars {
  uint64_t q_full, q_empty, kv_full[8], kv_empty[8], s_full[2], p_half[2], p_full[2], o_full[2];
  uint64_t item_full, item_taken, answer;
};

// One piece of work: two row tiles of one block of heads.
struct Item {
  SeqTile t;
  int h0, hk;  // first query head, key/value head
  int n;       // keys of the sequence
  int lo, hi;  // first and one past the last that may be valid
  bool last;   // there is no more work
};

template <typename T, int DP, bool PAGED, bool SCALED>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_fwd_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const __grid_constant__ FwdArgs f) {
  using L = Layout<DP>;
  constexpr int NS = L::kStages;
  // Half of a step's weights are announced too, which wakes the waiting MMA warp ahead of time: 402
  // instead of 454 us at 8192 keys, 16 heads of 64, but 534 instead of 503 at 128.
  constexpr bool kEarly = DP == 64;
  // Over an expanded e4m3 cache in fp16 the value's scale joins the weight, whose own running reference keeps the
  // product within fp16 for any scales.
  constexpr bool kWeighted = SCALED && std::is_same<T, __half>::value;
  constexpr float kShift = std::is_same<T, __half>::value && !SCALED ? kHalfShift : 0.f;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ Item s_item;
  __shared__ __align__(16) uint4 s_answer;
  __shared__ float s_max[2][2][kRows], s_sum[2][2][kRows];  // [tile][half of the keys][row]
  __shared__ float s_maxv[kWeighted ? 2 : 1][2][kWeighted ? kRows : 1];
  __shared__ uint32_t s_boxes[16];  // paged: which boxes of a key tile were loaded
  const AttnArgs& a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;

  if (warp == kSoftmaxWarps) {
    tc::alloc(&s_tmem, 512);
  } else if (warp == kSoftmaxWarps + 1 && lane == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 2);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&bars.kv_full[i], 1);
      mbar_init(&bars.kv_empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_half[i], kSoftmaxWarps / 2);
      mbar_init(&bars.p_full[i], kSoftmaxWarps / 2);
      mbar_init(&bars.o_full[i], 1);
    }
    mbar_init(&bars.item_full, 1);
    mbar_init(&bars.item_taken, kSoftmaxWarps + 3);
    mbar_init(&bars.answer, 1);
    fence_mbar_init();
    prefetch_tmap(&qmap);
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = s_tmem;

  // the it-th piece of work, for the warps that work on it; false: a wait ran out
  auto read_item = [&](int it, Item& x) -> bool {
    if (!tc::wait(&bars.item_full, it & 1)) return false;
    x = s_item;
    __syncwarp();
    return true;
  };
  auto taken = [&] {
    if (lane == 0) tc::arrive(&bars.item_taken);
  };
  auto take = [&](int it, Item& x) -> bool {
    if (!read_item(it, x)) return false;
    taken();
    return true;
  };
  // steps of 128 keys of the two tiles; j_lo: the first
  auto plan = [&](const Item& x, int (&first)[2], int (&steps)[2], int& j_lo, int& shift) {
    shift = PAGED ? x.n - x.t.n : 0;
    j_lo = x.lo / kRows;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      first[i] = x.t.first + i * f.tile_tokens;
      int end = x.hi;
      if (a.causal) end = min(end, min(first[i] + f.tile_tokens, x.t.n) + shift);
      steps[i] = first[i] < x.t.n ? max(0, (end + kRows - 1) / kRows - j_lo) : 0;
    }
  };
  // bit c of word i: key 32 i + c of the tile at j0 is one of the sequence's and valid; `kt`: running number of the tile
  auto key_words = [&](int n, const uint32_t* mask, int j0, int kt, uint32_t (&w)[4]) {
    tc::first_bits(n - j0, w);
    if constexpr (PAGED) {
      const uint32_t boxes = *reinterpret_cast<volatile uint32_t*>(&s_boxes[kt & 15]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!((boxes >> i) & 1u)) w[i >> 1] &= (i & 1) == 0 ? 0xffff0000u : 0x0000ffffu;
    } else if (mask != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n - j0 - 32 * i > 0) w[i] &= __ldg(mask + (j0 >> 5) + i);
    }
  };

  // 640 threads x 96 registers at launch = 4 x 128 x 104 + 128 x 64
  if (warp >= kSoftmaxWarps) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
   if (warp == kSoftmaxWarps + 2) {
    // ---------------- which work ----------------
    // The grid has a CTA per piece of work; a CTA that is done goes on with one that has not started.
    const int blocks = a.H / f.pack;
    bool ok = true;
    int id = blockIdx.x;
    for (int it = 0; ok; ++it) {
      if (it > 0) {
        // Every warp has begun the piece before, and its loads are all on their way.  Asked for
        // earlier, pieces of different lengths would be dealt out before it is known who is free:
        // 4 chunks over 1500 to 8192 keys took 315 us instead of 200.
        ok = tc::wait(&bars.item_taken, (it - 1) & 1);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars.answer, 16);
          tc::steal(&s_answer, &bars.answer);
        }
        ok = tc::wait(&bars.answer, (it - 1) & 1);
        if (!ok) break;
        id = tc::stolen(&s_answer);
      }
      Item x = {};
      x.last = id < 0;
      if (id >= 0) {
        const int hb = id % blocks;
        x.h0 = hb * f.pack;
        x.hk = x.h0 / (a.H / a.Hk);
        x.t = find_tile(a.cu, a.nseq, a.L, a.tiles, id / blocks, 2 * f.tile_tokens, a.causal, f.across,
                        f.seq_lens);
        x.n = x.hi = x.t.n;
        if constexpr (PAGED) {
          if (x.t.first < x.t.n) {
            x.n = __ldg(f.seq_lens + x.t.seq);
            const int64_t most = static_cast<int64_t>(f.table_width) * f.page;
            if ((x.n < 0 || x.n > most) && lane == 0) atomicExch(&g_tc_fwd_error, kDevBadIndex);
            x.n = x.n < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(x.n), most));
          }
          x.hi = x.n;
        } else {
          mask_range(a, x.t.batch, x.t.n, x.lo, x.hi);
        }
      }
      if (lane == 0) {
        s_item = x;
        tc::arrive(&bars.item_full);
      }
      __syncwarp();
      if (id < 0) break;
    }
    if (!ok && lane == 0) atomicExch(&g_tc_fwd_error, kDevTimeout);
   } else if (warp == kSoftmaxWarps + 1) {
    // ---------------- loads ----------------
    bool ok = true;
    int kv = 0, nq = 0;  // tiles loaded so far, Q loads so far
    for (int it = 0; ok; ++it) {
      Item x;
      ok = read_item(it, x);
      if (!ok || x.last) break;
      int first[2], steps[2], j_lo, shift;
      plan(x, first, steps, j_lo, shift);
      const int all = max(steps[0], steps[1]);
      if (all == 0) {
        taken();
        continue;
      }
      if (nq > 0) ok = tc::wait(&bars.q_empty, (nq - 1) & 1);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars.q_full, 2 * L::kTile);
        for (int i = 0; i < 2; ++i)
          for (int c = 0; c < DP / 64; ++c)
            tc::tma_load_4d(smem + i * L::kTile + c * L::kHalf, &qmap, &bars.q_full, 64 * c, x.h0,
                            static_cast<int>(x.t.row0) + first[i], x.t.batch);
      }
      ++nq;
      for (int y = 0; y < 2 * all; ++y) {
        const int stage = kv % NS;
        if (kv >= NS) ok = tc::wait(&bars.kv_empty[stage], ((kv / NS) - 1) & 1);
        if (!ok) break;
        const CUtensorMap* map = (y & 1) ? &vmap : &kmap;
        const uint32_t dst = smem + (2 + stage) * L::kTile;
        const int j0 = (j_lo + (y >> 1)) * kRows;
        if constexpr (PAGED) {
          // one lane per box; a box outside the sequence or the cache is left out
          const int boxes = kRows / f.box;
          const int key = j0 + lane * f.box;
          int page = -1;
          if (lane < boxes && key < x.n) {
            page = __ldg(f.table + x.t.seq * f.table_sB + key / f.page);
            if (page < 0 || page >= f.n_pages) {
              atomicExch(&g_tc_fwd_error, kDevBadIndex);
              page = -1;
            } else if (SCALED) {
              page = x.t.seq * f.table_width + key / f.page;
            }
          }
          const uint32_t got = __ballot_sync(0xffffffffu, page >= 0);
          if (lane == 0) {
            // one bit per 16 keys
            uint32_t bits = 0;
            const int per = f.box / 16;
            for (int b = 0; b < boxes; ++b)
              if ((got >> b) & 1u) bits |= ((1u << per) - 1u) << (b * per);
            *reinterpret_cast<volatile uint32_t*>(&s_boxes[(kv >> 1) & 15]) = bits;
            mbar_arrive_expect_tx(&bars.kv_full[stage], __popc(got) * f.box * 128 * (DP / 64));
          }
          __syncwarp();
          if (page >= 0)
            for (int c = 0; c < DP / 64; ++c)
              tc::tma_load_4d(dst + c * L::kHalf + lane * f.box * 128, map, &bars.kv_full[stage], 64 * c, x.hk,
                              key % f.page, page);
        } else if (lane == 0) {
          mbar_arrive_expect_tx(&bars.kv_full[stage], L::kTile);
          for (int c = 0; c < DP / 64; ++c)
            tc::tma_load_4d(dst + c * L::kHalf, map, &bars.kv_full[stage], 64 * c, x.hk,
                            static_cast<int>(x.t.row0) + j0, x.t.batch);
        }
        ++kv;
      }
      taken();
    }
    // nothing may still be in flight when the CTA ends: the MMA warp has waited for all of it unless a wait ran out
    if (!ok) {
      atomicExch(&g_tc_fwd_error, kDevTimeout);
      for (int y = max(0, kv - NS); y < kv; ++y) tc::wait(&bars.kv_full[y % NS], (y / NS) & 1);
      if (nq > 0) tc::wait(&bars.q_full, (nq - 1) & 1);
    }
   } else {
    // ---------------- products ----------------
    // One warp per row tile: a successful wait costs a hundred cycles or more, and with one warp for
    // both tiles those of one tile delayed the other's products (562 instead of 503 us at 8192 keys,
    // 16 heads of 128, 477 instead of 402 at 64).  Both free a key tile.
    const int i = warp == kSoftmaxWarps ? 0 : 1;
    constexpr uint32_t id_s = tc::idesc<T>(kRows, false), id_o = tc::idesc<T>(DP, true);
    const bool leader = tc::elect_one();
    bool ok = true;
    int kv = 0, nq = 0, ns = 0;  // running numbers: tiles, Q loads, steps of this row tile
    const uint32_t t_s = tmem + i * kRows, t_o = tmem + 2 * kRows + i * DP, q = smem + i * L::kTile;
    for (int it = 0; ok; ++it) {
      Item x;
      ok = take(it, x);
      if (!ok || x.last) break;
      int first[2], steps[2], j_lo, shift;
      plan(x, first, steps, j_lo, shift);
      const int all = max(steps[0], steps[1]), mine = i == 0 ? steps[0] : steps[1];
      if (all == 0) continue;
      ok = tc::wait(&bars.q_full, nq & 1);
      ++nq;
      const uint32_t* mask = !PAGED && a.mask != nullptr ? a.mask + x.t.batch * a.mask_words + kMaskHead : nullptr;
      auto kv_wait = [&](int y) { ok = ok && tc::wait(&bars.kv_full[(kv + y) % NS], ((kv + y) / NS) & 1); };
      auto kv_addr = [&](int y) { return smem + (2 + (kv + y) % NS) * L::kTile; };
      // scores of step j into the tile's buffer; keys are released by the step's end
      auto scores = [&](int j) {
        tc::product_nt<DP>(t_s, q, kv_addr(2 * j), id_s);
        tc::commit(&bars.s_full[i]);
        if (j + 1 == mine) tc::commit(&bars.q_empty);
      };
      kv_wait(0);
      tc::fence_after();
      if (ok && leader) {
        if (mine > 0) scores(0);
        else tc::commit(&bars.q_empty);
        tc::commit(&bars.kv_empty[kv % NS]);
      }
      __syncwarp();
      for (int j = 0; j < all && ok; ++j) {
        kv_wait(2 * j + 1);
        if (j + 1 < all) kv_wait(2 * j + 2);
        if (!ok) break;
        if (j < mine) {
          // values of keys that are not there or not valid may hold anything
          uint32_t w[4];
          const int j0 = (j_lo + j) * kRows;
          if (PAGED || mask != nullptr || j0 + kRows > x.n) {
            key_words(x.n, mask, j0, (kv >> 1) + j, w);
            if (!tc::all_set(w)) tc::clear_rows<DP / 64>(kv_addr(2 * j + 1), w);
          }
          // (Issuing the products of half the keys ahead of the others was tried: it costs more than it
          // hides, 643 instead of 534 us at 8192 keys, 16 heads of 128.)
          if (kEarly) ok = tc::wait(&bars.p_half[i], ns & 1);
          ok = ok && tc::wait(&bars.p_full[i], ns & 1);
          tc::fence_after();
          if (ok && leader) {
            tc::product_tn<64>(t_o, t_s, kv_addr(2 * j + 1), id_o, j > 0);
            if (j + 1 == mine) tc::commit(&bars.o_full[i]);
            else scores(j + 1);
          }
          ++ns;
        }
        if (ok && leader) {
          tc::commit(&bars.kv_empty[(kv + 2 * j + 1) % NS]);
          if (j + 1 < all) tc::commit(&bars.kv_empty[(kv + 2 * j + 2) % NS]);
        }
        __syncwarp();
      }
      kv += 2 * all;
    }
    if (!ok && lane == 0) atomicExch(&g_tc_fwd_error, kDevTimeout);
   }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---------------- softmax ----------------
    const int i = warp >> 3, half = (warp >> 2) & 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + i * kRows + half * 64;
    const uint32_t o_addr = tmem + lanes + 2 * kRows + i * DP + half * (DP / 2);
    const float c2 = a.scale * kLog2e;
    bool ok = true;
    int ns = 0, no = 0, kt = 0;  // running numbers: steps, outputs, key tiles
    for (int it = 0; ok; ++it) {
      Item x;
      ok = take(it, x);
      if (!ok || x.last) break;
      int first[2], steps[2], j_lo, shift;
      plan(x, first, steps, j_lo, shift);
      const int mine = i == 0 ? first[0] : first[1], count = i == 0 ? steps[0] : steps[1];
      const int all = max(steps[0], steps[1]);
      if (!PAGED && a.cu != nullptr && a.zero_tail && warp < 4 && x.t.n == 0) {
        // a tile behind the last sequence clears rows there
        for (int64_t r = x.t.row0 + x.t.tail_index; r < a.L; r += x.t.tail_count)
          for (int y = threadIdx.x; y < a.d * f.pack; y += kRows)
            static_cast<T*>(a.o)[r * a.os.t + (x.h0 + y / a.d) * a.os.h + y % a.d] = Elem<T>::from_f(0.f);
      }
      if (mine >= x.t.n) {
        kt += all;
        continue;
      }
      const int n = x.n;
      const uint32_t* mask = !PAGED && a.mask != nullptr ? a.mask + x.t.batch * a.mask_words + kMaskHead : nullptr;
      const int tok = mine + row / f.pack, h = x.h0 + row % f.pack;
      const bool live = tok < x.t.n;
      const int limit = a.causal ? tok + shift : n - 1;  // last key the row sees
      const int limit_all = mine + (warp & 3) * 32 / f.pack + shift;  // causal: last key all rows of the warp see
      T* out = static_cast<T*>(a.o) + x.t.batch * a.os.b + (x.t.row0 + tok) * a.os.t + h * a.os.h;
      float* lse = live && half == 0 && a.lse != nullptr ? a.lse + lse_index(a, x.t, h, tok) : nullptr;
      // the first fraction of this half's keys
      int res = SCALED ? (x.t.seq * a.Hk + x.hk) * static_cast<int>(residue_row(f.table_width * f.page)) +
                             j_lo * kRows + 64 * half
                       : 0;
      float m = neg_inf(), sum = 0.f;
      float mv = neg_inf();  // kWeighted: the reference of weight * scale, as an exponent of two
      for (int j = 0; j < count; ++j, ++ns, res += SCALED ? kRows : 0) {
        if (SCALED && lane < 4)  // two lines each of the step's fractions
          asm volatile("prefetch.global.L1 [%0];" ::"l"((lane < 2 ? f.k_res : f.v_res) + res + 32 * (lane & 1)));
        // After a wait that ran out a warp goes on without waiting to the end of the piece, so that
        // the named barriers below see all their warps.
        ok = ok && tc::wait(&bars.s_full[i], ns & 1);
        tc::fence_after();
        const int j0 = (j_lo + j) * kRows;
        uint32_t s[2][32];
        if (!SCALED) {
          tc::ld32(s_addr, s[0]);
          tc::ld32(s_addr + 32, s[1]);
        }
        // warp-uniform: every row of the warp sees all keys of the tile
        bool whole = j0 + kRows <= n && (!a.causal || j0 + kRows - 1 <= limit_all);
        uint32_t w[4];
        if (PAGED || mask != nullptr || !whole) {
          key_words(n, mask, j0, kt + j, w);
          whole = whole && tc::all_set(w);
        }
        if (!SCALED) tc::wait_ld(s[0], s[1]);
        // Fractions of the scales, 32 keys at a time: the scores are read from tensor memory once for the maximum and
        // once for the weights, which leaves registers for eight loads.  Bound by issue (77 % of the cycles of a busy
        // SM); with one read of both the loads wait for one another instead, 205 and 199 us for 32 chunks of 16
        // rows over 2048 keys.
        auto scale = [&](int c, uint32_t (&x)[32]) {
          tc::ld32(s_addr + 32 * c, x);
          float4 r[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = __ldg(reinterpret_cast<const float4*>(f.k_res + res + 32 * c) + e);
          tc::wait_ld(x);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 lo = mul2(make_float2(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1])),
                                   make_float2(r[e].x, r[e].y));
            const float2 hi = mul2(make_float2(__uint_as_float(x[4 * e + 2]), __uint_as_float(x[4 * e + 3])),
                                   make_float2(r[e].z, r[e].w));
            x[4 * e] = __float_as_uint(lo.x);
            x[4 * e + 1] = __float_as_uint(lo.y);
            x[4 * e + 2] = __float_as_uint(hi.x);
            x[4 * e + 3] = __float_as_uint(hi.y);
          }
        };
        auto hide = [&](int c, uint32_t (&x)[32]) {
          const int left = limit - j0 - 64 * half - 32 * c + 1;
          const uint32_t see =
              (half == 0 ? w[c] : w[2 + c]) & (left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((see >> e) & 1u)) x[e] = 0xff800000u;
        };
        float t[4], topv = mv;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t(&x)[32] = s[SCALED ? 0 : c];
          if (SCALED) scale(c, x);
          if (!whole) hide(c, x);
          if constexpr (kWeighted) {
            // score + logarithm of the value's scale
            float4 r[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) r[e] = __ldg(reinterpret_cast<const float4*>(f.v_res + res + 32 * c) + e);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 lo = fma2(make_float2(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1])), f2(c2),
                                     make_float2(r[e].x, r[e].y));
              const float2 hi = fma2(make_float2(__uint_as_float(x[4 * e + 2]), __uint_as_float(x[4 * e + 3])), f2(c2),
                                     make_float2(r[e].z, r[e].w));
              topv = tc::max3(tc::max3(lo.x, lo.y, hi.x), hi.y, topv);
            }
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float& z = t[2 * c + y];
            z = __uint_as_float(x[16 * y]);
#pragma unroll
            for (int e = 1; e < 15; e += 2)
              z = tc::max3(z, __uint_as_float(x[16 * y + e]), __uint_as_float(x[16 * y + e + 1]));
            z = fmaxf(z, __uint_as_float(x[16 * y + 15]));
          }
        }
        float top = tc::max3(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]), m);
        // The reference of a row moves when one of its halves has grown by more than kLazy past it (or
        // there was none): one barrier with a vote per step, and the halves' maxima only then.
        auto far = [&] {
          return (top > m && !((top - m) * c2 <= kLazy)) || (kWeighted && topv > mv && !(topv - mv <= kLazy));
        };
        if (tc::any_of(1 + i, 2 * kRows, far())) {
          s_max[i][half][row] = top;
          if constexpr (kWeighted) s_maxv[i][half][row] = topv;
          tc::sync_of(1 + i, 2 * kRows);
          top = fmaxf(top, s_max[i][half ^ 1][row]);
          if constexpr (kWeighted) topv = fmaxf(topv, s_maxv[i][half ^ 1][row]);
          const bool move = far();
          float shrink = 1.f;
          if constexpr (kWeighted) {
            if (move) {
              if (top > m) sum *= ex2((m - top) * c2);
              if (topv > mv) shrink = ex2(mv - topv);
              m = fmaxf(m, top);
              mv = fmaxf(mv, topv);
            }
          } else if (move) {
            shrink = ex2((m - top) * c2);
            sum *= shrink;
            m = top;
          }
          if (j > 0 && __any_sync(0xffffffffu, move)) {
            // the scores' barrier also covers the previous O += P V; each half has its half of the columns
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
              uint32_t o[16];
              tc::ld16(o_addr + 16 * c, o);
              tc::wait_ld(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
              tc::st16(o_addr + 16 * c, o);
            }
          }
        }
        const float base = m == neg_inf() ? 0.f : kShift - m * c2;
        const float2 c2v = f2(c2), bv = f2(base);
        const float2 vv = f2(mv == neg_inf() ? 0.f : kHalfShift - mv);
        float2 part = f2(0.f), part2 = f2(0.f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t p[16];
          uint32_t(&x)[32] = s[SCALED ? 0 : c];
          float4 r[SCALED ? 8 : 1];
          if constexpr (SCALED) {
            scale(c, x);
            if (!whole) hide(c, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) r[e] = __ldg(reinterpret_cast<const float4*>(f.v_res + res + 32 * c) + e);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 score = make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
            float2 y = fma2(score, c2v, bv);
            y.x = ex2(y.x);
            y.y = ex2(y.y);
            if (e & 1) part2 = add2(part2, y);
            else part = add2(part, y);
            if constexpr (SCALED) {
              const float4& z = r[e / 2];
              const float2 of_value = (e & 1) ? make_float2(z.z, z.w) : make_float2(z.x, z.y);
              if constexpr (kWeighted) {
                y = fma2(score, c2v, add2(of_value, vv));
                y.x = ex2(y.x);
                y.y = ex2(y.y);
              } else {
                y = mul2(y, of_value);
              }
            }
            p[e] = tc::pack2<T>(y.x, y.y);
          }
          // over this half's own scores: the other half may not have read its yet
          tc::st16(s_addr + 16 * c, p);
          tc::wait_st();
          tc::fence_before();
          __syncwarp();
          // one arrival per warp: 256 of them would queue up at the barrier
          if (c == 0 && kEarly && lane == 0) tc::arrive(&bars.p_half[i]);
          if (c == 1 && lane == 0) tc::arrive(&bars.p_full[i]);
        }
        part = add2(part, part2);
        sum += part.x + part.y;
      }
      kt += all;
      if (count > 0) {
        ok = ok && tc::wait(&bars.o_full[i], no & 1);
        ++no;
        tc::fence_after();
        s_sum[i][half][row] = sum;
        if (tc::any_of(1 + i, 2 * kRows, !ok)) {
          ok = false;
          break;  // all warps of the tile
        }
        sum += s_sum[i][half ^ 1][row];
      }
      // the factor between the references, which a scale past 2^120 takes out of fp32's range, and fp16's anyway
      const float unit = kWeighted ? ex2(fminf(mv - kHalfShift - m * c2, 127.f)) : 1.f;
      const float inv = sum > 0.f ? unit / sum : sum == 0.f ? 0.f : sum;  // NaN stays
      tc::store_rows<T, DP / 2>(o_addr, out, half * (DP / 2), a.d, inv, live, f.wide_out, count > 0);
      if (!PAGED && a.low != nullptr) {
        T* low = static_cast<T*>(a.low) + ((x.t.batch * a.L + x.t.row0 + tok) * a.H + h) * a.d;
        tc::store_rows<T, DP / 2, true>(o_addr, low, half * (DP / 2), a.d, inv, live, f.wide_low, count > 0);
      }
      if (lse != nullptr) *lse = sum == 0.f ? neg_inf() : (m * c2 + log2f(kShift == 0.f ? sum : sum * 0x1p-7f)) * kLn2;
      tc::fence_before();  // O has been read before the next piece's first weights are announced
    }
    if (!ok && lane == 0) atomicExch(&g_tc_fwd_error, kDevTimeout);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kSoftmaxWarps) tc::dealloc(tmem, 512);
}

template <typename T, int DP, bool PAGED, bool SCALED>
cudaError_t launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FwdArgs& f, int64_t ctas,
                   cudaStream_t st) {
  return launch_grid<attn_tc_fwd_kernel<T, DP, PAGED, SCALED>>(false, ctas, kThreads, Layout<DP>::kSmem, st, q, k, v, f);
}

template <bool PAGED, bool SCALED>
cudaError_t dispatch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FwdArgs& f, int dtype,
                     int64_t ctas, cudaStream_t st) {
  if (dtype == kBF16)
    return f.a.d <= 64 ? launch<__nv_bfloat16, 64, PAGED, SCALED>(q, k, v, f, ctas, st)
                       : launch<__nv_bfloat16, 128, PAGED, SCALED>(q, k, v, f, ctas, st);
  return f.a.d <= 64 ? launch<__half, 64, PAGED, SCALED>(q, k, v, f, ctas, st)
                     : launch<__half, 128, PAGED, SCALED>(q, k, v, f, ctas, st);
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
  f.wide_out = row_alignment(a.o, a.os, nb, a.H);
  f.wide_low = row_alignment(a.low, AttnStrides{a.L * a.H * a.d, static_cast<int64_t>(a.H) * a.d, a.d}, nb, a.H);
  int64_t tiles;
  const int rows = 2 * f.tile_tokens;
  if (a.cu != nullptr) {
    tiles = packed_tiles(a.L, a.nseq, rows);
    f.a.tiles = static_cast<int>(tiles);
  } else {
    f.a.tiles = static_cast<int>((a.L + rows - 1) / rows);
    tiles = static_cast<int64_t>(f.a.tiles) * a.nseq;
  }
  // Causal: with little work the long pieces of all sequences go first, else the ends are uneven (16 sequences of
  // 1024, 16/4 heads of 128, 1024 pieces: 106 and 112 us); with much of it a sequence's pieces stay together for
  // the keys' sake (24 such sequences, 32/8 heads, three times the pieces: 281 and 266 us).
  const int64_t pieces = tiles * (a.H / f.pack);
  f.across = a.cu != nullptr || (a.causal && pieces <= 12 * num_sms_here());
  *e = dispatch<false, false>(q, k, v, f, dtype, pieces, st);
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
  f.across = 1;
  f.table_width = p.table_width;
  f.page = p.page;
  f.n_pages = p.n_pages;
  f.k_res = p.k_res;
  f.v_res = p.v_res;
  f.box = std::min(p.page & -p.page, kRows);  // the largest power of two that divides a page
  f.wide_out = row_alignment(a.o, a.os, 1, a.H);
  // expanded pages are contiguous
  const int64_t pages = p.k_res != nullptr ? static_cast<int64_t>(p.B) * p.table_width : p.n_pages;
  const AttnStrides dense{static_cast<int64_t>(p.page) * p.Hk * p.d, static_cast<int64_t>(p.Hk) * p.d, p.d};
  const AttnStrides ks = p.k_res != nullptr ? dense : AttnStrides{p.kc_sP, p.kc_sS, p.kc_sH};
  const AttnStrides vs = p.k_res != nullptr ? dense : AttnStrides{p.vc_sP, p.vc_sS, p.vc_sH};
  CUtensorMap q, k, v;
  if (!attn_map(&q, p.q, dtype, 1, p.T, p.H, p.d, a.qs, f.pack, f.tile_tokens) ||
      !attn_map(&k, p.k_cache, dtype, pages, p.page, p.Hk, p.d, ks, 1, f.box) ||
      !attn_map(&v, p.v_cache, dtype, pages, p.page, p.Hk, p.d, vs, 1, f.box))
    return false;
  const int64_t tiles = packed_tiles(p.T, p.B, 2 * f.tile_tokens);
  a.tiles = static_cast<int>(tiles);
  const int64_t pieces = tiles * (p.H / f.pack);
  *e = p.k_res != nullptr ? dispatch<true, true>(q, k, v, f, dtype, pieces, st)
                          : dispatch<true, false>(q, k, v, f, dtype, pieces, st);
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
