// Attention forward on the tensor cores where rows do not see every key up to their own: prompts and chunks under a
// sliding window whose first keys stay visible, and the sums of a whole batch over the pages that all its sequences
// begin with.  The mathematics, the warps and the pipeline are those of attn_tc_fwd.cu, whose comments hold here too.
// What is different:
//
// * Window: the keys between the first ones and the windows of a piece's rows are passed over, in words of 32, so that
//   one step holds the first keys and where the windows begin; pages that no row of the piece sees are not loaded, nor are
//   their entries in the table trusted.
// * Prefix: the rows are those of all sequences, 256 (row, head) pairs to a piece, and the keys are cut into parts, so
//   that pieces fill the SMs; a part leaves its weighted values, maximum and sum in 32 bits for the join of the split
//   kernel (attn_paged.cu), which runs beside this one over the sequences' own keys.
// * Over e4m3 caches the scales' fractions come to shared memory with the values, and the keys' carry scale * log2(e).
//
// Bound like the forward by a step's chain of product, softmax and product, 2.0 us for the two tiles of a piece at dim
// 128, and by what a piece costs before and behind its steps, 5 to 6 us: in windows of 512 a piece of 64 tokens has five
// steps.  Measured, 32/8 heads of 128: 12 prompts of up to 4096 tokens, window 512, 4 first keys 417 us; chunks of 512 of 4
// sequences, window 1024, over e4m3 73 to 76 us; 64 rows over 8192 keys in 8 parts 38 us, in 16 parts 25
// (alone); 16384 tokens, 8 heads of 64, window 1024 105 us.
//
// Scores over e4m3 stay in registers in no variant: read from tensor memory a second time for the weights, chunks take 73 us;
// kept, with spills of 260 bytes, 94.
#include <algorithm>

#include "attn_tc_fwd.cuh"

namespace cta {

__device__ int g_tc_fwd_reach_error;

namespace {

using namespace tcfwd;

struct FwdArgs {
  AttnArgs a;
  int pack;          // heads per tile row block
  int tile_tokens;   // kRows / pack
  int warp_span;     // tokens from a warp's first row to its last
  int across;        // order of the work, see find_tile
  // paged keys
  const int32_t* table;
  int64_t table_sB;
  const int32_t* seq_lens;
  int table_width, page, n_pages, box;  // box: keys per TMA box
  // SCALED: page i of sequence b is page b * table_width + i, or with a window a key lies where CopySlots says (the table
  // still says which are valid), and these are what the expansion left out of its elements, see launch_cache_expand
  const float* k_res;
  const float* v_res;
  int copy_stride, copy_dense, copy_slots;
  int wide_out, wide_low;  // alignment of the outputs' rows, see store_rows
  // shared prefix: `splits` parts of `chunk` keys (whole tiles), whose sums go to part_o [splits, rows, heads, DP] and
  // part_ml [splits, rows, heads, 4] as the split kernel leaves them (attn_paged.cu)
  int splits, chunk, prefix;
  int64_t most_keys;  // of a sequence
  float* part_o;
  float* part_ml;
};

// what the two tiles of a piece go through
struct Plan {
  int first[2], steps[2], stop[2];  // first rows, steps, where the keys end
  int j0, edge, gap, shift;
  __device__ __forceinline__ int key(int at) const { return at + (at >= edge ? gap : 0); }
};

// kPrefix: all rows of a batch over the pages that it begins with
enum Form : int { kWindow = 0, kPrefix = 1 };
constexpr int kBox = 32;  // kWindow: keys per TMA box, see plan

// kPrefix: the last key that row `tok` sees, by its own sequence's length; rows behind the last sequence do not count
__device__ __forceinline__ int last_key(const FwdArgs& f, int tok) {
  const AttnArgs& a = f.a;
  int b = tok, from = tok, rows = 1;
  if (a.cu != nullptr) {
    // the last sequence that begins at or before the row
    int lo = 0, hi = a.nseq;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(a.cu + mid + 1) > tok) hi = mid;
      else lo = mid + 1;
    }
    if (lo == a.nseq) return 0x7fffffff;
    b = lo;
    int64_t begin;
    clamp_range(a.cu, b, a.L, begin, rows);
    from = static_cast<int>(begin);
  }
  const int n = static_cast<int>(min(static_cast<int64_t>(max(__ldg(f.seq_lens + b), 0)), f.most_keys));
  return n - rows + tok - from;
}

template <typename T, int DP, bool PAGED, bool SCALED, int FORM>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_reach_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
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
  // The keys' fractions carry scale * log2(e): one product less for each score.
  constexpr bool kFolded = SCALED;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ Item s_item;
  __shared__ __align__(16) uint4 s_answer;
  __shared__ float s_max[2][2][kRows], s_sum[2][2][kRows];  // [tile][half of the keys][row]
  __shared__ float s_maxv[kWeighted ? 2 : 1][2][kWeighted ? kRows : 1];
  __shared__ uint32_t s_boxes[16];  // paged: which boxes of a key tile were loaded
  // SCALED: the fractions of the key tiles in flight, keys' and values'.  They come with the values' tile, whose stage is
  // free only when the weights that need them are in O, so four of them are more than are in flight.
  __shared__ __align__(16) float s_res[SCALED ? 4 : 1][2][SCALED ? kRows : 1];
  const AttnArgs& a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
  if (FORM == kPrefix) pdl_launch_dependents();  // the split kernel's CTAs, for the sequences' own keys, may follow

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
  // Steps of 128 keys of the two tiles, from j0 on.  kWindow: the keys between the first ones and the windows are passed
  // over: the keys from `edge` on stand for those `gap` further on, so that a step may hold the first keys and where the
  // windows begin.  Words of 32 keys lie on one side.  (With the first keys in steps of their own, and windows from the
  // beginning of a whole tile, 12 prompts of up to 4096 tokens, 32/8 heads of 128, window 512, take 450 us instead of 417.)
  auto plan = [&](const Item& x) {
    Plan y;
    y.shift = PAGED && FORM != kPrefix ? x.n - x.t.n : 0;
    y.edge = 0x7fffffff;
    y.gap = 0;
    if constexpr (FORM == kWindow) {
      y.j0 = x.lo & ~31;
      const int from = max(x.lo, x.t.first + y.shift - a.window + 1) & ~31;
      const int edge = a.sinks == 0 ? y.j0 : (x.lo + a.sinks + 31) & ~31;
      if (from > edge) y.edge = edge, y.gap = from - edge;
    } else {
      y.j0 = x.lo / kRows * kRows;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      y.first[i] = x.t.first + i * f.tile_tokens;
      int end = x.hi;
      if (FORM == kWindow) end = min(end, min(y.first[i] + f.tile_tokens, x.t.n) + y.shift);
      if (end > y.edge) end = max(y.edge, end - y.gap);
      y.stop[i] = end;
      y.steps[i] = y.first[i] < x.t.n ? max(0, (end - y.j0 + kRows - 1) / kRows) : 0;
    }
    return y;
  };
  // first keys that stay visible to all: those before this one
  auto sinks_of = [&](const Item& x) { return FORM == kWindow && a.sinks > 0 ? x.lo + a.sinks : 0; };
  // A step of up to 32 keys takes a quarter of the products.  It pays where the softmax skips what no row of a warp
  // sees, which it does not at dim 128 over 16 bits: each step waits for the other tile there, and the votes cost more
  // than they save (12 prompts of up to 4096 tokens, 32/8 heads of 128, window 512: 451 and 424 us; 16384
  // tokens, 8 heads of 64, window 1024: 101 and 104; chunks of 512 over e4m3: 101 and 111).
  constexpr bool kSkip = FORM == kWindow && (SCALED || DP == 64);
  auto narrow = [&](int j0, int stop) { return kSkip && stop - j0 <= 32; };
  // bit c of word i: key c of the 32 that step j0's place 32 i stands for is one of the sequence's and valid; `kt`: running
  // number of the tile
  auto key_words = [&](int n, const uint32_t* mask, const Plan& y, int j0, int kt, uint32_t (&w)[4]) {
    const uint32_t boxes = PAGED ? *reinterpret_cast<volatile uint32_t*>(&s_boxes[kt & 15]) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = y.key(j0 + 32 * i);
      w[i] = ~tc::bits_from(n - at);
      if constexpr (PAGED) {
        if (!((boxes >> (2 * i)) & 1u)) w[i] &= 0xffff0000u;
        if (!((boxes >> (2 * i + 1)) & 1u)) w[i] &= 0x0000ffffu;
      } else if (mask != nullptr) {
        if (n - at > 0) w[i] &= __ldg(mask + (at >> 5));
      }
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
        if constexpr (FORM == kPrefix) {
          const int y = id / blocks, part = y % f.splits;
          x.t.n = static_cast<int>(a.L);
          x.t.first = y / f.splits * 2 * f.tile_tokens;
          x.lo = part * f.chunk;
          // what lies behind the longest sequence may hold anything
          int longest = 0;
          for (int b = lane; b < a.nseq; b += 32) longest = max(longest, __ldg(f.seq_lens + b));
          longest = __reduce_max_sync(0xffffffffu, longest);
          x.n = x.hi = min(min(f.prefix, x.lo + f.chunk), longest);
        } else {
          x.t = find_tile(a.cu, a.nseq, a.L, a.tiles, id / blocks, 2 * f.tile_tokens, true, f.across,
                          f.seq_lens);
          x.n = x.hi = x.t.n;
          if constexpr (PAGED) {
            if (x.t.first < x.t.n) {
              x.n = __ldg(f.seq_lens + x.t.seq);
              const int64_t most = static_cast<int64_t>(f.table_width) * f.page;
              if ((x.n < 0 || x.n > most) && lane == 0) atomicExch(&g_tc_fwd_reach_error, kDevBadIndex);
              x.n = x.n < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(x.n), most));
            }
            x.hi = x.n;
          } else {
            mask_range(a, x.t.batch, x.t.n, x.lo, x.hi);
          }
        }
      }
      if (lane == 0) {
        s_item = x;
        tc::arrive(&bars.item_full);
      }
      __syncwarp();
      if (id < 0) break;
    }
    if (!ok && lane == 0) atomicExch(&g_tc_fwd_reach_error, kDevTimeout);
   } else if (warp == kSoftmaxWarps + 1) {
    // ---------------- loads ----------------
    bool ok = true;
    int kv = 0, nq = 0;  // tiles loaded so far, Q loads so far
    for (int it = 0; ok; ++it) {
      Item x;
      ok = read_item(it, x);
      if (!ok || x.last) break;
      const Plan y = plan(x);
      const int all = max(y.steps[0], y.steps[1]);
      if (all == 0) {
        taken();
        continue;
      }
      constexpr bool kCopy = SCALED && FORM == kWindow;
      CopySlots copy = {};
      if constexpr (kCopy)
        copy = copy_slots(f.copy_stride, f.copy_dense, a.window, a.sinks, x.t.seq, x.t.row0, x.t.n, x.n);
      if (nq > 0) ok = tc::wait(&bars.q_empty, (nq - 1) & 1);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars.q_full, 2 * L::kTile);
        for (int i = 0; i < 2; ++i)
          for (int c = 0; c < DP / 64; ++c)
            tc::tma_load_4d(smem + i * L::kTile + c * L::kHalf, &qmap, &bars.q_full, 64 * c, x.h0,
                            static_cast<int>(x.t.row0) + y.first[i], x.t.batch);
      }
      ++nq;
      for (int step = 0; step < 2 * all; ++step) {
        const int stage = kv % NS, j0 = y.j0 + step / 2 * kRows;
        if (kv >= NS) ok = tc::wait(&bars.kv_empty[stage], ((kv / NS) - 1) & 1);
        if (!ok) break;
        const CUtensorMap* map = (step & 1) ? &vmap : &kmap;
        const uint32_t dst = smem + (2 + stage) * L::kTile;
        // one lane per box
        const int boxes = kRows / f.box, key = y.key(j0 + lane * f.box);
        if constexpr (PAGED) {
          // a box outside the sequence or the cache is left out
          int page = -1;
          // no row's window reaches it: the page may be gone
          const bool reached = FORM != kWindow || key < a.sinks || key + f.box > x.t.first + y.shift - a.window + 1;
          if (lane < boxes && key < x.n && reached) {
            page = __ldg(f.table + x.t.seq * f.table_sB + key / f.page);
            if (page < 0 || page >= f.n_pages) {
              atomicExch(&g_tc_fwd_reach_error, kDevBadIndex);
              page = -1;
            } else if (SCALED) {
              page = kCopy ? 0 : x.t.seq * f.table_width + key / f.page;
            }
          }
          const uint32_t got = __ballot_sync(0xffffffffu, page >= 0);
          // SCALED: lanes 0 to 3 fetch the keys' fractions, 32 each, the next four the values', with the values' tile; what
          // lies behind the row's end counts for nobody
          int64_t res_at = 0;
          uint32_t res = 0u;
          if (SCALED && (step & 1)) {
            const int64_t res_row = kCopy ? f.copy_slots : residue_row(static_cast<int64_t>(f.table_width) * f.page);
            const int res_key = y.key(j0 + (lane & 3) * 32), slot = kCopy ? copy.at(res_key) : res_key;
            res_at = (static_cast<int64_t>(kCopy ? 0 : x.t.seq) * a.Hk + x.hk) * res_row + slot;
            res = __ballot_sync(0xffffffffu, lane < 8 && slot >= 0 && slot < res_row);
          }
          if (lane == 0) {
            // one bit per 16 keys
            uint32_t bits = 0;
            const int per = f.box / 16;
            for (int b = 0; b < boxes; ++b)
              if ((got >> b) & 1u) bits |= ((1u << per) - 1u) << (b * per);
            *reinterpret_cast<volatile uint32_t*>(&s_boxes[(kv >> 1) & 15]) = bits;
            mbar_arrive_expect_tx(&bars.kv_full[stage], __popc(got) * f.box * 128 * (DP / 64) + __popc(res) * 128);
          }
          __syncwarp();
          if (SCALED && ((res >> lane) & 1u))
            tc::bulk_load(smem_addr(&s_res[(kv >> 1) & 3][lane >> 2][(lane & 3) * 32]), (lane < 4 ? f.k_res : f.v_res) + res_at,
                          128, &bars.kv_full[stage]);
          if (page >= 0)
            for (int c = 0; c < DP / 64; ++c)
              tc::tma_load_4d(dst + c * L::kHalf + lane * f.box * 128, map, &bars.kv_full[stage], 64 * c, x.hk,
                              kCopy ? copy.at(key) : key % f.page, page);
        } else {
          if (lane == 0) mbar_arrive_expect_tx(&bars.kv_full[stage], L::kTile);
          __syncwarp();
          if (lane < boxes)
            for (int c = 0; c < DP / 64; ++c)
              tc::tma_load_4d(dst + c * L::kHalf + lane * f.box * 128, map, &bars.kv_full[stage], 64 * c, x.hk,
                              static_cast<int>(x.t.row0) + key, x.t.batch);
        }
        ++kv;
      }
      taken();
    }
    // nothing may still be in flight when the CTA ends: the MMA warp has waited for all of it unless a wait ran out
    if (!ok) {
      atomicExch(&g_tc_fwd_reach_error, kDevTimeout);
      for (int y = max(0, kv - NS); y < kv; ++y) tc::wait(&bars.kv_full[y % NS], (y / NS) & 1);
      if (nq > 0) tc::wait(&bars.q_full, (nq - 1) & 1);
    }
   } else {
    // ---------------- products ----------------
    // One warp per row tile: a successful wait costs a hundred cycles or more, and with one warp for
    // both tiles those of one tile delayed the other's products (562 instead of 503 us at 8192 keys,
    // 16 heads of 128, 477 instead of 402 at 64).  Both free a key tile.
    const int i = warp == kSoftmaxWarps ? 0 : 1;
    constexpr uint32_t id_s = tc::idesc<T>(kRows, false), id_32 = tc::idesc<T>(32, false), id_o = tc::idesc<T>(DP, true);
    const bool leader = tc::elect_one();
    bool ok = true;
    int kv = 0, nq = 0, ns = 0;  // running numbers: tiles, Q loads, steps of this row tile
    const uint32_t t_s = tmem + i * kRows, t_o = tmem + 2 * kRows + i * DP, q = smem + i * L::kTile;
    for (int it = 0; ok; ++it) {
      Item x;
      ok = take(it, x);
      if (!ok || x.last) break;
      const Plan y = plan(x);
      const int all = max(y.steps[0], y.steps[1]), mine = i == 0 ? y.steps[0] : y.steps[1];
      const int stop = i == 0 ? y.stop[0] : y.stop[1];
      if (all == 0) continue;
      ok = tc::wait(&bars.q_full, nq & 1);
      ++nq;
      const uint32_t* mask = !PAGED && a.mask != nullptr ? a.mask + x.t.batch * a.mask_words + kMaskHead : nullptr;
      auto kv_wait = [&](int z) { ok = ok && tc::wait(&bars.kv_full[(kv + z) % NS], ((kv + z) / NS) & 1); };
      auto kv_addr = [&](int z) { return smem + (2 + (kv + z) % NS) * L::kTile; };
      // scores of step j into the tile's buffer; keys are released by the step's end
      auto scores = [&](int j, int at) {
        tc::product_nt<DP>(t_s, q, kv_addr(2 * j), narrow(at, stop) ? id_32 : id_s);
        tc::commit(&bars.s_full[i]);
        if (j + 1 == mine) tc::commit(&bars.q_empty);
      };
      kv_wait(0);
      tc::fence_after();
      if (ok && leader) {
        if (mine > 0) scores(0, y.j0);
        else tc::commit(&bars.q_empty);
        tc::commit(&bars.kv_empty[kv % NS]);
      }
      __syncwarp();
      for (int j = 0, j0 = y.j0; j < all && ok; ++j, j0 += kRows) {
        kv_wait(2 * j + 1);
        if (j + 1 < all) kv_wait(2 * j + 2);
        if (!ok) break;
        if (j < mine) {
          // values of keys that are not there or not valid may hold anything
          uint32_t w[4];
          if (PAGED || mask != nullptr || y.key(j0 + kRows - 1) >= x.n) {
            key_words(x.n, mask, y, j0, (kv >> 1) + j, w);
            if (!tc::all_set(w)) tc::clear_rows<DP / 64>(kv_addr(2 * j + 1), w);
          }
          // (Issuing the products of half the keys ahead of the others was tried: it costs more than it
          // hides, 643 instead of 534 us at 8192 keys, 16 heads of 128.)
          if (kEarly) ok = tc::wait(&bars.p_half[i], ns & 1);
          ok = ok && tc::wait(&bars.p_full[i], ns & 1);
          tc::fence_after();
          if (ok && leader) {
            if (narrow(j0, stop)) tc::product_tn<64, 2>(t_o, t_s, kv_addr(2 * j + 1), id_o, j > 0);
            else tc::product_tn<64>(t_o, t_s, kv_addr(2 * j + 1), id_o, j > 0);
            if (j + 1 == mine) {
              tc::commit(&bars.o_full[i]);
            } else {
              scores(j + 1, j0 + kRows);
            }
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
    if (!ok && lane == 0) atomicExch(&g_tc_fwd_reach_error, kDevTimeout);
   }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    // ---------------- softmax ----------------
    const int i = warp >> 3, half = (warp >> 2) & 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + i * kRows + half * 64;
    const uint32_t o_addr = tmem + lanes + 2 * kRows + i * DP + half * (DP / 2);
    const float c2 = kFolded ? 1.f : a.scale * kLog2e;
    bool ok = true;
    int ns = 0, no = 0, kt = 0;  // running numbers: steps, outputs, key tiles
    for (int it = 0; ok; ++it) {
      Item x;
      ok = take(it, x);
      if (!ok || x.last) break;
      const Plan y = plan(x);
      const int mine = i == 0 ? y.first[0] : y.first[1], count = i == 0 ? y.steps[0] : y.steps[1];
      const int all = max(y.steps[0], y.steps[1]);
      if (!PAGED && a.cu != nullptr && a.zero_tail && warp < 4 && x.t.n == 0) {
        // a tile behind the last sequence clears rows there
        for (int64_t r = x.t.row0 + x.t.tail_index; r < a.L; r += x.t.tail_count)
          for (int c = threadIdx.x; c < a.d * f.pack; c += kRows)
            static_cast<T*>(a.o)[r * a.os.t + (x.h0 + c / a.d) * a.os.h + c % a.d] = Elem<T>::from_f(0.f);
      }
      if (mine >= x.t.n) {
        kt += all;
        continue;
      }
      const int n = x.n;
      const uint32_t* mask = !PAGED && a.mask != nullptr ? a.mask + x.t.batch * a.mask_words + kMaskHead : nullptr;
      const int tok = mine + row / f.pack, h = x.h0 + row % f.pack;
      const bool live = tok < x.t.n;
      int limit = tok + y.shift;                                  // last key the row sees
      int limit_all = mine + (warp & 3) * 32 / f.pack + y.shift;  // and that all rows of the warp see
      if constexpr (FORM == kPrefix) {
        // of its own sequence, which may end here
        limit = live ? min(n - 1, last_key(f, tok)) : n - 1;
        limit_all = __reduce_min_sync(0xffffffffu, limit);
      }
      T* out = static_cast<T*>(a.o) + x.t.batch * a.os.b + (x.t.row0 + tok) * a.os.t + h * a.os.h;
      float* lse = live && half == 0 && a.lse != nullptr ? a.lse + lse_index(a, x.t, h, tok) : nullptr;
      const int sink_end = sinks_of(x);
      float m = neg_inf(), sum = 0.f;
      float mv = neg_inf();  // kWeighted: the reference of weight * scale, as an exponent of two
      for (int j = 0, j0 = y.j0; j < count; ++j, ++ns, j0 += kRows) {
        // After a wait that ran out a warp goes on without waiting to the end of the piece, so that
        // the named barriers below see all their warps.
        ok = ok && tc::wait(&bars.s_full[i], ns & 1);
        if (SCALED) ok = ok && tc::wait(&bars.kv_full[(2 * (kt + j) + 1) % NS], ((2 * (kt + j) + 1) / NS) & 1);
        tc::fence_after();
        uint32_t s[2][32];
        if (!SCALED) {
          tc::ld32(s_addr, s[0]);
          tc::ld32(s_addr + 32, s[1]);
        }
        // warp-uniform: every row of the warp sees all keys of the tile
        const int k0 = y.key(j0), k1 = y.key(j0 + kRows - 1);
        bool whole = k1 < n && k1 <= limit_all &&
                     (FORM != kWindow || k0 > limit_all + f.warp_span - a.window || k1 < sink_end);
        uint32_t w[4];
        if (PAGED || mask != nullptr || !whole) {
          key_words(n, mask, y, j0, kt + j, w);
          whole = whole && tc::all_set(w);
        }
        if (!SCALED) tc::wait_ld(s[0], s[1]);
        // Fractions of the scales, 32 keys at a time: the scores are read from tensor memory once for the maximum and
        // once for the weights, for want of registers.  From shared memory, where the loads' warp puts them: the
        // softmax waited for them 56 % of its time when each warp fetched them (512 rows of 4 sequences in windows
        // of 1024, 32/8 heads of 128: 106 and 83 us; 128 rows in fp16 over a prefix of 16384: 120 and 93).
        auto fractions = [&](int of, int c, float4 (&r)[8]) {
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = *reinterpret_cast<const float4*>(&s_res[(kt + j) & 3][of][64 * half + 32 * c + 4 * e]);
        };
        auto scale = [&](int c, uint32_t (&x)[32]) {
          tc::ld32(s_addr + 32 * c, x);
          float4 r[8];
          fractions(0, c, r);
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
        // false: none of these 32 keys counts for any row of the warp (kSkip; x is left as it is)
        auto hide = [&](int c, uint32_t (&x)[32]) -> bool {
          const int at = y.key(j0 + 64 * half + 32 * c), left = limit - at + 1;
          uint32_t see =
              (half == 0 ? w[c] : w[2 + c]) & (left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u);
          if constexpr (FORM == kWindow) see &= tc::bits_from(left - a.window) | ~tc::bits_from(sink_end - at);
          if constexpr (kSkip) {
            if (!__any_sync(0xffffffffu, see != 0u)) return false;
            if (__all_sync(0xffffffffu, see == 0xffffffffu)) return true;
          }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((see >> e) & 1u)) x[e] = 0xff800000u;
          return true;
        };
        bool some[2] = {true, true};
        float t[4], topv = mv;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t(&x)[32] = s[SCALED ? 0 : c];
          if (SCALED) scale(c, x);
          if (!whole) some[c] = hide(c, x);
          if (kSkip && !some[c]) {
            t[2 * c] = t[2 * c + 1] = neg_inf();
            continue;
          }
          if constexpr (kWeighted) {
            // score + logarithm of the value's scale
            float4 r[8];
            fractions(1, c, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 a0 = make_float2(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]));
              const float2 a1 = make_float2(__uint_as_float(x[4 * e + 2]), __uint_as_float(x[4 * e + 3]));
              const float2 v0 = make_float2(r[e].x, r[e].y), v1 = make_float2(r[e].z, r[e].w);
              const float2 lo = kFolded ? add2(a0, v0) : fma2(a0, f2(c2), v0);
              const float2 hi = kFolded ? add2(a1, v1) : fma2(a1, f2(c2), v1);
              topv = tc::max3(tc::max3(lo.x, lo.y, hi.x), hi.y, topv);
            }
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            float& z = t[2 * c + b];
            z = __uint_as_float(x[16 * b]);
#pragma unroll
            for (int e = 1; e < 15; e += 2)
              z = tc::max3(z, __uint_as_float(x[16 * b + e]), __uint_as_float(x[16 * b + e + 1]));
            z = fmaxf(z, __uint_as_float(x[16 * b + 15]));
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
          if (kSkip && !some[c]) {
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = 0u;
          } else {
            if constexpr (SCALED) {
              scale(c, x);
              if (!whole) hide(c, x);
              fractions(1, c, r);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 score = make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
              float2 w2 = kFolded ? add2(score, bv) : fma2(score, c2v, bv);
              w2.x = ex2(w2.x);
              w2.y = ex2(w2.y);
              if (e & 1) part2 = add2(part2, w2);
              else part = add2(part, w2);
              if constexpr (SCALED) {
                const float4& z = r[e / 2];
                const float2 of_value = (e & 1) ? make_float2(z.z, z.w) : make_float2(z.x, z.y);
                if constexpr (kWeighted) {
                  w2 = kFolded ? add2(score, add2(of_value, vv)) : fma2(score, c2v, add2(of_value, vv));
                  w2.x = ex2(w2.x);
                  w2.y = ex2(w2.y);
                } else {
                  w2 = mul2(w2, of_value);
                }
              }
              p[e] = tc::pack2<T>(w2.x, w2.y);
            }
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
      if constexpr (FORM == kPrefix) {
        // The part's sums as they are.  The join takes it that values of half products carry 2^7; bf16 weights over e4m3
        // codes do not.
        constexpr float kUnit = SCALED && !kWeighted ? 128.f : 1.f;
        const int64_t at = (static_cast<int64_t>(x.lo / f.chunk) * a.L + tok) * a.H + h;
        tc::store_floats<DP / 2>(o_addr, f.part_o + at * DP + half * (DP / 2), kUnit, live, count > 0);  // or the part lies behind all sequences
        if (live && half == 0)
          *reinterpret_cast<float4*>(f.part_ml + at * 4) =
              make_float4(m * c2, kShift == 0.f ? sum : sum * 0x1p-7f, kWeighted ? mv : m * c2, 0.f);
        tc::fence_before();
        continue;
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
    if (!ok && lane == 0) atomicExch(&g_tc_fwd_reach_error, kDevTimeout);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == kSoftmaxWarps) tc::dealloc(tmem, 512);
}

template <typename T, int DP, bool PAGED, bool SCALED, int FORM>
cudaError_t launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FwdArgs& f, int64_t ctas,
                   cudaStream_t st) {
  return launch_grid<attn_tc_reach_kernel<T, DP, PAGED, SCALED, FORM>>(false, ctas, kThreads, Layout<DP>::kSmem, st, q, k, v, f);
}

template <bool PAGED, bool SCALED, int FORM>
cudaError_t dispatch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const FwdArgs& f, int dtype,
                     int64_t ctas, cudaStream_t st) {
  if (dtype == kBF16)
    return f.a.d <= 64 ? launch<__nv_bfloat16, 64, PAGED, SCALED, FORM>(q, k, v, f, ctas, st)
                       : launch<__nv_bfloat16, 128, PAGED, SCALED, FORM>(q, k, v, f, ctas, st);
  return f.a.d <= 64 ? launch<__half, 64, PAGED, SCALED, FORM>(q, k, v, f, ctas, st)
                     : launch<__half, 128, PAGED, SCALED, FORM>(q, k, v, f, ctas, st);
}

}  // namespace

bool launch_attn_tc_fwd_window(const AttnArgs& a, int dtype, cudaStream_t st, cudaError_t* e) {
  if (dtype == kF32 || a.d % 8 != 0 || a.d > 128 || !(a.scale > 0.f)) return false;
  FwdArgs f = {};
  f.a = a;
  f.pack = attn_pack(a.H / a.Hk);
  f.tile_tokens = kRows / f.pack;
  f.warp_span = 31 / f.pack;
  f.box = kBox;
  const int64_t nb = a.cu != nullptr ? 1 : a.nseq;
  CUtensorMap q, k, v;
  if (!attn_map(&q, a.q, dtype, nb, a.L, a.H, a.d, a.qs, f.pack, f.tile_tokens) ||
      !attn_map(&k, a.k, dtype, nb, a.L, a.Hk, a.d, a.ks, 1, kBox) ||
      !attn_map(&v, a.v, dtype, nb, a.L, a.Hk, a.d, a.vs, 1, kBox))
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
  f.across = a.cu != nullptr || pieces <= 12 * num_sms_here();
  *e = dispatch<false, false, kWindow>(q, k, v, f, dtype, pieces, st);
  return true;
}

namespace {

// what chunks and prefixes have in common: the tensors and the pages
bool paged_maps(const PagedArgs& p, int dtype, int most_box, FwdArgs& f, CUtensorMap (&maps)[3]) {
  if (!(p.scale > 0.f)) return false;
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
  a.scale = p.scale;
  f.pack = attn_pack(p.H / p.Hk);
  f.tile_tokens = kRows / f.pack;
  f.warp_span = 31 / f.pack;
  f.table = p.table;
  f.table_sB = p.table_sB;
  f.seq_lens = p.seq_lens;
  f.table_width = p.table_width;
  f.page = p.page;
  f.n_pages = p.n_pages;
  f.k_res = p.k_res;
  f.v_res = p.v_res;
  f.box = std::min(p.page & -p.page, most_box);  // the largest power of two that divides a page
  // expanded pages are contiguous, the keys of a window one page
  const bool copy = p.k_res != nullptr && p.window > 0;
  f.copy_stride = p.copy_stride;
  f.copy_dense = p.copy_dense;
  f.copy_slots = static_cast<int>(p.copy_slots);
  const int64_t pages = copy ? 1 : p.k_res != nullptr ? p.expanded_pages : p.n_pages, page = copy ? p.copy_slots : p.page;
  const AttnStrides dense{page * p.Hk * p.d, static_cast<int64_t>(p.Hk) * p.d, p.d};
  const AttnStrides ks = p.k_res != nullptr ? dense : AttnStrides{p.kc_sP, p.kc_sS, p.kc_sH};
  const AttnStrides vs = p.k_res != nullptr ? dense : AttnStrides{p.vc_sP, p.vc_sS, p.vc_sH};
  return attn_map(&maps[0], p.q, dtype, 1, p.T, p.H, p.d, a.qs, f.pack, f.tile_tokens) &&
         attn_map(&maps[1], p.k_cache, dtype, pages, page, p.Hk, p.d, ks, 1, f.box) &&
         attn_map(&maps[2], p.v_cache, dtype, pages, page, p.Hk, p.d, vs, 1, f.box);
}

}  // namespace

bool launch_paged_tc_window(const PagedArgs& p, int dtype, cudaStream_t st, cudaError_t* e) {
  if (p.cu == nullptr) return false;
  FwdArgs f = {};
  CUtensorMap m[3];
  if (!paged_maps(p, dtype, kBox, f, m)) return false;
  f.a.causal = 1;
  f.a.window = p.window;
  f.a.sinks = p.sinks;
  f.across = 1;
  f.wide_out = row_alignment(f.a.o, f.a.os, 1, f.a.H);
  const int64_t tiles = packed_tiles(p.T, p.B, 2 * f.tile_tokens);
  f.a.tiles = static_cast<int>(tiles);
  const int64_t pieces = tiles * (p.H / f.pack);
  *e = p.k_res != nullptr ? dispatch<true, true, kWindow>(m[0], m[1], m[2], f, dtype, pieces, st)
                          : dispatch<true, false, kWindow>(m[0], m[1], m[2], f, dtype, pieces, st);
  return true;
}

// row tiles of 256 (row, head) pairs
int64_t prefix_tiles(const PagedArgs& p) {
  const int64_t rows = 2 * (kRows / attn_pack(p.H / p.Hk));
  return (p.T + rows - 1) / rows * (p.H / attn_pack(p.H / p.Hk));
}

bool launch_prefix_tc(const PagedArgs& p, int dtype, cudaStream_t st, cudaError_t* e) {
  FwdArgs f = {};
  CUtensorMap m[3];
  if (!paged_maps(p, dtype, kRows, f, m)) return false;
  f.splits = p.prefix_splits;
  f.chunk = p.prefix_chunk;
  f.prefix = p.skip;
  f.table_width = p.skip / p.page;
  f.most_keys = static_cast<int64_t>(p.table_width) * p.page;
  f.part_o = p.prefix_o;
  f.part_ml = p.prefix_ml;
  const int64_t pieces = prefix_tiles(p) * f.splits;
  *e = p.k_res != nullptr ? dispatch<true, true, kPrefix>(m[0], m[1], m[2], f, dtype, pieces, st)
                          : dispatch<true, false, kPrefix>(m[0], m[1], m[2], f, dtype, pieces, st);
  return true;
}

int read_device_error_tc_fwd_reach(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_tc_fwd_reach_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_tc_fwd_reach_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace cta
