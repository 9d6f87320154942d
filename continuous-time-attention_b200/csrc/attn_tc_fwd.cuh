// What the two units of the tensor-core forward share (attn_tc_fwd.cu, attn_tc_fwd_reach.cu).
#pragma once

#include "attn_tc.cuh"

namespace cta {
namespace tcfwd {

constexpr int kThreads = 640;  // five warpgroups
constexpr int kSoftmaxWarps = 16;
constexpr int kRows = 128;  // rows of a tile, and keys of a step
constexpr float kLazy = 8.f;
// fp16 weights carry 2^7, and so stay below 2^15; what is lost to subnormals is below 2^-32 of the reference
constexpr float kHalfShift = 7.f;
static_assert(kHalfShift == 7.f, "lse takes 2^-7 of the sum");

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

}  // namespace tcfwd
}  // namespace cta
