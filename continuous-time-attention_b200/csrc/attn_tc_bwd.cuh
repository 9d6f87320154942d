// What the two units of the tensor-core backward share (attn_tc_bwd.cu, attn_tc_bwd_window.cu).
#pragma once

#include "attn_tc.cuh"

namespace cta {
namespace tcbwd {

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

}  // namespace tcbwd
}  // namespace cta
