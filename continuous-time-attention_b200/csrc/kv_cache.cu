// Writing new keys and values into a paged cache, and reading slots back.
//
// A 16-bit cache takes the rows as they are.  An e4m3 cache takes, per token
// and head,  s = m / 448,  code = e4m3(448 x / m)  with m = max(max|x|,
// 2^-100): one pass over the row, the maximum by shuffles between the 16 (or,
// above 128 elements, 32) lanes that hold it.  The floor of m keeps the quotient
// finite, so a row of zeros needs no case of its own.  Where 7 divides m's
// fraction, 448 x / m is often in the middle of two codes, and x times a rounded
// 448 / m goes to either; so 448 x is formed exactly, multiplied by the rounded
// reciprocal of m, and the quotient corrected once by its remainder, which a fused
// multiply-add gives exactly (Markstein 1990).  A tie has 5 bits, and what the
// correction is off by, 2^-24 of a few units in the last place, rounds away; any
// other quotient lies at least 2^-17 from one, since 448 x and the tie times m are
// whole numbers of up to 17 bits.
// Reading back multiplies code by s in 32 bits and rounds once to the tensor's type.
//
// Its floor is HBM: 2 d bytes read and d + 4 (2 d) written per row; the e4m3 forms are
// bound by issue (in 74 to 78 % of the cycles), the 16-bit ones by HBM.  Each lane
// moves 16 bytes of the 16-bit row; kHeads rows per group of lanes are in flight
// together.  Measured: 16384 tokens of 8 heads of 128 into e4m3, 101 MB, 23 us (21
// without the correction), and back 17 us; 16-bit cache, 134 MB, 22 and 20 us, 6.0 and
// 6.7 TB/s in part from L2; 64 tokens 2 us each.
#include <algorithm>

#include "attn_common.cuh"

namespace cta {

__device__ int g_cache_error;

namespace {

constexpr float kE4m3Max = 448.f;
constexpr float kLeastMax = 7.888609052210118e-31f;  // 2^-100
constexpr int kThreads = 256;
constexpr int kHeads = 4;  // rows of a token per group of lanes

__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
__device__ __forceinline__ float2 from_e4m3x2(uint16_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <typename T>
__device__ __forceinline__ void unpack8(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::unpack(*reinterpret_cast<const typename Elem<T>::Pair*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const typename Elem<T>::Pair p = Elem<T>::pack(make_float2(x[2 * i], x[2 * i + 1]));
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// m = 2^n * fraction(m), in [1, 2)
__device__ __forceinline__ float fraction(float m) {
  return __uint_as_float((__float_as_uint(m) & 0x007fffffu) | 0x3f800000u);
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A group of GROUP lanes holds a row of at most 8 GROUP elements and takes
// kHeads consecutive heads of one token: the slot and its page are found once,
// the rows' loads are in flight together, and the divisions of all of them are
// one, each lane doing one row's.  gridDim.y: 0 keys, 1 values.
struct Place {
  unsigned t;   // token
  int h0;       // first head
  bool any;     // there is such a token
  int64_t slot;
};
template <int GROUP>
__device__ __forceinline__ Place place(const CacheArgs& a) {
  const unsigned group = (blockIdx.x * kThreads + threadIdx.x) / GROUP;
  const unsigned blocks = (a.Hk + kHeads - 1) / kHeads;
  Place p;
  p.t = group / blocks;
  p.h0 = static_cast<int>(group - p.t * blocks) * kHeads;
  p.any = p.t < static_cast<unsigned>(a.T);
  p.slot = p.any ? __ldg(a.slots + p.t) : -1;
  return p;
}
// past the cache: reported, and treated as padding
__device__ __forceinline__ bool in_cache(const CacheArgs& a, int64_t slot, bool report) {
  if (slot >= a.n_slots && report) atomicExch(&g_cache_error, kDevBadIndex);
  return slot >= 0 && slot < a.n_slots;
}

template <typename T, int GROUP, bool QUANT>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const __grid_constant__ CacheArgs a) {
  const bool second = blockIdx.y != 0;
  const T* in = static_cast<const T*>(second ? a.v_in : a.k_in);
  const int64_t sT = second ? a.v_sT : a.k_sT, sH = second ? a.v_sH : a.k_sH;
  const int64_t cP = second ? a.vc_sP : a.kc_sP, cS = second ? a.vc_sS : a.kc_sS, cH = second ? a.vc_sH : a.kc_sH;
  const int lane = threadIdx.x % GROUP, c = lane * 8;
  const Place at = place<GROUP>(a);
  uint4 x[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (at.any && at.h0 + i < a.Hk && c < a.d)
      x[i] = __ldg(reinterpret_cast<const uint4*>(in + at.t * sT + (at.h0 + i) * sH + c));
  }
  const bool keep = in_cache(a, at.slot, lane == 0);
  const unsigned page = static_cast<unsigned>(at.slot) / a.page, slot = static_cast<unsigned>(at.slot) - page * a.page;
  const int64_t base = page * cP + slot * cS + at.h0 * cH + c;
  if constexpr (QUANT) {
    uint8_t* cache = static_cast<uint8_t*>(second ? a.v_cache : a.k_cache);
    float* scale = second ? a.v_scale : a.k_scale;
    float m[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      float f[8];
      unpack8<T>(x[i], f);
      m[i] = kLeastMax;
#pragma unroll
      for (int e = 0; e < 8; ++e) m[i] = fmaxf(m[i], fabsf(f[e]));
#pragma unroll
      for (int o = 1; o < GROUP; o <<= 1) m[i] = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
    }
    // lane i of the first kHeads: 1 / the fraction of m[i], lane kHeads + i: m[i] / 448
    float mine = m[0];
#pragma unroll
    for (int i = 1; i < kHeads; ++i) mine = (lane % kHeads) == i ? m[i] : mine;
    const bool up = (lane / kHeads) % 2 == 0;
    const float ratio = __fdiv_rn(up ? 1.f : mine, up ? fraction(mine) : kE4m3Max);
    if (keep && lane >= kHeads && lane < 2 * kHeads && at.h0 + lane - kHeads < a.Hk)
      scale[(static_cast<int64_t>(page) * a.Hk + at.h0 + lane - kHeads) * a.page + slot] = ratio;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const float r = __shfl_sync(0xffffffffu, ratio, i, GROUP);
      const float2 rr = f2(r), div = f2(-fraction(m[i]));
      // 448 over m's power of two; an infinite m has one too
      const float2 num = f2(__uint_as_float(((262u - (__float_as_uint(m[i]) >> 23)) << 23) | 0x600000u));
      float f[8];
      unpack8<T>(x[i], f);
      float2 q[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = mul2(make_float2(f[2 * e], f[2 * e + 1]), num), q0 = mul2(y, rr);
        q[e] = fma2(fma2(q0, div, y), rr, q0);
      }
      uint2 code;
      code.x = to_e4m3x4(q[0].x, q[0].y, q[1].x, q[1].y);
      code.y = to_e4m3x4(q[2].x, q[2].y, q[3].x, q[3].y);
      if (keep && c < a.d && at.h0 + i < a.Hk) *reinterpret_cast<uint2*>(cache + base + i * cH) = code;
    }
  } else {
    T* cache = static_cast<T*>(second ? a.v_cache : a.k_cache);
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (keep && c < a.d && at.h0 + i < a.Hk) *reinterpret_cast<uint4*>(cache + base + i * cH) = x[i];
  }
}

template <typename T, int GROUP, bool QUANT>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ CacheArgs a) {
  const bool second = blockIdx.y != 0;
  T* out = static_cast<T*>(second ? a.v_out : a.k_out);
  const int64_t sT = second ? a.v_sT : a.k_sT, sH = second ? a.v_sH : a.k_sH;
  const int64_t cP = second ? a.vc_sP : a.kc_sP, cS = second ? a.vc_sS : a.kc_sS, cH = second ? a.vc_sH : a.kc_sH;
  const int lane = threadIdx.x % GROUP, c = lane * 8;
  const Place at = place<GROUP>(a);
  if (!at.any || c >= a.d) return;
  const bool have = in_cache(a, at.slot, lane == 0);
  const unsigned page = static_cast<unsigned>(at.slot) / a.page, slot = static_cast<unsigned>(at.slot) - page * a.page;
  const int64_t base = page * cP + slot * cS + at.h0 * cH + c;
  uint4 x[kHeads];
  float mul[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    mul[i] = 0.f;
    if (!have || at.h0 + i >= a.Hk) continue;
    if constexpr (QUANT) {
      const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(second ? a.v_cache : a.k_cache) + base + i * cH);
      x[i].x = w.x;
      x[i].y = w.y;
      mul[i] = (second ? a.v_scale : a.k_scale)[(static_cast<int64_t>(page) * a.Hk + at.h0 + i) * a.page + slot];
    } else {
      x[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(second ? a.v_cache : a.k_cache) + base + i * cH);
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (at.h0 + i >= a.Hk) continue;
    uint4 y = x[i];
    if constexpr (QUANT) {
      float f[8];
      const uint32_t w[2] = {x[i].x, x[i].y};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = from_e4m3x2(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
        f[2 * e] = v.x * mul[i];
        f[2 * e + 1] = v.y * mul[i];
      }
      y = pack8<T>(f);
    }
    *reinterpret_cast<uint4*>(out + at.t * sT + (at.h0 + i) * sH + c) = y;
  }
}

// Codes of the pages of each sequence, in order, as exact 16-bit rows.  bf16, whose exponents reach as far as fp32's:
// each times the power of two below its scale, whose fraction goes into k_res and v_res.  fp16: the codes alone, and
// beside them the key's scale and the logarithm of the value's (attn_tc_fwd.cu says why).  fold_scale: what is for
// the keys carries what takes a score to an exponent of two.  Window: `per_seq` is copy_stride, and the groups behind
// those of all sequences are the slots that they have for their rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) cache_expand_kernel(const __grid_constant__ PagedArgs a, T* k_out, T* v_out,
                                                                float* k_res, float* v_res, unsigned per_seq) {
  constexpr int GROUP = 16;
  const bool second = blockIdx.y != 0;
  const unsigned blocks = (a.Hk + kHeads - 1) / kHeads;
  const unsigned group = (blockIdx.x * kThreads + threadIdx.x) / GROUP;
  const unsigned slots = static_cast<unsigned>(a.table_width) * a.page;  // per sequence
  const unsigned at = group / blocks;
  unsigned b = at / per_seq, j = at - b * per_seq;
  const int h0 = static_cast<int>(group - at * blocks) * kHeads, lane = threadIdx.x % GROUP, c = lane * 8;
  if (a.window > 0 && at >= a.copy_slots) return;
  if (b >= static_cast<unsigned>(a.B)) {
    if (a.window == 0 || !a.copy_dense) return;
    // the last sequence whose rows begin in or before this slot's tile
    const unsigned t = at - static_cast<unsigned>(a.B) * per_seq;
    unsigned last = a.B - 1;
    int64_t begin;
    int rows;
    for (b = 0; b < last;) {
      const unsigned mid = (b + last + 1) / 2;
      clamp_range(a.cu, mid, a.T, begin, rows);
      if (static_cast<unsigned>(begin) / 128 * 128 <= t) b = mid;
      else last = mid - 1;
    }
    clamp_range(a.cu, b, a.T, begin, rows);
    if (t < static_cast<unsigned>(begin) / 128 * 128) return;
    j = per_seq + t - static_cast<unsigned>(begin) / 128 * 128;
  }
  // nullptr: all of the table; a length past it ends with it, as for the kernel that reads the pages (and reports it)
  const int n = a.seq_lens != nullptr ? min(max(__ldg(a.seq_lens + b), 0), static_cast<int>(slots)) : static_cast<int>(slots);
  int low = 0;  // window: the first key that the first row's window holds
  unsigned row = b * slots + j;  // where the key goes
  if (a.window > 0) {
    int64_t begin;
    int rows;
    clamp_range(a.cu, b, a.T, begin, rows);
    low = max(n - rows - a.window + 1, 0);
    const CopySlots copy = copy_slots(per_seq, a.copy_dense, a.window, a.sinks, b, begin, rows, n);
    row = copy.base + j;
    if (a.copy_dense) {
      // no further than the rows reach: what follows is the next sequence's
      if (j >= static_cast<unsigned>(copy.first + residue_row(a.window + rows + 127))) return;
      if (j >= static_cast<unsigned>(copy.first)) j += copy.gap;
    }
  }
  if (j >= slots) return;
  // what goes beside this key, and behind the last key up to the tile's end
  const int64_t res_row = a.window > 0 ? a.copy_slots : residue_row(slots);
  float* res = (second ? v_res : k_res) + (a.window > 0 ? h0 * res_row + row : (static_cast<int64_t>(b) * a.Hk + h0) * res_row + j);
  if (j + 1 == slots)
    for (int i = 0; i < kHeads && h0 + i < a.Hk; ++i)
      for (int x = 1 + lane; x <= residue_row(slots) - slots; x += GROUP) res[i * res_row + x] = 1.f;
  if (c >= a.d) return;
  bool there = j < static_cast<unsigned>(n);
  if (a.window > 0) {
    // Left out where no row's window reaches, but for boxes that the reader loads whole: what lies beside a key that
    // counts meets a zero weight, and must not be NaN.
    const int box = min(a.page & -a.page, 128), first = static_cast<int>(j) / box * box;
    there = there && (first < a.sinks || first + box > low);
  }
  const int page = there ? __ldg(a.table + b * a.table_sB + j / a.page) : -1;
  if (page < 0 || page >= a.n_pages) {
    // not there, or reported by the kernel that reads the pages, which leaves it out
    if (lane == 0)
      for (int i = 0; i < kHeads && h0 + i < a.Hk; ++i) res[i * res_row] = 1.f;
    return;
  }
  const unsigned slot = j % a.page;
  const uint8_t* in = static_cast<const uint8_t*>(second ? a.v_cache : a.k_cache) + c +
                      page * (second ? a.vc_sP : a.kc_sP) + slot * (second ? a.vc_sS : a.kc_sS);
  const int64_t sH = second ? a.vc_sH : a.kc_sH;
  const float* scale = (second ? a.v_scale : a.k_scale) + static_cast<int64_t>(page) * a.Hk * a.page + slot;
  T* out = (second ? v_out : k_out) + static_cast<int64_t>(row) * a.Hk * a.d + c;
  uint2 w[kHeads];
  float mul[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (h0 + i < a.Hk) {
      w[i] = __ldg(reinterpret_cast<const uint2*>(in + (h0 + i) * sH));
      mul[i] = __ldg(scale + (h0 + i) * a.page);
    }
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (h0 + i < a.Hk) {
      float pow = 1.f, rest;
      if constexpr (std::is_same<T, __half>::value) {
        // an infinite scale must not make a NaN of a weight that is zero
        rest = second ? fminf(__log2f(mul[i]), 128.f) : mul[i];
      } else {
        const uint32_t bits = __float_as_uint(mul[i]);
        pow = __uint_as_float(bits & 0xff800000u);
        rest = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
      }
      if (lane == 0) res[i * res_row] = second || !a.fold_scale ? rest : rest * (a.scale * kLog2e);
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = from_e4m3x2(static_cast<uint16_t>((e < 2 ? w[i].x : w[i].y) >> (16 * (e & 1))));
        f[2 * e] = v.x * pow;
        f[2 * e + 1] = v.y * pow;
      }
      *reinterpret_cast<uint4*>(out + (h0 + i) * a.d) = pack8<T>(f);
    }
}

template <typename T, int GROUP>
cudaError_t launch(const CacheArgs& a, bool write, cudaStream_t st) {
  const int64_t groups = a.T * ((a.Hk + kHeads - 1) / kHeads);
  const int64_t ctas = (groups + kThreads / GROUP - 1) / (kThreads / GROUP);
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(ctas), 2u);
  if (write) {
    if (a.quantized) cache_write_kernel<T, GROUP, true><<<grid, kThreads, 0, st>>>(a);
    else cache_write_kernel<T, GROUP, false><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (a.quantized) cache_read_kernel<T, GROUP, true><<<grid, kThreads, 0, st>>>(a);
    else cache_read_kernel<T, GROUP, false><<<grid, kThreads, 0, st>>>(a);
  }
  return cudaGetLastError();
}

cudaError_t dispatch(const CacheArgs& a, int dtype, bool write, cudaStream_t st) {
  const bool wide = a.d > 128;
  if (dtype == kBF16)
    return wide ? launch<__nv_bfloat16, 32>(a, write, st) : launch<__nv_bfloat16, 16>(a, write, st);
  return wide ? launch<__half, 32>(a, write, st) : launch<__half, 16>(a, write, st);
}


// ---------------------------------------------------------------------------
// rotation by position, on the way into the cache
// ---------------------------------------------------------------------------
// The first 2 P elements of a row of q or k are P pairs, (x_i, x_{P + i}), or interleaved (x_{2i}, x_{2i + 1}); pair i of
// a token at position p turns by the angle whose cosine and sine the table holds in [p, i] and [p, P + i]:
//   (a, b) -> (a cos - b sin, b cos + a sin)
// in fp32, rounded once: to q's type, the cache's type, or e4m3 straight from fp32 (an intermediate 16-bit row would
// round twice).
//
// A lane takes 16 elements of a row as two pieces of 16 bytes that hold whole pairs: pieces l and l + P / 8, or 2 l and
// 2 l + 1; the elements behind the pairs go by in the same steps.  So no pair is split between lanes, and out may be q
// itself.  GROUP lanes hold a row and take HEADS heads of one token, for which the angles are loaded once; a CTA has the
// same heads of 16 (8) tokens, so that whether they turn and where they go is one branch for all.
//
// Its floor is HBM: q read and written, k and v read, the cache written.  What is in flight is bound by registers: 6 CTAs
// of 128 threads an SM with four heads, or for e4m3 8 with two (4 with four heads: 68 and 81 us).  Measured, 16384
// tokens, 32/8 heads of 128: 16-bit cache, 402 MB, 66 us, 6.1 TB/s, 94 % of a copy; e4m3, 370 MB, 70 us, 5.3 TB/s;
// 64 tokens 2.5 us.
constexpr int kTurnThreads = 128;
template <typename T, bool TABLE16>
__device__ __forceinline__ void load_turn(const void* table, int64_t at, float (&x)[8]) {
  if constexpr (TABLE16) {
    unpack8<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(table) + at)), x);
  } else {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(table) + at);
    const float4 lo = __ldg(p), hi = __ldg(p + 1);
    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w;
    x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
  }
}

template <typename T, int GROUP, int HEADS, bool QUANT, bool TABLE16>
__global__ void __launch_bounds__(kTurnThreads, QUANT ? 8 : 6) rotary_write_kernel(const __grid_constant__ RotaryArgs r) {
  const CacheArgs& a = r.cache;
  const int lane = threadIdx.x % GROUP;
  // a CTA takes kTurnThreads / GROUP tokens of one block of heads: 0: q's, 1: k's, 2: v's
  const unsigned q_blocks = (r.H + HEADS - 1) / HEADS, k_blocks = (a.Hk + HEADS - 1) / HEADS;
  const unsigned tile = blockIdx.x / (q_blocks + 2 * k_blocks), block = blockIdx.x - tile * (q_blocks + 2 * k_blocks);
  const unsigned t = tile * (kTurnThreads / GROUP) + threadIdx.x / GROUP;
  const bool any = t < static_cast<unsigned>(a.T);
  const int what = block < q_blocks ? 0 : block < q_blocks + k_blocks ? 1 : 2;
  const int heads = what == 0 ? r.H : a.Hk;
  const int h0 = static_cast<int>(what == 0 ? block : what == 1 ? block - q_blocks : block - q_blocks - k_blocks) * HEADS;
  const int pairs = r.pairs;
  const bool turns = what != 2 && lane * 8 < pairs;  // this lane's elements are pairs
  const int c0 = turns && !r.interleaved ? 8 * lane : 16 * lane;
  const int c1 = turns && !r.interleaved ? 8 * lane + pairs : 16 * lane + 8;
  const bool live = any && 16 * lane < a.d;
  const T* in = static_cast<const T*>(what == 0 ? r.q : what == 1 ? a.k_in : a.v_in);
  const int64_t sT = what == 0 ? r.q_sT : what == 1 ? a.k_sT : a.v_sT, sH = what == 0 ? r.q_sH : what == 1 ? a.k_sH : a.v_sH;
  const int64_t slot_at = any ? __ldg(a.slots + t) : -1;
  const int64_t pos = any ? __ldg(r.positions + t) : -1;
  uint4 x0[HEADS], x1[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    x0[i] = x1[i] = make_uint4(0u, 0u, 0u, 0u);
    if (live && h0 + i < heads) {
      const T* row = in + t * sT + (h0 + i) * sH;
      x0[i] = *reinterpret_cast<const uint4*>(row + c0);
      x1[i] = *reinterpret_cast<const uint4*>(row + c1);
    }
  }
  // a position outside the table: reported; q's row is zero, the token is not written
  const bool placed = pos >= 0 && pos < r.positions_end;
  if (any && !placed && slot_at >= 0 && lane == 0) atomicExch(&g_cache_error, kDevBadIndex);
  float cs[8] = {}, sn[8] = {};
  if (turns && placed) {
    load_turn<T, TABLE16>(r.table, pos * r.table_sP + 8 * lane, cs);
    load_turn<T, TABLE16>(r.table, pos * r.table_sP + pairs + 8 * lane, sn);
  }
  auto rotated = [&](int i, float (&f)[16]) {
    float u[8], w[8];
    unpack8<T>(x0[i], u);
    unpack8<T>(x1[i], w);
    if (turns && r.interleaved) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = __fmaf_rn(u[2 * e], cs[e], -u[2 * e + 1] * sn[e]);
        f[2 * e + 1] = __fmaf_rn(u[2 * e + 1], cs[e], u[2 * e] * sn[e]);
        f[8 + 2 * e] = __fmaf_rn(w[2 * e], cs[4 + e], -w[2 * e + 1] * sn[4 + e]);
        f[9 + 2 * e] = __fmaf_rn(w[2 * e + 1], cs[4 + e], w[2 * e] * sn[4 + e]);
      }
    } else if (turns) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = __fmaf_rn(u[e], cs[e], -w[e] * sn[e]);
        f[8 + e] = __fmaf_rn(w[e], cs[e], u[e] * sn[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = u[e], f[8 + e] = w[e];
    }
  };
  auto halves = [&](const float (&f)[16], uint4& lo, uint4& hi) {
    float u[8], w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = f[e], w[e] = f[8 + e];
    lo = pack8<T>(u);
    hi = pack8<T>(w);
  };
  if (what == 0) {
    T* out = static_cast<T*>(r.q_out);
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      float f[16];
      rotated(i, f);
      uint4 lo, hi;
      halves(f, lo, hi);
      if (!placed) lo = hi = make_uint4(0u, 0u, 0u, 0u);
      if (live && h0 + i < heads) {
        T* row = out + t * r.o_sT + (h0 + i) * r.o_sH;
        *reinterpret_cast<uint4*>(row + c0) = lo;
        *reinterpret_cast<uint4*>(row + c1) = hi;
      }
    }
    return;
  }
  const bool second = what == 2;
  const bool there = in_cache(a, slot_at, any && lane == 0) && placed, keep = there && live;
  const unsigned page = static_cast<unsigned>(slot_at) / a.page, slot = static_cast<unsigned>(slot_at) - page * a.page;
  const int64_t cH = second ? a.vc_sH : a.kc_sH;
  const int64_t base = page * (second ? a.vc_sP : a.kc_sP) + slot * (second ? a.vc_sS : a.kc_sS) + h0 * cH;
  if constexpr (QUANT) {
    uint8_t* cache = static_cast<uint8_t*>(second ? a.v_cache : a.k_cache);
    float* scale = second ? a.v_scale : a.k_scale;
    float mine = 1.f;  // the largest magnitude of row `lane`
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      float f[16];
      rotated(i, f);
      float m = kLeastMax;
#pragma unroll
      for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(f[e]));
#pragma unroll
      for (int o = 1; o < GROUP; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      mine = lane == i ? m : mine;
      // as in cache_write_kernel, with the unit's reciprocal: the correction makes up for its last bit too
      const float2 rr = f2(rcp(fraction(m))), div = f2(-fraction(m));
      const float2 num = f2(__uint_as_float(((262u - (__float_as_uint(m) >> 23)) << 23) | 0x600000u));
      uint32_t code[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 y[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 z = mul2(make_float2(f[4 * e + 2 * x], f[4 * e + 2 * x + 1]), num), q0 = mul2(z, rr);
          y[x] = fma2(fma2(q0, div, z), rr, q0);
        }
        code[e] = to_e4m3x4(y[0].x, y[0].y, y[1].x, y[1].y);
      }
      if (keep && h0 + i < heads) {
        uint8_t* row = cache + base + i * cH;
        *reinterpret_cast<uint2*>(row + c0) = make_uint2(code[0], code[1]);
        *reinterpret_cast<uint2*>(row + c1) = make_uint2(code[2], code[3]);
      }
    }
    mine = __fdiv_rn(mine, kE4m3Max);
    if (there && lane < HEADS && h0 + lane < heads)
      scale[(static_cast<int64_t>(page) * a.Hk + h0 + lane) * a.page + slot] = mine;
  } else {
    T* cache = static_cast<T*>(second ? a.v_cache : a.k_cache);
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      uint4 lo = x0[i], hi = x1[i];
      if (!second) {
        float f[16];
        rotated(i, f);
        halves(f, lo, hi);
      }
      if (keep && h0 + i < heads) {
        T* row = cache + base + i * cH;
        *reinterpret_cast<uint4*>(row + c0) = lo;
        *reinterpret_cast<uint4*>(row + c1) = hi;
      }
    }
  }
}

template <typename T, int GROUP, int HEADS, bool QUANT>
cudaError_t launch_rotary(const RotaryArgs& r, bool table16, cudaStream_t st) {
  const int64_t blocks = (r.H + HEADS - 1) / HEADS + 2 * ((r.cache.Hk + HEADS - 1) / HEADS);
  const int64_t ctas = (r.cache.T + kTurnThreads / GROUP - 1) / (kTurnThreads / GROUP) * blocks;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const unsigned grid = static_cast<unsigned>(ctas);
  if (table16) rotary_write_kernel<T, GROUP, HEADS, QUANT, true><<<grid, kTurnThreads, 0, st>>>(r);
  else rotary_write_kernel<T, GROUP, HEADS, QUANT, false><<<grid, kTurnThreads, 0, st>>>(r);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_rotary(const RotaryArgs& r, bool table16, cudaStream_t st) {
  // 16 elements per lane
  if (r.cache.quantized)
    return r.cache.d > 128 ? launch_rotary<T, 16, 2, true>(r, table16, st) : launch_rotary<T, 8, 2, true>(r, table16, st);
  return r.cache.d > 128 ? launch_rotary<T, 16, 4, false>(r, table16, st) : launch_rotary<T, 8, 4, false>(r, table16, st);
}

}  // namespace

cudaError_t launch_cache_write(const CacheArgs& a, int dtype, cudaStream_t st) { return dispatch(a, dtype, true, st); }
cudaError_t launch_cache_read(const CacheArgs& a, int dtype, cudaStream_t st) { return dispatch(a, dtype, false, st); }

cudaError_t launch_rotary_write(const RotaryArgs& r, int dtype, bool table16, cudaStream_t st) {
  return dtype == kBF16 ? launch_rotary<__nv_bfloat16>(r, table16, st) : launch_rotary<__half>(r, table16, st);
}

void plan_copy_slots(PagedArgs& p) {
  const int64_t table = residue_row(static_cast<int64_t>(p.table_width) * p.page);
  const int64_t stride = residue_row(p.sinks) + residue_row(p.window) + 256, dense = p.B * stride + residue_row(p.T);
  p.copy_dense = dense < p.B * table;
  p.copy_stride = static_cast<int>(p.copy_dense ? stride : table);
  p.copy_slots = p.copy_dense ? dense : p.B * table;
}

cudaError_t launch_cache_expand(const PagedArgs& p, int dtype, void* k, void* v, float* k_res, float* v_res,
                                cudaStream_t st) {
  const int64_t per_seq = p.window > 0 ? p.copy_stride : static_cast<int64_t>(p.table_width) * p.page;
  const int64_t groups = (p.window > 0 ? p.copy_slots : p.B * per_seq) * ((p.Hk + kHeads - 1) / kHeads);
  const int64_t ctas = (groups * 16 + kThreads - 1) / kThreads;
  if (groups >= (1LL << 28)) return cudaErrorInvalidConfiguration;  // the caller's limit keeps it below
  const dim3 grid(static_cast<unsigned>(ctas), 2u);
  if (ctas == 0) return cudaSuccess;
  if (dtype == kBF16)
    cache_expand_kernel<<<grid, kThreads, 0, st>>>(p, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v),
                                                   k_res, v_res, static_cast<unsigned>(per_seq));
  else
    cache_expand_kernel<<<grid, kThreads, 0, st>>>(p, static_cast<__half*>(k), static_cast<__half*>(v), k_res,
                                                   v_res, static_cast<unsigned>(per_seq));
  return cudaGetLastError();
}

int read_device_error_cache(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_cache_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace cta
