// Attention of prompts on the FP32 pipes: every type, every head dim up to 256.
//
//   O_i = sum_j P_ij V_j,  P_ij = exp(c q_i.k_j - lse_i),  lse_i = log sum_j exp(c q_i.k_j)
//   D_i = dO_i.O_i,  dS_ij = P_ij (dO_i.V_j - D_i)
//   dQ_i = c sum_j dS_ij K_j,  dK_j = c sum_i dS_ij Q_i,  dV_j = sum_i P_ij dO_i
//
// 128 threads own a 64-row tile and march over the tiles of the other side; the
// scores of a tile pair live in registers (4 x 8 per thread), the softmax keeps
// a running maximum and sum.  The backward recomputes P from lse in two kernels,
// one that owns query rows (dQ) and one that owns keys (dK, dV): seven products
// instead of five, but no atomics, so the gradients do not depend on the order
// in which CTAs run, and shared key/value heads are summed in registers.
// This is the path of fp32 tensors, whose products need 24-bit operands (on tensor
// cores each would have to be split into several bf16 pieces: not built), of head dims
// above 128, and of the strides and dims that TMA cannot address.  Its ceiling is the
// FP32 pipes; what it reaches is bound by latency at the 7 warps an SM that registers
// and tiles leave (2 x 1024, 8 heads of 64: instructions issue in 40 % of the cycles).
// Measured, fp32, 4 x 512 causal, 8 heads of 64: forward 58 us, both gradients 127
// (dQ alone 83, dK and dV 113); 2 x 1024 not causal: 141 us, 30 TFLOP/s, and 459.
// bf16, 2048 tokens causal, 16 heads of 192: 1.8 and 6.2 ms.
// 256 threads with half the rows each took 1.4 times as long at 2 x 1024: twice the
// shared-memory reads per product.
#include "attn_common.cuh"

namespace cta {

namespace {

constexpr int kThreads = 128;
constexpr int kPad = 4;

// VEC consecutive elements as fp32
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    x[0] = Elem<T>::to_f(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    const float2 a = Elem<T>::unpack(*reinterpret_cast<const typename Elem<T>::Pair*>(&v.x));
    const float2 b = Elem<T>::unpack(*reinterpret_cast<const typename Elem<T>::Pair*>(&v.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  }
}

// rows [first, first + ROWS) of a head into shared memory as fp32; rows outside
// [0, n) and invalid keys (clear bits of `valid`, row first + r is bit r) are
// zero, so that no NaN of theirs meets a zero weight.  BATCH loads in flight.
template <typename T, int ROWS, int DP, int VEC>
__device__ __forceinline__ void load_rows_vec(float* dst, const T* p, int64_t stride, int first, int n, int d,
                                              uint64_t valid) {
  constexpr int kItems = ROWS * DP / VEC / kThreads, kBatch = kItems < 8 ? kItems : 8;
#pragma unroll 1
  for (int i0 = 0; i0 < kItems; i0 += kBatch) {
    float x[kBatch][VEC];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int at = (i0 + i) * kThreads + threadIdx.x;
      const int r = at / (DP / VEC), c = at % (DP / VEC) * VEC, j = first + r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[i][e] = 0.f;
      if (j < n && c < d && ((valid >> r) & 1u)) load_vec<T, VEC>(p + static_cast<int64_t>(j) * stride + c, x[i]);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int at = (i0 + i) * kThreads + threadIdx.x;
      float* o = dst + at / (DP / VEC) * (DP + kPad) + at % (DP / VEC) * VEC;
      if constexpr (VEC == 4) *reinterpret_cast<float4*>(o) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
      else o[0] = x[i][0];
    }
  }
}

template <typename T, int ROWS, int DP>
__device__ __forceinline__ void load_rows(float* dst, const void* base, const AttnStrides& s, const SeqTile& t, int h,
                                          int first, int n, int d, uint64_t valid) {
  const T* p = static_cast<const T*>(base) + t.batch * s.b + t.row0 * s.t + h * s.h;
  if (((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(s.t * sizeof(T))) & (4 * sizeof(T) - 1)) == 0 && d % 4 == 0)
    load_rows_vec<T, ROWS, DP, 4>(dst, p, s.t, first, n, d, valid);
  else
    load_rows_vec<T, ROWS, DP, 1>(dst, p, s.t, first, n, d, valid);
}

// validity of the ROWS (32 or 64) keys from `first` (a multiple of 32)
template <int ROWS>
__device__ __forceinline__ uint64_t valid_keys(const uint32_t* mask, int first, int n) {
  if (mask == nullptr) return ~0ull;
  uint64_t w = first < n ? __ldg(mask + kMaskHead + (first >> 5)) : 0u;
  if (ROWS == 64 && first + 32 < n) w |= static_cast<uint64_t>(__ldg(mask + kMaskHead + (first >> 5) + 1)) << 32;
  return w;
}

// acc[r][c] = A[ty + 16 r] . B[tx + 8 c] over DP; rows of A and B are DP + kPad apart
template <int R, int C, int DP>
__device__ __forceinline__ void mm_nt(float (&acc)[R][C], const float* A, const float* B, int ty, int tx) {
  float2 s[R][C];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) s[r][c] = make_float2(0.f, 0.f);
#pragma unroll 2
  for (int k = 0; k < DP; k += 4) {
    float4 a[R];
#pragma unroll
    for (int r = 0; r < R; ++r) a[r] = *reinterpret_cast<const float4*>(A + (ty + 16 * r) * (DP + kPad) + k);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float4 b = *reinterpret_cast<const float4*>(B + (tx + 8 * c) * (DP + kPad) + k);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[r][c] = fma2(make_float2(a[r].x, a[r].y), make_float2(b.x, b.y), s[r][c]);
        s[r][c] = fma2(make_float2(a[r].z, a[r].w), make_float2(b.z, b.w), s[r][c]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[r][c] = s[r][c].x + s[r][c].y;
}

// acc[r][x] += sum_j P[ty + 16 r][j] V[j][4 tx + 32 x ..]; V rows DP + kPad apart, P rows KT + kPad
template <int R, int DC, int KT, int DP>
__device__ __forceinline__ void mm_nn(float4 (&acc)[R][DC], const float* P, const float* V, int ty, int tx) {
#pragma unroll 1
  for (int j = 0; j < KT; j += 4) {
    float4 p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) p[r] = *reinterpret_cast<const float4*>(P + (ty + 16 * r) * (KT + kPad) + j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int x = 0; x < DC; ++x) {
        const float4 v = *reinterpret_cast<const float4*>(V + (j + i) * (DP + kPad) + 4 * tx + 32 * x);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float w = i == 0 ? p[r].x : i == 1 ? p[r].y : i == 2 ? p[r].z : p[r].w;
          const float2 lo = fma2(f2(w), make_float2(v.x, v.y), make_float2(acc[r][x].x, acc[r][x].y));
          const float2 hi = fma2(f2(w), make_float2(v.z, v.w), make_float2(acc[r][x].z, acc[r][x].w));
          acc[r][x] = make_float4(lo.x, lo.y, hi.x, hi.y);
        }
      }
    }
  }
}

template <typename T, int R, int DC, bool LOW = false>
__device__ __forceinline__ void store_rows(void* base, const AttnStrides& s, const SeqTile& t, int h,
                                           const float4 (&acc)[R][DC], const float (&mul)[R], int d, int ty, int tx) {
  T* p = static_cast<T*>(base) + t.batch * s.b + t.row0 * s.t + h * s.h;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = t.first + ty + 16 * r;
    if (i >= t.n) continue;
#pragma unroll
    for (int x = 0; x < DC; ++x) {
      const float v[4] = {acc[r][x].x, acc[r][x].y, acc[r][x].z, acc[r][x].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 4 * tx + 32 * x + e;
        if (c < d) p[static_cast<int64_t>(i) * s.t + c] = Elem<T>::from_f(LOW ? lost<T>(v[e] * mul[r]) : v[e] * mul[r]);
      }
    }
  }
}

__device__ __forceinline__ float max8(float x) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float sum8(float x) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ SeqTile block_tile(const AttnArgs& a, int tile, int rows, bool backwards) {
  __shared__ SeqTile t;
  if (threadIdx.x < 32) {
    const SeqTile x = find_tile(a.cu, a.nseq, a.L, a.tiles, tile, rows, backwards,
                                a.causal || a.cu != nullptr);
    if (threadIdx.x == 0) t = x;
  }
  __syncthreads();
  return t;
}

// keys per tile: 64, and 32 at head dim 256, where the tiles of four tensors have to fit shared memory
template <int DP> struct SimtTile { static constexpr int KT = DP == 256 ? 32 : 64; };

// WINDOW: rows see the keys of Reach; tiles between the first keys and the tile's window are passed over
template <typename T, int DP, bool WINDOW>
__global__ void __launch_bounds__(kThreads) attn_simt_fwd_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int KT = SimtTile<DP>::KT, C = KT / 8, DC = DP / 32, R = kSimtRows / 16;
  extern __shared__ float4 smem_raw[];
  float* Q = reinterpret_cast<float*>(smem_raw);
  float* K = Q + kSimtRows * (DP + kPad);
  float* V = K + KT * (DP + kPad);
  float* P = V + KT * (DP + kPad);
  const int h = blockIdx.x % a.H, hk = h / (a.H / a.Hk);
  const SeqTile t = block_tile(a, blockIdx.x / a.H, kSimtRows, a.causal);
  if (t.first >= t.n) {
    if (a.cu != nullptr && a.zero_tail) zero_rows<T>(a.o, a.os, t.row0, a.L, h, a.d, t.tail_index, t.tail_count);
    return;
  }
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  const uint32_t* mask = a.mask != nullptr ? a.mask + t.batch * a.mask_words : nullptr;
  int lo, hi;
  mask_range(a, t.batch, t.n, lo, hi);
  if (a.causal) hi = min(hi, t.first + kSimtRows);
  load_rows<T, kSimtRows, DP>(Q, a.q, a.qs, t, h, t.first, t.n, a.d, ~0ull);
  float m[R], l[R];
  float4 acc[R][DC];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = neg_inf();
    l[r] = 0.f;
#pragma unroll
    for (int x = 0; x < DC; ++x) acc[r][x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float c2 = a.scale * kLog2e;
  const Reach reach = reach_of(a, lo);
  for (int j0 = lo / KT * KT; j0 < hi; j0 += KT) {
    if (WINDOW && j0 >= reach.sink_end && j0 + KT <= reach.first(t.first)) {
      j0 = reach.first(t.first) / KT * KT;
      if (j0 >= hi) break;
    }
    __syncthreads();
    const uint64_t valid = valid_keys<KT>(mask, j0, t.n);
    load_rows<T, KT, DP>(K, a.k, a.ks, t, hk, j0, t.n, a.d, valid);
    load_rows<T, KT, DP>(V, a.v, a.vs, t, hk, j0, t.n, a.d, valid);
    __syncthreads();
    float s[R][C];
    mm_nt<R, C, DP>(s, Q, K, ty, tx);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = t.first + ty + 16 * r;
      float top = m[r];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int j = j0 + tx + 8 * c;
        const bool see = j < t.n && (!a.causal || j <= i) && (!WINDOW || reach.sees(i, j)) && ((valid >> (tx + 8 * c)) & 1u);
        s[r][c] = see ? s[r][c] * c2 : neg_inf();
        top = fmaxf(top, s[r][c]);
      }
      top = max8(top);
      const float base = top == neg_inf() ? 0.f : top;  // no key yet: every weight is exp(-inf) = 0
      const float shrink = ex2(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float p = ex2(s[r][c] - base);
        sum += p;
        P[(ty + 16 * r) * (KT + kPad) + tx + 8 * c] = p;
      }
      l[r] = l[r] * shrink + sum8(sum);
      m[r] = top;
#pragma unroll
      for (int x = 0; x < DC; ++x) {
        acc[r][x].x *= shrink;
        acc[r][x].y *= shrink;
        acc[r][x].z *= shrink;
        acc[r][x].w *= shrink;
      }
    }
    __syncwarp();  // a row of P is written and read by the same eight lanes
    mm_nn<R, DC, KT, DP>(acc, P, V, ty, tx);
  }
  float inv[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    inv[r] = l[r] == 0.f ? 0.f : 1.f / l[r];
    const int i = t.first + ty + 16 * r;
    if (tx == 0 && i < t.n && a.lse != nullptr)
      a.lse[lse_index(a, t, h, i)] = l[r] == 0.f ? neg_inf() : (m[r] + log2f(l[r])) * kLn2;
  }
  store_rows<T, R, DC>(a.o, a.os, t, h, acc, inv, a.d, ty, tx);
  if (!std::is_same<T, float>::value && a.low != nullptr)
    store_rows<T, R, DC, true>(a.low, AttnStrides{a.L * a.H * a.d, static_cast<int64_t>(a.H) * a.d, a.d}, t, h, acc, inv,
                               a.d, ty, tx);
}

// weights and d(scores) of a tile pair from the scores s and the products dp = dO.V
__device__ __forceinline__ void weight_grad(float s, float dp, float lse2, float delta, float c2, bool see, float& p,
                                            float& ds) {
  p = see ? ex2(s * c2 - lse2) : 0.f;
  ds = see ? p * (dp - delta) : 0.f;
}

template <typename T, int DP, bool WINDOW>
__global__ void __launch_bounds__(kThreads) attn_simt_dq_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int KT = SimtTile<DP>::KT, C = KT / 8, DC = DP / 32, R = kSimtRows / 16;
  extern __shared__ float4 smem_raw[];
  float* Q = reinterpret_cast<float*>(smem_raw);
  float* G = Q + kSimtRows * (DP + kPad);
  float* K = G + kSimtRows * (DP + kPad);
  float* V = K + KT * (DP + kPad);
  float* P = V + KT * (DP + kPad);
  const int h = blockIdx.x % a.H, hk = h / (a.H / a.Hk);
  const SeqTile t = block_tile(a, blockIdx.x / a.H, kSimtRows, a.causal);
  if (t.first >= t.n) {
    if (a.cu != nullptr) zero_rows<T>(a.dq, a.dqs, t.row0, a.L, h, a.d, t.tail_index, t.tail_count);
    pdl_wait();
    return;
  }
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  const uint32_t* mask = a.mask != nullptr ? a.mask + t.batch * a.mask_words : nullptr;
  int lo, hi;
  mask_range(a, t.batch, t.n, lo, hi);
  if (a.causal) hi = min(hi, t.first + kSimtRows);
  load_rows<T, kSimtRows, DP>(Q, a.q, a.qs, t, h, t.first, t.n, a.d, ~0ull);
  load_rows<T, kSimtRows, DP>(G, a.g, a.gs, t, h, t.first, t.n, a.d, ~0ull);
  float lse2[R], delta[R];
  float4 acc[R][DC];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = t.first + ty + 16 * r;
    lse2[r] = i < t.n ? a.lse[lse_index(a, t, h, i)] * kLog2e : neg_inf();
    delta[r] = i < t.n ? a.delta[lse_index(a, t, h, i)] : 0.f;
#pragma unroll
    for (int x = 0; x < DC; ++x) acc[r][x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float c2 = a.scale * kLog2e;
  const Reach reach = reach_of(a, lo);
  for (int j0 = lo / KT * KT; j0 < hi; j0 += KT) {
    if (WINDOW && j0 >= reach.sink_end && j0 + KT <= reach.first(t.first)) {
      j0 = reach.first(t.first) / KT * KT;
      if (j0 >= hi) break;
    }
    __syncthreads();
    const uint64_t valid = valid_keys<KT>(mask, j0, t.n);
    load_rows<T, KT, DP>(K, a.k, a.ks, t, hk, j0, t.n, a.d, valid);
    load_rows<T, KT, DP>(V, a.v, a.vs, t, hk, j0, t.n, a.d, valid);
    __syncthreads();
    float s[R][C], dp[R][C];
    mm_nt<R, C, DP>(s, Q, K, ty, tx);
    mm_nt<R, C, DP>(dp, G, V, ty, tx);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int i = t.first + ty + 16 * r, j = j0 + tx + 8 * c;
        const bool see = i < t.n && j < t.n && (!a.causal || j <= i) && (!WINDOW || reach.sees(i, j)) &&
                         ((valid >> (tx + 8 * c)) & 1u) && lse2[r] != neg_inf();
        float p, ds;
        weight_grad(s[r][c], dp[r][c], lse2[r], delta[r], c2, see, p, ds);
        P[(ty + 16 * r) * (KT + kPad) + tx + 8 * c] = ds;
      }
    __syncwarp();
    mm_nn<R, DC, KT, DP>(acc, P, K, ty, tx);
  }
  float mul[R];
#pragma unroll
  for (int r = 0; r < R; ++r) mul[r] = a.scale;
  store_rows<T, R, DC>(a.dq, a.dqs, t, h, acc, mul, a.d, ty, tx);
  pdl_wait();  // launched beside dK and dV
}

// A window's first keys are seen by all rows.  Those behind the window of such a key tile, the far ones, are another launch,
// a CTA per `chunk` rows, which leaves its sums over the first keys in 32 bits; the tile's own CTA adds them in order.  One
// sequence, 8 heads of 64, window 4 and 4 first keys: 16384 tokens 467 us in fp32, against 3200 (bf16) with the tile's CTA
// going through all rows; 1024 tokens 71 and 200.
struct FarRows {
  float* sums;  // nullptr: there are none
  int chunk, tiles, keys;  // rows of a CTA; tiles with first keys; first keys of a tile at most
};
enum DkvForm : int { kAll = 0, kNear = 1, kFar = 2 };

// owns KT keys of one key/value head; rows of the score tile are keys, columns are queries.  kNear, kFar: with a window.
template <typename T, int DP, int FORM>
__global__ void __launch_bounds__(kThreads) attn_simt_dkv_kernel(const __grid_constant__ AttnArgs a,
                                                                 const __grid_constant__ FarRows far) {
  constexpr bool WINDOW = FORM != kAll;
  constexpr int KT = SimtTile<DP>::KT, QT = KT, C = QT / 8, DC = DP / 32, R = KT / 16;
  extern __shared__ float4 smem_raw[];
  float* K = reinterpret_cast<float*>(smem_raw);
  float* V = K + KT * (DP + kPad);
  float* Q = V + KT * (DP + kPad);
  float* G = Q + QT * (DP + kPad);
  float* P = G + QT * (DP + kPad);
  __shared__ float s_lse[QT], s_delta[QT];
  const int hk = blockIdx.x % a.Hk, group = a.H / a.Hk;
  pdl_launch_dependents();  // dQ's CTAs may follow; kFar: the others'
  // early keys of a causal sequence meet the most queries: forwards is heaviest first
  SeqTile t = FORM == kFar ? block_tile(a, blockIdx.x / a.Hk / far.tiles, far.chunk, false)
                           : block_tile(a, blockIdx.x / a.Hk, KT, false);
  if (t.first >= t.n) {
    if (FORM == kNear) pdl_wait();
    if (FORM != kFar && a.cu != nullptr) {
      zero_rows<T>(a.dk, a.dks, t.row0, a.L, hk, a.d, t.tail_index, t.tail_count);
      zero_rows<T>(a.dv, a.dvs, t.row0, a.L, hk, a.d, t.tail_index, t.tail_count);
    }
    return;
  }
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  const uint32_t* mask = a.mask != nullptr ? a.mask + t.batch * a.mask_words : nullptr;
  int lo, hi;
  mask_range(a, t.batch, t.n, lo, hi);
  const Reach reach = reach_of(a, lo);
  int row_from = a.causal ? t.first : 0, row_to = t.n;
  if constexpr (WINDOW) {
    const int chunk_from = t.first;
    if constexpr (FORM == kFar) t.first = (lo / KT + static_cast<int>(blockIdx.x) / a.Hk % far.tiles) * KT;
    // rows behind the windows that hold the last of these keys see none of them, unless it is one of the first
    const int far_from = (min(t.n, t.first + KT - 1 + reach.window) + QT - 1) / QT * QT;
    if constexpr (FORM == kFar) {
      row_from = max(chunk_from, far_from);
      row_to = min(chunk_from + far.chunk, t.n);
      if (row_from >= row_to || t.first >= min(min(t.n, hi), reach.sink_end)) return;
    } else if (t.first >= reach.sink_end || far.sums != nullptr) {
      row_to = min(t.n, far_from);
    }
  }
  // the far rows' sums of chunk c over the first keys of this tile: dV, then dK, [far.keys][2][DP]
  auto far_at = [&](int c) {
    const int64_t slot = far_place(a, t, KT, far.chunk) + c;
    return far.sums + (((slot * far.tiles + (t.first / KT - lo / KT)) * a.Hk + hk) * far.keys - max(t.first, lo)) * 2 * DP;
  };
  const uint64_t valid = valid_keys<KT>(mask, t.first, t.n);
  load_rows<T, KT, DP>(K, a.k, a.ks, t, hk, t.first, t.n, a.d, valid);
  load_rows<T, KT, DP>(V, a.v, a.vs, t, hk, t.first, t.n, a.d, valid);
  bool key[R];
  float4 dk[R][DC], dv[R][DC];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = t.first + ty + 16 * r;
    key[r] = j < t.n && ((valid >> (ty + 16 * r)) & 1u);
#pragma unroll
    for (int x = 0; x < DC; ++x) dk[r][x] = dv[r][x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float c2 = a.scale * kLog2e;
  // rows that see no key, up to the first valid one, may hold anything
  const int from = lo >= hi ? t.n : a.causal ? lo : 0;
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    for (int i0 = row_from; i0 < row_to; i0 += QT) {
      if (from >= i0 + QT) continue;
      uint64_t seeing = from > i0 ? ~0ull << (from - i0) : ~0ull;
      if constexpr (WINDOW) {
        // a window may lie on masked keys alone: such a row sees nothing and may hold anything, as the padding may
#pragma unroll
        for (int x = 0; x < QT; x += 32) {
          const int i = i0 + x + static_cast<int>(threadIdx.x & 31);
          const unsigned some = __ballot_sync(0xffffffffu, i < t.n && a.lse[lse_index(a, t, h, i)] != neg_inf());
          seeing &= ~(static_cast<uint64_t>(~some) << x);
        }
      }
      __syncthreads();
      load_rows<T, QT, DP>(Q, a.q, a.qs, t, h, i0, t.n, a.d, seeing);
      load_rows<T, QT, DP>(G, a.g, a.gs, t, h, i0, t.n, a.d, seeing);
      if (threadIdx.x < QT) {
        const int i = i0 + threadIdx.x;
        s_lse[threadIdx.x] = i < t.n ? a.lse[lse_index(a, t, h, i)] * kLog2e : neg_inf();
        s_delta[threadIdx.x] = i < t.n ? a.delta[lse_index(a, t, h, i)] : 0.f;
      }
      __syncthreads();
      float s[R][C], dp[R][C];
      mm_nt<R, C, DP>(s, K, Q, ty, tx);
      mm_nt<R, C, DP>(dp, V, G, ty, tx);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int q = tx + 8 * c, i = i0 + q, j = t.first + ty + 16 * r;
          const bool see = key[r] && i < t.n && (!a.causal || j <= i) && (!WINDOW || reach.sees(i, j)) && s_lse[q] != neg_inf();
          float p;
          weight_grad(s[r][c], dp[r][c], s_lse[q], s_delta[q], c2, see, p, dp[r][c]);
          P[(ty + 16 * r) * (QT + kPad) + q] = p;
        }
      __syncwarp();
      mm_nn<R, DC, QT, DP>(dv, P, G, ty, tx);
      __syncwarp();
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) P[(ty + 16 * r) * (QT + kPad) + tx + 8 * c] = dp[r][c];
      __syncwarp();
      mm_nn<R, DC, QT, DP>(dk, P, Q, ty, tx);
    }
  }
  if constexpr (WINDOW) {
    if constexpr (FORM == kNear) pdl_wait();  // launched beside the far rows
    if (FORM == kFar || (far.sums != nullptr && row_to < t.n && t.first < min(hi, reach.sink_end))) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = t.first + ty + 16 * r;
        if (j < lo || j >= reach.sink_end) continue;
        const int c1 = FORM == kFar ? row_from / far.chunk + 1 : (t.n + far.chunk - 1) / far.chunk;
        for (int c = (FORM == kFar ? row_from : row_to) / far.chunk; c < c1; ++c) {
          float* sums = far_at(c) + static_cast<int64_t>(j) * 2 * DP + 4 * tx;
#pragma unroll
          for (int x = 0; x < DC; ++x) {
            float4* of_v = reinterpret_cast<float4*>(sums + 32 * x);
            float4* of_k = reinterpret_cast<float4*>(sums + DP + 32 * x);
            if constexpr (FORM == kFar) {
              *of_v = dv[r][x];
              *of_k = dk[r][x];
            } else {
              const float4 y = __ldcg(of_v), z = __ldcg(of_k);  // written while this kernel may already be there
              dv[r][x].x += y.x, dv[r][x].y += y.y, dv[r][x].z += y.z, dv[r][x].w += y.w;
              dk[r][x].x += z.x, dk[r][x].y += z.y, dk[r][x].z += z.z, dk[r][x].w += z.w;
            }
          }
        }
      }
    }
    if constexpr (FORM == kFar) return;
  }
  float mul[R], one[R];
#pragma unroll
  for (int r = 0; r < R; ++r) mul[r] = a.scale, one[r] = 1.f;
  store_rows<T, R, DC>(a.dk, a.dks, t, hk, dk, mul, a.d, ty, tx);
  store_rows<T, R, DC>(a.dv, a.dvs, t, hk, dv, one, a.d, ty, tx);
}

// delta_i = sum_d g_i o_i, o_i with what its rounding lost where that was kept.  GROUP lanes per (row, head), 16 bytes
// of each tensor per lane and step (VEC elements; one element where rows do not start on 16 bytes): bound by HBM, two
// or three tensors read once; 8 x 1024 tokens, 32 heads of 128 in bf16, two tensors: 40 us, 3.4 TB/s.
// For fp16 gradients on tensor cores it also leaves |g_i| and, of the first groups one key each, |v_j|: 55 us there
// with 8 key/value heads, 45 without the norms (groups of their own for the keys: 57); 16 x 512 tokens, 8 heads of 64: 11 and 7.
template <typename T, int GROUP, int VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 6 : 5) attn_delta_kernel(const __grid_constant__ AttnArgs a, int64_t rows, int64_t keys) {
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / GROUP;
  const int lane = threadIdx.x % GROUP;
  const bool norms = std::is_same<T, __half>::value && a.g_norm != nullptr;
  float s = 0.f, g2 = 0.f, v2 = 0.f;
  int64_t at = 0, key_at = 0, key_b = 0, key_i = 0;
  // token and head of the x-th row of a tensor with `heads`, and its place in [batch, heads, token]
  auto place = [&](int64_t x, int heads, int64_t& b, int64_t& i, int& h) {
    const int64_t r = x / heads;
    h = static_cast<int>(x - r * heads);
    b = a.cu != nullptr ? 0 : r / a.L;
    i = r - b * a.L;
    return (b * heads + h) * a.L + i;
  };
  if (w < rows) {
    int64_t b, i;
    int h, hk = 0;
    at = place(w, a.H, b, i, h);
    const T* o = static_cast<const T*>(a.o) + b * a.os.b + i * a.os.t + h * a.os.h;
    const T* g = static_cast<const T*>(a.g) + b * a.gs.b + i * a.gs.t + h * a.gs.h;
    const T* low = a.low != nullptr ? static_cast<const T*>(a.low) + w * a.d : nullptr;
    const T* v = nullptr;
    if (norms && w < keys) {
      key_at = place(w, a.Hk, key_b, key_i, hk);
      v = static_cast<const T*>(a.v) + key_b * a.vs.b + key_i * a.vs.t + hk * a.vs.h;
    }
    for (int c = lane * VEC; c < a.d; c += GROUP * VEC) {
      if constexpr (VEC == 1) {
        float x = Elem<T>::to_f(o[c]);
        if (low != nullptr) x = fmaf(Elem<T>::to_f(low[c]), 1.f / low_scale<T>(), x);
        const float y = Elem<T>::to_f(g[c]), z = v != nullptr ? Elem<T>::to_f(v[c]) : 0.f;
        s = fmaf(x, y, s);
        g2 = fmaf(y, y, g2);
        v2 = fmaf(z, z, v2);
      } else {
        float x[4], y[4], z[4];
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          load_vec<T, 4>(o + c + e, x);
          load_vec<T, 4>(g + c + e, y);
          if (low != nullptr) {
            load_vec<T, 4>(low + c + e, z);
#pragma unroll
            for (int w4 = 0; w4 < 4; ++w4) x[w4] = fmaf(z[w4], 1.f / low_scale<T>(), x[w4]);
          }
#pragma unroll
          for (int w4 = 0; w4 < 4; ++w4) s = fmaf(x[w4], y[w4], s);
          if (norms) {
#pragma unroll
            for (int w4 = 0; w4 < 4; ++w4) g2 = fmaf(y[w4], y[w4], g2);
          }
          if (v != nullptr) {
            load_vec<T, 4>(v + c + e, z);
#pragma unroll
            for (int w4 = 0; w4 < 4; ++w4) v2 = fmaf(z[w4], z[w4], v2);
          }
        }
      }
    }
  }
#pragma unroll
  for (int x = GROUP / 2; x > 0; x >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, x);
    if (norms) {
      g2 += __shfl_xor_sync(0xffffffffu, g2, x);
      v2 += __shfl_xor_sync(0xffffffffu, v2, x);
    }
  }
  if (lane != 0 || w >= rows) return;
  a.delta[at] = s;
  if (!norms) return;
  // what may hold anything does not count: masked keys, infinities and NaN
  const float inf = __int_as_float(0x7f800000);
  a.g_norm[at] = g2 < inf ? sqrtf(g2) : 0.f;
  if (w >= keys) return;
  const uint32_t* mask = a.mask != nullptr ? a.mask + key_b * a.mask_words : nullptr;
  a.v_norm[key_at] = mask_key(mask, static_cast<int>(key_i)) && v2 < inf ? sqrtf(v2) : 0.f;
}

// key mask words: one CTA per batch entry
__global__ void attn_mask_words_kernel(const void* mask, int dtype, int64_t sB, int64_t sL, int64_t L, uint32_t* out,
                                       int64_t words) {
  uint32_t* w = out + blockIdx.x * words;
  __shared__ int s_lo, s_hi;
  if (threadIdx.x == 0) {
    s_lo = static_cast<int>(L);
    s_hi = 0;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  int lo = static_cast<int>(L), hi = 0;
  for (int64_t i = threadIdx.x >> 5; i < words - kMaskHead; i += blockDim.x >> 5) {
    const int64_t j = i * 32 + lane;
    const bool ok = j < L && mask_valid(mask, dtype, blockIdx.x * sB + j * sL);
    const uint32_t bits = __ballot_sync(0xffffffffu, ok);
    if (lane == 0) w[kMaskHead + i] = bits;
    if (bits != 0u) {
      lo = min(lo, static_cast<int>(i * 32) + __ffs(bits) - 1);
      hi = static_cast<int>(i * 32) + 32 - __clz(bits);
    }
  }
  if (lane == 0) {
    atomicMin(&s_lo, lo);
    atomicMax(&s_hi, hi);
  }
  __syncthreads();
  if (threadIdx.x < kMaskHead) w[threadIdx.x] = threadIdx.x == 0 ? s_lo : threadIdx.x == 1 ? s_hi : 0u;
}

int64_t count_tiles(AttnArgs& a, int rows) {
  if (a.cu != nullptr) {
    a.tiles = static_cast<int>(packed_tiles(a.L, a.nseq, rows));
    return a.tiles;
  }
  a.tiles = static_cast<int>((a.L + rows - 1) / rows);
  return static_cast<int64_t>(a.tiles) * a.nseq;
}

// shared memory is the same for every launch of a kernel
template <typename T, int DP, bool WINDOW>
cudaError_t fwd(AttnArgs a, cudaStream_t st) {
  constexpr int KT = SimtTile<DP>::KT;
  constexpr int smem = sizeof(float) * ((kSimtRows + 2 * KT) * (DP + kPad) + kSimtRows * (KT + kPad));
  const int64_t tiles = count_tiles(a, kSimtRows);
  return launch_grid<attn_simt_fwd_kernel<T, DP, WINDOW>>(false, tiles * a.H, kThreads, smem, st, a);
}

int key_tile(int d) { return d > 128 ? SimtTile<256>::KT : SimtTile<64>::KT; }
int far_tiles(const AttnArgs& a) {
  const int kt = key_tile(a.d);
  return a.mask != nullptr ? (a.sinks + kt - 2) / kt + 1 : (a.sinks + kt - 1) / kt;
}
int64_t far_bytes_of(const AttnArgs& a, int64_t chunk) {
  const int kt = key_tile(a.d);
  return far_places(a, kt, chunk) * far_tiles(a) * a.Hk * std::min(a.sinks, kt) * 2 * (a.d <= 64 ? 64 : a.d <= 128 ? 128 : 256) *
         static_cast<int64_t>(sizeof(float));
}
// Rows of a far CTA: about as many as the others' windows; more where there would be more than 64 parts in a row, or
// more than 256 MB of them.
int far_chunk(const AttnArgs& a) {
  int64_t rows = std::max<int64_t>(std::max<int64_t>(a.window + key_tile(a.d), 128), (a.L + 63) / 64);
  rows = (rows + 63) / 64 * 64;
  while (rows < a.L && far_bytes_of(a, rows) > (256LL << 20)) rows *= 2;
  return static_cast<int>(rows);
}

template <typename T, int DP, bool WINDOW>
cudaError_t bwd(AttnArgs a, void* far_sums, cudaStream_t st) {
  constexpr int KT = SimtTile<DP>::KT;
  if (a.dk != nullptr) {
    constexpr int smem = sizeof(float) * (4 * KT * (DP + kPad) + KT * (KT + kPad));
    FarRows far = {};
    if (WINDOW && simt_far_bytes(a) > 0) {
      far = FarRows{static_cast<float*>(far_sums), far_chunk(a), far_tiles(a), std::min(a.sinks, KT)};
      const int64_t chunks = count_tiles(a, far.chunk);
      const cudaError_t e = launch_grid<attn_simt_dkv_kernel<T, DP, WINDOW ? kFar : kAll>>(
          false, chunks * far.tiles * a.Hk, kThreads, smem, st, a, far);
      if (e != cudaSuccess) return e;
    }
    const int64_t tiles = count_tiles(a, KT);
    const cudaError_t e = launch_grid<attn_simt_dkv_kernel<T, DP, WINDOW ? kNear : kAll>>(far.sums != nullptr, tiles * a.Hk,
                                                                                          kThreads, smem, st, a, far);
    if (e != cudaSuccess) return e;
  }
  if (a.dq == nullptr) return cudaSuccess;
  constexpr int smem = sizeof(float) * ((2 * kSimtRows + 2 * KT) * (DP + kPad) + kSimtRows * (KT + kPad));
  const int64_t tiles = count_tiles(a, kSimtRows);
  return launch_grid<attn_simt_dq_kernel<T, DP, WINDOW>>(a.dk != nullptr, tiles * a.H, kThreads, smem, st, a);
}

template <typename T, bool WINDOW>
cudaError_t dispatch_dim(const AttnArgs& a, bool backward, void* far, cudaStream_t st) {
  if (a.d <= 64) return backward ? bwd<T, 64, WINDOW>(a, far, st) : fwd<T, 64, WINDOW>(a, st);
  if (a.d <= 128) return backward ? bwd<T, 128, WINDOW>(a, far, st) : fwd<T, 128, WINDOW>(a, st);
  return backward ? bwd<T, 256, WINDOW>(a, far, st) : fwd<T, 256, WINDOW>(a, st);
}
template <typename T>
cudaError_t dispatch(const AttnArgs& a, bool backward, void* far, cudaStream_t st) {
  return a.window > 0 ? dispatch_dim<T, true>(a, backward, far, st) : dispatch_dim<T, false>(a, backward, far, st);
}

}  // namespace

int64_t simt_far_bytes(const AttnArgs& a) {
  // A launch pays for a few row tiles.  fp32 backward, 8 heads of 64, 4 first keys, with and without: 4 x 512 tokens, window
  // 128, 111 and 116 us; 4 x 1024, 212 and 273; 512, window 16, 46 and 100.
  if (a.window == 0 || a.sinks == 0 || a.L < a.window + 4 * key_tile(a.d)) return 0;
  return far_bytes_of(a, far_chunk(a));
}

cudaError_t launch_attn_simt_fwd(const AttnArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case kF32: return dispatch<float>(a, false, nullptr, st);
    case kBF16: return dispatch<__nv_bfloat16>(a, false, nullptr, st);
    default: return dispatch<__half>(a, false, nullptr, st);
  }
}

cudaError_t launch_attn_simt_bwd(const AttnArgs& a, int dtype, void* far, cudaStream_t st) {
  switch (dtype) {
    case kF32: return dispatch<float>(a, true, far, st);
    case kBF16: return dispatch<__nv_bfloat16>(a, true, far, st);
    default: return dispatch<__half>(a, true, far, st);
  }
}

namespace {
template <typename T>
bool rows_on16(const void* p, const AttnStrides& s) {
  return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>((s.b | s.t | s.h) * sizeof(T))) % 16 == 0;
}

template <typename T>
cudaError_t delta(const AttnArgs& a, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  const int64_t tokens = a.cu != nullptr ? a.L : a.L * a.nseq;
  const int64_t rows = tokens * a.H, keys = a.v_norm != nullptr ? tokens * a.Hk : 0;
  const bool vec = a.d % kVec == 0 && rows_on16<T>(a.o, a.os) && rows_on16<T>(a.g, a.gs) &&
                   reinterpret_cast<uintptr_t>(a.low) % 16 == 0 && (keys == 0 || rows_on16<T>(a.v, a.vs));
  const int group = vec && a.d <= 8 * kVec ? 8 : vec && a.d <= 16 * kVec ? 16 : 32;
  const int64_t ctas = (rows * group + 255) / 256;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const unsigned grid = static_cast<unsigned>(ctas);
  if (!vec) attn_delta_kernel<T, 32, 1><<<grid, 256, 0, st>>>(a, rows, keys);
  else if (group == 8) attn_delta_kernel<T, 8, kVec><<<grid, 256, 0, st>>>(a, rows, keys);
  else if (group == 16) attn_delta_kernel<T, 16, kVec><<<grid, 256, 0, st>>>(a, rows, keys);
  else attn_delta_kernel<T, 32, kVec><<<grid, 256, 0, st>>>(a, rows, keys);
  return cudaGetLastError();
}
}  // namespace

cudaError_t launch_attn_delta(const AttnArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case kF32: return delta<float>(a, st);
    case kBF16: return delta<__nv_bfloat16>(a, st);
    default: return delta<__half>(a, st);
  }
}

cudaError_t launch_attn_mask_words(const void* mask, int mask_dtype, int64_t sB, int64_t sL, int64_t B, int64_t L,
                                   uint32_t* words, int64_t words_per_batch, cudaStream_t st) {
  attn_mask_words_kernel<<<static_cast<unsigned>(B), 512, 0, st>>>(mask, mask_dtype, sB, sL, L, words,
                                                                   words_per_batch);
  return cudaGetLastError();
}

}  // namespace cta
