// Writing new keys and values into a paged cache, and reading slots back.
//
// A 16-bit cache takes the rows as they are.  An e4m3 cache takes, per token
// and head,  s = m / 448,  code = e4m3(x * (448 / m))  with m = max(max|x|,
// 2^-100): one pass over the row, the maximum by shuffles between the 16 (or,
// above 128 elements, 32) lanes that hold it.  The floor of m keeps 448 / m
// finite, so a row of zeros needs no case of its own.  The product is at most
// 448 (1 + 2^-23) and the conversion saturates.  Reading back multiplies code
// by s in 32 bits and rounds once to the tensor's type.
//
// Bound by HBM: 2 d bytes read and d + 4 (2 d) written per row.  Each lane
// moves 16 bytes of the 16-bit row; kRowsPerGroup rows per group of lanes are
// in flight together.
#include "attn_common.cuh"

namespace cta {

__device__ int g_cache_error;

namespace {

constexpr float kE4m3Max = 448.f;
constexpr float kLeastMax = 7.888609052210118e-31f;  // 2^-100
constexpr int kThreads = 256;
constexpr int kRowsPerGroup = 4;

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

// GROUP lanes hold one row of at most 8 GROUP elements.  gridDim.y: 0 keys, 1 values.
template <typename T, int GROUP, bool QUANT>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const __grid_constant__ CacheArgs a) {
  const bool second = blockIdx.y != 0;
  const T* in = static_cast<const T*>(second ? a.v_in : a.k_in);
  const int64_t sT = second ? a.v_sT : a.k_sT, sH = second ? a.v_sH : a.k_sH;
  const int64_t cP = second ? a.vc_sP : a.kc_sP, cS = second ? a.vc_sS : a.kc_sS, cH = second ? a.vc_sH : a.kc_sH;
  void* cache = second ? a.v_cache : a.k_cache;
  float* scale = second ? a.v_scale : a.k_scale;
  const unsigned group = (blockIdx.x * kThreads + threadIdx.x) / GROUP;
  const unsigned groups = gridDim.x * (kThreads / GROUP);
  const int c = (threadIdx.x % GROUP) * 8;
  const unsigned rows = static_cast<unsigned>(a.T) * a.Hk;  // < 2^30, checked by the caller
  uint4 x[kRowsPerGroup];
  int64_t slot[kRowsPerGroup];
#pragma unroll
  for (int i = 0; i < kRowsPerGroup; ++i) {
    const unsigned r = group + i * groups;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    slot[i] = -1;
    if (r < rows) {
      const unsigned t = r / a.Hk;
      slot[i] = __ldg(a.slots + t);
      if (c < a.d) x[i] = __ldg(reinterpret_cast<const uint4*>(in + static_cast<int64_t>(t) * sT + (r - t * a.Hk) * sH + c));
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsPerGroup; ++i) {
    const unsigned r = group + i * groups;
    const int h = r % a.Hk;
    const bool bad = slot[i] >= a.n_slots;
    if (bad && c == 0) atomicExch(&g_cache_error, kDevBadIndex);
    const bool keep = slot[i] >= 0 && !bad;  // a negative slot is padding
    const int64_t p = static_cast<unsigned>(slot[i]) / a.page, s = slot[i] - p * a.page;  // n_slots < 2^31
    if constexpr (QUANT) {
      float f[8];
      unpack8<T>(x[i], f);
      float m = kLeastMax;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(f[e]));
#pragma unroll
      for (int o = 1; o < GROUP; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float up = __fdiv_rn(kE4m3Max, m);
      if (keep && c < a.d) {
        uint2 code;
        code.x = to_e4m3x4(f[0] * up, f[1] * up, f[2] * up, f[3] * up);
        code.y = to_e4m3x4(f[4] * up, f[5] * up, f[6] * up, f[7] * up);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(cache) + p * cP + s * cS + h * cH + c) = code;
        if (c == 0) scale[(p * a.Hk + h) * a.page + s] = __fdiv_rn(m, kE4m3Max);
      }
    } else if (keep && c < a.d) {
      *reinterpret_cast<uint4*>(static_cast<T*>(cache) + p * cP + s * cS + h * cH + c) = x[i];
    }
  }
}

template <typename T, int GROUP, bool QUANT>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ CacheArgs a) {
  const bool second = blockIdx.y != 0;
  T* out = static_cast<T*>(second ? a.v_out : a.k_out);
  const int64_t sT = second ? a.v_sT : a.k_sT, sH = second ? a.v_sH : a.k_sH;
  const int64_t cP = second ? a.vc_sP : a.kc_sP, cS = second ? a.vc_sS : a.kc_sS, cH = second ? a.vc_sH : a.kc_sH;
  const void* cache = second ? a.v_cache : a.k_cache;
  const float* scale = second ? a.v_scale : a.k_scale;
  const unsigned group = (blockIdx.x * kThreads + threadIdx.x) / GROUP;
  const unsigned groups = gridDim.x * (kThreads / GROUP);
  const int c = (threadIdx.x % GROUP) * 8;
  if (c >= a.d) return;
  const unsigned rows = static_cast<unsigned>(a.T) * a.Hk;  // < 2^30, checked by the caller
  uint4 x[kRowsPerGroup];
  float mul[kRowsPerGroup];
#pragma unroll
  for (int i = 0; i < kRowsPerGroup; ++i) {
    const unsigned r = group + i * groups;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    mul[i] = 0.f;
    if (r >= rows) continue;
    const unsigned t = r / a.Hk;
    const int64_t slot = __ldg(a.slots + t);
    const int h = r - t * a.Hk;
    if (slot >= a.n_slots) {
      if (c == 0) atomicExch(&g_cache_error, kDevBadIndex);
    } else if (slot >= 0) {
      const int64_t p = static_cast<unsigned>(slot) / a.page, s = slot - p * a.page;
      const int64_t at = p * cP + s * cS + h * cH + c;
      if constexpr (QUANT) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(cache) + at);
        x[i].x = w.x;
        x[i].y = w.y;
        mul[i] = scale[(p * a.Hk + h) * a.page + s];
      } else {
        x[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(cache) + at);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kRowsPerGroup; ++i) {
    const unsigned r = group + i * groups;
    if (r >= rows) continue;
    const unsigned t = r / a.Hk;
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
    *reinterpret_cast<uint4*>(out + static_cast<int64_t>(t) * sT + (r - t * a.Hk) * sH + c) = y;
  }
}

template <typename T, int GROUP>
cudaError_t launch(const CacheArgs& a, bool write, cudaStream_t st) {
  const int64_t per_cta = static_cast<int64_t>(kThreads / GROUP) * kRowsPerGroup;
  const int64_t ctas = (a.T * a.Hk + per_cta - 1) / per_cta;
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

}  // namespace

cudaError_t launch_cache_write(const CacheArgs& a, int dtype, cudaStream_t st) { return dispatch(a, dtype, true, st); }
cudaError_t launch_cache_read(const CacheArgs& a, int dtype, cudaStream_t st) { return dispatch(a, dtype, false, st); }

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
