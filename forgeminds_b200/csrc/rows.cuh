// What the row-wise kernels (layernorm.cu, rotary.cu, distill.cu, route.cu) share: 16-byte vectors of bf16 or
// fp32 values, reductions over a warp, a part of a warp or the threads of a row, and a few instructions.
// These files are compiled without --use_fast_math: divisions, square roots and expf are the accurate ones
// unless a kernel says otherwise.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

namespace fmb {

template <typename T> struct Vec16;          // 16 bytes of T
template <> struct Vec16<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive values as fp32 from a 16-byte aligned address
template <typename T, int N> __device__ __forceinline__ void load_f32(const T* p, float (&f)[N]) {
  constexpr int M = Vec16<T>::N;
  if constexpr (N >= M) {
#pragma unroll
    for (int v = 0; v < N / M; ++v) {
      float part[M];
      Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4*>(p) + v), part);
#pragma unroll
      for (int j = 0; j < M; ++j) f[v * M + j] = part[j];
    }
  } else {
    static_assert(sizeof(T) * N == 8, "half a vector");
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
  }
}

// Sum and maximum over `W` neighbouring lanes (W a power of two); every lane gets the result.
template <int W> __device__ __forceinline__ float lanes_sum(float v, unsigned mask = 0xffffffffu) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}
template <int W> __device__ __forceinline__ float lanes_max(float v, unsigned mask = 0xffffffffu) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
  return v;
}

// 2^x, relative error 2^-22: the special function unit without the handling of subnormal results (they become 0)
__device__ __forceinline__ float exp2_unit(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two fp32 values in one register pair, for the instructions that take both at once
using F2 = float2;
__device__ __forceinline__ F2 f2(float lo, float hi) { return make_float2(lo, hi); }
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) { return __fmul2_rn(a, b); }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// SMs of the current device (asked once per device)
inline int sm_count() {
  static int known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (known[dev] == 0) {
    int n = 0;
    known[dev] = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
  }
  return known[dev];
}

}  // namespace fmb
