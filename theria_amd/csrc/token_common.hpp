// Device building blocks of the token-side kernels: vector loads to float32, sums over lanes, waves and workgroups.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace theria {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// VEC consecutive values as they lie in memory: 16-byte pieces, or one element.
template <typename T, int VEC>
struct RawVec {
  static constexpr int kBytes = VEC * (int)sizeof(T);
  static_assert(kBytes % 16 == 0, "whole 16-byte pieces");
  u32x4_t v[kBytes / 16];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) v[i] = reinterpret_cast<const u32x4_t*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<u32x4_t*>(p)[i] = v[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) v[i] = u32x4_t{0, 0, 0, 0};
  }
  __device__ __forceinline__ void get(float (&f)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (sizeof(T) == 4)
        f[i] = __uint_as_float(v[i / 4][i % 4]);
      else if constexpr (__is_same(T, __bf16))
        f[i] = __uint_as_float(i % 2 ? v[i / 8][i % 8 / 2] & 0xffff0000u : v[i / 8][i % 8 / 2] << 16);
      else
        f[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(v[i / 8][i % 8 / 2] >> (i % 2 * 16)));
    }
  }
  __device__ __forceinline__ void set(const float (&f)[VEC]) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          v[i][k] = __float_as_uint(f[4 * i + k]);
        } else {
          const uint32_t lo = __builtin_bit_cast(uint16_t, (T)f[8 * i + 2 * k]);
          const uint32_t hi = __builtin_bit_cast(uint16_t, (T)f[8 * i + 2 * k + 1]);
          v[i][k] = lo | hi << 16;
        }
      }
    }
  }
};

template <typename T>
struct RawVec<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void zero() { v = (T)0.0f; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = (float)v; }
  __device__ __forceinline__ void set(const float (&f)[1]) { v = (T)f[0]; }
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// Sum over aligned groups of W = 16 or 64 lanes, the same bits in every lane of a group (every step adds the same two
// partial sums in both of its lanes). Lane swaps within the register file: no LDS round trips.
template <int W>
__device__ __forceinline__ float lane_sum(float x) {
  static_assert(W == 16 || W == 64);
  x = dpp_add<0xB1>(x);   // lane ^ 1
  x = dpp_add<0x4E>(x);   // lane ^ 2
  x = dpp_add<0x141>(x);  // the other four of eight
  x = dpp_add<0x140>(x);  // the other eight of sixteen
  if constexpr (W == 64) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return x;
}

// Lanes 16 and 32 apart added: the four 16-lane groups of a wave, every group with the sum.
__device__ __forceinline__ float group16_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// K sums over groups of TPR threads: 16 or 64 lanes, or a whole workgroup of TPR threads through `red`, an LDS array
// of K * TPR / 64 floats (one barrier; a later call needs another array or a barrier of its own in between).
template <int TPR, int K>
__device__ __forceinline__ void team_sum(float (&s)[K], float* red) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = lane_sum<W>(s[k]);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[k * NW + wave] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = red[k * NW];
#pragma unroll
      for (int w = 1; w < NW; ++w) t += red[k * NW + w];
      s[k] = t;
    }
  }
}

// Column sums of `parts` rows of `cols` floats: the second step of a sum over many rows, in a fixed order. Columns
// [0, split) go to out0, the rest to out1, either of which may be null; times *factor where it is given.
template <typename T>
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* __restrict__ part, int parts, int64_t cols, int64_t split,
                                                          T* __restrict__ out0, T* __restrict__ out1, const float* factor) {
  __shared__ float red[16][65];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < cols) {
    int r = wave;
    for (; r + 48 < parts; r += 64) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += part[(int64_t)(r + 16 * u) * cols + c];
    }
    for (; r < parts; r += 16) s[0] += part[(int64_t)r * cols + c];
  }
  red[wave][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (wave == 0 && c < cols) {
    float t = red[0][lane];
#pragma unroll
    for (int w = 1; w < 16; ++w) t += red[w][lane];
    if (factor) t *= *factor;
    if (c < split) {
      if (out0) out0[c] = (T)t;
    } else {
      if (out1) out1[c - split] = (T)t;
    }
  }
}

}  // namespace theria
