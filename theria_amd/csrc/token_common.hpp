// Device building blocks of the token-side kernels: vector loads to float32, sums over lanes, waves and workgroups.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace theria {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_at2_t __attribute__((aligned(2)));
typedef u32x4_t u32x4_at4_t __attribute__((aligned(4)));

// VEC consecutive values as they lie in memory, whole 16-byte pieces of them. Memory only has to be aligned to its elements:
// global memory takes unaligned 16-byte accesses, so that rows of odd widths are read like others (layer norm of (4999,
// 1001) float16, forward 13.7 -> 7.6 us and backward 21.0 -> 13.6 us against single-element accesses). The last vector of a row may hold fewer: `have` of them.
template <typename T, int VEC>
struct RawVec {
  static constexpr int kPieces = VEC * (int)sizeof(T) / 16;
  static_assert(kPieces * 16 == VEC * (int)sizeof(T), "whole 16-byte pieces");
  using piece_t = typename std::conditional<sizeof(T) == 2, u32x4_at2_t, u32x4_at4_t>::type;
  u32x4_t v[kPieces];

  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) v[i] = reinterpret_cast<const piece_t*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<piece_t*>(p)[i] = v[i];
  }
  // The first `have` values (none where it is not positive), zeros behind them. TAIL false: all of them, or none.
  template <bool TAIL = true>
  __device__ __forceinline__ void load(const T* p, int have) {
    if (TAIL ? have >= VEC : have > 0) return load(p);
    zero();
    if (!TAIL || have <= 0) return;
    T t[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[e] = e < have ? p[e] : (T)0.f;
    __builtin_memcpy(v, t, sizeof(v));
  }
  template <bool TAIL = true>
  __device__ __forceinline__ void store(T* p, int have) const {
    if (TAIL ? have >= VEC : have > 0) return store(p);
    if (!TAIL) return;
    T t[VEC];
    __builtin_memcpy(t, v, sizeof(v));
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e < have) p[e] = t[e];
  }
  // The same past the caches: for a large result that is read much later, if at all, whose writes would push out what
  // the kernels around it read (embedding gradient of (16384, 32000, 2048) bfloat16: its rows 52 -> 37 us, the next
  // step's lookup 22 -> 17 us).
  __device__ __forceinline__ void stream(T* p, int have) const {
    if (have < VEC) return store(p, have);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) __builtin_nontemporal_store(v[i], reinterpret_cast<piece_t*>(p) + i);
  }
  // Values n < VEC places down, zeros behind them.
  __device__ __forceinline__ void shift_down(int n) {
    constexpr int N = 4 * kPieces;
    n *= (int)sizeof(T);
#pragma unroll
    for (int by = N / 2; by >= 1; by /= 2) {  // in registers
      if (!(n & 4 * by)) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i / 4][i % 4] = i + by < N ? v[(i + by) / 4 % kPieces][(i + by) % 4] : 0;
    }
    if (sizeof(T) == 2 && (n & 2)) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i / 4][i % 4] = v[i / 4][i % 4] >> 16 | (i + 1 < N ? v[(i + 1) / 4 % kPieces][(i + 1) % 4] << 16 : 0);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) v[i] = u32x4_t{0, 0, 0, 0};
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
    for (int i = 0; i < kPieces; ++i) {
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

// Four consecutive values as float32, zeros behind the first `have`; memory aligned to its elements.
template <typename T>
__device__ __forceinline__ void load_quad(float (&f)[4], const T* p, int have) {
  T t[4] = {(T)0.f, (T)0.f, (T)0.f, (T)0.f};
  if (have >= 4) {
    __builtin_memcpy(t, p, sizeof(t));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < have) t[e] = p[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = (float)t[e];
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// x of the lane 16 (or 32) away added.
__device__ __forceinline__ float swap16_add(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float swap32_add(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Sum over aligned groups of W = 8, 16, 32 or 64 lanes, the same bits in every lane of a group (every step adds the same two
// partial sums in both of its lanes). Lane swaps within the register file: no LDS round trips.
template <int W>
__device__ __forceinline__ float lane_sum(float x) {
  static_assert(W == 8 || W == 16 || W == 32 || W == 64);
  x = dpp_add<0xB1>(x);                             // lane ^ 1
  x = dpp_add<0x4E>(x);                             // lane ^ 2
  x = dpp_add<0x141>(x);                            // the other four of eight
  if constexpr (W >= 16) x = dpp_add<0x140>(x);     // the other eight of sixteen
  if constexpr (W >= 32) x = swap16_add(x);
  if constexpr (W >= 64) x = swap32_add(x);
  return x;
}

// The groups of W lanes of a wave added lane by lane, every group with the sum.
template <int W>
__device__ __forceinline__ float across_groups(float x) {
  if constexpr (W <= 8) x = dpp_add<0x128>(x);  // the lane 8 away, round sixteen
  if constexpr (W <= 16) x = swap16_add(x);
  if constexpr (W <= 32) x = swap32_add(x);
  return x;
}

// K sums over groups of TPR threads: 8 to 64 lanes, or a whole workgroup of TPR threads through `red`, an LDS array
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
      if constexpr (NW == 16) {
        s[k] = lane_sum<16>(red[k * NW + threadIdx.x % 16]);  // one read for each sum, not sixteen: they would fill the registers
      } else {
        float t = red[k * NW];
#pragma unroll
        for (int w = 1; w < NW; ++w) t += red[k * NW + w];
        s[k] = t;
      }
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
