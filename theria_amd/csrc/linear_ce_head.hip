// Cross entropy of a linear head with few classes, a classifier's: at most 16 classes of at most 512 elements (gfx950).
//
// The products of linear_ce.hip would be nearly all padding here, and their launches the cost. Instead a wave takes a row at a
// time, with the whole weight in its registers: the row's logits are sums over its lanes, taken together so that each lane
// ends with one of them. Forward and backward are a launch each, and a second one that adds the workgroups' sums (in a fixed order) where
// more than one workgroup has rows. All arithmetic is float32 on the inputs' values.
//
// Bound by the host for a classifier's batch, by instructions for many rows: (10^5, 64) of 16 classes float32 forward 72 us
// with a sum after the other, 49 us with class_sums.
#include "token_common.hpp"
#include "token_params.hpp"

namespace theria {
namespace {

constexpr int kWaves = 8;         // of a workgroup
constexpr int64_t kAloneRows = 64;  // most rows that one workgroup takes

// What a wave needs of a row: 64 E elements, lane l holding l, l + 64, ...
template <typename T, int E>
__device__ __forceinline__ void load_row(float (&x)[E], const void* base, int64_t sr, int64_t row, int width, int lane) {
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = e * 64 + lane < width ? (float)((const T*)base)[row * sr + e * 64 + lane] : 0.f;
}

__device__ __forceinline__ int64_t load_target(const CeParams& p, int64_t row) {
  return p.target64 ? ((const int64_t*)p.target)[row] : (int64_t)((const int32_t*)p.target)[row];
}

// The class whose logit a lane ends with: lane bits 0, 1, 3 and, with sixteen classes, 4. The others hold copies.
template <int V>
__device__ __forceinline__ int class_of(int lane) {
  return (lane & 3) | (lane >> 1 & (V == 16 ? 12 : 4));
}
__device__ __forceinline__ int lane_of(int v) { return (v & 3) | (v & 12) << 1; }

template <int CTRL>
__device__ __forceinline__ float dpp_take(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// One step of a sum of N values over lanes, which halves the values that a lane goes on with: it keeps those of its own side
// and gets the other lane's share of them.
template <int CTRL, int N>
__device__ __forceinline__ void halve(float (&s)[N], bool odd) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    const float a = s[2 * j], b = s[2 * j + 1];
    s[j] = (odd ? b : a) + dpp_take<CTRL>(odd ? a : b);
  }
}
// Sums over the lanes of V values; a lane gets class_of's, the copies the same bits. 43 instructions for eight values, where
// a sum after the other takes 64.
template <int V>
__device__ __forceinline__ float class_sums(float (&s)[V], int lane) {
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = dpp_add<0x141>(s[v]);  // the mirror lane of eight
  halve<0xB1, V>(s, lane & 1);
  halve<0x4E, V / 2>(reinterpret_cast<float(&)[V / 2]>(s), lane & 2);
  halve<0x128, V / 4>(reinterpret_cast<float(&)[V / 4]>(s), lane & 8);
  if constexpr (V == 16) {  // even rows of sixteen lanes go on with the first, odd ones with the second
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(s[0]), __float_as_uint(s[1]), false, false);
    return swap32_add(__uint_as_float(r[0]) + __uint_as_float(r[1]));
  } else {
    return swap32_add(swap16_add(s[0]));
  }
}
// Sum and largest over the classes.
template <int V>
__device__ __forceinline__ float over_classes_sum(float x) {
  x = dpp_add<0xB1>(x), x = dpp_add<0x4E>(x), x = dpp_add<0x128>(x);
  return V == 16 ? swap16_add(x) : x;
}
template <int V>
__device__ __forceinline__ float over_classes_max(float x) {
  x = fmaxf(x, dpp_take<0xB1>(x)), x = fmaxf(x, dpp_take<0x4E>(x)), x = fmaxf(x, dpp_take<0x128>(x));
  if constexpr (V == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return x;
}

// The weight in registers, and the bias of the lane's class: -inf past the last one.
template <typename T, int V, int E>
struct Head {
  float w[V][E], b;
  int lane, cls;
  __device__ __forceinline__ explicit Head(const CeParams& p) : lane(threadIdx.x % 64), cls(class_of<V>(lane)) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < E; ++e)
        w[v][e] = v < p.classes && e * 64 + lane < p.width ? (float)((const T*)p.w.p)[v * p.w.sr + e * 64 + lane] : 0.f;
    b = cls >= p.classes ? -__builtin_inff() : p.bias ? (float)((const T*)p.bias)[cls] : 0.f;
  }
  // The lane's class's logit less the largest one, the exponential of that, and the sum of all exponentials without the
  // largest one's, which is 1: so small losses keep their digits.
  __device__ __forceinline__ void softmax(const float (&x)[E], float& z, float& ex, float& rest) const {
    float s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s[v] = fmaf(x[e], w[v][e], s[v]);
    }
    z = class_sums<V>(s, lane) + b;
    const float top = over_classes_max<V>(z);
    const int first = class_of<V>(__ffsll(__ballot(z == top)) - 1);
    z -= top;
    ex = expf(z);
    rest = over_classes_sum<V>(cls == first ? ex - 1.f : ex);
  }
};

// part: [workgroup] of (sum of losses, kept rows), where there are several.
template <typename T, int V, int E>
__global__ __launch_bounds__(kWaves * 64) void head_fwd_kernel(CeParams p, float2* part) {
  __shared__ float2 red[kWaves];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Head<T, V, E> head(p);
  float total = 0.f;
  int kept = 0;
  for (int64_t row = (int64_t)blockIdx.x * kWaves + wave; row < p.n; row += (int64_t)gridDim.x * kWaves) {
    const int64_t t = load_target(p, row);
    float loss = 0.f;
    if (t != p.ignore) {
      if (t < 0 || t >= p.classes) {
        loss = __builtin_nanf("");
      } else {
        float x[E], z, ex, rest;
        load_row<T, E>(x, p.x.p, p.x.sr, row, p.width, lane);
        head.softmax(x, z, ex, rest);
        loss = log1pf(rest) - __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(z), __builtin_amdgcn_readfirstlane(lane_of((int)t))));
        ++kept;
      }
    }
    if (p.reduction == kCeNone) {
      if (lane == 0) p.loss[row] = loss;
    }
    total += loss;
  }
  if (p.reduction == kCeNone) return;
  if (lane == 0) red[wave] = float2{total, (float)kept};
  __syncthreads();
  if (threadIdx.x == 0) {
    float2 s = red[0];
    for (int w = 1; w < kWaves; ++w) s.x += red[w].x, s.y += red[w].y;
    if (gridDim.x == 1) {
      p.loss[0] = p.reduction == kCeMean ? s.x / s.y : s.x;
      p.stats[0] = s.y;
    } else {
      part[blockIdx.x] = s;
    }
  }
}

__global__ __launch_bounds__(64) void head_total_kernel(CeParams p, const float2* part, int parts) {
  float s[2] = {0.f, 0.f};
  for (int i = threadIdx.x; i < parts; i += 64) s[0] += part[i].x, s[1] += part[i].y;
  s[0] = lane_sum<64>(s[0]), s[1] = lane_sum<64>(s[1]);
  if (threadIdx.x == 0) {
    p.loss[0] = p.reduction == kCeMean ? s[0] / s[1] : s[0];
    p.stats[0] = s[1];
  }
}

// part: [workgroup][classes * width + classes], the sums of dweight and dbias, where there are several.
template <typename T, int V, int E>
__global__ __launch_bounds__(kWaves * 64) void head_bwd_kernel(CeParams p, float* part) {
  __shared__ float red[kWaves][64 * E];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Head<T, V, E> head(p);
  const bool sums = p.dw.p || p.db;
  float dw[V][E], db = 0.f;  // db: of the lane's class
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int e = 0; e < E; ++e) dw[v][e] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * kWaves + wave; row < p.n; row += (int64_t)gridDim.x * kWaves) {
    const int64_t t = load_target(p, row);
    float dx[E];
    if (t == p.ignore || t < 0 || t >= p.classes) {
#pragma unroll
      for (int e = 0; e < E; ++e) dx[e] = t == p.ignore ? 0.f : __builtin_nanf("");
    } else {
      const float g = p.reduction == kCeNone ? p.gout[row] : p.reduction == kCeMean ? p.gout[0] / p.stats[0] : p.gout[0];
      float x[E], z, ex, rest;
      load_row<T, E>(x, p.x.p, p.x.sr, row, p.width, lane);
      head.softmax(x, z, ex, rest);
      // the target's share less 1 is the others' sum: without cancellation
      const float others = over_classes_sum<V>(head.cls == t ? 0.f : ex);
      const float mine = (head.cls == t ? -others : ex) * (g / (1.f + rest));
      db += mine;
#pragma unroll
      for (int e = 0; e < E; ++e) dx[e] = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = v < p.classes ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), lane_of(v))) : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          dx[e] = fmaf(d, head.w[v][e], dx[e]);
          dw[v][e] = fmaf(d, x[e], dw[v][e]);
        }
      }
    }
    if (p.dx.p) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * 64 + lane < p.width) ((T*)p.dx.p)[row * p.dx.sr + e * 64 + lane] = (T)dx[e];
    }
  }
  if (!sums) return;
  const bool alone = gridDim.x == 1;
  const int64_t cols = p.classes * p.width;
  float* mine = part + (int64_t)blockIdx.x * (cols + p.classes);
  // class by class, the waves' sums added in order
  for (int v = 0; v < (int)p.classes; ++v) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) s = k == v ? dw[k][e] : s;
      red[wave][e * 64 + lane] = s;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.width; c += kWaves * 64) {
      float s = red[0][c];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) s += red[w][c];
      if (!alone)
        mine[(int64_t)v * p.width + c] = s;
      else if (p.dw.p)
        ((T*)p.dw.p)[(int64_t)v * p.dw.sr + c] = (T)s;
    }
  }
  __syncthreads();
  if (lane == lane_of(head.cls)) red[wave][head.cls] = db;
  __syncthreads();
  if (threadIdx.x < p.classes) {
    float s = red[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s += red[w][threadIdx.x];
    if (!alone)
      mine[cols + threadIdx.x] = s;
    else if (p.db)
      ((T*)p.db)[threadIdx.x] = (T)s;
  }
}

// Workgroups: one up to 64 rows (no second launch), else one for every 32 rows, at most four a CU where the weight takes eight
// registers and two where it takes more and the loads of a row are in flight together. Forward and backward in us with
// two and four a CU: (10^6, 64) of 5 classes float32 827 and 757, (10^5, 256) of 16 classes 190 and 230.
int groups(const CeParams& p) {
  const int64_t most = (p.classes <= 8 && p.width <= 64 ? 4 : 2) * (int64_t)device_cu_count(), want = (p.n + 4 * kWaves - 1) / (4 * kWaves);
  return (int)(p.n <= kAloneRows ? 1 : want < most ? want : most);
}

template <typename T, int V, int E>
hipError_t launch(const CeParams& p, bool backward, hipStream_t st) {
  if (!backward) {
    const int n = groups(p);
    head_fwd_kernel<T, V, E><<<n, kWaves * 64, 0, st>>>(p, (float2*)p.ws);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || n == 1 || p.reduction == kCeNone) return e;
    head_total_kernel<<<1, 64, 0, st>>>(p, (const float2*)p.ws, n);
    return hipGetLastError();
  }
  const int64_t cols = p.classes * p.width, all = cols + p.classes;
  // the second launch writes whole rows: a gradient whose rows are apart takes one workgroup
  const int n = p.dw.p && p.dw.sr != p.width ? 1 : groups(p);
  head_bwd_kernel<T, V, E><<<n, kWaves * 64, 0, st>>>(p, (float*)p.ws);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || n == 1 || !(p.dw.p || p.db)) return e;
  column_sum_kernel<T><<<dim3((unsigned)((all + 63) / 64)), 1024, 0, st>>>((const float*)p.ws, n, all, cols, (T*)p.dw.p, (T*)p.db, nullptr);
  return hipGetLastError();
}

template <typename T>
hipError_t by_size(const CeParams& p, bool backward, hipStream_t st) {
  if (p.classes <= 8) {
    if (p.width <= 64) return launch<T, 8, 1>(p, backward, st);
    if (p.width <= 128) return launch<T, 8, 2>(p, backward, st);
    if (p.width <= 256) return launch<T, 8, 4>(p, backward, st);
    return launch<T, 8, 8>(p, backward, st);
  }
  if (p.width <= 64) return launch<T, 16, 1>(p, backward, st);
  if (p.width <= 128) return launch<T, 16, 2>(p, backward, st);
  return launch<T, 16, 4>(p, backward, st);
}

}  // namespace

// The weight and its gradient's sums take up to 64 registers each. (A call's two halves decide alike: the gradients'
// strides are not asked.)
bool ce_head_takes(const CeParams& p) { return p.n > 0 && ((p.classes <= 8 && p.width <= 512) || (p.classes <= 16 && p.width <= 256)); }

int64_t ce_head_ws_bytes(const CeParams& p, bool backward) {
  return 256 + (int64_t)groups(p) * (backward ? 4 * (p.classes * p.width + p.classes) : (int64_t)sizeof(float2));
}

hipError_t launch_ce_head(const CeParams& p, bool backward, hipStream_t st) {
  if (p.dtype == 0) return by_size<float>(p, backward, st);
  if (p.dtype == 1) return by_size<_Float16>(p, backward, st);
  return by_size<__bf16>(p, backward, st);
}

}  // namespace theria
