// Layer norm over the last dimension: forward, backward and double backward (gfx950).
//
// With xh = (x - mu) r, r = (var + eps)^-1/2, gw = dout o w and, for a row t, P(t) = r (t - mean t - xh mean(t o xh)):
//   forward          y = xh o w + b, saving mu and r
//   backward         dx = P(gw), dw = sum_rows dout o xh, db = sum_rows dout
//   double backward  cotangents u of dx, a of dw, c of db:
//                      G_dout = w o P(u) + a o xh + c,   G_w = sum_rows dout o P(u),
//                      G_x = P(h) - r xh mean(u o dx),   h = a o dout - r (u mean(gw o xh) + gw mean(u o xh))
//                    (P(h) is the path through xh, the other term the one through r). Every sum it needs is one of seven
//                    sums over the row of products of the inputs, taken in one sweep: h enters them linearly.
//
// All are bound by memory: each tensor is read once and written once, a row held in registers between its sums and
// its outputs. A row belongs to a team of 8 to 64 lanes or of a whole workgroup, by its width, so that a thread holds
// at most 16 of its elements of each tensor. Sums over the rows (dw, db, G_w) stay in the threads' registers while a
// workgroup walks its rows; each workgroup writes one partial row of them and a second launch adds the partial rows in
// a fixed order (no atomics: the same bits on every run).
#include "token_common.hpp"
#include "token_params.hpp"

namespace theria {
namespace {

template <int TPR>
constexpr int kBlock = TPR > 256 ? TPR : 256;

// TAIL: the width is no multiple of VEC, so that a row's last vector is partly filled (a template parameter, since the
// branch costs whole vectors too: backward of (8192, 4096) bfloat16 56 us with it, 45 us without).
//
// The columns that thread t of a team holds: NPT vectors of VEC, TPR vectors apart.
template <int VEC, int TPR>
__device__ __forceinline__ int col_of(int i, int t) {
  return (i * TPR + t) * VEC;
}

template <typename T, int VEC, int NPT, int TPR, bool TAIL>
__device__ __forceinline__ void load_row(RawVec<T, VEC> (&raw)[NPT], const T* row, int t, int width, bool live) {
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int c = col_of<VEC, TPR>(i, t);
    raw[i].template load<TAIL>(row + c, live ? width - c : 0);
  }
}

// VEC parameters from column c, or the given constant where the parameter is absent.
template <typename WT, int VEC, bool TAIL>
__device__ __forceinline__ void load_param(float (&f)[VEC], const void* p, int c, int width, float absent) {
  if (p) {
    RawVec<WT, VEC> r;
    r.template load<TAIL>((const WT*)p + c, width - c);
    r.get(f);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = absent;
  }
}

template <typename T, typename WT, int VEC, int NPT, int TPR, bool TAIL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_fwd_kernel(NormParams p) {
  constexpr int TEAMS = kBlock<TPR> / TPR;
  __shared__ float red[2][16];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR;
  const bool live = row < p.rows;
  RawVec<T, VEC> raw[NPT];
  load_row<T, VEC, NPT, TPR, TAIL>(raw, (const T*)p.x.p + row * p.x.sr, t, p.width, live);
  float x[NPT][VEC];
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    raw[i].get(x[i]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[0] += x[i][e];
  }
  team_sum<TPR, 1>(s, red[0]);
  const float mean = s[0] / (float)p.width;
  // the variance from the centred values: no cancellation for rows far from zero
  float q[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int have = p.width - col_of<VEC, TPR>(i, t);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      x[i][e] -= mean;
      q[0] += e * TAIL < have ? x[i][e] * x[i][e] : 0.f;
    }
  }
  team_sum<TPR, 1>(q, red[1]);
  const float rstd = 1.0f / sqrtf(q[0] / (float)p.width + p.eps);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int c = col_of<VEC, TPR>(i, t);
    if (c >= p.width) continue;
    float w[VEC], b[VEC];
    load_param<WT, VEC, TAIL>(w, p.weight, c, p.width, 1.f);
    load_param<WT, VEC, TAIL>(b, p.bias, c, p.width, 0.f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[i][e] = x[i][e] * rstd * w[e] + b[e];
    RawVec<T, VEC> out;
    out.set(x[i]);
    out.template store<TAIL>((T*)p.y.p + row * p.y.sr + c, p.width - c);
  }
  if (t == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
}

// A workgroup's column sums: the teams' sums added and written as one partial row. acc: the thread's columns.
template <int VEC, int NPT, int TPR>
__device__ __forceinline__ void write_partial(float (&acc)[NPT][VEC], float* out, int width, float* lds) {
  constexpr int COLS = VEC * NPT * TPR, WAVES = 4;
  const int t = threadIdx.x % TPR, wave = threadIdx.x / 64;
  if constexpr (TPR < 64) {
#pragma unroll
    for (int i = 0; i < NPT; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[i][e] = across_groups<TPR>(acc[i][e]);
  }
  if constexpr (TPR <= 64) {
    __syncthreads();
    if (threadIdx.x % 64 < TPR) {
#pragma unroll
      for (int i = 0; i < NPT; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) lds[wave * COLS + col_of<VEC, TPR>(i, t) + e] = acc[i][e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += kBlock<TPR>) {
      float s = lds[c];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) s += lds[w * COLS + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int c = col_of<VEC, TPR>(i, t);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c + e < width) out[c + e] = acc[i][e];
    }
  }
}

template <int VEC, int NPT, int TPR>
constexpr int kPartialLds = TPR <= 64 ? 4 * VEC * NPT * TPR : 1;

template <typename T, typename WT, int VEC, int NPT, int TPR, bool TAIL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_bwd_kernel(NormParams p) {
  constexpr int TEAMS = kBlock<TPR> / TPR;
  __shared__ float red[2][2 * 16];
  __shared__ float lds[kPartialLds<VEC, NPT, TPR>];
  const int t = threadIdx.x % TPR, width = p.width;
  const float inv = 1.0f / (float)width;
  const bool sums = p.dw || p.db;
  float dw[NPT][VEC], db[NPT][VEC];
#pragma unroll
  for (int i = 0; i < NPT; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f;

  const int64_t step = (int64_t)gridDim.x * TEAMS;
  int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR;
  RawVec<T, VEC> rx[NPT], rg[NPT];
  load_row<T, VEC, NPT, TPR, TAIL>(rx, (const T*)p.x.p + row * p.x.sr, t, width, row < p.rows);
  load_row<T, VEC, NPT, TPR, TAIL>(rg, (const T*)p.dout.p + row * p.dout.sr, t, width, row < p.rows);
  int turn = 0;
  // teams of a wave leave the loop apart; a workgroup-wide team leaves it as one (its row is the workgroup's)
#pragma unroll 1
  while (row < p.rows) {
    float x[NPT][VEC], g[NPT][VEC];
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      rx[i].get(x[i]);
      rg[i].get(g[i]);
    }
    // the next row's loads go out before this row's sums
    const int64_t next = row + step;
    load_row<T, VEC, NPT, TPR, TAIL>(rx, (const T*)p.x.p + next * p.x.sr, t, width, next < p.rows);
    load_row<T, VEC, NPT, TPR, TAIL>(rg, (const T*)p.dout.p + next * p.dout.sr, t, width, next < p.rows);
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int c = col_of<VEC, TPR>(i, t);
      if (c < width) {
        float w[VEC];
        load_param<WT, VEC, TAIL>(w, p.weight, c, p.width, 1.f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          x[i][e] = (x[i][e] - mean) * rstd;
          dw[i][e] += g[i][e] * x[i][e];
          db[i][e] += g[i][e];
          g[i][e] *= w[e];
          s[0] += g[i][e];
          s[1] += g[i][e] * x[i][e];
        }
      }
    }
    if (p.dx.p) {
      team_sum<TPR, 2>(s, red[turn]);
      turn ^= 1;
      const float m1 = s[0] * inv, m2 = s[1] * inv;
#pragma unroll
      for (int i = 0; i < NPT; ++i) {
        const int c = col_of<VEC, TPR>(i, t);
        if (c < width) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) g[i][e] = rstd * (g[i][e] - m1 - x[i][e] * m2);
          RawVec<T, VEC> out;
          out.set(g[i]);
          out.template store<TAIL>((T*)p.dx.p + row * p.dx.sr + c, width - c);
        }
      }
    }
    row = next;
  }
  if (!sums) return;
  float* part = p.ws + (int64_t)blockIdx.x * 2 * width;
  write_partial<VEC, NPT, TPR>(dw, part, width, lds);
  write_partial<VEC, NPT, TPR>(db, part + width, width, lds);
}

template <typename T, typename WT, int VEC, int NPT, int TPR, bool TAIL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_bwd_bwd_kernel(NormParams p) {
  constexpr int TEAMS = kBlock<TPR> / TPR;
  __shared__ float red[2][7 * 16];
  __shared__ float lds[kPartialLds<VEC, NPT, TPR>];
  const int t = threadIdx.x % TPR, width = p.width;
  const float inv = 1.0f / (float)width;
  float gw_sum[NPT][VEC];
#pragma unroll
  for (int i = 0; i < NPT; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) gw_sum[i][e] = 0.f;

  int turn = 0;
#pragma unroll 1
  for (int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR; row < p.rows; row += (int64_t)gridDim.x * TEAMS) {
    RawVec<T, VEC> rx[NPT], rg[NPT], ru[NPT];
    load_row<T, VEC, NPT, TPR, TAIL>(rx, (const T*)p.x.p + row * p.x.sr, t, width, true);
    load_row<T, VEC, NPT, TPR, TAIL>(rg, (const T*)p.dout.p + row * p.dout.sr, t, width, true);
    load_row<T, VEC, NPT, TPR, TAIL>(ru, (const T*)p.gdx.p + row * p.gdx.sr, t, width, p.gdx.p != nullptr);
    const float mean = p.mean[row], rstd = p.rstd[row];
    float x[NPT][VEC], g[NPT][VEC], u[NPT][VEC];
    // sums over the row: gw, gw xh, u, u xh, u gw, a dout, a dout xh
    float s[7] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int c = col_of<VEC, TPR>(i, t);
      rx[i].get(x[i]);
      rg[i].get(g[i]);
      ru[i].get(u[i]);
      if (c < width) {
        float w[VEC], a[VEC];
        load_param<WT, VEC, TAIL>(w, p.weight, c, p.width, 1.f);
        load_param<WT, VEC, TAIL>(a, p.gdw, c, p.width, 0.f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          x[i][e] = (x[i][e] - mean) * rstd;
          const float gw = g[i][e] * w[e], ag = a[e] * g[i][e];
          s[0] += gw;
          s[1] += gw * x[i][e];
          s[2] += u[i][e];
          s[3] += u[i][e] * x[i][e];
          s[4] += u[i][e] * gw;
          s[5] += ag;
          s[6] += ag * x[i][e];
        }
      }
    }
    team_sum<TPR, 7>(s, red[turn]);
    turn ^= 1;
    const float m_gx = s[1] * inv, m_u = s[2] * inv, m_ux = s[3] * inv;
    // mean(u o dx) and the means of h and h o xh
    const float m_udx = rstd * (s[4] - s[2] * s[0] * inv - s[3] * m_gx) * inv;
    const float m_h = (s[5] - rstd * (s[2] * m_gx + s[0] * m_ux)) * inv;
    const float m_hx = (s[6] - rstd * (s[3] * m_gx + s[1] * m_ux)) * inv;
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int c = col_of<VEC, TPR>(i, t);
      if (c >= width) continue;
      float w[VEC], a[VEC], b[VEC];
      load_param<WT, VEC, TAIL>(w, p.weight, c, p.width, 1.f);
      load_param<WT, VEC, TAIL>(a, p.gdw, c, p.width, 0.f);
      load_param<WT, VEC, TAIL>(b, p.gdb, c, p.width, 0.f);
      float gx[VEC], gg[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float pu = rstd * (u[i][e] - m_u - x[i][e] * m_ux);
        const float h = a[e] * g[i][e] - rstd * (u[i][e] * m_gx + g[i][e] * w[e] * m_ux);
        gx[e] = rstd * (h - m_h - x[i][e] * (m_hx + m_udx));
        gg[e] = w[e] * pu + a[e] * x[i][e] + b[e];
        gw_sum[i][e] += g[i][e] * pu;
      }
      RawVec<T, VEC> out;
      if (p.out_gx.p) {
        out.set(gx);
        out.template store<TAIL>((T*)p.out_gx.p + row * p.out_gx.sr + c, width - c);
      }
      if (p.out_gdout.p) {
        out.set(gg);
        out.template store<TAIL>((T*)p.out_gdout.p + row * p.out_gdout.sr + c, width - c);
      }
    }
  }
  if (p.out_gw) write_partial<VEC, NPT, TPR>(gw_sum, p.ws + (int64_t)blockIdx.x * width, width, lds);
}

// Teams by width, in vectors of 16 bytes: at most 16 elements of a tensor for each thread.
struct Plan {
  int npt, tpr;
};
Plan plan_of(const NormParams& p) {
  const int vec = p.dtype == 0 ? 4 : 8, n = (p.width + vec - 1) / vec;
  if (n <= 64) return {1, n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : 64};
  if (n <= 128) return {2, 64};
  if (vec == 4) return n <= 256 ? Plan{4, 64} : n <= 512 ? Plan{2, 256} : n <= 1024 ? Plan{4, 256} : n <= 2048 ? Plan{2, 1024} : Plan{4, 1024};
  return n <= 256 ? Plan{1, 256} : n <= 512 ? Plan{2, 256} : n <= 1024 ? Plan{1, 1024} : Plan{2, 1024};
}

// Teams of a workgroup.
int teams_of(const Plan& pl) { return pl.tpr >= 256 ? 1 : 256 / pl.tpr; }

// Workgroups of a launch that sums over the rows. More hide more latency and write more partial rows, eight bytes of traffic
// a column each: two a CU while those are over a fourteenth of the rows' own bytes, up to four (16-bit) or three. Teams of
// 1024 threads, one a CU. Backward in us with 1, 2, 3, 4, 6 a CU: (8192, 4096) bfloat16 69, 53, 56, 60, 74; (65536, 2048)
// bfloat16 371, 214, 175, 169, 168, float32 399, 302, 303, 310, 318; (400000, 64) float32 102, 62, 56, 57, 62; (4096, 16384)
// bfloat16 109, 131, 159, 188, 244. Fewer where a team would get fewer than two rows.
int walkers(const NormParams& p, const Plan& pl) {
  const int64_t cus = device_cu_count(), two = 2 * teams_of(pl), want = (p.rows + two - 1) / two;
  int64_t most = cus;
  if (pl.tpr < 1024) {
    const int64_t few = 2 * cus, many = (p.dtype == 0 ? pl.tpr == 256 ? 2 : 3 : 4) * cus, cheap = p.rows * (p.dtype == 0 ? 4 : 2) / 76;
    most = cheap < few ? few : cheap < many ? cheap : many;
  }
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

struct Fwd {
  template <typename T, typename WT, int VEC, int NPT, int TPR, bool TAIL>
  static hipError_t run(const NormParams& p, hipStream_t st) {
    constexpr int TEAMS = kBlock<TPR> / TPR;
    constexpr int64_t most = int64_t(1) << 21;  // rows: a launch holds fewer than 2^32 threads
    for (int64_t r = 0; r < p.rows; r += most) {
      NormParams q = p;
      q.rows = p.rows - r < most ? p.rows - r : most;
      q.x.p = (const T*)p.x.p + r * p.x.sr;
      q.y.p = (T*)p.y.p + r * p.y.sr;
      q.mean = p.mean + r, q.rstd = p.rstd + r;
      norm_fwd_kernel<T, WT, VEC, NPT, TPR, TAIL><<<dim3((unsigned)((q.rows + TEAMS - 1) / TEAMS)), kBlock<TPR>, 0, st>>>(q);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
};

template <typename WT>
hipError_t finish(const NormParams& p, int parts, int64_t cols, void* out0, void* out1, hipStream_t st) {
  column_sum_kernel<WT><<<dim3((unsigned)((cols + 63) / 64)), 1024, 0, st>>>(p.ws, parts, cols, p.width, (WT*)out0, (WT*)out1, nullptr);
  return hipGetLastError();
}

struct Bwd {
  template <typename T, typename WT, int VEC, int NPT, int TPR, bool TAIL>
  static hipError_t run(const NormParams& p, hipStream_t st) {
    const int n = walkers(p, Plan{NPT, TPR});
    norm_bwd_kernel<T, WT, VEC, NPT, TPR, TAIL><<<n, kBlock<TPR>, 0, st>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !(p.dw || p.db)) return e;
    return finish<WT>(p, n, 2 * (int64_t)p.width, p.dw, p.db, st);
  }
};

struct BwdBwd {
  template <typename T, typename WT, int VEC, int NPT, int TPR, bool TAIL>
  static hipError_t run(const NormParams& p, hipStream_t st) {
    const int n = walkers(p, Plan{NPT, TPR});
    norm_bwd_bwd_kernel<T, WT, VEC, NPT, TPR, TAIL><<<n, kBlock<TPR>, 0, st>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.out_gw) return e;
    return finish<WT>(p, n, p.width, p.out_gw, nullptr, st);
  }
};

template <typename L, typename T, typename WT>
hipError_t by_plan(const NormParams& p, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const Plan pl = plan_of(p);
#define THERIA_NORM_CASE(NPT, TPR)               \
  if (pl.npt == NPT && pl.tpr == TPR)            \
    return p.width % V ? L::template run<T, WT, V, NPT, TPR, true>(p, st) : L::template run<T, WT, V, NPT, TPR, false>(p, st);
  THERIA_NORM_CASE(1, 8)
  THERIA_NORM_CASE(1, 16)
  THERIA_NORM_CASE(1, 32)
  THERIA_NORM_CASE(1, 64)
  THERIA_NORM_CASE(2, 64)
  THERIA_NORM_CASE(2, 256)
  THERIA_NORM_CASE(2, 1024)
  if constexpr (V == 4) {
    THERIA_NORM_CASE(4, 64)
    THERIA_NORM_CASE(4, 256)
    THERIA_NORM_CASE(4, 1024)
  } else {
    THERIA_NORM_CASE(1, 256)
    THERIA_NORM_CASE(1, 1024)
  }
#undef THERIA_NORM_CASE
  return hipErrorInvalidValue;
}

template <typename L>
hipError_t by_type(const NormParams& p, hipStream_t st) {
  if (p.dtype == 0) return by_plan<L, float, float>(p, st);
  if (p.dtype == 1) return p.param_dtype == 0 ? by_plan<L, _Float16, float>(p, st) : by_plan<L, _Float16, _Float16>(p, st);
  return p.param_dtype == 0 ? by_plan<L, __bf16, float>(p, st) : by_plan<L, __bf16, __bf16>(p, st);
}

}  // namespace

int64_t norm_ws_floats(const NormParams& p) {
  return p.rows > 0 ? (int64_t)walkers(p, plan_of(p)) * 2 * p.width : 0;
}
hipError_t launch_norm_fwd(const NormParams& p, hipStream_t st) { return by_type<Fwd>(p, st); }
hipError_t launch_norm_bwd(const NormParams& p, hipStream_t st) { return by_type<Bwd>(p, st); }
hipError_t launch_norm_bwd_bwd(const NormParams& p, hipStream_t st) { return by_type<BwdBwd>(p, st); }

}  // namespace theria
