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

// How a row's last vector is filled (a template parameter: a branch around loads costs whole vectors too, backward of (8192, 4096)
// bfloat16 56 us with one, 45 us without).
enum Tail {
  kWhole,  // the width is a multiple of VEC
  kOver,   // it is not: the last vector is loaded from VEC before the row's end and shifted when it is used. Loads of
           // single elements are waited for where they stand, and every load before them too: backward of (130000, 1001)
           // bfloat16 168 us against 153 us.
  kSingle  // the width is below VEC: single elements
};

// The columns that thread t of a team holds: NPT vectors of VEC, TPR vectors apart.
template <int VEC, int TPR>
__device__ __forceinline__ int col_of(int i, int t) {
  return (i * TPR + t) * VEC;
}

// The vector at column c of a row (zeros where there is none), and its values.
template <Tail TAIL, typename T, int VEC>
__device__ __forceinline__ void load_vec(RawVec<T, VEC>& raw, const T* row, int c, int width, bool live) {
  if constexpr (TAIL == kOver)
    raw.template load<false>(row + (c + VEC > width ? width - VEC : c), live ? width - c : 0);
  else
    raw.template load<TAIL == kSingle>(row + c, live ? width - c : 0);
}
template <Tail TAIL, typename T, int VEC>
__device__ __forceinline__ void values_of(float (&f)[VEC], RawVec<T, VEC> raw, int c, int width) {
  if (TAIL == kOver && c < width && c + VEC > width) raw.shift_down(VEC - width % VEC);
  raw.get(f);
}

template <typename T, int VEC, int NPT, int TPR, Tail TAIL>
__device__ __forceinline__ void load_row(RawVec<T, VEC> (&raw)[NPT], const T* row, int t, int width, bool live) {
#pragma unroll
  for (int i = 0; i < NPT; ++i) load_vec<TAIL>(raw[i], row, col_of<VEC, TPR>(i, t), width, live);
}
template <typename T, int VEC, int NPT, int TPR, Tail TAIL>
__device__ __forceinline__ void values(float (&f)[NPT][VEC], const RawVec<T, VEC> (&raw)[NPT], int t, int width) {
#pragma unroll
  for (int i = 0; i < NPT; ++i) values_of<TAIL>(f[i], raw[i], col_of<VEC, TPR>(i, t), width);
}

// VEC parameters from column c, or the given constant where the parameter is absent.
template <typename WT, int VEC, Tail TAIL>
__device__ __forceinline__ void load_param(float (&f)[VEC], const void* p, int c, int width, float absent) {
  if (p) {
    RawVec<WT, VEC> r;
    load_vec<TAIL>(r, (const WT*)p, c, width, true);
    values_of<TAIL>(f, r, c, width);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = absent;
  }
}

// A parameter's columns of a thread: held in registers (HOLD) by a team that walks its rows with the next row's loads on
// their way. Vector memory answers in order, so that a load behind those would wait for that row, too. Backward of (65536,
// 2048) bfloat16 173 -> 151 us, float32 301 -> 285 us.
template <typename WT, int VEC, int NPT, int TPR, Tail TAIL, bool HOLD>
struct HeldParam {
  const void* p;
  int t, width;
  float absent;
  RawVec<WT, VEC> raw[HOLD ? NPT : 1];

  __device__ __forceinline__ HeldParam(const void* p_, int t_, int width_, float absent_) : p(p_), t(t_), width(width_), absent(absent_) {
    if constexpr (HOLD) {
#pragma unroll
      for (int i = 0; i < NPT; ++i) {
        float f[VEC];
        load_param<WT, VEC, TAIL>(f, p, col_of<VEC, TPR>(i, t), width, absent);
        raw[i].set(f);
      }
    }
  }
  __device__ __forceinline__ void get(float (&f)[VEC], int i) const {
    if constexpr (HOLD)
      raw[i].get(f);
    else
      load_param<WT, VEC, TAIL>(f, p, col_of<VEC, TPR>(i, t), width, absent);
  }
};

template <typename T, typename WT, int VEC, int NPT, int TPR, Tail TAIL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_fwd_kernel(NormParams p) {
  constexpr int TEAMS = kBlock<TPR> / TPR;
  __shared__ float red[2][16];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR;
  const bool live = row < p.rows;
  RawVec<T, VEC> raw[NPT];
  load_row<T, VEC, NPT, TPR, TAIL>(raw, (const T*)p.x.p + row * p.x.sr, t, p.width, live);
  float x[NPT][VEC];
  values<T, VEC, NPT, TPR, TAIL>(x, raw, t, p.width);
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NPT; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[0] += x[i][e];
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
      q[0] += (TAIL == kWhole ? have > 0 : e < have) ? x[i][e] * x[i][e] : 0.f;
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
    out.template store<TAIL != kWhole>((T*)p.y.p + row * p.y.sr + c, p.width - c);
  }
  if (t == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
}

// A thread's sums over its rows. For float32 parameters every sixteen rows are added up first (TWO): one sum over 256 rows
// after the other loses half as much again as a library's tree (mean error of dweight of (65536, 2048) 2.9e-7 against
// 2.1e-7, with TWO 1.7e-7). 16-bit parameters round by far more, and 1024 threads with 16 columns each have no registers left.
template <int VEC, int NPT, bool TWO>
struct RowSums {
  float s[NPT][VEC], far[TWO ? NPT : 1][TWO ? VEC : 1];
  int rows = 0;
  __device__ __forceinline__ RowSums() {
#pragma unroll
    for (int i = 0; i < NPT; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s[i][e] = 0.f;
        if constexpr (TWO) far[i][e] = 0.f;
      }
  }
  __device__ __forceinline__ void end_row() {
    if constexpr (TWO) {
      if (++rows % 16 == 0) join();
    }
  }
  __device__ __forceinline__ void join() {
    if constexpr (TWO) {
#pragma unroll
      for (int i = 0; i < NPT; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) far[i][e] += s[i][e], s[i][e] = 0.f;
    }
  }
  __device__ __forceinline__ float (&total())[NPT][VEC] {
    if constexpr (TWO) {
      join();
      return far;
    } else {
      return s;
    }
  }
};
template <typename WT, int VEC, int NPT, int TPR>
constexpr bool kTwo = sizeof(WT) == 4 && !(TPR == 1024 && NPT * VEC == 16);

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

template <typename T, typename WT, int VEC, int NPT, int TPR, Tail TAIL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_bwd_kernel(NormParams p) {
  constexpr int TEAMS = kBlock<TPR> / TPR;
  constexpr bool HOLD = !(TPR == 1024 && NPT == 4);  // which has no registers left for the weight
  __shared__ float red[2][2 * 16];
  __shared__ float lds[kPartialLds<VEC, NPT, TPR>];
  const int t = threadIdx.x % TPR, width = p.width;
  const float inv = 1.0f / (float)width;
  const bool sums = p.dw || p.db;
  RowSums<VEC, NPT, kTwo<WT, VEC, NPT, TPR>> dw, db;

  const HeldParam<WT, VEC, NPT, TPR, TAIL, HOLD> weight(p.weight, t, width, 1.f);
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR;
  RawVec<T, VEC> rx[NPT], rg[NPT];
  float next_mean = 0.f, next_rstd = 0.f;
  const auto fetch = [&](int64_t r) {
    const bool live = r < p.rows;
    if (live) next_mean = p.mean[r], next_rstd = p.rstd[r];
    load_row<T, VEC, NPT, TPR, TAIL>(rx, (const T*)p.x.p + r * p.x.sr, t, width, live);
    load_row<T, VEC, NPT, TPR, TAIL>(rg, (const T*)p.dout.p + r * p.dout.sr, t, width, live);
  };
  fetch(row);
  int turn = 0;
  // teams of a wave leave the loop apart; a workgroup-wide team leaves it as one (its row is the workgroup's)
#pragma unroll 1
  for (; row < p.rows; row += step) {
    float x[NPT][VEC], g[NPT][VEC];
    values<T, VEC, NPT, TPR, TAIL>(x, rx, t, width);
    values<T, VEC, NPT, TPR, TAIL>(g, rg, t, width);
    const float mean = next_mean, rstd = next_rstd;
    fetch(row + step);  // before this row's sums
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int c = col_of<VEC, TPR>(i, t);
      if (c < width) {
        float w[VEC];
        weight.get(w, i);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          x[i][e] = (x[i][e] - mean) * rstd;
          dw.s[i][e] += g[i][e] * x[i][e];
          db.s[i][e] += g[i][e];
          g[i][e] *= w[e];
          s[0] += g[i][e];
          s[1] += g[i][e] * x[i][e];
        }
      }
    }
    dw.end_row(), db.end_row();
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
          out.template store<TAIL != kWhole>((T*)p.dx.p + row * p.dx.sr + c, width - c);
        }
      }
    }
  }
  if (!sums) return;
  float* part = p.ws + (int64_t)blockIdx.x * 2 * width;
  write_partial<VEC, NPT, TPR>(dw.total(), part, width, lds);
  write_partial<VEC, NPT, TPR>(db.total(), part + width, width, lds);
}

template <typename T, typename WT, int VEC, int NPT, int TPR, Tail TAIL>
__global__ __launch_bounds__(kBlock<TPR>) void norm_bwd_bwd_kernel(NormParams p) {
  constexpr int TEAMS = kBlock<TPR> / TPR;
  constexpr bool AHEAD = TPR < 1024;  // the next row's loads and the parameters in registers: 1024 threads have too few
  __shared__ float red[2][7 * 16];
  __shared__ float lds[kPartialLds<VEC, NPT, TPR>];
  const int t = threadIdx.x % TPR, width = p.width;
  const float inv = 1.0f / (float)width;
  RowSums<VEC, NPT, kTwo<WT, VEC, NPT, TPR>> gw_sum;
  const HeldParam<WT, VEC, NPT, TPR, TAIL, AHEAD> weight(p.weight, t, width, 1.f), gdw(p.gdw, t, width, 0.f), gdb(p.gdb, t, width, 0.f);
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR;
  RawVec<T, VEC> rx[NPT], rg[NPT], ru[NPT];
  float next_mean = 0.f, next_rstd = 0.f;
  const auto fetch = [&](int64_t r) {
    const bool live = r < p.rows;
    if (live) next_mean = p.mean[r], next_rstd = p.rstd[r];
    load_row<T, VEC, NPT, TPR, TAIL>(rx, (const T*)p.x.p + r * p.x.sr, t, width, live);
    load_row<T, VEC, NPT, TPR, TAIL>(rg, (const T*)p.dout.p + r * p.dout.sr, t, width, live);
    load_row<T, VEC, NPT, TPR, TAIL>(ru, (const T*)p.gdx.p + r * p.gdx.sr, t, width, live && p.gdx.p);
  };
  if constexpr (AHEAD) fetch(row);
  int turn = 0;
#pragma unroll 1
  for (; row < p.rows; row += step) {
    if constexpr (!AHEAD) fetch(row);
    float x[NPT][VEC], g[NPT][VEC], u[NPT][VEC];
    values<T, VEC, NPT, TPR, TAIL>(x, rx, t, width);
    values<T, VEC, NPT, TPR, TAIL>(g, rg, t, width);
    values<T, VEC, NPT, TPR, TAIL>(u, ru, t, width);
    const float mean = next_mean, rstd = next_rstd;
    if constexpr (AHEAD) fetch(row + step);
    // sums over the row: gw, gw xh, u, u xh, u gw, a dout, a dout xh
    float s[7] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int c = col_of<VEC, TPR>(i, t);
      if (c < width) {
        float w[VEC], a[VEC];
        weight.get(w, i);
        gdw.get(a, i);
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
      weight.get(w, i);
      gdw.get(a, i);
      gdb.get(b, i);
      float gx[VEC], gg[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float pu = rstd * (u[i][e] - m_u - x[i][e] * m_ux);
        const float h = a[e] * g[i][e] - rstd * (u[i][e] * m_gx + g[i][e] * w[e] * m_ux);
        gx[e] = rstd * (h - m_h - x[i][e] * (m_hx + m_udx));
        gg[e] = w[e] * pu + a[e] * x[i][e] + b[e];
        gw_sum.s[i][e] += g[i][e] * pu;
      }
      RawVec<T, VEC> out;
      if (p.out_gx.p) {
        out.set(gx);
        out.template store<TAIL != kWhole>((T*)p.out_gx.p + row * p.out_gx.sr + c, width - c);
      }
      if (p.out_gdout.p) {
        out.set(gg);
        out.template store<TAIL != kWhole>((T*)p.out_gdout.p + row * p.out_gdout.sr + c, width - c);
      }
    }
    gw_sum.end_row();
  }
  if (p.out_gw) write_partial<VEC, NPT, TPR>(gw_sum.total(), p.ws + (int64_t)blockIdx.x * width, width, lds);
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

// Workgroups of a launch that sums over the rows. A workgroup has the next rows of its teams on their way, 8 KiB of each
// tensor on a CU hide what latency there is, and every further workgroup writes another partial row: one a CU from
// 8 KiB of rows on, more below it, and two at least with 16-bit rows, whose unpacking takes longer. Backward in us with 1, 2, 3, 4 a CU:
// bfloat16 (65536, 2048) 217, 149, 149, 162; (80000, 1500) 326, 193, 149, 144; (130000, 1001) 182, 154, 163, 168; (16384,
// 4096) 86, 91, 97, 103, its double backward 162, 141, 149, 147; (10^6, 50) 120, 77, 65, 69; float32 (65000, 1001) 143, 157,
// 161, 164; (200000, 256) 169, 119, 120, 121. With few rows the partial rows count more: (2048, 4096) bfloat16 21, 26, 32, 39,
// so that a further one has to have six rows for each team (two for the first).
int walkers(const NormParams& p, const Plan& pl) {
  const int64_t cus = device_cu_count(), teams = teams_of(pl), bytes = teams * p.width * (p.dtype == 0 ? 4 : 2);
  int64_t each = 1;
  if (pl.tpr < 1024) {
    each = (8192 + bytes - 1) / bytes;
    if (p.dtype != 0 && each < 2) each = 2;
    if (each > 4) each = 4;
    while (each > 1 && p.rows < 6 * teams * each * cus) --each;
  }
  const int64_t want = (p.rows + 2 * teams - 1) / (2 * teams), most = each * cus;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

struct Fwd {
  template <typename T, typename WT, int VEC, int NPT, int TPR, Tail TAIL>
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
  template <typename T, typename WT, int VEC, int NPT, int TPR, Tail TAIL>
  static hipError_t run(const NormParams& p, hipStream_t st) {
    const int n = walkers(p, Plan{NPT, TPR});
    norm_bwd_kernel<T, WT, VEC, NPT, TPR, TAIL><<<n, kBlock<TPR>, 0, st>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !(p.dw || p.db)) return e;
    return finish<WT>(p, n, 2 * (int64_t)p.width, p.dw, p.db, st);
  }
};

struct BwdBwd {
  template <typename T, typename WT, int VEC, int NPT, int TPR, Tail TAIL>
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
  if (p.width < V) return L::template run<T, WT, V, 1, 8, kSingle>(p, st);
#define THERIA_NORM_CASE(NPT, TPR)               \
  if (pl.npt == NPT && pl.tpr == TPR)            \
    return p.width % V ? L::template run<T, WT, V, NPT, TPR, kOver>(p, st) : L::template run<T, WT, V, NPT, TPR, kWhole>(p, st);
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
