// Cross entropy of the logits z = x W^T + b of a linear head, and its gradient, without keeping the logits (gfx950).
//
//   forward    loss_n = log sum_v exp(z_nv) - z_{n, t_n}
//   backward   dz = (softmax(z) - onehot(t)) g_n;   dx = dz W,   dW = dz^T x,   db = sum_n dz
//
// Rows whose target is ignored cost nothing: a first launch lists the kept rows, a second one gathers them, and every
// product runs over those alone (what an ignored row holds is never read). Forward: tiles of z stay in the accumulators
// of the product, whose epilogue takes the largest logit and the sum of exponentials of each row over the tile's classes;
// a small launch joins the tiles. Backward: for a piece of the vocabulary at a time, z is formed again, dz leaves the
// epilogue in 16 bits, and two products turn the piece's dz into its rows of dW and its share of dx, which is summed in
// float32. 8 N V D operations, two of them the recomputed logits; the workspace is the piece's dz, whatever the vocabulary.
//
// dz enters the products in the inputs' 16-bit type, as an operand of a matrix product does everywhere here: one rounding
// of at most 2^-8 (bfloat16) or 2^-11 (float16) of each entry, which sums over many of them average out. A row's own target
// is the entry that no sum averages in dx: what its rounding left is kept in float32 and added to dx with the target's row
// of W (bfloat16 dx of (4000, 300, 64), relative error: 1.68e-3, of which 1.66e-3 is dx's own rounding; without, 2.44e-3).
// dz is held without the loss's own factor (1 / kept rows, or the largest |g|), which multiplies the float32 sums, and
// in float16 times 2^14, so that probabilities down to 2^-38 do not vanish.
//
// float32. Up to 256 rows the operands are multiplied as they are (v_mfma_f32_32x32x2_f32): reading W is most of the work. More
// rows take planes of 16-bit terms (token_gemm.hpp), laid out by a launch before. For the logits two float16 terms, x = h
// + m to 2^-22, and three products of them (m m, 2^-22 of the product at most and 2^-25 on average, is dropped): each row of
// x and W is first scaled by the power of two that brings its largest element to 2^13, which the epilogue takes back, so that
// nothing leaves float16's range. For the gradients, whose sums run over rows of any size, three bfloat16 terms and six
// products. ((48, 32000, 4096) forward and gradients: 0.76 ms as they are, 2 ms in planes; (2000, 10000, 1024): 0.87 ms in
// planes, of six products throughout 1.25 ms.)
#include <type_traits>

#include "token_common.hpp"
#include "token_gemm.hpp"
#include "token_params.hpp"

namespace theria {
namespace {

constexpr int64_t kPieceBytes = int64_t(256) << 20;  // most of a piece's dz
constexpr int64_t kLayBytes = int64_t(1) << 30;      // most of a piece of W laid out anew
constexpr int64_t kNativeRows = 256;                 // most rows of float32 products without planes

// The workspace's layout and the kernels that use it ask the same question.
bool takes_planes(const CeParams& p) { return p.dtype == 0 && p.n > kNativeRows; }

// ------------------------------------------------------------------------------------------ rows
struct Meta {
  int kept;
  float most;    // largest finite |g| of the kept rows (kCeNone)
  float factor;  // of the float32 sums that become gradients
};

constexpr int kScanPer = 4, kScan = 1024 * kScanPer;  // rows of a thread and of a workgroup in a round

struct RowTarget {
  int64_t target;
  bool keep, drop;
};
__device__ __forceinline__ RowTarget row_target(const CeParams& p, int64_t n) {
  if (n >= p.n) return {0, false, false};
  const int64_t t = p.target64 ? ((const int64_t*)p.target)[n] : (int64_t)((const int32_t*)p.target)[n];
  const bool valid = t != p.ignore && t >= 0 && t < p.classes;
  return {t, valid, !valid};
}

// Kept rows and largest finite |g| of each kScan rows, for the launch that lists them with several workgroups.
struct RowCount {
  int kept;
  float most;
};
__device__ __forceinline__ float kept_gradient(const CeParams& p, int64_t n) {
  const float g = fabsf(p.gout[n]);
  return g < THERIA_INF ? g : 0.f;
}
// The sum of `kept` and the largest `most` over a workgroup of 16 waves, in every thread.
__device__ __forceinline__ void block_count(int& kept, float& most, RowCount* red) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    kept += __shfl_xor(kept, o);
    most = fmaxf(most, __shfl_xor(most, o));
  }
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = {kept, most};
  __syncthreads();
  kept = 0;
  for (int w = 0; w < 16; ++w) kept += red[w].kept, most = fmaxf(most, red[w].most);
}
__global__ __launch_bounds__(1024) void ce_count_kernel(CeParams p, bool gradients, RowCount* counts) {
  __shared__ RowCount red[16];
  int kept = 0;
  float most = 0.f;
#pragma unroll
  for (int u = 0; u < kScanPer; ++u) {
    const int64_t n = (int64_t)blockIdx.x * kScan + u * 1024 + threadIdx.x;
    if (row_target(p, n).keep) {
      ++kept;
      if (gradients) most = fmaxf(most, kept_gradient(p, n));
    }
  }
  block_count(kept, most, red);
  if (threadIdx.x == 0) counts[blockIdx.x] = {kept, most};
}

// map: the kept rows in order, then from the end the dropped ones, ignored as n, invalid as -n - 1. target: of the kept.
// One workgroup for all rows, or with `counts` one for every kScan.
__global__ __launch_bounds__(1024) void ce_rows_kernel(CeParams p, bool backward, const RowCount* counts, int* map, int* target, Meta* meta) {
  __shared__ int wave_kept[2][16];
  __shared__ RowCount red[2][16];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const bool gradients = backward && p.reduction == kCeNone;
  int64_t first = 0, end = p.n;
  int kept = 0;  // before this round's rows
  int all_kept = 0;
  float most = 0.f;
  if (counts) {
    const int blocks = gridDim.x;
    float none = 0.f;
    for (int b = threadIdx.x; b < blocks; b += 1024) {
      all_kept += counts[b].kept;
      kept += b < (int)blockIdx.x ? counts[b].kept : 0;
      most = fmaxf(most, counts[b].most);
    }
    block_count(all_kept, most, red[0]);
    block_count(kept, none, red[1]);
    first = (int64_t)blockIdx.x * kScan;
    end = first + kScan < p.n ? first + kScan : p.n;
  }
  int turn = 0;
  for (int64_t base = first; base < end; base += kScan, turn ^= 1) {
    const int64_t n0 = base + threadIdx.x * kScanPer;
    RowTarget t[kScanPer];
    int mine = 0;
#pragma unroll
    for (int u = 0; u < kScanPer; ++u) {
      t[u] = row_target(p, n0 + u);
      mine += t[u].keep;
      if (gradients && !counts && t[u].keep) most = fmaxf(most, kept_gradient(p, n0 + u));
    }
    int upto = mine;  // inclusive sum over the wave's lanes
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int add = __shfl_up(upto, o);
      if (lane >= o) upto += add;
    }
    if (lane == 63) wave_kept[turn][wave] = upto;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < 16; ++w) {
      before += w < wave ? wave_kept[turn][w] : 0;
      all += wave_kept[turn][w];
    }
    int64_t at = kept + before + upto - mine;
#pragma unroll
    for (int u = 0; u < kScanPer; ++u) {
      const int64_t n = n0 + u;
      if (t[u].keep) {
        map[at] = (int)n;
        target[at] = (int)t[u].target;
        ++at;
      } else if (t[u].drop) {
        map[p.n - 1 - (n - at)] = t[u].target == p.ignore ? (int)n : (int)(-n - 1);
      }
    }
    kept += all;
  }
  if (!counts) {
    int none = 0;
    block_count(none, most, red[0]);
    all_kept = kept;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    meta->kept = all_kept;
    meta->most = most;
    if (backward) {
      const float unit = p.dtype == 1 ? 0x1p-14f : 1.f;
      // no kept row: zero, not the zero over zero of an empty mean
      meta->factor = all_kept == 0 ? 0.f : unit * (p.reduction == kCeNone ? most : p.reduction == kCeMean ? p.gout[0] / (float)all_kept : p.gout[0]);
    }
  }
}

// Rows laid out for the products: `width` elements, zeros up to kp, a wave for a row. With map: the kept rows of src.
// SPLIT false: a copy. true (float32): two scaled float16 planes and the exponent of each row's scale at `logits`, and three
// bfloat16 planes at `grads` unless it is null.
struct LayTo {
  char *logits, *grads;
  int* exponent;
  int64_t plane;  // bytes from plane to plane
  int kp;
  MutRows dx;     // with map: the dropped rows of this matrix become zero, NaN where the target is invalid; or absent
};
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void ce_lay_kernel(Rows src, int64_t rows, int width, const int* map, const Meta* meta, LayTo to) {
  const int lane = threadIdx.x % 64;
  const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (i >= rows) return;
  if (map && i >= meta->kept) {
    const int m = map[i];
    if (!to.dx.p) return;
    const T fill = m < 0 ? (T)__builtin_nanf("") : (T)0.f;
    T* row = (T*)to.dx.p + (m < 0 ? -(int64_t)m - 1 : (int64_t)m) * to.dx.sr;
    for (int c = lane; c < width; c += 64) row[c] = fill;
    return;
  }
  const T* row = (const T*)src.p + (map ? (int64_t)map[i] : i) * src.sr;
  RawVec<T, 8> raw;
  int scale = 0;
  if constexpr (SPLIT) {
    float most = 0.f;  // of the finite elements
    for (int c = lane * 8; c < width; c += 512) {
      float v[8];
      raw.load(row + c, width - c);
      raw.get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fabsf(v[e]) < THERIA_INF ? fmaxf(most, fabsf(v[e])) : most;
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) most = fmaxf(most, __shfl_xor(most, o));
    int e = 0;
    if (most > 0.f) frexpf(most, &e), scale = 14 - e;
    if (lane == 0) to.exponent[i] = -scale;
  }
  for (int c = lane * 8; c < to.kp; c += 512) {
    raw.load(row + c, width - c);
    const int64_t at = (i * to.kp + c) * 2;
    if constexpr (!SPLIT) {
      raw.store((T*)to.logits + i * to.kp + c);
    } else {
      float v[8];
      raw.get(v);
      f16x8_t h, m;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = ldexpf(v[e], scale);
        h[e] = (_Float16)x;
        m[e] = fabsf(x) < THERIA_INF ? (_Float16)(x - (float)h[e]) : (_Float16)0.f;
      }
      *reinterpret_cast<f16x8_t*>(to.logits + at) = h;
      *reinterpret_cast<f16x8_t*>(to.logits + to.plane + at) = m;
      if (!to.grads) continue;
      bf16x8_t a, b, d;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        __bf16 x, y, z;
        split3(v[e], x, y, z);
        a[e] = x, b[e] = y, d[e] = z;
      }
      *reinterpret_cast<bf16x8_t*>(to.grads + at) = a;
      *reinterpret_cast<bf16x8_t*>(to.grads + to.plane + at) = b;
      *reinterpret_cast<bf16x8_t*>(to.grads + 2 * to.plane + at) = d;
    }
  }
}

// ------------------------------------------------------------------------------------------ epilogues
// What the logits' two epilogues share. Classes are i of the product, rows j.
// SCALED: products of scaled planes.
template <typename T, bool SCALED>
struct LogitBase {
  const T* bias;      // of the piece's classes, or null
  int64_t v0;         // the piece's first class
  const int* target;  // of the kept rows
  const int *exponent_w, *exponent_x;  // float32 operands: of the scales of the classes' and of the rows' planes

  // Four elements from i of an array of the classes, those past the end as they are in `q`.
  template <typename Q, typename E>
  __device__ __forceinline__ static void load4(Q& q, const E* p, int i, int I) {
    if ((uintptr_t)p % (4 * sizeof(E)) == 0 && i + 4 <= I) {
      q = *reinterpret_cast<const Q*>(p + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < I) q[e] = p[i + e];
    }
  }

  // The accumulators' first values: the bias (loaded while the first stage's copies are on their way), or zeros. Scaled
  // products get their bias at the end.
  template <class S>
  __device__ __forceinline__ void start(f32x16_t (&z)[S::FI][S::FJ], const GemmTile& t) const {
    typedef T quad_t __attribute__((ext_vector_type(4)));
    if (SCALED || !bias) return gemm_zero<S>(z);
    const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        quad_t b = {(T)0.f, (T)0.f, (T)0.f, (T)0.f};
        load4(b, bias, t.i0 + 32 * fi + 8 * q + 4 * g, t.I);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int fj = 0; fj < S::FJ; ++fj) z[fi][fj][4 * q + e] = (float)b[e];
      }
  }

  // The logits: scales taken back and bias added where start() could not; classes past the piece's end become -inf.
  template <class S>
  __device__ __forceinline__ void finish(f32x16_t (&z)[S::FI][S::FJ], const GemmTile& t) const {
    const int li = threadIdx.x & 31, g = (threadIdx.x >> 5) & 1;
    if constexpr (SCALED) {
      int ex[S::FJ];
#pragma unroll
      for (int fj = 0; fj < S::FJ; ++fj) ex[fj] = t.j0 + 32 * fj + li < t.J ? exponent_x[t.j0 + 32 * fj + li] : 0;
#pragma unroll
      for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = t.i0 + 32 * fi + 8 * q + 4 * g;
          i32x4_t ew = {0, 0, 0, 0};
          f32x4_t b = {0.f, 0.f, 0.f, 0.f};
          load4(ew, exponent_w, i, t.I);
          if (bias) load4(b, bias, i, t.I);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int fj = 0; fj < S::FJ; ++fj) z[fi][fj][4 * q + e] = ldexpf(z[fi][fj][4 * q + e], ew[e] + ex[fj]) + b[e];
          __builtin_amdgcn_sched_barrier(0);  // the loads of a whole tile do not fit the registers
        }
    }
    if (t.i0 + 32 * S::FI <= t.I) return;
    const int room = t.I - t.i0 - 4 * g;
#pragma unroll
    for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int fj = 0; fj < S::FJ; ++fj)
          if (32 * fi + 8 * (r >> 2) + (r & 3) >= room) z[fi][fj][r] = -THERIA_INF;
  }
};

// What a softmax's sum is kept as: the largest logit, and the sum of exp(logit - largest) without the largest one's 1 (-1 where
// there is nothing but -inf). So the loss of a row that is well predicted, log1p of it, keeps its digits: next to the 1 they
// would be rounded off with every term.
__device__ __forceinline__ float2 joined(float2 a, float2 b) {
  const bool swap = b.x > a.x;
  const float2 hi = swap ? b : a, lo = swap ? a : b;
  const float off = hi.x == -THERIA_INF ? 0.f : hi.x;
  return float2{hi.x, hi.y + (1.f + lo.y) * fast_exp2((lo.x - off) * kLog2e)};
}

// Forward: of each row (column j of the tile) that pair over the tile's classes, and the target's logit where it lies in the
// tile.
template <typename T, bool SCALED>
struct LogitStats : LogitBase<T, SCALED> {
  float* at_target;   // one of each kept row
  float2* part;       // [tile][n]
  int64_t n;
  int tile0;          // the piece's first tile

  template <class S>
  __device__ __forceinline__ void run(f32x16_t (&z)[S::FI][S::FJ], const GemmTile& t, char*) const {
    __shared__ float2 red[S::WI][S::TJ];
    const int lane = threadIdx.x & 63, li = lane & 31, g = lane >> 5;
    this->template finish<S>(z, t);
#pragma unroll
    for (int fj = 0; fj < S::FJ; ++fj) {
      const int j = t.j0 + 32 * fj + li;
      if (j < t.J) {
        const int64_t want = (int64_t)this->target[j] - this->v0 - t.i0;
        const int w = (int)want - 4 * g;  // the wanted one's place among this half's rows, if it is there
        if (want >= 0 && want < 32 * S::FI && (want >> 2 & 1) == g) {
          float at = 0.f;
#pragma unroll
          for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
            for (int r = 0; r < 16; ++r) at = w == 32 * fi + 8 * (r >> 2) + (r & 3) ? z[fi][fj][r] : at;
          at_target[j] = at;
        }
      }
      float top = -THERIA_INF;
#pragma unroll
      for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, z[fi][fj][r]);
      top = pair_max(top);
      const float off = top == -THERIA_INF ? 0.f : top;  // nothing but -inf: a sum of zeros
      float part4[4] = {0.f, 0.f, 0.f, 0.f};
      int tops = 0;
#pragma unroll
      for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool it = z[fi][fj][r] == top;
          part4[r & 3] += it ? 0.f : fast_exp2((z[fi][fj][r] - off) * kLog2e);
          tops += it;
        }
      const float others = pair_sum((part4[0] + part4[1]) + (part4[2] + part4[3])), more = pair_sum((float)tops) - 1.f;
      const float rest = top == THERIA_INF ? __builtin_nanf("") : others + (top == -THERIA_INF ? -1.f : more);
      if (g == 0) red[t.wave_i][t.wave_j * (S::TJ / S::WJ) + 32 * fj + li] = float2{top, rest};
    }
    __syncthreads();
    for (int c = threadIdx.x; c < S::TJ; c += S::NW * 64) {
      const int j = t.tile_j * S::TJ + c;
      if (j >= t.J) continue;
      float2 all = red[0][c];
#pragma unroll
      for (int w = 1; w < S::WI; ++w) all = joined(all, red[w][c]);
      part[(int64_t)(tile0 + t.tile_i) * n + j] = all;
    }
  }
};

// Backward: dz of the tile in the operands' type, or of scaled products in three bfloat16 planes; rows j of ld elements.
template <typename T, bool SCALED>
struct LogitGrad : LogitBase<T, SCALED> {
  static constexpr int PLANES = SCALED ? 3 : 1;
  const int* map;
  const float* stats;  // [2][n]: largest logit, sum
  int64_t n;
  const float* gout;   // of each row (kCeNone), or null: 1
  const Meta* meta;
  float* rest;         // of each kept row: what the rounding of its target's entry left (16-bit inputs)
  char* dz;
  int ld;              // the piece's classes rounded up to 64: the rest are zeros
  int64_t plane;

  template <class S>
  __device__ __forceinline__ void run(f32x16_t (&z)[S::FI][S::FJ], const GemmTile& t, char* lds) const {
    using H = typename std::conditional<PLANES == 1, typename S::H, __bf16>::type;
    const int lane = threadIdx.x & 63, li = lane & 31, g = lane >> 5;
    this->template finish<S>(z, t);
#pragma unroll
    for (int fj = 0; fj < S::FJ; ++fj) {
      const int j = t.j0 + 32 * fj + li;
      const bool in = j < t.J;
      const float top = in ? stats[j] : 0.f, inv = in ? 1.0f / stats[n + j] : 0.f;
      float unit = __is_same(T, _Float16) ? 0x1p14f : 1.f;
      if (in && gout) {
        const float go = gout[map[j]], most = meta->most;
        // a gradient that is not finite keeps its own value: it is not in `most`
        unit *= !(fabsf(go) < THERIA_INF) ? go : most > 0.f ? go / most : 0.f;
      }
      // softmax times the unit; classes past the piece's end have z = -inf, so zeros
#pragma unroll
      for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
        for (int r = 0; r < 16; ++r) z[fi][fj][r] = fast_exp2((z[fi][fj][r] - top) * kLog2e) * inv;
      const int64_t want = in ? (int64_t)this->target[j] - this->v0 - t.i0 : -1;
      if (want >= 0 && want < 32 * S::FI && (want >> 2 & 1) == g) {
        const int w = (int)want - 4 * g;
        float at = 0.f;
#pragma unroll
        for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool it = w == 32 * fi + 8 * (r >> 2) + (r & 3);
            z[fi][fj][r] -= it ? 1.f : 0.f;
            at = it ? z[fi][fj][r] * unit : at;
          }
        if constexpr (sizeof(T) == 2) rest[j] = at - (float)(H)at;
      }
#pragma unroll
      for (int fi = 0; fi < S::FI; ++fi) z[fi][fj] *= unit;
    }
    using Stage = GemmStage<S, (int)sizeof(H)>;
    // the share holds every row of 16-bit values, or one block's rows of float32 ones
    constexpr int kBlocks = sizeof(H) == 2 ? S::FJ : 1;
    // one plane after another through the same LDS
#pragma unroll 1
    for (int k = 0; k < PLANES; ++k) {
#pragma unroll
      for (int f0 = 0; f0 < S::FJ; f0 += kBlocks) {
#pragma unroll
        for (int fj = f0; fj < f0 + kBlocks; ++fj)
#pragma unroll
          for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              H out[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float v = z[fi][fj][4 * q + e];
                if constexpr (PLANES == 1) {
                  out[e] = (H)v;
                } else {
                  __bf16 h, m, l;
                  asm volatile("" : "+v"(v));  // split anew for each plane: the three of a whole tile do not fit the registers
                  split3(v, h, m, l);
                  out[e] = k == 0 ? h : k == 1 ? m : l;
                }
              }
              Stage::put(lds, 32 * (fj - f0) + li, fi, q, g, out);
            }
        const int j0 = t.j0 + 32 * f0;
        Stage::each(lds, 32 * kBlocks, [&](int r, int i, const i32x4_t& v) {
          if (j0 + r < t.J && t.i0 + i < ld)
            *reinterpret_cast<i32x4_t*>(dz + k * plane + ((int64_t)(j0 + r) * ld + t.i0 + i) * sizeof(H)) = v;
        });
      }
    }
  }
};

// float32 sums, one set for each part of k: [split][J][ld], added to what is there or written.
struct SumTile {
  float* sums;
  int64_t rows;  // of a split
  int ld;        // a multiple of 8
  bool add;

  template <class S>
  __device__ __forceinline__ void start(f32x16_t (&z)[S::FI][S::FJ], const GemmTile&) const {
    gemm_zero<S>(z);
  }
  template <class S>
  __device__ __forceinline__ void run(f32x16_t (&z)[S::FI][S::FJ], const GemmTile& t, char* lds) const {
    const int lane = threadIdx.x & 63, li = lane & 31, g = lane >> 5;
    using Stage = GemmStage<S, 4>;
#pragma unroll
    for (int fj = 0; fj < S::FJ; ++fj) {
#pragma unroll
      for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4_t v = {z[fi][fj][4 * q], z[fi][fj][4 * q + 1], z[fi][fj][4 * q + 2], z[fi][fj][4 * q + 3]};
          Stage::put(lds, li, fi, q, g, &v);
        }
      const int j0 = t.j0 + 32 * fj;
      Stage::each(lds, 32, [&](int r, int i, const i32x4_t& c) {
        if (j0 + r >= t.J || t.i0 + i >= ld) return;
        f32x4_t* to = reinterpret_cast<f32x4_t*>(sums + (t.split * rows + j0 + r) * ld + t.i0 + i);
        f32x4_t v = __builtin_bit_cast(f32x4_t, c);
        if (add) v += *to;
        *to = v;
      });
    }
  }
};

// The tile times the factor, in the output's type. Rows j go to map[j] where there is a map, and `rest` is as in
// ce_join_rows_kernel.
template <typename T>
struct OutTile {
  T* out;
  int64_t sr;
  const Meta* meta;
  const int* map;
  const float* rest;
  const int* target;
  Rows w;

  template <class S>
  __device__ __forceinline__ void start(f32x16_t (&z)[S::FI][S::FJ], const GemmTile&) const {
    gemm_zero<S>(z);
  }
  template <class S>
  __device__ __forceinline__ void run(f32x16_t (&z)[S::FI][S::FJ], const GemmTile& t, char* lds) const {
    const int lane = threadIdx.x & 63, li = lane & 31, g = lane >> 5;
    const float f = meta->factor;
    if (rest) {
#pragma unroll
      for (int fj = 0; fj < S::FJ; ++fj) {
        const int j = t.j0 + 32 * fj + li;
        const float left = j < t.J ? rest[j] : 0.f;
        if (left == 0.f) continue;
        const T* row = (const T*)w.p + target[j] * w.sr;
#pragma unroll
        for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int i = t.i0 + 32 * fi + 8 * q + 4 * g;
            float f4[4];
            load_quad(f4, row + i, t.I - i);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[fi][fj][4 * q + e] += left * f4[e];
          }
      }
    }
    using Stage = GemmStage<S, (int)sizeof(T)>;
    // the share holds every row of 16-bit results, or one block's rows of float32 ones
    constexpr int kBlocks = sizeof(T) == 2 ? S::FJ : 1, kPer = 16 / (int)sizeof(T);
#pragma unroll
    for (int f0 = 0; f0 < S::FJ; f0 += kBlocks) {
#pragma unroll
      for (int fj = f0; fj < f0 + kBlocks; ++fj)
#pragma unroll
        for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            T v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(z[fi][fj][4 * q + e] * f);
            Stage::put(lds, 32 * (fj - f0) + li, fi, q, g, v);
          }
      const int j0 = t.j0 + 32 * f0;
      Stage::each(lds, 32 * kBlocks, [&](int r, int i, const i32x4_t& c) {
        if (j0 + r >= t.J || t.i0 + i >= t.I) return;
        T* to = out + (map ? (int64_t)map[j0 + r] : (int64_t)(j0 + r)) * sr + t.i0 + i;
        RawVec<T, kPer> v;
        __builtin_memcpy(v.v, &c, 16);
        v.store(to, t.I - t.i0 - i);
      });
    }
  }
};

// ------------------------------------------------------------------------------------------ joins
// R rows a workgroup, each one's tiles spread over 256 / R threads. Dropped rows: zero, or NaN where the target is invalid.
template <int R>
__global__ __launch_bounds__(256) void ce_join_kernel(CeParams p, int tiles, const float2* part, const float* at_target, const int* map,
                                                      const Meta* meta, float* row_loss) {
  constexpr int S = 256 / R;
  __shared__ float2 red[S][R + 1];
  const int r = threadIdx.x % R, s = threadIdx.x / R;
  const int64_t j = (int64_t)blockIdx.x * R + r;
  const int kept = meta->kept;
  float2 all{-THERIA_INF, -1.f};
  if (j < kept) {
    float top = -THERIA_INF, rest = 0.f;
    bool seen = false;
#pragma unroll 4
    for (int k = s; k < tiles; k += S) top = fmaxf(top, part[(int64_t)k * p.n + j].x);
    const float off = top == -THERIA_INF ? 0.f : top;
#pragma unroll 4
    for (int k = s; k < tiles; k += S) {
      const float2 v = part[(int64_t)k * p.n + j];
      const bool it = v.x == top && !seen;
      rest += it ? v.y : (1.f + v.y) * fast_exp2((v.x - off) * kLog2e);
      seen = seen || it;
    }
    all = float2{top, seen ? rest : -1.f};
  }
  red[s][r] = all;
  // halves of the slices joined in turn, in an order that does not depend on the run
#pragma unroll
  for (int o = S / 2; o > 0; o /= 2) {
    __syncthreads();
    if (s < o) red[s][r] = all = joined(red[s][r], red[s + o][r]);
  }
  if (s != 0 || j >= p.n) return;
  if (j >= kept) {
    if (row_loss) {
      const int row = map[j];
      row_loss[row < 0 ? -row - 1 : row] = row < 0 ? __builtin_nanf("") : 0.f;
    }
    return;
  }
  p.stats[j] = all.x;
  p.stats[p.n + j] = 1.f + all.y;
  if (row_loss) row_loss[map[j]] = log1pf(all.y) - (at_target[j] - all.x);
}

// The mean or sum of the rows' losses, by one workgroup in a fixed order.
__global__ __launch_bounds__(1024) void ce_total_kernel(CeParams p, const float* row_loss, const Meta* meta) {
  __shared__ float red[16];
  float s[1] = {0.f};
#pragma unroll 8
  for (int64_t n = threadIdx.x; n < p.n; n += 1024) s[0] += row_loss[n];
  team_sum<1024, 1>(s, red);
  if (threadIdx.x == 0) p.loss[0] = p.reduction == kCeMean ? s[0] / (float)meta->kept : s[0];
}

// out[row] = the sum over the splits of sums[split][i], times the factor. map: row map[i] for each kept row; without: row i.
// rest: what the rounding of the kept rows' target entries left, to be added with the target's row of w.
template <typename T>
__global__ __launch_bounds__(256) void ce_join_rows_kernel(const float* sums, int splits, int64_t rows, int ld, int width, const int* map,
                                                           const Meta* meta, T* out, int64_t sr, const float* rest,
                                                           const int* target, Rows w) {
  const int c = blockIdx.y * 512 + threadIdx.x % 64 * 8;
  const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (i >= (map ? (int64_t)meta->kept : rows) || c >= width) return;
  const float f = meta->factor, left = rest ? rest[i] : 0.f;
  f32x4_t a = {0.f, 0.f, 0.f, 0.f}, b = a;  // ld is a multiple of 8
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const f32x4_t* from = reinterpret_cast<const f32x4_t*>(sums + (s * rows + i) * ld + c);
    a += from[0], b += from[1];
  }
  float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  RawVec<T, 8> o;
  if (left != 0.f) {
    float w8[8];
    o.load((const T*)w.p + target[i] * w.sr + c, width - c);
    o.get(w8);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += left * w8[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= f;
  o.set(v);
  o.store(out + (map ? (int64_t)map[i] : i) * sr + c, width - c);
}

// Column sums of a piece's dz: a thread adds eight columns over its share of the kept rows.
template <typename H, int PLANES>
__global__ __launch_bounds__(256) void ce_bias_kernel(const char* dz, int ld, int64_t plane, const Meta* meta, float* part) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * 8, kept = meta->kept;
  if (c >= ld) return;
  const int per = (kept + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = min(kept, r0 + per);
  float s[8] = {};
#pragma unroll 4
  for (int r = r0; r < r1; ++r) {
#pragma unroll
    for (int k = PLANES - 1; k >= 0; --k) {
      RawVec<H, 8> v;
      v.load((const H*)(dz + k * plane) + (int64_t)r * ld + c);
      float f[8];
      v.get(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += f[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[(int64_t)blockIdx.y * ld + c + e] = s[e];
}

// ------------------------------------------------------------------------------------------ layout of a call
int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// Product tiles, and parts of k for products with few of them. A workgroup of 256 x 256 holds a CU by itself and reads half
// the operand bytes of 128 x 128 for each product; two of those share a CU, and one's epilogue runs beside the other's
// products. Up to 64 rows, and for float32 operands as they are: 128 x 64.
enum class Tile { kFew, kMid, kLarge };
int tile_i(Tile t) { return t == Tile::kLarge ? 256 : 128; }
int tile_j(Tile t) { return t == Tile::kLarge ? 256 : t == Tile::kMid ? 128 : 64; }
int64_t tiles_of(Tile t, int64_t I, int64_t J) { return up(I, tile_i(t)) / tile_i(t) * (up(J, tile_j(t)) / tile_j(t)); }

struct Pick {
  Tile tile;
  int splits;
};

// The pick with the least time for I x J results of K k by a model of the measured kernels, in us: a step of 64 k takes 1.65
// in a large workgroup, 1.1 in two small ones on a CU and 0.9 in one alone, an epilogue 6 and 3, and a part's float32 sums
// are written and read at 4.5 TB/s. (Before, large tiles wherever they alone filled the GPU, dx of (4096, 32000, 1024)
// bfloat16 took 461 us, and takes 264 us in four parts; forward of (2000, 10000, 512) takes 48 us in small tiles and 54 us in large ones, of (4096,
// 32000, 512) 181 and 172.) parts: most parts of k. Parts have at least 8 steps.
Pick pick(int64_t I, int64_t J, int64_t K, int segments, bool few, bool large, bool parts) {
  const int64_t cus = device_cu_count();
  const bool narrow = few && (J <= 64 || !large);
  if (I == 0 || J == 0) return {narrow ? Tile::kFew : Tile::kMid, 1};
  const int64_t most = !parts || K < 1024 ? 1 : K / 512 < 256 ? K / 512 : 256;
  if (narrow || !large) {
    // bound by reading one operand, or by few products: parts until there are two workgroups for each CU
    const Tile t = narrow ? Tile::kFew : Tile::kMid;
    const int64_t tiles = tiles_of(t, I, J), want = tiles >= cus ? 1 : (2 * cus + tiles - 1) / tiles;
    return {t, (int)(want < most ? want : most)};
  }
  Pick best{Tile::kLarge, 1};
  double least = 1e30;
  for (int s = 1; s <= most; s += s < 4 ? 1 : s < 16 ? s / 4 : s / 2) {
    const double steps = (double)((K + 64 * s - 1) / (64 * s)) * segments, sums = parts && s > 1 ? s * 8.0 * I * J / 4.5e6 : 0;
    const int64_t nl = tiles_of(Tile::kLarge, I, J) * s, nm = tiles_of(Tile::kMid, I, J) * s;
    const double tl = (double)((nl + cus - 1) / cus) * (1.65 * steps + 6) + sums;
    const double tm = nm <= cus ? 0.9 * steps + 3 + sums : (double)((nm + 2 * cus - 1) / (2 * cus)) * (1.1 * steps + 3) + sums;
    if (tl < least) least = tl, best = {Tile::kLarge, s};
    if (tm < least) least = tm, best = {Tile::kMid, s};
  }
  return best;
}

// Where everything lies in the workspace.
struct Layout {
  bool planes;      // float32: operands in planes of 16-bit terms
  bool lay_w;       // W is laid out anew, a piece at a time
  int kp;           // width rounded up to 64
  int64_t piece;    // classes of a piece
  int ldz;          // of a piece's dz
  Pick f, x, w;     // of the logits, dx, dW
  bool direct_x;    // dx leaves its product finished: one piece, one part
  int ldx;          // of the float32 sums
  int tiles;        // of classes, over all pieces
  int bias_parts;
  int64_t map, target, counts, meta, xs, xs_grad, ws_w, ws_w_grad, ex_x, ex_w, at_target, part, row_loss, rest, dz, sum_x, sum_w, bias_part, bytes;
};

Layout layout_of(const CeParams& p, bool backward) {
  Layout l{};
  l.planes = takes_planes(p);
  const bool f32 = p.dtype == 0, native = f32 && !l.planes;
  // bytes of an element of the logits' operands and of the gradients', all planes
  const int es = f32 ? 4 : 2, bl = es, bg = l.planes ? 6 : es, per = 16 / es;
  l.kp = (int)up(p.width, 64);
  // the copies take 16-byte pieces and 32-bit offsets inside a tile
  l.lay_w = l.planes || p.width % per || p.w.sr % per || (uintptr_t)p.w.p % 16 || p.w.sr > (1 << 20);
  l.piece = up(p.classes, 64);
  auto limit = [&](int64_t bytes, int64_t row_bytes) {  // bytes of one class
    const int64_t most = bytes / row_bytes / 256 * 256;
    if (l.piece > most) l.piece = most < 256 ? 256 : most;
  };
  if (l.lay_w) limit(kLayBytes, (bl + (l.planes && backward ? bg : 0)) * (int64_t)l.kp);
  if (backward && p.n > 0) limit(kPieceBytes, bg * p.n);
  l.ldz = (int)l.piece;
  const int segments_l = l.planes ? 3 : 1, segments_g = l.planes ? 6 : 1;
  l.f = pick(l.piece, p.n, p.width, segments_l, true, !native, false);
  l.x = pick(p.width, p.n, l.piece, segments_g, true, !native, true);
  l.w = pick(p.width, l.piece, p.n, segments_g, false, !native, true);
  l.direct_x = l.piece >= p.classes && l.x.splits == 1;
  l.ldx = (int)up(p.width, 8);
  l.bias_parts = (int)(p.n < 64 ? 1 : p.n / 64 < 64 ? p.n / 64 : 64);
  for (int64_t v = 0; v < p.classes; v += l.piece)
    l.tiles += (int)(up(p.classes - v < l.piece ? p.classes - v : l.piece, tile_i(l.f.tile)) / tile_i(l.f.tile));
  auto take = [&](int64_t bytes) {
    const int64_t at = l.bytes;
    l.bytes += up(bytes, 256);
    return at;
  };
  l.meta = take(sizeof(Meta));
  l.map = take(4 * p.n);
  l.target = take(4 * p.n);
  l.counts = take(sizeof(RowCount) * (p.n / kScan + 1));
  l.xs = take(bl * p.n * l.kp);
  if (l.lay_w) l.ws_w = take(bl * l.piece * l.kp);
  if (l.planes) {
    l.ex_x = take(4 * p.n);
    l.ex_w = take(4 * l.piece);
    if (backward) l.xs_grad = take(bg * p.n * l.kp), l.ws_w_grad = take(bg * l.piece * l.kp);
  }
  if (!backward) {
    l.at_target = take(4 * p.n);
    l.part = take(8 * l.tiles * p.n);
    l.row_loss = take(4 * p.n);
  } else {
    l.rest = take(4 * p.n);
    l.dz = take(bg * p.n * l.ldz);
    if (p.dx.p && !l.direct_x) l.sum_x = take(4 * l.x.splits * p.n * l.ldx);
    if (p.dw.p && l.w.splits > 1) l.sum_w = take(4 * l.w.splits * l.piece * l.ldx);
    if (p.db) l.bias_part = take(4 * (int64_t)l.bias_parts * l.ldz);
  }
  return l;
}

template <typename H, bool A, bool B, class Epi>
hipError_t gemm(Tile t, const GemmParams& g, const Epi& e, hipStream_t st) {
  switch (t) {
    case Tile::kLarge:
      if constexpr (sizeof(H) == 2) return launch_gemm<GemmShape<H, 256, 256, 2, 4, A, B>>(g, e, st);
      break;
    case Tile::kMid: return launch_gemm<GemmShape<H, 128, 128, 2, 2, A, B>>(g, e, st);
    case Tile::kFew:
      if constexpr (!B) return launch_gemm<GemmShape<H, 128, 64, 4, 1, A, B>>(g, e, st);
  }
  return hipErrorInvalidValue;
}

#define THERIA_TRY(call)                \
  do {                                  \
    const hipError_t e_ = (call);       \
    if (e_ != hipSuccess) return e_;    \
  } while (0)

// SPLIT: float32 operands in planes.
template <typename T, bool SPLIT>
struct Call {
  using L = typename std::conditional<SPLIT, _Float16, T>::type;  // operands of the logits
  using H = typename std::conditional<SPLIT, __bf16, T>::type;    // operands of the gradients
  const CeParams& p;
  const Layout l;
  hipStream_t st;
  char* ws;
  int* map;
  int* target;
  Meta* meta;

  Call(const CeParams& p_, bool backward, hipStream_t st_)
      : p(p_), l(layout_of(p_, backward)), st(st_), ws((char*)p_.ws), map((int*)(ws + l.map)), target((int*)(ws + l.target)), meta((Meta*)(ws + l.meta)) {}

  static constexpr int ES = sizeof(H);
  static_assert(sizeof(L) == ES);
  int64_t plane_x() const { return ES * p.n * l.kp; }
  int64_t plane_w() const { return ES * l.piece * l.kp; }
  int64_t plane_z() const { return ES * p.n * l.ldz; }
  static constexpr int kLogitSegments = SPLIT ? 3 : 1, kGradSegments = SPLIT ? 6 : 1;
  // Operands along k belong to the logits, but for dz; those across k to the gradients.
  GemmOperand x_operand(bool across) const {
    return {ws + (across && SPLIT ? l.xs_grad : l.xs), ES * (int64_t)l.kp, plane_x(), across ? l.kp : (int)p.n};
  }
  GemmOperand z_operand(bool across) const { return {ws + l.dz, ES * (int64_t)l.ldz, plane_z(), across ? l.ldz : (int)p.n}; }
  // classes [v, v + have)
  GemmOperand w_operand(bool across, int64_t v, int have) const {
    if (l.lay_w) return {ws + (across && SPLIT ? l.ws_w_grad : l.ws_w), ES * (int64_t)l.kp, plane_w(), across ? l.kp : have};
    return {(const char*)p.w.p + v * p.w.sr * ES, ES * p.w.sr, 0, across ? p.width : have};
  }
  const float* rest() const { return sizeof(T) == 4 ? nullptr : (const float*)(ws + l.rest); }
  LogitBase<T, SPLIT> base(int64_t v) const {
    return {p.bias ? (const T*)p.bias + v : nullptr, v, target, (const int*)(ws + l.ex_w), (const int*)(ws + l.ex_x)};
  }

  hipError_t rows(bool backward) {
    // many rows: counted first, so that several workgroups can list them (100000: 87 -> 12 us)
    if (p.n > 4 * kScan) {
      const unsigned blocks = (unsigned)((p.n + kScan - 1) / kScan);
      RowCount* counts = (RowCount*)(ws + l.counts);
      ce_count_kernel<<<blocks, 1024, 0, st>>>(p, backward && p.reduction == kCeNone, counts);
      ce_rows_kernel<<<blocks, 1024, 0, st>>>(p, backward, counts, map, target, meta);
    } else {
      ce_rows_kernel<<<1, 1024, 0, st>>>(p, backward, nullptr, map, target, meta);
    }
    THERIA_TRY(hipGetLastError());
    if (p.n == 0) return hipSuccess;
    ce_lay_kernel<T, SPLIT><<<dim3((unsigned)((p.n + 3) / 4)), 256, 0, st>>>(p.x, p.n, p.width, map, meta, LayTo{ws + l.xs, backward && SPLIT ? ws + l.xs_grad : nullptr, (int*)(ws + l.ex_x), plane_x(), l.kp, backward ? p.dx : MutRows{}});
    return hipGetLastError();
  }
  hipError_t lay_piece(bool backward, int64_t v, int have) {
    if (!l.lay_w) return hipSuccess;
    const Rows src{(const T*)p.w.p + v * p.w.sr, p.w.sr};
    ce_lay_kernel<T, SPLIT><<<dim3((unsigned)((have + 3) / 4)), 256, 0, st>>>(src, have, p.width, nullptr, meta, LayTo{ws + l.ws_w, backward && SPLIT ? ws + l.ws_w_grad : nullptr, (int*)(ws + l.ex_w), plane_w(), l.kp, MutRows{}});
    return hipGetLastError();
  }

  hipError_t forward() {
    THERIA_TRY(rows(false));
    int tile0 = 0;
    for (int64_t v = 0; v < p.classes && p.n > 0; v += l.piece) {
      const int have = (int)(p.classes - v < l.piece ? p.classes - v : l.piece);
      THERIA_TRY(lay_piece(false, v, have));
      const GemmParams g{w_operand(false, v, have), x_operand(false), have, (int)p.n, p.width, 1, kLogitSegments, &meta->kept, true, false};
      const LogitStats<T, SPLIT> e{base(v), (float*)(ws + l.at_target), (float2*)(ws + l.part), p.n, tile0};
      THERIA_TRY((gemm<L, false, false>(l.f.tile, g, e, st)));
      tile0 += (int)(up(have, tile_i(l.f.tile)) / tile_i(l.f.tile));
    }
    float* row_loss = p.reduction == kCeNone ? p.loss : (float*)(ws + l.row_loss);
    // few rows: a workgroup for each, so that the tiles' partial sums are read by more threads
    if (p.n > 0) {
      const float2* part = (const float2*)(ws + l.part);
      const float* at = (const float*)(ws + l.at_target);
      if (p.n <= 1024)
        ce_join_kernel<1><<<dim3((unsigned)p.n), 256, 0, st>>>(p, l.tiles, part, at, map, meta, row_loss);
      else
        ce_join_kernel<8><<<dim3((unsigned)((p.n + 7) / 8)), 256, 0, st>>>(p, l.tiles, part, at, map, meta, row_loss);
    }
    THERIA_TRY(hipGetLastError());
    if (p.reduction != kCeNone) ce_total_kernel<<<1, 1024, 0, st>>>(p, row_loss, meta);
    return hipGetLastError();
  }

  hipError_t backward() {
    constexpr int PLANES = SPLIT ? 3 : 1;
    THERIA_TRY(rows(true));
    for (int64_t v = 0; v < p.classes; v += l.piece) {
      const int have = (int)(p.classes - v < l.piece ? p.classes - v : l.piece);
      THERIA_TRY(lay_piece(true, v, have));
      {
        const GemmParams g{w_operand(false, v, have), x_operand(false), have, (int)p.n, p.width, 1, kLogitSegments, &meta->kept, true, false};
        const LogitGrad<T, SPLIT> e{base(v), map, p.stats, p.n, p.reduction == kCeNone ? p.gout : nullptr, meta, (float*)(ws + l.rest), ws + l.dz, l.ldz, plane_z()};
        THERIA_TRY((gemm<L, false, false>(l.f.tile, g, e, st)));
      }
      if (p.dx.p) {
        const GemmParams g{w_operand(true, v, have), z_operand(false), p.width, (int)p.n, have, l.x.splits, kGradSegments, &meta->kept, true, false};
        if (l.direct_x) {
          THERIA_TRY((gemm<H, true, false>(l.x.tile, g, OutTile<T>{(T*)p.dx.p, p.dx.sr, meta, map, rest(), target, p.w}, st)));
        } else {
          const SumTile e{(float*)(ws + l.sum_x), p.n, l.ldx, v > 0};
          THERIA_TRY((gemm<H, true, false>(l.x.tile, g, e, st)));
        }
      }
      if (p.dw.p) {
        T* out = (T*)p.dw.p + v * p.dw.sr;
        const GemmParams g{x_operand(true), z_operand(true), p.width, have, (int)p.n, l.w.splits, kGradSegments, &meta->kept, false, true};
        if (l.w.splits == 1) {
          THERIA_TRY((gemm<H, true, true>(l.w.tile, g, OutTile<T>{out, p.dw.sr, meta, nullptr, nullptr, nullptr, Rows{}}, st)));
        } else {
          float* sums = (float*)(ws + l.sum_w);
          THERIA_TRY((gemm<H, true, true>(l.w.tile, g, SumTile{sums, l.piece, l.ldx, false}, st)));
          ce_join_rows_kernel<T><<<dim3((unsigned)((have + 3) / 4), (p.width + 511) / 512), 256, 0, st>>>(sums, l.w.splits, l.piece, l.ldx, p.width, nullptr, meta, out, p.dw.sr, nullptr, nullptr, Rows{});
          THERIA_TRY(hipGetLastError());
        }
      }
      if (p.db) {
        float* part = (float*)(ws + l.bias_part);
        ce_bias_kernel<H, PLANES><<<dim3((unsigned)((l.ldz + 2047) / 2048), (unsigned)l.bias_parts), 256, 0, st>>>(ws + l.dz, l.ldz, plane_z(), meta, part);
        THERIA_TRY(hipGetLastError());
        column_sum_kernel<T><<<dim3((unsigned)((l.ldz + 63) / 64)), 1024, 0, st>>>(part, l.bias_parts, l.ldz, have, (T*)p.db + v, nullptr, &meta->factor);
        THERIA_TRY(hipGetLastError());
      }
    }
    if (p.dx.p && p.n > 0 && !l.direct_x) {
      ce_join_rows_kernel<T><<<dim3((unsigned)((p.n + 3) / 4), (p.width + 511) / 512), 256, 0, st>>>((const float*)(ws + l.sum_x), l.x.splits, p.n, l.ldx, p.width, map, meta, (T*)p.dx.p, p.dx.sr, rest(), target, p.w);
      THERIA_TRY(hipGetLastError());
    }
    return hipSuccess;
  }
};

template <typename T, bool SPLIT>
hipError_t run(const CeParams& p, bool backward, hipStream_t st) {
  Call<T, SPLIT> c(p, backward, st);
  return backward ? c.backward() : c.forward();
}

hipError_t by_type(const CeParams& p, bool backward, hipStream_t st) {
  if (p.dtype == 0) return takes_planes(p) ? run<float, true>(p, backward, st) : run<float, false>(p, backward, st);
  if (p.dtype == 1) return run<_Float16, false>(p, backward, st);
  return run<__bf16, false>(p, backward, st);
}

}  // namespace

int64_t ce_ws_bytes(const CeParams& p, bool backward) { return ce_head_takes(p) ? ce_head_ws_bytes(p, backward) : layout_of(p, backward).bytes; }
hipError_t launch_ce_fwd(const CeParams& p, hipStream_t st) { return ce_head_takes(p) ? launch_ce_head(p, false, st) : by_type(p, false, st); }
hipError_t launch_ce_bwd(const CeParams& p, hipStream_t st) { return ce_head_takes(p) ? launch_ce_head(p, true, st) : by_type(p, true, st); }

}  // namespace theria
