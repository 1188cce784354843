// Matrix products for the linear cross entropy: C[i][j] = sum_k A[i][k] B[j][k] on MFMA (gfx950).
//
// Either operand lies in memory "along k" (rows i, k contiguous) or "across k" (rows k, i contiguous); the second kind is
// transposed on its way from LDS to registers (ds_read_b64_tr_b16), so that no transposed copy is ever made. A workgroup
// owns a tile of TI x TJ results, walks k in steps of 128 bytes (64 elements of 16 bits) and keeps two stages of both
// operands in LDS, filled by LDS DMA: the next step's copies run while this step's products do.
//
// float32 operands either go to v_mfma_f32_32x32x2_f32 as they are (H = float; a sixteenth of the 16-bit rate, but nothing
// is laid out anew), or come as planes of 16-bit terms. Two each, x = h + m: three passes over k (m h, h m, h h). Three
// each, x = h + m + l (split3): six passes (m m, l h, h l, m h, h m, h h), whose dropped terms are at most 2^-24 of the
// product. The smallest come first.
//
// The accumulators have i along registers and j along lanes: lane l holds column j = l % 32 of a 32 x 32 block and four
// consecutive i in each group of four registers, so sums over i stay inside a lane and i is written in pieces of four.
#pragma once

#include "sdpa_lds.hpp"

namespace theria {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

// Operand fragments of 32 x 32 results: 16 bytes a lane, 16 k (float32: 8 k, as four instructions of two).
template <typename H>
struct GemmMma {
  using frag_t = typename Mfma<H>::frag_t;
  __device__ __forceinline__ static f32x16_t mma(frag_t a, frag_t b, f32x16_t c) { return Mfma<H>::mma(a, b, c); }
};
template <>
struct GemmMma<float> {
  using frag_t = f32x4_t;
  __device__ __forceinline__ static f32x16_t mma(frag_t a, frag_t b, f32x16_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

struct GemmOperand {
  const char* base;
  int64_t ld;     // bytes from row to row, a multiple of 16
  int64_t plane;  // bytes from plane to plane (float32 operands)
  int extent;     // along k: its rows (i or j); across k: its columns, a multiple of 8
};

struct GemmParams {
  GemmOperand a, b;
  int I, J, K;
  int splits;       // parts of k, each a workgroup of its own
  int segments;     // 1; 3 for operands in two planes, 6 in three
  const int* kept;  // kept rows of the problem, read on the device
  bool j_kept, k_kept;  // J (and b's extent), or K, is *kept instead
};

// x as three bfloat16 terms, each the nearest to what is left; infinities, NaN and values that would round past the
// largest bfloat16 keep their whole value in the first two terms.
__device__ __forceinline__ void split3(float x, __bf16& h, __bf16& m, __bf16& l) {
  const uint32_t u = __float_as_uint(x), e = u & 0x7fffffffu;
  h = e > 0x7f7f0000u ? __builtin_bit_cast(__bf16, (uint16_t)(e > 0x7f800000u ? 0x7fc0u : u >> 16)) : (__bf16)x;
  const float r = e >= 0x7f800000u ? 0.f : x - (float)h;
  m = (__bf16)r;
  l = (__bf16)(r - (float)m);
}

// Slot of 16-byte chunk `chunk` in row k of an across-k tile of 128 columns, for elements of ES bytes. 16 bits: see swz<128>.
// float32: rows 4 apart, which the two halves of a wave read at once, take different halves of the banks.
template <int ES>
__device__ __forceinline__ int across_slot(int k, int chunk) {
  return ES == 2 ? chunk ^ swz<128>(k) : chunk ^ ((k >> 2 & 1) << 3);
}

// Copies of one operand's tile: EXT rows or columns of a step, EXT / 8 wave instructions over NW waves. Every address is
// inside the operand: a lane whose row, column or k lies outside uses an offset past the buffer's end and gets zeros.
template <int ES, bool ACROSS, int EXT, int NW>
struct GemmLoader {
  static constexpr int NQ = EXT / 8 / NW, kStep = 128 / ES, kChunk = 16 / ES, kLanes = 8 * ES;  // lanes of an across row
  static constexpr uint32_t kOut = 0x80000000u, kRange = 0x7fffffffu;
  static_assert(NQ * NW * 8 == EXT && (!ACROSS || EXT % 128 == 0));
  uint32_t off[NQ];
  int at[NQ];  // k of what the lane copies, from the step's first
  int wave;

  __device__ __forceinline__ void init(int w, int lane, int64_t ld, int valid) {
    wave = w;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int piece = q * NW + w;
      if constexpr (ACROSS) {
        const int row = piece % 16 * (64 / kLanes) + lane / kLanes, col = piece / 16 * 128 + across_slot<ES>(row, lane % kLanes) * kChunk;
        off[q] = col < valid ? (uint32_t)(row * ld) + col * ES : kOut;
        at[q] = row;
      } else {
        const int row = piece * 8 + lane / 8, chunk = (lane % 8) ^ swz<64>(row);
        off[q] = row < valid ? (uint32_t)(row * ld) + chunk * 16 : kOut;
        at[q] = chunk * kChunk;
      }
    }
  }
  // base: the tile at this step's first k, of which `left` remain.
  __device__ __forceinline__ void issue(const char* base, char* lds, int left) const {
    const rsrc_t r = make_rsrc(base, kRange);
    if (left >= kStep) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) dma16(r, lds + (q * NW + wave) * 1024, off[q], 0);
    } else {
#pragma unroll
      for (int q = 0; q < NQ; ++q) dma16(r, lds + (q * NW + wave) * 1024, at[q] < left ? off[q] : kOut, 0);
    }
  }
};

// A lane's addresses in a tile for fragments of 32 rows from row r0 + 32 f, k chunk c (a quarter of the step). Both kinds
// hand lane half g the same k: 8 g + e of a 16-bit chunk, 4 g + e of a float32 one. The swizzles separate: along k it
// depends on c and the lane alone (32 f rows are a constant distance), across k on f and the lane (a chunk's rows are),
// so that a few offsets serve every fragment of a step.
template <typename H, bool ACROSS, int NF>
struct GemmFrags {
  static constexpr int ES = sizeof(H), N = !ACROSS ? 4 : ES == 2 ? 2 * NF : NF;
  using frag_t = typename GemmMma<H>::frag_t;
  uint32_t off[N];

  __device__ __forceinline__ void init(int r0) {
    const int lane = threadIdx.x & 63, g = lane >> 5;
    if constexpr (!ACROSS) {
      const int row = r0 + (lane & 31);
#pragma unroll
      for (int c = 0; c < N; ++c) off[c] = row * 128 + (((2 * c + g) ^ swz<64>(row)) << 4);
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int r = r0 + 32 * f, sub = r / 128 * 16384;
        if constexpr (ES == 2) {
          const int s = lane & 15, col = r % 128 + 16 * ((lane >> 4) & 1) + 4 * (s & 3);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int k = 8 * g + 4 * b + (s >> 2);
            off[2 * f + b] = sub + k * 256 + (across_slot<ES>(k, col >> 3) << 4) + (col & 7) * 2;
          }
        } else {
          const int col = r % 128 + (lane & 31), k = 4 * g;
          off[f] = sub + k * 512 + (across_slot<ES>(k, col >> 2) << 4) + (col & 3) * 4;
        }
      }
    }
  }
  __device__ __forceinline__ frag_t get(const char* tile, int f, int c) const {
    if constexpr (!ACROSS) {
      return __builtin_bit_cast(frag_t, *reinterpret_cast<const i16x8_t*>(tile + off[c] + f * 4096));
    } else if constexpr (ES == 2) {
      const i16x4_t a = ds_read_tr16(tile + off[2 * f] + c * 4096), b = ds_read_tr16(tile + off[2 * f + 1] + c * 4096);
      const i16x8_t v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      return __builtin_bit_cast(frag_t, v);
    } else {
      frag_t v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float*>(tile + off[f] + c * 4096 + e * 512);
      return v;
    }
  }
};

// What a tile's epilogue gets: its place and this wave's.
struct GemmTile {
  int i0, j0;      // the wave's first row and column
  int tile_i, tile_j, split;
  int I, J, K;     // valid extents
  int wave_i, wave_j;
};

template <typename H_, int TI_, int TJ_, int WI_, int WJ_, bool A_, bool B_>
struct GemmShape {
  using H = H_;
  static constexpr int ES = sizeof(H_), K = 128 / ES;  // bytes of an element, k of a step
  static constexpr int TI = TI_, TJ = TJ_, WI = WI_, WJ = WJ_, NW = WI_ * WJ_;
  static constexpr bool A = A_, B = B_;
  static constexpr int FI = TI_ / WI_ / 32, FJ = TJ_ / WJ_ / 32;
};

// A wave's results on their way to memory through its share of the LDS: a lane has four consecutive i of one j, memory
// wants whole rows of i. Rows j of 32 FI elements, in 16-byte chunks swizzled by the row. Element: 2 or 4 bytes; a
// 2-byte piece is half a chunk. (Stores of 8 bytes from the accumulators' layout touch 32 rows each.)
template <class S, int ELEM>
struct GemmStage {
  static constexpr int kChunks = 32 * S::FI * ELEM / 16, kRow = 16 * kChunks;
  __device__ __forceinline__ static int at(int row, int chunk) { return row * kRow + ((chunk ^ row) % kChunks << 4); }
  // four values of row `row` from i = 32 fi + 8 q + 4 g
  __device__ __forceinline__ static void put(char* lds, int row, int fi, int q, int g, const void* v) {
    if constexpr (ELEM == 2)
      *reinterpret_cast<uint2*>(lds + at(row, 4 * fi + q) + 8 * g) = *static_cast<const uint2*>(v);
    else
      *reinterpret_cast<i32x4_t*>(lds + at(row, 8 * fi + 2 * q + g)) = *static_cast<const i32x4_t*>(v);
  }
  // f(row, i, chunk) for every chunk of `rows` rows, a wave instruction over whole rows
  template <class F>
  __device__ __forceinline__ static void each(const char* lds, int rows, const F& f) {
    constexpr int kRows = 64 / kChunks;  // rows of an instruction
    const int lane = threadIdx.x & 63;
    wave_order();
#pragma unroll 4
    for (int r = lane / kChunks; r < rows; r += kRows)
      f(r, lane % kChunks * (16 / ELEM), *reinterpret_cast<const i32x4_t*>(lds + at(r, lane % kChunks)));
    wave_order();
  }
  // The lanes of a wave read what others of its lanes wrote: LDS keeps a wave's order, and so must the compiler.
  __device__ __forceinline__ static void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
};

template <class S>
__device__ __forceinline__ void gemm_zero(f32x16_t (&z)[S::FI][S::FJ]) {
#pragma unroll
  for (int i = 0; i < S::FI; ++i)
#pragma unroll
    for (int j = 0; j < S::FJ; ++j) z[i][j] = zero16();
}

template <class S, class Epi>
__global__ __launch_bounds__(S::NW * 64, S::ES == 4 ? 2 : 1) void gemm_kernel(GemmParams p, Epi epi) {
  using H = typename S::H;
  constexpr int TI = S::TI, TJ = S::TJ, FI = S::FI, FJ = S::FJ, NW = S::NW, ES = S::ES;
  // two stages as arrays of their own, so that the reads of one are known not to wait for the copies into the other
  __shared__ __align__(1024) char a0[TI * 128], b0[TJ * 128], a1[TI * 128], b1[TJ * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // Place. Workgroups go round the eight XCDs, each with an L2 of its own: an XCD takes a run of consecutive tiles, in
  // which groups of eight columns of tiles are walked row by row, so that its workgroups share their operands' rows.
  const int kept = (p.j_kept || p.k_kept) ? *p.kept : 0;
  const int J = p.j_kept ? kept : p.J, K = p.k_kept ? kept : p.K;
  const int ni = (p.I + TI - 1) / TI, nj = (J + TJ - 1) / TJ, total = ni * nj * p.splits;
  const int per = (total + 7) / 8, place = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || place >= total) return;
  GemmTile t;
  t.split = place / (ni * nj);
  const int tile = place % (ni * nj), group = tile / (8 * ni), wide = min(8, nj - 8 * group), in = tile % (8 * ni);
  t.tile_i = in / wide;
  t.tile_j = 8 * group + in % wide;
  t.I = p.I, t.J = J, t.K = K;
  t.wave_i = wave / S::WJ, t.wave_j = wave % S::WJ;
  t.i0 = t.tile_i * TI + t.wave_i * (TI / S::WI);
  t.j0 = t.tile_j * TJ + t.wave_j * (TJ / S::WJ);

  // this part's k, in whole steps
  const int steps_all = (K + S::K - 1) / S::K, steps_per = (steps_all + p.splits - 1) / p.splits;
  const int first = min(t.split * steps_per, steps_all), ksteps = min(steps_per, steps_all - first), steps = ksteps * p.segments;

  const int ti0 = t.tile_i * TI, tj0 = t.tile_j * TJ;
  GemmLoader<ES, S::A, TI, NW> la;
  GemmLoader<ES, S::B, TJ, NW> lb;
  la.init(wave, lane, p.a.ld, p.a.extent - ti0);
  lb.init(wave, lane, p.b.ld, (p.j_kept ? kept : p.b.extent) - tj0);
  const int64_t astep = S::A ? S::K * p.a.ld : 128, bstep = S::B ? S::K * p.b.ld : 128;
  const char* abase = p.a.base + (S::A ? (int64_t)ti0 * ES : (int64_t)ti0 * p.a.ld) + first * astep;
  const char* bbase = p.b.base + (S::B ? (int64_t)tj0 * ES : (int64_t)tj0 * p.b.ld) + first * bstep;
  // planes of the segments, two bits each, the first segment lowest: a = m l h m h h, b = m h l h m h; or m h h, h m h
  const uint32_t planes_a = p.segments == 6 ? 0x049u : p.segments == 3 ? 0x01u : 0u;
  const uint32_t planes_b = p.segments == 6 ? 0x121u : p.segments == 3 ? 0x04u : 0u;

  f32x16_t acc[FI][FJ];

  int seg = 0, ks = 0;  // of the next step to copy
  auto copy = [&](char* a, char* b) {
    const int left = K - (first + ks) * S::K;
    la.issue(abase + (int64_t)(planes_a >> (2 * seg) & 3) * p.a.plane + ks * astep, a, left);
    lb.issue(bbase + (int64_t)(planes_b >> (2 * seg) & 3) * p.b.plane + ks * bstep, b, left);
    if (++ks == ksteps) ks = 0, ++seg;
  };
  GemmFrags<H, S::A, FI> ra;
  GemmFrags<H, S::B, FJ> rb;
  ra.init(t.wave_i * (TI / S::WI));
  rb.init(t.wave_j * (TJ / S::WJ));
  // A stage's products, chunk by chunk: chunk c + 1 is read while chunk c's products run, and no earlier (the barriers
  // bound the registers). The last chunk's products wait for the next stage, whose first chunk is read meanwhile: after
  // the workgroup's barrier every wave has products to run.
  constexpr int NC = 4;
  typename GemmMma<H>::frag_t fa[2][FI], fb[2][FJ];
  auto read = [&](const char* a, const char* b, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FI; ++i) fa[c & 1][i] = ra.get(a, i, c);
#pragma unroll
    for (int j = 0; j < FJ; ++j) fb[c & 1][j] = rb.get(b, j, c);
  };
  // float32: a stage's products are a sum of their own. An instruction adds two products, so that one sum over all k would
  // round most: the error of dx of 158 rows of 5 classes at k = 2880 is 1.1e-6 so,
  // 4.5e-6 in one sum (in the registers of two waves a SIMD, out of the accumulation registers, at 2% of the time).
  constexpr bool OWN = ES == 4;
  f32x16_t own[OWN ? FI : 1][OWN ? FJ : 1];
  auto products = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        if constexpr (OWN) {
          own[i][j] = GemmMma<H>::mma(fa[c & 1][i], fb[c & 1][j], c == 0 ? zero16() : own[i][j]);
          if (c == NC - 1) acc[i][j] += own[i][j];
        } else {
          acc[i][j] = GemmMma<H>::mma(fa[c & 1][i], fb[c & 1][j], acc[i][j]);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto stage = [&](const char* a, const char* b, bool first) __attribute__((always_inline)) {
    read(a, b, 0);
    if (!first) products(NC - 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c + 1 < NC; ++c) {
      read(a, b, c + 1);
      products(c);
    }
  };
  auto arrive = [&]() __attribute__((always_inline)) {
    wait_vm_all();
    __syncthreads();  // a stage is there for every wave, and every wave has read the other one
  };
  if (steps > 0) copy(a0, b0);
  epi.template start<S>(acc, t);
  if (steps > 0) {
    arrive();
    if (steps > 1) copy(a1, b1);
    stage(a0, b0, true);
    int s = 1;
    for (; s + 2 <= steps; s += 2) {
      arrive();
      copy(a0, b0);
      stage(a1, b1, false);
      arrive();
      if (s + 2 < steps) copy(a1, b1);
      stage(a0, b0, false);
    }
    if (s < steps) {
      arrive();
      stage(a1, b1, false);
    }
    products(NC - 1);
  }
  __syncthreads();  // the tiles are read: each wave takes 2 KB of their LDS for a 32 x 32 block
  constexpr int kShare = FI * FJ * 2048, kPer = TI * 128 / kShare;
  static_assert(NW <= kPer || (TI == TJ && NW <= 4 * kPer));
  const int part = wave / kPer;
  char* const lds = part == 0 ? a0 : part == 1 ? b0 : part == 2 ? a1 : b1;
  epi.template run<S>(acc, t, lds + wave % kPer * kShare);
}

template <class S, class Epi>
hipError_t launch_gemm(const GemmParams& p, const Epi& epi, hipStream_t st) {
  // p.J is the most that the kept rows can be: workgroups beyond the tiles that there are return at once
  const int64_t tiles = (int64_t)((p.I + S::TI - 1) / S::TI) * ((p.J + S::TJ - 1) / S::TJ) * p.splits;
  if (tiles == 0) return hipSuccess;
  if (tiles * S::NW * 64 >= (int64_t(1) << 32)) return hipErrorInvalidValue;  // more threads than a launch holds
  gemm_kernel<S, Epi><<<dim3((unsigned)((tiles + 7) / 8 * 8)), S::NW * 64, 0, st>>>(p, epi);
  return hipGetLastError();
}

}  // namespace theria
