// Embedding lookup with a scale, and its gradient by sorted tokens (gfx950).
//
//   lookup    out[n] = s W[ids[n]]
//   gradient  dW[v] = s sum of dout[n] over the n with ids[n] = v, zeros for ids that no token has
//
// Both are bound by memory. The gradient orders the tokens by (id, n) first: every row of dW then has a known run of
// tokens and is summed in float32 and written once, in an order that does not depend on the run (no float atomics, no
// float32 copy of the table, no clearing pass).
//
//   order   up to kRankTokens tokens: one launch in which every token counts the tokens before it (n^2 comparisons out
//           of LDS, spread over the GPU). More: a stable radix sort, digits of at most 10 bits, two launches a digit.
//   pieces  frequent ids: every aligned run of 64 sorted tokens that holds one id alone is summed by a workgroup of its
//           own into a float32 row of the workspace, so that an id with thousands of tokens is spread over the GPU.
//   rows    every table row: the tokens before its first whole piece, the pieces, and the tokens after its last one. Of
//           few tokens and rows this launch is the only one (own_launch): each workgroup finds its rows' tokens itself.
#include "token_common.hpp"
#include "token_params.hpp"

namespace theria {
namespace {

constexpr int kPiece = 64;         // sorted tokens of a piece
// Most tokens ordered by counting: 12 us for 4096 and 20 us for 8192 tokens, where two passes of the sort take 25 us; 16384
// tokens would take 35 us against 25 us.
constexpr int kRankTokens = 8192;
constexpr int kSortMost = 1024;     // digits of a radix sort's pass

__device__ __forceinline__ int64_t load_id(const void* ids, bool ids64, int64_t n) {
  return ids64 ? ((const int64_t*)ids)[n] : (int64_t)((const int32_t*)ids)[n];
}

// The sort key of an id: the id, or `classes` (behind every row) for padding and for ids outside the table.
__device__ __forceinline__ uint32_t key_of(const EmbedParams& p, int64_t n) {
  const int64_t id = load_id(p.ids, p.ids64, n);
  return id < 0 || id >= p.classes || id == p.padding ? (uint32_t)p.classes : (uint32_t)id;
}

// ------------------------------------------------------------------------------------------ lookup
// Teams of TPR threads, one for each token; a thread moves two vectors of the row (grid.y covers wide rows).
template <typename T, int VEC, int TPR>
__global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedParams p) {
  constexpr int TEAMS = 256 / TPR;
  const int t = threadIdx.x % TPR;
  const int64_t n = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TPR;
  if (n >= p.n) return;
  const int64_t id = load_id(p.ids, p.ids64, n);
  const bool known = id >= 0 && id < p.classes, zero = p.zero_padding && id == p.padding;
  const T* row = (const T*)p.table.p + (known ? id : 0) * p.table.sr;
  RawVec<T, VEC> raw[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = ((2 * blockIdx.y + i) * TPR + t) * VEC;
    raw[i].load(row + c, known ? p.width - c : 0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = ((2 * blockIdx.y + i) * TPR + t) * VEC;
    if (c >= p.width) continue;
    float f[VEC];
    raw[i].get(f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = zero ? 0.f : known ? f[e] * p.scale : __builtin_nanf("");
    raw[i].set(f);
    raw[i].store((T*)p.out.p + n * p.out.sr + c, p.width - c);
  }
}

// ------------------------------------------------------------------------------------------ order
// No tokens for any row yet: a share of the first launch.
__device__ __forceinline__ void clear_bounds(int2* bounds, int64_t classes) {
  for (int64_t v = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; v < classes; v += (int64_t)gridDim.x * blockDim.x) bounds[v] = int2{0, 0};
}

// keys[r], order[r]: the token of rank r. A workgroup ranks 64 tokens, each of its 16 waves against a sixteenth of all.
__global__ __launch_bounds__(1024) void rank_kernel(EmbedParams p, uint32_t* keys, uint32_t* order, int2* bounds) {
  __shared__ __align__(16) uint32_t all[kRankTokens + 64];
  __shared__ int part[16][64];
  const int n = (int)p.n, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  clear_bounds(bounds, p.classes);
  const int slice = (n + 63) / 64 * 4;  // tokens of a wave, a multiple of 4; 16 slices cover n
  for (int i = threadIdx.x; i < 16 * slice; i += 1024) all[i] = i < n ? key_of(p, i) : 0xffffffffu;
  __syncthreads();
  const int i = blockIdx.x * 64 + lane;
  const uint32_t mine = all[min(i, n - 1)];
  const int j0 = wave * slice, j1 = j0 + slice;
  // tokens of the same id count when they come earlier: compare with mine + 1 before this workgroup's tokens, mine after
  const int own0 = blockIdx.x * 64, own1 = own0 + 64;
  const int before = min(max(own0, j0), j1), after = min(max(own1, j0), j1);  // multiples of 4
  int rank = 0;
  for (int j = j0; j < before; j += 4) {
    const u32x4_t k = *reinterpret_cast<const u32x4_t*>(all + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) rank += k[e] <= mine;
  }
  for (int j = before; j < after; ++j) rank += all[j] < mine || (all[j] == mine && j < i);
  for (int j = after; j < j1; j += 4) {
    const u32x4_t k = *reinterpret_cast<const u32x4_t*>(all + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) rank += k[e] < mine;
  }
  part[wave][lane] = rank;
  __syncthreads();
  if (wave == 0 && i < n) {
    int r = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) r += part[w][lane];
    keys[r] = mine;
    order[r] = (uint32_t)i;
  }
}

// One digit of the radix sort. from == nullptr: the keys are taken from the ids, the tokens in order.
struct SortPass {
  const uint32_t *from_key, *from_order;
  uint32_t *to_key, *to_order;
  uint32_t* hist;  // [tiles][digits]
  int2* bounds;
  int shift, bits, tiles;
};

__device__ __forceinline__ uint32_t sort_key(const EmbedParams& p, const SortPass& s, int64_t n) {
  return s.from_key ? s.from_key[n] : key_of(p, n);
}

// ROUNDS rounds of 64 tokens for each of a workgroup's four waves.
template <int ROUNDS>
__global__ __launch_bounds__(256) void sort_count_kernel(EmbedParams p, SortPass s) {
  __shared__ uint32_t count[kSortMost];
  const int digits = 1 << s.bits;
  if (!s.from_key) clear_bounds(s.bounds, p.classes);
  for (int d = threadIdx.x; d < digits; d += 256) count[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * 256 * ROUNDS;
#pragma unroll 4
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t n = base + r * 256 + threadIdx.x;
    if (n < p.n) atomicAdd(&count[sort_key(p, s, n) >> s.shift & (digits - 1)], 1u);  // whole numbers: any order
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += 256) s.hist[(int64_t)blockIdx.x * digits + d] = count[d];
}

// Places of a tile's tokens: the tokens of smaller digits, of the same digit in earlier tiles, in earlier waves of this
// tile (a wave takes consecutive tokens), and before it in its wave (by ballots over the digit's bits).
template <int ROUNDS>
__global__ __launch_bounds__(256) void sort_place_kernel(EmbedParams p, SortPass s) {
  __shared__ uint32_t count[4][kSortMost];  // a wave's tokens of each digit so far; then the place of its first
  __shared__ uint32_t sums[256];
  const int digits = 1 << s.bits, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  for (int d = threadIdx.x; d < 4 * kSortMost; d += 256) count[d / kSortMost][d % kSortMost] = 0;
  __syncthreads();
  const int64_t base = ((int64_t)blockIdx.x * 4 + wave) * 64 * ROUNDS;
  uint32_t key[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t n = base + r * 64 + lane;
    key[r] = n < p.n ? sort_key(p, s, n) : 0;
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool in = base + r * 64 + lane < p.n;
    const uint32_t d = key[r] >> s.shift & (digits - 1);
    uint64_t same = __ballot(in);
    for (int b = 0; b < s.bits; ++b) {
      const uint64_t set = __ballot(d >> b & 1);
      same &= d >> b & 1 ? set : ~set;
    }
    const uint32_t earlier = __popcll(same & ((1ull << lane) - 1));
    if (in) rank[r] = count[wave][d] + earlier;
    __builtin_amdgcn_wave_barrier();  // every lane has read the count before one of its digit raises it
    if (in && earlier == 0) count[wave][d] += (uint32_t)__popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
  // digits 4 t .. 4 t + 3 belong to thread t: their tokens in all tiles and in the tiles before this one
  const int per = (digits + 255) / 256;
  uint32_t total[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0}, mine = 0;
  for (int q = 0; q < per; ++q) {
    const int d = threadIdx.x * per + q;
    if (d >= digits) break;
#pragma unroll 8
    for (int b = 0; b < s.tiles; ++b) {
      const uint32_t h = s.hist[(int64_t)b * digits + d];
      total[q] += h;
      before[q] += b < (int)blockIdx.x ? h : 0;
    }
    mine += total[q];
  }
  sums[threadIdx.x] = mine;
  __syncthreads();
  for (int o = 1; o < 256; o *= 2) {  // inclusive scan over the threads
    const uint32_t add = (int)threadIdx.x >= o ? sums[threadIdx.x - o] : 0;
    __syncthreads();
    sums[threadIdx.x] += add;
    __syncthreads();
  }
  uint32_t place = sums[threadIdx.x] - mine;
  for (int q = 0; q < per; ++q) {
    const int d = threadIdx.x * per + q;
    if (d >= digits) break;
    uint32_t at = place + before[q];
    for (int w = 0; w < 4; ++w) {
      const uint32_t c = count[w][d];
      count[w][d] = at;
      at += c;
    }
    place += total[q];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t n = base + r * 64 + lane;
    if (n < p.n) {
      const uint32_t at = count[wave][key[r] >> s.shift & (digits - 1)] + rank[r];
      s.to_key[at] = key[r];
      s.to_order[at] = s.from_order ? s.from_order[n] : (uint32_t)n;
    }
  }
}

// ------------------------------------------------------------------------------------------ sums
// Tokens [s, e) of the order, every `step`-th from s + first: the thread's vector of their rows added to acc, eight rows
// in flight.
template <typename T, int VEC>
__device__ __forceinline__ void add_tokens(float (&acc)[VEC], const EmbedParams& p, const uint32_t* order, uint32_t s, uint32_t e, int first, int step,
                                           int c) {
  constexpr int U = 8;
  for (uint32_t j = s + first; j < e; j += U * step) {
    RawVec<T, VEC> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t at = j + u * step;
      raw[u].zero();
      if (at < e) raw[u].load((const T*)p.dout.p + (int64_t)order[at] * p.dout.sr + c, p.width - c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[VEC];
      raw[u].get(f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += f[k];
    }
  }
}

// acc summed over a workgroup's teams in team 0's threads, in the teams' order.
template <int VEC, int TPR>
__device__ __forceinline__ void join_teams(float (&acc)[VEC], float* lds) {
  constexpr int TEAMS = 256 / TPR;
  const int t = threadIdx.x % TPR, team = threadIdx.x / TPR;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < VEC; ++k) lds[(team * TPR + t) * (VEC + 1) + k] = acc[k];
  __syncthreads();
  if (team == 0) {
#pragma unroll
    for (int q = 1; q < TEAMS; ++q)
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += lds[(q * TPR + t) * (VEC + 1) + k];
  }
}

// Sums of the pieces that hold one id, and every row's bounds in the order: the tokens where the id changes write them.
template <typename T, int VEC, int TPR>
__global__ __launch_bounds__(256) void embed_piece_kernel(EmbedParams p, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order,
                                                          int2* __restrict__ bounds, float* __restrict__ pieces) {
  constexpr int TEAMS = 256 / TPR;
  __shared__ float lds[256 * (VEC + 1)];
  const int64_t s = (int64_t)blockIdx.x * kPiece;
  if (blockIdx.y == 0 && threadIdx.x < kPiece && s + threadIdx.x < p.n) {
    const int64_t i = s + threadIdx.x;
    const uint32_t key = keys[i];
    if (key < p.classes) {
      if (i == 0 || keys[i - 1] != key) bounds[key].x = (int)i;
      if (i + 1 == p.n || keys[i + 1] != key) bounds[key].y = (int)i + 1;
    }
  }
  if (s + kPiece > p.n) return;
  const uint32_t key = keys[s];
  if (key != keys[s + kPiece - 1] || key >= p.classes) return;
  const int t = threadIdx.x % TPR, team = threadIdx.x / TPR, c = (blockIdx.y * TPR + t) * VEC;
  float acc[VEC] = {};
  add_tokens<T, VEC>(acc, p, order, (uint32_t)s, (uint32_t)s + kPiece, team, TEAMS, c);
  join_teams<VEC, TPR>(acc, lds);
  if (team == 0 && c < p.width) {
    RawVec<float, VEC> out;
    out.set(acc);
    out.store(pieces + (int64_t)blockIdx.x * p.width + c, p.width - c);
  }
}

constexpr int kRowsMost = 16;   // table rows of a workgroup
constexpr int kOwnTokens = 512;  // most tokens whose gradient may be one launch instead of three
constexpr int kTeamTokens = 8;  // most tokens that a team sums alone

// The tokens of table rows v0 to v0 + have, in order, and each row's run of them, found by the workgroup itself: every one
// looks at every id, which takes less than a launch while they are few.
__device__ __forceinline__ void own_order(const EmbedParams& p, int64_t v0, int have, uint32_t* order, int2* bound, int (&count)[kOwnTokens / 64][kRowsMost]) {
  constexpr int PER = kOwnTokens / 256;
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  int row[PER], before[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int n = u * 256 + threadIdx.x;
    const int64_t at = n < p.n ? (int64_t)key_of(p, n) - v0 : -1;
    row[u] = at >= 0 && at < have ? (int)at : -1;
    before[u] = 0;
    for (int r = 0; r < have; ++r) {
      const uint64_t all = __ballot(row[u] == r);
      if (lane == 0) count[4 * u + wave][r] = __popcll(all);
      if (row[u] == r) before[u] = __popcll(all & ((uint64_t(1) << lane) - 1));
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < kRowsMost) {  // each row's counts to places in it, and its tokens
    int sum = 0;
    if ((int)threadIdx.x < have)
#pragma unroll
      for (int k = 0; k < kOwnTokens / 64; ++k) {
        const int c = count[k][threadIdx.x];
        count[k][threadIdx.x] = sum;
        sum += c;
      }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < kRowsMost; o *= 2) {
      const int add = __shfl_up(upto, o, kRowsMost);
      if ((int)threadIdx.x >= o) upto += add;
    }
    bound[threadIdx.x] = int2{upto - sum, upto};
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (row[u] >= 0) order[bound[row[u]].x + count[4 * u + wave][row[u]] + before[u]] = u * 256 + threadIdx.x;
  __syncthreads();
}

// `rows` table rows of a workgroup, one for each team in turn; rows with more tokens take all the teams. OWN: the gradient of at
// most kOwnTokens tokens, in this launch alone.
template <typename T, int VEC, int TPR, bool OWN>
__global__ __launch_bounds__(256) void embed_rows_kernel(EmbedParams p, int64_t first, const uint32_t* __restrict__ sorted, const int2* __restrict__ bounds,
                                                         const float* __restrict__ pieces, int rows, int cols) {
  constexpr int TEAMS = 256 / TPR;
  __shared__ float lds[256 * (VEC + 1)];
  __shared__ int2 bound[kRowsMost];
  const int64_t v0 = (int64_t)(blockIdx.x / cols) * rows;  // from `first`
  const int have = (int)min((int64_t)rows, p.classes - first - v0);
  __shared__ uint32_t own[OWN ? kOwnTokens : 1];
  __shared__ int count[OWN ? kOwnTokens / 64 : 1][kRowsMost];
  const uint32_t* order;
  if constexpr (OWN) {
    own_order(p, first + v0, have, own, bound, count);
    order = own;
  } else {
    if ((int)threadIdx.x < have) bound[threadIdx.x] = bounds[first + v0 + threadIdx.x];
    __syncthreads();
    order = sorted;
  }
  const int t = threadIdx.x % TPR, team = threadIdx.x / TPR, c = ((int)(blockIdx.x % cols) * TPR + t) * VEC;
  auto write = [&](const float(&acc)[VEC], int64_t v) {
    if (c >= p.width) return;
    float f[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = acc[k] * p.scale;
    RawVec<T, VEC> out;
    out.set(f);
    out.stream((T*)p.out.p + v * p.out.sr + c, p.width - c);
  };
  for (int r = team; r < have; r += TEAMS) {
    const int2 at = bound[r];
    if (at.y - at.x > kTeamTokens) continue;
    float acc[VEC] = {};
    add_tokens<T, VEC>(acc, p, order, at.x, at.y, 0, 1, c);
    write(acc, v0 + r);
  }
  for (int r = 0; r < have; ++r) {
    const int s = bound[r].x, e = bound[r].y;
    if (e - s <= kTeamTokens) continue;
    const int a = (s + kPiece - 1) / kPiece, b = e / kPiece;  // whole pieces [a, b)
    float acc[VEC] = {};
    if (!OWN && a < b) {
      add_tokens<T, VEC>(acc, p, order, s, a * kPiece, team, TEAMS, c);
      if (c < p.width) {
#pragma unroll 4
        for (int q = a + team; q < b; q += TEAMS) {
          RawVec<float, VEC> raw;
          raw.load(pieces + (int64_t)q * p.width + c, p.width - c);
          float f[VEC];
          raw.get(f);
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += f[k];
        }
      }
      add_tokens<T, VEC>(acc, p, order, b * kPiece, e, team, TEAMS, c);
    } else {
      add_tokens<T, VEC>(acc, p, order, s, e, team, TEAMS, c);
    }
    join_teams<VEC, TPR>(acc, lds);
    if (team == 0) write(acc, v0 + r);
  }
}

// ------------------------------------------------------------------------------------------ launches
int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

int key_bits(int64_t classes) {  // keys run from 0 to classes
  int b = 1;
  while (b < 32 && classes >> b) ++b;
  return b;
}

template <typename T, int VEC, int TPR>
hipError_t fwd(const EmbedParams& p, hipStream_t st) {
  constexpr int TEAMS = 256 / TPR, COLS = 2 * TPR * VEC;
  // a launch holds fewer than 2^32 threads in x
  for (int64_t n = 0; n < p.n; n += int64_t(1) << 23) {
    EmbedParams q = p;
    q.n = p.n - n < int64_t(1) << 23 ? p.n - n : int64_t(1) << 23;
    q.ids = (const char*)p.ids + n * (p.ids64 ? 8 : 4);
    q.out.p = (T*)p.out.p + n * p.out.sr;
    embed_fwd_kernel<T, VEC, TPR><<<dim3((unsigned)((q.n + TEAMS - 1) / TEAMS), (p.width + COLS - 1) / COLS), 256, 0, st>>>(q);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

struct Order {
  uint32_t *keys, *order;
  int2* bounds;
  float* pieces;
};

// A radix sort's workgroup takes 1024 tokens, or 4096 where so many workgroups would each read too many others' counts.
constexpr int64_t kSmallSort = 131072;
int sort_tiles(int64_t n) { return (int)((n + 1023) / 1024 <= kSmallSort / 1024 ? (n + 1023) / 1024 : (n + 4095) / 4096); }

// The workspace: keys and order twice, the digits' counts, the rows' bounds, and a float32 row for each piece.
struct Space {
  int64_t each, hist, bounds, pieces, bytes;
  explicit Space(const EmbedParams& p)
      : each(align256(4 * p.n)),
        hist(4 * each),
        bounds(hist + align256(4 * kSortMost * (int64_t)sort_tiles(p.n))),
        pieces(bounds + align256(8 * p.classes)),
        bytes(pieces + 4 * (p.n / kPiece) * p.width) {}
};

hipError_t sort_tokens(const EmbedParams& p, Order& o, hipStream_t st) {
  char* ws = (char*)p.ws;
  const Space at(p);
  uint32_t *key[2] = {(uint32_t*)ws, (uint32_t*)(ws + at.each)}, *ord[2] = {(uint32_t*)(ws + 2 * at.each), (uint32_t*)(ws + 3 * at.each)};
  o = {key[0], ord[0], (int2*)(ws + at.bounds), (float*)(ws + at.pieces)};
  if (p.n <= kRankTokens) {
    rank_kernel<<<dim3((unsigned)((p.n + 63) / 64)), 1024, 0, st>>>(p, o.keys, o.order, o.bounds);
    return hipGetLastError();
  }
  const int bits = key_bits(p.classes), passes = (bits + 9) / 10, each_bits = (bits + passes - 1) / passes;
  const int tiles = sort_tiles(p.n);
  SortPass s{nullptr, nullptr, key[0], ord[0], (uint32_t*)(ws + at.hist), o.bounds, 0, each_bits, tiles};
  for (int q = 0; q < passes; ++q) {
    s.to_key = key[q & 1], s.to_order = ord[q & 1];
    if (p.n <= kSmallSort) {
      sort_count_kernel<4><<<dim3((unsigned)tiles), 256, 0, st>>>(p, s);
      sort_place_kernel<4><<<dim3((unsigned)tiles), 256, 0, st>>>(p, s);
    } else {
      sort_count_kernel<16><<<dim3((unsigned)tiles), 256, 0, st>>>(p, s);
      sort_place_kernel<16><<<dim3((unsigned)tiles), 256, 0, st>>>(p, s);
    }
    s.from_key = s.to_key, s.from_order = s.to_order;
    s.shift += each_bits;
  }
  o.keys = s.to_key, o.order = s.to_order;
  return hipGetLastError();
}

// Columns of workgroups of the gradient, and its table rows for each (several once they fill the GPU).
int grad_team(const EmbedParams& p) { return p.width <= 16 * (p.dtype == 0 ? 4 : 8) ? 16 : 64; }
int64_t grad_cols(const EmbedParams& p) {
  const int64_t cols = (int64_t)grad_team(p) * (p.dtype == 0 ? 4 : 8);
  return (p.width + cols - 1) / cols;
}
int64_t grad_rows(const EmbedParams& p) {
  const int64_t per = p.classes * grad_cols(p) / (16 * (int64_t)device_cu_count());
  return per < 1 ? 1 : per < kRowsMost ? per : kRowsMost;
}
// Whether the gradient is one launch. (512, 32 to 1000, up to 4096) bfloat16: 44 us a call with its lookup against 50 us, 6 to 7 us
// against 12 to 13 in a graph; an id that all 512 tokens share 21 us against 17. More workgroups than those with fewer
// than kRowsMost rows each lose it again, (512, 128000, 1024) 62 us against 58; more tokens than these wait for the one id.
bool own_launch(const EmbedParams& p) { return p.n <= kOwnTokens && grad_rows(p) < kRowsMost; }

template <typename T, int VEC, int TPR>
hipError_t bwd(const EmbedParams& p, hipStream_t st) {
  const unsigned cols = (unsigned)grad_cols(p);
  const bool own = own_launch(p) || p.n == 0;
  Order o{};
  if (!own) {
    hipError_t e = sort_tokens(p, o, st);
    if (e != hipSuccess) return e;
    embed_piece_kernel<T, VEC, TPR><<<dim3((unsigned)((p.n + kPiece - 1) / kPiece), cols), 256, 0, st>>>(p, o.keys, o.order, o.bounds, o.pieces);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int rows = (int)grad_rows(p);
  const int64_t most = (int64_t(1) << 23) / cols * rows;  // table rows: a launch holds fewer than 2^32 threads
  for (int64_t v = 0; v < p.classes; v += most) {
    const int64_t have = p.classes - v < most ? p.classes - v : most;
    EmbedParams q = p;
    q.out.p = (T*)p.out.p + v * p.out.sr;
    const auto kernel = own ? embed_rows_kernel<T, VEC, TPR, true> : embed_rows_kernel<T, VEC, TPR, false>;
    kernel<<<dim3((unsigned)((have + rows - 1) / rows * cols)), 256, 0, st>>>(q, v, o.order, o.bounds, o.pieces, rows, (int)cols);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, bool GRAD>
hipError_t by_width(const EmbedParams& p, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const int n = (p.width + V - 1) / V;
  if constexpr (GRAD) {
    return grad_team(p) == 16 ? bwd<T, V, 16>(p, st) : bwd<T, V, 64>(p, st);
  } else {
    if (n <= 16) return fwd<T, V, 16>(p, st);
    return n <= 128 ? fwd<T, V, 64>(p, st) : fwd<T, V, 256>(p, st);
  }
}

template <bool GRAD>
hipError_t by_type(const EmbedParams& p, hipStream_t st) {
  if (p.dtype == 0) return by_width<float, GRAD>(p, st);
  if (p.dtype == 1) return by_width<_Float16, GRAD>(p, st);
  return by_width<__bf16, GRAD>(p, st);
}

}  // namespace

int64_t embed_ws_bytes(const EmbedParams& p) { return Space(p).bytes; }
hipError_t launch_embed_fwd(const EmbedParams& p, hipStream_t st) { return by_type<false>(p, st); }
hipError_t launch_embed_bwd(const EmbedParams& p, hipStream_t st) { return by_type<true>(p, st); }

}  // namespace theria
