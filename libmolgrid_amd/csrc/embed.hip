// Type vectors out of a learned table (mg_embed_types) and the gradients of the table and of a
// per-token scale.
//
//   y[n,c] = s_n W[t_n,c]                 zero where t_n names no row of W
//   dW[v,c] = sum over n with t_n = v of s_n g[n,c]        in float, in a fixed order
//   ds_n = sum over c of g[n,c] W[t_n,c]
//
// The sums by row come in two ways.  A table of few rows is summed where the tokens are read: every
// wave keeps a copy of it in LDS and adds its tokens there, and the copies are added afterwards; no
// order of the tokens is better or worse for it.  For any other table the tokens are sorted by row
// first and a team of lanes adds the tokens of a row; rows of many tokens are cut into pieces.
#include <type_traits>

#include "kernels.h"
#include "row_team.h"

namespace mg {
namespace {

constexpr int kThreads = 256;
constexpr int kResident = 2048;   // workgroups of 256 threads that fill the chip

// Rows that a team of LANES lanes holds with a pack each: it takes kTokens tokens at a time, whose
// indices, and then rows, are loaded together.  204,000 tokens of 28 channels of float: 8.3 us (23 MB
// written); the waits for index and row are what is left.
constexpr int kTokens = 4;

template <typename T, int VEC, int LANES>
__global__ __launch_bounds__(kThreads) void embed_narrow_kernel(TokenArg t, const T* __restrict__ table,
                                                                float scale,
                                                                const float* __restrict__ scales,
                                                                T* __restrict__ out) {
  constexpr int kTeams = kThreads / LANES;
  const int c = threadIdx.x % LANES * VEC, team = threadIdx.x / LANES;
  const uint32_t ntokens = (uint32_t)t.ntokens;
  for (uint32_t n0 = blockIdx.x * kTeams * kTokens; n0 < ntokens; n0 += gridDim.x * kTeams * kTokens) {
    uint32_t n[kTokens];
    int row[kTokens];
    float by[kTokens], v[kTokens][VEC];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) n[u] = n0 + u * kTeams + team;
    token_rows(t, n, ntokens, row);
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      by[u] = scales ? scales[n[u] < ntokens ? n[u] : 0] : scale;
      if (t.nrows > 0)
        load_floats<T, VEC>(table + (size_t)(row[u] < 0 ? 0 : row[u]) * t.channels + (c < t.channels ? c : 0), v[u]);
    }
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      if (n[u] >= ntokens || c >= t.channels) continue;
      // (a row that is not there is zero whatever the scale is)
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[u][i] = row[u] < 0 ? 0.f : by[u] * v[u][i];
      store_floats<T, VEC>(out + (size_t)n[u] * t.channels + c, v[u]);
    }
  }
}

// Wider rows: a wave takes one token at a time; the index of its next token is read ahead.  Memory
// bound: 65,536 tokens of 4,096 channels of bfloat16 in 153 us (0.54 GB written, 0.16 GB of rows read
// at least once: 4.6 TB/s).
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void embed_kernel(TokenArg t, const T* __restrict__ table,
                                                         float scale,
                                                         const float* __restrict__ scales,
                                                         T* __restrict__ out) {
  constexpr int LANES = kWave, kTeams = kThreads / LANES, kUnroll = 4;
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const uint32_t step = gridDim.x * kTeams, ntokens = (uint32_t)t.ntokens;
  uint32_t n = blockIdx.x * kTeams + team;
  int row = n < ntokens ? token_row(t, n) : -1;
  float s = scales && n < ntokens ? scales[n] : scale;
  for (; n < ntokens; n += step) {
    const T* from = table + (size_t)(row < 0 ? 0 : row) * t.channels;
    T* to = out + (size_t)n * t.channels;
    const int at = row;
    const float by = s;
    if (n + step < ntokens) {
      row = token_row(t, n + step);
      if (scales) s = scales[n + step];
    }
    for (int c0 = lane * VEC; c0 < t.channels; c0 += LANES * VEC * kUnroll) {
      float v[kUnroll][VEC];
      if (t.nrows > 0)
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {   // (beyond the last channel: the first ones, not used)
          const int c = c0 + u * LANES * VEC;
          load_floats<T, VEC>(from + (c < t.channels ? c : 0), v[u]);
        }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int c = c0 + u * LANES * VEC;
        if (c >= t.channels) break;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[u][i] = at < 0 ? 0.f : by * v[u][i];
        store_floats<T, VEC>(to + c, v[u]);
      }
    }
  }
}

// ds: a team takes one token at a time: 16,384 tokens of 1,024 bfloat16 in 11 us.  Where a small table's
// gradient is summed, ds comes out there.
template <typename T, int VEC, int LANES>
__global__ __launch_bounds__(kThreads) void scale_gradient_kernel(TokenArg t,
                                                                  const T* __restrict__ grad,
                                                                  const T* __restrict__ table,
                                                                  float* __restrict__ out) {
  constexpr int kTeams = kThreads / LANES;
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const uint32_t step = gridDim.x * kTeams, ntokens = (uint32_t)t.ntokens;
  for (uint32_t n0 = blockIdx.x * kTeams; n0 < ntokens; n0 += step) {
    const uint32_t n = n0 + team;
    const int row = n < ntokens ? token_row(t, n) : -1;
    float sum = 0.f;
    if (row >= 0)
      for (int c = lane * VEC; c < t.channels; c += LANES * VEC) {
        float g[VEC], w[VEC];
        load_floats<T, VEC>(grad + (size_t)n * t.channels + c, g);
        load_floats<T, VEC>(table + (size_t)row * t.channels + c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum = fmaf(g[i], w[i], sum);
      }
    sum = team_sum_in_wave<LANES>(sum);
    if (n < ntokens && lane == 0) out[n] = sum;
  }
}

// What is added up: the gradient's rows, times the tokens' scale, dropped out.
struct SumArg {
  float scale;
  const float* scales;
  DropArg drop;
};
template <bool DROP, int VEC>
__device__ __forceinline__ void add_token(size_t e, const SumArg& a, float by, uint64_t seed,
                                          uint64_t offset, float (&g)[VEC], float (&acc)[VEC]) {
  if (DROP) drop<VEC>(e, a.drop, seed, offset, g);
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = DROP ? acc[i] + g[i] : fmaf(by, g[i], acc[i]);
}

// ---- few rows: a copy of the table for every team, in LDS -----------------------------------------
//
// A workgroup takes a share of the tokens and LANES packs of channels; its teams take the share's
// tokens in turn and add them to a copy of the table of their own, so that every sum is added up
// by one lane in the tokens' order.  A copy holds element i of pack l of a row at
// (row VEC + i) LANES + l: the lanes of a team never meet in a bank.  The LDS for it is
// 256 nrows VEC bytes a wave whatever LANES is, and LDS is what limits the waves on a CU.
constexpr int kTableLds = 64 << 10;   // of a workgroup, so that two share a CU
constexpr int kTableUnroll = 8;       // tokens of a team in flight

//
// The tokens of a team go through in rounds of kTableUnroll, a round's loads in flight while the
// round before it is added: 204,000 tokens, 28 rows of 28 floats with SCALES in 19 us, 121,250 of 32
// floats with DROP in 16.5 us, of 28 bfloat16, an element a load, in 30 us, and 4 us for the second launch.
// SCALES: the gradients of the tokens' scales come out on the way (one tile of channels then holds a
// row), with the table itself in LDS behind the copies.
template <typename T, int VEC, int LANES, bool DROP, bool SCALES>
__global__ __launch_bounds__(kThreads) void few_rows_kernel(TokenArg t, const T* __restrict__ grad,
                                                            SumArg a, int share, const T* __restrict__ table,
                                                            float* __restrict__ grad_scales, T* out,
                                                            float* partial, uint32_t* __restrict__ named) {
  HIP_DYNAMIC_SHARED(float, copies);
  __shared__ uint32_t any_named;
  uint32_t my_named = 0;
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const int teams = blockDim.x / LANES;
  const int copy = t.nrows * VEC * LANES;
  float* mine = copies + team * copy + lane;
  const float* own = copies + teams * copy + lane;
  const int c = (blockIdx.y * LANES + lane) * VEC;
  const bool inside = c < t.channels;
  const uint32_t begin = blockIdx.x * (uint32_t)share;
  const uint32_t end = min(begin + (uint32_t)share, (uint32_t)t.ntokens);
  struct Round {
    int row[kTableUnroll];
    float by[kTableUnroll];
    Pack<T, VEC> g[kTableUnroll];
  };
  const auto fetch = [&](uint32_t n0, Round& r) {
    uint32_t n[kTableUnroll];
#pragma unroll
    for (int u = 0; u < kTableUnroll; ++u) n[u] = n0 + u * teams;
    token_rows(t, n, end, r.row);
#pragma unroll
    for (int u = 0; u < kTableUnroll; ++u) {
      const uint32_t m = n[u] < end ? n[u] : begin;   // (a token that is there)
      r.by[u] = a.scales ? a.scales[m] : a.scale;
      r.g[u] = *reinterpret_cast<const Pack<T, VEC>*>(grad + (size_t)m * t.channels + (inside ? c : 0));
    }
  };
  Round next;
  fetch(begin + team, next);
  for (int i = 0; i < t.nrows * VEC; ++i) mine[i * LANES] = 0.f;
  if (SCALES) {
    float* to = copies + teams * copy;
#pragma unroll 8
    for (int i = threadIdx.x; i < copy; i += blockDim.x) {
      const int at = i % LANES * VEC + i / LANES % VEC;
      to[i] = at < t.channels ? widen(table[(size_t)(i / (LANES * VEC)) * t.channels + at]) : 0.f;
    }
    __syncthreads();
  }
  uint64_t seed = 0, offset = 0;
  if (DROP) drop_key(a.drop, seed, offset);
  for (uint32_t b0 = begin; b0 < end; b0 += teams * kTableUnroll) {
    const uint32_t n0 = b0 + team;
    const Round now = next;
    fetch(n0 + teams * kTableUnroll, next);
#pragma unroll
    for (int u = 0; u < kTableUnroll; ++u) {
      const uint32_t n = n0 + u * teams;
      float g[VEC], dot = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[i] = now.g[u][i];
      if (now.row[u] >= 0 && inside) {
        const int at = now.row[u] * VEC * LANES;
        my_named |= 1u << now.row[u];
        if (SCALES)
#pragma unroll
          for (int i = 0; i < VEC; ++i) dot = fmaf(g[i], own[at + i * LANES], dot);
        float sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = mine[at + i * LANES];
        add_token<DROP, VEC>((size_t)n * t.channels + c, a, now.by[u], seed, offset, g, sum);
#pragma unroll
        for (int i = 0; i < VEC; ++i) mine[at + i * LANES] = sum[i];
      }
      if (SCALES) {
        dot = team_sum_in_wave<LANES>(dot);
        if (lane == 0 && n < end) grad_scales[n] = dot;
      }
    }
  }
  if (named && threadIdx.x == 0) any_named = 0;
  __syncthreads();
  if (named) {   // (a bit a row: a table of few rows has no more than a word has bits)
    atomicOr(&any_named, my_named);
    __syncthreads();
    if (threadIdx.x == 0 && blockIdx.y == 0) named[blockIdx.x] = any_named;
  }
  for (int i = threadIdx.x; i < copy; i += blockDim.x) {
    float sum = 0.f;
#pragma unroll 16
    for (int k = 0; k < teams; ++k) sum += copies[k * copy + i];
    const int at = blockIdx.y * LANES * VEC + (i % LANES) * VEC + i / LANES % VEC;
    if (at >= t.channels) continue;
    const size_t e = (size_t)(i / (LANES * VEC)) * t.channels + at;
    if (partial)
      partial[(size_t)blockIdx.x * t.nrows * t.channels + e] = sum;
    else
      out[e] = narrow<T>(sum);
  }
}

// The workgroups' tables, added up: a workgroup takes 64 elements, its waves a share of the tables
// each.
constexpr int kSumWaves = 16;

template <typename O>
__global__ __launch_bounds__(kWave* kSumWaves) void sum_tables_kernel(
    const float* __restrict__ partial, int parts, size_t elements, O* __restrict__ out) {
  __shared__ float sums[kSumWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const size_t e = (size_t)blockIdx.x * kWave + lane;
  const int share = (parts + kSumWaves - 1) / kSumWaves;
  const int end = min(parts, (wave + 1) * share);
  float sum = e < elements ? column_sum(partial, elements, e, wave * share, end) : 0.f;
  sums[wave][lane] = sum;
  lds_barrier();
  if (wave != 0 || e >= elements) return;
  for (int w = 1; w < kSumWaves; ++w) sum += sums[w][lane];
  out[e] = narrow<O>(sum);
}

// ---- any table: the tokens sorted by row ----------------------------------------------------------
//
// Up to kOneLaunchTokens tokens are sorted by one launch (sort_tokens_kernel): a workgroup owns a range
// of rows, reads every index and keeps those of its range.  Every compute unit reads all indices
// then, and the workgroup of a frequent row has most of the placing to do: 7 us for 1,000 tokens and
// 16 us for 16,384 of a vocabulary (131,072 rows).  More tokens are sorted by digits of their row, two
// or three launches for each of 9 bits.  Both give the same order: rows ascending, and the tokens of a
// row as they were.
// (Table gradients of eight floats a row, one launch and digits: 27 and 45 us for 12,000 tokens, 44 and
// 51 us for 32,768.)
constexpr int kOneLaunchTokens = 32768;

// A row of up to kDirect tokens is added up by one team.  Longer ones are cut into pieces that
// start at multiples of their length from the row's start, a multiple of kBlock tokens, so that the
// tokens of a piece and the pieces of a row, which are added up one after the other, stay balanced.
// A piece's sum has slot 2 b + f, where b is the block of kBlock positions of the order that the piece
// starts in and f whether it is its row's first: of a block's positions at most two start pieces, a
// first one (its row then holds the block's last position) and a later one (its row then holds the
// block's first position).
constexpr int kBlock = 16, kDirect = 16;

__device__ __forceinline__ int piece_length(int count) {
  return ((int)(0.5f * sqrtf((float)count)) / kBlock + 1) * kBlock;
}
__device__ __forceinline__ int piece_slot(int from, int length, int j) {
  return (from + j * length) / kBlock * 2 + (j == 0 ? 1 : 0);
}

struct Sorted {
  int32_t* start;   // [nrows + 1]: where a row's tokens begin in order
  int32_t* order;   // [ntokens]; start[nrows] of them have a row
  int32_t* row;     // [ntokens]: the row of the token at a position of order
};

// The one launch: first a workgroup counts its rows' tokens, and the tokens of lower rows, which is
// where its part of the order begins; then it goes again through the steps of 64 tokens that held one
// of its own and writes those in place.  Each of its waves goes through a piece of the tokens of its
// own, with counters of its own, so the order within a row is that of the tokens.
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kSortRange = 960;   // most rows of a workgroup: 60 KB of counters

__device__ __forceinline__ int wave_inclusive_sum(int v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int below = __shfl_up(v, d);
    if (lane >= d) v += below;
  }
  return v;
}

template <typename I>
__global__ __launch_bounds__(kSortThreads) void sort_tokens_kernel(const I* __restrict__ index,
                                                                   uint32_t ntokens, int nrows,
                                                                   int range, Sorted sorted) {
  HIP_DYNAMIC_SHARED(int, count);   // [kSortWaves][range]
  __shared__ int sums[kSortWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int row0 = blockIdx.x * range, rows = min(range, nrows - row0);
  for (int i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) count[i] = 0;
  __syncthreads();
  const uint32_t steps = (ntokens + kSortThreads - 1) / kSortThreads;   // of 64 tokens, for each wave
  const uint32_t begin = wave * steps * kWave;
  const uint32_t end = ntokens < begin + steps * kWave ? ntokens : begin + steps * kWave;
  int* mine = count + wave * range;
  constexpr int kAhead = 8;   // indices of a lane in flight
  const auto fetch = [&](uint32_t n) { return n < end ? table_row(index[n], nrows) : -1; };
  int lower = 0;
  static_assert(kOneLaunchTokens <= 32 * kSortThreads, "a bit for every step");
  uint32_t held = 0;   // steps that have a token of this workgroup's rows
  for (uint32_t s0 = 0; s0 < steps; s0 += kAhead) {
    uint32_t row[kAhead];   // (no row: larger than any)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) row[u] = (uint32_t)fetch(begin + (s0 + u) * kWave + lane);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      lower += row[u] < (uint32_t)row0 ? 1 : 0;
      const uint32_t r = row[u] - (uint32_t)row0, s = s0 + u;
      const bool inside = r < (uint32_t)rows;
      if (__ballot(inside)) {
        if (inside) atomicAdd(&mine[r], 1);
        held |= 1u << s;
      }
    }
  }
  lower = wave_inclusive_sum(lower, lane);
  if (lane == kWave - 1) sums[wave] = lower;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kSortWaves; ++w) base += sums[w];
  __syncthreads();
  // where the tokens of every row, and of every wave in it, begin
  const int r = threadIdx.x;   // (a row a thread: a range has fewer rows than a workgroup threads)
  int total = 0;
  if (r < rows)
    for (int w = 0; w < kSortWaves; ++w) total += count[w * range + r];
  const int through = wave_inclusive_sum(total, lane);
  if (lane == kWave - 1) sums[wave] = through;
  __syncthreads();
  int at = base + through - total;
  for (int w = 0; w < wave; ++w) at += sums[w];
  if (r < rows) {
    sorted.start[row0 + r] = at;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count[w * range + r];
      count[w * range + r] = at;
      at += c;
    }
    if (row0 + r == nrows - 1) sorted.start[nrows] = at;
  }
  __syncthreads();
  const unsigned long long below = (1ull << lane) - 1;
  const auto place = [&](uint32_t n, int row) {
    const int r = row - row0;
    const bool inside = row >= 0 && (uint32_t)r < (uint32_t)rows;
    unsigned long long left = __ballot(inside);
    while (left) {   // one turn for each row among the wave's tokens
      const int first = __builtin_amdgcn_readlane(r, (int)__builtin_ctzll(left));
      const unsigned long long same = __ballot(inside && r == first);
      const int to = mine[first];
      wave_lds_fence();
      if (inside && r == first) {
        const int rank = __popcll(same & below);
        sorted.order[to + rank] = (int32_t)n;
        sorted.row[to + rank] = row;
        if (rank == 0) mine[first] = to + __popcll(same);
      }
      wave_lds_fence();
      left &= ~same;
    }
  };
  constexpr int kTogether = 4;
  while (held) {
    uint32_t n[kTogether];
    int row[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const uint32_t s = held ? (uint32_t)__builtin_ctz(held) : steps;
      held &= held - 1;
      n[u] = begin + s * kWave + lane;
      row[u] = s < steps ? fetch(n[u]) : -1;
    }
#pragma unroll
    for (int u = 0; u < kTogether; ++u) place(n[u], row[u]);
  }
}

// By digits: the tokens of a tile are counted by their digit, then every tile's workgroup works out
// where each of its digits begins from all tiles' counts, ranks its tokens (those of a wave by the
// lanes of equal digit, those of its waves one after the other) and moves them.  FIRST: the rows come
// from the indices; a token without a row gets the row behind the last one.  Every workgroup would read
// the counts of every tile, which grows with the square of the tokens: beyond kMostTilesRead tiles a
// launch between the two sums them over the tiles.  Table gradients of one float a row, 1,000 rows, counts
// read and summed: 524,288 tokens (128 tiles) 64 and 67 us, 1,048,576 108 and 104, 4,194,304 515 and 370,
// 16,777,216 3,810 and 1,350.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits, kTile = 4096, kTileSteps = kTile / kSortThreads;
constexpr int kMostTilesRead = 128;

template <bool FIRST>
__device__ __forceinline__ uint32_t tile_row(const TokenArg& t, const int32_t* rows, uint32_t i) {
  if (!FIRST) return (uint32_t)rows[i];
  const int row = token_row(t, i);
  return row < 0 ? (uint32_t)t.nrows : (uint32_t)row;
}

template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void count_digits_kernel(TokenArg t, const int32_t* __restrict__ rows,
                                                                    int shift, int32_t* __restrict__ counts) {
  __shared__ int count[kDigits];
  for (int i = threadIdx.x; i < kDigits; i += kSortThreads) count[i] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k) {
    const uint32_t i = blockIdx.x * (uint32_t)kTile + k * kSortThreads + threadIdx.x;
    if (i < (uint32_t)t.ntokens) atomicAdd(&count[tile_row<FIRST>(t, rows, i) >> shift & (kDigits - 1)], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kDigits; i += kSortThreads) counts[(size_t)blockIdx.x * kDigits + i] = count[i];
}

// Counts [tiles][kDigits] become those of the tiles before, with the sum over all tiles behind the last: a
// workgroup takes 64 digits, its waves a share of the tiles each.
__global__ __launch_bounds__(kSortThreads) void sum_digits_kernel(int32_t* counts, int tiles) {
  __shared__ int sums[kSortWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int share = (tiles + kSortWaves - 1) / kSortWaves;
  const int begin = min(wave * share, tiles), end = min(begin + share, tiles);
  int32_t* column = counts + blockIdx.x * kWave + lane;
  int sum = 0;
#pragma unroll 16
  for (int k = begin; k < end; ++k) sum += column[(size_t)k * kDigits];
  sums[wave][lane] = sum;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; ++w) before += sums[w][lane];
  constexpr int U = 16;   // loads in flight
  for (int k0 = begin; k0 < end; k0 += U) {
    int count[U];
#pragma unroll
    for (int u = 0; u < U; ++u) count[u] = column[(size_t)min(k0 + u, end - 1) * kDigits];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u >= end) break;
      column[(size_t)(k0 + u) * kDigits] = before;
      before += count[u];
    }
  }
  if (wave == kSortWaves - 1) column[(size_t)tiles * kDigits] = before;
}

// SUMMED: the counts went through sum_digits_kernel.
template <bool FIRST, bool SUMMED>
__global__ __launch_bounds__(kSortThreads) void move_digits_kernel(
    TokenArg t, const int32_t* __restrict__ rows, const int32_t* __restrict__ order, int shift,
    const int32_t* __restrict__ counts, int32_t* __restrict__ to_rows, int32_t* __restrict__ to_order) {
  __shared__ int count[kSortWaves][kDigits];   // of a wave's tokens, then where they go
  __shared__ int totals[2][kDigits], befores[2][kDigits], sums[kSortWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads) (&count[0][0])[i] = 0;
  // the tiles' counts of a digit: all of them, and those of the tiles before this one
  const int digit = threadIdx.x % kDigits, half = threadIdx.x / kDigits;
  int total = 0, before = 0;
  if (SUMMED) {   // (a half of the workgroup one each, the halves are added)
    const int v = counts[(size_t)(half ? gridDim.x : blockIdx.x) * kDigits + digit];
    if (half)
      total = v;
    else
      before = v;
  } else {
#pragma unroll 8
    for (int k = half; k < (int)gridDim.x; k += kSortThreads / kDigits) {
      const int v = counts[(size_t)k * kDigits + digit];
      total += v;
      before += k < (int)blockIdx.x ? v : 0;
    }
  }
  totals[half][digit] = total;
  befores[half][digit] = before;
  uint32_t row[kTileSteps];
  int token[kTileSteps], rank[kTileSteps];
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k) {
    const uint32_t i = blockIdx.x * (uint32_t)kTile + (wave * kTileSteps + k) * kWave + lane;
    const bool there = i < (uint32_t)t.ntokens;
    row[k] = there ? tile_row<FIRST>(t, rows, i) : 0xFFFFFFFFu;
    token[k] = FIRST || !there ? (int)i : order[i];
  }
  __syncthreads();
  const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k) {
    const bool there = row[k] != 0xFFFFFFFFu;
    const int d = row[k] >> shift & (kDigits - 1);
    unsigned long long same = __ballot(there);   // the lanes of this lane's digit
#pragma unroll
    for (int b = 0; b < kDigitBits; ++b) {
      const unsigned long long set = __ballot(d >> b & 1);
      same &= d >> b & 1 ? set : ~set;
    }
    const int at = count[wave][d];
    rank[k] = at + __popcll(same & below);
    wave_lds_fence();
    if (there && (same & below) == 0) count[wave][d] = at + __popcll(same);
    wave_lds_fence();
  }
  __syncthreads();
  int mine = 0;   // threads of the first half: a digit each
  if (half == 0) mine = totals[0][digit] + totals[1][digit];
  const int through = wave_inclusive_sum(mine, lane);
  if (lane == kWave - 1) sums[wave] = through;
  __syncthreads();
  if (half == 0) {
    int at = through - mine + befores[0][digit] + befores[1][digit];
    for (int w = 0; w < wave; ++w) at += sums[w];
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count[w][digit];
      count[w][digit] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k)
    if (row[k] != 0xFFFFFFFFu) {
      const int to = count[wave][row[k] >> shift & (kDigits - 1)] + rank[k];
      to_rows[to] = (int32_t)row[k];
      to_order[to] = token[k];
    }
}

// Where the rows begin, out of the sorted tokens' rows: a thread a position (and one behind the last)
// fills in the rows that begin there, a wave those of a wide gap.
__global__ __launch_bounds__(kThreads) void row_starts_kernel(TokenArg t, Sorted sorted) {
  const int lane = threadIdx.x & (kWave - 1);
  const uint32_t i = blockIdx.x * (uint32_t)kThreads + threadIdx.x, ntokens = (uint32_t)t.ntokens;
  const bool there = i <= ntokens;
  const int from = there && i > 0 ? sorted.row[i - 1] + 1 : 0;   // first row to fill in
  const int to = !there ? 0 : i < ntokens ? sorted.row[i] : t.nrows;
  const bool wide = there && to - from >= 8;
  if (there && !wide)
    for (int r = from; r <= to; ++r) sorted.start[r] = (int32_t)i;
  for (unsigned long long left = __ballot(wide); left; left &= left - 1) {
    const int who = (int)__builtin_ctzll(left);
    const int a = __builtin_amdgcn_readlane(from, who), b = __builtin_amdgcn_readlane(to, who);
    const int at = __builtin_amdgcn_readlane((int)i, who);
    for (int64_t r = (int64_t)a + lane; r <= b; r += kWave) sorted.start[r] = at;
  }
}

// Tokens of a team in flight, and the first ones of order[begin .. end)
constexpr int tokens_ahead(int packs) { return packs == 1 ? 8 : packs <= 4 ? 4 : 2; }
template <int U>
__device__ __forceinline__ void first_tokens(const int32_t* order, int begin, int end, uint32_t (&n)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (begin + u < end) n[u] = (uint32_t)order[begin + u];
}

// Adds channels c0 + ... of the tokens order[begin .. end) to acc, in that order; `n` are the first of
// them.  The next ones are read while the gradients of these are under way.
template <typename T, int VEC, int LANES, int K, bool DROP, int U>
__device__ __forceinline__ void add_tokens(const TokenArg& t, const T* grad, const SumArg& a,
                                           const int32_t* order, int begin, int end, int c0, int lane,
                                           uint64_t seed, uint64_t offset, uint32_t (&n)[U],
                                           float (&acc)[K][VEC]) {
  for (int i0 = begin; i0 < end; i0 += U) {
    RowPacks<T, VEC, K> g[U];
    uint32_t now[U];
    float by[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= end) break;
      now[u] = n[u];
      by[u] = a.scales ? a.scales[n[u]] : a.scale;
      load_row<T, VEC, LANES, K>(grad + (size_t)n[u] * t.channels + c0, t.channels - c0, lane, true, g[u]);
    }
    first_tokens(order, i0 + U, end, n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= end) break;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = g[u].pack[k][i];
        add_token<DROP, VEC>((size_t)now[u] * t.channels + c0 + (k * LANES + lane) * VEC, a, by[u], seed, offset, v,
                             acc[k]);
        one_after_the_other();
      }
    }
  }
}

template <typename O, int VEC, int LANES, int K>
__device__ __forceinline__ void store_row(O* to, int channels, int lane, const float (&v)[K][VEC]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * LANES + lane) * VEC;
    if (c < channels) store_floats<O, VEC>(to + c, v[k]);
  }
}

// The pieces of long rows, a team a slot; tiles of channels along the grid's y.
template <typename T, int VEC, int LANES, int K, bool DROP>
__global__ __launch_bounds__(kThreads) void pieces_kernel(TokenArg t, const T* __restrict__ grad,
                                                          SumArg a, Sorted sorted,
                                                          float* __restrict__ partial) {
  const int lane = threadIdx.x % LANES;
  const int slot = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int block = slot / 2, c0 = blockIdx.y * LANES * K * VEC;
  const int64_t position = (int64_t)block * kBlock + (slot & 1 ? kBlock - 1 : 0);
  if (position >= sorted.start[t.nrows]) return;
  const int row = sorted.row[position], from = sorted.start[row], to = sorted.start[row + 1];
  const int first = block * kBlock, length = piece_length(to - from);
  if (to - from <= kDirect) return;
  // the row's first piece, if it starts in this block, or the one that does, if it is a later one
  const int j = slot & 1 ? 0 : (first - from + length - 1) / length;
  const int begin = from + j * length, end = min(begin + length, to);
  if (slot & 1 ? from < first : j == 0 || begin >= to || begin >= first + kBlock) return;
  uint64_t seed = 0, offset = 0;
  if (DROP) drop_key(a.drop, seed, offset);
  float acc[K][VEC] = {};
  constexpr int U = tokens_ahead(K);
  uint32_t n[U];
  first_tokens(sorted.order, begin, end, n);
  add_tokens<T, VEC, LANES, K, DROP, U>(t, grad, a, sorted.order, begin, end, c0, lane, seed, offset, n, acc);
  store_row<float, VEC, LANES, K>(partial + (size_t)slot * t.channels + c0, t.channels - c0, lane, acc);
}

// What a row's sum goes through when the vectors were normed rows of the scaled table
struct TableNorm {
  const void* table;
  float scale;
  NormArg norm;
  bool to_table, to_params;
  ParamSums params;
};

// Every row of the table: the sum of its tokens, or of its pieces; tiles of channels along the
// grid's y.  65,536 tokens into 131,072 rows of 4,096 bfloat16: 273 us (1.07 GB written, 0.27 GB read:
// 4.9 TB/s), and 81 us for the pieces (0.27 GB); with NORM, 32,768 tokens into 32,000 rows of 2,048:
// 80 and 30 us, bound by the waits of one row after the other.  One row that holds all of 204,000 tokens
// (28 floats): 58 us for its 900 pieces, and 118 for the team that adds them up.  What the next rows need is
// read ahead: their bounds two rows, their first tokens one.
// NORM: the sum is the gradient of the row's normed vector, which is taken back through the norm
// while it is here (a team then holds the whole row); the workgroups stay, and their teams' shares
// of the gradients of weight and bias are added up at the end.
constexpr int rows_waves(int elements, bool norm) {   // a SIMD should hold
  return elements <= 8 ? 4 : elements <= 16 && !norm ? 4 : norm && elements > 16 ? 1 : 2;
}
template <typename T, typename O, int VEC, int LANES, int K, bool DROP, bool NORM>
__global__ __launch_bounds__((TeamShape<LANES, K>::THREADS), (rows_waves(K * VEC, NORM))) void rows_kernel(
    TokenArg t, const T* __restrict__ grad, SumArg a, Sorted sorted,
    const float* __restrict__ partial, O* __restrict__ out, TableNorm norm) {
  using Shape = TeamShape<LANES, K>;
  __shared__ float slots[3][2 * Shape::WAVES];
  HIP_DYNAMIC_SHARED(float, param_sums);
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const int c0 = NORM ? 0 : blockIdx.y * LANES * K * VEC, channels = t.channels - c0;
  const uint32_t nrows = (uint32_t)t.nrows, step = gridDim.x * Shape::TEAMS;
  uint64_t seed = 0, offset = 0;
  if (DROP) drop_key(a.drop, seed, offset);
  float w[K][VEC], dw[K][VEC], db[K][VEC];
  if (NORM) {
    load_param<T, VEC, LANES, K>(norm.norm.weight, norm.params.is_float, 1.f, channels, lane, w);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) dw[k][i] = db[k][i] = 0.f;
  }
  constexpr int U = NORM ? (K == 1 ? 3 : 2) : K <= 2 ? 4 : 2;   // most rows have a token or two
  const auto bounds = [&](uint32_t row, int& from, int& to) {
    from = row < nrows ? sorted.start[row] : 0;
    to = row < nrows ? sorted.start[row + 1] : 0;
  };
  int from1, to1, from2, to2;   // of the next row and the one after it
  uint32_t n1[U];
  const uint32_t mine = blockIdx.x * Shape::TEAMS + team;
  bounds(mine, from1, to1);
  bounds(mine + step, from2, to2);
  first_tokens(sorted.order, from1, to1, n1);
  for (uint32_t row0 = blockIdx.x * Shape::TEAMS; row0 < nrows; row0 += step) {
    const uint32_t row = row0 + team;
    const int from = from1, to = to1;
    uint32_t n[U];
#pragma unroll
    for (int u = 0; u < U; ++u) n[u] = n1[u];
    from1 = from2;
    to1 = to2;
    first_tokens(sorted.order, from1, to1, n1);
    bounds(row + 2 * step, from2, to2);
    const bool some = to > from;
    float v[K][VEC] = {};
    RowPacks<T, VEC, K> x;
    if (NORM && some)
      load_row<T, VEC, LANES, K>(static_cast<const T*>(norm.table) + (size_t)row * channels, channels, lane, true, x);
    if (to - from <= kDirect) {
      add_tokens<T, VEC, LANES, K, DROP, U>(t, grad, a, sorted.order, from, to, c0, lane, seed, offset, n, v);
    } else {
      const int length = piece_length(to - from), pieces = (to - from + length - 1) / length;
      constexpr int P = K == 1 ? (NORM ? 3 : 4) : 2;   // pieces in flight
      for (int j0 = 0; j0 < pieces; j0 += P) {
        RowPacks<float, VEC, K> p[P];
#pragma unroll
        for (int u = 0; u < P; ++u) {
          if (j0 + u >= pieces) break;
          load_row<float, VEC, LANES, K>(partial + (size_t)piece_slot(from, length, j0 + u) * t.channels + c0,
                                         channels, lane, true, p[u]);
        }
#pragma unroll
        for (int u = 0; u < P; ++u) {
          if (j0 + u >= pieces) break;
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[k][i] += p[u].pack[k][i];
        }
      }
    }
    // (all teams of a wave come along, and a team of several waves is a workgroup)
    if (NORM && __ballot(some)) {
      float h[K][VEC];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[k][i] = some ? norm.scale * x.pack[k][i] : 0.f;
      float mean, rstd;
      team_stats<VEC, LANES, K>(h, channels, lane, norm.norm.eps, slots[0], slots[1], mean, rstd);
      float both[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          h[k][i] *= rstd;
          const float q = v[k][i] * w[k][i];
          both[0] += q;
          both[1] = fmaf(q, h[k][i], both[1]);
          if (some) dw[k][i] = fmaf(v[k][i], h[k][i], dw[k][i]);
          db[k][i] += v[k][i];
        }
      team_sums<LANES>(both, slots[2]);
      const float mean_q = both[0] / channels, mean_qh = both[1] / channels;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          v[k][i] = some ? norm.scale * rstd * (v[k][i] * w[k][i] - mean_q - h[k][i] * mean_qh) : 0.f;
    }
    if (row < nrows && (!NORM || norm.to_table))
      store_row<O, VEC, LANES, K>(out + (size_t)row * t.channels + c0, channels, lane, v);
  }
  if (NORM && norm.to_params) add_up_params<T, VEC, LANES, K>(dw, db, lane, channels, param_sums, norm.params);
}

// ---- launches -------------------------------------------------------------------------------------
unsigned at_most(size_t blocks, size_t most) { return (unsigned)(blocks < most ? (blocks ? blocks : 1) : most); }

// The lanes of a team for rows of `packs` packs where wider rows are gone through in steps
template <int VEC, typename F>
void with_lanes(int packs, F f) {
  if constexpr (VEC > 1) {
    if (packs <= 4) return f(std::integral_constant<int, 4>());
    if (packs <= 8) return f(std::integral_constant<int, 8>());
    if (packs > 16 && packs <= 32) return f(std::integral_constant<int, 32>());
  }
  if (packs <= 16) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 64>());
}
template <typename T, typename F>
void with_packs_of(int channels, uintptr_t where, F f) {
  if (whole_packs<T>(channels, where))
    f(std::integral_constant<int, 16 / (int)sizeof(T)>());
  else
    f(std::integral_constant<int, 1>());
}

template <typename T>
hipError_t embed(const TokenArg& t, const void* table, float scale, const float* scales, void* out,
                 hipStream_t stream) {
  with_packs_of<T>(t.channels, address(table) | address(out), [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    with_lanes<VEC>(t.channels / VEC, [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      const size_t blocks = ((size_t)t.ntokens * LANES + kThreads - 1) / kThreads;
      if (t.channels <= LANES * VEC)
        hipLaunchKernelGGL((embed_narrow_kernel<T, VEC, LANES>), dim3(at_most((blocks + kTokens - 1) / kTokens, kResident)),
                           dim3(kThreads), 0, stream, t, (const T*)table, scale, scales, (T*)out);
      else
        hipLaunchKernelGGL((embed_kernel<T, VEC>), dim3(at_most(blocks, kResident)), dim3(kThreads), 0, stream, t,
                           (const T*)table, scale, scales, (T*)out);
    });
  });
  return hipGetLastError();
}

template <typename T>
hipError_t scale_gradient(const TokenArg& t, const void* grad, const void* table, float* out,
                          hipStream_t stream) {
  with_packs_of<T>(t.channels, address(table) | address(grad), [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    with_lanes<VEC>(t.channels / VEC, [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      const size_t blocks = ((size_t)t.ntokens * LANES + kThreads - 1) / kThreads;
      hipLaunchKernelGGL((scale_gradient_kernel<T, VEC, LANES>), dim3(at_most(blocks, kResident)),
                         dim3(kThreads), 0, stream, t, (const T*)grad, (const T*)table, out);
    });
  });
  return hipGetLastError();
}

size_t round_up(size_t bytes) { return (bytes + 255) / 256 * 256; }

// How the few-row kernel shares the tokens out.  It is for tables of up to kFewRows rows, where a
// wave's copies fit the LDS of a workgroup.
constexpr int kFewRows = 32;
constexpr int kFewRowsParts = 512;   // two workgroups on each of 256 CUs
struct FewRowsPlan {
  int waves, share, parts;
};
FewRowsPlan few_rows_plan(int ntokens, int nrows, int vec, int lanes, int column_blocks) {
  FewRowsPlan p;
  const int wave_bytes = 256 * nrows * vec;
  p.waves = kTableLds / wave_bytes;
  if (p.waves > kThreads / kWave) p.waves = kThreads / kWave;
  if (p.waves < 1) p.waves = 1;
  const int teams = p.waves * kWave / lanes;
  // kFewRowsParts workgroups, but no fewer than two rounds of loads for each
  size_t share = ((size_t)ntokens * column_blocks + kFewRowsParts - 1) / kFewRowsParts;
  const size_t least = (size_t)teams * kTableUnroll * 2;
  if (share < least) share = least;
  if (share > (size_t)ntokens) share = ntokens;
  p.share = (int)share;
  p.parts = (int)(((size_t)ntokens + share - 1) / share);
  return p;
}
size_t few_rows_bytes(int ntokens, int nrows, int channels) {
  // (the smallest share is that of one team)
  size_t parts = ((size_t)ntokens + 2 * kTableUnroll - 1) / (2 * kTableUnroll);
  if (parts > kFewRowsParts) parts = kFewRowsParts;
  return round_up(parts * nrows * channels * sizeof(float));
}

// Whether the copies are the better way: where the workgroups' tables, which are written and read
// again, are no more than two thirds of the gradient, or a single one is enough.  Sums alone, copies
// and sorted: 204,000 tokens, 28 rows of 28 floats 17 and 56 us, 30,000 x 28 x 256 floats 28 and 45
// us, 2,000 x 28 x 32 bfloat16 14 and 15 us; but 2,000 x 28 x 256 floats 21 and 15 us, 20,000 x 32 x
// 512 bfloat16 66 and 33 us, 2,000 x 28 x 2,048 bfloat16 57 and 16 us.
template <typename T>
bool copies_pay(const TokenArg& t, const void* grad) {
  if (t.nrows > kFewRows) return false;
  bool pay = false;
  with_packs_of<T>(t.channels, address(grad), [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    with_lanes<VEC>(t.channels / VEC, [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      const FewRowsPlan p = few_rows_plan(t.ntokens, t.nrows, VEC, LANES,
                                          (t.channels + LANES * VEC - 1) / (LANES * VEC));
      pay = p.parts == 1 || (size_t)3 * t.nrows * sizeof(float) <= (size_t)2 * p.share * sizeof(T);
    });
  });
  return pay;
}

struct SortedLayout {
  size_t order, row, other_order, other_row, counts, partial, bytes;   // offsets; start is first
  int slots, tiles;
};
SortedLayout sorted_layout(int ntokens, int nrows, int channels) {
  SortedLayout l;
  l.slots = ntokens > kDirect ? (ntokens + kBlock - 1) / kBlock * 2 : 0;
  l.tiles = ntokens > kOneLaunchTokens ? (ntokens + kTile - 1) / kTile : 0;
  const size_t list = round_up((size_t)ntokens * sizeof(int32_t));
  l.order = round_up(((size_t)nrows + 1) * sizeof(int32_t));
  l.row = l.order + list;
  l.other_order = l.row + list;
  l.other_row = l.other_order + (l.tiles ? list : 0);
  l.counts = l.other_row + (l.tiles ? list : 0);
  l.partial = l.counts + round_up(((size_t)l.tiles + (l.tiles > kMostTilesRead)) * kDigits * sizeof(int32_t));
  l.bytes = l.partial + round_up((size_t)l.slots * channels * sizeof(float));
  return l;
}

// scales_done: whether the gradients of the scales (if any are wanted) came out as well.  named: where
// the rows that tokens name are written down, a word of bits for each of the workgroups.
template <typename T, typename O, bool DROP>
hipError_t few_rows(const TokenArg& t, const void* grad, const SumArg& a, const void* table, float* grad_scales,
                    bool* scales_done, void* out, float* partial, NamedRows* named, hipStream_t stream) {
  with_packs_of<T>(t.channels, address(grad), [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    with_lanes<VEC>(t.channels / VEC, [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      const int column_blocks = (t.channels + LANES * VEC - 1) / (LANES * VEC);
      const FewRowsPlan p = few_rows_plan(t.ntokens, t.nrows, VEC, LANES, column_blocks);
      const bool direct = p.parts == 1 && std::is_same<T, O>::value;
      const size_t copies = (size_t)p.waves * 256 * t.nrows * VEC;
      const size_t own = (size_t)t.nrows * VEC * LANES * sizeof(float);
      const dim3 grid(p.parts, column_blocks), block(p.waves * kWave);
      uint32_t* words = named ? const_cast<uint32_t*>(named->words) : nullptr;
      if (named) named->count = p.parts;
      if (!DROP && grad_scales && column_blocks == 1 && copies + own <= kTableLds) {
        if (scales_done) *scales_done = true;
        hipLaunchKernelGGL((few_rows_kernel<T, VEC, LANES, DROP, !DROP>), grid, block, copies + own, stream, t,
                           (const T*)grad, a, p.share, (const T*)table, grad_scales, direct ? (T*)out : nullptr,
                           direct ? nullptr : partial, words);
      } else {
        hipLaunchKernelGGL((few_rows_kernel<T, VEC, LANES, DROP, false>), grid, block, copies, stream, t,
                           (const T*)grad, a, p.share, (const T*)table, grad_scales, direct ? (T*)out : nullptr,
                           direct ? nullptr : partial, words);
      }
      if (direct) return;
      const size_t elements = (size_t)t.nrows * t.channels;
      hipLaunchKernelGGL((sum_tables_kernel<O>), dim3((unsigned)((elements + kWave - 1) / kWave)),
                         dim3(kWave * kSumWaves), 0, stream, partial, p.parts, elements, (O*)out);
    });
  });
  return hipGetLastError();
}

Sorted sort_tokens(const TokenArg& t, const SortedLayout& l, char* base, hipStream_t stream) {
  const auto list = [&](size_t at) { return reinterpret_cast<int32_t*>(base + at); };
  const Sorted sorted{list(0), list(l.order), list(l.row)};
  if (l.tiles) {
    int passes = 1;   // digits of 0 .. nrows
    while (passes < 4 && (uint32_t)t.nrows >> (passes * kDigitBits)) ++passes;
    const Sorted other{nullptr, list(l.other_order), list(l.other_row)};
    for (int p = 0; p < passes; ++p) {
      const bool last = (passes - 1 - p) % 2 == 0;   // the last pass ends in `sorted`
      const Sorted &to = last ? sorted : other, &from = last ? other : sorted;
      const auto pass = [&](auto first, const int32_t* rows, const int32_t* order) {
        constexpr bool FIRST = decltype(first)::value;
        const dim3 grid(l.tiles), block(kSortThreads);
        int32_t* counts = list(l.counts);
        hipLaunchKernelGGL(count_digits_kernel<FIRST>, grid, block, 0, stream, t, rows, p * kDigitBits, counts);
        if (l.tiles > kMostTilesRead) {
          hipLaunchKernelGGL(sum_digits_kernel, dim3(kDigits / kWave), block, 0, stream, counts, l.tiles);
          hipLaunchKernelGGL((move_digits_kernel<FIRST, true>), grid, block, 0, stream, t, rows, order, p * kDigitBits,
                             counts, to.row, to.order);
        } else {
          hipLaunchKernelGGL((move_digits_kernel<FIRST, false>), grid, block, 0, stream, t, rows, order, p * kDigitBits,
                             counts, to.row, to.order);
        }
      };
      if (p == 0)
        pass(std::true_type(), nullptr, nullptr);
      else
        pass(std::false_type(), from.row, from.order);
    }
    hipLaunchKernelGGL(row_starts_kernel, dim3(((unsigned)t.ntokens + kThreads) / kThreads), dim3(kThreads), 0,
                       stream, t, sorted);
    return sorted;
  }
  int range = (t.nrows + 255) / 256;
  if (range > kSortRange) range = kSortRange;
  const dim3 grid((t.nrows + range - 1) / range), block(kSortThreads);
  const size_t shared = (size_t)kSortWaves * range * sizeof(int);
  if (t.index_kind == MG_INDEX_FLOAT32)
    hipLaunchKernelGGL(sort_tokens_kernel<float>, grid, block, shared, stream, (const float*)t.index,
                       (uint32_t)t.ntokens, t.nrows, range, sorted);
  else if (t.index_kind == MG_INDEX_INT32)
    hipLaunchKernelGGL(sort_tokens_kernel<int32_t>, grid, block, shared, stream, (const int32_t*)t.index,
                       (uint32_t)t.ntokens, t.nrows, range, sorted);
  else
    hipLaunchKernelGGL(sort_tokens_kernel<int64_t>, grid, block, shared, stream, (const int64_t*)t.index,
                       (uint32_t)t.ntokens, t.nrows, range, sorted);
  return sorted;
}

// Workgroups of rows_kernel that stay, for the sums over all rows
constexpr int kRowParts = 1024;

// The sums by row of a table of more than kFewRows rows, or (NORM) what follows from them.
template <typename T, typename O, bool DROP, bool NORM>
hipError_t sorted_rows(const TokenArg& t, const void* grad, const SumArg& a, void* out, void* workspace,
                       const TableNorm& norm, hipStream_t stream) {
  const SortedLayout l = sorted_layout(t.ntokens, t.nrows, t.channels);
  char* base = static_cast<char*>(workspace);
  float* partial = reinterpret_cast<float*>(base + l.partial);
  const Sorted sorted = sort_tokens(t, l, base, stream);
  int parts = 0;
  with_packs_of<T>(t.channels, address(grad) | address(out) | address(NORM ? norm.table : nullptr), [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    const int packs = (t.channels + VEC - 1) / VEC;
    const auto tiles = [&](auto shape) {
      using S = decltype(shape);
      return (unsigned)((packs + S::LANES * S::K - 1) / (S::LANES * S::K));
    };
    if (l.slots)
      with_tile<VEC, VEC == 1 ? 4 : 1>(packs, [&](auto shape) {
        using S = decltype(shape);
        hipLaunchKernelGGL((pieces_kernel<T, VEC, S::LANES, S::K, DROP>),
                           dim3((l.slots + S::TEAMS - 1) / S::TEAMS, tiles(shape)), dim3(kThreads), 0, stream, t,
                           (const T*)grad, a, sorted, partial);
      });
    const auto rows = [&](auto shape, size_t most, unsigned y) {
      using S = decltype(shape);
      parts = (int)at_most(((size_t)t.nrows + S::TEAMS - 1) / S::TEAMS, most);
      const size_t shared = NORM && S::LANES <= kWave ? (size_t)2 * t.channels * sizeof(float) : 0;
      hipLaunchKernelGGL((rows_kernel<T, O, VEC, S::LANES, S::K, DROP, NORM>), dim3(parts, y), dim3(S::THREADS),
                         shared, stream, t, (const T*)grad, a, sorted, partial, (O*)out, norm);
    };
    if constexpr (NORM)
      with_team<VEC>(packs, [&](auto shape) { rows(shape, kRowParts, 1); });
    else
      with_tile<VEC, 4>(packs, [&](auto shape) { rows(shape, kResident, tiles(shape)); });
  });
  if (NORM && norm.to_params && parts > 1)
    return launch_sum_partials(norm.norm, norm.params.partial, parts, norm.params.weight, norm.params.bias,
                               stream);
  return hipGetLastError();
}

// A table that no token can name a row of
template <typename O>
__global__ __launch_bounds__(kThreads) void zero_kernel(O* out, size_t n) {
  for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (size_t)gridDim.x * kThreads)
    out[i] = narrow<O>(0.f);
}
template <typename O>
hipError_t zero(void* out, size_t n, hipStream_t stream) {
  hipLaunchKernelGGL((zero_kernel<O>), dim3(at_most((n + kThreads - 1) / kThreads, kResident)), dim3(kThreads), 0,
                     stream, (O*)out, n);
  return hipGetLastError();
}

}  // namespace

#define MG_FOR_TYPE(dtype, FN)                \
  switch (dtype) {                            \
    case MG_FLOAT32: return FN(float);        \
    case MG_FLOAT16: return FN(Half);         \
    case MG_BFLOAT16: return FN(Bfloat16);    \
  }                                           \
  return hipErrorInvalidValue

size_t embed_backward_workspace_bytes(int ntokens, int nrows, int channels) {
  // (whichever way is taken: that depends on the type and alignment of the call's arrays)
  const size_t few = nrows <= kFewRows ? few_rows_bytes(ntokens, nrows, channels) : 0;
  const size_t sorted = sorted_layout(ntokens, nrows, channels).bytes;
  return few > sorted ? few : sorted;
}

hipError_t launch_embed(const TokenArg& t, const void* table, float scale, const float* scales,
                        void* out, hipStream_t stream) {
#define MG_CALL(T) embed<T>(t, table, scale, scales, out, stream)
  MG_FOR_TYPE(t.dtype, MG_CALL);
#undef MG_CALL
}

namespace {
template <typename T>
hipError_t embed_backward(const TokenArg& t, const void* grad, const void* table, const SumArg& a,
                          void* grad_table, float* grad_scales, void* workspace, hipStream_t stream) {
  hipError_t e = hipSuccess;
  bool scales_done = false;
  if (grad_table && t.nrows > 0 && t.channels > 0)
    e = t.ntokens == 0 ? zero<T>(grad_table, (size_t)t.nrows * t.channels, stream)
        : copies_pay<T>(t, grad)
            ? few_rows<T, T, false>(t, grad, a, table, grad_scales, &scales_done, grad_table, (float*)workspace, nullptr,
                                    stream)
            : sorted_rows<T, T, false, false>(t, grad, a, grad_table, workspace, TableNorm(), stream);
  if (e != hipSuccess || !grad_scales || t.ntokens == 0 || scales_done) return e;
  return scale_gradient<T>(t, grad, table, grad_scales, stream);
}
}  // namespace

hipError_t launch_embed_backward(const TokenArg& t, const void* grad, const void* table, float scale,
                                 const float* scales, void* grad_table, float* grad_scales,
                                 void* workspace, hipStream_t stream) {
  const SumArg a{scale, scales, DropArg()};
#define MG_CALL(T) embed_backward<T>(t, grad, table, a, grad_table, grad_scales, workspace, stream)
  MG_FOR_TYPE(t.dtype, MG_CALL);
#undef MG_CALL
}

// encode's backward pass: rows in teams are summed and normed back in one launch; otherwise the sums
// of all rows go through memory (first in the workspace), and layer_norm.hip takes them back.
namespace {
struct EncodeLayout {
  size_t params, named, rest, bytes;   // offsets: partial sums of weight and bias, bits of the rows that
                                       // tokens name, workspace of the row sums
};
EncodeLayout encode_layout(int ntokens, int nrows, int channels, bool in_memory) {
  EncodeLayout l;
  l.params = in_memory ? round_up((size_t)nrows * channels * sizeof(float)) : 0;
  l.named = l.params + round_up(in_memory
                                    ? norm_backward_workspace_bytes(nrows, channels)
                                    : (size_t)(nrows < kRowParts ? nrows : kRowParts) * 2 * channels * sizeof(float));
  l.rest = l.named + (nrows <= kFewRows ? kFewRowsParts * sizeof(uint32_t) : 0);
  l.bytes = l.rest + (ntokens ? embed_backward_workspace_bytes(ntokens, nrows, channels) : 0);
  return l;
}
template <typename T>
hipError_t encode_backward(const TokenArg& t, const NormArg& n, const void* grad, const void* table, float scale,
                           const DropArg& drop, void* grad_table, void* grad_weight, void* grad_bias,
                           char* workspace, hipStream_t stream) {
  const bool copies = t.ntokens > 0 && t.nrows > 0 && copies_pay<T>(t, grad);
  const bool in_memory = t.ntokens == 0 || t.nrows == 0 || copies || t.channels > kMostTeamChannels;
  const EncodeLayout l = encode_layout(t.ntokens, t.nrows, t.channels, in_memory);
  const SumArg a{1.f, nullptr, drop};
  float* params = reinterpret_cast<float*>(workspace + l.params);
  if (!in_memory) {
    const TableNorm norm{table, scale, n, grad_table != nullptr, grad_weight || grad_bias,
                         {params, grad_weight, grad_bias, n.param_dtype == MG_FLOAT32}};
    return sorted_rows<T, T, true, true>(t, grad, a, grad_table, workspace + l.rest, norm, stream);
  }
  float* sums = reinterpret_cast<float*>(workspace);
  // which rows tokens name: the others have no part in the gradients, whatever stands in them
  NamedRows named{reinterpret_cast<uint32_t*>(workspace + l.named), 0, nullptr};
  if (!copies && t.ntokens > 0 && t.nrows > 0) named = NamedRows{nullptr, 0, reinterpret_cast<int32_t*>(workspace + l.rest)};
  hipError_t e = t.nrows == 0 ? hipSuccess
                 : t.ntokens == 0 ? zero<float>(sums, (size_t)t.nrows * t.channels, stream)
                 : copies
                     ? few_rows<T, float, true>(t, grad, a, nullptr, nullptr, nullptr, sums, (float*)(workspace + l.rest),
                                                &named, stream)
                     : sorted_rows<T, float, true, false>(t, grad, a, sums, workspace + l.rest, TableNorm(), stream);
  if (e != hipSuccess) return e;
  return launch_table_norm_backward(n, sums, table, scale, named, grad_table, grad_weight, grad_bias, params, stream);
}
}  // namespace

size_t encode_backward_workspace_bytes(int ntokens, int nrows, int channels) {
  const bool wide = channels > kMostTeamChannels;   // (whichever ways a call of these sizes can take)
  const size_t in_memory =
      ntokens == 0 || nrows <= kFewRows || wide ? encode_layout(ntokens, nrows, channels, true).bytes : 0;
  const size_t other = ntokens == 0 || wide ? 0 : encode_layout(ntokens, nrows, channels, false).bytes;
  return in_memory > other ? in_memory : other;
}
hipError_t launch_encode_backward(const TokenArg& t, const NormArg& a, const void* grad, const void* table,
                                  float scale, const DropArg& drop, void* grad_table, void* grad_weight,
                                  void* grad_bias, void* workspace, hipStream_t stream) {
#define MG_CALL(T) \
  encode_backward<T>(t, a, grad, table, scale, drop, grad_table, grad_weight, grad_bias, (char*)workspace, stream)
  MG_FOR_TYPE(t.dtype, MG_CALL);
#undef MG_CALL
}

}  // namespace mg
