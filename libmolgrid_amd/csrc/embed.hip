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

// A team takes one token at a time; the index of its next token is read ahead.
template <typename T, int VEC, int LANES>
__global__ __launch_bounds__(kThreads) void embed_kernel(TokenArg t, const T* __restrict__ table,
                                                         float scale,
                                                         const float* __restrict__ scales,
                                                         T* __restrict__ out) {
  constexpr int kTeams = kThreads / LANES, kUnroll = 4;
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
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int c = c0 + u * LANES * VEC;
        if (at >= 0 && c < t.channels)
          load_floats<T, VEC>(from + c, v[u]);
        else
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[u][i] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int c = c0 + u * LANES * VEC;
        if (c >= t.channels) break;
        // (a row that is not there is zero whatever the scale is)
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[u][i] = at < 0 ? 0.f : by * v[u][i];
        store_floats<T, VEC>(to + c, v[u]);
      }
    }
  }
}

// ds: a team takes one token at a time.
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

template <typename T, int VEC, int LANES, bool DROP>
__global__ __launch_bounds__(kThreads) void few_rows_kernel(TokenArg t, const T* __restrict__ grad,
                                                            SumArg a, int share, T* out,
                                                            float* partial) {
  HIP_DYNAMIC_SHARED(float, copies);
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const int teams = blockDim.x / LANES;
  const int copy = t.nrows * VEC * LANES;
  float* mine = copies + team * copy + lane;
  for (int i = 0; i < t.nrows * VEC; ++i) mine[i * LANES] = 0.f;
  uint64_t seed = 0, offset = 0;
  if (DROP) drop_key(a.drop, seed, offset);
  const int c = (blockIdx.y * LANES + lane) * VEC;
  const uint32_t begin = blockIdx.x * (uint32_t)share;
  const uint32_t end = min(begin + (uint32_t)share, (uint32_t)t.ntokens);
  if (c < t.channels)
    for (uint32_t n0 = begin + team; n0 < end; n0 += teams * kTableUnroll) {
      int row[kTableUnroll];
      float by[kTableUnroll], g[kTableUnroll][VEC];
#pragma unroll
      for (int u = 0; u < kTableUnroll; ++u) {
        const uint32_t n = n0 + u * teams;
        row[u] = n < end ? token_row(t, n) : -1;
        by[u] = a.scales && n < end ? a.scales[n] : a.scale;
        if (n < end) load_floats<T, VEC>(grad + (size_t)n * t.channels + c, g[u]);
      }
#pragma unroll
      for (int u = 0; u < kTableUnroll; ++u) {
        if (row[u] < 0) continue;
        float sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = mine[(row[u] * VEC + i) * LANES];
        add_token<DROP, VEC>((size_t)(n0 + u * teams) * t.channels + c, a, by[u], seed, offset, g[u], sum);
#pragma unroll
        for (int i = 0; i < VEC; ++i) mine[(row[u] * VEC + i) * LANES] = sum[i];
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < copy; i += blockDim.x) {
    float sum = 0.f;
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
  float sum = 0.f;
  if (e < elements)
#pragma unroll 8
    for (int i = wave * share; i < end; ++i) sum += partial[(size_t)i * elements + e];
  sums[wave][lane] = sum;
  lds_barrier();
  if (wave != 0 || e >= elements) return;
  for (int w = 1; w < kSumWaves; ++w) sum += sums[w][lane];
  out[e] = narrow<O>(sum);
}

// ---- any table: the tokens sorted by row ----------------------------------------------------------
//
// One launch sorts: a workgroup owns a range of rows, reads every index twice and keeps those of its
// range.  First it counts its rows' tokens, and the tokens of lower rows, which is where its part of
// the order begins; then it writes its tokens in place.  Each of its waves goes through a piece of
// the tokens of its own, with counters of its own, so the order within a row is that of the
// tokens.  All workgroups read all indices (out of the L2 after the first), which costs less than
// the launches of a sort by digits for up to about 2^18 tokens.
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

__global__ __launch_bounds__(kSortThreads) void sort_tokens_kernel(TokenArg t, int range,
                                                                   int32_t* __restrict__ start,
                                                                   int32_t* __restrict__ order) {
  HIP_DYNAMIC_SHARED(int, count);   // [kSortWaves][range]
  __shared__ int sums[kSortWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int row0 = blockIdx.x * range, rows = min(range, t.nrows - row0);
  for (int i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) count[i] = 0;
  __syncthreads();
  const uint32_t ntokens = (uint32_t)t.ntokens;
  const uint32_t piece = (ntokens + kSortThreads - 1) / kSortThreads * kWave;
  const uint32_t begin = wave * piece, end = min(begin + piece, ntokens);
  int* mine = count + wave * range;
  constexpr int kAhead = 8;   // indices of a lane in flight
  int lower = 0;
  for (uint32_t n0 = begin; n0 < end; n0 += kAhead * kWave) {
    int row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t n = n0 + u * kWave + lane;
      row[u] = n < end ? token_row(t, n) : -1;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      lower += row[u] >= 0 && row[u] < row0 ? 1 : 0;
      const int r = row[u] - row0;
      if (row[u] >= row0 && r < rows) atomicAdd(&mine[r], 1);
    }
  }
  lower = wave_inclusive_sum(lower, lane);
  if (lane == kWave - 1) sums[wave] = lower;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kSortWaves; ++w) base += sums[w];
  __syncthreads();
  // where the tokens of every row, and of every wave in it, begin
  const int per_thread = (range + kSortThreads - 1) / kSortThreads;
  const int r0 = threadIdx.x * per_thread, r1 = min(r0 + per_thread, rows);
  int total = 0;
  for (int r = r0; r < r1; ++r)
    for (int w = 0; w < kSortWaves; ++w) total += count[w * range + r];
  const int through = wave_inclusive_sum(total, lane);
  if (lane == kWave - 1) sums[wave] = through;
  __syncthreads();
  int at = base + through - total;
  for (int w = 0; w < wave; ++w) at += sums[w];
  for (int r = r0; r < r1; ++r) {
    start[row0 + r] = at;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count[w * range + r];
      count[w * range + r] = at;
      at += c;
    }
    if (row0 + r == t.nrows - 1) start[t.nrows] = at;
  }
  __syncthreads();
  const unsigned long long below = (1ull << lane) - 1;
  for (uint32_t n0 = begin; n0 < end; n0 += kAhead * kWave) {
    int row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t n = n0 + u * kWave + lane;
      row[u] = n < end ? token_row(t, n) : -1;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int r = row[u] - row0;
      const bool inside = row[u] >= row0 && r < rows;
      unsigned long long left = __ballot(inside);
      while (left) {   // one turn for each row among the wave's tokens
        const int first = __builtin_amdgcn_readlane(r, (int)__builtin_ctzll(left));
        const unsigned long long same = __ballot(inside && r == first);
        const int to = mine[first];
        wave_lds_fence();
        if (inside && r == first) {
          const int rank = __popcll(same & below);
          order[to + rank] = (int32_t)(n0 + u * kWave + lane);
          if (rank == 0) mine[first] = to + __popcll(same);
        }
        wave_lds_fence();
        left &= ~same;
      }
    }
  }
}

// Tokens of a row that one team adds; rows of more are cut where the order's multiples of it are.
constexpr int kPiece = 128;

struct Sorted {
  const int32_t* start;   // [nrows + 1]: where a row's tokens begin in order
  const int32_t* order;
};

// Adds the tokens order[begin .. end) to acc, in that order.
template <typename T, int VEC, int LANES, int K, bool DROP>
__device__ __forceinline__ void add_tokens(const TokenArg& t, const T* grad, const SumArg& a,
                                           const int32_t* order, int begin, int end, int lane,
                                           uint64_t seed, uint64_t offset, float (&acc)[K][VEC]) {
  constexpr int kAhead = K * VEC <= 8 ? 4 : 2;
  for (int i0 = begin; i0 < end; i0 += kAhead) {
    RowPacks<T, VEC, K> g[kAhead];
    uint32_t n[kAhead];
    float by[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool live = i0 + u < end;
      n[u] = live ? (uint32_t)order[i0 + u] : 0;
      by[u] = !live ? 0.f : a.scales ? a.scales[n[u]] : a.scale;
      load_row<T, VEC, LANES, K>(grad + (size_t)n[u] * t.channels, t.channels, lane, live, g[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u >= end) break;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = widen(g[u].pack[k].v[i]);
        add_token<DROP, VEC>((size_t)n[u] * t.channels + (k * LANES + lane) * VEC, a, by[u], seed, offset, v,
                             acc[k]);
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

// The first `piece_blocks` workgroups take pieces of long rows, whose sums go to `partial`
// (piece i: the row that its first token is of, then the row that its last one is of), the others
// rows.
template <typename T, typename O, int VEC, int LANES, int K, bool DROP>
__global__ __launch_bounds__((TeamShape<LANES, K>::THREADS)) void sorted_rows_kernel(
    TokenArg t, const T* __restrict__ grad, SumArg a, Sorted sorted, int piece_blocks,
    O* __restrict__ out, float* __restrict__ partial) {
  using Shape = TeamShape<LANES, K>;
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  uint64_t seed = 0, offset = 0;
  if (DROP) drop_key(a.drop, seed, offset);
  const int blocks = gridDim.x - piece_blocks;
  if ((int)blockIdx.x < piece_blocks) {
    const int total = sorted.start[t.nrows];
    const int i = blockIdx.x * Shape::TEAMS + team;
    if (i > (total - 1) / kPiece || total == 0) return;
    const int begin = i * kPiece, end = total - begin < kPiece ? total : begin + kPiece;
    const int first = token_row(t, (uint32_t)sorted.order[begin]);
    const int last = token_row(t, (uint32_t)sorted.order[end - 1]);
    for (int which = 0; which < (first == last ? 1 : 2); ++which) {
      const int row = which ? last : first;
      const int from = sorted.start[row], to = sorted.start[row + 1];
      if (to - from <= kPiece) continue;
      float acc[K][VEC] = {};
      add_tokens<T, VEC, LANES, K, DROP>(t, grad, a, sorted.order, max(from, begin), min(to, end), lane,
                                         seed, offset, acc);
      store_row<float, VEC, LANES, K>(partial + ((size_t)i * 2 + which) * t.channels, t.channels, lane, acc);
    }
    return;
  }
  for (uint32_t row = (blockIdx.x - piece_blocks) * Shape::TEAMS + team; row < (uint32_t)t.nrows;
       row += blocks * Shape::TEAMS) {
    const int from = sorted.start[row], to = sorted.start[row + 1];
    if (to - from > kPiece) continue;
    float acc[K][VEC] = {};
    add_tokens<T, VEC, LANES, K, DROP>(t, grad, a, sorted.order, from, to, lane, seed, offset, acc);
    store_row<O, VEC, LANES, K>(out + (size_t)row * t.channels, t.channels, lane, acc);
  }
}

// Long rows: the workgroup of the piece that such a row begins in adds the row's pieces, a wave
// every fourth one.
template <typename O>
__global__ __launch_bounds__(kThreads) void long_rows_kernel(TokenArg t, Sorted sorted,
                                                             const float* __restrict__ partial,
                                                             O* __restrict__ out) {
  constexpr int kWaves = kThreads / kWave;
  __shared__ float sums[kWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int total = sorted.start[t.nrows];
  const int piece = blockIdx.x, begin = piece * kPiece;
  if (begin >= total) return;
  const int end = total - begin < kPiece ? total : begin + kPiece;
  const int row = token_row(t, (uint32_t)sorted.order[end - 1]);
  const int from = sorted.start[row], to = sorted.start[row + 1];
  if (to - from <= kPiece || from < begin) return;
  const int last = (to - 1) / kPiece;
  const int first_slot = from > begin ? 1 : 0;   // behind another row in its first piece
  for (int c0 = 0; c0 < t.channels; c0 += kWave) {
    const int c = c0 + lane;
    float sum = 0.f;
    if (c < t.channels)
#pragma unroll 4
      for (int i = piece + wave; i <= last; i += kWaves)
        sum += partial[((size_t)i * 2 + (i == piece ? first_slot : 0)) * t.channels + c];
    lds_barrier();
    sums[wave][lane] = sum;
    lds_barrier();
    if (wave == 0 && c < t.channels) {
      for (int w = 1; w < kWaves; ++w) sum += sums[w][lane];
      out[(size_t)row * t.channels + c] = narrow<O>(sum);
    }
  }
}

// Rows wider than any team: a workgroup a row, a thread a channel.
template <typename T, typename O, bool DROP>
__global__ __launch_bounds__(kThreads) void wide_rows_kernel(TokenArg t, const T* __restrict__ grad,
                                                             SumArg a, Sorted sorted,
                                                             O* __restrict__ out) {
  uint64_t seed = 0, offset = 0;
  if (DROP) drop_key(a.drop, seed, offset);
  for (uint32_t row = blockIdx.x; row < (uint32_t)t.nrows; row += gridDim.x) {
    const int from = sorted.start[row], to = sorted.start[row + 1];
    for (int c = blockIdx.y * kThreads + threadIdx.x; c < t.channels; c += gridDim.y * kThreads) {
      float acc[1] = {0.f};
      for (int i = from; i < to; ++i) {
        const uint32_t n = (uint32_t)sorted.order[i];
        float g[1] = {widen(grad[(size_t)n * t.channels + c])};
        add_token<DROP, 1>((size_t)n * t.channels + c, a, a.scales ? a.scales[n] : a.scale, seed, offset, g, acc);
      }
      out[(size_t)row * t.channels + c] = narrow<O>(acc[0]);
    }
  }
}

// ---- launches -------------------------------------------------------------------------------------
unsigned at_most(size_t blocks, size_t most) { return (unsigned)(blocks < most ? (blocks ? blocks : 1) : most); }

// The lanes of a team for rows of `packs` packs where wider rows are gone through in steps
template <int VEC, typename F>
void with_lanes(int packs, F f) {
  if (VEC > 1 && packs <= 4) return f(std::integral_constant<int, 4>());
  if (VEC > 1 && packs <= 8) return f(std::integral_constant<int, 8>());
  if (packs <= 16) return f(std::integral_constant<int, 16>());
  if (VEC > 1 && packs <= 32) return f(std::integral_constant<int, 32>());
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
      hipLaunchKernelGGL((embed_kernel<T, VEC, LANES>), dim3(at_most(blocks, kResident)), dim3(kThreads), 0,
                         stream, t, (const T*)table, scale, scales, (T*)out);
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

// How the few-row kernel shares the tokens out.  It is taken for tables of up to kFewRows rows,
// where a wave's copies fit the LDS of a workgroup.
constexpr int kFewRows = 32;
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
  // two workgroups on each of 256 CUs, but no fewer than two rounds of loads for each
  size_t share = ((size_t)ntokens * column_blocks + 511) / 512;
  const size_t least = (size_t)teams * kTableUnroll * 2;
  if (share < least) share = least;
  p.share = (int)share;
  p.parts = (int)(((size_t)ntokens + share - 1) / share);
  return p;
}
// (its partial tables are never more than the 512 workgroups')
size_t few_rows_bytes(int ntokens, int nrows, int channels) {
  // (the smallest share is that of one team)
  size_t parts = ((size_t)ntokens + 2 * kTableUnroll - 1) / (2 * kTableUnroll);
  if (parts > 512) parts = 512;
  return round_up(parts * nrows * channels * sizeof(float));
}

struct SortedLayout {
  size_t start, order, partial, bytes;   // offsets into the workspace
  int pieces;
};
SortedLayout sorted_layout(int ntokens, int nrows, int channels) {
  SortedLayout l;
  l.start = 0;
  l.order = round_up(((size_t)nrows + 1) * sizeof(int32_t));
  l.partial = l.order + round_up((size_t)ntokens * sizeof(int32_t));
  l.pieces = ntokens > kPiece ? (ntokens + kPiece - 1) / kPiece : 0;
  l.bytes = l.partial + round_up((size_t)l.pieces * 2 * channels * sizeof(float));
  return l;
}

template <typename T, typename O, bool DROP>
hipError_t few_rows(const TokenArg& t, const void* grad, const SumArg& a, void* out,
                    float* partial, hipStream_t stream) {
  with_packs_of<T>(t.channels, address(grad), [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    with_lanes<VEC>(t.channels / VEC, [&](auto lanes) {
      constexpr int LANES = decltype(lanes)::value;
      const int column_blocks = (t.channels + LANES * VEC - 1) / (LANES * VEC);
      const FewRowsPlan p = few_rows_plan(t.ntokens, t.nrows, VEC, LANES, column_blocks);
      const bool direct = p.parts == 1 && std::is_same<T, O>::value;
      hipLaunchKernelGGL((few_rows_kernel<T, VEC, LANES, DROP>), dim3(p.parts, column_blocks),
                         dim3(p.waves * kWave), (size_t)p.waves * 256 * t.nrows * VEC, stream, t,
                         (const T*)grad, a, p.share, direct ? (T*)out : nullptr,
                         direct ? nullptr : partial);
      if (direct) return;
      const size_t elements = (size_t)t.nrows * t.channels;
      hipLaunchKernelGGL((sum_tables_kernel<O>), dim3((unsigned)((elements + kWave - 1) / kWave)),
                         dim3(kWave * kSumWaves), 0, stream, partial, p.parts, elements, (O*)out);
    });
  });
  return hipGetLastError();
}

template <typename T, typename O, bool DROP>
hipError_t row_sums(const TokenArg& t, const void* grad, const SumArg& a, void* out, void* workspace,
                    hipStream_t stream) {
  if (t.nrows <= kFewRows) return few_rows<T, O, DROP>(t, grad, a, out, (float*)workspace, stream);
  const SortedLayout l = sorted_layout(t.ntokens, t.nrows, t.channels);
  char* base = static_cast<char*>(workspace);
  int32_t* start = reinterpret_cast<int32_t*>(base + l.start);
  int32_t* order = reinterpret_cast<int32_t*>(base + l.order);
  float* partial = reinterpret_cast<float*>(base + l.partial);
  int range = (t.nrows + 255) / 256;
  if (range > kSortRange) range = kSortRange;
  hipLaunchKernelGGL(sort_tokens_kernel, dim3((t.nrows + range - 1) / range), dim3(kSortThreads),
                     (size_t)kSortWaves * range * sizeof(int), stream, t, range, start, order);
  const Sorted sorted{start, order};
  bool done = false;
  with_packs_of<T>(t.channels, address(grad) | address(out), [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    done = with_team<VEC>((t.channels + VEC - 1) / VEC, [&](auto shape) {
      using S = decltype(shape);
      const int piece_blocks = (l.pieces + S::TEAMS - 1) / S::TEAMS;
      const unsigned blocks = at_most(((size_t)t.nrows + S::TEAMS - 1) / S::TEAMS, kResident * 4);
      hipLaunchKernelGGL((sorted_rows_kernel<T, O, VEC, S::LANES, S::K, DROP>),
                         dim3(blocks + piece_blocks), dim3(S::THREADS), 0, stream, t, (const T*)grad, a,
                         sorted, piece_blocks, (O*)out, partial);
    });
  });
  if (!done)
    hipLaunchKernelGGL((wide_rows_kernel<T, O, DROP>), dim3(at_most(t.nrows, 8192), 16), dim3(kThreads), 0,
                       stream, t, (const T*)grad, a, sorted, (O*)out);
  else if (l.pieces > 0)
    hipLaunchKernelGGL((long_rows_kernel<O>), dim3(l.pieces), dim3(kThreads), 0, stream, t, sorted, partial,
                       (O*)out);
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

size_t row_sums_workspace_bytes(int ntokens, int nrows, int channels) {
  if (nrows <= kFewRows) return few_rows_bytes(ntokens, nrows, channels);
  return sorted_layout(ntokens, nrows, channels).bytes;
}

hipError_t launch_embed(const TokenArg& t, const void* table, float scale, const float* scales,
                        void* out, hipStream_t stream) {
#define MG_CALL(T) embed<T>(t, table, scale, scales, out, stream)
  MG_FOR_TYPE(t.dtype, MG_CALL);
#undef MG_CALL
}

hipError_t launch_embed_backward(const TokenArg& t, const void* grad, float scale,
                                 const float* scales, void* grad_table, void* workspace,
                                 hipStream_t stream) {
  const SumArg a{scale, scales, DropArg()};
  const size_t elements = (size_t)t.nrows * t.channels;
#define MG_CALL(T)                                             \
  t.ntokens == 0 ? zero<T>(grad_table, elements, stream)       \
                 : row_sums<T, T, false>(t, grad, a, grad_table, workspace, stream)
  MG_FOR_TYPE(t.dtype, MG_CALL);
#undef MG_CALL
}

hipError_t launch_row_sums(const TokenArg& t, const void* grad, const DropArg& drop, float* out,
                           void* workspace, hipStream_t stream) {
  const SumArg a{1.f, nullptr, drop};
  if (t.ntokens == 0) return zero<float>(out, (size_t)t.nrows * t.channels, stream);
#define MG_CALL(T) row_sums<T, float, true>(t, grad, a, out, workspace, stream)
  MG_FOR_TYPE(t.dtype, MG_CALL);
#undef MG_CALL
}

hipError_t launch_scale_gradient(const TokenArg& t, const void* grad, const void* table,
                                 float* grad_scales, hipStream_t stream) {
#define MG_CALL(T) scale_gradient<T>(t, grad, table, grad_scales, stream)
  MG_FOR_TYPE(t.dtype, MG_CALL);
#undef MG_CALL
}

}  // namespace mg
