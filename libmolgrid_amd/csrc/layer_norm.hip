// Layer norm over the channels of type vectors (mg_layer_norm), its gradients, and the whole way
// from type indices to dropped-out, normed vectors of a table (mg_encode_types).
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   q = g w, dx = r (q - mean q - h mean (q h)), dw = sum over rows of g h, db = sum over rows of g
//
// The variance is that of the differences, not mean x^2 - m^2, which loses its digits where |m| is
// large beside the spread.  Statistics and sums are float throughout.
#include <type_traits>

#include "kernels.h"
#include "row_team.h"

namespace mg {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

struct Stats {
  float mean, rstd;
};

template <typename T>
__device__ __forceinline__ float param_at(const void* p, bool is_float, int c, float absent) {
  if (p == nullptr) return absent;
  return is_float ? static_cast<const float*>(p)[c] : widen(static_cast<const T*>(p)[c]);
}

// Statistics of one row by the whole workgroup.
template <typename T>
__device__ __forceinline__ Stats wide_row_stats(const T* x, int channels, float scale, float eps,
                                                float (&slots)[2][kWaves]) {
  float sum[1] = {0.f}, squares[1] = {0.f};
  for (int c = threadIdx.x; c < channels; c += kThreads) sum[0] += scale * widen(x[c]);
  team_sums<kThreads>(sum, slots[0]);
  const float mean = sum[0] / channels;
  for (int c = threadIdx.x; c < channels; c += kThreads) {
    const float d = scale * widen(x[c]) - mean;
    squares[0] = fmaf(d, d, squares[0]);
  }
  team_sums<kThreads>(squares, slots[1]);
  return Stats{mean, 1.f / sqrtf(squares[0] / channels + eps)};
}

// Forward: a team holds a row in registers, sums it and its squared differences and writes it once.
// The workgroups stay (kResident of them) and go through the rows, so that a lane reads its share of
// weight and bias once; the next row's loads are in flight while a row is summed.
// 32,768 x 8,192 bfloat16: 201 us (1.07 GB, 5.3 TB/s; a copy of as much reaches 5.1); 121,231 x 28
// floats: 7.7 us; 32,768 x 2,048 bfloat16 off a 16-byte boundary, an element a load: 93 us.
// ENCODE: the rows are those of a scaled table, by the tokens' indices, and are dropped out.  32,768 x
// 2,048 bfloat16: 50 to 55 us, 44 where nothing is dropped.  Its 22 million vector instructions, 8 million of
// them the generator's, take 36 us to issue at 2.4 GHz.
constexpr int kResident = 2048;

template <typename T, int VEC, int LANES, int K, bool ENCODE>
__global__ __launch_bounds__((TeamShape<LANES, K>::THREADS)) void norm_kernel(
    const T* x, TokenArg tokens, float scale, NormArg a, const void* __restrict__ bias, DropArg arg,
    T* out, float* __restrict__ means, float* __restrict__ rstds) {
  using Shape = TeamShape<LANES, K>;
  __shared__ float slots[2][Shape::WAVES];
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const int channels = a.channels;
  const uint32_t nrows = (uint32_t)(ENCODE ? tokens.ntokens : a.nrows);
  uint64_t seed = 0, offset = 0;
  if (ENCODE) drop_key(arg, seed, offset);
  float w[K][VEC], b[K][VEC];
  load_param<T, VEC, LANES, K>(a.weight, a.param_dtype == MG_FLOAT32, 1.f, channels, lane, w);
  load_param<T, VEC, LANES, K>(bias, a.param_dtype == MG_FLOAT32, 0.f, channels, lane, b);
  if (ENCODE) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        w[k][i] *= arg.factor;
        b[k][i] *= arg.factor;
      }
    arg.factor = 1.f;
  }
  const uint32_t step = gridDim.x * Shape::TEAMS;

  RowPacks<T, VEC, K> next;
  bool next_named = true;
  const auto fetch = [&](uint32_t n) {
    size_t at = n;
    bool live = n < nrows;
    if (!live) at = 0;
    if (ENCODE) {
      const int row = live ? token_row(tokens, n) : -1;
      at = row < 0 ? 0 : row;
      live = next_named = row >= 0;
    }
    load_row<T, VEC, LANES, K>(x + at * channels, channels, lane, live, next);
  };
  fetch(blockIdx.x * Shape::TEAMS + team);
  for (uint32_t n0 = blockIdx.x * Shape::TEAMS; n0 < nrows; n0 += step) {
    const uint32_t n = n0 + team;
    const RowPacks<T, VEC, K> packs = next;
    const bool named = next_named;
    fetch(n + step);
    float v[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        v[k][i] = ENCODE ? scale * packs.pack[k][i] : packs.pack[k][i];
    float mean, rstd;
    team_stats<VEC, LANES, K>(v, channels, lane, a.eps, slots[0], slots[1], mean, rstd);
    if (n >= nrows) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * LANES + lane) * VEC;
      if (c >= channels) break;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[k][i] = fmaf(v[k][i] * rstd, w[k][i], b[k][i]);
      const size_t e = (size_t)n * channels + c;
      if (ENCODE) {
        drop<VEC>(e, arg, seed, offset, v[k]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k][i] = named ? v[k][i] : 0.f;
      }
      store_floats<T, VEC>(out + e, v[k]);
    }
    if (!ENCODE && means && lane == 0) {
      means[n] = mean;
      rstds[n] = rstd;
    }
  }
}

// ENCODE with a table of few rows: every workgroup norms the table once, into LDS, and goes through
// the result in groups of eight elements, each with one counter of the generator and one store,
// whatever the channels are.
constexpr int kFewRowsFloats = 8192;   // of a table: 32 KB
constexpr size_t kFewRowsBlocks = 1024;
constexpr int kFewRowsLanes = 8, kFewRowsTeams = kThreads / kFewRowsLanes;   // that share a row; rows normed at a time

// Whether it pays.  Norming the table takes each workgroup about 0.5 us a round of kFewRowsTeams rows and 0.16 us
// for every eight channels of one, which the tokens have to bring in: a team a token draws a counter for each pack,
// so eight times as many where an element is a pack and twice as many for floats.  This kernel and a team
// a token, us, 28 rows and 20,000 | 121,250 tokens unless said:
//   one-element packs:   27 channels of bfloat16 6.5, 8.1 | 9.9, 33;  255 22, 18 | 45, 80;  300 rows of 27 22, 8.0 | 28, 34
//   packs of floats:     32 channels 4.7, 4.4 | 8.9, 9.6;  256 16, 12 | 35, 44;  64 rows of 128 15, 7.6 | 26, 26
//   packs of 16 bits:    32 channels 4.6, 4.3 | 7.2, 7.9;  256 15, 9.0 | 32, 29;  64 rows of 32 5.8, 4.3 | 9.0, 7.9
// and few tokens of wide rows: 300 tokens, one row of 8,192 floats 202, 13.
bool few_rows_pay(const TokenArg& t, size_t element, bool packs) {
  if (t.nrows == 0) return true;   // zeros
  if ((size_t)t.nrows * t.channels > (size_t)kFewRowsFloats) return false;
  const int rounds = (t.nrows + kFewRowsTeams - 1) / kFewRowsTeams;
  if (!packs) return t.ntokens >= 10000 * (rounds + 1);
  return rounds == 1 && t.ntokens >= 50000 && (element == 4 || t.channels <= 64);
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void few_rows_encode_kernel(
    const T* __restrict__ table, TokenArg t, float scale, NormArg a, const void* __restrict__ bias,
    DropArg arg, uint32_t step_tokens, int step_channels, T* __restrict__ out) {
  HIP_DYNAMIC_SHARED(float, vectors);   // [nrows][channels]
  uint64_t seed, offset;
  drop_key(arg, seed, offset);
  constexpr int LANES = kFewRowsLanes, kTeams = kFewRowsTeams;
  const int lane = threadIdx.x % LANES, channels = t.channels;
  const bool is_float = a.param_dtype == MG_FLOAT32;
  for (int row0 = 0; row0 < t.nrows; row0 += kTeams) {
    const int row = row0 + threadIdx.x / LANES, count = row < t.nrows ? channels : 0;
    float* v = vectors + row * channels;
    float sum = 0.f, squares = 0.f;
#pragma unroll 4
    for (int c = lane; c < count; c += LANES) {
      v[c] = scale * widen(table[(size_t)row * channels + c]);
      sum += v[c];
    }
    const float mean = team_sum_in_wave<LANES>(sum) / channels;
    for (int c = lane; c < count; c += LANES) {   // (every lane its own elements)
      const float d = v[c] - mean;
      squares = fmaf(d, d, squares);
    }
    const float rstd = 1.f / sqrtf(team_sum_in_wave<LANES>(squares) / channels + a.eps);
#pragma unroll 4
    for (int c = lane; c < count; c += LANES)
      v[c] = fmaf((v[c] - mean) * rstd, param_at<T>(a.weight, is_float, c, 1.f), param_at<T>(bias, is_float, c, 0.f));
  }
  __syncthreads();
  const size_t total = (size_t)t.ntokens * channels, step = (size_t)gridDim.x * kThreads * 8;
  size_t e = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  uint32_t n = (uint32_t)(e / channels);
  int c = (int)(e % channels);
  for (; e < total; e += step) {
    float v[8];
    if (WHOLE) {   // rows are whole groups
      const int row = token_row(t, n);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = row < 0 ? 0.f : vectors[row * channels + c + i];
    } else {
      uint32_t m = n;
      int at = c, row = token_row(t, m);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = row < 0 ? 0.f : vectors[row * channels + at];
        if (++at == channels) {
          at = 0;
          ++m;
          row = m < (uint32_t)t.ntokens ? token_row(t, m) : -1;
        }
      }
    }
    drop<8>(e, arg, seed, offset, v);
    if (WHOLE || (e + 8 <= total && (reinterpret_cast<uintptr_t>(out) & 15) == 0)) {
      store_floats<T, 8>(out + e, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e + i < total) out[e + i] = narrow<T>(v[i]);
    }
    n += step_tokens;
    c += step_channels;
    if (c >= channels) {
      c -= channels;
      ++n;
    }
  }
}

// Rows wider than any team (more than 8,192 channels): a workgroup goes over the row three times,
// which stays in the caches, an element a load: 8,192 x 12,288 bfloat16 in 255 us (1.6 TB/s).
template <typename T, bool ENCODE>
__global__ __launch_bounds__(kThreads) void wide_norm_kernel(const T* x, TokenArg tokens,
                                                             float scale, NormArg a,
                                                             const void* __restrict__ bias,
                                                             DropArg arg, T* out,
                                                             float* __restrict__ means,
                                                             float* __restrict__ rstds) {
  __shared__ float slots[2][kWaves];
  uint64_t seed = 0, offset = 0;
  if (ENCODE) drop_key(arg, seed, offset);
  const bool is_float = a.param_dtype == MG_FLOAT32;
  const uint32_t nrows = (uint32_t)(ENCODE ? tokens.ntokens : a.nrows);
  for (uint32_t n = blockIdx.x; n < nrows; n += gridDim.x) {
    const int at = ENCODE ? token_row(tokens, n) : 0;
    T* to = out + (size_t)n * a.channels;
    if (at < 0) {
      for (int c = threadIdx.x; c < a.channels; c += kThreads) to[c] = narrow<T>(0.f);
      continue;
    }
    const T* row = x + (size_t)(ENCODE ? (uint32_t)at : n) * a.channels;
    const Stats s = wide_row_stats(row, a.channels, ENCODE ? scale : 1.f, a.eps, slots);
    for (int c = threadIdx.x; c < a.channels; c += kThreads) {
      const float h = ((ENCODE ? scale : 1.f) * widen(row[c]) - s.mean) * s.rstd;
      float y[1] = {fmaf(h, param_at<T>(a.weight, is_float, c, 1.f), param_at<T>(bias, is_float, c, 0.f))};
      if (ENCODE) drop<1>((size_t)n * a.channels + c, arg, seed, offset, y);
      to[c] = narrow<T>(y[0]);
    }
    if (!ENCODE && means && threadIdx.x == 0) {
      means[n] = s.mean;
      rstds[n] = s.rstd;
    }
  }
}

// The words of NamedRows, ORed by the workgroup.
__device__ __forceinline__ uint32_t named_word(const NamedRows& named) {
  __shared__ uint32_t all;
  if (threadIdx.x == 0) all = 0;
  __syncthreads();
  uint32_t mine = 0;
  for (int i = threadIdx.x; i < named.count; i += blockDim.x) mine |= named.words[i];
  if (mine) atomicOr(&all, mine);
  __syncthreads();
  return all;
}
__device__ __forceinline__ bool is_named(const NamedRows& named, uint32_t word, uint32_t n) {
  return named.start ? named.start[n + 1] > named.start[n] : n < 32 && (word >> n & 1);
}

// Backward: a team holds the rows of x and of the gradient, writes dx, and a lane adds its share of
// dw and db up over all rows that its team takes.  32,768 x 8,192 bfloat16: 329 us (1.6 GB, 4.9 TB/s) and
// 8 us for the partial sums; 121,231 x 28 floats: 10 and 6 us.  G: type of the gradient; TABLE: x is a scaled
// table, whose statistics are computed here.
constexpr int kParts = 512, kNarrowParts = 1024;   // workgroups that share the rows

template <typename T, typename G, int VEC, int LANES, int K, bool TABLE>
__global__ __launch_bounds__((TeamShape<LANES, K>::THREADS)) void norm_backward_kernel(
    const G* __restrict__ grad, const T* __restrict__ x, float scale, NormArg a,
    const float* __restrict__ means, const float* __restrict__ rstds, NamedRows named,
    T* __restrict__ grad_x, bool to_params, ParamSums params) {
  using Shape = TeamShape<LANES, K>;
  __shared__ float slots[4][2 * Shape::WAVES];
  HIP_DYNAMIC_SHARED(float, sums);   // dw and db of a workgroup with several teams
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const int channels = a.channels;
  const uint32_t nrows = (uint32_t)a.nrows;
  float w[K][VEC], dw[K][VEC], db[K][VEC];
  load_param<T, VEC, LANES, K>(a.weight, a.param_dtype == MG_FLOAT32, 1.f, channels, lane, w);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = db[k][i] = 0.f;
  const float inv = 1.f / channels;
  const uint32_t step = gridDim.x * Shape::TEAMS;

  const uint32_t word = TABLE ? named_word(named) : 0;

  RowPacks<T, VEC, K> next_x;
  RowPacks<G, VEC, K> next_g;
  float next_mean = 0.f, next_rstd = 0.f;
  bool next_named = false;
  const auto fetch = [&](uint32_t n) {
    const bool live = n < nrows;
    const size_t at = live ? (size_t)n * channels : 0;
    next_named = live && (!TABLE || is_named(named, word, n));
    load_row<T, VEC, LANES, K>(x + at, channels, lane, next_named, next_x);
    load_row<G, VEC, LANES, K>(grad + at, channels, lane, live, next_g);
    if (!TABLE && live) {
      next_mean = means[n];
      next_rstd = rstds[n];
    }
  };
  fetch(blockIdx.x * Shape::TEAMS + team);
  int parity = 0;   // a row's sums must not meet those of the row before in the same slots
  for (uint32_t n0 = blockIdx.x * Shape::TEAMS; n0 < nrows; n0 += step, parity ^= 1) {
    const uint32_t n = n0 + team;
    const RowPacks<T, VEC, K> px = next_x;
    const RowPacks<G, VEC, K> pg = next_g;
    float mean = next_mean, rstd = next_rstd;
    const bool has_part = next_named;
    fetch(n + step);
    float h[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[k][i] = TABLE ? scale * px.pack[k][i] : px.pack[k][i];
    if (TABLE) {
      team_stats<VEC, LANES, K>(h, channels, lane, a.eps, slots[2], slots[3], mean, rstd);
      mean = 0.f;   // (taken out already)
    }
    float both[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float g = pg.pack[k][i];
        h[k][i] = (h[k][i] - mean) * rstd;
        const float q = g * w[k][i];
        both[0] += q;
        both[1] = fmaf(q, h[k][i], both[1]);
        if (has_part) dw[k][i] = fmaf(g, h[k][i], dw[k][i]);
        db[k][i] += g;
      }
    team_sums<LANES>(both, slots[parity]);
    if (grad_x == nullptr || n >= nrows) continue;
    const float mean_q = both[0] * inv, mean_qh = both[1] * inv;
    const float factor = TABLE ? scale * rstd : rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * LANES + lane) * VEC;
      if (c >= channels) break;
      float d[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float q = pg.pack[k][i] * w[k][i];
        d[i] = has_part ? factor * (q - mean_q - h[k][i] * mean_qh) : 0.f;
      }
      store_floats<T, VEC>(grad_x + (size_t)n * channels + c, d);
    }
  }
  if (to_params) add_up_params<T, VEC, LANES, K>(dw, db, lane, channels, sums, params);
}

// The same for rows wider than any team: dx, a workgroup a row, and dw and db, a thread a channel, which
// are kept in the workgroup's row of partial sums: 8,192 x 12,288 bfloat16 in 243 and 1,085 us.
template <typename T, typename G>
__global__ __launch_bounds__(kThreads) void wide_norm_backward_kernel(
    const G* __restrict__ grad, const T* __restrict__ x, float scale, NormArg a, const float* means,
    const float* rstds, NamedRows named, T* __restrict__ grad_x) {
  __shared__ float slots[2][kWaves];
  __shared__ float both_slots[2 * kWaves];
  const bool is_float = a.param_dtype == MG_FLOAT32;
  const uint32_t word = means ? 0 : named_word(named);
  for (uint32_t n = blockIdx.x; n < (uint32_t)a.nrows; n += gridDim.x) {
    const size_t at = (size_t)n * a.channels;
    if (!means && !is_named(named, word, n)) {
      for (int c = threadIdx.x; c < a.channels; c += kThreads) grad_x[at + c] = narrow<T>(0.f);
      continue;
    }
    const Stats s = means ? Stats{means[n], rstds[n]}
                          : wide_row_stats(x + at, a.channels, scale, a.eps, slots);
    float both[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.channels; c += kThreads) {
      const float q = widen(grad[at + c]) * param_at<T>(a.weight, is_float, c, 1.f);
      both[0] += q;
      both[1] = fmaf(q, (scale * widen(x[at + c]) - s.mean) * s.rstd, both[1]);
    }
    lds_barrier();
    team_sums<kThreads>(both, both_slots);
    const float mean_q = both[0] / a.channels, mean_qh = both[1] / a.channels;
    for (int c = threadIdx.x; c < a.channels; c += kThreads) {
      const float q = widen(grad[at + c]) * param_at<T>(a.weight, is_float, c, 1.f);
      const float h = (scale * widen(x[at + c]) - s.mean) * s.rstd;
      grad_x[at + c] = narrow<T>(scale * s.rstd * (q - mean_q - h * mean_qh));
    }
  }
}

template <typename T, typename G>
__global__ __launch_bounds__(kThreads) void wide_norm_params_kernel(
    const G* __restrict__ grad, const T* __restrict__ x, float scale, NormArg a, const float* means,
    const float* rstds, NamedRows named, float* __restrict__ partial) {
  __shared__ float slots[2][kWaves];
  float* row = partial + (size_t)blockIdx.x * 2 * a.channels;
  for (int c = threadIdx.x; c < a.channels; c += kThreads) row[c] = row[a.channels + c] = 0.f;
  const uint32_t word = means ? 0 : named_word(named);
  for (uint32_t n = blockIdx.x; n < (uint32_t)a.nrows; n += gridDim.x) {
    const size_t at = (size_t)n * a.channels;
    if (!means && !is_named(named, word, n)) continue;
    const Stats s = means ? Stats{means[n], rstds[n]}
                          : wide_row_stats(x + at, a.channels, scale, a.eps, slots);
    for (int c = threadIdx.x; c < a.channels; c += kThreads) {   // (the same thread all along)
      const float g = widen(grad[at + c]);
      row[c] = fmaf(g, (scale * widen(x[at + c]) - s.mean) * s.rstd, row[c]);
      row[a.channels + c] += g;
    }
  }
}

// The rows of `partial`, summed: a workgroup takes 64 columns (of dw, then db), its waves a share
// of the rows each, which are then added in their order.
constexpr int kSumWaves = 16;

template <typename P>
__global__ __launch_bounds__(kWave* kSumWaves) void sum_partials_kernel(
    const float* __restrict__ partial, int parts, int channels, P* __restrict__ grad_weight,
    P* __restrict__ grad_bias) {
  __shared__ float sums[kSumWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const size_t columns = (size_t)2 * channels, c = (size_t)blockIdx.x * kWave + lane;
  const int share = (parts + kSumWaves - 1) / kSumWaves;
  const int end = min(parts, (wave + 1) * share);
  float sum = c < columns ? column_sum(partial, columns, c, wave * share, end) : 0.f;
  sums[wave][lane] = sum;
  lds_barrier();
  if (wave != 0 || c >= columns) return;
  for (int w = 1; w < kSumWaves; ++w) sum += sums[w][lane];
  P* to = c < (size_t)channels ? grad_weight : grad_bias;
  if (to) to[c < (size_t)channels ? c : c - channels] = narrow<P>(sum);
}

int wide_parts(int nrows) { return nrows < 256 ? nrows : 256; }

template <typename P>
hipError_t sum_partials(const float* partial, int parts, int channels, void* grad_weight, void* grad_bias,
                  hipStream_t stream) {
  hipLaunchKernelGGL((sum_partials_kernel<P>), dim3(((size_t)2 * channels + kWave - 1) / kWave),
                     dim3(kWave * kSumWaves), 0, stream, partial, parts, channels, (P*)grad_weight,
                     (P*)grad_bias);
  return hipGetLastError();
}

// The encoder's rows take more arithmetic than a norm's, so as many elements a lane as go: what is done
// once a row (a division and a square root, the sums over the lanes) is then shared by more of them:
// 2,048 channels of bfloat16 by 64 lanes 57 us, by 256 lanes 65 us.
template <int VEC, bool ENCODE, typename F>
bool with_norm_team(int packs, F f) {
  if constexpr (ENCODE && VEC == 8)
    if (packs > 128 && packs <= 256) return f(TeamShape<64, 4>()), true;
  return with_team<VEC>(packs, f);
}

template <typename T, bool ENCODE>
hipError_t norm(const NormArg& a, const TokenArg& t, float scale, const void* x, const void* bias,
                const DropArg& drop, void* out, float* means, float* rstds, hipStream_t stream) {
  const uint32_t nrows = (uint32_t)(ENCODE ? t.ntokens : a.nrows);
  const bool packs = whole_packs<T>(a.channels, address(x) | address(out));
  if (ENCODE && few_rows_pay(t, sizeof(T), packs)) {
    const size_t groups = ((size_t)t.ntokens * t.channels + 7) / 8;
    const size_t all = (groups + kThreads - 1) / kThreads, blocks = all < kFewRowsBlocks ? all : kFewRowsBlocks;
    const size_t step = blocks * kThreads * 8, shared = (size_t)t.nrows * t.channels * sizeof(float);
    const bool whole = t.channels % 8 == 0 && address(out) % 16 == 0;
    const uint32_t step_tokens = (uint32_t)(step / t.channels);
    const int step_channels = (int)(step % t.channels);
    if (whole)
      hipLaunchKernelGGL((few_rows_encode_kernel<T, true>), dim3((unsigned)blocks), dim3(kThreads), shared, stream,
                         (const T*)x, t, scale, a, bias, drop, step_tokens, step_channels, (T*)out);
    else
      hipLaunchKernelGGL((few_rows_encode_kernel<T, false>), dim3((unsigned)blocks), dim3(kThreads), shared, stream,
                         (const T*)x, t, scale, a, bias, drop, step_tokens, step_channels, (T*)out);
    return hipGetLastError();
  }
  const auto with_packs = [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    return with_norm_team<VEC, ENCODE>((a.channels + VEC - 1) / VEC, [&](auto shape) {
      using S = decltype(shape);
      const uint32_t blocks = (nrows + S::TEAMS - 1) / S::TEAMS;
      const uint32_t resident = kResident * 256 / S::THREADS;
      hipLaunchKernelGGL((norm_kernel<T, VEC, S::LANES, S::K, ENCODE>),
                         dim3(blocks < resident ? blocks : resident), dim3(S::THREADS), 0, stream,
                         (const T*)x, t, scale, a, bias, drop, (T*)out, means, rstds);
    });
  };
  const bool done = packs ? with_packs(std::integral_constant<int, 16 / (int)sizeof(T)>())
                          : with_packs(std::integral_constant<int, 1>());
  if (!done)
    hipLaunchKernelGGL((wide_norm_kernel<T, ENCODE>), dim3(nrows < 4096 ? nrows : 4096),
                       dim3(kThreads), 0, stream, (const T*)x, t, scale, a, bias, drop, (T*)out,
                       means, rstds);
  return hipGetLastError();
}

// Workgroups that share the rows, each with its row of partial sums (8 bytes a channel): as many as
// fill the chip, more of them where rows are narrow and many share a workgroup.
int norm_parts(int nrows, int teams) {
  const size_t rounds = ((size_t)nrows + teams - 1) / teams;
  const size_t most = teams > 4 ? kNarrowParts : kParts;
  return (int)(rounds < most ? rounds : most);
}

template <typename T, typename G, bool TABLE>
hipError_t norm_backward(const NormArg& a, const void* grad, const void* x, float scale,
                         const float* means, const float* rstds, const NamedRows& named, void* grad_x,
                         void* grad_weight, void* grad_bias, void* workspace, hipStream_t stream) {
  const bool to_params = grad_weight || grad_bias;
  float* partial = to_params ? static_cast<float*>(workspace) : nullptr;
  const ParamSums params{partial, grad_weight, grad_bias, a.param_dtype == MG_FLOAT32};
  int parts = 0;
  bool done = false;
  if (a.nrows > 0) {
    const auto with_packs = [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      return with_team<VEC>((a.channels + VEC - 1) / VEC, [&](auto shape) {
        using S = decltype(shape);
        parts = norm_parts(a.nrows, S::TEAMS);
        const size_t shared = S::LANES <= kWave ? (size_t)2 * a.channels * sizeof(float) : 0;
        hipLaunchKernelGGL((norm_backward_kernel<T, G, VEC, S::LANES, S::K, TABLE>), dim3(parts),
                           dim3(S::THREADS), shared, stream, (const G*)grad, (const T*)x, scale, a,
                           means, rstds, named, (T*)grad_x, to_params, params);
      });
    };
    const bool whole = whole_packs<T>(a.channels, address(x) | address(grad) | address(grad_x));
    done = whole ? with_packs(std::integral_constant<int, 16 / (int)sizeof(T)>())
                 : with_packs(std::integral_constant<int, 1>());
    if (!done) {
      parts = wide_parts(a.nrows);
      if (grad_x)
        hipLaunchKernelGGL((wide_norm_backward_kernel<T, G>), dim3(a.nrows < 4096 ? a.nrows : 4096),
                           dim3(kThreads), 0, stream, (const G*)grad, (const T*)x, scale, a, means,
                           rstds, named, (T*)grad_x);
      if (partial)
        hipLaunchKernelGGL((wide_norm_params_kernel<T, G>), dim3(parts), dim3(kThreads), 0, stream,
                           (const G*)grad, (const T*)x, scale, a, means, rstds, named, partial);
    }
  }
  if (to_params && !(done && parts == 1))
    return launch_sum_partials(a, partial, parts, grad_weight, grad_bias, stream);
  return hipGetLastError();
}

}  // namespace

size_t norm_backward_workspace_bytes(int nrows, int channels) {
  size_t parts = 0;   // (whichever team takes the rows)
  for (int teams = 1; teams <= 64; teams *= 2)
    if ((size_t)norm_parts(nrows, teams) > parts) parts = norm_parts(nrows, teams);
  return parts * 2 * channels * sizeof(float);
}

#define MG_FOR_TYPE(dtype, FN)                \
  switch (dtype) {                            \
    case MG_FLOAT32: return FN(float);        \
    case MG_FLOAT16: return FN(Half);         \
    case MG_BFLOAT16: return FN(Bfloat16);    \
  }                                           \
  return hipErrorInvalidValue

hipError_t launch_sum_partials(const NormArg& a, const float* partial, int parts, void* grad_weight,
                               void* grad_bias, hipStream_t stream) {
#define MG_CALL(T) sum_partials<T>(partial, parts, a.channels, grad_weight, grad_bias, stream)
  MG_FOR_TYPE(a.param_dtype, MG_CALL);
#undef MG_CALL
}

hipError_t launch_norm(const NormArg& a, const void* x, const void* bias, void* out, float* means,
                       float* rstds, hipStream_t stream) {
#define MG_CALL(T) norm<T, false>(a, TokenArg(), 1.f, x, bias, DropArg(), out, means, rstds, stream)
  MG_FOR_TYPE(a.dtype, MG_CALL);
#undef MG_CALL
}

hipError_t launch_encode(const TokenArg& t, const NormArg& a, const void* table, float scale,
                         const void* bias, const DropArg& drop, void* out, hipStream_t stream) {
#define MG_CALL(T) norm<T, true>(a, t, scale, table, bias, drop, out, nullptr, nullptr, stream)
  MG_FOR_TYPE(a.dtype, MG_CALL);
#undef MG_CALL
}

hipError_t launch_norm_backward(const NormArg& a, const void* grad, const void* x,
                                const float* means, const float* rstds, void* grad_x,
                                void* grad_weight, void* grad_bias, void* workspace,
                                hipStream_t stream) {
#define MG_CALL(T)                                                                              \
  norm_backward<T, T, false>(a, grad, x, 1.f, means, rstds, NamedRows(), grad_x, grad_weight, grad_bias, workspace, \
                             stream)
  MG_FOR_TYPE(a.dtype, MG_CALL);
#undef MG_CALL
}

hipError_t launch_table_norm_backward(const NormArg& a, const float* sums, const void* table,
                                      float scale, const NamedRows& named, void* grad_table, void* grad_weight,
                                      void* grad_bias, void* workspace, hipStream_t stream) {
#define MG_CALL(T)                                                                            \
  norm_backward<T, float, true>(a, sums, table, scale, nullptr, nullptr, named, grad_table, grad_weight, \
                                grad_bias, workspace, stream)
  MG_FOR_TYPE(a.dtype, MG_CALL);
#undef MG_CALL
}

}  // namespace mg
