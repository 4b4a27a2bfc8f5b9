// A team of LANES lanes holds one row of type vectors in registers: K packs of VEC elements a lane,
// pack k of lane l at element (k LANES + l) VEC, so that every load and store of the team is
// contiguous.  Narrow rows share a wave, wide ones take a workgroup.
#ifndef LIBMOLGRID_AMD_ROW_TEAM_H_
#define LIBMOLGRID_AMD_ROW_TEAM_H_

#include "element_types.h"
#include "sweep.h"

namespace mg {

template <int LANES_, int K_>
struct TeamShape {
  static constexpr int LANES = LANES_, K = K_;
  static constexpr int THREADS = LANES > 256 ? LANES : 256;
  static constexpr int TEAMS = THREADS / LANES;   // rows that a workgroup holds at a time
  static constexpr int WAVES = THREADS / kWave;
};

constexpr int kMostTeamChannels = 8192;   // of rows that a team can hold

// Calls f with the shape for rows of `packs` packs.  Few elements a lane (up to 32 of 16-bit types, 16
// of any other) leave room for many waves, whose loads hide one another; four-wave teams pay with a
// barrier a sum.  1001 channels of float16, one element a pack: 64 lanes of 16 packs take 16 us where
// 256 lanes of four take 10 (4099 rows).  False: no team is wide enough.
template <int VEC, typename F>
bool with_team(int packs, F f) {
  if constexpr (VEC == 1) {
    if (packs <= 16) return f(TeamShape<16, 1>()), true;
    if (packs <= 64) return f(TeamShape<64, 1>()), true;
    if (packs <= 256) return f(TeamShape<64, 4>()), true;
    if (packs <= 1024) return f(TeamShape<256, 4>()), true;
    if (packs <= 4096) return f(TeamShape<256, 16>()), true;
    if (packs <= 8192) return f(TeamShape<1024, 8>()), true;
  } else {
    if (packs <= 4) return f(TeamShape<4, 1>()), true;
    if (packs <= 8) return f(TeamShape<8, 1>()), true;
    if (packs <= 16) return f(TeamShape<16, 1>()), true;
    if (packs <= 32) return f(TeamShape<32, 1>()), true;
    if (packs <= 64) return f(TeamShape<64, 1>()), true;
    if (packs <= 128) return f(TeamShape<64, 2>()), true;
    if (packs <= 256) return f(TeamShape<256, 1>()), true;
    if (packs <= 512) return f(TeamShape<256, 2>()), true;
    if (packs <= 1024) return f(TeamShape<256, 4>()), true;
    if constexpr (VEC == 4)
      if (packs <= 2048) return f(TeamShape<1024, 2>()), true;
  }
  return false;
}

// Teams of a wave or less for rows that are gone through in tiles of up to `most` packs a lane
template <int VEC, int MOST, typename F>
void with_tile(int packs, F f) {
  if constexpr (VEC > 1) {
    if (packs <= 4) return f(TeamShape<4, 1>());
    if (packs <= 8) return f(TeamShape<8, 1>());
    if (packs > 16 && packs <= 32) return f(TeamShape<32, 1>());
  }
  if (packs <= 16) return f(TeamShape<16, 1>());
  if constexpr (MOST > 1) {
    if (packs > 64 && packs <= 128) return f(TeamShape<64, 2>());
    if (packs > 128) return f(TeamShape<64, 4>());
  }
  return f(TeamShape<64, 1>());
}

// Elements of a pack for rows of `channels` elements in arrays whose addresses are ORed together in
// `where`: 16 bytes where every row of every array starts on a 16-byte boundary, one element
// otherwise.
template <typename T>
bool whole_packs(int channels, uintptr_t where) {
  return channels % (16 / (int)sizeof(T)) == 0 && where % 16 == 0;
}
inline uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}

// Sum over the team's lanes that share a wave, in each of them.  Every lane of the wave calls it.
template <int LANES>
__device__ __forceinline__ float team_sum_in_wave(float v) {
  v = add_dpp<kDppQuadPerm1032>(v);
  v = add_dpp<kDppQuadPerm2301>(v);
  if (LANES >= 8) v = add_dpp<kDppRowHalfMirror>(v);
  if (LANES >= 16) v = add_dpp<kDppRowMirror>(v);
  if (LANES >= 32) v += __shfl_xor(v, 16);
  if (LANES >= 64) v += __shfl_xor(v, 32);
  return v;
}

// Two sums over the team's lanes, in each of them.  A team of several waves meets at a barrier:
// every thread of the workgroup calls it, and two calls in a row must not get the same `slots`
// (one float for each wave and sum).
template <int LANES, int SUMS>
__device__ __forceinline__ void team_sums(float (&v)[SUMS], float* slots) {
#pragma unroll
  for (int s = 0; s < SUMS; ++s) v[s] = team_sum_in_wave<LANES>(v[s]);
  if (LANES <= kWave) return;
  constexpr int kWaves = LANES <= kWave ? 1 : LANES / kWave;
  if ((threadIdx.x & (kWave - 1)) == 0) {
#pragma unroll
    for (int s = 0; s < SUMS; ++s) slots[s * kWaves + threadIdx.x / kWave] = v[s];
  }
  lds_barrier();
#pragma unroll
  for (int s = 0; s < SUMS; ++s) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += slots[s * kWaves + w];
    v[s] = sum;
  }
}

// K packs of a row, as they stand in memory
template <typename T, int VEC, int K>
struct RowPacks {
  Pack<T, VEC> pack[K];
};
// Lanes beyond the last channel read the row's first pack, which is there, and get zeros: a branch
// around every load would be issued one after the other.
template <typename T, int VEC, int LANES, int K>
__device__ __forceinline__ void load_row(const T* row, int channels, int lane, bool live,
                                         RowPacks<T, VEC, K>& out) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * LANES + lane) * VEC;
    out.pack[k] = *reinterpret_cast<const Pack<T, VEC>*>(row + (c < channels ? c : 0));
  }
#pragma unroll
  for (int k = 0; k < K; ++k) out.pack[k].zero_unless(live && (k * LANES + lane) * VEC < channels);
}

// A lane's share of a parameter (float or of type T, or absent)
template <typename S, int VEC, int LANES, int K>
__device__ __forceinline__ void load_param_as(const S* p, int channels, int lane, float (&out)[K][VEC]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * LANES + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[k][i] = c < channels ? widen(p[c + i]) : 0.f;
  }
}
template <typename T, int VEC, int LANES, int K>
__device__ __forceinline__ void load_param(const void* p, bool is_float, float absent, int channels,
                                           int lane, float (&out)[K][VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[k][i] = absent;
  } else if (is_float) {
    load_param_as<float, VEC, LANES, K>(static_cast<const float*>(p), channels, lane, out);
  } else {
    load_param_as<T, VEC, LANES, K>(static_cast<const T*>(p), channels, lane, out);
  }
}

// The rows of tokens n[0 .. U) below `end`, -1 for the others: all their indices are loaded together.
template <int U>
__device__ __forceinline__ void token_rows(const TokenArg& t, const uint32_t (&n)[U], uint32_t end,
                                           int (&row)[U]) {
#define MG_ROWS(S)                                                                  \
  {                                                                                 \
    S index[U];                                                                     \
    _Pragma("unroll") for (int u = 0; u < U; ++u)                                   \
      index[u] = n[u] < end ? static_cast<const S*>(t.index)[n[u]] : (S)-1;         \
    _Pragma("unroll") for (int u = 0; u < U; ++u) row[u] = table_row(index[u], t.nrows); \
  }
  if (t.index_kind == MG_INDEX_FLOAT32)
    MG_ROWS(float)
  else if (t.index_kind == MG_INDEX_INT32)
    MG_ROWS(int32_t)
  else
    MG_ROWS(int64_t)
#undef MG_ROWS
}

// Statistics of the row that a team holds in v, which becomes its differences from the mean; two
// slots arrays as in team_sums.
template <int VEC, int LANES, int K>
__device__ __forceinline__ void team_stats(float (&v)[K][VEC], int channels, int lane, float eps,
                                           float* slots_a, float* slots_b, float& mean, float& rstd) {
  float sum[1] = {0.f}, squares[1] = {0.f};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[0] += v[k][i];
  team_sums<LANES>(sum, slots_a);
  mean = sum[0] / channels;   // (a product could be contracted into the differences)
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if ((k * LANES + lane) * VEC < channels)   // (zeros beyond)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[k][i] -= mean;
        squares[0] = fmaf(v[k][i], v[k][i], squares[0]);
      }
  }
  team_sums<LANES>(squares, slots_b);
  rstd = 1.f / sqrtf(squares[0] / channels + eps);
}

// Column `at` of rows begin .. end - 1 (of `stride` floats) added up, sixteen loads at a time, the last
// ones too.
__device__ __forceinline__ float column_sum(const float* rows, size_t stride, size_t at, int begin, int end) {
  constexpr int U = 16;
  float sum = 0.f;
  for (int i0 = begin; i0 < end; i0 += U) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = rows[(size_t)min(i0 + u, end - 1) * stride + at];
#pragma unroll
    for (int u = 0; u < U; ++u) sum += i0 + u < end ? v[u] : 0.f;
  }
  return sum;
}

// Where the sums of a norm's parameter gradients go: as they are if one workgroup has them all,
// else into the workgroup's row of `partial` (weight, then bias).
struct ParamSums {
  float* partial;
  void *weight, *bias;   // of param_dtype; either may be nullptr
  int is_float;
};
template <typename T>
__device__ __forceinline__ void store_param_sum(const ParamSums& to, int channels, int c, float dw, float db) {
  if (gridDim.x > 1) {
    float* row = to.partial + (size_t)blockIdx.x * 2 * channels;
    row[c] = dw;
    row[channels + c] = db;
  } else if (to.is_float) {
    if (to.weight) static_cast<float*>(to.weight)[c] = dw;
    if (to.bias) static_cast<float*>(to.bias)[c] = db;
  } else {
    if (to.weight) static_cast<T*>(to.weight)[c] = narrow<T>(dw);
    if (to.bias) static_cast<T*>(to.bias)[c] = narrow<T>(db);
  }
}

// Adds the teams' shares of dw and db up in their order: those of a wave first, then the waves one
// after the other through `sums` (2 channels floats of LDS, where a workgroup has several teams).
template <typename T, int VEC, int LANES, int K>
__device__ __forceinline__ void add_up_params(float (&dw)[K][VEC], float (&db)[K][VEC], int lane, int channels,
                                              float* sums, const ParamSums& to) {
  using Shape = TeamShape<LANES, K>;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
      for (int m = LANES; m < kWave; m *= 2) {
        dw[k][i] += __shfl_xor(dw[k][i], m);
        db[k][i] += __shfl_xor(db[k][i], m);
      }
    }
  constexpr int kTurns = LANES < kWave ? Shape::WAVES : Shape::TEAMS;
  const int turn = LANES < kWave ? threadIdx.x / kWave : threadIdx.x / LANES;
  const bool speaks = LANES >= kWave || (threadIdx.x & (kWave - 1)) < LANES;
  for (int t = 0; t < kTurns; ++t) {
    if (t > 0) lds_barrier();
    if (turn != t || !speaks) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * LANES + lane) * VEC;
      if (c >= channels) break;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (t > 0) {
          dw[k][i] += sums[c + i];
          db[k][i] += sums[channels + c + i];
        }
        if (t + 1 < kTurns) {
          sums[c + i] = dw[k][i];
          sums[channels + c + i] = db[k][i];
        } else {
          store_param_sum<T>(to, channels, c + i, dw[k][i], db[k][i]);
        }
      }
    }
  }
}

// Drops elements e .. e + VEC - 1 of v (see DropArg); e is a multiple of VEC.
template <int VEC>
__device__ __forceinline__ void drop(size_t e, const DropArg& a, uint64_t seed, uint64_t offset,
                                     float (&v)[VEC]) {
  if (a.limit == 0) return;
  const Words4 words = philox(e >> 3, offset, seed);
  const uint32_t upper = 0u - ((uint32_t)(e >> 2) & 1u);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    // (selections by bits: an index that depends on e would put the words into memory)
    uint32_t half;
    if (VEC == 8) {
      half = drop_half(words, i);
    } else if (VEC == 4) {
      const uint32_t w = words.w[i / 2] ^ ((words.w[i / 2] ^ words.w[2 + i / 2]) & upper);
      half = i & 1 ? w >> 16 : w & 0xFFFFu;
    } else {
      const uint32_t odd = 0u - ((uint32_t)(e >> 1) & 1u);
      const uint32_t w0 = words.w[0] ^ ((words.w[0] ^ words.w[2]) & upper);
      const uint32_t w1 = words.w[1] ^ ((words.w[1] ^ words.w[3]) & upper);
      const uint32_t w = w0 ^ ((w0 ^ w1) & odd);
      half = (e & 1) ? w >> 16 : w & 0xFFFFu;
    }
    v[i] = half >= a.limit ? v[i] * a.factor : 0.f;
  }
}

}  // namespace mg

#endif
