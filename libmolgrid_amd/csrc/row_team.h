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

// Calls f with the shape for rows of `packs` packs: the narrowest team that holds them, in which a
// lane holds up to 32 elements of 16-bit types, 16 of any other.  False: no team is wide enough.
template <int VEC, typename F>
bool with_team(int packs, F f) {
  if constexpr (VEC == 1) {
    if (packs <= 16) return f(TeamShape<16, 1>()), true;
    if (packs <= 64) return f(TeamShape<64, 1>()), true;
    if (packs <= 256) return f(TeamShape<64, 4>()), true;
    if (packs <= 1024) return f(TeamShape<64, 16>()), true;
    if (packs <= 4096) return f(TeamShape<256, 16>()), true;
    if (packs <= 16384) return f(TeamShape<1024, 16>()), true;
  } else {
    if (packs <= 4) return f(TeamShape<4, 1>()), true;
    if (packs <= 8) return f(TeamShape<8, 1>()), true;
    if (packs <= 16) return f(TeamShape<16, 1>()), true;
    if (packs <= 32) return f(TeamShape<32, 1>()), true;
    if (packs <= 64) return f(TeamShape<64, 1>()), true;
    if (packs <= 128) return f(TeamShape<64, 2>()), true;
    if (packs <= 256) return f(TeamShape<64, 4>()), true;
    if (packs <= 512) return f(TeamShape<256, 2>()), true;
    if (packs <= 1024) return f(TeamShape<256, 4>()), true;
    if (packs <= 4096 * 4 / VEC) return f(TeamShape<1024, 16 / VEC>()), true;
  }
  return false;
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
template <typename T, int VEC, int LANES, int K>
__device__ __forceinline__ void load_row(const T* row, int channels, int lane, bool live,
                                         RowPacks<T, VEC, K>& out) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * LANES + lane) * VEC;
    if (live && c < channels)
      out.pack[k] = *reinterpret_cast<const Pack<T, VEC>*>(row + c);
    else
#pragma unroll
      for (int i = 0; i < VEC; ++i) out.pack[k].v[i] = T();
  }
}

// A lane's share of a parameter (float or of type T, or absent)
template <typename T, int VEC, int LANES, int K>
__device__ __forceinline__ void load_param(const void* p, bool is_float, float absent, int channels,
                                           int lane, float (&out)[K][VEC]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * LANES + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[k][i] = absent;
    if (p == nullptr || c >= channels) continue;
    if (is_float) {
      const float* f = static_cast<const float*>(p) + c;
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[k][i] = f[i];
    } else {
      const T* t = static_cast<const T*>(p) + c;
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[k][i] = widen(t[i]);
    }
  }
}

// Drops elements e .. e + VEC - 1 of v (see DropArg); e is a multiple of VEC.
template <int VEC>
__device__ __forceinline__ void drop(size_t e, const DropArg& a, uint64_t seed, uint64_t offset,
                                     float (&v)[VEC]) {
  if (a.limit == 0) return;
  const Words4 words = philox(e >> 3, offset, seed);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    uint32_t half;
    if (VEC == 8) {
      half = drop_half(words, i);
    } else if (VEC == 4) {
      const uint32_t w = (e & 4) ? words.w[2 + i / 2] : words.w[i / 2];
      half = i & 1 ? w >> 16 : w & 0xFFFFu;
    } else {
      const uint32_t pair = (e & 4) ? ((e & 2) ? words.w[3] : words.w[2]) : ((e & 2) ? words.w[1] : words.w[0]);
      half = (e & 1) ? pair >> 16 : pair & 0xFFFFu;
    }
    v[i] = half >= a.limit ? v[i] * a.factor : 0.f;
  }
}

}  // namespace mg

#endif
