// Type vectors out of a learned table (mg_embed_types) and the gradients of the table and of a
// per-token scale.
//
//   y[n,c] = s_n W[t_n,c]                 zero where t_n names no row of W
//   dW[v,c] = sum over n with t_n = v of s_n g[n,c]        in the order of n, in float
//   ds_n = sum over c of g[n,c] W[t_n,c]
#include "element_types.h"
#include "kernels.h"

namespace mg {
namespace {

constexpr int kThreads = 256;

template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void embed_kernel(const I* __restrict__ index,
                                                         const T* __restrict__ table, int ntokens,
                                                         int nrows, int channels, float scale,
                                                         const float* __restrict__ scales,
                                                         T* __restrict__ out) {
  for (int n = blockIdx.x; n < ntokens; n += gridDim.x) {
    const int row = table_row(index[n], nrows);
    const float s = scales ? scales[n] : scale;
    for (int c = threadIdx.x; c < channels; c += kThreads)
      out[(size_t)n * channels + c] =
          narrow<T>(row < 0 ? 0.f : s * widen(table[(size_t)row * channels + c]));
  }
}

// One thread owns one element of the gradient and reads every index.
template <typename T, typename I, typename O, bool DROP>
__global__ __launch_bounds__(kThreads) void row_sums_kernel(const I* __restrict__ index,
                                                            const T* __restrict__ grad, int ntokens,
                                                            int nrows, int channels, float scale,
                                                            const float* __restrict__ scales,
                                                            DropArg drop, O* __restrict__ out) {
  uint64_t seed = 0, offset = 0;
  if (DROP) drop_key(drop, seed, offset);
  const size_t total = (size_t)nrows * channels;
  const size_t stride = (size_t)gridDim.x * kThreads;
  for (size_t e = (size_t)blockIdx.x * kThreads + threadIdx.x; e < total; e += stride) {
    const int row = (int)(e / channels), c = (int)(e % channels);
    float sum = 0.f;
    for (int n = 0; n < ntokens; ++n) {
      if (table_row(index[n], nrows) != row) continue;
      const size_t at = (size_t)n * channels + c;
      float g = widen(grad[at]);
      if (DROP) {
        const Words4 words = philox(at >> 3, offset, seed);
        g = drop_half(words, (int)(at & 7)) >= drop.limit ? g * drop.factor : 0.f;
      }
      sum += (scales ? scales[n] : scale) * g;
    }
    out[e] = narrow<O>(sum);
  }
}

template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void scale_gradient_kernel(
    const I* __restrict__ index, const T* __restrict__ grad, const T* __restrict__ table,
    int ntokens, int nrows, int channels, float* __restrict__ out) {
  const int lane = threadIdx.x & (kWave - 1);
  const int waves = gridDim.x * (kThreads / kWave);
  for (int n = blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave; n < ntokens; n += waves) {
    const int row = table_row(index[n], nrows);
    float sum = 0.f;
    if (row >= 0)
      for (int c = lane; c < channels; c += kWave)
        sum = fmaf(widen(grad[(size_t)n * channels + c]), widen(table[(size_t)row * channels + c]),
                   sum);
    sum = lanes_sum(sum);
    if (lane == 0) out[n] = sum;
  }
}

unsigned blocks_for(size_t work) { return (unsigned)(work < 65536 ? (work ? work : 1) : 65536); }

template <typename T, typename I>
hipError_t embed(const TokenArg& t, const void* table, float scale, const float* scales, void* out,
                 hipStream_t stream) {
  hipLaunchKernelGGL((embed_kernel<T, I>), dim3(blocks_for(t.ntokens)), dim3(kThreads), 0, stream,
                     (const I*)t.index, (const T*)table, t.ntokens, t.nrows, t.channels, scale,
                     scales, (T*)out);
  return hipGetLastError();
}

template <typename T, typename I, typename O, bool DROP>
hipError_t row_sums(const TokenArg& t, const void* grad, float scale, const float* scales,
                    const DropArg& drop, void* out, hipStream_t stream) {
  const size_t total = (size_t)t.nrows * t.channels;
  hipLaunchKernelGGL((row_sums_kernel<T, I, O, DROP>),
                     dim3(blocks_for((total + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream,
                     (const I*)t.index, (const T*)grad, t.ntokens, t.nrows, t.channels, scale,
                     scales, drop, (O*)out);
  return hipGetLastError();
}

template <typename T, typename I>
hipError_t scale_gradient(const TokenArg& t, const void* grad, const void* table, float* out,
                          hipStream_t stream) {
  hipLaunchKernelGGL((scale_gradient_kernel<T, I>), dim3(blocks_for(((size_t)t.ntokens + 3) / 4)),
                     dim3(kThreads), 0, stream, (const I*)t.index, (const T*)grad, (const T*)table,
                     t.ntokens, t.nrows, t.channels, out);
  return hipGetLastError();
}

}  // namespace

// One instance for each element type and kind of index.
#define MG_FOR_TOKENS(t, FN, ...)                                        \
  switch ((t).dtype * 3 + (t).index_kind) {                              \
    case MG_FLOAT32 * 3 + MG_INDEX_FLOAT32: FN(float, float, __VA_ARGS__)      \
    case MG_FLOAT32 * 3 + MG_INDEX_INT32: FN(float, int32_t, __VA_ARGS__)      \
    case MG_FLOAT32 * 3 + MG_INDEX_INT64: FN(float, int64_t, __VA_ARGS__)      \
    case MG_FLOAT16 * 3 + MG_INDEX_FLOAT32: FN(Half, float, __VA_ARGS__)       \
    case MG_FLOAT16 * 3 + MG_INDEX_INT32: FN(Half, int32_t, __VA_ARGS__)       \
    case MG_FLOAT16 * 3 + MG_INDEX_INT64: FN(Half, int64_t, __VA_ARGS__)       \
    case MG_BFLOAT16 * 3 + MG_INDEX_FLOAT32: FN(Bfloat16, float, __VA_ARGS__)  \
    case MG_BFLOAT16 * 3 + MG_INDEX_INT32: FN(Bfloat16, int32_t, __VA_ARGS__)  \
    case MG_BFLOAT16 * 3 + MG_INDEX_INT64: FN(Bfloat16, int64_t, __VA_ARGS__)  \
  }                                                                      \
  return hipErrorInvalidValue

hipError_t launch_embed(const TokenArg& t, const void* table, float scale, const float* scales,
                        void* out, hipStream_t stream) {
#define MG_CALL(T, I, ...) return embed<T, I>(__VA_ARGS__);
  MG_FOR_TOKENS(t, MG_CALL, t, table, scale, scales, out, stream);
#undef MG_CALL
}

hipError_t launch_embed_backward(const TokenArg& t, const void* grad, float scale,
                                 const float* scales, void* grad_table, void* workspace,
                                 size_t workspace_bytes, hipStream_t stream) {
#define MG_CALL(T, I, ...) return row_sums<T, I, T, false>(__VA_ARGS__);
  MG_FOR_TOKENS(t, MG_CALL, t, grad, scale, scales, DropArg(), grad_table, stream);
#undef MG_CALL
}

hipError_t launch_row_sums(const TokenArg& t, const void* grad, const DropArg& drop, float* out,
                           void* workspace, size_t workspace_bytes, hipStream_t stream) {
#define MG_CALL(T, I, ...) return row_sums<T, I, float, true>(__VA_ARGS__);
  MG_FOR_TOKENS(t, MG_CALL, t, grad, 1.f, (const float*)nullptr, drop, out, stream);
#undef MG_CALL
}

hipError_t launch_scale_gradient(const TokenArg& t, const void* grad, const void* table,
                                 float* grad_scales, hipStream_t stream) {
#define MG_CALL(T, I, ...) return scale_gradient<T, I>(__VA_ARGS__);
  MG_FOR_TOKENS(t, MG_CALL, t, grad, table, grad_scales, stream);
#undef MG_CALL
}

size_t row_sums_workspace_bytes(int ntokens, int nrows, int channels) { return 0; }

}  // namespace mg
