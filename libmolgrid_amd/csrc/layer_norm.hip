// Layer norm over the channels of type vectors (mg_layer_norm), its gradients, and the whole way
// from type indices to dropped-out, normed vectors of a table (mg_encode_types).
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   q = g w, dx = r (q - mean q - h mean (q h)), dw = sum over rows of g h, db = sum over rows of g
//
// The variance is that of the differences, not mean x^2 - m^2, which loses its digits where |m| is
// large beside the spread.  Statistics and sums are float throughout.
#include "element_types.h"
#include "kernels.h"

namespace mg {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

struct Stats {
  float mean, rstd;
};

template <typename T>
__device__ __forceinline__ Stats row_stats(const T* x, int channels, float scale, float eps,
                                           int lane) {
  float sum = 0.f;
  for (int c = lane; c < channels; c += kWave) sum += scale * widen(x[c]);
  const float mean = lanes_sum(sum) / channels;
  float squares = 0.f;
  for (int c = lane; c < channels; c += kWave) {
    const float d = scale * widen(x[c]) - mean;
    squares = fmaf(d, d, squares);
  }
  return Stats{mean, 1.f / sqrtf(lanes_sum(squares) / channels + eps)};
}

// A wave takes one row.
template <typename T, typename P>
__global__ __launch_bounds__(kThreads) void norm_kernel(const T* x, int nrows, int channels,
                                                        const P* __restrict__ weight,
                                                        const P* __restrict__ bias, float eps,
                                                        T* out, float* __restrict__ means,
                                                        float* __restrict__ rstds) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int n = blockIdx.x * kWaves + threadIdx.x / kWave; n < nrows; n += gridDim.x * kWaves) {
    const T* row = x + (size_t)n * channels;
    const Stats s = row_stats(row, channels, 1.f, eps, lane);
    for (int c = lane; c < channels; c += kWave) {
      const float h = (widen(row[c]) - s.mean) * s.rstd;
      out[(size_t)n * channels + c] =
          narrow<T>(fmaf(h, weight ? widen(weight[c]) : 1.f, bias ? widen(bias[c]) : 0.f));
    }
    if (lane == 0 && means) {
      means[n] = s.mean;
      rstds[n] = s.rstd;
    }
  }
}

template <typename T, typename P, typename I>
__global__ __launch_bounds__(kThreads) void encode_kernel(const I* __restrict__ index,
                                                          const T* __restrict__ table, int ntokens,
                                                          int nrows, int channels, float scale,
                                                          const P* __restrict__ weight,
                                                          const P* __restrict__ bias, float eps,
                                                          DropArg drop, T* __restrict__ out) {
  uint64_t seed, offset;
  drop_key(drop, seed, offset);
  const int lane = threadIdx.x & (kWave - 1);
  for (int n = blockIdx.x * kWaves + threadIdx.x / kWave; n < ntokens; n += gridDim.x * kWaves) {
    const int at = table_row(index[n], nrows);
    if (at < 0) {
      for (int c = lane; c < channels; c += kWave)
        out[(size_t)n * channels + c] = narrow<T>(0.f);
      continue;
    }
    const T* row = table + (size_t)at * channels;
    const Stats s = row_stats(row, channels, scale, eps, lane);
    for (int c = lane; c < channels; c += kWave) {
      const float h = (scale * widen(row[c]) - s.mean) * s.rstd;
      const float y = fmaf(h, weight ? widen(weight[c]) : 1.f, bias ? widen(bias[c]) : 0.f);
      const size_t e = (size_t)n * channels + c;
      const Words4 words = philox(e >> 3, offset, seed);
      out[e] = narrow<T>(drop_half(words, (int)(e & 7)) >= drop.limit ? y * drop.factor : 0.f);
    }
  }
}

// dx; a wave takes one row.  G is float where the gradient is a sum over tokens.
template <typename T, typename P, typename G>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(
    const G* grad, const T* x, int nrows, int channels, float scale, const float* means,
    const float* rstds, const P* __restrict__ weight, float eps, T* grad_x) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int n = blockIdx.x * kWaves + threadIdx.x / kWave; n < nrows; n += gridDim.x * kWaves) {
    const size_t at = (size_t)n * channels;
    const Stats s = means ? Stats{means[n], rstds[n]} : row_stats(x + at, channels, scale, eps, lane);
    float sum = 0.f, sum_h = 0.f;
    for (int c = lane; c < channels; c += kWave) {
      const float q = widen(grad[at + c]) * (weight ? widen(weight[c]) : 1.f);
      sum += q;
      sum_h = fmaf(q, (scale * widen(x[at + c]) - s.mean) * s.rstd, sum_h);
    }
    sum = lanes_sum(sum) / channels;
    sum_h = lanes_sum(sum_h) / channels;
    for (int c = lane; c < channels; c += kWave) {
      const float q = widen(grad[at + c]) * (weight ? widen(weight[c]) : 1.f);
      const float h = (scale * widen(x[at + c]) - s.mean) * s.rstd;
      grad_x[at + c] = narrow<T>(scale * s.rstd * (q - sum - h * sum_h));
    }
  }
}

// dw and db, first step: the workgroup's share of the rows is summed into its own row of `partial`
// (weight, then bias).
template <typename T, typename G>
__global__ __launch_bounds__(kThreads) void norm_params_kernel(const G* grad, const T* x, int nrows,
                                                               int channels, float scale,
                                                               const float* means,
                                                               const float* rstds, float eps,
                                                               float* __restrict__ partial) {
  __shared__ Stats stats[kThreads];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  for (int c0 = 0; c0 < channels; c0 += kThreads) {
    const int c = c0 + threadIdx.x;
    float dw = 0.f, db = 0.f;
    for (int n0 = blockIdx.x * kThreads; n0 < nrows; n0 += gridDim.x * kThreads) {
      const int count = min(kThreads, nrows - n0);
      __syncthreads();
      if (means) {
        if ((int)threadIdx.x < count) stats[threadIdx.x] = Stats{means[n0 + threadIdx.x], rstds[n0 + threadIdx.x]};
      } else {
        for (int i = wave; i < count; i += kWaves)
          stats[i] = row_stats(x + (size_t)(n0 + i) * channels, channels, scale, eps, lane);
      }
      __syncthreads();
      if (c < channels)
        for (int i = 0; i < count; ++i) {
          const size_t at = (size_t)(n0 + i) * channels + c;
          const float g = widen(grad[at]);
          dw = fmaf(g, (scale * widen(x[at]) - stats[i].mean) * stats[i].rstd, dw);
          db += g;
        }
    }
    if (c < channels) {
      partial[(size_t)blockIdx.x * 2 * channels + c] = dw;
      partial[((size_t)blockIdx.x * 2 + 1) * channels + c] = db;
    }
  }
}

// Second step: the partial rows are summed in their order.
template <typename P>
__global__ __launch_bounds__(kThreads) void norm_params_sum_kernel(const float* __restrict__ partial,
                                                                   int parts, int channels,
                                                                   P* __restrict__ grad_weight,
                                                                   P* __restrict__ grad_bias) {
  for (int c = blockIdx.x * kThreads + threadIdx.x; c < channels; c += gridDim.x * kThreads) {
    float dw = 0.f, db = 0.f;
    for (int i = 0; i < parts; ++i) {
      dw += partial[(size_t)i * 2 * channels + c];
      db += partial[((size_t)i * 2 + 1) * channels + c];
    }
    if (grad_weight) grad_weight[c] = narrow<P>(dw);
    if (grad_bias) grad_bias[c] = narrow<P>(db);
  }
}

unsigned row_blocks(int nrows) {
  const size_t blocks = ((size_t)nrows + kWaves - 1) / kWaves;
  return (unsigned)(blocks < 65536 ? (blocks ? blocks : 1) : 65536);
}
int norm_parts(int nrows) { return nrows >= 512 * 256 ? 512 : (nrows + 255) / 256; }

template <typename T, typename P>
hipError_t norm(const NormArg& a, const void* x, const void* bias, void* out, float* means,
                float* rstds, hipStream_t stream) {
  hipLaunchKernelGGL((norm_kernel<T, P>), dim3(row_blocks(a.nrows)), dim3(kThreads), 0, stream,
                     (const T*)x, a.nrows, a.channels, (const P*)a.weight, (const P*)bias, a.eps,
                     (T*)out, means, rstds);
  return hipGetLastError();
}

template <typename T, typename P, typename G>
hipError_t norm_backward(const NormArg& a, const void* grad, const void* x, float scale,
                         const float* means, const float* rstds, void* grad_x, void* grad_weight,
                         void* grad_bias, void* workspace, hipStream_t stream) {
  if (grad_x && a.nrows > 0)
    hipLaunchKernelGGL((norm_backward_kernel<T, P, G>), dim3(row_blocks(a.nrows)), dim3(kThreads), 0,
                       stream, (const G*)grad, (const T*)x, a.nrows, a.channels, scale, means, rstds,
                       (const P*)a.weight, a.eps, (T*)grad_x);
  if (grad_weight || grad_bias) {
    const int parts = norm_parts(a.nrows);
    if (parts > 0)
      hipLaunchKernelGGL((norm_params_kernel<T, G>), dim3(parts), dim3(kThreads), 0, stream,
                         (const G*)grad, (const T*)x, a.nrows, a.channels, scale, means, rstds, a.eps,
                         (float*)workspace);
    hipLaunchKernelGGL((norm_params_sum_kernel<P>), dim3((a.channels + kThreads - 1) / kThreads),
                       dim3(kThreads), 0, stream, (const float*)workspace, parts, a.channels,
                       (P*)grad_weight, (P*)grad_bias);
  }
  return hipGetLastError();
}

template <typename T, typename P, typename I>
hipError_t encode(const TokenArg& t, const NormArg& a, const void* table, float scale,
                  const void* bias, const DropArg& drop, void* out, hipStream_t stream) {
  hipLaunchKernelGGL((encode_kernel<T, P, I>), dim3(row_blocks(t.ntokens)), dim3(kThreads), 0,
                     stream, (const I*)t.index, (const T*)table, t.ntokens, t.nrows, t.channels,
                     scale, (const P*)a.weight, (const P*)bias, a.eps, drop, (T*)out);
  return hipGetLastError();
}

}  // namespace

// Parameters are float or of the type of the vectors.
#define MG_FOR_NORM(dtype, param, FN, ...)                                   \
  switch (dtype) {                                                           \
    case MG_FLOAT32: return FN(float, float, __VA_ARGS__);                   \
    case MG_FLOAT16:                                                         \
      if (param == MG_FLOAT32) return FN(Half, float, __VA_ARGS__);          \
      return FN(Half, Half, __VA_ARGS__);                                    \
    case MG_BFLOAT16:                                                        \
      if (param == MG_FLOAT32) return FN(Bfloat16, float, __VA_ARGS__);      \
      return FN(Bfloat16, Bfloat16, __VA_ARGS__);                            \
  }                                                                          \
  return hipErrorInvalidValue

size_t norm_backward_workspace_bytes(int nrows, int channels) {
  return (size_t)norm_parts(nrows) * 2 * channels * sizeof(float);
}

hipError_t launch_norm(const NormArg& a, const void* x, const void* bias, void* out, float* means,
                       float* rstds, hipStream_t stream) {
#define MG_CALL(T, P, ...) norm<T, P>(__VA_ARGS__)
  MG_FOR_NORM(a.dtype, a.param_dtype, MG_CALL, a, x, bias, out, means, rstds, stream);
#undef MG_CALL
}

hipError_t launch_norm_backward(const NormArg& a, const void* grad, const void* x,
                                const float* means, const float* rstds, void* grad_x,
                                void* grad_weight, void* grad_bias, void* workspace,
                                hipStream_t stream) {
#define MG_CALL(T, P, ...) norm_backward<T, P, T>(__VA_ARGS__)
  MG_FOR_NORM(a.dtype, a.param_dtype, MG_CALL, a, grad, x, 1.f, means, rstds, grad_x, grad_weight,
              grad_bias, workspace, stream);
#undef MG_CALL
}

hipError_t launch_table_norm_backward(const NormArg& a, const float* sums, const void* table,
                                      float scale, void* grad_table, void* grad_weight,
                                      void* grad_bias, void* workspace, hipStream_t stream) {
#define MG_CALL(T, P, ...) norm_backward<T, P, float>(__VA_ARGS__)
  MG_FOR_NORM(a.dtype, a.param_dtype, MG_CALL, a, sums, table, scale, (const float*)nullptr,
              (const float*)nullptr, grad_table, grad_weight, grad_bias, workspace, stream);
#undef MG_CALL
}

hipError_t launch_encode(const TokenArg& t, const NormArg& a, const void* table, float scale,
                         const void* bias, const DropArg& drop, void* out, hipStream_t stream) {
#define MG_CALL_F(T, P, ...) encode<T, P, float>(__VA_ARGS__)
#define MG_CALL_I(T, P, ...) encode<T, P, int32_t>(__VA_ARGS__)
#define MG_CALL_L(T, P, ...) encode<T, P, int64_t>(__VA_ARGS__)
  if (t.index_kind == MG_INDEX_FLOAT32) {
    MG_FOR_NORM(a.dtype, a.param_dtype, MG_CALL_F, t, a, table, scale, bias, drop, out, stream);
  }
  if (t.index_kind == MG_INDEX_INT32) {
    MG_FOR_NORM(a.dtype, a.param_dtype, MG_CALL_I, t, a, table, scale, bias, drop, out, stream);
  }
  MG_FOR_NORM(a.dtype, a.param_dtype, MG_CALL_L, t, a, table, scale, bias, drop, out, stream);
#undef MG_CALL_F
#undef MG_CALL_I
#undef MG_CALL_L
}

}  // namespace mg
