// Dropout whose mask is never stored (mg_dropout): it is a function of seed, offset and position,
// so the backward pass is the same call on the gradient.
#include "element_types.h"
#include "kernels.h"

namespace mg {
namespace {

constexpr int kThreads = 256;

// One thread takes one group of eight elements, i.e. one counter of the generator.
template <typename T>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const T* in, size_t n, DropArg drop,
                                                           T* out) {
  uint64_t seed, offset;
  drop_key(drop, seed, offset);
  const size_t groups = (n + 7) / 8, stride = (size_t)gridDim.x * kThreads;
  for (size_t g = (size_t)blockIdx.x * kThreads + threadIdx.x; g < groups; g += stride) {
    const Words4 words = philox(g, offset, seed);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const size_t e = g * 8 + i;
      if (e >= n) break;
      const float v = widen(in[e]) * drop.factor;
      out[e] = narrow<T>(drop_half(words, i) >= drop.limit ? v : 0.f);
    }
  }
}

template <typename T>
hipError_t dropout(const void* in, size_t n, const DropArg& drop, void* out, hipStream_t stream) {
  size_t blocks = ((n + 7) / 8 + kThreads - 1) / kThreads;
  if (blocks > 65536) blocks = 65536;
  hipLaunchKernelGGL((dropout_kernel<T>), dim3((unsigned)blocks), dim3(kThreads), 0, stream,
                     (const T*)in, n, drop, (T*)out);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(const void* in, size_t n, int dtype, const DropArg& drop, void* out,
                          hipStream_t stream) {
  switch (dtype) {
    case MG_FLOAT32: return dropout<float>(in, n, drop, out, stream);
    case MG_FLOAT16: return dropout<Half>(in, n, drop, out, stream);
    case MG_BFLOAT16: return dropout<Bfloat16>(in, n, drop, out, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace mg
