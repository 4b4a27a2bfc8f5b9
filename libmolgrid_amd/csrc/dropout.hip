// Dropout whose mask is never stored (mg_dropout): it is a function of seed, offset and position,
// so the backward pass is the same call on the gradient.
#include "element_types.h"
#include "kernels.h"
#include "row_team.h"

namespace mg {
namespace {

constexpr int kThreads = 256;

// A thread takes kGroups groups of eight elements, i.e. as many counters of the generator, and has
// their loads in flight together.  Memory bound: 268 million bfloat16 in 189 us (1.07 GB, 5.7 TB/s), and
// in 186 us where nothing is dropped and the generator left out.  WHOLE: the arrays start on 16-byte
// boundaries; 67 million bfloat16 that do not take 120 us, an element a load, and 39 us where they do.
constexpr int kGroups = 2;

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const T* in, size_t n, DropArg arg,
                                                           T* out) {
  uint64_t seed, offset;
  drop_key(arg, seed, offset);
  const size_t groups = (n + 7) / 8;
  for (size_t g0 = (size_t)blockIdx.x * kThreads * kGroups + threadIdx.x; g0 < groups;
       g0 += (size_t)gridDim.x * kThreads * kGroups) {
    float v[kGroups][8];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const size_t e = (g0 + (size_t)j * kThreads) * 8;
      if (WHOLE && e + 8 <= n) {
        load_floats<T, 8>(in + e, v[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = e + i < n ? widen(in[e + i]) : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      const size_t e = (g0 + (size_t)j * kThreads) * 8;
      drop<8>(e, arg, seed, offset, v[j]);
      if (WHOLE && e + 8 <= n) {
        store_floats<T, 8>(out + e, v[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i < n) out[e + i] = narrow<T>(v[j][i]);
      }
    }
  }
}

template <typename T>
hipError_t dropout(const void* in, size_t n, const DropArg& arg, void* out, hipStream_t stream) {
  const size_t share = (size_t)kThreads * kGroups * 8;
  size_t blocks = (n + share - 1) / share;
  if (blocks > 1u << 20) blocks = 1u << 20;
  if ((address(in) | address(out)) % 16 == 0)
    hipLaunchKernelGGL((dropout_kernel<T, true>), dim3((unsigned)blocks), dim3(kThreads), 0, stream,
                       (const T*)in, n, arg, (T*)out);
  else
    hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)blocks), dim3(kThreads), 0, stream,
                       (const T*)in, n, arg, (T*)out);
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
