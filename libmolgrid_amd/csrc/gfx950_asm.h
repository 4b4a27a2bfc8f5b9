// The inline assembly of the gfx950 kernels and their conversions of 16-bit types, in one place.
#ifndef LIBMOLGRID_AMD_GFX950_ASM_H_
#define LIBMOLGRID_AMD_GFX950_ASM_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mg {

// a * b with 0 * anything = 0 (also infinities and NaNs): v_mul_legacy_f32
__device__ __forceinline__ float mul_legacy(float a, float b) {
  float r;
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

// keeps a wave-uniform value in a vector register (an fma takes one scalar operand)
__device__ __forceinline__ void keep_in_vgpr(float& v) { asm volatile("" : "+v"(v)); }

// The same for an integer, used the other way round: what is computed from the value after this
// point cannot be moved in front of it (out of a loop, where it would occupy registers -- or
// scratch memory -- for the whole loop).
__device__ __forceinline__ void compute_here(int& v) { asm volatile("" : "+v"(v)); }

// workgroup barrier that waits for the wave's LDS traffic only (not for its global loads and
// stores, which __syncthreads would also wait for)
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Inside a branch on a scalar condition: keeps the compiler from turning the branch into
// unconditional code plus a select (it would for a few cheap-looking instructions, among them the
// transcendental ones this is used to skip).
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// Between the LDS writes of a wave and its own reads of what other lanes wrote (and the other
// way round).  The lanes of a wave execute an instruction together and the LDS keeps the order of
// a wave's accesses, so the hardware needs no instruction here; this only keeps the compiler from
// moving LDS accesses across the point.
__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_wave_barrier(); }

// Keeps the compiler's scheduler from mixing what comes before with what comes after: independent
// pieces of work done side by side need the registers of all of them.
__device__ __forceinline__ void one_after_the_other() { __builtin_amdgcn_sched_barrier(0); }

// a ^ b ^ c
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

// Bits of a 16-bit float type from a float (to the nearest, ties to even) and back.
__device__ __forceinline__ float half_bits_to_float(uint16_t bits) {
  return (float)__builtin_bit_cast(_Float16, bits);
}
__device__ __forceinline__ uint16_t float_to_half_bits(float v) {
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ uint16_t float_to_bfloat16_bits(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);
}
// Two at once, the first in the low half.
__device__ __forceinline__ uint32_t floats_to_half_bits(float a, float b) {
  typedef float Floats __attribute__((ext_vector_type(2)));
  typedef _Float16 Halves __attribute__((ext_vector_type(2)));
  const Floats v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, Halves));
}
__device__ __forceinline__ uint32_t floats_to_bfloat16_bits(float a, float b) {
  typedef float Floats __attribute__((ext_vector_type(2)));
  typedef __bf16 Halves __attribute__((ext_vector_type(2)));
  const Floats v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, Halves));
}

}  // namespace mg

#endif
