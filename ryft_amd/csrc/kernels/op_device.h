// Shared by the decoding operators' kernels: 16-bit floats and f32, to and from f32 values, and partial results that workgroups
// of one launch hand to each other.
#pragma once

#include "ew_device.h"

namespace ryft {

struct ElemBF16 {
  typedef uint16_t raw;
  __device__ static __forceinline__ float get(raw x) { return bf16_bits_to_f32(x); }
  __device__ static __forceinline__ raw put(float x) { return f32_to_bf16_bits(x); }
};
struct ElemF16 {
  typedef uint16_t raw;
  __device__ static __forceinline__ float get(raw x) { return (float)__builtin_bit_cast(_Float16, x); }
  __device__ static __forceinline__ raw put(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};
struct ElemF32 {
  typedef float raw;
  __device__ static __forceinline__ float get(raw x) { return x; }
  __device__ static __forceinline__ raw put(float x) { return x; }
};

// Calls f with the element type that `dtype` names (bf16, f16 or f32: custom_call.cc lets no other through).
template <class F>
inline void with_elem(int32_t dtype, F&& f) {
  if (dtype == DT_BF16) f(ElemBF16{});
  else if (dtype == DT_F16) f(ElemF16{});
  else f(ElemF32{});
}

typedef float f32x4p __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4p __attribute__((ext_vector_type(4)));
typedef float f32x16p __attribute__((__vector_size__(16 * sizeof(float))));

// Partial results move between workgroups of one launch past the XCDs' L2s (agent scope: sc1).
constexpr int kAgent = 16;
typedef uint32_t u32x4w __attribute__((__vector_size__(16)));
typedef uint32_t u32x2w __attribute__((__vector_size__(8)));
__device__ __forceinline__ void agent_put4(__amdgpu_buffer_rsrc_t r, uint32_t byte, f32x4p v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4w, v), r, (int)byte, 0, kAgent);
}
__device__ __forceinline__ f32x4p agent_get4(__amdgpu_buffer_rsrc_t r, uint32_t byte) {
  return __builtin_bit_cast(f32x4p, __builtin_amdgcn_raw_buffer_load_b128(r, (int)byte, 0, kAgent));
}
__device__ __forceinline__ void agent_put2(__amdgpu_buffer_rsrc_t r, uint32_t byte, float x, float y) {
  __builtin_amdgcn_raw_buffer_store_b64(u32x2w{__float_as_uint(x), __float_as_uint(y)}, r, (int)byte, 0, kAgent);
}
__device__ __forceinline__ float2 agent_get2(__amdgpu_buffer_rsrc_t r, uint32_t byte) {
  const u32x2w v = __builtin_amdgcn_raw_buffer_load_b64(r, (int)byte, 0, kAgent);
  return float2{__uint_as_float(v[0]), __uint_as_float(v[1])};
}

// Whether this workgroup is the last of `parts` to arrive at a counter, once all its own stores are complete. Every
// thread calls it; `last`: a word of LDS. The counter is back at zero when the last has arrived.
__device__ __forceinline__ bool last_to_arrive(int32_t* counter, int parts, int* last) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const int arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    if (arrived == parts) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *last = arrived == parts;
  }
  __syncthreads();
  return *(volatile int*)last != 0;
}

}  // namespace ryft
