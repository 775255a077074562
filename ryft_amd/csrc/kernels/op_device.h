// Element access shared by the decoding operators' kernels: 16-bit floats and f32, to and from f32 values.
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

}  // namespace ryft
