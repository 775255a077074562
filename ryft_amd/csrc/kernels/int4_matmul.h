// Shared by the kernels of ryft.int4_matmul on the matrix cores (the definition stands at Int4Args in kernel_abi.h): 4-bit
// values as matrix operands, and the scales of their groups.
//
// A value q becomes 16 + q in x's own 16-bit type, exactly: four bits of the mantissa under a fixed exponent, for two values
// in a shift, and one instruction that masks and joins. What that adds, and the zero point, is taken off where a group's sum
// begins: (q - z) · x summed over a group = Σ (16 + q) x - (16 + z) Σ x. The group's scale multiplies the finished sum, in f32.
//
// The eight values of a word come out in the order 0 4, 1 5, 2 6, 3 7; x is put into that order.
#pragma once

#include <hip/hip_runtime.h>

#include "kernels.h"
#include "op_device.h"

namespace ryft {

struct Int4BF16 {
  typedef __bf16 x8 __attribute__((__vector_size__(8 * sizeof(__bf16))));
  static constexpr uint32_t BASE = 0x41804180u, MASK = 0x00780078u, ONES = 0x3f803f80u;
  static constexpr int SHIFT = 3;  // of the mantissa's bit that is worth 1
  __device__ static __forceinline__ f32x4p mma16(const u32x4p& a, const u32x4p& b, f32x4p c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x16p mma32(const u32x4p& a, const u32x4p& b, f32x16p c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  __device__ static __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  __device__ static __forceinline__ uint16_t put(float x) { return f32_to_bf16_bits(x); }
};
struct Int4F16 {
  typedef _Float16 x8 __attribute__((__vector_size__(8 * sizeof(_Float16))));
  static constexpr uint32_t BASE = 0x4c004c00u, MASK = 0x03c003c0u, ONES = 0x3c003c00u;
  static constexpr int SHIFT = 6;
  __device__ static __forceinline__ f32x4p mma16(const u32x4p& a, const u32x4p& b, f32x4p c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x16p mma32(const u32x4p& a, const u32x4p& b, f32x16p c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)w); }
  __device__ static __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)); }
  __device__ static __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};

// A word's eight values as 16 + q, in the order above. The constants are kept in registers: with a literal, masking and joining
// are two instructions.
template <class X>
struct Int4Operand {
  uint32_t mask = X::MASK, base = X::BASE;
  __device__ __forceinline__ Int4Operand() {
    asm volatile("" : "+s"(mask));
    asm volatile("" : "+v"(base));
  }
  __device__ __forceinline__ u32x4p operator()(uint32_t w) const {
    u32x4p f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr int S = X::SHIFT;
      const uint32_t v = 4 * i >= S ? w >> (4 * i >= S ? 4 * i - S : 0) : w << (4 * i < S ? S - 4 * i : 0);
      f[i] = (v & mask) | base;
    }
    return f;
  }
};
// Eight consecutive values of x in that order.
__device__ __forceinline__ u32x4p int4_order(const u32x4p& v) {
  return u32x4p{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// Loads go through buffer descriptors: one address register a lane for the whole loop. No lane's place is outside its buffer, so
// that nothing here depends on the hardware's check.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t int4_buffer(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, (int)max((int64_t)0, min(bytes, (int64_t)0x7fffffff)), 0x00020000);
}
constexpr int kOnce = 2;  // nt: read once, past the caches' use for it

// A workgroup's range of the K loop's steps.
__device__ __forceinline__ void int4_range(const Int4Args& A, int part, int& lo, int& hi) {
  const uint32_t each = (uint32_t)A.steps / (uint32_t)A.parts, more = (uint32_t)A.steps - each * (uint32_t)A.parts;
  lo = part * (int)each + min(part, (int)more);
  hi = lo + (int)each + (part < (int)more ? 1 : 0);
}

// k_int4_tile.hip
void int4_tile_plan(Int4Args& a, int64_t room, int64_t* ws_floats);
void launch_int4_tile(const Int4Args& a, hipStream_t stream, hipEvent_t done);

}  // namespace ryft
