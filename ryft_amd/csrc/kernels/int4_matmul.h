// Shared by the kernels of ryft.int4_matmul on the matrix cores (the definition stands at Int4Args in kernel_abi.h): 4-bit
// values as matrix operands, and the scales of their groups.
//
// A value q becomes 16 + q in x's own 16-bit type, exactly: four bits of the mantissa under a fixed exponent, for two values
// in a shift, and one instruction that masks and joins. What that adds, and the zero point, is taken off where a group's sum begins: (q - z) · x
// summed over a group = Σ (16 + q) x - (16 + z) Σ x. The group's scale multiplies the finished sum, in f32.
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

// A word's eight values as 16 + q, in the order above.
template <class X>
__device__ __forceinline__ u32x4p int4_operand(uint32_t w) {
  auto pair = [](uint32_t v) { return (v & X::MASK) | X::BASE; };
  u32x4p f;
  f[0] = pair(w << X::SHIFT);
#pragma unroll
  for (int i = 1; i < 4; ++i) f[i] = pair(4 * i > X::SHIFT ? w >> (4 * i - X::SHIFT > 0 ? 4 * i - X::SHIFT : 0) : w << (X::SHIFT - 4 * i > 0 ? X::SHIFT - 4 * i : 0));
  return f;
}
// Eight consecutive values of x in that order.
__device__ __forceinline__ u32x4p int4_order(const u32x4p& v) {
  return u32x4p{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// 16 bytes (32 values) of a row of the weight, read once: past the caches' use for them.
__device__ __forceinline__ u32x4p int4_load(const uint8_t* p) { return __builtin_nontemporal_load((const u32x4p*)p); }

// Scales and zero points of `C` consecutive spans of row n from value k on (those past the row's end: of its last group),
// and what the group's sum begins with, per unit of Σ x: -(16 + zero).
template <int SPAN, int C, class X>
__device__ __forceinline__ void int4_scales(const Int4Args& A, int64_t n, int64_t k, float (&s)[C], float (&c)[C]) {
  const int64_t groups = A.K / A.G;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    int64_t g = A.G == SPAN ? k / SPAN + i : (k + i * SPAN) / A.G;
    g = n * groups + (g < groups ? g : groups - 1);
    if (A.scale_dtype == DT_F32) s[i] = ((const float*)A.scale)[g];
    else s[i] = X::lo(((const uint16_t*)A.scale)[g]);
    c[i] = A.zero ? -16.f - (float)A.zero[g] : -24.f;
  }
}

// k_int4_tile.hip
void int4_tile_plan(Int4Args& a, int64_t* ws_floats, int64_t* counters);
void launch_int4_tile(const Int4Args& a, hipStream_t stream, hipEvent_t done);

}  // namespace ryft
