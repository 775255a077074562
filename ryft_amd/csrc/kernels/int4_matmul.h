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

// Loads through buffer descriptors: one address register a lane for the whole loop, `step` bytes on in it. A lane's place is
// inside the buffer or kOutside, which reads zeros; `step` alone never passes the buffer's end, so that nothing here depends on
// whether the hardware's check counts it.
constexpr uint32_t kOutside = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t int4_buffer(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, (int)max((int64_t)0, min(bytes, (int64_t)0x7fffffff)), 0x00020000);
}
template <int AUX>
__device__ __forceinline__ u32x4p int4_load(__amdgpu_buffer_rsrc_t r, uint32_t at, int step) {
  return __builtin_bit_cast(u32x4p, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, step, AUX));
}
constexpr int kOnce = 2;  // nt: read once, past the caches' use for it

// The groups of the rows of a weight from row n0 < N on.
struct Int4Groups {
  __amdgpu_buffer_rsrc_t s, z;
  __device__ __forceinline__ Int4Groups(const Int4Args& A, int64_t n0) {
    const int es = A.scale_dtype == DT_F32 ? 4 : 2;
    const int64_t first = n0 * A.groups, rest = (A.N - n0) * A.groups;
    s = int4_buffer((const char*)A.scale + first * es, rest * es);
    z = int4_buffer(A.zero ? (const void*)(A.zero + first) : A.scale, A.zero ? rest : 0);
  }
};
// Scales and zero points of `C` consecutive spans from value k on of the row whose groups begin `at` groups into them (spans
// past the row's end: of its last group), as they lie in memory: nothing waits for them here.
template <int SPAN, int C>
struct Int4Scales {
  uint32_t s[C], z[C];
  __device__ __forceinline__ void load(const Int4Args& A, const Int4Groups& G, uint32_t at, int k) {
    int g[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      g[i] = k / SPAN + i;
      if (A.group_spans > 1) g[i] = (int)((uint32_t)g[i] / (uint32_t)A.group_spans);
      g[i] = min(g[i], A.groups - 1);
    }
    if (A.scale_dtype == DT_F32) {
#pragma unroll
      for (int i = 0; i < C; ++i) s[i] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(G.s, (int)(4 * at), 4 * g[i], 0);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) s[i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(G.s, (int)(2 * at), 2 * g[i], 0);
    }
    if (A.zero) {
#pragma unroll
      for (int i = 0; i < C; ++i) z[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(G.z, (int)at, g[i], 0);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) z[i] = 8;
    }
  }
  template <class X>
  __device__ __forceinline__ float scale(const Int4Args& A, int i) const {
    return A.scale_dtype == DT_F32 ? __uint_as_float(s[i]) : X::lo(s[i]);
  }
};

// A workgroup's range of the K loop's steps.
__device__ __forceinline__ void int4_range(const Int4Args& A, int part, int& lo, int& hi) {
  const uint32_t each = (uint32_t)A.steps / (uint32_t)A.parts, more = (uint32_t)A.steps - each * (uint32_t)A.parts;
  lo = part * (int)each + min(part, (int)more);
  hi = lo + (int)each + (part < (int)more ? 1 : 0);
}

// k_int4_tile.hip
void int4_tile_plan(Int4Args& a, int64_t* ws_floats, int64_t* counters);
void launch_int4_tile(const Int4Args& a, hipStream_t stream, hipEvent_t done);

}  // namespace ryft
