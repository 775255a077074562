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

// Results that are not finite, summed again by a wavefront in 64 bits. The sums above carry 16 + q and 16 + z: an infinity of x is
// in both of them, and they may pass f32's range where the result does not (x from 2^112 on). What that leaves is infinite or NaN
// to the end, so that finite results need nothing more than the look at them, a product with 0 each (16 rows against 28672 x 4096:
// 20.0 us with and without; 2048 against 12288 x 4096: 221.5 and 220). With a NaN in every row the two take 0.1 and 2 ms, with an
// infinity 1.6 and 58 ms, with an infinity in one row 0.14 and 3.6 ms.
__device__ __forceinline__ bool int4_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// y[t, n] from its definition, eight values a lane at a time; `nan`: whether row t of x has a NaN, of which every result is NaN.
template <class X>
__device__ __forceinline__ float int4_again(const Int4Args& A, int64_t t, int64_t n, bool& nan) {
  const uint16_t* const x = (const uint16_t*)A.x + t * A.K;
  const uint32_t* const w = (const uint32_t*)(A.w + n * (A.K / 2));
  const int64_t g0 = n * A.groups;
  double sum = 0;
  bool odd = false;
#pragma unroll 1
  for (int k = 8 * (threadIdx.x & 63); k < (int)A.K; k += 512) {
    const int64_t g = g0 + (uint32_t)k / (uint32_t)A.G;
    const double s = A.scale_dtype == DT_F32 ? ((const float*)A.scale)[g] : X::lo(((const uint16_t*)A.scale)[g]);
    const int z = A.zero ? A.zero[g] : 8;
    const u32x4p v = *(const u32x4p*)(x + k);
    const uint32_t q = w[k / 8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = e & 1 ? X::hi(v[e >> 1]) : X::lo(v[e >> 1] & 0xffffu);
      odd |= f != f;
      sum = __builtin_fma(s * (double)((int)(q >> (4 * e) & 15) - z), (double)f, sum);
    }
  }
  for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m, 64);
  nan = __any(odd);
  return (float)sum;
}

// Each lane's v is y[t, n]; where `bad`, it is summed again. All lanes of the wavefront call it.
template <class X>
__device__ __forceinline__ float int4_mend(const Int4Args& A, bool bad, int64_t t, int64_t n, float v) {
  uint64_t todo = __ballot(bad);
  while (todo) {
    const int lane = __builtin_ctzll(todo);
    const int64_t row = __shfl(t, lane, 64);
    bool nan;
    const float y = int4_again<X>(A, row, __shfl(n, lane, 64), nan);
    if (nan) {  // (it is in every sum of the row already)
      todo &= ~__ballot(t == row);
      continue;
    }
    if ((int)(threadIdx.x & 63) == lane) v = y;
    todo &= todo - 1;
  }
  return v;
}

// The kernel's first argument, read again: so that what the seldom taken way needs of it is not kept in registers on the other
// (16 rows against 28672 x 4096: 20.4 us where it was).
__device__ __forceinline__ const Int4Args& int4_args_again() {
  const void* p = (const void*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Int4Args*)p;
}

// The same for y[t, n] where it lies, by the lane that has written it: at the end of a kernel, for registers that are free there.
template <class X>
__device__ __forceinline__ void int4_mend_stored(const Int4Args& A, bool mine, int64_t t, int64_t n) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const int64_t at = t * A.N + n;
  float v = 0.f;
  if (mine) v = A.y_dtype == DT_F32 ? ((const float*)A.y)[at] : X::lo(((const uint16_t*)A.y)[at]);
  const bool bad = !int4_finite(v);
  v = int4_mend<X>(A, bad, t, n, v);
  if (bad && A.y_dtype == DT_F32) ((float*)A.y)[at] = v;
  if (bad && A.y_dtype != DT_F32) ((uint16_t*)A.y)[at] = X::put(v);
}

// k_int4_tile.hip
bool int4_tile_plan(Int4Args& a, int64_t room, int64_t* ws_floats);  // false: not with that workspace
void launch_int4_tile(const Int4Args& a, hipStream_t stream, hipEvent_t done);

}  // namespace ryft
