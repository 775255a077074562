// ryft.int4_matmul: products with 4-bit weights that have a scale, and perhaps a zero point, for each group of a row's values
// (the definition stands at Int4Args in kernel_abi.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../common.h"
#include "kernels.h"
#include "launch.h"
#include "op_device.h"

namespace ryft {

namespace {

__device__ __forceinline__ float read_any(const void* p, int64_t i, int dtype) {
  if (dtype == DT_BF16) return ElemBF16::get(((const uint16_t*)p)[i]);
  if (dtype == DT_F16) return ElemF16::get(((const uint16_t*)p)[i]);
  return ((const float*)p)[i];
}
__device__ __forceinline__ void write_any(void* p, int64_t i, int dtype, float v) {
  if (dtype == DT_BF16) ((uint16_t*)p)[i] = ElemBF16::put(v);
  else if (dtype == DT_F16) ((uint16_t*)p)[i] = ElemF16::put(v);
  else ((float*)p)[i] = v;
}

// Any types and groups: a wavefront a row of the weight and up to eight rows of x, a byte (two values) a lane at a time.
constexpr int ANY_ROWS = 8;
__global__ void __launch_bounds__(256) int4_matmul_any_kernel(const Int4Args A) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = (int64_t)blockIdx.x * 4 + wave, groups = A.K / A.G;
  if (n >= A.N) return;
  const uint8_t* const w = A.w + n * (A.K / 2);
  for (int64_t t0 = (int64_t)blockIdx.y * ANY_ROWS; t0 < A.T; t0 += (int64_t)gridDim.y * ANY_ROWS) {
    float acc[ANY_ROWS] = {};
    for (int64_t j = lane; j < A.K / 2; j += 64) {
      const int64_t g = 2 * j / A.G;
      const float s = read_any(A.scale, n * groups + g, A.scale_dtype);
      const int z = A.zero ? A.zero[n * groups + g] : 8, b = w[j];
      const float w0 = s * (float)((b & 15) - z), w1 = s * (float)((b >> 4) - z);
#pragma unroll
      for (int r = 0; r < ANY_ROWS; ++r)
        if (t0 + r < A.T) {
          const int64_t at = (t0 + r) * A.xs + 2 * j;
          acc[r] = __builtin_fmaf(w0, read_any(A.x, at, A.x_dtype), acc[r]);
          acc[r] = __builtin_fmaf(w1, read_any(A.x, at + 1, A.x_dtype), acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < ANY_ROWS; ++r) {
      for (int x = 32; x; x >>= 1) acc[r] += __shfl_xor(acc[r], x, 64);
      if (lane == 0 && t0 + r < A.T) write_any(A.y, (t0 + r) * A.N + n, A.y_dtype, acc[r]);
    }
  }
}

}  // namespace

void launch_int4_matmul(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.K < 2 || a.K % 2 || a.N < 1 || a.G < 2 || a.G % 2 || a.K % a.G)
    fail(PJRT_Error_Code_INTERNAL, "int4_matmul of a shape the kernels do not take");
  if (a.T == 0) return record_done(done, stream);
  const dim3 grid((unsigned)((a.N + 3) / 4), (unsigned)std::min<int64_t>(65535, (a.T + ANY_ROWS - 1) / ANY_ROWS));
  launch_k(done, int4_matmul_any_kernel, grid, dim3(256), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("int4_matmul launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
