// ryft.int4_matmul: products with 4-bit weights that have a scale, and perhaps a zero point, for each group of a row's values
// (the definition stands at Int4Args in kernel_abi.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../common.h"
#include "int4_matmul.h"
#include "launch.h"

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

// ------------------------------------------------------------------------------------------------ up to 16 rows of x
// bf16 and f16, groups of a multiple of 32: the weight's bytes bound it, so they go from memory into registers once, and
// nothing else is waited for on their way. A workgroup has NT tiles of 16 rows of the weight, its eight wavefronts take every
// eighth step of 256 values, and meet in LDS at the end, in one order; where that leaves the chip idle, `parts` workgroups
// share a tile, and the last of them to arrive adds the parts, in their order too. A step's bytes are on their way while the
// one before is multiplied.
//
// Scores the 16 rows of x as the first operand: a lane's four sums are of one row of the weight, so that it needs one scale
// a group. A lane loads 32 values of a row, four lanes 128 together; the exchange between them leaves each with the values
// that a matrix instruction takes from it. Σ x comes from a product with ones.
constexpr int FEW_WAVES = 8;
constexpr int FEW_STEP = 256;

template <class X, int NT, int SPAN>
__global__ void __launch_bounds__(64 * FEW_WAVES, 2) int4_few_kernel(const Int4Args A) {
  constexpr int SPANS = FEW_STEP / SPAN, BLOCKS = SPAN / 32;
  __shared__ f32x4p sums[FEW_WAVES][NT][64];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g16 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
  const int part = blockIdx.y, K = (int)A.K;
  int lo, hi;
  int4_range(A, part, lo, hi);

  const __amdgpu_buffer_rsrc_t wb = int4_buffer(A.w + n0 * (K / 2), (A.N - n0) * (K / 2)), xb = int4_buffer(A.x, A.T * A.xs * 2);
  const Int4Groups groups(A, n0);
  uint32_t w[NT], row[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int r = (int)min((int64_t)(16 * i + l16), A.N - 1 - n0);  // (rows past the last are computed and not stored)
    w[i] = (uint32_t)r * (uint32_t)(K / 2) + 16 * g16;
    row[i] = (uint32_t)r * (uint32_t)A.groups;
  }
  const uint32_t x = l16 < A.T ? (uint32_t)(l16 * (int)A.xs + 8 * g16) * 2 : kOutside;

  struct Step {
    u32x4p w[NT][2], x[8];
    Int4Scales<SPAN, SPANS> s[NT];
  };
  auto load = [&](Step& v, int step) {
    const int k = step * FEW_STEP;
    if (k + FEW_STEP <= K) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) v.w[i][j] = int4_load<kOnce>(wb, w[i], k / 2 + 64 * j);
#pragma unroll
      for (int b = 0; b < 8; ++b) v.x[b] = int4_load<0>(xb, x, 2 * (k + 32 * b));
    } else {
      // (the row ends within the step)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          v.w[i][j] = int4_load<kOnce>(wb, k + 128 * j + 32 * g16 < K ? w[i] + (uint32_t)(k / 2 + 64 * j) : kOutside, 0);
#pragma unroll
      for (int b = 0; b < 8; ++b)
        v.x[b] = int4_load<0>(xb, k + 32 * b < K && x != kOutside ? x + (uint32_t)(2 * (k + 32 * b)) : kOutside, 0);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) v.s[i].load(A, groups, row[i], k);
  };

  f32x4p y[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) y[i] = f32x4p{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Step& v) {
    const u32x4p ones = {X::ONES, X::ONES, X::ONES, X::ONES};
    // word of block b that this lane has: the four words of lane group g are blocks' words, exchanged between the groups
    u32x4p q[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4p d = v.w[i][j];
        const auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false), b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
        const auto e = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), f = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
        q[i][j] = u32x4p{e[0], e[1], f[0], f[1]};
      }
#pragma unroll
    for (int p = 0; p < SPANS; ++p) {
      u32x4p xf[BLOCKS];
      f32x4p sx = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        xf[b] = int4_order(v.x[p * BLOCKS + b]);
        sx = X::mma16(xf[b], ones, sx);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float scale = v.s[i].template scale<X>(A, p), c = -16.f - (float)v.s[i].z[p];
        f32x4p acc;
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = c * sx[r];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
          const int at = p * BLOCKS + b;
          acc = X::mma16(xf[b], int4_operand<X>(q[i][at >> 2][at & 3]), acc);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) y[i][r] = __builtin_fmaf(scale, acc[r], y[i][r]);
      }
    }
  };
  int step = lo + wave;
  if (step < hi) {
    Step a, b;
    load(a, step);
    while (true) {
      if (step + FEW_WAVES < hi) load(b, step + FEW_WAVES);
      multiply(a);
      step += FEW_WAVES;
      if (step >= hi) break;
      if (step + FEW_WAVES < hi) load(a, step + FEW_WAVES);
      multiply(b);
      step += FEW_WAVES;
      if (step >= hi) break;
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) sums[wave][i][lane] = y[i];
  __syncthreads();
  // thread i of the first NT · 64: lane i % 64 of tile i / 64
  const int i = tid >> 6;
  f32x4p sum = {0.f, 0.f, 0.f, 0.f};
  if (i < NT) {
#pragma unroll
    for (int u = 0; u < FEW_WAVES; ++u) sum += sums[u][i][lane];
  }
  if (A.parts > 1) {
    const __amdgpu_buffer_rsrc_t ws = __builtin_amdgcn_make_buffer_rsrc((void*)(A.ws + (int64_t)blockIdx.x * A.parts * (NT * 256)), (short)0, -1, 0x00020000);
    if (i < NT) agent_put4(ws, (uint32_t)(part * NT * 64 + tid) * 16, sum);
    if (!last_to_arrive(A.counters + blockIdx.x, A.parts, &last)) return;
    if (i < NT) {
      sum = f32x4p{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int u = 0; u < A.parts; ++u) sum += agent_get4(ws, (uint32_t)(u * NT * 64 + tid) * 16);
    }
  }
  const int64_t n = n0 + 16 * i + l16;
  if (i >= NT || n >= A.N) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t t = 4 * g16 + r;
    if (t >= A.T) continue;
    if (A.y_dtype == DT_F32) ((float*)A.y)[t * A.N + n] = sum[r];
    else ((uint16_t*)A.y)[t * A.N + n] = X::put(sum[r]);
  }
}

template <class X, int NT>
void launch_few(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  const dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)a.parts), block(64 * FEW_WAVES);
  if (a.span == 128) launch_k(done, int4_few_kernel<X, NT, 128>, grid, block, 0, stream, a);
  else if (a.span == 64) launch_k(done, int4_few_kernel<X, NT, 64>, grid, block, 0, stream, a);
  else launch_k(done, int4_few_kernel<X, NT, 32>, grid, block, 0, stream, a);
}

void few_plan(Int4Args& a, int64_t* ws_floats, int64_t* counters) {
  a.kernel = INT4_FEW;
  a.tiles_t = 1;
  const int64_t steps = (a.K + FEW_STEP - 1) / FEW_STEP;
  a.steps = (int32_t)steps;
  a.tiles_n = a.N >= 16384 ? 2 : 1;
  const int64_t tiles = (a.N + 16 * a.tiles_n - 1) / (16 * a.tiles_n);
  // ranges of K until there are two workgroups a CU, each with a step for every wavefront
  a.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>(512 / tiles, steps / FEW_WAVES));
  if (a.parts > 1) {
    *ws_floats = tiles * a.parts * a.tiles_n * 256;
    *counters = tiles;
  }
}

}  // namespace

void int4_matmul_plan(Int4Args& a, int64_t* ws_floats, int64_t* counters) {
  *ws_floats = *counters = 0;
  a.kernel = INT4_ANY;
  a.parts = 1;
  if ((a.x_dtype != DT_BF16 && a.x_dtype != DT_F16) || a.G % 32 || a.T == 0) return;
  // (offsets within a tile's rows are 31 bits)
  if (a.K > (1 << 22)) return;
  a.span = a.G % 128 == 0 ? 128 : a.G % 64 == 0 ? 64 : 32;
  a.groups = (int32_t)(a.K / a.G);
  a.group_spans = a.G / a.span;
  if (a.T <= 16) return few_plan(a, ws_floats, counters);
  int4_tile_plan(a, ws_floats, counters);
}

void launch_int4_matmul(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.K < 2 || a.K % 2 || a.N < 1 || a.G < 2 || a.G % 2 || a.K % a.G)
    fail(PJRT_Error_Code_INTERNAL, "int4_matmul of a shape the kernels do not take");
  if (a.T == 0) return record_done(done, stream);
  if (a.kernel != INT4_ANY && a.parts > 1 && (!a.ws || !a.counters)) fail(PJRT_Error_Code_INTERNAL, "int4_matmul without a workspace");
  if (a.kernel == INT4_FEW) {
    if (a.T > 16) fail(PJRT_Error_Code_INTERNAL, "int4_matmul's kernel for few rows with many");
    if (a.x_dtype == DT_BF16) a.tiles_n == 2 ? launch_few<Int4BF16, 2>(a, stream, done) : launch_few<Int4BF16, 1>(a, stream, done);
    else a.tiles_n == 2 ? launch_few<Int4F16, 2>(a, stream, done) : launch_few<Int4F16, 1>(a, stream, done);
  } else if (a.kernel == INT4_TILE) {
    launch_int4_tile(a, stream, done);
  } else {
    const dim3 grid((unsigned)((a.N + 3) / 4), (unsigned)std::min<int64_t>(65535, (a.T + ANY_ROWS - 1) / ANY_ROWS));
    launch_k(done, int4_matmul_any_kernel, grid, dim3(256), 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("int4_matmul launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
