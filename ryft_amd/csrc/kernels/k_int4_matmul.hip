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

// y[t, n] in 64 bits, by a wavefront: for a sum that left f32's range.
__device__ __forceinline__ float any_again(const Int4Args& A, int64_t t, int64_t n) {
  double sum = 0;
#pragma unroll 1
  for (uint32_t j = threadIdx.x & 63; j < (uint32_t)(A.K / 2); j += 64) {
    const int64_t g = n * ((uint32_t)A.K / (uint32_t)A.G) + 2 * j / (uint32_t)A.G;
    const double s = read_any(A.scale, g, A.scale_dtype);
    const int z = A.zero ? A.zero[g] : 8, b = A.w[n * (A.K / 2) + j];
    sum = __builtin_fma(s * (double)((b & 15) - z), (double)read_any(A.x, t * A.K + 2 * j, A.x_dtype), sum);
    sum = __builtin_fma(s * (double)((b >> 4) - z), (double)read_any(A.x, t * A.K + 2 * j + 1, A.x_dtype), sum);
  }
  for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m, 64);
  return (float)sum;
}

// Any types and groups: a wavefront a row of the weight and up to eight rows of x, a byte (two values) a lane at a time. Float and
// integer instructions bound it, two products and an address a value and row: 16 rows, 28672 x 4096: 0.85 ms in f32, 1.06 in bf16
// with groups of 16 (with the group divided for in 64 bits 1.14 and 1.52).
constexpr int ANY_ROWS = 8;
__global__ void __launch_bounds__(256) int4_matmul_any_kernel(const Int4Args A) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = (int64_t)blockIdx.x * 4 + wave;
  if (n >= A.N) return;
  const uint8_t* const w = A.w + n * (A.K / 2);
  const uint32_t half = (uint32_t)(A.K / 2);
  const int64_t groups = (uint32_t)A.K / (uint32_t)A.G;
  for (int64_t t0 = (int64_t)blockIdx.y * ANY_ROWS; t0 < A.T; t0 += (int64_t)gridDim.y * ANY_ROWS) {
    float acc[ANY_ROWS] = {};
    for (uint32_t j = lane; j < half; j += 64) {  // (K is 2^24 at most)
      const uint32_t g = 2 * j / (uint32_t)A.G;
      const float s = read_any(A.scale, n * groups + g, A.scale_dtype);
      const int z = A.zero ? A.zero[n * groups + g] : 8, b = w[j];
      const float w0 = s * (float)((b & 15) - z), w1 = s * (float)((b >> 4) - z);
#pragma unroll
      for (int r = 0; r < ANY_ROWS; ++r)
        if (t0 + r < A.T) {
          const int64_t at = (t0 + r) * A.K + 2 * j;
          acc[r] = __builtin_fmaf(w0, read_any(A.x, at, A.x_dtype), acc[r]);
          acc[r] = __builtin_fmaf(w1, read_any(A.x, at + 1, A.x_dtype), acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < ANY_ROWS; ++r) {
      for (int x = 32; x; x >>= 1) acc[r] += __shfl_xor(acc[r], x, 64);
      if (t0 + r < A.T && !int4_finite(acc[r])) acc[r] = any_again(A, t0 + r, n);
      if (lane == 0 && t0 + r < A.T) write_any(A.y, (t0 + r) * A.N + n, A.y_dtype, acc[r]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ 16 rows of x at a time
// bf16 and f16, groups of a multiple of 32: the weight's bytes bound it. A workgroup takes tiles of 16 rows of the weight, one
// after the other; its wavefronts take every W-th step of 256 values, and meet in LDS at the tile's end, in one order.
//
// Each wavefront streams its steps, weight, scales and zero points, from memory straight into a ring of its own in LDS, DEPTH
// steps deep, over the tiles' borders, in whole lines (a lane that loaded its own 16 bytes of a row, as the matrix instructions
// take them, had each of 16 neighbours on another line: 58 MB took 29 us so, 2.0 TB/s), and waits for its own loads only.
//
// x: where the wavefronts' steps of a row are S or fewer each and there is more than a tile a workgroup, every wavefront keeps
// its part of x in registers for all its tiles. Otherwise x comes through the ring, as the weight does.
//
// The products have the 16 rows of x as the first operand: a lane's four sums are of one row of the weight, so that it needs one
// scale a group. A lane reads 32 values of a row, four lanes 128 together; the exchange between them leaves each with the values
// that a matrix instruction takes from it. Σ x comes from a product with ones.
constexpr int FEW_STEP = 256, CUS = 256;

// XL: loads of two rows of x each, at least as many as there are rows. S: steps of x in registers, 0: x through the ring.
template <int SPAN, int XL, int S>
struct FewCfg {
  static constexpr int W = S || XL <= 4 ? 8 : 4;     // wavefronts (with 16 rows of x in the rings there is no room for eight)
  static constexpr int SPANS = FEW_STEP / SPAN;
  static constexpr int SL = SPANS > 4 ? 2 : 1;       // loads of a tile's scales: SPANS words a row
  static constexpr int SW = SPANS, ZW = SPANS > 4 ? 4 : 2;  // words a row of scales, of zero points
  static constexpr int X0 = 2048, S0 = X0 + (S ? 0 : XL * 1024), Z0 = S0 + SL * 256, SLOT = Z0 + 512;
  static constexpr int SUMS = W * 1024;              // bytes of a tile's sums
  static constexpr int depth(int shares) { return (160 * 1024 / shares - 256 - 2 * SUMS) / (W * SLOT); }  // with that many on a CU
  static constexpr int SHARES = !S && depth(2) >= 2 ? 2 : 1;
  static constexpr int DEPTH = depth(SHARES) < 7 ? depth(SHARES) : 7;
  static constexpr int LDS = W * DEPTH * SLOT + 2 * SUMS;
  static constexpr int LOADS = 3 + SL + (S ? 0 : XL);  // of a step
  static_assert(DEPTH >= 2, "");
};

typedef __attribute__((address_space(3))) void few_lds;

// LDS reads that the compiler does not order behind the loads on their way: waited for in their statement.
__device__ __forceinline__ void few_read_x(u32x4p (&f)[8], uint32_t a, uint32_t b) {
  asm volatile(
      "ds_read_b128 %0, %8\n ds_read_b128 %1, %9\n ds_read_b128 %2, %8 offset:128\n ds_read_b128 %3, %9 offset:128\n"
      "ds_read_b128 %4, %8 offset:256\n ds_read_b128 %5, %9 offset:256\n ds_read_b128 %6, %8 offset:384\n ds_read_b128 %7, %9 offset:384\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]), "=&v"(f[7])
      : "v"(a), "v"(b)
      : "memory");
}
// A row's 32 bytes of the weight, and its words of scales and zero points.
typedef uint32_t u32x2f __attribute__((ext_vector_type(2)));
template <int SPANS>
__device__ __forceinline__ void few_read_w(u32x4p (&f)[2], uint32_t (&s)[8], uint32_t (&z)[4], uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  if constexpr (SPANS == 2) {
    u32x2f u, v;
    asm volatile("ds_read_b64 %2, %6\n ds_read_b64 %3, %7\n ds_read_b128 %0, %4\n ds_read_b128 %1, %5\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(u), "=&v"(v)
                 : "v"(a), "v"(b), "v"(c), "v"(d)
                 : "memory");
    s[0] = u[0], s[1] = u[1], z[0] = v[0], z[1] = v[1];
  } else if constexpr (SPANS == 4) {
    u32x4p u;
    u32x2f v;
    asm volatile("ds_read_b128 %2, %6\n ds_read_b64 %3, %7\n ds_read_b128 %0, %4\n ds_read_b128 %1, %5\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(u), "=&v"(v)
                 : "v"(a), "v"(b), "v"(c), "v"(d)
                 : "memory");
    s[0] = u[0], s[1] = u[1], s[2] = u[2], s[3] = u[3], z[0] = v[0], z[1] = v[1];
  } else {
    u32x4p u, w, v;
    asm volatile("ds_read_b128 %2, %7\n ds_read_b128 %3, %7 offset:16\n ds_read_b128 %4, %8\n"
                 "ds_read_b128 %0, %5\n ds_read_b128 %1, %6\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(u), "=&v"(w), "=&v"(v)
                 : "v"(a), "v"(b), "v"(c), "v"(d)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = u[i], s[4 + i] = w[i], z[i] = v[i];
  }
}

template <int N>
__device__ __forceinline__ void few_wait() {  // until N loads or fewer are on their way
  constexpr int n = N > 63 ? 63 : N;
  __builtin_amdgcn_s_waitcnt(0x0F70 | (n & 15) | (n >> 4) << 14);
}

template <class X, int SPAN, int XL, int S>
__global__ void __launch_bounds__((64 * FewCfg<SPAN, XL, S>::W), 2) int4_few_kernel(const Int4Args A) {
  typedef FewCfg<SPAN, XL, S> C;
  constexpr int SPANS = C::SPANS, BLOCKS = SPAN / 32, W = C::W;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g16 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = (int)A.K, T = (int)A.T, N = (int)A.N, steps = A.steps;
  const int tiles = (N + 15) / 16;

  const int es = A.scale_dtype == DT_F32 ? 4 : 2;
  const __amdgpu_buffer_rsrc_t xb = int4_buffer(A.x, A.T * A.K * 2);
  uint32_t x_row[XL];  // position c of row r holds chunk c ^ (r mod 8)
#pragma unroll
  for (int h = 0; h < XL; ++h)
    x_row[h] = (uint32_t)min(2 * h + (lane >> 5), T - 1) * (uint32_t)(2 * A.K) + 16 * ((lane & 31) ^ ((2 * h + (lane >> 5)) & 7));
  const int w_chunk = (lane & 7) ^ (lane >> 3);
  char* const ring = smem + wave * (C::DEPTH * C::SLOT);
  const uint32_t ring_at = (uint32_t)(uintptr_t)(few_lds*)ring;
  if (!A.zero) {
    // (the zero points that the loads below leave alone)
#pragma unroll
    for (int d = 0; d < C::DEPTH; ++d) ((uint32_t*)(ring + d * C::SLOT + C::Z0))[lane] = 0x08080808u;
  }

  // First group of step `step`, of those that a row has.
  auto first_group = [&](int step) {
    int g = step * SPANS;
    if (A.group_spans > 1) g = (int)((uint32_t)g / (uint32_t)A.group_spans);
    return min(g, A.groups - 1);
  };
  // Steps on one line: of tile blockIdx.x, + gridDim.x, ... one after the other.
  struct Place {
    int tile, step;
  };
  auto rows_of = [&](int tile) { return min(16, N - tile * 16); };  // (rows past the last are computed as it, not stored)
  // Loads of a step at `ahead`: places of a lane within its tile's rows. A row of the weight has eight chunks of 16 bytes a step,
  // one of x 32: position c of row r holds chunk c ^ (r mod 8), so that the reads below take different banks. Scales and zero
  // points come in whole words (a tile's begin with one; the last of an odd number of 16-bit scales lies in one with two bytes that belong to no one, as
  // the last zero points may). Loads never leave the buffers: of a step that a row ends in, chunks past its end are read from
  // its beginning, and words past the last as that.
  Place ahead;
  uint32_t w_row[2], s_row[C::SL], z_row;
  __amdgpu_buffer_rsrc_t wb, sb, zb;
  uint32_t s_last = 0, z_last = 0;
  const int64_t w_next = (int64_t)16 * (K / 2), s_next = (int64_t)16 * A.groups * es, z_next = (int64_t)16 * A.groups;  // bytes of a tile: whole words
  auto places = [&](int rows) {
#pragma unroll
    for (int h = 0; h < 2; ++h) w_row[h] = (uint32_t)min(8 * h + (lane >> 3), rows - 1) * (uint32_t)(K / 2) + 16 * w_chunk;
#pragma unroll
    for (int h = 0; h < C::SL; ++h) s_row[h] = (uint32_t)(min((64 * h + lane) / C::SW, rows - 1) * A.groups) * es;
    z_row = (uint32_t)(min(lane / C::ZW, rows - 1) * A.groups);
  };
  auto enter = [&]() {  // `ahead` is at a tile's first step
    const int rows = rows_of(ahead.tile);
    const uint32_t s_bytes = (uint32_t)min((int64_t)(N - ahead.tile * 16) * A.groups * es + 3, (int64_t)0x7ffffffc) & ~3u;
    const uint32_t z_bytes = (uint32_t)min((int64_t)(N - ahead.tile * 16) * A.groups + 3, (int64_t)0x7ffffffc) & ~3u;
    wb = int4_buffer(A.w + ahead.tile * w_next, (int64_t)rows * (K / 2));
    sb = int4_buffer((const char*)A.scale + ahead.tile * s_next, s_bytes);
    zb = A.zero ? int4_buffer(A.zero + ahead.tile * z_next, z_bytes) : sb;
    s_last = s_bytes - 4, z_last = (A.zero ? z_bytes : s_bytes) - 4;
    if (rows < 16) places(rows);
  };
  const int z_to = A.zero ? C::Z0 : C::Z0 + 256;
  auto fetch = [&](int slot) {
    const int step = ahead.step, k = step * FEW_STEP;
    char* const to = ring + slot * C::SLOT;
    const bool whole = k + FEW_STEP <= K;
    if (whole) {
#pragma unroll
      for (int h = 0; h < 2; ++h) __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, (few_lds*)(to + h * 1024), 16, (int)w_row[h], k / 2, 0, kOnce);
      if constexpr (S == 0) {
#pragma unroll
        for (int h = 0; h < XL; ++h) __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, (few_lds*)(to + C::X0 + h * 1024), 16, (int)x_row[h], 2 * k, 0, 0);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = k + 32 * w_chunk < K ? w_row[h] + k / 2 : w_row[h] - 16 * w_chunk;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, (few_lds*)(to + h * 1024), 16, (int)at, 0, 0, kOnce);
      }
      if constexpr (S == 0) {
#pragma unroll
        for (int h = 0; h < XL; ++h) {
          const int chunk = (lane & 31) ^ ((2 * h + (lane >> 5)) & 7);
          const uint32_t at = k + 8 * chunk < K ? x_row[h] + 2 * k : x_row[h] - 16 * chunk;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, (few_lds*)(to + C::X0 + h * 1024), 16, (int)at, 0, 0, 0);
        }
      }
    }
    const uint32_t g = (uint32_t)first_group(step);
#pragma unroll
    for (int h = 0; h < C::SL; ++h) {
      const uint32_t at = ((s_row[h] + g * es) & ~3u) + 4 * ((64 * h + lane) % C::SW);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sb, (few_lds*)(to + C::S0 + h * 256), 4, (int)min(at, s_last), 0, 0, 0);
    }
    // (without zero points some of the scales, to a place that no one reads: for the number of loads)
    const uint32_t z = ((z_row + g) & ~3u) + 4 * (lane % C::ZW);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(zb, (few_lds*)(to + z_to), 4, (int)min(z, z_last), 0, 0, 0);
    ahead.step += W;
    if (ahead.step >= steps) {
      ahead.step = wave, ahead.tile += (int)gridDim.x;
      if (ahead.tile < tiles) enter();
    }
  };
  // Waits until the oldest of `later` + 1 steps on their way is there.
  auto arrived = [&](int later) {
    asm volatile("" ::: "memory");
    constexpr int L = C::LOADS, D = C::DEPTH - 1;
    if (later >= D) few_wait<D * L>();
    else if (D > 4 && later >= 4) few_wait<4 * L>();
    else if (D > 2 && later >= 2) few_wait<2 * L>();
    else if (D > 1 && later == 1) few_wait<L>();
    else few_wait<0>();
    asm volatile("" ::: "memory");
  };

  const Int4Operand<X> operand;
  const u32x4p ones = {X::ONES, X::ONES, X::ONES, X::ONES};
  f32x4p y;
  uint32_t row;  // groups before this lane's row of the tile
  const int xl = min(l16, 2 * XL - 1);  // (rows that there are not: of the last, and not stored)
  const uint32_t w_at = ring_at + l16 * 128, w_pos = 16 * (g16 ^ (l16 & 7)), x_at = ring_at + C::X0 + xl * 512, x_pos = 16 * (g16 ^ (xl & 7));
  const uint32_t s_at = ring_at + C::S0 + l16 * (4 * C::SW), z_at = ring_at + C::Z0 + l16 * (4 * C::ZW);
  // the part of x in registers, in a word's order, and its sums where they are few
  constexpr bool SUMMED = S > 0 && SPAN == 128;
  u32x4p x_own[S ? S : 1][8];
  f32x4p x_sum[SUMMED ? S : 1][SPANS];
  if constexpr (S > 0) {
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int at = 0; at < 8; ++at) {
        const int k = (wave + W * s) * FEW_STEP + 32 * at + 8 * g16;
        x_own[s][at] = u32x4p{0u, 0u, 0u, 0u};
        if (k < K) x_own[s][at] = *(const u32x4p*)((const uint16_t*)A.x + (int64_t)min(l16, T - 1) * A.K + k);
      }
  }
  auto multiply = [&](int step, int slot, const u32x4p (&xo)[8], const f32x4p (&xs)[SPANS]) {
    const uint32_t off = (uint32_t)slot * C::SLOT;
    u32x4p xv[8], wv[2];
    uint32_t sv[8], zv[4];
    if constexpr (S == 0) few_read_x(xv, x_at + off + x_pos, x_at + off + (x_pos ^ 64));
    few_read_w<SPANS>(wv, sv, zv, w_at + off + w_pos, w_at + off + (w_pos ^ 64), s_at + off, z_at + off);
    // scales and zero points of the step's spans (0 past the row's end)
    float scale[SPANS], c[SPANS];
    const uint32_t g0 = (uint32_t)first_group(step);
    const int left = (K - step * FEW_STEP) / SPAN;
    const uint32_t before = row + g0;
#pragma unroll
    for (int p = 0; p < SPANS; p += 4) {
      const uint32_t z = __builtin_amdgcn_alignbyte(zv[p / 4 + 1], zv[p / 4], A.zero ? before & 3 : 0);
#pragma unroll
      for (int e = 0; e < 4 && p + e < SPANS; ++e) c[p + e] = -16.f - (float)(z >> (8 * e) & 255u);
    }
    if (es == 4) {
#pragma unroll
      for (int p = 0; p < SPANS; ++p) scale[p] = __uint_as_float(sv[p]);
    } else {
#pragma unroll
      for (int p = 0; p < SPANS; p += 2) {
        const uint32_t w = __builtin_amdgcn_alignbyte(sv[p / 2 + 1], sv[p / 2], 2 * before & 2);
        scale[p] = X::lo(w & 0xffffu), scale[p + 1] = X::hi(w);
      }
    }
    if (A.group_spans > 1) {
      // (several spans a group: of the groups that were read, each the one that it lies in)
      float s1[SPANS], c1[SPANS];
#pragma unroll
      for (int p = 0; p < SPANS; ++p) {
        const int g = (int)((uint32_t)(step * SPANS + p) / (uint32_t)A.group_spans) - (int)g0;
        s1[p] = scale[0], c1[p] = c[0];
#pragma unroll
        for (int j = 1; j < SPANS; ++j) s1[p] = g == j ? scale[j] : s1[p], c1[p] = g == j ? c[j] : c1[p];
      }
#pragma unroll
      for (int p = 0; p < SPANS; ++p) scale[p] = s1[p], c[p] = c1[p];
    }
    if (left < SPANS) {
#pragma unroll
      for (int p = 1; p < SPANS; ++p)
        if (p >= left) scale[p] = 0.f;
    }
    // word of block b that this lane has: the four words of lane group g are blocks' words, exchanged between the groups
    u32x4p q[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4p d = wv[j];
      const auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false), b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
      const auto e = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), f = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
      q[j] = u32x4p{e[0], e[1], f[0], f[1]};
    }
#pragma unroll
    for (int p = 0; p < SPANS; ++p) {
      f32x4p sx = {0.f, 0.f, 0.f, 0.f}, acc = {0.f, 0.f, 0.f, 0.f};
      if constexpr (SUMMED) sx = xs[p];
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const int at = p * BLOCKS + b;
        const u32x4p xf = S ? xo[at] : int4_order(xv[at]);
        if constexpr (!SUMMED) sx = X::mma16(xf, ones, sx);
        acc = X::mma16(xf, operand(q[at >> 2][at & 3]), acc);
      }
#pragma unroll
      for (int r = 0; r < (XL == 1 ? 2 : 4); ++r) y[r] = __builtin_fmaf(scale[p], __builtin_fmaf(c[p], sx[r], acc[r]), y[r]);
    }
  };
  Place here{(int)blockIdx.x, wave};
  if (here.step >= steps) here.tile = tiles;  // (a wavefront without steps only takes part in the sums)
  ahead = here;
  places(16);
  if (ahead.tile < tiles) enter();
  int slot = 0, to = 0, count = 0;  // count: steps on their way
#pragma unroll 1
  for (int d = 0; d < C::DEPTH - 1 && ahead.tile < tiles; ++d, ++count, ++to) fetch(to);
  if constexpr (S > 0) {
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int at = 0; at < 8; ++at) x_own[s][at] = int4_order(x_own[s][at]);
    if constexpr (SUMMED) {
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int p = 0; p < SPANS; ++p) {
          x_sum[s][p] = f32x4p{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b) x_sum[s][p] = X::mma16(x_own[s][p * BLOCKS + b], ones, x_sum[s][p]);
        }
    }
  }
  int turn = 0;
  float odd = 0.f;  // NaN where a sum of the tiles that this wavefront has finished is not finite (in a vector register: those are left)
  auto forward = [&]() {  // has the next step loaded and waits for the oldest
    if (ahead.tile < tiles) {
      fetch(to);
      ++count;
      if (++to == C::DEPTH) to = 0;
    }
    arrived(--count);
  };
  for (int tile = blockIdx.x; tile < tiles; tile += (int)gridDim.x, ++turn) {
    y = f32x4p{0.f, 0.f, 0.f, 0.f};
    row = (uint32_t)(min(l16, rows_of(tile) - 1) * A.groups);
    if constexpr (S > 0) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (wave + W * s >= steps) break;
        forward();
        multiply(wave + W * s, slot, x_own[s], x_sum[SUMMED ? s : 0]);
        if (++slot == C::DEPTH) slot = 0;
      }
    } else {
#pragma unroll 1
      while (here.tile == tile) {
        forward();
        multiply(here.step, slot, x_own[0], x_sum[0]);
        if (++slot == C::DEPTH) slot = 0;
        here.step += W;
        if (here.step >= steps) here.step = wave, here.tile += (int)gridDim.x;
      }
    }
    // The wavefronts' sums, by turns in one of two places: a wavefront writes one again only after all have passed the barrier
    // of the tile between.
    const uint32_t sums = (uint32_t)(uintptr_t)(few_lds*)(smem + W * C::DEPTH * C::SLOT + (turn & 1) * C::SUMS);  // [W][64]
    asm volatile("ds_write_b128 %0, %1\n s_waitcnt lgkmcnt(0)" ::"v"(sums + (wave * 64 + lane) * 16), "v"(y) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (wave != turn % W) continue;  // (the wavefronts finish tiles by turns)
    f32x4p sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < W; u += 4) {
      f32x4p v[4];
      asm volatile("ds_read_b128 %0, %4\n ds_read_b128 %1, %4 offset:%5\n ds_read_b128 %2, %4 offset:%6\n"
                   "ds_read_b128 %3, %4 offset:%7\n s_waitcnt lgkmcnt(0)"
                   : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
                   : "v"(sums + (u * 64 + lane) * 16), "i"(1024), "i"(2 * 1024), "i"(3 * 1024)
                   : "memory");
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += v[j];
    }
    const int n = tile * 16 + l16;
#pragma unroll
    for (int r = 0; r < 4; ++r) odd = __builtin_fmaf(sum[r], 0.f, odd);
    if (n >= N) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 4 * g16 + r;
      if (t >= T) continue;
      if (A.y_dtype == DT_F32) ((float*)A.y)[(int64_t)t * N + n] = sum[r];
      else ((uint16_t*)A.y)[(int64_t)t * N + n] = X::put(sum[r]);
    }
  }
  if (!__any(odd != odd)) return;
  const Int4Args& B = int4_args_again();
  turn = 0;
#pragma unroll 1
  for (int64_t n0 = (int64_t)blockIdx.x * 16; n0 < B.N; n0 += (int64_t)gridDim.x * 16, ++turn) {
    if (wave != turn % W) continue;
#pragma unroll 1
    for (int t = 4 * g16; t < 4 * g16 + 4; ++t) int4_mend_stored<X>(B, t < B.T && n0 + l16 < B.N, t, n0 + l16);
  }
}

template <class X, int SPAN, int XL, int S>
void launch_few_of(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  typedef FewCfg<SPAN, XL, S> C;
  const hipError_t e = hipFuncSetAttribute((const void*)int4_few_kernel<X, SPAN, XL, S>, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("int4_matmul LDS attribute: ") + hipGetErrorString(e));
  const dim3 grid((unsigned)std::min<int64_t>((a.N + 15) / 16, C::SHARES * CUS));
  const int ys = a.y_dtype == DT_F32 ? 4 : 2;
  for (int64_t t0 = 0; t0 < a.T; t0 += 16) {
    Int4Args b = a;
    b.x = (const char*)a.x + t0 * a.K * 2;
    b.y = (char*)a.y + t0 * a.N * ys;
    b.T = std::min<int64_t>(16, a.T - t0);
    launch_k(t0 + 16 >= a.T ? done : nullptr, int4_few_kernel<X, SPAN, XL, S>, grid, dim3(64 * C::W), C::LDS, stream, b);
  }
}
template <class X, int SPAN>
void launch_few_span(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.x_steps == 1) launch_few_of<X, SPAN, 8, 1>(a, stream, done);
  else if (a.x_steps == 2) launch_few_of<X, SPAN, 8, 2>(a, stream, done);
  else if (a.x_steps == 4) launch_few_of<X, SPAN, 8, 4>(a, stream, done);
  else if (a.T <= 2) launch_few_of<X, SPAN, 1, 0>(a, stream, done);
  else if (a.T <= 8) launch_few_of<X, SPAN, 4, 0>(a, stream, done);
  else launch_few_of<X, SPAN, 8, 0>(a, stream, done);
}
template <class X>
void launch_few(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.span == 128) launch_few_span<X, 128>(a, stream, done);
  else if (a.span == 64) launch_few_span<X, 64>(a, stream, done);
  else launch_few_span<X, 32>(a, stream, done);
}

void few_plan(Int4Args& a) {
  a.kernel = INT4_FEW;
  a.steps = (int32_t)((a.K + FEW_STEP - 1) / FEW_STEP);
  // x in registers: 16 rows, 4096 values against 28672 rows of the weight, bf16: 20.5 us, through the ring 29.8; 4 rows against
  // 12288: 11.2 and 11.6. Not for one or two rows, of which a step's x is an eighth of the weight's bytes (28672 rows: 19.4 and
  // 17.5), nor with a tile or less a workgroup (4096 x 4096, one row: 6.3 and 5.4).
  if ((a.N + 15) / 16 > CUS && a.T > 2) a.x_steps = a.steps <= 8 ? 1 : a.steps <= 16 ? 2 : a.steps <= 32 ? 4 : 0;
}

}  // namespace

void int4_matmul_plan(Int4Args& a, int64_t room, int64_t* ws_floats) {
  *ws_floats = 0;
  a.kernel = INT4_ANY;
  a.parts = 1;
  if ((a.x_dtype != DT_BF16 && a.x_dtype != DT_F16) || a.G % 32 || a.T == 0) return;
  // (offsets within a tile's rows are 31 bits)
  if (a.K > (1 << 22)) return;
  a.span = a.G % 128 == 0 ? 128 : a.G % 64 == 0 ? 64 : 32;
  a.groups = (int32_t)(a.K / a.G);
  a.group_spans = a.G / a.span;
  // (16 rows, 4096 x 28672: 20.5 us, with tiles 30; 14336 x 4096: 16.7 and 24; 4096 x 4096: 7.2 and 15. From 17 rows on a
  // second pass over the weight would be needed.)
  if (a.T <= 16) return few_plan(a);
  // Rows too long for tiles in that workspace go 16 at a time: 32 rows of 2^20 values take 71 MB or more, 17 of 2^22 151 or more,
  // and the scratch of allocation-free executions is 64 MiB.
  if (!int4_tile_plan(a, room, ws_floats)) few_plan(a);
}

void launch_int4_matmul(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.K < 2 || a.K % 2 || a.N < 1 || a.G < 2 || a.G % 2 || a.K % a.G)
    fail(PJRT_Error_Code_INTERNAL, "int4_matmul of a shape the kernels do not take");
  if (a.T == 0) return record_done(done, stream);
  if (a.kernel == INT4_FEW) {
    if (a.x_dtype == DT_BF16) launch_few<Int4BF16>(a, stream, done);
    else launch_few<Int4F16>(a, stream, done);
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
