// ryft.int4_matmul with more than 16 rows of x, bf16 and f16, groups of a multiple of 32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../common.h"
#include "int4_matmul.h"
#include "launch.h"

namespace ryft {

namespace {

constexpr int STAGE = 128;  // values of x a stage

template <int MT, int SPAN>
struct TileCfg {
  static constexpr int BM = 32 * MT, SPANS = STAGE / SPAN;
  static constexpr int XB = BM * STAGE * 2;         // bytes of a stage's x
  static constexpr int LDS1 = XB + BM * SPANS * 16;  // and of the terms of its sums
};

// Sum over the lanes of 4, 8 or 16 that have a span's chunks of eight values.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
template <int SPAN>
__device__ __forceinline__ float span_sum(float v) {
  v = dpp_add<0xb1>(v);  // quad_perm 1 0 3 2
  v = dpp_add<0x4e>(v);  // quad_perm 2 3 0 1
  if constexpr (SPAN >= 64) v = dpp_add<0x141>(v);   // row_half_mirror
  if constexpr (SPAN >= 128) v = dpp_add<0x140>(v);  // row_mirror
  return v;
}

// Terms of a span's sum S that a matrix instruction multiplies by -(16 + z): S = a · H + b + c, each rounded to 16 bits (a: a
// power of two that keeps f16 from overflowing), so that nothing of S's 24 bits is lost.
template <class X>
struct SumTerms;
template <>
struct SumTerms<Int4BF16> {
  static constexpr float H = 1.f;
};
template <>
struct SumTerms<Int4F16> {
  static constexpr float H = 256.f;
};
template <class X>
__device__ __forceinline__ u32x4p sum_terms(float s) {
  const uint32_t a = X::put(s * (1.f / SumTerms<X>::H));
  const float r = s - SumTerms<X>::H * X::lo(a);
  const uint32_t b = X::put(r), c = X::put(r - X::lo(b));
  return u32x4p{a | b << 16, c | a << 16, b | c << 16, 0u};
}
template <class X>
__device__ __forceinline__ u32x4p sum_factors(uint32_t zero, bool mine) {
  if (!mine) return u32x4p{0u, 0u, 0u, 0u};
  const float z = (float)zero;
  const uint32_t a1 = X::put(-16.f * SumTerms<X>::H), b1 = X::put(-16.f), a2 = X::put(-z * SumTerms<X>::H), b2 = X::put(-z);
  return u32x4p{a1 | b1 << 16, b1 | a2 << 16, b2 | b2 << 16, 0u};
}

__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <class X, int MT, int NW, int SPAN, int OCC>
__global__ void __launch_bounds__(256, OCC) int4_tile_kernel(const Int4Args A) {
  typedef TileCfg<MT, SPAN> C;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int last;
  constexpr int BN = 128 * NW, SPANS = C::SPANS, FR = SPAN / 16, CH = C::BM * 16 / 256;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles_n = (int)((A.N + BN - 1) / BN), tiles_t = (int)((A.T + C::BM - 1) / C::BM);
  const int tile = blockIdx.x;
  const int tn = tile / tiles_t, tt = tile - tn * tiles_t, part = blockIdx.y;
  const int64_t t0 = (int64_t)tt * C::BM, n0 = (int64_t)tn * BN;
  const int K = (int)A.K;
  int lo, hi;
  int4_range(A, part, lo, hi);

  const __amdgpu_buffer_rsrc_t wb = int4_buffer(A.w + n0 * (K / 2), (A.N - n0) * (K / 2));
  const __amdgpu_buffer_rsrc_t xb = int4_buffer((const uint16_t*)A.x + t0 * A.xs, (A.T - t0) * A.xs * 2);
  const Int4Groups groups(A, n0);
  uint32_t w[NW], row[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int r = (int)min((int64_t)(wave * (32 * NW) + 32 * i + l32), A.N - 1 - n0);  // (rows past the last are computed and not stored)
    w[i] = (uint32_t)r * (uint32_t)(K / 2) + 16 * half;
    row[i] = (uint32_t)r * (uint32_t)A.groups;
  }
  // chunk j of this thread: row 16 j + tid / 16 of the tile, values 8 · (tid % 16) on
  const int xr = tid >> 4, xc = tid & 15;
  uint32_t x[CH];
#pragma unroll
  for (int j = 0; j < CH; ++j)
    x[j] = t0 + 16 * j + xr < A.T ? (uint32_t)((16 * j + xr) * (int)A.xs + 8 * xc) * 2 : kOutside;

  u32x4p xs[CH], q[NW][2];
  Int4Scales<SPAN, SPANS> sc[NW];
  auto load_x = [&](int stage) {
    const int k = stage * STAGE;
    if (k + STAGE <= K) {
#pragma unroll
      for (int j = 0; j < CH; ++j) xs[j] = int4_load<0>(xb, x[j], 2 * k);
    } else {
      // (the row ends within the stage)
#pragma unroll
      for (int j = 0; j < CH; ++j) xs[j] = int4_load<0>(xb, k + 8 * xc < K && x[j] != kOutside ? x[j] + (uint32_t)(2 * k) : kOutside, 0);
    }
  };
  auto load_w = [&](int stage) {
    const int k = stage * STAGE;
    const bool whole = k + STAGE <= K;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (whole) q[i][j] = int4_load<0>(wb, w[i], k / 2 + 32 * j);
        else q[i][j] = int4_load<0>(wb, k + 64 * j + 32 * half < K ? w[i] + (uint32_t)(k / 2 + 32 * j) : kOutside, 0);
      }
      sc[i].load(A, groups, row[i], k);
    }
  };
  auto store_x = [&](int buffer) {
    char* const to = smem + buffer * C::LDS1;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int r = 16 * j + xr;
      float v = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) v += X::lo(xs[j][e]) + X::hi(xs[j][e]);
      v = span_sum<SPAN>(v);
      *(u32x4p*)(to + r * (STAGE * 2) + 16 * (xc ^ (r & 15))) = int4_order(xs[j]);
      if (xc % (SPAN / 8) == 0) *(u32x4p*)(to + C::XB + (xc / (SPAN / 8) * C::BM + r) * 16) = sum_terms<X>(v);
    }
  };

  // where a lane's block f of a stage's first span lies: row l32, chunk 2 f + half (and 32 FR bytes on, by exclusive or, the next)
  uint32_t chunk[FR];
#pragma unroll
  for (int f = 0; f < FR; ++f) chunk[f] = l32 * (STAGE * 2) + 16 * ((2 * f + half) ^ (l32 & 15));

  f32x16p y[MT][NW];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < NW; ++i) y[m][i] = f32x16p{};

  if (lo < hi) {
    load_x(lo);
    load_w(lo);
    store_x(0);
    lds_barrier();
    for (int stage = lo; stage < hi; ++stage) {
      const char* const from = smem + ((stage - lo) & 1) * C::LDS1;
      // the words that the matrix instructions take: block f of 16 values, words exchanged between the half-waves
      uint32_t word[NW][8];
      Int4Scales<SPAN, SPANS> now[NW];
#pragma unroll
      for (int i = 0; i < NW; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const auto a = __builtin_amdgcn_permlane32_swap(q[i][j][0], q[i][j][1], false, false);
          const auto b = __builtin_amdgcn_permlane32_swap(q[i][j][2], q[i][j][3], false, false);
          word[i][4 * j] = a[0], word[i][4 * j + 1] = b[0], word[i][4 * j + 2] = a[1], word[i][4 * j + 3] = b[1];
        }
        now[i] = sc[i];
      }
      if (stage + 1 < hi) {
        load_x(stage + 1);
        load_w(stage + 1);
      }
      // (a loop: the compiler would put off the sums of one span behind the products of the next, past the registers)
#pragma unroll 1
      for (int p = 0; p < SPANS; ++p) {
        u32x4p wf[NW][FR], zf[NW];
        float scale[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          zf[i] = sum_factors<X>(now[i].z[0], half == 0);
          scale[i] = now[i].template scale<X>(A, 0);
#pragma unroll
          for (int f = 0; f < FR; ++f) wf[i][f] = int4_operand<X>(word[i][f]);
#pragma unroll
          for (int f = 0; f + FR < 8; ++f) word[i][f] = word[i][f + FR];  // (the next span's come first)
#pragma unroll
          for (int j = 0; j + 1 < SPANS; ++j) now[i].s[j] = now[i].s[j + 1], now[i].z[j] = now[i].z[j + 1];
        }
        const char* const sums = from + C::XB + (p * C::BM + l32) * 16;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          f32x16p acc[NW];
          const u32x4p sf = *(const u32x4p*)(sums + 32 * m * 16);
#pragma unroll
          for (int i = 0; i < NW; ++i) acc[i] = X::mma32(sf, zf[i], f32x16p{});
#pragma unroll
          for (int f = 0; f < FR; ++f) {
            const u32x4p xf = *(const u32x4p*)(from + (chunk[f] ^ (p * (32 * FR))) + 32 * m * (STAGE * 2));
#pragma unroll
            for (int i = 0; i < NW; ++i) acc[i] = X::mma32(xf, wf[i][f], acc[i]);
          }
#pragma unroll
          for (int i = 0; i < NW; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) y[m][i][e] = __builtin_fmaf(scale[i], acc[i][e], y[m][i][e]);
        }
      }
      if (stage + 1 < hi) {
        store_x((stage + 1 - lo) & 1);
        lds_barrier();
      }
    }
  }
  if (A.parts > 1) {
    // (partial sums as they lie in the registers: 16 bytes a lane)
    constexpr int PART = MT * NW * 4096;  // floats of a workgroup's tile
    const __amdgpu_buffer_rsrc_t ws = __builtin_amdgcn_make_buffer_rsrc((void*)(A.ws + (int64_t)tile * A.parts * PART), (short)0, -1, 0x00020000);
    auto at = [&](int u, int m, int i, int e) { return (uint32_t)((u * (MT * NW * 4) + (m * NW + i) * 4 + e) * 256 + tid) * 16; };
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) agent_put4(ws, at(part, m, i, e), f32x4p{y[m][i][4 * e], y[m][i][4 * e + 1], y[m][i][4 * e + 2], y[m][i][4 * e + 3]});
    if (!last_to_arrive(A.counters + tile, A.parts, &last)) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < NW; ++i) y[m][i] = f32x16p{};
    for (int u = 0; u < A.parts; ++u) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < NW; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x4p v = agent_get4(ws, at(u, m, i, e));
#pragma unroll
            for (int f = 0; f < 4; ++f) y[m][i][4 * e + f] += v[f];
          }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const int64_t n = n0 + wave * (32 * NW) + 32 * i + l32;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t t = t0 + 32 * m + 8 * (e >> 2) + 4 * half + (e & 3);
        if (n < A.N && t < A.T) {
          if (A.y_dtype == DT_F32) ((float*)A.y)[t * A.N + n] = y[m][i][e];
          else ((uint16_t*)A.y)[t * A.N + n] = X::put(y[m][i][e]);
        }
      }
    }
}

template <class X, int MT, int NW, int OCC>
void launch_tile(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  const int64_t tiles = ((a.T + 32 * MT - 1) / (32 * MT)) * ((a.N + 128 * NW - 1) / (128 * NW));
  if (tiles > INT32_MAX) fail(PJRT_Error_Code_INTERNAL, "int4_matmul of too many tiles");
  const dim3 grid((unsigned)tiles, (unsigned)a.parts), block(256);
  auto go = [&](auto kernel, int lds) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("int4_matmul LDS attribute: ") + hipGetErrorString(e));
    launch_k(done, kernel, grid, block, lds, stream, a);
  };
  if (a.span == 128) go(int4_tile_kernel<X, MT, NW, 128, OCC>, 2 * TileCfg<MT, 128>::LDS1);
  else if (a.span == 64) go(int4_tile_kernel<X, MT, NW, 64, OCC>, 2 * TileCfg<MT, 64>::LDS1);
  else go(int4_tile_kernel<X, MT, NW, 32, OCC>, 2 * TileCfg<MT, 32>::LDS1);
}
template <class X>
void launch_type(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.tiles_t == 1) return launch_tile<X, 1, 1, 4>(a, stream, done);
  if (a.tiles_t == 2) return launch_tile<X, 2, 1, 3>(a, stream, done);
  launch_tile<X, 4, 2, 1>(a, stream, done);
}

}  // namespace

void int4_tile_plan(Int4Args& a, int64_t* ws_floats, int64_t* counters) {
  a.kernel = INT4_TILE;
  a.tiles_t = a.T <= 32 ? 1 : a.T <= 64 ? 2 : 4;
  a.tiles_n = a.tiles_t == 4 ? 2 : 1;
  const int64_t bm = 32 * a.tiles_t, bn = 128 * a.tiles_n;
  const int64_t tiles = ((a.T + bm - 1) / bm) * ((a.N + bn - 1) / bn), stages = (a.K + STAGE - 1) / STAGE;
  if (tiles > INT32_MAX) { a.kernel = INT4_ANY; return; }
  a.steps = (int32_t)stages;
  a.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>(256 / tiles, stages / 4));
  if (a.parts > 1) {
    *ws_floats = tiles * a.parts * (bm * bn);
    *counters = tiles;
  }
}

void launch_int4_tile(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.x_dtype == DT_BF16) launch_type<Int4BF16>(a, stream, done);
  else launch_type<Int4F16>(a, stream, done);
}

}  // namespace ryft
