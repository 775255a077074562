// ryft.int4_matmul with more than a few rows of x, bf16 and f16, groups of a multiple of 32.
//
// Two or three launches. The first puts x into the order and the places that the second's LDS has, and sums it over every span
// of values that share a scale: done by each workgroup of the second for itself it was most of its float and integer
// instructions (2048 rows against 12288 x 4096: 361 us; 205 to 222 and 8 so, with the card's clock: 0.93 to 1.0 PFLOP/s). The
// second multiplies tiles of 32 MT rows of x, which a workgroup's eight wavefronts share through a ring in LDS, with 32 rows of
// the weight a wavefront, which come through a ring of its own. A lane's sums are of one row of the weight, 16 rows of x each: one
// scale a span. Tiles are cut into ranges of K where they leave the chip idle; the third adds the parts in their order.
//
// At 2048 rows that is 0.67 to 0.72 of what a library product of 16-bit weights reaches on a large square (1.40). The matrix
// instructions are 9/8 of a product's, for the zero points: 166 us at that rate. What is beside them is traffic through LDS: of
// 213 us 208 are left without scaling, 218 without making operands, 169 without reading more of x than the first block, 169
// without loads, 137 without both. Wavefronts of 64 x 64, which read half as much of x and make each operand twice, take 223 us;
// words and groups read a stage ahead, or waits for fewer loads at the ranges' ends, change nothing.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../common.h"
#include "int4_matmul.h"
#include "launch.h"

namespace ryft {

namespace {

constexpr int STAGE = 128;  // values of x a stage
constexpr int CUS = 256, LEAST = 4;  // workgroups that run at a time (LDS has room for one a CU); stages a range of K
constexpr int AHEAD = 5;    // fragments of x on their way from LDS

// x as the second launch has it, for `rows` rows: of stage s and row t 256 bytes at (s · rows + t) · 256, chunk c (eight values,
// in a word's order) at position c ^ (t mod 16); then of span p and row t 16 bytes at (p · rows + t) · 16: the terms of its sum.
// A tile of the last rows reads on past them, whatever is there, and stores nothing of it: both parts end with room for that.
constexpr int MOST_ROWS = 128;
__host__ __device__ inline int64_t tile_x_bytes(int64_t steps, int64_t rows) { return (steps * rows + MOST_ROWS) * (STAGE * 2); }
__host__ __device__ inline int64_t tile_ws_bytes(int64_t steps, int64_t rows, int span) {
  return tile_x_bytes(steps, rows) + (steps * (STAGE / span) * rows + MOST_ROWS) * 16;
}

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

// Terms of a span's sum S that a matrix instruction multiplies by -(16 + z): S = a · H + b + c, each rounded to 16 bits (H: a
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

template <class X, int SPAN>
__global__ void __launch_bounds__(256) int4_prepare_kernel(const Int4Args A, int64_t t0, int rows) {
  const int c = threadIdx.x & 15, K = (int)A.K, t = (int)blockIdx.x * 16 + (threadIdx.x >> 4), stage = blockIdx.y, k = stage * STAGE + 8 * c;
  if (t >= rows) return;  // (whole groups of 16 lanes)
  const int64_t st = (int64_t)stage * rows + t;
  u32x4p v = {0, 0, 0, 0};
  if (k < K) v = *(const u32x4p*)((const uint16_t*)A.x + (t0 + t) * A.K + k);
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum += X::lo(v[e]) + X::hi(v[e]);
  sum = span_sum<SPAN>(sum);
  char* const ws = (char*)A.ws;
  *(u32x4p*)(ws + st * (STAGE * 2) + 16 * (c ^ (t & 15))) = int4_order(v);
  constexpr int CS = SPAN / 8;
  if (c % CS == 0)
    *(u32x4p*)(ws + tile_x_bytes(A.steps, rows) + ((int64_t)(stage * (STAGE / SPAN) + c / CS) * rows + t) * 16) = sum_terms<X>(sum);
}

// Floats from one part of `count` results to the next: parts begin at 16 bytes.
__host__ __device__ inline int64_t part_floats(int64_t count) { return (count + 3) & ~(int64_t)3; }

constexpr int WAVES = 8, BN = 32 * WAVES;  // wavefronts of a workgroup, each with 32 rows of the weight

// Rings in LDS: stages of x and its sums, DX of them, which all wavefronts read; stages of a wavefront's weight, scales and zero
// points, DW of them, which have further to come.
template <int MT, int SPAN>
struct TileCfg {
  static constexpr int BM = 32 * MT, SPANS = STAGE / SPAN;
  static constexpr int XB = BM * STAGE * 2;                          // bytes of a stage's x
  static constexpr int XS = XB + (BM * SPANS * 16 + 1023) / 1024 * 1024;  // and of the terms of its sums
  static constexpr int SW = SPANS, SL = SPANS > 2 ? 2 : 1;           // words a row of scales, loads of them
  static constexpr int ZW = SPANS > 1 ? 2 : 1;                       // words a row of zero points
  static constexpr int S0 = 2048, Z0 = S0 + SL * 256, WS = Z0 + 256;  // of a wavefront's stage
  static constexpr int DX = MT == 1 ? 3 : 2;
  static constexpr int ROOM = 160 * 1024 - 1536 - DX * XS;
  static constexpr int DW = ROOM / (WAVES * WS) < 6 ? ROOM / (WAVES * WS) : 6;
  static constexpr int YP = BN + 4, YB = 32 * YP * 4;                // 32 rows of the result: pitch, bytes
  static constexpr int DUMP = DX * XS + WAVES * DW * WS;             // a place for loads that are made for their number alone
  static constexpr int LDS = DUMP + 1024;
  static_assert(DW > DX && LDS >= YB);
};

typedef __attribute__((address_space(3))) void tile_lds;

template <int N>
__device__ __forceinline__ void tile_wait() {  // until N loads or fewer are on their way, and all LDS accesses are done
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
  asm volatile("" ::: "memory");
}

// parts > 1: partial sums as f32 rows, [part][row][N], part_floats() from part to part, behind the prepared x.
// MANY: several spans a group.
template <class X, int MT, int SPAN, bool MANY>
__global__ void __launch_bounds__(64 * WAVES, 2) int4_tile_kernel(const Int4Args A, int64_t t_base, int x_rows) {
  typedef TileCfg<MT, SPAN> C;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int SPANS = C::SPANS, FR = SPAN / 16, CH = C::BM * 16 / (64 * WAVES);
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles_t = (x_rows + C::BM - 1) / C::BM;
  const int tile = blockIdx.x;
  const int tn = tile / tiles_t, tt = tile - tn * tiles_t, part = blockIdx.y;
  const int t0 = tt * C::BM;  // (of the prepared rows)
  const int64_t n0 = (int64_t)tn * BN;
  const int K = (int)A.K;
  int lo, hi;
  int4_range(A, part, lo, hi);

  // A wavefront's own rows of the weight: four lanes load a row's 64 bytes of a stage, chunk c of 16 bytes of row r to position
  // c ^ (r / 4 mod 4), so that eight rows' reads take different banks. Scales and zero points come in whole words (the last of
  // an odd number of 16-bit scales lies in one with two bytes that belong to no one, as the last zero points may). Loads never
  // leave the buffers: chunks past a row's end are read from its beginning (x is 0 there), rows past the last are read as it
  // and not stored, and words past the last as that.
  const int es = A.scale_dtype == DT_F32 ? 4 : 2, most = (int)min(A.N - 1 - n0, (int64_t)(BN - 1));
  const int64_t first = n0 * A.groups, rest = (A.N - n0) * A.groups;
  const uint32_t s_off = (uint32_t)(first * es & 3), z_off = (uint32_t)(first & 3);
  const uint32_t s_bytes = (uint32_t)min(rest * es + s_off + 3, (int64_t)0x7ffffffc) & ~3u;
  const uint32_t z_bytes = (uint32_t)min(rest + z_off + 3, (int64_t)0x7ffffffc) & ~3u;
  const __amdgpu_buffer_rsrc_t wb = int4_buffer(A.w + n0 * (K / 2), (A.N - n0) * (K / 2));
  const __amdgpu_buffer_rsrc_t sb = int4_buffer((const char*)A.scale + (first * es & ~(int64_t)3), s_bytes);
  const __amdgpu_buffer_rsrc_t zb = A.zero ? int4_buffer(A.zero + (first & ~(int64_t)3), z_bytes) : sb;
  const int r0 = 32 * wave, wc = (lane & 3) ^ (lane >> 4);
  // (kept as they are: the compiler would compute them again in every stage)
  auto keep = [](uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
  };
  const uint32_t w0 = keep((uint32_t)min(r0 + (lane >> 2), most) * (uint32_t)(K / 2) + 16 * wc);
  const uint32_t w1 = keep((uint32_t)min(r0 + 16 + (lane >> 2), most) * (uint32_t)(K / 2) + 16 * wc);
  uint32_t s_row[C::SL];
#pragma unroll
  for (int h = 0; h < C::SL; ++h)
    s_row[h] = keep(s_off + (uint32_t)(min(r0 + min((64 * h + lane) / C::SW, 31), most) * A.groups) * es + 4 * ((64 * h + lane) % C::SW));
  const uint32_t z_row = keep(z_off + (uint32_t)(min(r0 + min(lane / C::ZW, 31), most) * A.groups) + 4 * (lane % C::ZW));
  // groups before this lane's row, from a whole word on
  const uint32_t own = keep((uint32_t)(first & 3) + (uint32_t)(min(r0 + l32, most) * A.groups));
  char* const w_ring = smem + C::DX * C::XS + wave * (C::DW * C::WS);
  if (!A.zero) {
    // (the zero points that the loads below leave alone)
#pragma unroll
    for (int d = 0; d < C::DW; ++d) ((uint32_t*)(w_ring + d * C::WS + C::Z0))[lane] = 0x08080808u;
  }
  // x and the terms of its sums, as they lie in the workspace
  const char* const xp = (const char*)A.ws;
  const char* const tp = xp + tile_x_bytes(A.steps, x_rows);
  const __amdgpu_buffer_rsrc_t xb = int4_buffer(xp, tile_x_bytes(A.steps, x_rows));
  const __amdgpu_buffer_rsrc_t tb = int4_buffer(tp, tile_ws_bytes(A.steps, x_rows, SPAN) - tile_x_bytes(A.steps, x_rows));
  const uint32_t x_at = keep((uint32_t)t0 * (STAGE * 2) + tid * 16);
  // (64 rows of a span and wavefront; wavefronts that none is left for load the first again, and let it be)
  const uint32_t t_to = 64 * wave < C::BM * SPANS ? C::XB + wave * 1024 : (uint32_t)C::DUMP;
  const int ti = 64 * wave < C::BM * SPANS ? min(tid, C::BM * SPANS - 1) : 0;
  const uint32_t t_at = keep((uint32_t)(ti / C::BM * x_rows + t0 + ti % C::BM) * 16);

  auto group_of = [&](int span) { return min(MANY ? (int)((uint32_t)span / (uint32_t)A.group_spans) : span, A.groups - 1); };
  auto load_x = [&](int stage, int slot) {
    char* const to = smem + slot * C::XS;
#pragma unroll
    for (int j = 0; j < CH; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, (tile_lds*)(to + j * (1024 * WAVES) + wave * 1024), 16, (int)x_at,
                                               stage * x_rows * (STAGE * 2) + j * (1024 * WAVES), 0, 0);
    char* const t_base = t_to == C::DUMP ? smem : to;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(tb, (tile_lds*)(t_base + t_to), 16, (int)t_at, stage * x_rows * (SPANS * 16), 0, 0);
  };
  const int z_to = A.zero ? C::Z0 : C::DUMP;
  auto load_w = [&](int stage, int slot) {
    const int k = stage * STAGE;
    char* const to = w_ring + slot * C::WS;
    if (k + STAGE <= K) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, (tile_lds*)to, 16, (int)w0, k / 2, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, (tile_lds*)(to + 1024), 16, (int)w1, k / 2, 0, 0);
    } else {
      const uint32_t off = k + 32 * wc < K ? (uint32_t)(k / 2) : (uint32_t)(-16 * wc);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, (tile_lds*)to, 16, (int)(w0 + off), 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, (tile_lds*)(to + 1024), 16, (int)(w1 + off), 0, 0, 0);
    }
    const uint32_t g = (uint32_t)group_of(stage * SPANS);
#pragma unroll
    for (int h = 0; h < C::SL; ++h) {
      const uint32_t at = min((s_row[h] + g * es) & ~3u, s_bytes - 4);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sb, (tile_lds*)(to + C::S0 + h * 256), 4, (int)at, 0, 0, 0);
    }
    // (without zero points, some of the scales, for the number of loads)
    const uint32_t z = min((z_row + g) & ~3u, (A.zero ? z_bytes : s_bytes) - 4);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(zb, (tile_lds*)((A.zero ? to : smem) + z_to), 4, (int)z, 0, 0, 0);
  };
  // Waits for a stage's loads, by how many were made after them. In the first stage those of DW - 2 weights; later those of DX - 2
  // stages and of one weight more, for x, whose weight's loads are older. Where there are no more weights to load, for all.
  auto arrived = [&](int stage) {
    constexpr int NW = 3 + C::SL, NX = CH + 1;
    if (stage + C::DW - 2 >= hi) tile_wait<0>();
    else if (stage == lo) tile_wait<(C::DW - 2) * NW>();
    else tile_wait<(C::DX - 2) * (NX + NW) + NW>();
  };
  // where a lane's first block of a stage lies: row l32, chunk `half` (and by exclusive or with 32 bytes the next, and so on)
  uint32_t chunk = l32 * (STAGE * 2) + 16 * (half ^ (l32 & 15));
  const uint32_t w_lane = keep(l32 * 64 + 16 * (half ^ (l32 >> 2 & 3))), sums_at = keep(C::XB + l32 * 16);
  const uint32_t s_lane = keep(C::S0 + l32 * (4 * C::SW)), z_lane = keep(C::Z0 + (A.zero ? l32 * (4 * C::ZW) : 0));
  const uint32_t s_step = es == 4 ? 0 : 2, z_step = A.zero ? 3 : 0, s_up = es == 4 ? 0 : 16;
  const Int4Operand<X> operand;

  f32x16p y[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) y[m] = f32x16p{};

  {
    int xi = 0, wi = 0, xo = C::DX - 1, wo = C::DW - 1;  // slots of this stage, and of those that are loaded in it
    for (int d = 0; d < C::DX - 1 && lo + d < hi; ++d) load_x(lo + d, d);
    for (int d = 0; d < C::DW - 1 && lo + d < hi; ++d) load_w(lo + d, d);
    for (int stage = lo; stage < hi; ++stage) {
      arrived(stage);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (stage + C::DX - 1 < hi) load_x(stage + C::DX - 1, xo);
      if (stage + C::DW - 1 < hi) load_w(stage + C::DW - 1, wo);
      const char* const from = smem + xi * C::XS;
      const char* const wf_at = w_ring + wi * C::WS;
      if (++xi == C::DX) xi = 0;
      if (++wi == C::DW) wi = 0;
      if (++xo == C::DX) xo = 0;
      if (++wo == C::DW) wo = 0;
      // the words that the matrix instructions take: of block f of 16 values, one for each half-wave
      uint32_t word[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4p v = *(const u32x4p*)(wf_at + (w_lane ^ (32 * j)));
        const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[1], false, false);
        const auto b = __builtin_amdgcn_permlane32_swap(v[2], v[3], false, false);
        word[4 * j] = a[0], word[4 * j + 1] = b[0], word[4 * j + 2] = a[1], word[4 * j + 3] = b[1];
      }
      const int g0 = group_of(stage * SPANS);
      // scales and zero points (of the groups that there are; past the row's end x is 0: its last one's)
      float scale[SPANS];
      u32x4p zf[SPANS];
#pragma unroll
      for (int p = 0; p < SPANS; ++p) {
        const int g = group_of(stage * SPANS + p) - g0;
        const uint32_t s_byte = es == 4 ? 4 * g : ((own + g0) << 1 & s_step) + 2 * g, z_byte = A.zero ? ((own + g0) & z_step) + g : 0;
        uint32_t s_word = *(const uint32_t*)(wf_at + s_lane + (s_byte & ~3u));
        s_word >>= s_byte << 3 & s_up;
        scale[p] = es == 4 ? __uint_as_float(s_word) : X::lo(s_word & 0xffffu);
        zf[p] = sum_factors<X>(*(const uint8_t*)(wf_at + z_lane + z_byte), half == 0);
      }
      u32x4p wf[8];
#pragma unroll
      for (int f = 0; f < 8; ++f) wf[f] = operand(word[f]);
      asm volatile("" : "+v"(chunk));  // (or all its neighbours would be kept in registers over the stages)
      const char* const sums = from + sums_at;
      // Blocks of a span and 32 rows of x, one after the other. Fragments of x are read AHEAD matrix instructions before they are
      // multiplied, and a block's sums are scaled while the next one's products run: the order is forced, since the compiler's own
      // reads each one, waits and multiplies.
      constexpr int F1 = FR + 1, BLOCKS = SPANS * MT, ALL = BLOCKS * F1;
      u32x4p ring[AHEAD + 1];
      f32x16p acc[2];
      auto read = [&](int at) {
        const int b = at / F1, f = at % F1, p = b / MT, m = b % MT;
        if (f == 0) return *(const u32x4p*)(sums + (p * C::BM + 32 * m) * 16);
        return *(const u32x4p*)(from + (chunk ^ (32 * (p * FR + f - 1))) + 32 * m * (STAGE * 2));
      };
      auto add = [&](int b) {
#pragma unroll
        for (int e = 0; e < 16; ++e) y[b % MT][e] = __builtin_fmaf(scale[b / MT], acc[b & 1][e], y[b % MT][e]);
        asm volatile("" : "+v"(y[b % MT]));  // (or they would be put off past all products)
      };
#pragma unroll
      for (int at = 0; at < AHEAD && at < ALL; ++at) ring[at] = read(at);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
        for (int f = 0; f < F1; ++f) {
          const int at = b * F1 + f;
          if (at + AHEAD < ALL) ring[(at + AHEAD) % (AHEAD + 1)] = read(at + AHEAD);
          const u32x4p x = ring[at % (AHEAD + 1)];
          acc[b & 1] = f == 0 ? X::mma32(x, zf[b / MT], f32x16p{}) : X::mma32(x, wf[b / MT * FR + (f > 0 ? f - 1 : 0)], acc[b & 1]);
        }
        if (b > 0) add(b - 1);
#pragma unroll
        for (int f = 0; f < F1; ++f) {
          if (b * F1 + f + AHEAD < ALL) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (b > 0) __builtin_amdgcn_sched_group_barrier(0x002, (16 + F1 - 1) / F1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      add(BLOCKS - 1);
    }
  }
  // The tile's rows, 32 at a time, through LDS: a thread stores 16 bytes of a row together where rows begin at such places.
  const bool whole = A.parts == 1;
  const int ys = whole && A.y_dtype != DT_F32 ? 2 : 4, per = 16 / ys;
  const bool wide = A.N % per == 0;
  const int n_here = (int)min((int64_t)BN, A.N - n0);
  char* const out = whole ? (char*)A.y + (t_base + t0) * A.N * ys
                          : (char*)A.ws + tile_ws_bytes(A.steps, x_rows, SPAN) + (part * part_floats(x_rows * A.N) + t0 * A.N) * 4;
  float* const rows_at = (float*)smem;
  float odd = 0.f;  // NaN where a value that this thread stores is not finite
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) rows_at[(8 * (e >> 2) + 4 * half + (e & 3)) * C::YP + 32 * wave + l32] = y[m][e];
    __syncthreads();
    const int t_here = min(32, x_rows - t0 - 32 * m);
    char* const to = out + ((int64_t)32 * m * A.N + n0) * ys;
    if (wide) {
      const int chunks = BN / per;
      for (int i = tid; i < 32 * chunks; i += 64 * WAVES) {
        const int r = i / chunks, c = (i - r * chunks) * per;
        if (r >= t_here || c >= n_here) continue;
        const f32x4p a = *(const f32x4p*)(rows_at + r * C::YP + c);
        char* const at = to + ((int64_t)r * A.N + c) * ys;
#pragma unroll
        for (int e = 0; e < 4; ++e) odd = __builtin_fmaf(a[e], 0.f, odd);
        if (ys == 4) {
          *(f32x4p*)at = a;
        } else {
          const f32x4p b = *(const f32x4p*)(rows_at + r * C::YP + c + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd = __builtin_fmaf(b[e], 0.f, odd);
          *(u32x4p*)at = u32x4p{X::put(a[0]) | (uint32_t)X::put(a[1]) << 16, X::put(a[2]) | (uint32_t)X::put(a[3]) << 16,
                                X::put(b[0]) | (uint32_t)X::put(b[1]) << 16, X::put(b[2]) | (uint32_t)X::put(b[3]) << 16};
        }
      }
    } else {
      for (int i = tid; i < 32 * BN; i += 64 * WAVES) {
        const int r = i / BN, c = i % BN;
        if (r >= t_here || c >= n_here) continue;
        const float v = rows_at[r * C::YP + c];
        char* const at = to + ((int64_t)r * A.N + c) * ys;
        odd = __builtin_fmaf(v, 0.f, odd);
        if (ys == 4) *(float*)at = v;
        else *(uint16_t*)at = X::put(v);
      }
    }
  }
  if (!whole || !__any(odd != odd)) return;  // (parts are looked at when they are added)
  const Int4Args& B = int4_args_again();
  const int each = wide ? per : 1, chunks = BN / each;
#pragma unroll 1
  for (int i = tid; i < C::BM * chunks; i += 64 * WAVES) {  // what this thread has stored; the wavefront together
    const int r = i / chunks, c = (i - r * chunks) * each;
#pragma unroll 1
    for (int e = 0; e < each; ++e) int4_mend_stored<X>(B, t0 + r < x_rows && c + e < n_here, t_base + t0 + r, n0 + c + e);
  }
}

// Adds the parts of `count` elements, in their order, from `parts` (of the workspace, part_floats() apart) into y from element
// `at` on, a multiple of four: four elements a thread.
template <class X>
__global__ void __launch_bounds__(256, 6) int4_join_kernel(const Int4Args A, const float* parts, int64_t at, int64_t count) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i - 4 * (threadIdx.x & 63) >= count) return;  // (whole wavefronts)
  f32x4p v = {0.f, 0.f, 0.f, 0.f};
  if (i < count) {
#pragma unroll 8
    for (int p = 0; p < A.parts; ++p) v += *(const f32x4p*)(parts + p * part_floats(count) + i);
  }
  if (count - i >= 4) {
    if (A.y_dtype == DT_F32) *(f32x4p*)((float*)A.y + at + i) = v;
    else *(uint2*)((uint16_t*)A.y + at + i) = uint2{X::put(v[0]) | (uint32_t)X::put(v[1]) << 16, X::put(v[2]) | (uint32_t)X::put(v[3]) << 16};
  } else {
    for (int e = 0; e < (int)(count - i); ++e) {
      if (A.y_dtype == DT_F32) ((float*)A.y)[at + i + e] = v[e];
      else ((uint16_t*)A.y)[at + i + e] = X::put(v[e]);
    }
  }
  if (!__any(!int4_finite(v[0]) || !int4_finite(v[1]) || !int4_finite(v[2]) || !int4_finite(v[3]))) return;
#pragma unroll 1
  for (int e = 0; e < 4; ++e) {
    const int64_t t = (at + i + e) / A.N;
    int4_mend_stored<X>(A, i + e < count, t, at + i + e - t * A.N);
  }
}

template <class X, int MT, int SPAN>
void launch_tile_span(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  typedef TileCfg<MT, SPAN> C;
  const auto kernel = a.group_spans > 1 ? int4_tile_kernel<X, MT, SPAN, true> : int4_tile_kernel<X, MT, SPAN, false>;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("int4_matmul LDS attribute: ") + hipGetErrorString(e));
  const int64_t each = a.rows;
  for (int64_t t0 = 0; t0 < a.T; t0 += each) {
    const int rows = (int)std::min(each, a.T - t0);
    hipEvent_t const end = t0 + each >= a.T ? done : nullptr;
    launch_k(nullptr, int4_prepare_kernel<X, SPAN>, dim3((unsigned)((rows + 15) / 16), (unsigned)a.steps), dim3(256), 0, stream, a, t0, rows);
    const int64_t tiles = ((int64_t)(rows + C::BM - 1) / C::BM) * ((a.N + BN - 1) / BN);
    launch_k(a.parts > 1 ? nullptr : end, kernel, dim3((unsigned)tiles, (unsigned)a.parts), dim3(64 * WAVES), C::LDS, stream, a, t0, rows);
    if (a.parts == 1) continue;
    const int64_t count = rows * a.N;
    launch_k(end, int4_join_kernel<X>, dim3((unsigned)((count + 1023) / 1024)), dim3(256), 0, stream, a,
             (const float*)((char*)a.ws + tile_ws_bytes(a.steps, rows, SPAN)), t0 * a.N, count);
  }
}
template <class X, int MT>
void launch_tile(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.span == 128) launch_tile_span<X, MT, 128>(a, stream, done);
  else if (a.span == 64) launch_tile_span<X, MT, 64>(a, stream, done);
  else launch_tile_span<X, MT, 32>(a, stream, done);
}
template <class X>
void launch_type(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (a.tile == 1) launch_tile<X, 1>(a, stream, done);
  else if (a.tile == 2) launch_tile<X, 2>(a, stream, done);
  else launch_tile<X, 4>(a, stream, done);
}

}  // namespace

bool int4_tile_plan(Int4Args& a, int64_t room, int64_t* ws_floats) {
  const int64_t stages = (a.K + STAGE - 1) / STAGE;
  a.steps = (int32_t)stages;
  // Rows at a time: equal shares, in whole tiles, of at most 32 MiB (838 rows of 13248 values against 3518 rows, once 768 and 70 at
  // a time: 226 us) and half of the room: parts may take as much (a tile of 128 KiB for each of 256 workgroups).
  const int64_t row = stages * (STAGE * 2 + STAGE / a.span * 16);
  int64_t most = std::max<int64_t>(1, std::min<int64_t>(32ll << 20, room / 2) / (row * MOST_ROWS)) * MOST_ROWS, unit = MOST_ROWS;
  if (tile_ws_bytes(stages, std::min(a.T, most), a.span) > room) {  // (fewer rows than the highest tile has)
    most = (room - tile_ws_bytes(stages, 0, a.span)) / row / 32 * 32, unit = 32;
    if (most < 32) return false;
  }
  const int64_t goes = (a.T + most - 1) / most, each = (a.T + goes - 1) / goes;
  const int64_t rows = std::min(a.T, (each + unit - 1) / unit * unit);
  const int64_t x_bytes = tile_ws_bytes(stages, rows, a.span), part = 4 * part_floats(rows * a.N);
  // Tile and ranges of K by what they are estimated to take, in us: 4 for the launch, 3 for a tile's way to its stages and from
  // them, a stage's time by rows of the tile and values of a span (2048 rows against 12288 x 4096: 219, 267 and 389 us with 128, 64
  // and 32 rows in spans of 128, 256, 320 and 468 of 64, 324, 406 and 593 of 32), 4 for the third launch and 0.3 a MB of parts,
  // written and read. Estimated and measured with 128, 64 and 32 rows: 256 rows against 4096 x 4096 30, 27, 29 and 27, 24, 28; 234
  // against 13226 x 1472 in spans of 64 34, 27, 37 and 33, 27, 38; 373 against 940 x 9216 27, 26, 27 and 24, 24, 27; 100 against
  // 8192 x 608 in spans of 32 24, 18, 15 and 20, 13, 12.
  static constexpr double STAGE_US[3][3] = {{0.95, 1.37, 2.2}, {1.13, 1.65, 2.6}, {1.5, 2.1, 3.3}};
  if (stages > 65535 || rows * ((a.N + 31) / 32) >= INT32_MAX) return false;  // (the grids' limits)
  double best = 1e30;
  for (int tile = 1; tile <= 4; tile *= 2) {
    const double stage = STAGE_US[a.span == 128 ? 0 : a.span == 64 ? 1 : 2][tile / 2];
    const int64_t tiles = ((rows + 32 * tile - 1) / (32 * tile)) * ((a.N + BN - 1) / BN);
    for (int64_t parts = 1; parts == 1 || (parts * tiles <= CUS && parts <= stages / LEAST && x_bytes + parts * part <= room); ++parts) {
      double us = 4 + (double)((tiles * parts + CUS - 1) / CUS) * (3 + stage * (double)((stages + parts - 1) / parts));
      if (parts > 1) us += 4 + 0.3e-6 * (double)(parts * part);
      if (us < best) best = us, a.tile = tile, a.parts = (int32_t)parts;
    }
  }
  a.kernel = INT4_TILE;
  a.rows = (int32_t)rows;
  *ws_floats = (x_bytes + (a.parts > 1 ? a.parts * part : 0)) / 4;
  return true;
}

void launch_int4_tile(const Int4Args& a, hipStream_t stream, hipEvent_t done) {
  if (!a.ws) fail(PJRT_Error_Code_INTERNAL, "int4_matmul without a workspace");
  if (a.x_dtype == DT_BF16) launch_type<Int4BF16>(a, stream, done);
  else launch_type<Int4F16>(a, stream, done);
}

}  // namespace ryft
