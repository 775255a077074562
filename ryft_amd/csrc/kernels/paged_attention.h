// Shared by the kernels of ryft.paged_attention (the definition stands at PagedAttnArgs in kernel_abi.h): what a sequence
// of the ragged batch has, scores, the 16-bit matrix operands, and the join of partial results of key ranges.
#pragma once

#include "op_device.h"

namespace ryft {

constexpr float kLog2e = 1.4426950408889634f;

typedef float f32x2p __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2p __attribute__((ext_vector_type(2)));

// 16-bit matrix operands of one type: products into f32, pairs of values rounded to it (nearest even), and what that leaves
// of them, rounded to it too. Probabilities go to the product with the values as both terms, 2^-17 (f16: 2^-22) off, so that
// an output is as exact as f32 ones make it. The first term alone added 14 to 26% to its error against 64 bits (prompts of
// bf16 2.0e-3 of the norm, 1.6e-3 so). The second costs half of the matrix instructions again and three float instructions a
// score: four prompts of up to 2048 tokens 112 -> 129 us, two chunks of 512 35.5 -> 39.1; decoding steps, which HBM bounds,
// nothing (64 sequences of up to 4096 keys 111 us). LIFT: the power of two by which probabilities stand above 1 at the
// running maximum, so that f16 keeps its full precision down to 2^-21 of it (and may exceed it by 2^8: below 2^16).
struct MmaBF16 {
  typedef __bf16 x8 __attribute__((__vector_size__(8 * sizeof(__bf16))));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static constexpr float LIFT = 0.f;
  __device__ static __forceinline__ f32x4p mma16(const u32x4p& a, const u32x4p& b, f32x4p c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x16p mma32(const u32x4p& a, const u32x4p& b, f32x16p c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, x2));
  }
  __device__ static __forceinline__ uint32_t rest(uint32_t w, float lo, float hi) {
    return pack(lo - __uint_as_float(w << 16), hi - __uint_as_float(w & 0xffff0000u));
  }
};
struct MmaF16 {
  typedef _Float16 x8 __attribute__((__vector_size__(8 * sizeof(_Float16))));
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  static constexpr float LIFT = 7.f;
  __device__ static __forceinline__ f32x4p mma16(const u32x4p& a, const u32x4p& b, f32x4p c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x16p mma32(const u32x4p& a, const u32x4p& b, f32x16p c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, x2));
  }
  __device__ static __forceinline__ uint32_t rest(uint32_t w, float lo, float hi) {
    const x2 h = __builtin_bit_cast(x2, w);
    return pack(lo - (float)h[0], hi - (float)h[1]);
  }
};

// starts are clamped to [0, T], lengths to [0, M · P] (0 over an empty cache).
__device__ __forceinline__ int paged_start(const PagedAttnArgs& A, int b) {
  return (int)min(max((int64_t)A.starts[b], (int64_t)0), A.T);
}
__device__ __forceinline__ int paged_length(const PagedAttnArgs& A, int b) {
  return A.pages > 0 ? min(max(A.lengths[b], 0), A.M * A.P) : 0;
}
// key / P for a key below 2^31 (PagedAttnArgs::page_mul)
__device__ __forceinline__ int page_of(const PagedAttnArgs& A, int key) {
  return (int)(((uint64_t)(uint32_t)key * A.page_mul) >> A.page_shift);
}

// Trees of drafted tokens (PagedAttnArgs::visible). The 64 bits of token t's row from bit `from` on: ones before bit 0, which
// stand for the tokens before the tree, zeros past the row's end.
__device__ __forceinline__ uint64_t tree_bits(const PagedAttnArgs& A, int64_t t, int from) {
  const uint32_t* const row = A.visible + t * A.W;
  auto word = [&](int i) -> uint32_t { return i < 0 ? 0xffffffffu : i < A.W ? row[i] : 0u; };
  const int i = from >> 5, s = from & 31;  // (rounded down)
  const uint64_t lo = (uint64_t)word(i + 1) << 32 | word(i);
  return s ? lo >> s | (uint64_t)word(i + 2) << (64 - s) : lo;
}
// The first key that a token of a tree of n sees, under a window; the tree starts at position pos0.
__device__ __forceinline__ int tree_first(const PagedAttnArgs& A, int64_t t, int n, int pos0) {
  if (A.window <= 0) return 0;
  int seen = 0;
  for (int i = 0; i < A.W && 32 * i < n; ++i) {
    const uint32_t w = A.visible[t * A.W + i];
    seen += __popc(n - 32 * i < 32 ? w & ((1u << (n - 32 * i)) - 1) : w);
  }
  return (int)max((int64_t)0, min((int64_t)pos0, (int64_t)pos0 + seen - A.window));
}

// Scores in the log2 domain, constants of a launch. A cap is held by two forms, with z = s / cap: cap - 2 · cap / (e^(2 z) + 1),
// which saturates at both ends and is off by 2^-22 of the cap, for all scores up to a cap of kFarCap (log2; 2^-15 there, a
// twentieth of half a step of f16 in a probability; four prompts of up to 2048 tokens capped at 50 129 us, 135 with the other
// form where it would do); and above it where z is past 1/2, below that s · (tanh z / z), tanh z / z by a polynomial in z²
// that interpolates at Chebyshev nodes (2^-25 off), which leaves a score far below its cap as it is. Constants past f32's
// range are its largest numbers: a cap that small is reached by every score, one that large by none.
constexpr float kFarCap = 128.f;
struct PagedScore {
  float sl2, capr, capz, cap2;  // scale · log2 e; scale / cap; 2 · capr · log2 e; cap · log2 e (0: none)
  __device__ explicit PagedScore(const PagedAttnArgs& A) {
    auto bounded = [](float x, float most) { return fminf(fmaxf(x, -most), most); };
    sl2 = bounded(A.scale * kLog2e, 0x1p127f);
    capr = A.softcap > 0.f ? bounded(A.scale / A.softcap, 0x1p127f) : 0.f;
    capz = bounded(2.f * capr * kLog2e, 0x1p127f);
    cap2 = fminf(A.softcap * kLog2e, 0x1p126f);
  }
  // z of the larger half, or NaN
  __device__ __forceinline__ bool far(float dot) const { return !(fabsf(dot * capr) <= 0.5f); }
  __device__ __forceinline__ float near_cap(float dot, float bias) const {
    const float z = dot * capr, zz = z * z;
    float p = __builtin_fmaf(zz, 0x1.18d7e8p-6f, -0x1.b2167ep-5f);
    p = __builtin_fmaf(zz, p, 0x1.10e47ap-3f);
    p = __builtin_fmaf(zz, p, -0x1.5554a6p-2f);
    return __builtin_fmaf(__builtin_fmaf(zz, p, 1.f), dot * sl2, bias);
  }
  __device__ __forceinline__ float far_cap(float dot, float bias) const {
    const float e = __builtin_amdgcn_exp2f(dot * capz);
    return __builtin_fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(e + 1.f), cap2 + bias);
  }
  // N scores of a block of keys, the bias of score i bias(i)
  template <int N, class S, class B>
  __device__ __forceinline__ void cap(S& st, B&& bias) const {
    if (cap2 <= kFarCap) {
#pragma unroll
      for (int i = 0; i < N; ++i) st(i) = far_cap(st(i), bias(i));
      return;
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(st(i)));
    if (__builtin_amdgcn_ballot_w64(far(top))) {
#pragma unroll
      for (int i = 0; i < N; ++i) st(i) = far(st(i)) ? far_cap(st(i), bias(i)) : near_cap(st(i), bias(i));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) st(i) = near_cap(st(i), bias(i));
    }
  }
};

// Largest of a lane's value and those of the lanes 16, 32 and 48 away; the same for sums.
__device__ __forceinline__ float max_rows16(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_rows16(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// ------------------------------------------------------------------------------------------------ one row
// One query and head over the keys [first, last), by a workgroup of 256, for any type, head dim up to 256 and page size;
// nothing that the query does not see is read. pos: the query's position, of a tree that of its first token. Leaves the
// maximum (log2), the sum and, at thread d, element d of the unnormalised output. Each wavefront takes every fourth block of 64 keys, a lane a key for the scores and an element
// of the head for the output; the four meet in LDS at the end.
struct PagedRowLds {
  int64_t base[4][64];
  float prob[4][64];
  float q[256];
  float part[4][256 + 2];
};
template <class E, bool TREE>
__device__ __forceinline__ float paged_row(const PagedAttnArgs& A, int b, int64_t t, int h, int pos, int first, int last,
                                           PagedRowLds& sh, float* m_out, float* l_out) {
  typedef typename E::raw raw;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = A.D;
  const raw* const qg = (const raw*)A.q + t * A.qs[0] + h * A.qs[1];
  __syncthreads();
  for (int i = tid; i < D; i += 256) sh.q[i] = E::get(qg[i]);
  __syncthreads();
  const int hk = h / (A.Hq / A.Hkv);
  const float slope = A.slopes ? A.slopes[h] * kLog2e : 0.f;
  const PagedScore score(A);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = first; k0 < last; k0 += 256) {
    const int key = k0 + wave * 64 + lane;
    float s = -INFINITY;
    int64_t at = -1;
    if (key < last && (!TREE || key < pos || (tree_bits(A, t, key - pos) & 1))) {
      const int pi = page_of(A, key);
      const int page = A.table[(int64_t)b * A.M + pi];
      if (page >= 0 && page < A.pages) {
        at = (((int64_t)page * A.Hkv + hk) * A.P + (key - pi * A.P)) * D;
        const raw* const kr = (const raw*)A.k_cache + at;
        float x = 0.f;
        for (int i = 0; i < D; ++i) x = __builtin_fmaf(sh.q[i], E::get(kr[i]), x);
        s = !(score.cap2 > 0.f) ? x * score.sl2 : score.far(x) ? score.cap2 * tanhf(x * score.capr) : score.near_cap(x, 0.f);
        s += slope * (float)(key - pos);
      }
    }
    sh.base[wave][lane] = at;
    float mb = s;
    for (int x = 32; x; x >>= 1) mb = fmaxf(mb, __shfl_xor(mb, x, 64));
    const float mn = fmaxf(m, mb), ref = mn == -INFINITY ? 0.f : mn;
    const float p = exp2f(s - ref), alpha = exp2f(m - ref);
    m = mn;
    l *= alpha;
    for (int c = 0; c < 4; ++c) o[c] *= alpha;
    float pb = p;
    for (int x = 32; x; x >>= 1) pb += __shfl_xor(pb, x, 64);
    l += pb;
    sh.prob[wave][lane] = p;
    __syncthreads();
    for (int j = 0; j < 64; ++j) {
      if (sh.base[wave][j] < 0) continue;
      const raw* const vr = (const raw*)A.v_cache + sh.base[wave][j];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < D) o[c] = __builtin_fmaf(sh.prob[wave][j], E::get(vr[lane + 64 * c]), o[c]);
    }
    __syncthreads();
  }
  for (int c = 0; c < 4; ++c) sh.part[wave][lane + 64 * c] = o[c];
  if (lane == 0) sh.part[wave][256] = m, sh.part[wave][257] = l;
  __syncthreads();
  float mt = -INFINITY, lt = 0.f, x = 0.f;
  for (int w = 0; w < 4; ++w) mt = fmaxf(mt, sh.part[w][256]);
  const float ref = mt == -INFINITY ? 0.f : mt;
  for (int w = 0; w < 4; ++w) {
    const float f = exp2f(sh.part[w][256] - ref);
    lt += sh.part[w][257] * f;
    x += sh.part[w][tid] * f;
  }
  *m_out = mt;
  *l_out = lt;
  return x;
}

// ------------------------------------------------------------------------------------------------ tiles of rows
// The rows of a sequence's tile are pairs (query, head of one key head's group), flat = query · group + head: queries
// and the heads that share their keys fill a tile together.
struct PagedTile {
  int b, s0, n;   // the sequence, its first token and number of queries
  int pos0, len;  // position of its first query, its length
  int hk, row0;   // key head, first flat row
};

// Partial results move between workgroups of one launch past the XCDs' L2s (agent scope: sc1).
constexpr int kAgent = 16;
typedef uint32_t u32x4w __attribute__((__vector_size__(16)));
typedef uint32_t u32x2w __attribute__((__vector_size__(8)));
__device__ __forceinline__ void agent_put4(__amdgpu_buffer_rsrc_t r, uint32_t byte, f32x4p v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4w, v), r, (int)byte, 0, kAgent);
}
__device__ __forceinline__ f32x4p agent_get4(__amdgpu_buffer_rsrc_t r, uint32_t byte) {
  return __builtin_bit_cast(f32x4p, __builtin_amdgcn_raw_buffer_load_b128(r, (int)byte, 0, kAgent));
}
__device__ __forceinline__ void agent_put2(__amdgpu_buffer_rsrc_t r, uint32_t byte, float x, float y) {
  __builtin_amdgcn_raw_buffer_store_b64(u32x2w{__float_as_uint(x), __float_as_uint(y)}, r, (int)byte, 0, kAgent);
}
__device__ __forceinline__ float2 agent_get2(__amdgpu_buffer_rsrc_t r, uint32_t byte) {
  const u32x2w v = __builtin_amdgcn_raw_buffer_load_b64(r, (int)byte, 0, kAgent);
  return float2{__uint_as_float(v[0]), __uint_as_float(v[1])};
}

// Whether this workgroup is the last of `parts` to arrive at a counter, once all its own stores are complete. Every
// thread calls it; `last`: a word of LDS. The counter is back at zero when the last has arrived.
__device__ __forceinline__ bool last_to_arrive(int32_t* counter, int parts, int* last) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const int arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    if (arrived == parts) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *last = arrived == parts;
  }
  __syncthreads();
  return *(volatile int*)last != 0;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t paged_ws(const PagedAttnArgs& A) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)A.ws, (short)0, -1, 0x00020000);
}

// Partial result of a tile in the workspace: unnormalised rows [rows][D], then (maximum, sum) [rows][2].
__host__ __device__ inline int64_t paged_part_floats(int rows, int D) { return (int64_t)rows * (D + 2); }

// Four elements of a finished row.
template <class E>
__device__ __forceinline__ void paged_put4(const PagedAttnArgs& A, int D, int64_t token, int head, int d, f32x4p v) {
  *(u32x2p*)((uint16_t*)A.o + (token * A.Hq + head) * D + d) = u32x2p{E::pack(v.x, v.y), E::pack(v.z, v.w)};
}
template <class E, int D>
__device__ __forceinline__ void paged_store4(const PagedAttnArgs& A, const PagedTile& t, int row, int d, f32x4p v) {
  const int G = A.Hq / A.Hkv, flat = t.row0 + row, q = flat / G, g = flat - q * G;
  paged_put4<E>(A, D, t.s0 + q, t.hk * G + g, d, v);
}

// Joins the partial results of a tile's `parts` ranges (slot(i): the workspace slot of range i) into its output rows.
// Maxima and sums of as many ranges as LDS holds (`sh`: 64 KB) come there first, so that the loads of the rows depend on
// nothing: 16 of a thread's are in flight (112 parts of 8 rows × 128: 40 us with 8 in flight and 32 ranges at a time).
template <class E, int D, int ROWS, class F>
__device__ __forceinline__ void paged_join(const PagedAttnArgs& A, const PagedTile& t, int rows, int parts, F&& slot, float* sh) {
  constexpr int CH = 8192 / ROWS;
  const __amdgpu_buffer_rsrc_t ws = paged_ws(A);
  const int tid = threadIdx.x;
  const uint32_t part_bytes = (uint32_t)paged_part_floats(ROWS, D) * 4;
  constexpr int PER = (ROWS * D / 4 + 255) / 256;
  f32x4p o[PER];
  float m[PER], l[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) o[k] = f32x4p{0.f, 0.f, 0.f, 0.f}, m[k] = -INFINITY, l[k] = 0.f;
  for (int p0 = 0; p0 < parts; p0 += CH) {
    const int np = min(CH, parts - p0);
    __syncthreads();
    for (int i = tid; i < np * rows; i += 256) {
      const int p = i / rows, r = i - p * rows;
      const float2 v = agent_get2(ws, (uint32_t)slot(p0 + p) * part_bytes + (ROWS * D + 2 * r) * 4);
      sh[2 * (p * ROWS + r)] = v.x;
      sh[2 * (p * ROWS + r) + 1] = v.y;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = tid + 256 * k, r = i / (D / 4), d = 4 * (i % (D / 4));
      if (r >= rows) continue;
      float mn = m[k];
      for (int p = 0; p < np; ++p) mn = fmaxf(mn, sh[2 * (p * ROWS + r)]);
      const float ref = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m[k] - ref);
      m[k] = mn;
      l[k] *= alpha;
      o[k] *= alpha;
#pragma unroll 16
      for (int p = 0; p < np; ++p) {
        const f32x4p v = agent_get4(ws, (uint32_t)slot(p0 + p) * part_bytes + (r * D + d) * 4);
        const float w = __builtin_amdgcn_exp2f(sh[2 * (p * ROWS + r)] - ref);
        l[k] = __builtin_fmaf(sh[2 * (p * ROWS + r) + 1], w, l[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][e] = __builtin_fmaf(v[e], w, o[k][e]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = tid + 256 * k, r = i / (D / 4), d = 4 * (i % (D / 4));
    if (r < rows) paged_store4<E, D>(A, t, r, d, o[k] * (l[k] == 0.f ? 0.f : 1.f / l[k]));
  }
}

}  // namespace ryft
