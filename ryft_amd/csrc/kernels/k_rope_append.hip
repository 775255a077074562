// ryft.rope_append: RMSNorm of query and key heads, rotation by position, and keys and values written to their slots of
// a paged cache, in one pass (the definition stands at RopeAppendArgs in kernel_abi.h). Everything is computed in f32
// and rounded once, on store; the angles in f64: at position 10^6 an f32 product would be off by up to 0.06 radians.
#include <hip/hip_runtime.h>

#include <string>

#include "../common.h"
#include "kernels.h"
#include "launch.h"
#include "op_device.h"

namespace ryft {

namespace {

// cos and sin of position · freq, times the magnitude: the angle in turns and its reduction in f64, the functions of the
// remaining half turn in f32.
__device__ __forceinline__ float2 rotation(int32_t position, float freq, float magnitude) {
  const double turns = (double)position * (double)freq * 0.15915494309189533577;
  const float rest = (float)(turns - __builtin_rint(turns));
  float s, c;
  sincospif(2.f * rest, &s, &c);
  return float2{c * magnitude, s * magnitude};
}

// Destination row of head h of token t: the queries' result, or a slot of a cache (null: nothing is written).
template <class E>
__device__ __forceinline__ typename E::raw* rope_out(const RopeAppendArgs& A, int64_t t, int h, int slot) {
  typedef typename E::raw raw;
  if (h < A.Hq) return (raw*)A.q_out + (t * A.Hq + h) * A.D;
  if (slot < 0 || slot >= A.pages * A.P) return nullptr;
  const bool key = h < A.Hq + A.Hkv;
  const int64_t row = ((int64_t)(slot / A.P) * A.Hkv + (h - A.Hq - (key ? 0 : A.Hkv))) * A.P + slot % A.P;
  return (raw*)(key ? A.k_cache : A.v_cache) + row * A.D;
}
template <class E>
__device__ __forceinline__ const typename E::raw* rope_in(const RopeAppendArgs& A, int64_t t, int h) {
  typedef typename E::raw raw;
  if (h < A.Hq) return (const raw*)A.q + t * A.qs[0] + h * A.qs[1];
  if (h < A.Hq + A.Hkv) return (const raw*)A.k + t * A.ks[0] + (h - A.Hq) * A.ks[1];
  return (const raw*)A.v + t * A.vs[0] + (h - A.Hq - A.Hkv) * A.vs[1];
}

// Any head dim up to 256, any rotated part: a wavefront a head, an element a lane and step. Workgroup x is token x; its
// wavefronts take its heads in turn, the token's rotations computed once.
template <class E>
__global__ void __launch_bounds__(256) rope_append_any_kernel(const RopeAppendArgs A) {
  typedef typename E::raw raw;
  __shared__ float2 turn[128];
  __shared__ float row[4][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t t = blockIdx.x;
  const int half = A.R / 2, heads = A.Hq + 2 * A.Hkv, D = A.D;
  for (int i = tid; i < half; i += 256) turn[i] = rotation(A.positions[t], A.inv_freq[i], A.magnitude);
  __syncthreads();
  const int slot = A.slots[t];
  for (int h0 = 0; h0 < heads; h0 += 4) {
    const int h = h0 + wave;
    const bool live = h < heads;
    const bool key = h >= A.Hq, value = h >= A.Hq + A.Hkv;
    if (live) {
      const raw* const x = rope_in<E>(A, t, h);
      const raw* const w = value ? nullptr : (const raw*)(key ? A.k_weight : A.q_weight);
      float sq = 0.f;
      for (int i = lane; i < D; i += 64) {
        const float f = E::get(x[i]);
        row[wave][i] = f;
        sq = __builtin_fmaf(f, f, sq);
      }
      if (w) {
        for (int m = 32; m; m >>= 1) sq += __shfl_xor(sq, m, 64);
        const float inv = rsqrtf(sq / (float)D + A.eps);
        for (int i = lane; i < D; i += 64) row[wave][i] *= inv * E::get(w[i]);
      }
    }
    __syncthreads();
    raw* const y = live ? rope_out<E>(A, t, h, slot) : nullptr;
    if (y) {
      for (int i = lane; i < D; i += 64) {
        float f = row[wave][i];
        if (i < A.R && !value) {
          const int pair = A.interleaved ? i >> 1 : i < half ? i : i - half;
          const bool second = A.interleaved ? i & 1 : i >= half;
          const float other = row[wave][A.interleaved ? i ^ 1 : second ? i - half : i + half];
          const float2 cs = turn[pair];
          f = second ? f * cs.x + other * cs.y : f * cs.x - other * cs.y;
        }
        y[i] = E::put(f);
      }
    }
    __syncthreads();
  }
}

// 16-bit heads of 16, 32, 64, 128 or 256 values, the rotated part a multiple of 16: a lane has 16 values of a head in two
// 16-byte loads, the two halves of its pairs (half layout: 8 c and R / 2 + 8 c on; interleaved: 16 c and 16 c + 8 on; past
// the rotated part the same), so that a rotation needs no other lane, and D / 16 lanes have a head, 64 · 16 / D heads a
// wavefront. It moves each value in and out once and is bound by HBM where there are many tokens (8192 of 48 heads of 128,
// half of each rotated, 201 MB: 42 us, 4.8 TB/s, where every pass has other tensors, 38 where it writes the queries to the
// same memory, 32 over all the same again, which the last-level cache holds in part; a torch copy of that size 39 and 28;
// slots in order change nothing. With three times as many heads a wavefront, all loads first, 48; a workgroup a token with a
// value a lane, 97) and by latency where there are few (256 tokens of the same 10 us and 17). A wavefront turns its lane
// number into one rotation of its token, and the lanes take theirs from LDS.
typedef uint32_t u32x4r __attribute__((ext_vector_type(4)));
template <class E>
__global__ void __launch_bounds__(256) rope_append_rows_kernel(const RopeAppendArgs A, int passes) {
  typedef typename E::raw raw;
  __shared__ float2 turns[4][128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = (int64_t)blockIdx.x * 4 + wave, t = id / passes;
  const int pass = (int)(id - t * passes);
  if (t >= A.T) return;
  const int D = A.D, R = A.R, half = R / 2, lph = D / 16, heads = A.Hq + 2 * A.Hkv;
  const int c = lane % lph, per = 64 / lph;
  const bool turned = 16 * c < R;
  const int a0 = turned && !A.interleaved ? 8 * c : 16 * c, a1 = turned && !A.interleaved ? half + 8 * c : 16 * c + 8;
  const int h = pass * per + lane / lph;
  const bool live = h < heads, value = h >= A.Hq + A.Hkv, key = h >= A.Hq;
  u32x4r x0 = {0, 0, 0, 0}, x1 = {0, 0, 0, 0};
  if (live) {
    const raw* const x = rope_in<E>(A, t, h);
    x0 = *(const u32x4r*)(x + a0), x1 = *(const u32x4r*)(x + a1);
  }
  const int position = A.positions[t], slot = A.slots[t];
  for (int i = lane; i < half; i += 64) turns[wave][i] = rotation(position, A.inv_freq[i], A.magnitude);
  float2 cs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = turned ? turns[wave][8 * c + i] : float2{1.f, 0.f};
  raw* const y = live ? rope_out<E>(A, t, h, slot) : nullptr;
  float f[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = E::get((raw)x0[i]), f[2 * i + 1] = E::get((raw)(x0[i] >> 16));
    f[8 + 2 * i] = E::get((raw)x1[i]), f[8 + 2 * i + 1] = E::get((raw)(x1[i] >> 16));
  }
  if (A.q_weight) {
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sq = __builtin_fmaf(f[i], f[i], sq);
    for (int m = 1; m < lph; m <<= 1) sq += __shfl_xor(sq, m, 64);
    const raw* const w = (const raw*)(key ? A.k_weight : A.q_weight);
    const u32x4r w0 = *(const u32x4r*)(w + a0), w1 = *(const u32x4r*)(w + a1);
    const float inv = rsqrtf(sq / (float)D + A.eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] *= inv * E::get((raw)w0[i]), f[2 * i + 1] *= inv * E::get((raw)(w0[i] >> 16));
      f[8 + 2 * i] *= inv * E::get((raw)w1[i]), f[8 + 2 * i + 1] *= inv * E::get((raw)(w1[i] >> 16));
    }
  }
  if (!y) return;
  u32x4r y0 = x0, y1 = x1;
  if (!value && (turned || A.q_weight)) {
    // pairs (p, q) → (p c - q s, q c + p s)
    if (turned && A.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = f[2 * i], q = f[2 * i + 1];
        f[2 * i] = p * cs[i].x - q * cs[i].y, f[2 * i + 1] = q * cs[i].x + p * cs[i].y;
      }
    } else if (turned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = f[i], q = f[8 + i];
        f[i] = p * cs[i].x - q * cs[i].y, f[8 + i] = q * cs[i].x + p * cs[i].y;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y0[i] = (uint32_t)E::put(f[2 * i]) | (uint32_t)E::put(f[2 * i + 1]) << 16;
      y1[i] = (uint32_t)E::put(f[8 + 2 * i]) | (uint32_t)E::put(f[8 + 2 * i + 1]) << 16;
    }
  }
  *(u32x4r*)(y + a0) = y0;
  *(u32x4r*)(y + a1) = y1;
}

template <class E>
void launch_rows(const RopeAppendArgs& a, hipStream_t stream, hipEvent_t done) {
  const int per = 64 / (a.D / 16), passes = (a.Hq + 2 * a.Hkv + per - 1) / per;
  const int64_t blocks = (a.T * passes + 3) / 4;
  if (blocks > INT32_MAX) fail(PJRT_Error_Code_INTERNAL, "rope_append of too many tokens");
  launch_k(done, rope_append_rows_kernel<E>, dim3((unsigned)blocks), dim3(256), 0, stream, a, passes);
}

bool rows_supported(const RopeAppendArgs& a) {
  return (a.dtype == DT_BF16 || a.dtype == DT_F16) && (a.D == 16 || a.D == 32 || a.D == 64 || a.D == 128 || a.D == 256) &&
         a.R % 16 == 0 && !((a.qs[0] | a.qs[1] | a.ks[0] | a.ks[1] | a.vs[0] | a.vs[1]) & 7);
}

}  // namespace

void launch_rope_append(const RopeAppendArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.D < 1 || a.D > 256 || a.R < 0 || a.R > a.D || a.R % 2 || a.Hq < 1 || a.Hkv < 1 || a.P < 1)
    fail(PJRT_Error_Code_INTERNAL, "rope_append of a shape the kernels do not take");
  if (a.T == 0) return record_done(done, stream);
  if (rows_supported(a)) {
    if (a.dtype == DT_BF16) launch_rows<ElemBF16>(a, stream, done);
    else launch_rows<ElemF16>(a, stream, done);
  } else with_elem(a.dtype, [&](auto e) {
    launch_k(done, rope_append_any_kernel<decltype(e)>, dim3((unsigned)a.T), dim3(256), 0, stream, a);
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("rope_append launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
