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

}  // namespace

void launch_rope_append(const RopeAppendArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.D < 1 || a.D > 256 || a.R < 0 || a.R > a.D || a.R % 2 || a.Hq < 1 || a.Hkv < 1 || a.P < 1)
    fail(PJRT_Error_Code_INTERNAL, "rope_append of a shape the kernels do not take");
  if (a.T == 0) return record_done(done, stream);
  with_elem(a.dtype, [&](auto e) {
    launch_k(done, rope_append_any_kernel<decltype(e)>, dim3((unsigned)a.T), dim3(256), 0, stream, a);
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("rope_append launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
