// ryft.paged_attention: attention of a ragged batch of queries over a paged key / value cache (the definition stands at
// PagedAttnArgs in kernel_abi.h). Scores, softmax statistics and outputs are f32 and rounded once, on store.
#include <hip/hip_runtime.h>

#include <string>

#include "../common.h"
#include "kernels.h"
#include "launch.h"
#include "op_device.h"

namespace ryft {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int clamp_start(const PagedAttnArgs& A, int b) {
  return (int)min(max((int64_t)A.starts[b], (int64_t)0), A.T);
}
__device__ __forceinline__ int clamp_length(const PagedAttnArgs& A, int b) {
  return min(max(A.lengths[b], 0), A.M * A.P);
}

// Any type and head dim up to 256: a workgroup a query and head. Each wavefront takes every fourth block of 64 keys, a
// lane a key for the scores and an element of the head for the output; the four meet in LDS at the end.
template <class E>
__global__ void __launch_bounds__(256) paged_attention_any_kernel(const PagedAttnArgs A) {
  typedef typename E::raw raw;
  __shared__ float q[256];
  __shared__ float prob[4][64];
  __shared__ int64_t base[4][64];
  __shared__ float part[4][256 + 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, D = A.D;
  // the last sequence that starts at or before the token
  int lo = 0, hi = A.B;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (clamp_start(A, mid) <= t) lo = mid + 1;
    else hi = mid;
  }
  const int b = lo - 1;
  int first = 0, last = 0, pos = 0;  // the keys [first, last)
  if (b >= 0 && t < clamp_start(A, b + 1)) {
    const int len = clamp_length(A, b);
    pos = len - (clamp_start(A, b + 1) - (int)t);
    last = A.causal ? min(len, pos + 1) : len;
    if (A.window > 0) first = (int)max((int64_t)0, (int64_t)pos - A.window + 1);
  }
  const raw* const qg = (const raw*)A.q + t * A.qs[0] + h * A.qs[1];
  for (int i = tid; i < D; i += 256) q[i] = E::get(qg[i]);
  __syncthreads();
  const int hk = h / (A.Hq / A.Hkv);
  const float slope = A.slopes ? A.slopes[h] * kLog2e : 0.f;
  const float cap = A.softcap, sl2 = A.scale * kLog2e;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = first; k0 < last; k0 += 256) {
    const int key = k0 + wave * 64 + lane;
    float s = -INFINITY;
    int64_t at = -1;
    if (key < last) {
      const int page = A.table[(int64_t)b * A.M + key / A.P];
      if (page >= 0 && page < A.pages) {
        at = (((int64_t)page * A.Hkv + hk) * A.P + key % A.P) * D;
        const raw* const kr = (const raw*)A.k_cache + at;
        float x = 0.f;
        for (int i = 0; i < D; ++i) x = __builtin_fmaf(q[i], E::get(kr[i]), x);
        s = (cap > 0.f ? cap * tanhf(x * A.scale / cap) * kLog2e : x * sl2) + slope * (float)(key - pos);
      }
    }
    prob[wave][lane] = s;
    base[wave][lane] = at;
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
    prob[wave][lane] = p;
    __syncthreads();
    for (int j = 0; j < 64; ++j) {
      if (base[wave][j] < 0) continue;
      const raw* const vr = (const raw*)A.v_cache + base[wave][j];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < D) o[c] = __builtin_fmaf(prob[wave][j], E::get(vr[lane + 64 * c]), o[c]);
    }
    __syncthreads();
  }
  for (int c = 0; c < 4; ++c) part[wave][lane + 64 * c] = o[c];
  if (lane == 0) part[wave][256] = m, part[wave][257] = l;
  __syncthreads();
  float mt = -INFINITY, lt = 0.f, x = 0.f;
  for (int w = 0; w < 4; ++w) mt = fmaxf(mt, part[w][256]);
  const float ref = mt == -INFINITY ? 0.f : mt;
  for (int w = 0; w < 4; ++w) {
    const float f = exp2f(part[w][256] - ref);
    lt += part[w][257] * f;
    x += part[w][tid] * f;
  }
  if (tid < D) ((raw*)A.o)[(t * A.Hq + h) * D + tid] = E::put(lt == 0.f ? 0.f : x / lt);
}

}  // namespace

void launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.D < 1 || a.D > 256 || a.Hkv < 1 || a.Hq < 1 || a.Hq > 65535 || a.Hq % a.Hkv || a.P < 1)
    fail(PJRT_Error_Code_INTERNAL, "paged_attention of a shape the kernels do not take");
  if (a.T == 0) return record_done(done, stream);
  with_elem(a.dtype, [&](auto e) {
    launch_k(done, paged_attention_any_kernel<decltype(e)>, dim3((unsigned)a.T, (unsigned)a.Hq), dim3(256), 0, stream, a);
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("paged_attention launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
