// ryft.sample: a token for each row of logits (the definition stands at SampleArgs in kernel_abi.h).
//
// Weights are exp((x - max) / temperature) in f64, held as 64-bit integers of the largest power-of-two scale at which a
// row's sum cannot overflow (2^45 for 2^17 tokens): sums of integers do not depend on their order, so the result does
// not depend on how the row is split over lanes, wavefronts and workgroups, and a token within one part in 2^45 of a
// border falls on the side the 64-bit definition puts it on. Logits are ordered by a 32-bit key (equal for -0 and +0).
#include <hip/hip_runtime.h>

#include <string>

#include "../common.h"
#include "kernels.h"
#include "launch.h"
#include "op_device.h"

namespace ryft {

namespace {

// Unsigned order of the keys = order of the values; 0: NaN and -inf, which are never drawn.
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
  return (uint32_t)__shfl_xor((int)(uint32_t)v, m, 64) | (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), m, 64) << 32;
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
  for (int m = 32; m; m >>= 1) v += shfl_xor64(v, m);
  return v;
}

constexpr int SW = 16;  // wavefronts of a workgroup

// One workgroup a row.
template <class E>
__global__ void __launch_bounds__(SW * 64) sample_row_kernel(const SampleArgs A) {
  typedef typename E::raw raw;
  __shared__ uint64_t hist[256];
  __shared__ uint64_t sums[SW];
  __shared__ uint32_t word[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = (int)A.V;
  const int64_t r = blockIdx.x;
  const raw* const x = (const raw*)A.logits + r * A.V;
  auto key_at = [&](int i) { return logit_key(E::get(x[i])); };

  // the largest key
  uint32_t top = 0;
  for (int i = tid; i < V; i += SW * 64) top = max(top, key_at(i));
  for (int m = 32; m; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
  if (lane == 0) sums[wave] = top;
  __syncthreads();
  for (int w = 0; w < SW; ++w) top = max(top, (uint32_t)sums[w]);
  __syncthreads();
  if (top == 0) {
    if (tid == 0) A.token[r] = -1, A.logprob[r] = -INFINITY;
    return;
  }
  const float temp = A.temperature[r];
  const bool greedy = !(temp > 0.f);
  const double best = key_logit(top), t = temp;
  const double scale = (double)((uint64_t)1 << (62 - (32 - __clz(V))));
  auto real_weight = [&](uint32_t k) { return k == top ? 1.0 : exp(((double)key_logit(k) - best) / t); };
  auto weight = [&](uint32_t k) -> uint64_t {
    if (k == top) return (uint64_t)scale;
    return k == 0 || greedy ? 0 : (uint64_t)__double2ll_rn(real_weight(k) * scale);
  };
  const double minp = A.min_p[r];

  // total of f over the row
  auto total = [&](auto f) {
    uint64_t s = 0;
    for (int i = tid; i < V; i += SW * 64) s += f(i, key_at(i));
    s = wave_sum(s);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < SW; ++w) s += sums[w];
    __syncthreads();
    return s;
  };
  // the first index whose running sum of f exceeds target (< the total)
  auto find = [&](auto f, uint64_t target) {
    int begin = 0, end = V;
    while (end - begin > 1) {
      const int chunk = (end - begin + SW - 1) / SW, b = min(end, begin + wave * chunk), e = min(end, b + chunk);
      uint64_t s = 0;
      for (int i = b + lane; i < e; i += 64) s += f(i, key_at(i));
      s = wave_sum(s);
      if (lane == 0) sums[wave] = s;
      __syncthreads();
      int w = 0;
      for (; w < SW - 1 && sums[w] <= target; ++w) target -= sums[w];
      __syncthreads();
      begin = min(end, begin + w * chunk);
      end = min(end, begin + chunk);
    }
    return min(begin, V - 1);
  };
  // the key at which the running sum of f over keys in falling order reaches target (>= 1, <= the total), and what is
  // left of the target there: a radix search, 8 bits of the key at a time
  auto select = [&](auto f, uint64_t target, uint64_t* left) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += SW * 64) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += SW * 64) {
        const uint32_t k = key_at(i);
        if (shift == 24 || k >> (shift + 8) == prefix >> (shift + 8))
          if (const uint64_t v = f(i, k)) atomicAdd((unsigned long long*)&hist[k >> shift & 255], (unsigned long long)v);
      }
      __syncthreads();
      int d = 255;
      for (; d > 0 && hist[d] < target; --d) target -= hist[d];
      __syncthreads();
      prefix |= (uint32_t)d << shift;
    }
    *left = target;
    return prefix;
  };

  // kept: keys above `low`, and `low` itself up to index `low_last`
  uint32_t low = 1;
  int low_last = V;
  const int k = A.top_k[r];
  auto kept = [&](int i, uint32_t key) {
    return (key > low || (key == low && i <= low_last)) && (key == top || !(real_weight(key) < minp));
  };
  if (greedy) {
    low = top;
    low_last = find([&](int, uint32_t key) -> uint64_t { return key == top; }, 0);
  } else {
    if (k > 0 && k < V) {
      auto one = [&](int, uint32_t key) -> uint64_t { return key != 0; };
      const uint64_t n = total(one);
      if ((uint64_t)k < n) {
        uint64_t left;
        low = select(one, (uint64_t)k, &left);
        low_last = find([&](int, uint32_t key) -> uint64_t { return key == low; }, left - 1);
      }
    }
    const double p = A.top_p[r];
    if (p < 1.0) {
      auto mass = [&](int i, uint32_t key) -> uint64_t { return kept(i, key) ? weight(key) : 0; };
      const double want = p * (double)total(mass);
      const uint64_t target = want > 1.0 ? (uint64_t)__builtin_ceil(want) : 1;
      uint64_t left;
      const uint32_t cut = select(mass, target, &left);
      const uint64_t w = max(weight(cut), (uint64_t)1), n = (left + w - 1) / w;  // so many tokens of that key
      auto same = [&](int i, uint32_t key) -> uint64_t { return key == cut && kept(i, key); };
      const int cut_last = find(same, n - 1);
      low = cut;
      low_last = cut_last;
    }
  }
  auto mass = [&](int i, uint32_t key) -> uint64_t { return kept(i, key) ? weight(key) : 0; };
  const uint64_t z = total(mass);
  const double want = (double)A.uniform[r] * (double)z;
  const uint64_t target = want > 0 ? min((uint64_t)want, z - 1) : 0;
  const int token = find(mass, target);
  if (tid == 0) {
    A.token[r] = token;
    A.logprob[r] = (float)log(real_weight(key_at(token)) / ((double)z / scale));
  }
}

}  // namespace

void launch_sample(const SampleArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.V < 1 || a.V > (1 << 24)) fail(PJRT_Error_Code_INTERNAL, "sample of a vocabulary the kernels do not take");
  if (a.B == 0) return record_done(done, stream);
  with_elem(a.dtype, [&](auto e) {
    launch_k(done, sample_row_kernel<decltype(e)>, dim3((unsigned)a.B), dim3(SW * 64), 0, stream, a);
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("sample launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
