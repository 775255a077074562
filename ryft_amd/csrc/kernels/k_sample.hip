// ryft.sample: a token for each row of logits (the definition stands at SampleArgs in kernel_abi.h).
//
// Weights are 2^((x - max) log2 e / temperature) in 64 bits. What is kept is always the tokens down to one place (a key
// and, among equal keys, an index) in the order of the logits, whatever mix of top-k, min-p and top-p asked for it, so
// every filter is a search for a place, and the draw a search by index:
//  - sample_chunk: a row is cut into chunks, one a workgroup, which reads its chunk once into LDS and leaves its maximum,
//    the sum of weights of each of its wavefronts' stretches and, for a row that is filtered, the counts and sums of 512
//    bins of 1/8 octave below its top and the tokens of its topmost bins (its picks).
//  - sample_draw: a workgroup a row joins them (a chunk's weights are relative to its own maximum; bins are cut at
//    multiples of 1/8 octave of the logits, the same in every chunk), finds the bin of the place from the sums, and the
//    place itself from the bin's tokens: the picks where they reach that far, else one pass over the row. The token is
//    looked for in the one stretch whose running sum passes the uniform number, or among the picks.
// Within a chunk weights are summed as integers of the scale 2^48, across chunks in f64 in a fixed order: no sum depends on
// the order in which lanes, wavefronts or workgroups finish. A weight is rounded to within 2^-49 of its chunk's largest, so a
// sum over a chunk is off by 2^-36 of that at most: a token farther from a border falls on the side that the 64-bit
// definition puts it on. Logits are ordered by a 32-bit key (equal for -0 and +0). Rows whose tokens crowd into few bins
// (more than LDS holds), that have an infinite logit, or temperatures at which f32 logits are too coarse are searched key
// digit by digit (sample_row, in integers of the scale 2^51 or 2^62 / V).
//
// Two launches and small code are on purpose: joined by the workgroup that finished last, the chunks kept the registers and
// LDS of the search and ran two to a CU where four fit; and with every search inlined and unrolled (175 KB) a workgroup
// spent most of its time waiting for instructions.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../common.h"
#include "kernels.h"
#include "launch.h"
#include "op_device.h"

namespace ryft {

namespace {

constexpr int SW = 8;          // wavefronts of a workgroup
constexpr int ST = SW * 64;
constexpr int kChunk = 8192;   // logits of a chunk, at most
constexpr int kMaxChunks = 64;
constexpr int kBits = 48;      // weights of a chunk are whole numbers of the scale 2^kBits
constexpr int NB = 512;        // bins of a chunk: 64 octaves below its top; what is in the last is 2^-63 of it and left out
constexpr int kPicks = 1024;   // a chunk's picks, at most
constexpr int kList = 3840;    // tokens that LDS holds
constexpr int kAll = 1024;     // tokens up to which all that is kept is listed, if it need not be (3800: 29 us, as one bin 17)
constexpr int kFew = 1024;     // top_k up to which the counts alone lead to a list of all that is kept (64 rows 33 us; sums too: 41)
constexpr int kStretch = kChunk / SW;
constexpr int kStats = 4 + SW; // words of a chunk's results before its bins

// Unsigned order of the keys = order of the values; 0: NaN and -inf, which are never drawn.
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// Running results over a wavefront's lanes (inclusive; all lanes take part), by moves between lanes inside the registers: a
// search is little else than these, and each took six trips through LDS (one filtered row of 32000 logits 24 us, 20 so; 64
// mixed rows of 128256 70 and 58).
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T from_lane(T v, T none) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
  } else {
    const uint64_t a = __builtin_bit_cast(uint64_t, v), b = __builtin_bit_cast(uint64_t, none);
    const uint32_t lo = __builtin_amdgcn_update_dpp((int)(uint32_t)b, (int)(uint32_t)a, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp((int)(b >> 32), (int)(a >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
  }
}
template <class T, class F>
__device__ __forceinline__ T running(T v, T none, F&& op) {
  v = op(v, from_lane<0x111, 0xf>(v, none));  // from 1, 2, 4 and 8 lanes below, in rows of 16
  v = op(v, from_lane<0x112, 0xf>(v, none));
  v = op(v, from_lane<0x114, 0xf>(v, none));
  v = op(v, from_lane<0x118, 0xf>(v, none));
  v = op(v, from_lane<0x142, 0xa>(v, none));  // from lane 15 of the row below, for rows 1 and 3
  v = op(v, from_lane<0x143, 0xc>(v, none));  // from lane 31, for rows 2 and 3
  return v;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32;
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
  return __builtin_bit_cast(double, lane64(__builtin_bit_cast(uint64_t, v), lane));
}
__device__ __forceinline__ uint64_t scan64(uint64_t v) {
  return running(v, (uint64_t)0, [](uint64_t a, uint64_t b) { return a + b; });
}
__device__ __forceinline__ int scan32(int v) {
  return running(v, 0, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ double scan_f64(double v) {
  return running(v, 0.0, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return lane64(scan64(v), 63); }
__device__ __forceinline__ uint64_t wave_min(uint64_t v) {
  return lane64(running(v, ~(uint64_t)0, [](uint64_t a, uint64_t b) { return min(a, b); }), 63);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  return lane64(running(v, (uint64_t)0, [](uint64_t a, uint64_t b) { return max(a, b); }), 63);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  return __builtin_amdgcn_readlane((int)running(v, 0u, [](uint32_t a, uint32_t b) { return max(a, b); }), 63);
}

// 2^y for y <= 0, scaled by 2^bits and rounded to a whole number (2^y 2^bits < 2^52): a polynomial that interpolates
// (2^f - 1) / f at Chebyshev nodes on [-1/2, 1/2], 2^-50 off, exact at 0. The sum with 2^52 leaves the whole number in
// the low bits; kWhole is what else is in them.
constexpr uint64_t kWhole = 0x4330000000000000ull;
__device__ __forceinline__ double exp2_poly(double f) {
  double p = 0x1.e66fb851eb852p-28;
  p = __builtin_fma(p, f, 0x1.b6557a28f5c29p-24);
  p = __builtin_fma(p, f, 0x1.62bf9fba8f5c3p-20);
  p = __builtin_fma(p, f, 0x1.ffcb77e7acccdp-17);
  p = __builtin_fma(p, f, 0x1.4309131abdeb8p-13);
  p = __builtin_fma(p, f, 0x1.5d87fe902d461p-10);
  p = __builtin_fma(p, f, 0x1.3b2ab6fb9dbeep-7);
  p = __builtin_fma(p, f, 0x1.c6b08d7044325p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff82c5a9p-3);
  p = __builtin_fma(p, f, 0x1.62e42fefa39f7p-1);
  return __builtin_fma(p, f, 1.0);
}
__device__ __forceinline__ double exp2_neg(double y, int bits) {
  y = fmax(y, -2000.0);  // (NaN too: infinity less infinity, or its product with 0)
  const double n = __builtin_rint(y);
  return __builtin_ldexp(exp2_poly(y - n), (int)n + bits);
}

// Weights of a row relative to one of its logits.
struct Weights {
  double at, c;  // the logit; log2 e / temperature
  int bits;
  __device__ double real(float x) const { return (double)x == at ? 1.0 : exp2_neg(((double)x - at) * c, 0); }
  __device__ __forceinline__ uint64_t raw(float x) const {  // + kWhole; x > -inf
    const double w = (double)x == at ? __builtin_ldexp(1.0, bits) : exp2_neg(((double)x - at) * c, bits);
    return __builtin_bit_cast(uint64_t, w + 4503599627370496.0);
  }
  __device__ uint64_t whole(float x) const { return raw(x) - kWhole; }
};

// Weights relative to a maximum, many at a time: no branches, where every distance to it is finite and f32 fine enough
// (`usual`). What is below `least` counts as it (its weight is 0), NaN too.
struct FastWeights {
  double at, c;
  float least;
  bool usual;
  __device__ __forceinline__ FastWeights(float top, double c_) : at(top), c(c_) {
    least = (float)((double)top - 1000.0 / c_);
    const double y = ((double)least - at) * c;
    usual = y > -1020.0 && y < -100.0;
  }
  __device__ __forceinline__ uint64_t raw(float x) const {  // of the scale 2^kBits, + kWhole
    constexpr double kRint = 6755399441055744.0;  // 1.5 · 2^52: a sum with it is rounded to a whole number, in its low bits
    const double d = (double)fmaxf(x, least) - at, t = __builtin_fma(d, c, kRint);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
    const double p = exp2_poly(__builtin_fma(d, c, kRint - t));
    const uint64_t w = __builtin_bit_cast(uint64_t, p) + ((uint64_t)((n + kBits) << 20) << 32);
    return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, w) + 4503599627370496.0);
  }
  __device__ __forceinline__ uint64_t whole(float x) const { return raw(x) - kWhole; }
};

typedef uint32_t u32x4s __attribute__((ext_vector_type(4)));
typedef float f32x4s __attribute__((ext_vector_type(4)));

// The launch's arguments where they are (asked for in a kernel only). What is not inlined takes these: a reference to a kernel's own copy would put the
// copy, and the functions' frames, into scratch memory. (No kernel here has any.)
__device__ __forceinline__ const SampleArgs& sample_args() {
  return *(const SampleArgs*)(const void*)__builtin_amdgcn_kernarg_segment_ptr();
}

// What a workgroup has in LDS.
struct ChunkLds {
  float x[kChunk];
  uint64_t mass[NB];
  uint32_t count[NB];  // then running counts
  uint32_t top[SW];
  int count_sums[SW];
  int n, index;
};
struct SampleLds {
  uint64_t list[kList];                  // tokens: key << 32 | ~index
  uint64_t weight[kList];                // relative to the row's maximum, at least 1
  double row_mass[NB];                   // the row's bins, running sums of falling order
  uint32_t row_count[NB];
  uint64_t digits[256];
  uint32_t digit_count[256];
  uint64_t sums[SW], low[SW], high[SW];
  double mass_sums[SW];
  int count_sums[SW];
  uint64_t kept[kMaxChunks];             // sum of a chunk's kept weights, relative to its own maximum
  double factor[kMaxChunks];             // its maximum's weight
  uint32_t top[kMaxChunks];
  int shift[kMaxChunks];                 // bins from the row's top to the chunk's
  int pick_bin[kMaxChunks], picks[kMaxChunks];
  uint64_t place;
  int n, index;
};
static_assert(sizeof(ChunkLds) <= 40 * 1024 && sizeof(SampleLds) <= 80 * 1024, "four workgroups share a CU, and two");

// A row in chunks of whole 16 bytes of the operand's own grid (it is 16-byte aligned, its rows need not be): chunk ch has
// the grid's 16 bytes [ch · per, (ch + 1) · per) from the row's first on.
template <class E>
struct Rows {
  typedef typename E::raw raw;
  static constexpr int ES = sizeof(raw), VEC = 16 / ES;
  const raw* x;
  int64_t off, v0, end;  // the row's first element, the 16 bytes that hold it, whole 16 bytes of the operand
  int V, vecs, per;
  __device__ Rows(const SampleArgs& A, int64_t row) : x((const raw*)A.logits), off(row * A.V), V((int)A.V) {
    v0 = off / VEC;
    end = A.B * A.V / VEC;
    vecs = (int)((off + V + VEC - 1) / VEC - v0);
    per = A.chunks ? (vecs + A.chunks - 1) / A.chunks : vecs;
  }
  __device__ __forceinline__ float at(int i) const { return E::get(x[off + i]); }
  // index in the row of element 0 of its 16 bytes v
  __device__ __forceinline__ int index(int v) const { return (int)((v0 + v) * VEC - off); }
  // the chunk that an index lies in
  __device__ __forceinline__ int chunk(int i) const { return (int)(((off + i) / VEC - v0) / per); }
  // 16 bytes v (read as the operand's last whole ones where they end past it)
  __device__ __forceinline__ u32x4s load(int v) const { return ((const __attribute__((address_space(1))) u32x4s*)x)[min(v0 + v, end - 1)]; }
  __device__ __forceinline__ float get(const u32x4s& w, int e) const {
    if constexpr (ES == 4) return __uint_as_float(w[e]);
    else return E::get((raw)(w[e / 2] >> (16 * (e % 2))));
  }
  // Chunk ch as f32 in LDS, at element p what has index first + p in the row, -inf where that is none. Every thread calls.
  __device__ __forceinline__ int stage(ChunkLds& sh, int ch) const {
    constexpr int U = kChunk / VEC / ST;
    const int tid = threadIdx.x, b = ch * per, n = min(per, vecs - b), first = index(b);
    u32x4s w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = load(min(b + u * ST + tid, vecs - 1));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = u * ST + tid;
#pragma unroll
      for (int q = 0; q < VEC / 4; ++q) {
        f32x4s f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = v < n ? get(w[u], 4 * q + e) : -INFINITY;
        *(f32x4s*)(sh.x + v * VEC + 4 * q) = f;
      }
    }
    __syncthreads();
    // the row's first and last 16 bytes, element by element: they may hold another row's, and end past the operand
    if (tid < 2 * VEC) {
      const int v = tid < VEC ? 0 : vecs - 1, e = tid % VEC, i = index(v) + e;
      if (v >= b && v < b + n) sh.x[(v - b) * VEC + e] = i >= 0 && i < V ? at(i) : -INFINITY;
    }
    __syncthreads();
    return first;
  }
};

// Results of a row's chunk in the workspace: top key and first index of it, last picked bin and number of picks, whether
// its weights could be summed, the sums of its stretches; the bins' sums, their counts (two a word); the picks.
constexpr int kChunkWords = kStats + NB + NB / 2 + kPicks;
struct ChunkWs {
  uint64_t *stats, *mass, *picks;
  uint32_t* count;
  // (each kind together, so that a row's chunks lie next to each other)
  __device__ __forceinline__ ChunkWs(const SampleArgs& A, int64_t rc) {
    const int64_t all = (int64_t)A.rows * A.chunks;
    uint64_t* const ws = (uint64_t*)A.ws;
    stats = ws + rc * kStats;
    mass = ws + all * kStats + rc * NB;
    count = (uint32_t*)(ws + all * (kStats + NB)) + rc * NB;
    picks = ws + all * (kStats + NB + NB / 2) + rc * kPicks;
  }
};

__device__ __forceinline__ uint64_t block_sum(uint64_t s, SampleLds& sh) {
  const int tid = threadIdx.x;
  s = wave_sum(s);
  __syncthreads();
  if ((tid & 63) == 0) sh.sums[tid >> 6] = s;
  __syncthreads();
  s = 0;
  for (int w = 0; w < SW; ++w) s += sh.sums[w];
  return s;
}

// The first index of [begin, end) at which the running sum of f(index, logit) passes target (below the sum). Each step
// leaves the segment of one wavefront, then the lanes of one.
template <class E, class F>
__device__ __forceinline__ int find_index(const SampleArgs& A, int64_t row, int begin, int end, uint64_t target, SampleLds& sh, F&& f) {
  typedef typename E::raw raw;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const raw* const x = (const raw*)A.logits + row * A.V;
  const int last = end - 1;
  while (end - begin > 64) {
    const int part = (end - begin + SW - 1) / SW, b = min(end, begin + wave * part), e = min(end, b + part);
    uint64_t s = 0;
#pragma unroll 1
    for (int i = b + lane; i < e; i += 64) s += f(i, E::get(x[i]));
    s = wave_sum(s);
    __syncthreads();
    if (lane == 0) sh.sums[wave] = s;
    __syncthreads();
    int w = 0;
#pragma unroll 1
    for (; w < SW - 1 && sh.sums[w] <= target; ++w) target -= sh.sums[w];
    begin = min(end, begin + w * part);
    end = min(end, begin + part);
  }
  const uint64_t s = scan64(begin + lane < end ? f(begin + lane, E::get(x[begin + lane])) : 0);
  const uint64_t past = __builtin_amdgcn_ballot_w64(s > target);
  return past ? min(last, begin + __builtin_ctzll(past)) : last;
}

// A whole row by one workgroup, key digit by digit, with no list: every search is four passes over the row, however its
// logits crowd.
template <class E>
__device__ __attribute__((noinline)) void sample_row(const SampleArgs& A, int64_t r, uint32_t top, SampleLds& sh) {
  typedef typename E::raw raw;
  uint64_t* const hist = sh.digits;
  const int tid = threadIdx.x, V = (int)A.V;
  const raw* const x = (const raw*)A.logits + r * A.V;
  auto key_at = [&](int i) { return logit_key(E::get(x[i])); };
  const double t = A.temperature[r], best = key_logit(top);
  const int bits = 62 - (32 - __clz(V));
  const Weights wt{best, 1.4426950408889634 / t, min(bits, 51)};
  auto weight = [&](uint32_t k) -> uint64_t { return k == 0 ? 0 : wt.whole(key_logit(k)); };
  const double minp = A.min_p[r];
  auto total = [&](auto f) {
    uint64_t s = 0;
#pragma unroll 1
    for (int i = tid; i < V; i += ST) s += f(i, key_at(i));
    return block_sum(s, sh);
  };
  auto find = [&](auto f, uint64_t target) {
    return find_index<E>(A, r, 0, V, target, sh, [&](int i, float v) { return f(i, logit_key(v)); });
  };
  // the key at which the running sum of f over keys in falling order reaches target (>= 1, <= the total), and what is
  // left of the target there: a radix search, 8 bits of the key at a time
  auto select = [&](auto f, uint64_t target, uint64_t* left) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = tid; i < 256; i += ST) hist[i] = 0;
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < V; i += ST) {
        const uint32_t k = key_at(i);
        if (shift == 24 || k >> (shift + 8) == prefix >> (shift + 8))
          if (const uint64_t v = f(i, k)) atomicAdd((unsigned long long*)&hist[k >> shift & 255], (unsigned long long)v);
      }
      __syncthreads();
      int d = 255;
#pragma unroll 1
      for (; d > 0 && hist[d] < target; --d) target -= hist[d];
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
    return (key > low || (key == low && i <= low_last)) && !(wt.real(key_logit(key)) < minp);
  };
  if (k > 0 && k < V) {
    auto one = [&](int, uint32_t key) -> uint64_t { return key != 0; };
    const uint64_t n = total(one);
    if ((uint64_t)k < n) {
      uint64_t left;
      low = select(one, (uint64_t)k, &left);
      low_last = find([&](int, uint32_t key) -> uint64_t { return key == low; }, left - 1);
    }
  }
  auto mass = [&](int i, uint32_t key) -> uint64_t { return kept(i, key) ? weight(key) : 0; };
  const double p = A.top_p[r];
  if (p < 1.0) {
    const double want = p * (double)total(mass);
    const uint64_t target = want > 1.0 ? (uint64_t)__builtin_ceil(want) : 1;
    uint64_t left;
    const uint32_t cut = select(mass, target, &left);
    const uint64_t w = max(weight(cut), (uint64_t)1), n = (left + w - 1) / w;  // so many tokens of that key
    const int cut_last = find([&](int i, uint32_t key) -> uint64_t { return key == cut && kept(i, key); }, n - 1);
    low = cut;
    low_last = cut_last;
  }
  const uint64_t z = total(mass);
  const double want = (double)A.uniform[r] * (double)z;
  // (no target: the first token kept that has any weight, however little)
  const int token = want > 0 ? find(mass, min((uint64_t)want, z - 1))
                             : find([&](int i, uint32_t key) -> uint64_t { return key && kept(i, key) && wt.real(key_logit(key)) > 0; }, 0);
  if (tid == 0) {
    A.token[r] = token;
    A.logprob[r] = (float)log(wt.real(key_logit(key_at(token))) / __builtin_ldexp((double)z, -wt.bits));
  }
}

// Bin of a logit below one of at least its size: whole eighths of an octave, monotone in the logit, and the same
// wherever it is asked relative to `top8`, the floor of a maximum's eighths.
__device__ __forceinline__ float eighths(float x, float c8) { return __builtin_floorf(x * c8); }
__device__ __forceinline__ int bin_below(float top8, float x, float c8, bool is_top) {
  if (is_top) return 0;
  const float d = top8 - eighths(x, c8);
  return d < (float)(NB - 1) ? (int)d : NB - 1;  // (NaN: NB - 1)
}

// The smallest key in [1, top] for which f holds (it holds for top, and for every key above one for which it does): 64
// keys at a time.
template <class F>
__device__ __forceinline__ uint32_t lowest_key(uint32_t top, F&& f) {
  uint64_t lo = 0, hi = top;  // f does not hold at lo (0 stands for none), holds at hi
  const int lane = threadIdx.x & 63;
  while (hi - lo > 1) {
    const uint64_t step = (hi - lo + 63) / 64, k = lo + step * (lane + 1);
    const uint64_t holds = __builtin_amdgcn_ballot_w64(k < hi ? f((uint32_t)k) : true);
    const int first = __builtin_ctzll(holds);
    const uint64_t nlo = lo + step * first;
    hi = min(hi, nlo + step);
    lo = nlo;
  }
  return (uint32_t)hi;
}

// The same, looked for next to a guess first.
template <class F>
__device__ __forceinline__ uint32_t lowest_key_near(uint32_t guess, uint32_t top, F&& f) {
  if (guess > 64 && guess < top) {
    const uint32_t k = guess - 32 + (threadIdx.x & 63);
    const uint64_t holds = __builtin_amdgcn_ballot_w64(k < top ? f(k) : true);
    if (holds && !(holds & 1)) return min(top, guess - 32 + (uint32_t)__builtin_ctzll(holds));
  }
  return lowest_key(top, f);
}
// The smallest key whose bin below `top8` is at most `bin`.
__device__ __attribute__((noinline)) uint32_t lowest_of_bin(uint32_t top, float top8, float c8, int bin) {
  const float ftop = key_logit(top);
  return lowest_key_near(logit_key((top8 - (float)bin) / c8), top, [&](uint32_t key) {
    const float x = key_logit(key);
    return bin_below(top8, x, c8, x == ftop) <= bin;
  });
}
// The smallest key whose weight is at least minp.
__device__ __attribute__((noinline)) uint32_t lowest_of_weight(uint32_t top, double at, double c, double minp) {
  const Weights w{at, c, 0};
  return lowest_key_near(logit_key((float)(at + (double)log2f((float)minp) / c)), top, [&](uint32_t key) { return !(w.real(key_logit(key)) < minp); });
}

// Room for `mine` entries of each lane in a list of *n so far: where this lane's begin. One atomic a wavefront.
__device__ __forceinline__ int list_room(int* n, int mine) {
  const int incl = scan32(mine);
  int base = 0;
  if ((threadIdx.x & 63) == 63 && incl) base = atomicAdd(n, incl);
  return __builtin_amdgcn_readlane(base, 63) + incl - mine;
}

// Of the list's entries of at least `cut`, in falling order (by_index: in rising order of their indexes): the one at which
// the running sum of their weights (ones: of 1) reaches target, the last if it never does. Its value, or the lower half of
// it. The bits in which the entries differ, 8 at a time, until one entry is left.
__device__ __attribute__((noinline)) uint64_t list_select(SampleLds& sh, uint64_t cut, bool by_index, bool ones, uint64_t target) {
  const int tid = threadIdx.x, lane = tid & 63, n = sh.n;
  const uint64_t mask = by_index ? 0xffffffffu : ~(uint64_t)0;
  uint64_t low = ~(uint64_t)0, high = 0;
  for (int i = tid; i < n; i += ST) {
    const uint64_t e = sh.list[i];
    if (e >= cut) low = min(low, e & mask), high = max(high, e & mask);
  }
  low = wave_min(low), high = wave_max(high);
  __syncthreads();
  if (lane == 0) sh.low[tid >> 6] = low, sh.high[tid >> 6] = high;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SW; ++w) low = min(low, sh.low[w]), high = max(high, sh.high[w]);
  int bits = low >= high ? 0 : 64 - __clzll(low ^ high);  // (what is left of a value; above them all agree with prefix)
  uint64_t prefix = bits < 64 ? high >> bits : 0;
  while (bits > 0) {
    const int step = min(8, bits), above = bits;
    bits -= step;
    if (tid < 256) sh.digits[tid] = 0, sh.digit_count[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += ST) {
      const uint64_t e = sh.list[i], v = e & mask;
      if (e >= cut && (above == 64 || v >> above == prefix)) {
        const int d = (int)(v >> bits) & ((1 << step) - 1);
        atomicAdd((unsigned long long*)&sh.digits[d], ones ? 1ull : (unsigned long long)sh.weight[i]);
        atomicAdd(&sh.digit_count[d], 1u);
      }
    }
    __syncthreads();
    // every wavefront: lane l has the digits 255 - 4 l and the three below
    uint64_t d[4], s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = sh.digits[255 - 4 * lane - i], s += d[i];
    const uint64_t incl = scan64(s);
    const uint64_t reach = __builtin_amdgcn_ballot_w64(incl >= target), some = __builtin_amdgcn_ballot_w64(s > 0);
    const int who = reach ? __builtin_ctzll(reach) : some ? 63 - __builtin_clzll(some) : 0;
    uint64_t before = incl - s, at = before;
    int digit = 255 - 4 * lane;
    bool got = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!got && d[i] > 0) digit = 255 - 4 * lane - i, at = before, got = before + d[i] >= target;
      before += d[i];
    }
    digit = __builtin_amdgcn_readlane(digit, who);
    at = lane64(at, who);
    target = target > at ? target - at : 0;
    prefix = prefix << step | (uint64_t)digit;
    const bool one = sh.digit_count[digit] == 1;
    __syncthreads();
    if (one) {
      for (int i = tid; i < n; i += ST) {
        const uint64_t e = sh.list[i];
        if (e >= cut && ((e & mask) >> bits) == prefix) sh.place = e & mask;
      }
      __syncthreads();
      return sh.place;
    }
  }
  return prefix;
}

// i & bit ? a : b, as one instruction (the compiler makes an array in memory of a tree of these)
__device__ __forceinline__ float select_bit(int i, int bit, float a, float b) {
  float y;
  asm("v_cndmask_b32 %0, %1, %2, %3" : "=v"(y) : "v"(b), "v"(a), "s"(__builtin_amdgcn_ballot_w64(i & bit)));
  return y;
}
// The list: the row's tokens with keys in [from, to), by a pass over the row, 32 logits a thread in flight.
template <class E>
__device__ __attribute__((noinline)) void list_row(const SampleArgs& A, int64_t r, SampleLds& sh, uint32_t from, uint32_t to) {
  constexpr int VEC = Rows<E>::VEC;
  const Rows<E> row(A, r);
  const int tid = threadIdx.x;
  const float least = key_logit(from), past = key_logit(to);  // (NaN: past +inf)
  // (between the row's first and last 16 bytes)
  constexpr int U = 32 / VEC;
  u32x4s next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = row.load(min(1 + u * ST + tid, row.vecs - 1));
  for (int b = 1; b < row.vecs - 1; b += U * ST) {
    float x[32];
    uint32_t hits = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        x[u * VEC + e] = row.get(next[u], e);
        bits |= (x[u * VEC + e] >= least && !(x[u * VEC + e] >= past) ? 1u : 0u) << e;
      }
      if (b + u * ST + tid < row.vecs - 1) hits |= bits << (u * VEC);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = row.load(min(b + (U + u) * ST + tid, row.vecs - 1));
    int at = list_room(&sh.n, __builtin_popcount(hits));
    // (from the registers, by a tree of selections: a branch for each logit took 3 us a pass, read again every token waited
    // for memory)
    while (hits) {
      const int i = __builtin_ctz(hits);
      hits &= hits - 1;
      float y[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) y[k] = select_bit(i, 16, x[k + 16], x[k]);
#pragma unroll
      for (int half = 8; half; half >>= 1)
#pragma unroll
        for (int k = 0; k < half; ++k) y[k] = select_bit(i, half, y[k + half], y[k]);
      if (at < kList) sh.list[at] = (uint64_t)logit_key(y[0]) << 32 | (uint32_t)~(row.index(b + i / VEC * ST + tid) + i % VEC);
      ++at;
    }
  }
  if (tid < 64) {
    const int i = tid < VEC ? row.index(0) + tid : row.vecs > 1 && tid < 2 * VEC ? row.index(row.vecs - 1) + tid - VEC : -1;
    const uint32_t key = i >= 0 && i < row.V ? logit_key(row.at(i)) : 0;
    const int at = list_room(&sh.n, key >= from && key < to);
    if (key >= from && key < to && at < kList) sh.list[at] = (uint64_t)key << 32 | (uint32_t)~i;
  }
}

// Whether a row takes the first of its largest logits: no weight is at least a min_p above 1, and the largest is kept.
__device__ __forceinline__ bool greedy_row(const SampleArgs& A, int64_t r) { return !(A.temperature[r] > 0.f) || !(A.min_p[r] <= 1.f); }

// What a row asks for.
struct Wanted {
  bool greedy, by_count, by_weight, by_mass, filtered;
  bool few;           // no sums of weights are needed: all that can be kept will be listed
  int k;
  double minp, p, c;  // log2 e / temperature
  float c8;           // eighths of an octave a unit of logit
  __device__ __forceinline__ Wanted(const SampleArgs& A, int64_t r) {
    const float temp = A.temperature[r];
    k = A.top_k[r];
    minp = A.min_p[r], p = A.top_p[r];
    greedy = greedy_row(A, r);
    by_count = k > 0 && k < A.V, by_weight = minp > 0.0, by_mass = p < 1.0;
    filtered = !greedy && (by_count || by_weight || by_mass);
    few = filtered && by_count && k <= kFew;
    c = 1.4426950408889634 / (double)temp;
    c8 = (float)(8.0 * c);
  }
};

template <class E>
__global__ void __launch_bounds__(ST, 8) sample_chunk_kernel(const SampleArgs A) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  ChunkLds& sh = *(ChunkLds*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, C = A.chunks;
  const int64_t r = blockIdx.x / C + A.row0;
  const Rows<E> row(A, r);
  const int first = row.stage(sh, blockIdx.x % C);
  const Wanted want(A, r);
  const ChunkWs ws(A, blockIdx.x);
  auto each = [&](auto&& f) {  // f(place in LDS, logit), for the wavefront's stretch
#pragma unroll 1
    for (int u = 0; u < kStretch / 256; ++u) {
      const int at = wave * kStretch + u * 256 + lane * 4;
      const f32x4s x = *(const f32x4s*)(sh.x + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) f(at + e, x[e]);
    }
  };
  float best = -INFINITY;
  each([&](int, float x) { best = fmaxf(best, x); });
  const uint32_t wave_top = wave_max(logit_key(best));
  if (lane == 0) sh.top[wave] = wave_top;
  if (want.filtered) sh.mass[tid] = 0, sh.count[tid] = 0;
  if (tid == 0) sh.index = row.V, sh.n = 0;
  __syncthreads();
  uint32_t top = 0;
#pragma unroll
  for (int w = 0; w < SW; ++w) top = max(top, sh.top[w]);
  const float ctop = key_logit(top), ctop8 = eighths(ctop, want.c8);
  const FastWeights fast(ctop, want.c);
  const bool usual = !top || want.greedy || fast.usual;
  uint64_t sum = 0;
  if (top && want.greedy) {
    int i0 = row.V;
    each([&](int at, float x) { if (x == ctop) i0 = min(i0, first + at); });
    if (i0 < row.V) atomicMin(&sh.index, i0);
    __syncthreads();
  } else if (top && want.few) {
    each([&](int, float x) {
      const float d = ctop8 - eighths(x, want.c8);
      if (d < (float)(NB - 1)) atomicAdd(&sh.count[(int)d], 1u);
    });
  } else if (top && usual) {
    each([&](int, float x) {
      const uint64_t w = fast.raw(x);
      sum += w;
      if (want.filtered) {
        const float d = ctop8 - eighths(x, want.c8);
        if (d < (float)(NB - 1)) {  // (NaN and -inf: not)
          atomicAdd((unsigned long long*)&sh.mass[(int)d], (unsigned long long)(w - kWhole));
          atomicAdd(&sh.count[(int)d], 1u);
        }
      }
    });
    sum = wave_sum(sum - (uint64_t)(kChunk / ST) * kWhole);
  }
  if (lane == 0) ws.stats[4 + wave] = sum;
  int picked = -1;
  if (want.filtered) {
    __syncthreads();
    if (!want.few) ws.mass[tid] = sh.mass[tid];
    ws.count[tid] = sh.count[tid];
    // The picks: whole bins from the top, as many as fit and can matter. (What top_k or min_p keep of the row's tokens is
    // among what they would keep of the chunk's.)
    int n = scan32(sh.count[tid]);
    if (lane == 63) sh.count_sums[wave] = n;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SW; ++w) n += w < wave ? sh.count_sums[w] : 0;
    sh.count[tid] = n;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NB / 64; ++i) picked += __builtin_popcountll(__builtin_amdgcn_ballot_w64(sh.count[64 * i + lane] <= kPicks));
    picked = min(picked, NB - 2);
    if (want.by_count) {
      int below = 0;  // bins before the one that reaches k
#pragma unroll
      for (int i = 0; i < NB / 64; ++i) below += __builtin_popcountll(__builtin_amdgcn_ballot_w64(sh.count[64 * i + lane] < (uint32_t)want.k));
      picked = min(picked, below);
    }
    if (want.by_weight) picked = (int)fminf((float)picked, 2.f - 8.f * log2f((float)want.minp));
    if (picked >= 0 && top && usual) {
      const float least = key_logit(lowest_of_bin(top, ctop8, want.c8, picked));
      int mine = 0;
      each([&](int, float x) { mine += x >= least; });
      int to = list_room(&sh.n, mine);
      if (__builtin_amdgcn_ballot_w64(mine > 0))
        each([&](int at, float x) {
          if (x >= least && to < kPicks) ws.picks[to++] = (uint64_t)logit_key(x) << 32 | (uint32_t)~(first + at);
        });
    }
    __syncthreads();
  }
  if (tid == 0) {
    ws.stats[0] = top | (uint64_t)(uint32_t)sh.index << 32;
    ws.stats[1] = (uint32_t)picked | (uint64_t)(uint32_t)sh.n << 32;
    ws.stats[2] = usual;
  }
}

// The place down to which a filtered row's tokens are kept, in sh.kept each chunk's kept weights; or 0, and the draw is
// done.
template <class E>
__device__ __forceinline__ uint64_t filtered(const SampleArgs& A, int64_t r, uint32_t key_top, double all, SampleLds& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, C = A.chunks;
  const int64_t rc0 = (r - A.row0) * C;
  const Rows<E> row(A, r);
  const Wanted want(A, r);
  const double unit = __builtin_ldexp(1.0, -kBits), uniform = A.uniform[r];
  const float ftop = key_logit(key_top), top8 = eighths(ftop, want.c8);
  const Weights rw{(double)ftop, want.c, 0};
  uint64_t cut = (uint64_t)1 << 32;  // kept: entries key << 32 | ~index of at least this
  auto bin_of = [&](uint32_t key) { const float f = key_logit(key); return bin_below(top8, f, want.c8, f == ftop); };
  // bins of the row, then running sums over them
  double m = 0;
  int n = 0;
  const ChunkWs ws(A, rc0);
  for (int i0 = 0; i0 < C; i0 += 16) {  // (16 chunks' loads in flight)
    uint64_t w[16];
    uint32_t q[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int i = min(i0 + u, C - 1), b = min(max(tid - sh.shift[i], 0), NB - 1);
      q[u] = ws.count[i * NB + b];
      w[u] = 0;
    }
    if (!want.few)  // (a branch for all of them: with one each they followed each other)
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const int i = min(i0 + u, C - 1);
        w[u] = ws.mass[i * NB + min(max(tid - sh.shift[i], 0), NB - 1)];
      }
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int i = min(i0 + u, C - 1);
      const bool in = i0 + u < C && tid >= sh.shift[i] && tid - sh.shift[i] < NB - 1;
      m += in ? (double)w[u] * unit * sh.factor[i] : 0.0;
      n += in ? (int)q[u] : 0;
    }
  }
  m = scan_f64(m);
  n = scan32(n);
  if (lane == 63) sh.mass_sums[wave] = m, sh.count_sums[wave] = n;
  __syncthreads();
  double before = 0;
#pragma unroll
  for (int w = 0; w < SW; ++w) before += w < wave ? sh.mass_sums[w] : 0.0, n += w < wave ? sh.count_sums[w] : 0;
  sh.row_mass[tid] = before + m, sh.row_count[tid] = n;
  __syncthreads();
  // the first bin whose running count or sum reaches a target (NB: none does)
  auto first_bin_of = [&](auto&& reaches) {
    int b = NB;
    for (int i = NB / 64 - 1; i >= 0; --i)
      if (const uint64_t m = __builtin_amdgcn_ballot_w64(reaches(64 * i + lane))) b = 64 * i + __builtin_ctzll(m);
    return b;
  };
  bool crowded = false;
  int first_bin = NB, last_bin = -1;  // bins whose tokens the list has
  // `bin` and, where they are not too many to search, all above: from the picks if they reach that far, else from the row
  auto collect = [&](int bin) {
    const uint32_t above = bin ? sh.row_count[bin - 1] : 0;
    first_bin = sh.row_count[bin] <= (want.few ? kList : kAll) ? 0 : bin;
    last_bin = bin;
    crowded = sh.row_count[bin] - (first_bin ? above : 0) > kList;
    if (crowded) return;
    const bool reach = !__builtin_amdgcn_ballot_w64(sh.top[lane] && bin - sh.shift[lane] > sh.pick_bin[lane]);
    __syncthreads();
    if (tid == 0) sh.n = 0;
    __syncthreads();
    if (reach) {
      // a chunk's picks to a wavefront, four loads in flight
      for (int ch = wave; ch < C; ch += SW) {
        const uint64_t* const picks = ws.picks + ch * kPicks;
        for (int i0 = 0; i0 < sh.picks[ch]; i0 += 4 * 64) {
          uint64_t e[4];
          bool in[4];
          int mine = 0;
#pragma unroll
          for (int u = 0; u < 4; ++u) e[u] = i0 + 64 * u + lane < sh.picks[ch] ? picks[i0 + 64 * u + lane] : 0;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int b = e[u] ? bin_of((uint32_t)(e[u] >> 32)) : NB;
            in[u] = b <= bin && b >= first_bin;
            mine += in[u];
          }
          int to = list_room(&sh.n, mine);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (in[u]) {
              if (to < kList) sh.list[to] = e[u];
              ++to;
            }
        }
      }
    } else {
      list_row<E>(sample_args(), r, sh, lowest_of_bin(key_top, top8, want.c8, bin), first_bin ? lowest_of_bin(key_top, top8, want.c8, bin - 1) : key_top + 1);
    }
    __syncthreads();
    crowded = sh.n > kList;
    const FastWeights fast(ftop, want.c);
    for (int i = tid; i < min(sh.n, kList); i += ST) sh.weight[i] = max(fast.whole(key_logit((uint32_t)(sh.list[i] >> 32))), (uint64_t)1);
    __syncthreads();
  };
  // sum of the listed weights from the cut on
  auto listed = [&]() {
    uint64_t s = 0;
    for (int i = tid; i < sh.n; i += ST)
      if (sh.list[i] >= cut) s += sh.weight[i];
    return block_sum(s, sh);
  };
  int cut_bin = NB;
  if (want.by_weight) {
    const uint32_t key = lowest_of_weight(key_top, ftop, want.c, want.minp);
    if (bin_of(key) < NB - 1) cut = (uint64_t)key << 32, cut_bin = bin_of(key);
  }
  int count_bin = want.by_count ? first_bin_of([&](int i) { return sh.row_count[i] >= (uint32_t)want.k; }) : NB;
  if (want.few) count_bin = min(count_bin, NB - 2);  // (fewer than k in all bins: those)
  const bool cut_by_count = count_bin < NB - 1 && count_bin <= cut_bin;
  if (cut_by_count || cut_bin < NB) collect(cut_by_count ? count_bin : cut_bin);
  if (cut_by_count && !crowded) {
    // (of the list's bins from the top: all, or the last alone)
    const uint64_t e = list_select(sh, 0, false, true, (uint64_t)want.k - (first_bin ? sh.row_count[first_bin - 1] : 0));
    if (e > cut) cut = e;
    cut_bin = count_bin;
  }
  // Here the list has the cut's bin. The weights before it, and of it.
  if (want.by_mass && !crowded) {
    const double total = cut_bin < NB ? (double)listed() * unit + (first_bin ? sh.row_mass[first_bin - 1] : 0.0) : all;
    const double target = want.p * total;
    const int b = min(first_bin_of([&](int i) { return sh.row_mass[i] >= target; }), cut_bin);
    if (b < NB - 1) {
      if (b < first_bin || b > last_bin) collect(b);
      if (!crowded) {
        const double rest = __builtin_ldexp(target - (first_bin ? sh.row_mass[first_bin - 1] : 0.0), kBits);
        cut = list_select(sh, cut, false, false, rest > 1.0 ? (uint64_t)__builtin_ceil(rest) : 1);
        cut_bin = b;
      }
    }
  }
  // What top_k or min_p cut off past the bins is less than a sum over the row shows, and is left out of it: only a uniform
  // number of 0 asks for what is kept of that.
  const bool past = (want.by_count || want.by_weight) && (cut_bin == NB || (want.few && !want.by_mass && sh.row_count[NB - 2] < (uint32_t)want.k));
  if (crowded || (want.few && first_bin != 0) || (past && !(uniform > 0))) {
    sample_row<E>(sample_args(), r, key_top, sh);
    return 0;
  }
  if (cut_bin < NB && first_bin == 0) {
    // all that is kept is listed: the draw is a search by index
    const uint64_t total = listed();
    const uint64_t target = min((uint64_t)(uniform * (double)total), total - 1) + 1;
    const uint32_t at = (uint32_t)list_select(sh, cut, true, false, target);
    for (int i = tid; i < sh.n; i += ST)
      if ((uint32_t)sh.list[i] == at) {
        A.token[r] = (int)~at;
        A.logprob[r] = (float)log(rw.real(key_logit((uint32_t)(sh.list[i] >> 32))) / ((double)total * unit));
      }
    return 0;
  }
  if (cut_bin < NB) {
    // each chunk's kept weights: its bins above the cut's, and its tokens of that bin (as its own sums have them, to the
    // last bit)
    for (int i = wave; i < C; i += SW) {
      uint64_t s = 0;
      for (int b = lane; b < cut_bin - sh.shift[i]; b += 64) s += ws.mass[i * NB + b];
      s = wave_sum(s);
      if (lane == 0) sh.kept[i] = s;
    }
    __syncthreads();
    for (int i = tid; i < sh.n; i += ST) {
      const uint64_t e = sh.list[i];
      if (e < cut || bin_of((uint32_t)(e >> 32)) != cut_bin) continue;
      const int at = row.chunk((int)~(uint32_t)e);
      atomicAdd((unsigned long long*)&sh.kept[at],
                (unsigned long long)FastWeights(key_logit(sh.top[at]), want.c).whole(key_logit((uint32_t)(e >> 32))));
    }
    __syncthreads();
  }
  return cut;
}

template <class E>
__global__ void __launch_bounds__(ST, 2) sample_draw_kernel(const SampleArgs A) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  SampleLds& sh = *(SampleLds*)smem;
  constexpr int VEC = Rows<E>::VEC;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, C = A.chunks;
  const int64_t r = blockIdx.x + A.row0, rc0 = (int64_t)blockIdx.x * C;
  const Rows<E> row(A, r);
  const Wanted want(A, r);
  const double unit = __builtin_ldexp(1.0, -kBits), uniform = A.uniform[r];

  // ---- the chunks, one a lane, in every wavefront
  uint64_t head = 0, kept = 0, pick = 0, ok = 1;
  if (lane < C) {
    const uint64_t* const ws = ChunkWs(A, rc0 + lane).stats;
    head = ws[0], pick = ws[1], ok = ws[2];
#pragma unroll
    for (int w = 0; w < SW; ++w) kept += ws[4 + w];
  }
  const uint32_t top = (uint32_t)head;
  const uint32_t key_top = wave_max(top);
  if (key_top == 0 || want.greedy) {
    const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(top == key_top));
    const int index = __builtin_amdgcn_readlane((int)(head >> 32), who);
    if (tid == 0) A.token[r] = key_top ? index : -1, A.logprob[r] = key_top ? 0.f : -INFINITY;
    return;
  }
  if (__builtin_amdgcn_ballot_w64(ok == 0)) return sample_row<E>(sample_args(), r, key_top, sh);
  const float ftop = key_logit(key_top);
  const Weights rw{(double)ftop, want.c, 0};  // relative to the row's maximum
  const float ctop = key_logit(top);
  const double factor = top ? rw.real(ctop) : 0.0;
  double upto = scan_f64((double)kept * unit * factor), all = lane_f64(upto, 63);

  uint64_t cut = (uint64_t)1 << 32;  // kept: entries key << 32 | ~index of at least this
  if (want.filtered) {
    if (wave == 0) {
      sh.top[lane] = top, sh.factor[lane] = factor, sh.kept[lane] = kept;
      sh.shift[lane] = top ? bin_below(eighths(ftop, want.c8), ctop, want.c8, ctop == ftop) : NB - 1;
      sh.pick_bin[lane] = (int)(uint32_t)pick, sh.picks[lane] = lane < C ? min((int)(pick >> 32), kPicks) : 0;
    }
    __syncthreads();
    cut = filtered<E>(A, r, key_top, all, sh);
    if (!cut) return;
    kept = sh.kept[lane];
    upto = scan_f64((double)kept * unit * factor);
    all = lane_f64(upto, 63);
  }

  // ---- the draw: the chunk whose running sum passes the uniform number, its stretch, and the index in that
  const double aim = uniform * all;
  const bool none = !(aim > 0);  // the first that has any weight, however little
  const bool cut_off = cut > (uint64_t)1 << 32;
  const uint64_t passed = __builtin_amdgcn_ballot_w64(upto > aim), some = __builtin_amdgcn_ballot_w64(kept > 0 && factor > 0);
  // (none passed: rounding of the sums alone)
  int at = passed ? __builtin_ctzll(passed) : 63 - __builtin_clzll(some);
  const uint64_t have = lane64(kept, at);
  const double in = (aim - (at ? lane_f64(upto, at - 1) : 0.0)) / (unit * lane_f64(factor, at));
  uint64_t target = none ? 0 : !passed ? have - 1 : in > 0 ? min((uint64_t)in, have - 1) : 0;
  for (at = none ? 0 : at; at < C; ++at) {
    const FastWeights w(key_logit(__builtin_amdgcn_readlane(top, at)), want.c);
    const int f0 = row.index(at * row.per), places = min(row.per, row.vecs - at * row.per) * VEC;
    auto value = [&](int place) {
      const int i = f0 + place;
      const float x = row.at(min(max(i, 0), row.V - 1));
      return place < places && i >= 0 && i < row.V ? x : -INFINITY;
    };
    auto weight = [&](float x, int place) -> uint64_t {
      const bool in = x > -INFINITY && ((uint64_t)logit_key(x) << 32 | (uint32_t)~(f0 + place)) >= cut;
      return in ? none ? rw.real(x) > 0 : w.whole(x) : 0;
    };
    // the sums of its stretches: as the chunk left them, or of what is kept
    uint64_t s = 0;
    if (none || cut_off) {
      float x[kStretch / 64];
#pragma unroll
      for (int u = 0; u < kStretch / 64; ++u) x[u] = value(wave * kStretch + u * 64 + lane);
#pragma unroll
      for (int u = 0; u < kStretch / 64; ++u) s += weight(x[u], wave * kStretch + u * 64 + lane);
      s = wave_sum(s);
      __syncthreads();
      if (lane == 0) sh.sums[wave] = s;
      __syncthreads();
      s = lane < SW ? sh.sums[lane] : 0;
    } else {
      s = lane < SW ? ChunkWs(A, rc0 + at).stats[4 + lane] : 0;
    }
    const uint64_t ends = scan64(s), reach = __builtin_amdgcn_ballot_w64(ends > target);
    if (!reach && none) continue;
    const int st = reach ? min(__builtin_ctzll(reach), SW - 1) : SW - 1;
    target -= min(target, lane64(ends - s, st));
    // two logits a thread
    const int p0 = st * kStretch + 2 * tid;
    const float xa = value(p0), xb = value(p0 + 1);
    const uint64_t a = weight(xa, p0), b = weight(xb, p0 + 1);
    uint64_t incl = scan64(a + b);
    __syncthreads();
    if (tid == 0) sh.index = 0;
    if (lane == 63) sh.low[wave] = incl;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SW; ++i) incl += i < wave ? sh.low[i] : 0;
    // (a chunk's kept weights add up to `have` to the last bit, so one finds itself here)
    if (incl > target && incl - a - b <= target) sh.index = f0 + p0 + (incl - b <= target);
    __syncthreads();
    if (tid == 0) {
      const int token = sh.index;
      A.token[r] = token;
      A.logprob[r] = (float)log(rw.real(row.at(token)) / all);
    }
    return;
  }
}

// One workgroup a row, for vocabularies past kMaxChunks chunks, and operands of less than 16 bytes.
template <class E>
__global__ void __launch_bounds__(ST) sample_whole_kernel(const SampleArgs A) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  SampleLds& sh = *(SampleLds*)smem;
  const int tid = threadIdx.x, V = (int)A.V;
  const int64_t r = blockIdx.x;
  uint32_t top = 0;
  for (int i = tid; i < V; i += ST) top = max(top, logit_key(E::get(((const typename E::raw*)A.logits)[r * A.V + i])));
  top = wave_max(top);
  if ((tid & 63) == 0) sh.high[tid >> 6] = top;
  __syncthreads();
  for (int w = 0; w < SW; ++w) top = max(top, (uint32_t)sh.high[w]);
  if (top == 0) {
    if (tid == 0) A.token[r] = -1, A.logprob[r] = -INFINITY;
    return;
  }
  if (greedy_row(A, r)) {
    const int i = find_index<E>(A, r, 0, V, 0, sh, [&](int, float x) -> uint64_t { return logit_key(x) == top; });
    if (tid == 0) A.token[r] = i, A.logprob[r] = 0.f;
    return;
  }
  sample_row<E>(sample_args(), r, top, sh);
}

// Rows that share the workspace: 32 MB of it.
int64_t rows_at_once(const SampleArgs& a) {
  return a.chunks ? std::max<int64_t>(1, std::min<int64_t>(a.B, (32 << 20) / (a.chunks * 8 * kChunkWords))) : a.B;
}

}  // namespace

void sample_plan(SampleArgs& a, int64_t* ws_bytes) {
  const int64_t vec = 16 / (a.dtype == DT_F32 ? 4 : 2);
  // As few chunks as LDS holds (with room for a row that begins and ends inside 16 bytes). Of few rows, up to 256 smaller ones
  // are no faster: the search is longer by them (one row of 128256 logits, all filters: 22 us in 16 chunks, 25 in 31). A
  // workgroup a row, for vocabularies that need more than 64, takes much longer: that row 773 us, 64 of them 1.1 ms and 33 us.
  const int64_t least = (a.V + 2 * vec + kChunk - 1) / kChunk;
  a.chunks = least > kMaxChunks || a.B * a.V < vec ? 0 : (int32_t)least;
  a.rows = (int32_t)rows_at_once(a);
  *ws_bytes = a.chunks ? a.rows * (int64_t)a.chunks * 8 * kChunkWords : 0;
}

void launch_sample(const SampleArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.V < 1 || a.V > (1 << 24) || a.chunks < 0 || a.chunks > kMaxChunks)
    fail(PJRT_Error_Code_INTERNAL, "sample of a vocabulary the kernels do not take");
  if (a.chunks && !a.ws) fail(PJRT_Error_Code_INTERNAL, "sample without a workspace");
  if (a.B == 0) return record_done(done, stream);
  with_elem(a.dtype, [&](auto e) {
    typedef decltype(e) E;
    // (per device and kernel, so asked for at every launch: it costs no device work)
    const auto kernel = a.chunks ? sample_draw_kernel<E> : sample_whole_kernel<E>;
    const hipError_t s = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, sizeof(SampleLds));
    if (s != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("sample LDS attribute: ") + hipGetErrorString(s));
    const int64_t rows = a.rows;
    for (int64_t r = 0; r < a.B; r += rows) {
      SampleArgs part = a;
      part.row0 = r;
      const int64_t n = std::min(rows, a.B - r);
      if (a.chunks) launch_k(nullptr, sample_chunk_kernel<E>, dim3((unsigned)(n * a.chunks)), dim3(ST), sizeof(ChunkLds), stream, part);
      launch_k(r + rows >= a.B ? done : nullptr, kernel, dim3((unsigned)n), dim3(ST), sizeof(SampleLds), stream, part);
    }
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("sample launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
