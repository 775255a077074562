// ryft.paged_attention: attention of a ragged batch of queries over a paged key / value cache (the definition stands at
// PagedAttnArgs in kernel_abi.h). Scores, softmax statistics and outputs are f32 and rounded once, on store; 16-bit types
// round the probabilities to their type for the product with the values, and sum what they rounded.
//
// Three kernels: few rows a sequence (here: a decoding step), many (k_paged_prompt.hip), and any type and head dim (here).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../common.h"
#include "kernels.h"
#include "launch.h"
#include "paged_attention.h"
#include "paged_prompt.h"

namespace ryft {

namespace {

// Any type and head dim up to 256: a workgroup a query and head.
template <class E>
__global__ void __launch_bounds__(256) paged_attention_any_kernel(const PagedAttnArgs A) {
  __shared__ PagedRowLds sh;
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, D = A.D, tid = threadIdx.x;
  // the last sequence that starts at or before the token
  int lo = 0, hi = A.B;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (paged_start(A, mid) <= t) lo = mid + 1;
    else hi = mid;
  }
  const int b = lo - 1;
  int first = 0, last = 0, pos = 0;  // the keys [first, last)
  if (b >= 0 && t < paged_start(A, b + 1)) {
    const int len = paged_length(A, b);
    pos = len - (paged_start(A, b + 1) - (int)t);
    last = A.causal ? min(len, pos + 1) : len;
    if (A.window > 0) first = (int)max((int64_t)0, (int64_t)pos - A.window + 1);
  }
  float m, l;
  const float x = paged_row<E>(A, b, t, h, pos, first, last, sh, &m, &l);
  if (tid < D) ((typename E::raw*)A.o)[(t * A.Hq + h) * D + tid] = E::put(l == 0.f ? 0.f : x / l);
}

// ------------------------------------------------------------------------------------------------ few rows a sequence
// A decoding step: a tile is the 16 or 32 rows (query, head of a group) of a sequence that share a key head, and the
// work is reading that head's keys and values once. The matrix cores take 16 rows at the cost of one, so what bounds
// it is HBM, as long as enough loads are in flight and the workgroups finish together:
//  - the (tile, 4 blocks of keys) units of the whole batch are one line, cut into equal stretches, one a workgroup (two
//    workgroups on a CU): ragged lengths need no balancing. The batch's lengths are on the device, so every wavefront
//    finds its stretch itself, a sequence a lane. A stretch that covers a tile in part leaves its maximum, sum and
//    output rows in the workspace, and the workgroup that arrives last joins the parts.
//  - each wavefront streams blocks of its own (8 KB of keys, 8 KB of values) from the cache straight into its own part
//    of LDS, and waits for its own loads only: no barriers inside a stretch. While the scores are computed the values
//    are in flight, while the values are weighed the next keys.
// Scores come transposed, S = K · Qᵀ, so that a lane has one row's scores and the probabilities, rounded and packed, are
// the second operand of Oᵀ = Vᵀ · Pᵀ as they are; transposing LDS reads give the first.
constexpr int FEW_WAVES = 4;

// LDS position of 16-byte chunk c of row r: c ^ few_swz(r). Key fragments (16 rows, one chunk) need a bijection of
// r mod 16 onto the banks, value fragments (8 rows, two neighbouring chunks) distinct pairs.
template <int D>
__device__ __forceinline__ int few_swz(int r) {
  if constexpr (D == 128) return ((r & 7) << 1) | ((r >> 3) & 1);
  else return (((r >> 1) & 3) << 1) | ((r >> 3) & 1);
}

template <int D>
struct FewCfg {
  static constexpr int RB = 2 * D;              // bytes a row
  static constexpr int KB = 8192 / RB;          // keys a block: 32 or 64
  static constexpr int KT = KB / 16;            // 16-key tiles of a block
  static constexpr int UNIT = FEW_WAVES * KB;   // keys a unit
  static constexpr int PIECE_ROWS = 1024 / RB;  // rows of a wave-wide load
  static constexpr int WAVE = 16384;            // bytes of LDS a wavefront
  static constexpr int OP = D + 4;              // pitch of staged output rows, floats
};

// All fragments of a 16-key tile: D / 32 reads, waited for in the same statement.
template <int D>
__device__ __forceinline__ void few_read_k(u32x4p (&f)[D / 32], const uint32_t (&a)[D / 32], uint32_t tile) {
  if constexpr (D == 128)
    asm volatile("ds_read_b128 %0, %4\n ds_read_b128 %1, %5\n ds_read_b128 %2, %6\n ds_read_b128 %3, %7\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
                 : "v"(a[0] + tile), "v"(a[1] + tile), "v"(a[2] + tile), "v"(a[3] + tile)
                 : "memory");
  else
    asm volatile("ds_read_b128 %0, %2\n ds_read_b128 %1, %3\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1])
                 : "v"(a[0] + tile), "v"(a[1] + tile)
                 : "memory");
}
// Transposed value fragments of four 16-column tiles for 32 keys: keys 4g .. 4g+3 of the first 16-key tile and of the
// second (16 rows on) in lanes of group g = lane / 16, the order of the scores' registers.
template <int RB>
__device__ __forceinline__ void few_read_v(u32x2p (&f)[8], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n ds_read_b64_tr_b16 %1, %8 offset:%12\n"
      "ds_read_b64_tr_b16 %2, %9\n ds_read_b64_tr_b16 %3, %9 offset:%12\n"
      "ds_read_b64_tr_b16 %4, %10\n ds_read_b64_tr_b16 %5, %10 offset:%12\n"
      "ds_read_b64_tr_b16 %6, %11\n ds_read_b64_tr_b16 %7, %11 offset:%12\n s_waitcnt lgkmcnt(0)"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]), "=&v"(f[7])
      : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "i"(16 * RB)
      : "memory");
}

typedef __attribute__((address_space(3))) void few_lds;
typedef const __attribute__((address_space(1))) void few_glb;

// A value that is the same in all lanes, in scalar registers.
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uni(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)uni((int)(x >> 32)) << 32 | (uint32_t)uni((int)x));
}
__device__ __forceinline__ int64_t lane64(int64_t x, int lane) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
                   (uint32_t)__builtin_amdgcn_readlane((int)x, lane));
}

// What a lane knows of its sequence: how many units its tiles are together.
struct FewSeq {
  int s0, n, len, units, tiles;  // units: of one tile
  __device__ int64_t total() const { return (int64_t)units * tiles; }
};
// (a 64-bit division is some hundred instructions: taken only where it is needed)
__device__ __forceinline__ int64_t few_div(int64_t a, int64_t b) {
  return (a | b) >> 32 ? (int64_t)((uint64_t)a / (uint64_t)b) : (int64_t)((uint32_t)a / (uint32_t)b);
}

template <class X, class E, int D, int NR>
__global__ void __launch_bounds__(256, 2) paged_attention_few_kernel(const PagedAttnArgs A) {
  typedef FewCfg<D> C;
  constexpr int TR = 16 * NR;  // rows of a tile
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float part_ml[FEW_WAVES][TR][2];
  __shared__ uint32_t bad_rows;
  __shared__ int last_word;
  const int tid = threadIdx.x, lane = tid & 63, g16 = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = A.Hq / A.Hkv, W = (int)gridDim.x;
  const PagedScore score(A);

  // rows of no sequence
  for (int64_t t = blockIdx.x; t < A.T; t += W) {
    if (t >= paged_start(A, 0) && t < paged_start(A, A.B)) continue;
    for (int64_t i = tid; i < (int64_t)A.Hq * D; i += 256) ((uint16_t*)A.o)[t * A.Hq * D + i] = 0;
  }

  auto sequence = [&](int b) {
    FewSeq s{0, 0, 0, 0, 0};
    if (b < A.B) {
      s.s0 = paged_start(A, b);
      s.n = max(0, paged_start(A, b + 1) - s.s0);
      s.len = paged_length(A, b);
      if (s.n > 0) {
        const int first = A.window > 0 ? (int)max((int64_t)0, (int64_t)s.len - s.n - A.window + 1) / C::KB * C::KB : 0;
        s.units = max(1, (s.len - first + C::UNIT - 1) / C::UNIT);
        s.tiles = (int)(((uint32_t)s.n * (uint32_t)G + TR - 1) / TR) * A.Hkv;
      }
    }
    return s;
  };
  auto scan = [&](int64_t v) {  // inclusive, over the wavefront
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t o = __shfl_up(v, off, 64);
      if (lane >= off) v += o;
    }
    return v;
  };
  // the whole line's length, then this workgroup's stretch [at, end) of it
  FewSeq seq = sequence(lane);
  int64_t incl = scan(seq.total());
  int64_t all = lane64(incl, 63);
  for (int b0 = 64; b0 < A.B; b0 += 64) all += lane64(scan(sequence(b0 + lane).total()), 63);
  const int64_t per = uni(max(few_div(all + W - 1, W), (int64_t)A.min_units));
  int64_t at = (int64_t)blockIdx.x * per;
  const int64_t end = min(all, at + per);
  int b0 = 0;
  int64_t before = 0;  // units of the sequences before b0
  int64_t tiles_before = 0;
  while (at < end) {
    // the sequence, its tile and the unit within it (the same in every wavefront)
    int64_t here = lane64(incl, 63);
    while (at >= before + here) {
      before += here;
      tiles_before += lane64(scan(seq.tiles), 63);
      b0 += 64;
      seq = sequence(b0 + lane);
      incl = scan(seq.total());
      here = lane64(incl, 63);
    }
    const int64_t tiles_incl = scan(seq.tiles);
    const uint64_t mine = __builtin_amdgcn_ballot_w64(before + incl > at);
    const int who = __builtin_ctzll(mine);
    PagedTile t;
    t.b = b0 + who;
    t.s0 = __builtin_amdgcn_readlane(seq.s0, who);
    t.n = __builtin_amdgcn_readlane(seq.n, who);
    t.len = __builtin_amdgcn_readlane(seq.len, who);
    t.pos0 = t.len - t.n;
    const int units = __builtin_amdgcn_readlane(seq.units, who);
    const int tiles = __builtin_amdgcn_readlane(seq.tiles, who);
    const int64_t r = at - (before + lane64(incl, who) - (int64_t)tiles * units);
    const int tile = uni((int)few_div(r, units)), u0 = (int)(r - (int64_t)tile * units);
    const int64_t tile_index = tiles_before + lane64(tiles_incl, who) - tiles + tile;
    const int64_t tile_at = at - u0;
    const int u1 = (int)min((int64_t)units, u0 + (end - at));
    at += u1 - u0;
    t.hk = uni(tile % A.Hkv);
    t.row0 = uni(tile / A.Hkv) * TR;
    const int rows = (int)min((int64_t)TR, (int64_t)t.n * G - t.row0);
    const int kfirst = A.window > 0 ? (int)max((int64_t)0, (int64_t)t.pos0 - A.window + 1) / C::KB * C::KB : 0;

    // this lane's rows: one a 16-row tile
    int lo[NR], hi[NR], pos[NR];
    float slope[NR];
    u32x4p qf[NR][D / 32];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const int row = 16 * k + l16, flat = t.row0 + row, qi = flat / G, h = t.hk * G + (flat - qi * G);
      const bool live = row < rows;
      pos[k] = t.pos0 + qi;
      hi[k] = live ? (A.causal ? min(t.len - 1, pos[k]) : t.len - 1) : -1;
      lo[k] = A.window > 0 ? (int)max((int64_t)0, (int64_t)pos[k] - A.window + 1) : 0;
      slope[k] = A.slopes && live ? A.slopes[h] * kLog2e : 0.f;
      const uint16_t* const qg = (const uint16_t*)A.q + (int64_t)(t.s0 + qi) * A.qs[0] + h * A.qs[1] + 8 * g16;
#pragma unroll
      for (int s = 0; s < D / 32; ++s) qf[k][s] = live ? *(const u32x4p*)(qg + 32 * s) : u32x4p{0, 0, 0, 0};
    }
    // the keys that every row sees, and those that any does
    const int q_first = uni(t.row0 / G), q_last = uni((t.row0 + rows - 1) / G);
    const int all_hi = A.causal ? min(t.len - 1, t.pos0 + q_first) : t.len - 1;
    const int any_hi = A.causal ? min(t.len - 1, t.pos0 + q_last) : t.len - 1;
    const int all_lo = A.window > 0 ? (int)max((int64_t)0, (int64_t)t.pos0 + q_last - A.window + 1) : 0;

    __builtin_amdgcn_s_waitcnt(0x0F70);  // the queries: waited for inside the loop, the wait would run every iteration

    float m[NR], l[NR];
    f32x4p o[NR][D / 16];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      m[k] = -INFINITY, l[k] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[k][d] = f32x4p{0.f, 0.f, 0.f, 0.f};
    }

    // blocks of this wavefront: first key kfirst + (4 u + wave) · KB
    const int64_t kstart = (int64_t)kfirst + (int64_t)u0 * C::UNIT + wave * C::KB;
    const int64_t klimit = min((int64_t)any_hi + 1, (int64_t)kfirst + (int64_t)u1 * C::UNIT);
    const int blocks = klimit > kstart ? (int)((klimit - kstart + C::UNIT - 1) / C::UNIT) : 0;

    char* const lds = smem + wave * C::WAVE;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(few_lds*)lds;
    // entries [page0, page0 + 64) of the page table, one a lane
    const int32_t* const table = A.table + (int64_t)t.b * A.M;
    int page0 = -64, entry = -1;
    uint64_t bad = 0;             // keys of the block whose page is outside the cache
    uint32_t row[8];              // cache row of each of the lane's eight loads
    const int prow = lane / (C::RB / 16);
    auto locate = [&](int kb) {   // (the lane of key kb + lane)
      const int key = min(kb + (lane & (C::KB - 1)), any_hi);
      const int pi = page_of(A, key);
      const int p_first = __builtin_amdgcn_readlane(pi, 0), p_last = __builtin_amdgcn_readlane(pi, C::KB - 1);
      if (p_last >= page0 + 64) {
        page0 = p_first;
        entry = page0 + lane < A.M ? table[page0 + lane] : -1;
        __builtin_amdgcn_s_waitcnt(0x0F70);  // (waited for at its use, it would be waited for in every iteration)
      }
      const int page = __shfl(entry, pi - page0, 64);
      const bool ok = page >= 0 && page < A.pages;
      bad = __builtin_amdgcn_ballot_w64(!ok);
      const uint32_t cache_row = ok ? ((uint32_t)page * A.Hkv + t.hk) * A.P + (key - pi * A.P) : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) row[i] = __shfl(cache_row, i * C::PIECE_ROWS + prow, 64);
    };
    // Eight wave-wide loads of 1 KB; the lane that fills chunk position c of row r takes chunk c ^ few_swz(r). (r of a
    // load: a multiple of 16 of rows, or 4, 8 or 12 more.)
    auto fetch = [&](const void* cache, int to) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * C::PIECE_ROWS + prow, c = lane % (C::RB / 16) ^ few_swz<D>(r);
        const char* const src = (const char*)cache + (uint64_t)row[i] * C::RB + 16 * c;
        __builtin_amdgcn_global_load_lds((few_glb*)src, (few_lds*)(lds + to + i * 1024), 16, 0, 0);
      }
    };
    uint32_t ka[D / 32];
#pragma unroll
    for (int s = 0; s < D / 32; ++s) ka[s] = lds0 + l16 * C::RB + 16 * ((4 * s + g16) ^ few_swz<D>(l16));
    const int vrow = 4 * g16 + (l16 >> 2), vc = (l16 & 3) >> 1;
    const uint32_t va = lds0 + 8192 + vrow * C::RB + 8 * (l16 & 1);
    const int vsw = few_swz<D>(vrow);

    if (blocks > 0) {
      locate((int)kstart);
      fetch(A.k_cache, 0);
      fetch(A.v_cache, 8192);
    }
    for (int j = 0; j < blocks; ++j) {
      const int kb = (int)kstart + j * C::UNIT;
      const bool more = j + 1 < blocks;
      const uint64_t bad_now = bad;
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8): the keys are there, the values may be on their way
      asm volatile("" ::: "memory");
      f32x4p st[NR][C::KT];
#pragma unroll
      for (int tt = 0; tt < C::KT; ++tt) {
        u32x4p kf[D / 32];
        few_read_k<D>(kf, ka, tt * 16 * C::RB);
#pragma unroll
        for (int k = 0; k < NR; ++k) {
          f32x4p acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < D / 32; ++s) acc = X::mma16(kf[s], qf[k][s], acc);
          st[k][tt] = acc;
        }
      }
      // (from here on `row` and `bad` are the next block's; the values of this one are on their way already)
      if (more) {
        locate(kb + C::UNIT);
        fetch(A.k_cache, 0);
      }
      const bool mask = kb + C::KB - 1 > all_hi || kb < all_lo;
      uint32_t pf[NR][C::KT * 2];
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        if (score.cap2 > 0.f) {
#pragma unroll
          for (int tt = 0; tt < C::KT; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) st[k][tt][i] = score.capped(st[k][tt][i]);
        } else {
#pragma unroll
          for (int tt = 0; tt < C::KT; ++tt) st[k][tt] *= score.sl2;
        }
        if (A.slopes) {
#pragma unroll
          for (int tt = 0; tt < C::KT; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              st[k][tt][i] = __builtin_fmaf(slope[k], (float)(kb + 16 * tt + 4 * g16 + i - pos[k]), st[k][tt][i]);
        }
        if (mask) {
#pragma unroll
          for (int tt = 0; tt < C::KT; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int rel = 16 * tt + 4 * g16 + i, key = kb + rel;
              st[k][tt][i] = key <= hi[k] && key >= lo[k] ? st[k][tt][i] : -INFINITY;
            }
        }
        if (bad_now) {
#pragma unroll
          for (int tt = 0; tt < C::KT; ++tt) {
            const uint32_t bits = (uint32_t)(bad_now >> (16 * tt)) >> (4 * g16);
#pragma unroll
            for (int i = 0; i < 4; ++i) st[k][tt][i] = bits >> i & 1 ? -INFINITY : st[k][tt][i];
          }
        }
        float mb = st[k][0][0];
#pragma unroll
        for (int tt = 0; tt < C::KT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) mb = fmaxf(mb, st[k][tt][i]);
        mb = max_rows16(mb) - X::LIFT;
        if (__builtin_amdgcn_ballot_w64(mb > m[k])) {
          const float mn = fmaxf(m[k], mb);
          const float alpha = m[k] == mn ? 1.f : __builtin_amdgcn_exp2f(m[k] - mn);  // (equal: also -inf, nothing seen)
          m[k] = mn;
          l[k] *= alpha;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) o[k][d] *= alpha;
        }
        const float ref = m[k] == -INFINITY ? 0.f : m[k];
#pragma unroll
        for (int tt = 0; tt < C::KT; ++tt) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(st[k][tt][i] - ref);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w = X::pack(p[2 * i], p[2 * i + 1]);
            l[k] = X::sum2(w, l[k]);
            pf[k][2 * tt + i] = w;
          }
        }
      }
      // the values; of what was issued after them, the eight loads of the next keys may still run
      asm volatile("" ::: "memory");
      if (more) __builtin_amdgcn_s_waitcnt(0x0F78);
      else __builtin_amdgcn_s_waitcnt(0x0F70);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int s = 0; s < C::KT / 2; ++s) {
#pragma unroll
        for (int d4 = 0; d4 < D / 64; ++d4) {
          u32x2p f[8];
          const uint32_t a = va + s * 32 * C::RB;
          few_read_v<C::RB>(f, a + 16 * ((8 * d4 + 0 + vc) ^ vsw), a + 16 * ((8 * d4 + 2 + vc) ^ vsw),
                            a + 16 * ((8 * d4 + 4 + vc) ^ vsw), a + 16 * ((8 * d4 + 6 + vc) ^ vsw));
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const u32x4p vf = {f[2 * d].x, f[2 * d].y, f[2 * d + 1].x, f[2 * d + 1].y};
#pragma unroll
            for (int k = 0; k < NR; ++k)
              o[k][4 * d4 + d] = X::mma16(vf, u32x4p{pf[k][4 * s], pf[k][4 * s + 1], pf[k][4 * s + 2], pf[k][4 * s + 3]}, o[k][4 * d4 + d]);
          }
        }
      }
      if (more) fetch(A.v_cache, 8192);
    }

    // join the wavefronts, 16 rows at a time: staged outputs [wave][16][OP], then the joined rows [16][OP] in place of the
    // first wavefront's
    const bool whole = u0 == 0 && u1 == units;
    const __amdgpu_buffer_rsrc_t ws = paged_ws(A);
    const uint32_t slot = 2 * blockIdx.x + (u0 == 0 ? 1 : 0);
    const uint32_t slot_byte = slot * (uint32_t)paged_part_floats(TR, D) * 4;
    float* const so = (float*)smem;
#pragma unroll
    for (int k = 0; k < NR; ++k) l[k] = sum_rows16(l[k]);
    __syncthreads();
    if (tid == 0) bad_rows = 0;
#pragma unroll
    for (int k = 0; k < NR; ++k)
      if (g16 == 0) part_ml[wave][16 * k + l16][0] = m[k], part_ml[wave][16 * k + l16][1] = l[k];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      if (16 * k >= rows) break;
      float* const mine_o = so + (wave * 16 + l16) * C::OP + 4 * g16;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) *(f32x4p*)(mine_o + 16 * d) = o[k][d];
      __syncthreads();
      f32x4p x[D / 64];
      float mt[D / 64], lt[D / 64];
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int idx = tid + 256 * i, r = idx / (D / 4), d = 4 * (idx % (D / 4));
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) mm = fmaxf(mm, part_ml[w][16 * k + r][0]);
        const float ref = mm == -INFINITY ? 0.f : mm;
        f32x4p v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) {
          const float f = __builtin_amdgcn_exp2f(part_ml[w][16 * k + r][0] - ref);
          ll = __builtin_fmaf(part_ml[w][16 * k + r][1], f, ll);
          const f32x4p y = *(const f32x4p*)(so + (w * 16 + r) * C::OP + d);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(y[e], f, v[e]);
        }
        x[i] = v, mt[i] = mm, lt[i] = ll;
        const bool finite = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))) < INFINITY &&
                            !(v.x != v.x) && !(v.y != v.y) && !(v.z != v.z) && !(v.w != v.w);
        if (!finite && 16 * k + r < rows) atomicOr(&bad_rows, 1u << r);
      }
      __syncthreads();
      // A value that a row does not see has probability 0, which an infinity or NaN in it would still turn into NaN:
      // rows with such outputs are computed again from what they see alone.
      uint32_t again = bad_rows;
      while (again) {
        const int r = __builtin_ctz(again);
        again &= again - 1;
        const int flat = t.row0 + 16 * k + r, qi = flat / G, p = t.pos0 + qi;
        const int64_t first = max((int64_t)kfirst + (int64_t)u0 * C::UNIT, A.window > 0 ? (int64_t)p - A.window + 1 : 0);
        const int64_t last = min((int64_t)kfirst + (int64_t)u1 * C::UNIT, (int64_t)(A.causal ? min(t.len, p + 1) : t.len));
        float rm, rl;
        const float v = paged_row<E>(A, t.b, t.s0 + qi, t.hk * G + (flat - qi * G), p, (int)max(first, (int64_t)0), (int)max(last, (int64_t)0),
                                     *(PagedRowLds*)smem, &rm, &rl);
        __syncthreads();
        if (tid < D) so[tid] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const int idx = tid + 256 * i, d = 4 * (idx % (D / 4));
          if (idx / (D / 4) == r) x[i] = *(const f32x4p*)(so + d), mt[i] = rm, lt[i] = rl;
        }
        __syncthreads();
        if (tid == 0) bad_rows = 0;
      }
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int idx = tid + 256 * i, r = 16 * k + idx / (D / 4), d = 4 * (idx % (D / 4));
        if (r < rows) {
          if (whole) {
            paged_store4<X, D>(A, t, r, d, x[i] * (lt[i] == 0.f ? 0.f : 1.f / lt[i]));
          } else {
            agent_put4(ws, slot_byte + (r * D + d) * 4, x[i]);
            if (d == 0) agent_put2(ws, slot_byte + (TR * D + 2 * r) * 4, mt[i], lt[i]);
          }
        }
      }
      __syncthreads();
    }
    if (!whole && tile_index < A.max_tiles) {
      // the workgroups of this tile's parts: the first has it from its beginning, the others in their first slot
      const int w0 = uni((int)few_div(tile_at, per)), w1 = uni((int)few_div(tile_at + units - 1, per)), parts = w1 - w0 + 1;
      if (paged_arrive(A.counters + tile_index, parts, &last_word))
        paged_join<X, D, TR>(A, t, rows, parts, [&](int i) { return 2 * (w0 + i) + (i == 0 ? 1 : 0); }, so);
      __syncthreads();
    }
  }
}

template <class X, class E, int D, int NR>
void launch_few(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done) {
  constexpr int lds = FEW_WAVES * FewCfg<D>::WAVE;
  launch_k(done, paged_attention_few_kernel<X, E, D, NR>, dim3((unsigned)a.groups), dim3(256), lds, stream, a);
}

template <class X, class E>
void launch_matrix(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.tile_rows == kPromptRows) return launch_paged_prompt(a, stream, done);
  if (a.D == 128) a.tile_rows == 16 ? launch_few<X, E, 128, 1>(a, stream, done) : launch_few<X, E, 128, 2>(a, stream, done);
  else a.tile_rows == 16 ? launch_few<X, E, 64, 1>(a, stream, done) : launch_few<X, E, 64, 2>(a, stream, done);
}

}  // namespace

void paged_attention_plan(PagedAttnArgs& a, int64_t* ws_floats, int64_t* counters) {
  *ws_floats = *counters = 0;
  a.tile_rows = 0;
  // key / P = key · page_mul >> page_shift for key < 2^31 (page_mul = ⌈2^(31 + s) / P⌉, s = ⌈log2 P⌉)
  int s = 0;
  while (((int64_t)1 << s) < a.P) ++s;
  a.page_shift = 31 + s;
  a.page_mul = (((uint64_t)1 << a.page_shift) + a.P - 1) / a.P;
  if ((a.dtype != DT_BF16 && a.dtype != DT_F16) || (a.D != 64 && a.D != 128) || a.T == 0 || a.B == 0) return;
  // (rows of the cache are numbered in 32 bits, and the queries' rows read 16 bytes at a time)
  if (a.pages * a.Hkv * a.P > (int64_t)UINT32_MAX || (a.qs[0] | a.qs[1]) & 7) return;
  const int G = a.Hq / a.Hkv;
  const double rows = (double)a.T * G / a.B;  // rows a sequence has of a key head, on average
  if (rows > 32) return paged_prompt_plan(a, ws_floats, counters);
  a.tile_rows = rows > 16 ? 32 : 16;
  const int unit = a.D == 128 ? 128 : 256;
  a.min_units = 512 / unit;
  const int64_t tiles = (a.T * G / a.tile_rows + a.B) * a.Hkv;
  if (a.T * a.Hq > INT32_MAX || tiles > INT32_MAX) { a.tile_rows = 0; return; }
  a.max_tiles = (int32_t)tiles;
  // two workgroups a CU, fewer if even the longest sequences have no work for them
  const int64_t most = tiles * (((int64_t)a.M * a.P + 511) / 512 + 1);
  a.groups = (int32_t)std::max<int64_t>(1, std::min<int64_t>(512, most));
  *ws_floats = 2 * a.groups * paged_part_floats(a.tile_rows, a.D);
  *counters = a.max_tiles;
}

void launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.D < 1 || a.D > 256 || a.Hkv < 1 || a.Hq < 1 || a.Hq > 65535 || a.Hq % a.Hkv || a.P < 1)
    fail(PJRT_Error_Code_INTERNAL, "paged_attention of a shape the kernels do not take");
  if (a.T == 0) return record_done(done, stream);
  if (a.tile_rows) {
    if (a.groups < 1 || (a.tile_rows != kPromptRows && (!a.ws || !a.counters))) fail(PJRT_Error_Code_INTERNAL, "paged_attention without a workspace");
    if (a.dtype == DT_BF16) launch_matrix<MmaBF16, ElemBF16>(a, stream, done);
    else launch_matrix<MmaF16, ElemF16>(a, stream, done);
  } else {
    with_elem(a.dtype, [&](auto e) {
      launch_k(done, paged_attention_any_kernel<decltype(e)>, dim3((unsigned)a.T, (unsigned)a.Hq), dim3(256), 0, stream, a);
    });
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("paged_attention launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
