// ryft.paged_attention: attention of a ragged batch of queries over a paged key / value cache (the definition stands at
// PagedAttnArgs in kernel_abi.h). Scores, softmax statistics and outputs are f32 and rounded once, on store; probabilities
// go to the matrix cores as two terms of a 16-bit type (paged_attention.h).
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
// A decoding step: a tile is up to 16 rows (query, head of a group) of a sequence that share a key head, and the
// work is reading that head's keys and values once. The matrix cores take 16 rows at the cost of one, so what bounds
// it is HBM, as long as enough loads are in flight and the workgroups finish together:
//  - the (tile, 4 blocks of keys) units of the whole batch are one line, cut into equal stretches, one a workgroup (two
//    workgroups on a CU): ragged lengths need no balancing. The batch's lengths are on the device, so every wavefront
//    finds its stretch itself, a sequence a lane. A stretch that covers a tile in part leaves its maximum, sum and
//    output rows in the workspace, and the workgroup that arrives last joins the parts.
//  - each wavefront streams blocks of its own (8 KB of keys, 8 KB of values) from the cache straight into its own part
//    of LDS, and waits for its own loads only: no barriers inside a stretch. While the scores are computed the values
//    are in flight, while the values are weighed the next keys.
// Scores come transposed, S = K · Qᵀ, so that a lane has one row's scores and the probabilities, packed, are
// the second operand of Oᵀ = Vᵀ · Pᵀ as they are; transposing LDS reads give the first. Measured: 64 sequences of 8 to 4096
// keys, 32 heads on 8 of 128: 111 us (4.7 TB/s; all of 4096: 6.0); 8 x 2 queries over 20000 keys of 8 heads of 64: 68 us
// (4.8 TB/s); one query of 8 heads over 500 keys: 9 us, as any launch from the host.
constexpr int FEW_WAVES = 4;
constexpr int TR = 16;  // rows of a tile

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
  static constexpr int STAGE_ROWS = 7 * 128 / D;  // rows of all wavefronts that fit beside the blocks, with two workgroups a CU
  static constexpr int LDS = FEW_WAVES * (WAVE + STAGE_ROWS * OP * 4);
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

// A barrier that waits for this wavefront's LDS accesses and no others: __syncthreads would wait for the blocks on their way.
__device__ __forceinline__ void few_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// LDS accesses while blocks are on their way: the compiler, which cannot tell their places apart, would wait for the blocks
// before each of its own. Reads are waited for in their statement, writes by few_barrier.
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ void lds_put4(uint32_t a, f32x4p v) { asm volatile("ds_write_b128 %0, %1" ::"v"(a), "v"(v) : "memory"); }
__device__ __forceinline__ void lds_put2(uint32_t a, float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  asm volatile("ds_write_b64 %0, %1" ::"v"(a), "v"(f2{x, y}) : "memory");
}
__device__ __forceinline__ void lds_put1(uint32_t a, uint32_t v) { asm volatile("ds_write_b32 %0, %1" ::"v"(a), "v"(v) : "memory"); }
__device__ __forceinline__ uint32_t lds_get1(uint32_t a) {
  uint32_t v;
  asm volatile("ds_read_b32 %0, %1\n s_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(a) : "memory");
  return v;
}
// (maximum, sum) and four elements of a row from each of the four wavefronts, `ml` and `o` bytes apart
__device__ __forceinline__ void lds_get_parts(f32x4p (&v)[4], f32x2p (&w)[4], uint32_t a, uint32_t o, uint32_t b, uint32_t ml) {
  asm volatile(
      "ds_read_b64 %4, %12\n ds_read_b64 %5, %13\n ds_read_b64 %6, %14\n ds_read_b64 %7, %15\n"
      "ds_read_b128 %0, %8\n ds_read_b128 %1, %9\n ds_read_b128 %2, %10\n ds_read_b128 %3, %11\n s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3])
      : "v"(a), "v"(a + o), "v"(a + 2 * o), "v"(a + 3 * o), "v"(b), "v"(b + ml), "v"(b + 2 * ml), "v"(b + 3 * ml)
      : "memory");
}

typedef __attribute__((address_space(3))) void few_lds;
typedef const __attribute__((address_space(1))) void few_glb;

// A value that is the same in all lanes, in a scalar register.
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What a lane knows of its sequence: its tiles, and the units of each.
struct FewSeq {
  int s0, n, len, units, tiles;
};
// A stretch's part of a tile: the units [u0, u1) of it.
struct FewRange {
  PagedTile t;
  int rows, kfirst;       // its rows, the key that its units count from
  int units, u0, u1;
  int at, index;          // its first unit on the line, its number
};
// A part that waits to be joined: the rows' place, the workgroups [w0, w0 + parts) that have the others, its counter.
struct FewPart {
  PagedTile t;
  int rows, w0, parts, index;
};

template <class X, class E, int D>
__global__ void __launch_bounds__(256, 2) paged_attention_few_kernel(const PagedAttnArgs A) {
  typedef FewCfg<D> C;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float part_ml[FEW_WAVES][TR][2];
  __shared__ uint32_t bad_rows;
  __shared__ int last_word;
  const int tid = threadIdx.x, lane = tid & 63, g16 = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = A.Hq / A.Hkv, W = (int)gridDim.x;
  const PagedScore score(A);

  bool falls = false;  // of the lane's sequences, one ends before it begins
  auto sequence = [&](int b) {
    FewSeq s{0, 0, 0, 0, 0};
    if (b < A.B) {
      s.s0 = paged_start(A, b);
      s.n = paged_start(A, b + 1) - s.s0;
      falls |= s.n < 0;
      s.len = paged_length(A, b);
      if (s.n > 0) {
        const int first = A.window > 0 ? (int)max((int64_t)0, (int64_t)s.len - s.n - A.window + 1) / C::KB * C::KB : 0;
        s.units = max(1, (s.len - first + C::UNIT - 1) / C::UNIT);
        s.tiles = (int)(((uint32_t)s.n * (uint32_t)G + TR - 1) / TR) * A.Hkv;
      }
    }
    return s;
  };
  auto scan = [&](int v) {  // inclusive, over the wavefront
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(v, off, 64);
      if (lane >= off) v += o;
    }
    return v;
  };
  auto last_lane = [&](int v) { return __builtin_amdgcn_readlane(v, 63); };
  // The whole line's length (paged_attention_plan keeps it below 2^30); workgroup w has [w q + min(w, r), ...) of it, a
  // unit more where w < r.
  FewSeq seq = sequence(lane);
  int incl = scan(seq.units * seq.tiles), tiles_incl = scan(seq.tiles);
  int all = last_lane(incl);
  for (int b = 64; b < A.B; b += 64) {
    const FewSeq s = sequence(b + lane);
    all += last_lane(scan(s.units * s.tiles));
  }
  // Rows of no sequence; all of them where starts decrease. Those may name more tiles than there are counters for, and a line
  // longer than 32 bits count, whose parts would wait for workgroups that never come and leave their counters behind for
  // the next launch.
  const bool none = __builtin_amdgcn_ballot_w64(falls) != 0;
  for (int64_t t = blockIdx.x; t < A.T; t += W) {
    if (!none && t >= paged_start(A, 0) && t < paged_start(A, A.B)) continue;
    for (int64_t i = tid; i < (int64_t)A.Hq * D; i += 256) ((uint16_t*)A.o)[t * A.Hq * D + i] = 0;
  }
  if (none) return;
  // (down to a unit a stretch: with 4 as the least, 16 queries over 5624 keys took 27 us, 17 so, and 35 sequences of up to 18
  // keys 22 and 9)
  const int working = uni(max(1, min(W, all)));
  const int q_units = uni(all / working), r_units = all - q_units * working;
  const int w = blockIdx.x;
  if (w >= working) return;
  auto owner = [&](int unit) {
    const int wide = r_units * (q_units + 1);
    return uni(unit < wide ? unit / (q_units + 1) : r_units + (unit - wide) / q_units);
  };
  int at = w * q_units + min(w, r_units);
  const int end = at + q_units + (w < r_units ? 1 : 0);
  if (at >= end) return;
  int b0 = 0, before = 0, tiles_before = 0;  // units and tiles of the sequences before b0
  auto next_range = [&]() {  // (the same in every wavefront; `at` lies on the line)
    FewRange R;
    int here = last_lane(incl);
    while (at >= before + here) {
      before += here;
      tiles_before += last_lane(tiles_incl);
      b0 += 64;
      seq = sequence(b0 + lane);
      incl = scan(seq.units * seq.tiles), tiles_incl = scan(seq.tiles);
      here = last_lane(incl);
    }
    PagedTile& t = R.t;
    const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + incl > at));
    t.b = b0 + who;
    t.s0 = __builtin_amdgcn_readlane(seq.s0, who);
    t.n = __builtin_amdgcn_readlane(seq.n, who);
    t.len = __builtin_amdgcn_readlane(seq.len, who);
    t.pos0 = t.len - t.n;
    R.units = __builtin_amdgcn_readlane(seq.units, who);
    const int tiles = __builtin_amdgcn_readlane(seq.tiles, who);
    const int r = at - (before + __builtin_amdgcn_readlane(incl, who) - tiles * R.units), tile = uni(r / R.units);
    R.index = tiles_before + __builtin_amdgcn_readlane(tiles_incl, who) - tiles + tile;
    R.u0 = r - tile * R.units;
    R.u1 = min(R.units, R.u0 + (end - at));
    R.at = at - R.u0;
    at += R.u1 - R.u0;
    const int group = uni(tile / A.Hkv);
    t.hk = tile - group * A.Hkv;
    t.row0 = group * TR;
    R.rows = min(TR, t.n * G - t.row0);
    R.kfirst = A.window > 0 ? (int)max((int64_t)0, (int64_t)t.pos0 - A.window + 1) / C::KB * C::KB : 0;
    return R;
  };
  auto last_key = [&](const PagedTile& t, int q) { return A.causal ? min(t.len - 1, t.pos0 + q) : t.len - 1; };
  auto first_key = [&](const PagedTile& t, int q) { return A.window > 0 ? (int)max((int64_t)0, (int64_t)t.pos0 + q - A.window + 1) : 0; };

  // this wavefront's blocks of a range, first key kfirst + (4 u + wave) · KB, and what it needs to load them
  char* const lds = smem + wave * C::WAVE;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(few_lds*)lds;
  const int prow = lane / (C::RB / 16);
  int kstart = 0, blocks = 0, any_hi = 0, hk = 0;
  const int32_t* table = nullptr;
  int page0 = -64, entry = -1;  // entries [page0, page0 + 64) of the page table, one a lane
  uint64_t bad = 0;             // keys of the block whose page is outside the cache
  uint32_t row[8];              // cache row of each of the lane's eight loads
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
    const uint32_t cache_row = ok ? ((uint32_t)page * A.Hkv + hk) * A.P + (key - pi * A.P) : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) row[i] = __shfl(cache_row, i * C::PIECE_ROWS + prow, 64);
  };
  // Eight wave-wide loads of 1 KB; the lane that fills chunk position c of row r takes chunk c ^ few_swz(r).
  auto fetch = [&](const void* cache, int to) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * C::PIECE_ROWS + prow, c = lane % (C::RB / 16) ^ few_swz<D>(r);
      const char* const src = (const char*)cache + (uint64_t)row[i] * C::RB + 16 * c;
      __builtin_amdgcn_global_load_lds((few_glb*)src, (few_lds*)(lds + to + i * 1024), 16, 0, 0);
    }
  };
  // A range's queries, then its first block on its way: everything that was loaded before has arrived when it returns.
  auto begin = [&](const FewRange& R, u32x4p (&qn)[D / 32]) {
    const int flat = R.t.row0 + l16, qi = flat / G, h = R.t.hk * G + (flat - qi * G);
    const uint16_t* const qg = (const uint16_t*)A.q + (int64_t)(R.t.s0 + qi) * A.qs[0] + h * A.qs[1] + 8 * g16;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) qn[s] = l16 < R.rows ? *(const u32x4p*)(qg + 32 * s) : u32x4p{0, 0, 0, 0};
    hk = R.t.hk;
    table = A.table + (int64_t)R.t.b * A.M;
    page0 = -64;
    any_hi = last_key(R.t, uni((R.t.row0 + R.rows - 1) / G));
    const int64_t first = (int64_t)R.kfirst + (int64_t)R.u0 * C::UNIT + wave * C::KB;
    const int64_t limit = min((int64_t)any_hi + 1, (int64_t)R.kfirst + (int64_t)R.u1 * C::UNIT);
    blocks = limit > first ? (int)((limit - first + C::UNIT - 1) / C::UNIT) : 0;
    kstart = (int)first;
    if (blocks > 0) locate(kstart);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    // (the queries pass through a statement, or they would be waited for at their use, in every iteration)
#pragma unroll
    for (int s = 0; s < D / 32; ++s) asm volatile("" : "+v"(qn[s]));
    if (blocks > 0) {
      fetch(A.k_cache, 0);
      fetch(A.v_cache, 8192);
    }
  };
  uint32_t ka[D / 32];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) ka[s] = lds0 + l16 * C::RB + 16 * ((4 * s + g16) ^ few_swz<D>(l16));
  const int vrow = 4 * g16 + (l16 >> 2), vc = (l16 & 3) >> 1;
  const uint32_t va = lds0 + 8192 + vrow * C::RB + 8 * (l16 & 1);
  const int vsw = few_swz<D>(vrow);

  FewPart part[2];
  int parts = 0;
  u32x4p qf[D / 32];
  FewRange R = next_range();
  begin(R, qf);
  while (true) {
    const PagedTile t = R.t;
    const int rows = R.rows;
    // this lane's row
    const int flat = t.row0 + l16, qi = flat / G, pos = t.pos0 + qi;
    const int hi = l16 < rows ? last_key(t, qi) : -1, lo = first_key(t, qi);
    float slope = 0.f;
    if (A.slopes) {
      slope = A.slopes[l16 < rows ? t.hk * G + (flat - qi * G) : 0] * kLog2e;
      __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    // the keys that every row sees
    const int all_hi = last_key(t, uni(t.row0 / G)), all_lo = first_key(t, uni((t.row0 + rows - 1) / G));

    float m = -INFINITY, l = 0.f;
    f32x4p o[D / 16];
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = f32x4p{0.f, 0.f, 0.f, 0.f};

    for (int j = 0; j < blocks; ++j) {
      const int kb = kstart + j * C::UNIT;
      const bool more = j + 1 < blocks;
      const uint64_t bad_now = bad;
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8): the keys are there, the values may be on their way
      asm volatile("" ::: "memory");
      f32x4p st[C::KT];
#pragma unroll
      for (int tt = 0; tt < C::KT; ++tt) {
        u32x4p kf[D / 32];
        few_read_k<D>(kf, ka, tt * 16 * C::RB);
        f32x4p acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < D / 32; ++s) acc = X::mma16(kf[s], qf[s], acc);
        st[tt] = acc;
      }
      // (from here on `row` and `bad` are the next block's; the values of this one are on their way already)
      if (more) {
        locate(kb + C::UNIT);
        fetch(A.k_cache, 0);
      }
      const bool mask = kb + C::KB - 1 > all_hi || kb < all_lo;
      uint32_t pf[C::KT * 2], pr[C::KT * 2];  // probabilities: rounded, and what that leaves of them
      if (score.cap2 > 0.f) {
        auto at = [&](int i) -> float& { return ((float*)st)[i]; };
        score.cap<C::KT * 4>(at, [](int) { return 0.f; });
      } else {
#pragma unroll
        for (int tt = 0; tt < C::KT; ++tt) st[tt] *= score.sl2;
      }
      if (A.slopes) {
#pragma unroll
        for (int tt = 0; tt < C::KT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st[tt][i] = __builtin_fmaf(slope, (float)(kb + 16 * tt + 4 * g16 + i - pos), st[tt][i]);
      }
      if (mask) {
#pragma unroll
        for (int tt = 0; tt < C::KT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rel = 16 * tt + 4 * g16 + i, key = kb + rel;
            st[tt][i] = key <= hi && key >= lo ? st[tt][i] : -INFINITY;
          }
      }
      if (bad_now) {
#pragma unroll
        for (int tt = 0; tt < C::KT; ++tt) {
          const uint32_t bits = (uint32_t)(bad_now >> (16 * tt)) >> (4 * g16);
#pragma unroll
          for (int i = 0; i < 4; ++i) st[tt][i] = bits >> i & 1 ? -INFINITY : st[tt][i];
        }
      }
      float mb = st[0][0];
#pragma unroll
      for (int tt = 0; tt < C::KT; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mb = fmaxf(mb, st[tt][i]);
      mb = max_rows16(mb) - X::LIFT;
      if (__builtin_amdgcn_ballot_w64(mb > m)) {
        const float mn = fmaxf(m, mb);
        const float alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);  // (equal: also -inf, nothing seen)
        m = mn;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[d] *= alpha;
      }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int tt = 0; tt < C::KT; ++tt) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(st[tt][i] - ref);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l += p[2 * i] + p[2 * i + 1];
          pf[2 * tt + i] = X::pack(p[2 * i], p[2 * i + 1]);
          pr[2 * tt + i] = X::rest(pf[2 * tt + i], p[2 * i], p[2 * i + 1]);
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
            o[4 * d4 + d] = X::mma16(vf, u32x4p{pf[4 * s], pf[4 * s + 1], pf[4 * s + 2], pf[4 * s + 3]}, o[4 * d4 + d]);
            o[4 * d4 + d] = X::mma16(vf, u32x4p{pr[4 * s], pr[4 * s + 1], pr[4 * s + 2], pr[4 * s + 3]}, o[4 * d4 + d]);
          }
        }
      }
      if (more) fetch(A.v_cache, 8192);
    }

    // The next range's first block is on its way before the wavefronts join this one's rows, where the rows fit beside the
    // ring: waiting for each other, for the workspace and for that block one after the other took as long as two blocks.
    const bool early = rows <= C::STAGE_ROWS;
    const bool more_ranges = at < end;
    const FewRange cur = R;
    u32x4p qn[D / 32];
    if (more_ranges) R = next_range();
    if (early && more_ranges) begin(R, qn);
    // staged outputs [wave][rows][OP], summed by all threads
    const bool whole = cur.u0 == 0 && cur.u1 == cur.units;
    const __amdgpu_buffer_rsrc_t ws = paged_ws(A);
    const uint32_t slot_byte = (2 * (uint32_t)w + (cur.u0 == 0 ? 1 : 0)) * (uint32_t)paged_part_floats(TR, D) * 4;
    float* const so = (float*)(early ? smem + FEW_WAVES * C::WAVE : smem);
    l = sum_rows16(l);
    few_barrier();
    if (tid == 0) lds_put1(lds_at(&bad_rows), 0);
    if (g16 == 0) lds_put2(lds_at(part_ml[wave][l16]), m, l);
    if (l16 < rows) {
      const uint32_t mine_o = lds_at(so + (wave * rows + l16) * C::OP + 4 * g16);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) lds_put4(mine_o + 64 * d, o[d]);
    }
    few_barrier();
    f32x4p x[D / 64];
    float mt[D / 64], lt[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int idx = tid + 256 * i, r = idx / (D / 4), d = 4 * (idx % (D / 4));
      float mm = -INFINITY, ll = 0.f;
      f32x4p v = {0.f, 0.f, 0.f, 0.f};
      if (r < rows) {
        f32x4p y[4];
        f32x2p ml[4];
        lds_get_parts(y, ml, lds_at(so + r * C::OP + d), rows * C::OP * 4, lds_at(part_ml[0][r]), sizeof(part_ml[0]));
#pragma unroll
        for (int u = 0; u < FEW_WAVES; ++u) mm = fmaxf(mm, ml[u].x);
        const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int u = 0; u < FEW_WAVES; ++u) {
          const float f = __builtin_amdgcn_exp2f(ml[u].x - ref);
          ll = __builtin_fmaf(ml[u].y, f, ll);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(y[u][e], f, v[e]);
        }
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) finite &= fabsf(v[e]) < INFINITY;
        if (!finite) asm volatile("ds_or_b32 %0, %1" ::"v"(lds_at(&bad_rows)), "v"(1u << r) : "memory");
      }
      x[i] = v, mt[i] = mm, lt[i] = ll;
    }
    few_barrier();
    // A value that a row does not see has probability 0, which an infinity or NaN in it would still turn into NaN:
    // rows with such outputs are computed again from what they see alone.
    uint32_t again = uni((int)lds_get1(lds_at(&bad_rows)));
    while (again) {
      const int r = __builtin_ctz(again);
      again &= again - 1;
      const int flat = t.row0 + r, qi = flat / G;
      const int64_t first = max((int64_t)cur.kfirst + (int64_t)cur.u0 * C::UNIT, (int64_t)first_key(t, qi));
      const int64_t last = min((int64_t)cur.kfirst + (int64_t)cur.u1 * C::UNIT, (int64_t)last_key(t, qi) + 1);
      float rm, rl;
      const float v = paged_row<E>(A, t.b, t.s0 + qi, t.hk * G + (flat - qi * G), t.pos0 + qi, (int)first, (int)max(last, (int64_t)0),
                                   *(PagedRowLds*)so, &rm, &rl);
      float* const one = so + sizeof(PagedRowLds) / 4;
      if (tid < D) one[tid] = v;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int idx = tid + 256 * i, d = 4 * (idx % (D / 4));
        if (idx / (D / 4) == r) x[i] = *(const f32x4p*)(one + d), mt[i] = rm, lt[i] = rl;
      }
      __syncthreads();
      if (tid == 0) lds_put1(lds_at(&bad_rows), 0);
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int idx = tid + 256 * i, r = idx / (D / 4), d = 4 * (idx % (D / 4));
      if (r < rows) {
        if (whole) {
          paged_store4<X, D>(A, t, r, d, x[i] * (lt[i] == 0.f ? 0.f : 1.f / lt[i]));
        } else {
          agent_put4(ws, slot_byte + (r * D + d) * 4, x[i]);
          if (d == 0) agent_put2(ws, slot_byte + (TR * D + 2 * r) * 4, mt[i], lt[i]);
        }
      }
    }
    few_barrier();
    if (!whole) {
      // (its first range and its last: no workgroup has more parts than two)
      const int w0 = owner(cur.at), w1 = owner(cur.at + cur.units - 1);
      const FewPart P{t, rows, w0, w1 - w0 + 1, cur.index};
      if (parts == 0) part[0] = P;
      else part[1] = P;
      ++parts;
    }
    if (!more_ranges) break;
    if (early) {
#pragma unroll
      for (int s = 0; s < D / 32; ++s) qf[s] = qn[s];
    } else {
      begin(R, qf);
    }
  }
  // The workgroup of a tile that arrives last joins its parts: the first workgroup has it from its beginning, the others in
  // their first slot.
  for (int p = 0; p < parts; ++p) {
    const FewPart P = p == 0 ? part[0] : part[1];
    if (paged_arrive(A.counters + P.index, P.parts, &last_word))
      paged_join<X, D, TR>(A, P.t, P.rows, P.parts, [&](int i) { return 2 * (P.w0 + i) + (i == 0 ? 1 : 0); }, (float*)smem);
    __syncthreads();
  }
}

template <class X, class E, int D>
void launch_few(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done) {
  constexpr int lds = FewCfg<D>::LDS;
  const hipError_t e = hipFuncSetAttribute((const void*)paged_attention_few_kernel<X, E, D>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("paged_attention LDS attribute: ") + hipGetErrorString(e));
  launch_k(done, paged_attention_few_kernel<X, E, D>, dim3((unsigned)a.groups), dim3(256), lds, stream, a);
}

template <class X, class E>
void launch_matrix(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.tile_rows == kPromptRows) return launch_paged_prompt(a, stream, done);
  if (a.D == 128) return launch_few<X, E, 128>(a, stream, done);
  launch_few<X, E, 64>(a, stream, done);
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
  // The other kernel takes tiles of up to 128 rows, and its parts are joined by a second launch of the whole chip, here a
  // tile's by one workgroup. Heads of 128 over 4 x 4 queries of 8 sequences of 16000 keys: 104 us there, 132 here in tiles
  // of 32 rows; 3 x 5 queries of 5 heads of 64 over 12811 keys 25 and 38. With 16 rows or fewer it is the parts of a tile
  // that decide, many where tiles are few and long. How long is on the device; the table's room is what is known here. With
  // the lengths that the room is for: 1 tile of 30000 keys 20 us there and 55 here, 2 tiles 20 and 37, 4 tiles of 100001
  // keys 51 and 56, 8 of 30000 18 and 22, but 1 of 9000 14 and 12, and 16 of 9000 17 and 19, 32 of 9000 39 and 41. In a
  // table for 32768 keys, one sequence of 8 tiles: 12 and 9 us for 100 keys, 14 and 11 for 2000, 16 and 14 for 4000, 20 and
  // 24 for 8000, 23 and 37 for 16000, 36 and 34 for 32768; four sequences 15 and 11 for 500, 24 and 19 for 4000, 58 and 58
  // for 16000, 104 and 98 for 32768. So 8 tiles at most, which lose 3 us where they are short.
  const int64_t tiles128 = (a.T * G / kPromptRows + a.B) * a.Hkv, keys = (int64_t)a.M * a.P;
  if (rows > 16 || (tiles128 <= 8 && keys >= 16384)) return paged_prompt_plan(a, ws_floats);
  a.tile_rows = TR;
  const int unit = a.D == 128 ? 128 : 256;
  const int64_t tiles = (a.T * G / a.tile_rows + a.B) * a.Hkv;
  // (units are counted in 32 bits)
  if (a.T * a.Hq > INT32_MAX || tiles > (1 << 30) / ((int64_t)a.M * a.P / unit + 1)) { a.tile_rows = 0; return; }
  a.max_tiles = (int32_t)tiles;
  // two workgroups a CU, fewer if even the longest sequences have no work for them
  const int64_t most = tiles * (((int64_t)a.M * a.P + unit - 1) / unit + 1);
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
