// ryft.paged_attention with many rows a sequence (prompts, chunks of prompts, wide groups), bf16 and f16, head dim 64 or
// 128: a tile is 128 rows (query, head of a group) of a sequence that share a key head, 32 a wavefront; blocks of 64 keys
// and values stream through LDS, two stages, loaded straight from the rows of the cache that the page table names.
//
// Where the tiles do not fill the chip, each is cut into ranges of keys, which a second launch joins.
//
// Scores come transposed, S = K · Qᵀ, so that a lane has one row and half its keys: the running maximum and sum take one
// exchange between the half-waves, and the probabilities, packed, are the second operand of Oᵀ = Vᵀ · Pᵀ as they are.
// The matrix products and the exponentials bound it (a wavefront's float instructions and matrix instructions add up):
// the exponent reference moves only when a block exceeds it by 2^8, and masks are applied only in the blocks that need
// one. Two or three workgroups share a CU, so that one's waits for LDS are the others' work. Measured, heads of 128 and 64: four
// prompts of 875 to 1824 tokens, 32 heads, capped, 129 us (490 TFLOP/s, counting a product with the values once), uncapped 117;
// two chunks of 512 with a window of 4096, 39 us; 256 x 4 queries of two sequences of 60000 keys 106 us (590 TFLOP/s); 4 x 5
// queries each of 8 x 8 tiles over 16000 keys 104 us (5.0 TB/s).
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

constexpr int BKV = kPromptKeys;
// Workgroups that share a CU, by registers and LDS (2048 queries of two heads of 64 over 65000 keys: 128 us with three, 136
// with two; prompts of heads of 64 capped and biased, which keep 4 registers in scratch for it, 100 and 106).
__host__ __device__ constexpr int prompt_shares(int D) { return D == 64 ? 3 : 2; }
// Workgroups where tiles are cut into ranges of keys, at most
__host__ __device__ constexpr int prompt_ranges(int D) { return 256 * prompt_shares(D); }
constexpr int kMaxParts = 128;  // ranges of a tile (two tiles of 85 rows × 31072 keys: 24 us with at most 128, 30 with 243)

// The workspace of a launch with ranges: the parts (one a workgroup, of kPromptRows rows), the number of tiles, and for each
// of max_tiles {first token of its sequence, first flat row, rows + 256 parts, first workgroup}.
__host__ __device__ inline int64_t prompt_part(int D) { return paged_part_floats(kPromptRows, D); }
__device__ __forceinline__ int32_t* prompt_head(const PagedAttnArgs& A, int D) { return (int32_t*)(A.ws + (int64_t)A.groups * prompt_part(D)); }

template <int D>
struct PromptCfg {
  static constexpr int RB = 2 * D;              // bytes a row
  static constexpr int KBYTES = BKV * RB;       // a block of keys (or values)
  static constexpr int STAGE = 2 * KBYTES;
  static constexpr int PPW = KBYTES / 4096;     // wave-wide loads of 1 KB a wavefront and tensor
  static constexpr int PROWS = 4096 / RB;       // rows between a wavefront's consecutive loads
  static constexpr int OP = D + 4;              // pitch of staged output rows, floats
  static constexpr int LDS = 2 * STAGE > kPromptRows * OP * 4 ? 2 * STAGE : kPromptRows * OP * 4;
};

// LDS position of 16-byte chunk c of key row r: c ^ prompt_swz(r). Key fragments (16 rows, one chunk) need a bijection of
// r mod 16, value fragments (4 rows, 4 chunks) the rows' quads on distinct banks.
template <int D>
__device__ __forceinline__ int prompt_swz(int r) {
  if constexpr (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

typedef __attribute__((address_space(3))) void prompt_lds;
typedef const __attribute__((address_space(1))) void prompt_glb;

// Key fragments of four k-steps for both 32-key tiles (T2: bytes from one to the other), waited for in the statement.
template <int T2>
__device__ __forceinline__ void prompt_read_k(u32x4p (&f)[8], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
  asm volatile(
      "ds_read_b128 %0, %8\n ds_read_b128 %1, %8 offset:%12\n ds_read_b128 %2, %9\n ds_read_b128 %3, %9 offset:%12\n"
      "ds_read_b128 %4, %10\n ds_read_b128 %5, %10 offset:%12\n ds_read_b128 %6, %11\n ds_read_b128 %7, %11 offset:%12\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]), "=&v"(f[7])
      : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "i"(T2)
      : "memory");
}
// Transposed value fragments: two reads (keys 4 and 8 + 4 rows on) of four 32-column tiles at one k-step (head dim 128),
// or of two at two k-steps (64).
__device__ __forceinline__ void prompt_read_v(u32x2p (&f)[8], const uint32_t (&a)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n ds_read_b64_tr_b16 %1, %9\n ds_read_b64_tr_b16 %2, %10\n ds_read_b64_tr_b16 %3, %11\n"
      "ds_read_b64_tr_b16 %4, %12\n ds_read_b64_tr_b16 %5, %13\n ds_read_b64_tr_b16 %6, %14\n ds_read_b64_tr_b16 %7, %15\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]), "=&v"(f[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
      : "memory");
}

// Sums and maxima over the wavefront in scalar registers (DPP, no LDS), and an inclusive scan.
template <int CTRL, int MASK>
__device__ __forceinline__ int dpp_int(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, MASK, 0xf, false); }
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_int<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8: within 16 lanes
  v += dpp_int<0x112, 0xf>(v);
  v += dpp_int<0x114, 0xf>(v);
  v += dpp_int<0x118, 0xf>(v);
  v += dpp_int<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3
  v += dpp_int<0x143, 0xc>(v);  // row_bcast 31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
__device__ __forceinline__ int wave_max(int v) {  // (of values of at least 0)
  v = max(v, dpp_int<0x111, 0xf>(v));
  v = max(v, dpp_int<0x112, 0xf>(v));
  v = max(v, dpp_int<0x114, 0xf>(v));
  v = max(v, dpp_int<0x118, 0xf>(v));
  v = max(v, dpp_int<0x142, 0xa>(v));
  v = max(v, dpp_int<0x143, 0xc>(v));
  return __builtin_amdgcn_readlane(v, 63);
}

// prompt_nth_tile's sequences, one a lane.
struct PromptWave {
  PromptSeq own;
  template <class F>
  __device__ __forceinline__ int sum(F&& f) const { return wave_total(f(own)); }
  template <class F>
  __device__ __forceinline__ int largest(F&& f) const { return wave_max(f(own)); }
  template <class F>
  __device__ __forceinline__ int first_past(F&& f, int target, int* before) const {
    const int v = f(own), incl = wave_scan(v);
    const uint64_t past = __builtin_amdgcn_ballot_w64(incl > target);
    if (!past) return -1;
    const int who = __builtin_ctzll(past);
    *before = __builtin_amdgcn_readlane(incl - v, who);
    return who;
  }
  template <class F>
  __device__ __forceinline__ int at(int who, F&& f) const { return __builtin_amdgcn_readlane(f(own), who); }
};

// CAP, BIAS: scores are capped, biased by distance. TREE: the queries are a tree of drafted tokens (PagedAttnArgs::visible).
template <class X, class E, int D, bool CAP, bool BIAS, bool TREE>
__global__ void __launch_bounds__(256, prompt_shares(D)) paged_prompt_kernel(const PagedAttnArgs A) {
  typedef PromptCfg<D> C;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float row_ml[kPromptRows][2];
  __shared__ PagedRowLds row_lds;
  __shared__ uint32_t bad_rows[4];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = A.Hq / A.Hkv;
  const PagedScore score(A);

  // rows of no sequence
  for (int64_t t = blockIdx.x; t < A.T; t += gridDim.x) {
    if (t >= paged_start(A, 0) && t < paged_start(A, A.B)) continue;
    for (int64_t i = tid; i < (int64_t)A.Hq * D; i += 256) ((uint16_t*)A.o)[t * A.Hq * D + i] = 0;
  }

  // Key heads are dealt first: with 8 of them each XCD (workgroup mod 8) reads one head's keys.
  const int x = blockIdx.x, want = x / A.Hkv;
  PagedTile t;
  t.hk = x % A.Hkv;
  int s0 = 0, n = 0, len = 0, tiles = 0;  // of a sequence a lane
  auto sequence = [&](int b) {
    s0 = 0, n = 0, len = 0;
    if (b >= 0 && b < A.B) {
      s0 = paged_start(A, b);
      n = max(0, paged_start(A, b + 1) - s0);
      len = paged_length(A, b);
    }
    tiles = (int)(((uint32_t)n * (uint32_t)G + kPromptRows - 1) / kPromptRows);
  };
  // blocks of a tile: to its last query's key, at most those of a window and the tile's own queries (an estimate where causality
  // does not end them: the order and the ranges of tiles go by it, not what they read)
  const int most = A.window > 0 ? A.window / BKV + kPromptRows / G / BKV + 2 : INT32_MAX;
  int split = 0, cuts = 1, tile_no = 0;  // this workgroup's range of the tile, ranges that the tile has at most
  if (A.splits > 1) {
    // Every tile in ranges of about `each` blocks (a sequence's tiles in as many as its last has), the least with which all
    // fit into the launch: ragged lengths need no other balancing.
    auto cuts_of = [&](int each) { return max(1, min((int)A.splits, (min((len + BKV - 1) / BKV, most) + each - 1) / each)); };
    int room = min(prompt_ranges(D), A.groups) / A.Hkv;
    auto over = [&](auto&& f) {  // the sum of f over the sequences, at most 2^24
      int sum = 0;
      for (int b = 0; b < A.B; b += 64) {
        if (A.B > 64) sequence(b + lane);
        sum = min(1 << 24, sum + wave_total(min(1 << 18, f())));
      }
      return sum;
    };
    sequence(lane);
    const int total = over([&]() { return tiles; });
    int each = 1 << 30;
    if (total <= room) {
      const int work = over([&]() { return (int)min((int64_t)1 << 18, (int64_t)tiles * min((len + BKV - 1) / BKV, most)); });
      // (a third workgroup a CU where that leaves ranges of four blocks: two times 4 x 5 rows over 16000 keys of 4 heads 18
      // us, 20 with it)
      if (work / room < 4 && total <= 512 / A.Hkv) room = min(room, 512 / A.Hkv);
      each = max(2, work / room);
      while (over([&]() { return tiles * cuts_of(each); }) > room) each += max(1, each / 16);
    }
    if (x == 0 && tid == 0) *prompt_head(A, D) = total <= room ? min(total * A.Hkv, A.max_tiles) : 0;
    int sum = 0, before = 0, found = -1;
    for (int b = 0; b < A.B && found < 0; b += 64) {
      if (A.B > 64) sequence(b + lane);
      const int own = cuts_of(each), incl = wave_scan(tiles * own), tiles_incl = wave_scan(tiles);
      const uint64_t here = __builtin_amdgcn_ballot_w64(sum + incl > want);
      if (here) {
        found = __builtin_ctzll(here);
        t.b = b + found;
        t.s0 = __builtin_amdgcn_readlane(s0, found);
        t.n = __builtin_amdgcn_readlane(n, found);
        cuts = __builtin_amdgcn_readlane(own, found);
        const int count = __builtin_amdgcn_readlane(tiles, found);
        const int rest = want - (sum + __builtin_amdgcn_readlane(incl, found) - count * cuts);
        const int turn = __builtin_amdgcn_readfirstlane(rest / cuts), tile = count - 1 - turn;  // (long ones first)
        split = rest - turn * cuts;
        t.row0 = tile * kPromptRows;
        tile_no = (before + __builtin_amdgcn_readlane(tiles_incl, found) - count + tile) * A.Hkv + t.hk;
      } else {
        sum += __builtin_amdgcn_readlane(incl, 63);
        before += __builtin_amdgcn_readlane(tiles_incl, 63);
      }
    }
    if (found < 0) return;
  } else if (A.B <= 64) {
    // Row tiles in falling order of the blocks of keys they see, over all sequences, so that the chip does not wait for
    // long ones that began late (four causal prompts of 875 to 1824 tokens: the last workgroup ended 26% after the mean).
    sequence(lane);
    int tile = 0;
    if (!prompt_nth_tile(PromptWave{PromptSeq{n, len, tiles}}, G, A.causal, most, want, &t.b, &tile)) return;
    t.s0 = __builtin_amdgcn_readlane(s0, t.b);
    t.n = __builtin_amdgcn_readlane(n, t.b);
    t.row0 = tile * kPromptRows;
  } else {
    // from the last sequence to the first, 64 at a time, each from its last tile
    int sum = 0, found = -1;
    for (int b1 = A.B; b1 > 0 && found < 0; b1 -= 64) {
      sequence(b1 - 1 - lane);
      const int incl = wave_scan(tiles);
      const uint64_t here = __builtin_amdgcn_ballot_w64(sum + incl > want);
      if (here) {
        found = __builtin_ctzll(here);
        t.b = b1 - 1 - found;
        t.s0 = __builtin_amdgcn_readlane(s0, found);
        t.n = __builtin_amdgcn_readlane(n, found);
        t.row0 = (sum + __builtin_amdgcn_readlane(incl, found) - 1 - want) * kPromptRows;
      } else {
        sum += __builtin_amdgcn_readlane(incl, 63);
      }
    }
    if (found < 0) return;
  }
  t.len = __builtin_amdgcn_readfirstlane(paged_length(A, t.b));
  t.pos0 = t.len - t.n;
  const int rows = min(kPromptRows, t.n * G - t.row0);
  auto last_key = [&](int q) { return A.causal ? min(t.len - 1, t.pos0 + q) : t.len - 1; };
  auto first_key = [&](int q) { return A.window > 0 ? (int)max((int64_t)0, (int64_t)t.pos0 + q - A.window + 1) : 0; };
  const int q_first = __builtin_amdgcn_readfirstlane(t.row0 / G), q_last = __builtin_amdgcn_readfirstlane((t.row0 + rows - 1) / G);
  // this range's blocks [j0, j1) of 64 keys
  const int any_hi = last_key(q_last);
  // (a drafted token that sees none of the tree sees one key more of a window than the first query otherwise)
  const int tree_lo = A.window > 0 ? (int)max((int64_t)0, (int64_t)t.pos0 - A.window) : 0;
  const int jfirst = (TREE ? tree_lo : first_key(q_first)) / BKV, blocks = max(0, any_hi / BKV + (any_hi >= 0 ? 1 : 0) - jfirst);
  const int parts = max(1, min(cuts, blocks / 2));
  if (A.splits > 1 && split == 0 && tid == 0 && tile_no < A.max_tiles) {  // for the join
    int32_t* const at = prompt_head(A, D) + 4 + 4 * tile_no;
    at[0] = t.s0, at[1] = t.row0, at[2] = rows + 256 * parts, at[3] = x;
  }
  if (split >= parts) return;
  const int each = (blocks + parts - 1) / parts;
  const int j0 = jfirst + min(blocks, split * each), j1 = jfirst + min(blocks, (split + 1) * each);

  // this wavefront's rows, and this lane's
  const int wrows = min(32, rows - 32 * wave);
  const bool wlive = wrows > 0;
  const int wq0 = __builtin_amdgcn_readfirstlane((t.row0 + 32 * wave) / G);
  const int wq1 = __builtin_amdgcn_readfirstlane((t.row0 + 32 * wave + max(wrows, 1) - 1) / G);
  const int w_all_hi = TREE ? t.pos0 - 1 : last_key(wq0), w_any_hi = last_key(wq1);
  const int w_all_lo = first_key(TREE ? t.n - 1 : wq1), w_any_lo = TREE ? tree_lo : first_key(wq0);
  const int flat = t.row0 + min(32 * wave + (lane & 31), rows - 1), qi = flat / G, h = t.hk * G + (flat - qi * G);
  const int pos = t.pos0 + qi, hi = last_key(qi), lo = TREE ? tree_first(A, t.s0 + qi, t.n, t.pos0) : first_key(qi);
  const float slope = BIAS ? A.slopes[h] * kLog2e : 0.f;

  // Blocks into LDS: a wave-wide load fills 1 KB, the lane that fills chunk position c of row r takes chunk c ^ swz(r).
  // (The swizzle depends on r mod 16, the same for all loads of a lane.)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(prompt_lds*)smem;
  const int r0 = (wave * 1024 + lane * 16) / C::RB;
  const uint32_t c0 = 16 * (lane % (C::RB / 16) ^ prompt_swz<D>(r0));
  const int32_t* const table = A.table + (int64_t)t.b * A.M;
  int page0 = -64, entry = -1;   // entries [page0, page0 + 64) of the page table, one a lane
  uint64_t bad = 0;              // keys of the block whose page is outside the cache
  auto fetch = [&](int j) {
    const int key = min(j * BKV + lane, any_hi);
    const int pi = page_of(A, key);
    const int p_first = __builtin_amdgcn_readlane(pi, 0), p_last = __builtin_amdgcn_readlane(pi, 63);
    if (p_last >= page0 + 64) {
      page0 = p_first;
      entry = page0 + lane < A.M ? table[page0 + lane] : -1;
      __builtin_amdgcn_s_waitcnt(0x0F70);  // (waited for at its use, it would be waited for in every iteration)
    }
    const int page = __shfl(entry, pi - page0, 64);
    const bool ok = page >= 0 && page < A.pages;
    bad = __builtin_amdgcn_ballot_w64(!ok);
    const uint32_t cache_row = ok ? ((uint32_t)page * A.Hkv + t.hk) * A.P + (key - pi * A.P) : 0;
    char* const to = smem + (j & 1) * C::STAGE + wave * 1024;
#pragma unroll
    for (int i = 0; i < C::PPW; ++i) {
      const uint64_t at = (uint64_t)(uint32_t)__shfl(cache_row, r0 + i * C::PROWS, 64) * C::RB + c0;
      __builtin_amdgcn_global_load_lds((prompt_glb*)((const char*)A.k_cache + at), (prompt_lds*)(to + i * 4096), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((prompt_glb*)((const char*)A.v_cache + at), (prompt_lds*)(to + C::KBYTES + i * 4096), 16, 0, 0);
    }
  };
  auto arrived = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
  };

  // key fragment: row t·32 + l % 32, chunk 2 s + l / 32: byte k_lane ^ 32 s (+ 32 rows)
  const uint32_t k_lane = (lane & 31) * C::RB + 16 * (prompt_swz<D>(lane & 15) ^ half);
  // value fragment: rows 16 s + vr (+ 8), chunk 4 dt + vc: byte v_lane ^ 64 dt, plus 16 s rows
  const int vr = 4 * half + ((lane & 15) >> 2), vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_lo = vr * C::RB + 16 * (vc ^ prompt_swz<D>(vr)) + 8 * (lane & 1);
  const uint32_t v_hi = (vr + 8) * C::RB + 16 * (vc ^ prompt_swz<D>(vr + 8)) + 8 * (lane & 1);

  // m: the row's exponent reference (log2), -inf until its first visible score
  float m = -INFINITY, l = 0.f;
  f32x16p o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) o[d] = f32x16p{};

  if (j0 < j1) fetch(j0);
  u32x4p qf[D / 16];
  const uint16_t* const qg = (const uint16_t*)A.q + (int64_t)(t.s0 + qi) * A.qs[0] + h * A.qs[1] + 8 * half;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qf[s] = *(const u32x4p*)(qg + 16 * s);
  arrived();
  // (they pass through a statement here, or they would be waited for at their use, in every iteration)
#pragma unroll
  for (int s = 0; s < D / 16; ++s) asm volatile("" : "+v"(qf[s]));
  for (int j = j0; j < j1; ++j) {
    const uint64_t bad_now = bad;
    if (j + 1 < j1) fetch(j + 1);
    const int kb = j * BKV;
    // a wavefront without rows, or none of whose rows sees a key of this block, only takes part in the loads
    if (!wlive || kb > w_any_hi || kb + BKV <= w_any_lo) {
      arrived();
      continue;
    }
    uint64_t vis = ~(uint64_t)0;
    if constexpr (TREE) {
      if (kb + BKV - 1 > w_all_hi) vis = tree_bits(A, t.s0 + qi, kb - t.pos0) >> (4 * half);
    }
    const uint32_t sk = lds0 + (j & 1) * C::STAGE, sv = sk + C::KBYTES;
    f32x16p st[2] = {f32x16p{}, f32x16p{}};
#pragma unroll
    for (int s4 = 0; s4 < D / 64; ++s4) {
      u32x4p f[8];
      const int s = 4 * s4;
      prompt_read_k<32 * C::RB>(f, sk + (k_lane ^ (32 * s)), sk + (k_lane ^ (32 * s + 32)), sk + (k_lane ^ (32 * s + 64)),
                                sk + (k_lane ^ (32 * s + 96)));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) st[tt] = X::mma32(f[2 * i + tt], qf[s + i], st[tt]);
    }
    // exponents relative to the reference, masked; key of register r: kb + 32 tt + 8 (r / 4) + 4 half + r % 4
    const float ref = m == -INFINITY ? 0.f : m;
    // (the last operation of every form adds the bias: none costs one for it)
    const float base = BIAS ? slope * (float)(kb + 4 * half - pos) - ref : -ref;
    auto bias = [&](int tt, int r) { return BIAS ? __builtin_fmaf(slope, (float)(32 * tt + 8 * (r >> 2) + (r & 3)), base) : base; };
    if constexpr (CAP) {
      auto at = [&](int i) -> float& { return ((float*)st)[i]; };
      score.cap<32>(at, [&](int i) { return bias(i >> 4, i & 15); });
    } else {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[tt][r] = __builtin_fmaf(st[tt][r], score.sl2, bias(tt, r));
    }
    if (kb + BKV - 1 > w_all_hi || kb < w_all_lo) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kb + 4 * half + 32 * tt + 8 * (r >> 2) + (r & 3);
          const bool seen = !TREE || ((uint32_t)(vis >> (32 * tt)) >> (8 * (r >> 2) + (r & 3)) & 1);
          st[tt][r] = key <= hi && key >= lo && seen ? st[tt][r] : -INFINITY;
        }
    }
    if (bad_now) {
      const uint64_t bits = bad_now >> (4 * half);
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          st[tt][r] = (uint32_t)(bits >> (32 * tt)) >> (8 * (r >> 2) + (r & 3)) & 1 ? -INFINITY : st[tt][r];
    }
    // The largest exponent, as signed integers over the bit patterns: in order among positive floats, and every negative
    // one is a negative integer, so it tells whether any exceeds 8 (integer instructions run beside another wavefront's
    // matrix instructions, float ones do not)
    int top = (int)0x80000000u;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = max(top, (int)__float_as_uint(st[tt][r]));
    {
      const auto sw = __builtin_amdgcn_permlane32_swap((uint32_t)top, (uint32_t)top, false, false);
      top = max((int)sw[0], (int)sw[1]);
    }
    // the reference moves when a row's block exceeds it by more than 8, or with its first visible score
    if (__builtin_amdgcn_ballot_w64((top > (int)0x41000000) | (m == -INFINITY))) {
      float mb = -INFINITY;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mb = fmaxf(mb, st[tt][r]);
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mb), __float_as_uint(mb), false, false);
      mb = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      const bool move = (mb > 8.f) | ((m == -INFINITY) & (mb != -INFINITY));
      const float shift = move ? mb - X::LIFT : 0.f, mn = move ? ref + shift : m;
      const float alpha = move ? __builtin_amdgcn_exp2f(m - mn) : 1.f;  // (0 from -inf)
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[tt][r] -= shift;
    }
    // probabilities of 16 keys a k-step, in the accumulator's key order (16 s + 8 (e / 4) + 4 half + e % 4): rounded, and what
    // that leaves of them
    u32x4p pf[4], pr[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = __builtin_amdgcn_exp2f(st[s >> 1][8 * (s & 1) + 2 * i]);
        const float b = __builtin_amdgcn_exp2f(st[s >> 1][8 * (s & 1) + 2 * i + 1]);
        pf[s][i] = X::pack(a, b);
        pr[s][i] = X::rest(pf[s][i], a, b);
        l += a + b;
      }
    }
#pragma unroll
    for (int s = 0; s < 4; s += 128 / D) {
      u32x2p f[8];
      uint32_t a[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int dt = i % (D / 32), ss = s + i / (D / 32);
        a[2 * i] = sv + (v_lo ^ (64 * dt)) + 16 * ss * C::RB;
        a[2 * i + 1] = sv + (v_hi ^ (64 * dt)) + 16 * ss * C::RB;
      }
      prompt_read_v(f, a);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int dt = i % (D / 32), ss = s + i / (D / 32);
        const u32x4p vf = {f[2 * i].x, f[2 * i].y, f[2 * i + 1].x, f[2 * i + 1].y};
        o[dt] = X::mma32(vf, pf[ss], o[dt]);
        o[dt] = X::mma32(vf, pr[ss], o[dt]);
      }
    }
    arrived();
  }

  // rows through LDS: unnormalised outputs [128][OP], (maximum, sum) beside them
  float* const so = (float*)smem;
  {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    const int row = 32 * wave + (lane & 31);
    if (half == 0) row_ml[row][0] = m, row_ml[row][1] = l;
    if (tid < 4) bad_rows[tid] = 0;
    bool finite = true;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const f32x4p v = {o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        *(f32x4p*)(so + row * C::OP + 32 * d + 2 * r + 4 * half) = v;
#pragma unroll
        for (int e = 0; e < 4; ++e) finite &= fabsf(v[e]) < INFINITY;
      }
    __syncthreads();
    if (!finite && row < rows) atomicOr(&bad_rows[wave], 1u << (lane & 31));
    __syncthreads();
  }
  // A value that a row does not see has probability 0, which an infinity or NaN in it would still turn into NaN: rows with
  // such outputs are computed again from what they see alone.
  for (int w = 0; w < 4; ++w) {
    uint32_t again = bad_rows[w];
    while (again) {
      const int row = 32 * w + __builtin_ctz(again);
      again &= again - 1;
      const int f = t.row0 + row, q = f / G;
      const int k0 = max(TREE ? tree_first(A, t.s0 + q, t.n, t.pos0) : first_key(q), j0 * BKV), k1 = min(last_key(q) + 1, j1 * BKV);
      float rm, rl;
      const float v = paged_row<E, TREE>(A, t.b, t.s0 + q, t.hk * G + (f - q * G), TREE ? t.pos0 : t.pos0 + q, k0, max(k1, 0), row_lds, &rm, &rl);
      if (tid < D) so[row * C::OP + tid] = v;
      if (tid == 0) row_ml[row][0] = rm, row_ml[row][1] = rl;
      __syncthreads();
    }
  }
  if (parts == 1) {
    // (a row is a query and a head of the group; the thread's next one is 1024 / D on: no division a row)
    constexpr int STEP = 1024 / D;
    const int d = 4 * (tid % (D / 4)), dq = STEP / G, dg = STEP - dq * G;
    int q = (t.row0 + tid / (D / 4)) / G, g = t.row0 + tid / (D / 4) - q * G;
    for (int r = tid / (D / 4); r < rows; r += STEP) {
      const float sum_r = row_ml[r][1];
      paged_put4<X>(A, D, t.s0 + q, t.hk * G + g, d, *(const f32x4p*)(so + r * C::OP + d) * (sum_r == 0.f ? 0.f : 1.f / sum_r));
      q += dq, g += dg;
      if (g >= G) g -= G, ++q;
    }
    return;
  }
  float* const part = A.ws + (int64_t)x * prompt_part(D);
  for (int i = tid; i < rows * (D / 4); i += 256) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    *(f32x4p*)(part + r * D + d) = *(const f32x4p*)(so + r * C::OP + d);
  }
  for (int r = tid; r < rows; r += 256) *(f32x2p*)(part + kPromptRows * D + 2 * r) = f32x2p{row_ml[r][0], row_ml[r][1]};
}

// Joins the parts of every tile: four elements of a row a thread, or of a quarter of its parts (PG = 4). In a launch of its
// own: joined by the range that arrived last, 16 parts of 128 rows took one workgroup 25 us.
template <class X, int D, int PG>
__global__ void __launch_bounds__(256) paged_prompt_join_kernel(const PagedAttnArgs A) {
  constexpr int ITEMS = 256 / PG, CHUNKS = kPromptRows * D / 4 / ITEMS, U = 8;
  __shared__ f32x4p join_o[PG][ITEMS];
  __shared__ f32x2p join_ml[PG][ITEMS];
  const int tid = threadIdx.x, tile = blockIdx.x / CHUNKS, item = blockIdx.x % CHUNKS * ITEMS + tid % ITEMS, pg = tid / ITEMS;
  const int r = item / (D / 4), d = 4 * (item % (D / 4));
  const int32_t* const head = prompt_head(A, D);
  const int tiles = head[0], word = head[6 + 4 * tile], first = head[7 + 4 * tile];
  PagedTile t;
  t.hk = tile % A.Hkv;
  t.s0 = head[4 + 4 * tile], t.row0 = head[5 + 4 * tile];
  const int rows = word & 255, parts = word >> 8;
  if (tile >= tiles || parts < 2) return;
  float m = -INFINITY, l = 0.f;
  f32x4p o = {0.f, 0.f, 0.f, 0.f};
  if (r < rows) {
    for (int p0 = pg; p0 < parts; p0 += PG * U) {
      f32x4p v[U];
      f32x2p w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* const part = A.ws + (int64_t)(first + min(p0 + PG * u, parts - 1) * A.Hkv) * prompt_part(D);
        v[u] = *(const f32x4p*)(part + r * D + d);
        w[u] = *(const f32x2p*)(part + kPromptRows * D + 2 * r);
        if (p0 + PG * u >= parts) w[u].x = -INFINITY, v[u] = f32x4p{0.f, 0.f, 0.f, 0.f};
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, w[u].x);
      const float ref = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - ref);
      m = mn, l *= alpha, o *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float f = __builtin_amdgcn_exp2f(w[u].x - ref);
        l = __builtin_fmaf(w[u].y, f, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[u][e], f, o[e]);
      }
    }
  }
  if constexpr (PG > 1) {
    join_o[pg][tid % ITEMS] = o;
    join_ml[pg][tid % ITEMS] = f32x2p{m, l};
    __syncthreads();
    if (pg) return;
    float mt = -INFINITY;
#pragma unroll
    for (int g = 0; g < PG; ++g) mt = fmaxf(mt, join_ml[g][tid].x);
    const float ref = mt == -INFINITY ? 0.f : mt;
    l = 0.f, o = f32x4p{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < PG; ++g) {
      const float f = __builtin_amdgcn_exp2f(join_ml[g][tid].x - ref);
      l = __builtin_fmaf(join_ml[g][tid].y, f, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(join_o[g][tid][e], f, o[e]);
    }
  }
  if (r < rows) paged_store4<X, D>(A, t, r, d, o * (l == 0.f ? 0.f : 1.f / l));
}

template <class X, class E, int D>
void launch_prompt(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done) {
  constexpr int lds = PromptCfg<D>::LDS;
  const dim3 grid((unsigned)a.groups), block(256);
  auto go = [&](auto kernel) {
    // (per device and kernel, so asked for at every launch: it costs no device work)
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("paged_attention LDS attribute: ") + hipGetErrorString(e));
    launch_k(a.splits > 1 ? nullptr : done, kernel, grid, block, lds, stream, a);
  };
  if (a.visible) a.softcap > 0.f ? go(paged_prompt_kernel<X, E, D, true, false, true>) : go(paged_prompt_kernel<X, E, D, false, false, true>);
  else if (a.softcap > 0.f) a.slopes ? go(paged_prompt_kernel<X, E, D, true, true, false>) : go(paged_prompt_kernel<X, E, D, true, false, false>);
  else a.slopes ? go(paged_prompt_kernel<X, E, D, false, true, false>) : go(paged_prompt_kernel<X, E, D, false, false, false>);
  if (a.splits <= 1) return;
  const unsigned tiles = (unsigned)a.max_tiles, chunks = kPromptRows * D / 4 / 256;
  if (tiles <= 32) launch_k(done, paged_prompt_join_kernel<X, D, 4>, dim3(tiles * chunks * 4), block, 0, stream, a);
  else launch_k(done, paged_prompt_join_kernel<X, D, 1>, dim3(tiles * chunks), block, 0, stream, a);
}

}  // namespace

void paged_prompt_plan(PagedAttnArgs& a, int64_t* ws_floats) {
  const int64_t tiles = (a.T * (a.Hq / a.Hkv) / kPromptRows + a.B) * a.Hkv;  // (at most)
  if (a.T * a.Hq > INT32_MAX || tiles > INT32_MAX) return;
  a.tile_rows = kPromptRows;
  a.max_tiles = (int32_t)tiles;
  // Ranges of keys where the tiles alone may leave the chip short of two workgroups a CU (one tile of 85 rows × 31072 keys
  // of two heads: 68 us in 16 ranges, 24 in 121). Of two blocks at least; under 8 blocks the second launch costs more than
  // they save (300 queries of their own: 17.9 us, 18.5 with ranges).
  a.splits = tiles <= 512 && (int64_t)a.M * a.P >= 8 * BKV ? (int32_t)std::max<int64_t>(1, std::min<int64_t>(kMaxParts, (int64_t)a.M * a.P / (2 * BKV))) : 1;
  // (of ranges no more than the tiles can be cut into; those that the kernel has no room for end at once)
  a.groups = (int32_t)(a.splits > 1 ? std::min<int64_t>(prompt_ranges((int)a.D), tiles * a.splits) : tiles);
  if (a.splits > 1) *ws_floats = a.groups * prompt_part((int)a.D) + 4 + 4 * tiles;
}

void launch_paged_prompt(const PagedAttnArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.splits > 1 && !a.ws) fail(PJRT_Error_Code_INTERNAL, "paged_attention ranges without a workspace");
  if (a.dtype == DT_BF16) a.D == 128 ? launch_prompt<MmaBF16, ElemBF16, 128>(a, stream, done) : launch_prompt<MmaBF16, ElemBF16, 64>(a, stream, done);
  else a.D == 128 ? launch_prompt<MmaF16, ElemF16, 128>(a, stream, done) : launch_prompt<MmaF16, ElemF16, 64>(a, stream, done);
}

}  // namespace ryft
