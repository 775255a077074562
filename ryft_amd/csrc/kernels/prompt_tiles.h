// Which row tile of ryft.paged_attention's kernel for many rows a workgroup takes, where a wavefront holds all sequences of
// the batch: the rule alone, so that the host can run it too (tests/sanitize/prompt_tiles_check.cc).
#pragma once

#include <hip/hip_runtime.h>

namespace ryft {

constexpr int kPromptRows = 128;  // rows (query, head of a group) of a tile
constexpr int kPromptKeys = 64;   // keys of a block

// A sequence's queries, its length, its row tiles of one key head.
struct PromptSeq {
  int n, len, tiles;
};

__host__ __device__ __forceinline__ int prompt_blocks(int len) { return (len + kPromptKeys - 1) / kPromptKeys; }

// Tiles of a sequence that see `c` blocks of keys or more (`most`: as many as any tile sees): all for c = 0, fewer or as
// many for every block more. A sequence's queries may be more than its keys; the first of them then see none.
__host__ __device__ __forceinline__ int prompt_reach(const PromptSeq& s, int c, int G, bool causal, int most) {
  if (c <= 0) return s.tiles;
  if (c > most) return 0;
  if (!causal) return prompt_blocks(s.len) >= c ? s.tiles : 0;
  const int q = kPromptKeys * (c - 1) - (s.len - s.n);  // the first query that does
  if (q <= 0) return s.tiles;
  return q >= s.n ? 0 : s.tiles - (int)(((unsigned)G * (unsigned)q) / kPromptRows);
}

// The tile at place `want` in falling order of the blocks of keys that tiles see, over the sequences that `w` holds: its
// sequence and its number there; false past the last. Without a sort: the number of blocks that as many tiles reach by
// bisection, then the tile among those of that number. `w` gives the sum and the maximum of a function of the sequences,
// the first sequence at which the running sum of one passes a number (-1: none; `before`: the sum before it), and the
// value of one at a sequence.
template <class W>
__host__ __device__ __forceinline__ bool prompt_nth_tile(const W& w, int G, bool causal, int most, int want, int* seq, int* tile) {
  if (want >= w.sum([&](const PromptSeq& s) { return s.tiles; })) return false;
  // more than `want` tiles see lo blocks, not more see hi
  int lo = 0, hi = w.largest([&](const PromptSeq& s) { return prompt_blocks(s.len) < most ? prompt_blocks(s.len) : most; }) + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (w.sum([&](const PromptSeq& s) { return prompt_reach(s, mid, G, causal, most); }) > want) lo = mid;
    else hi = mid;
  }
  const int rest = want - w.sum([&](const PromptSeq& s) { return prompt_reach(s, hi, G, causal, most); });
  int before = 0;
  const int who = w.first_past(
      [&](const PromptSeq& s) { return prompt_reach(s, lo, G, causal, most) - prompt_reach(s, hi, G, causal, most); }, rest, &before);
  if (who < 0) return false;
  // (the last tiles of a sequence see more blocks, the ones before those as many)
  *seq = who;
  *tile = w.at(who, [&](const PromptSeq& s) { return s.tiles - prompt_reach(s, lo, G, causal, most); }) + rest - before;
  return true;
}

}  // namespace ryft
