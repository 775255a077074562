// The choice of row tiles of paged attention's kernel for many rows (kernels/prompt_tiles.h) over ragged batches on the
// host, a wavefront's lanes as an array: every tile is found at exactly one place, none past the last, and in falling
// order of the blocks of keys that tiles see. Prints what it found wrong and ends with 1.
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <set>
#include <vector>

#include "kernels/prompt_tiles.h"

using namespace ryft;

namespace {

struct HostWave {
  std::vector<PromptSeq> own;  // 64 of them
  template <class F>
  int sum(F&& f) const {
    int v = 0;
    for (const PromptSeq& s : own) v += f(s);
    return v;
  }
  template <class F>
  int largest(F&& f) const {
    int v = 0;
    for (const PromptSeq& s : own) v = std::max(v, f(s));
    return v;
  }
  template <class F>
  int first_past(F&& f, int target, int* before) const {
    int v = 0;
    for (size_t i = 0; i < own.size(); ++i) {
      *before = v;
      if ((v += f(own[i])) > target) return (int)i;
    }
    return -1;
  }
  template <class F>
  int at(int who, F&& f) const { return f(own.at((size_t)who)); }
};

long cases = 0;

void check(const std::vector<int>& n, const std::vector<int>& len, int G, bool causal, int window) {
  HostWave w;
  int total = 0;
  for (size_t b = 0; b < 64; ++b) {
    PromptSeq s{0, 0, 0};
    if (b < n.size()) s = PromptSeq{n[b], len[b], (n[b] * G + kPromptRows - 1) / kPromptRows};
    total += s.tiles;
    w.own.push_back(s);
  }
  const int most = window > 0 ? window / kPromptKeys + kPromptRows / G / kPromptKeys + 2 : 0x7fffffff;
  std::set<std::pair<int, int>> found;
  int last = 0x7fffffff;
  bool ok = true;
  for (int want = 0; want < total + 3; ++want) {
    int b = -1, tile = -1;
    const bool got = prompt_nth_tile(w, G, causal, most, want, &b, &tile);
    ok &= got == (want < total);
    if (!got) continue;
    ok &= b >= 0 && b < (int)n.size() && tile >= 0 && tile < w.own[(size_t)b].tiles && found.insert({b, tile}).second;
    if (!ok) break;
    // blocks from the first key on that the tile's last query sees, as far as `most`
    const PromptSeq& s = w.own[(size_t)b];
    const int q = std::min(s.n, ((tile + 1) * kPromptRows + G - 1) / G) - 1;
    const int keys = causal ? std::max(0, std::min(s.len, s.len - s.n + q + 1)) : s.len;
    const int blocks = std::min(prompt_blocks(keys), most);
    ok &= blocks <= last;
    last = blocks;
  }
  ++cases;
  if (ok && (int)found.size() == total) return;
  printf("%d of %d tiles found: group %d, %s, window %d, queries/length", (int)found.size(), total, G, causal ? "causal" : "not causal", window);
  for (size_t b = 0; b < n.size() && b < 8; ++b) printf(" %d/%d", n[b], len[b]);
  printf(" (%d sequences)\n", (int)n.size());
  exit(1);
}

}  // namespace

int main() {
  // more queries than keys: alone, and behind a batch that fills the chip
  for (int window : {0, 1, 100, 4096})
    for (bool causal : {true, false})
      for (int G : {1, 3, 4, 5, 8, 40, 128, 200}) {
        check({200}, {0}, G, causal, window);
        check({200}, {10}, G, causal, window);
        check({300, 0, 1}, {100, 50, 0}, G, causal, window);
        std::vector<int> n(8, 2048), len(8, 2048);
        n.push_back(300), len.push_back(0);
        check(n, len, G, causal, window);
        check(std::vector<int>(64, 100), std::vector<int>(64, 20), G, causal, window);
        check({}, {}, G, causal, window);
        check({0, 0}, {0, 9}, G, causal, window);
      }
  std::mt19937 r(1);
  for (int i = 0; i < 3000; ++i) {
    const int count = 1 + (int)(r() % (i % 10 ? 9 : 64)), G = (int)std::vector<int>{1, 2, 4, 5, 8, 16, 40}[r() % 7];
    std::vector<int> n, len;
    for (int b = 0; b < count; ++b) {
      n.push_back((int)(r() % (r() % 3 ? 700 : 70)));
      // from none to beyond the queries
      len.push_back(r() % 4 == 0 ? 0 : r() % 3 == 0 ? (int)(r() % (n.back() + 1)) : n.back() + (int)(r() % 600));
    }
    check(n, len, G, r() % 4 != 0, r() % 3 ? 0 : (int)(1 + r() % 500));
  }
  printf("prompt tiles: %ld batches\n", cases);
  return 0;
}
