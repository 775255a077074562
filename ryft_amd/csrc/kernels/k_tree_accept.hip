// ryft.tree_accept: the longest path of each tree of drafted tokens that the model's choices agree with, and its keys and
// values moved to the positions behind the committed ones (the definition stands at TreeAcceptArgs in kernel_abi.h).
//
// One launch, for every layer's caches: a workgroup a sequence and cache, each of which walks its sequence's tree itself,
// since that takes two reads of a few words and nothing else has to be waited for. Latency bounds it: a node's word goes
// through memory three times (starts; tokens, parents and slots; the parent's target) and the walk through LDS once a node
// of the path.
//
// The walk: every node that its parent's choice names enters its number into its parent's word of LDS, the smallest stays,
// and one lane follows the words from the root. A node's children come after it, so that the walk ends.
//
// The move: a thread takes one chunk of a head's row along the whole path, eight nodes' chunks read before any of them is
// written. The j-th node of the path has a number of j or more, so that no chunk is read after its place was written:
// nodes read later have numbers past every place written before.
#include <hip/hip_runtime.h>

#include <string>

#include "../common.h"
#include "kernels.h"
#include "launch.h"

namespace ryft {

namespace {

constexpr int kTreeNodes = 8192;  // of a tree whose words LDS holds

// The lowest child of node i that its choice names (n: none), all threads over the nodes after it: for trees past LDS.
__device__ int next_node(const TreeAcceptArgs& A, int s0, int n, int i, int* low) {
  const int want = A.targets[s0 + i];
  for (int c0 = i + 1; c0 < n; c0 += 256) {
    __syncthreads();
    if (threadIdx.x == 0) *low = n;
    __syncthreads();
    const int c = c0 + (int)threadIdx.x;
    if (c < n && A.parents[s0 + c] == i && A.tokens[s0 + c] == want) atomicMin(low, c);
    __syncthreads();
    if (*low < n) return *low;
  }
  return n;
}

// V: a chunk of a row
template <class V>
__global__ void __launch_bounds__(256) tree_accept_kernel(const TreeAcceptArgs A) {
  __shared__ int next[kTreeNodes];  // the child that a node's choice names; then, from the front, the path
  __shared__ int low, length;
  const int b = blockIdx.x, tid = threadIdx.x;
  const bool first = blockIdx.y == 0;  // (of the workgroups of a sequence, the one that writes the results)
  if (A.B == 0) {
    for (int64_t t = tid; first && t < A.T; t += 256) A.emitted[t] = -1, A.path[t] = -1;
    return;
  }
  auto start = [&](int i) { return (int)min(max((int64_t)A.starts[i], (int64_t)0), A.T); };
  const int s0 = start(b), n = start(b + 1) - s0;
  if (first) {
    // rows of no sequence
    const int lo = start(0), hi = start(A.B);
    for (int64_t t = (int64_t)b * 256 + tid; t < A.T; t += (int64_t)A.B * 256)
      if (t < lo || t >= hi) A.emitted[t] = -1, A.path[t] = -1;
    if (n <= 0 && tid == 0) A.counts[b] = 0;
  }
  if (n <= 0) return;
  const bool small = n <= kTreeNodes;
  if (small) {
    for (int i = tid; i < n; i += 256) next[i] = n;
    __syncthreads();
    for (int i = 1 + tid; i < n; i += 256) {
      const int p = A.parents[s0 + i];
      if (p >= 0 && p < i && A.tokens[s0 + i] == A.targets[s0 + p]) atomicMin(&next[p], i);
    }
    __syncthreads();
    if (tid == 0) {
      // (word j of the path is written when word at >= j has been read)
      int at = 0, j = 0;
      while (at < n) {
        const int to = next[at];
        next[j++] = at;
        at = to;
      }
      length = j;
    }
    __syncthreads();
    if (first) {
      if (tid == 0) A.counts[b] = length;
      for (int i = tid; i < n; i += 256) {
        A.emitted[s0 + i] = i < length ? A.targets[s0 + next[i]] : -1;
        A.path[s0 + i] = i < length ? next[i] : -1;
      }
    }
  } else if (first) {
    int j = 0;
    for (int at = 0; at < n; at = next_node(A, s0, n, at, &low), ++j)
      if (tid == 0) A.emitted[s0 + j] = A.targets[s0 + at], A.path[s0 + j] = at;
    if (tid == 0) A.counts[b] = j;
    for (int i = j + tid; i < n; i += 256) A.emitted[s0 + i] = -1, A.path[s0 + i] = -1;
  }
  if (!A.n_caches) return;
  char* const cache = (char*)A.caches[blockIdx.y];
  const int chunks = A.row_bytes / (int)sizeof(V), items = A.Hkv * chunks;
  const int64_t all = A.pages * A.P;
  // where a node's chunk of head h lies, -1 outside the cache
  auto place = [&](int node, int h, int c) -> int64_t {
    const int slot = A.slots[s0 + node];
    if (slot < 0 || slot >= all) return -1;
    const int page = slot / A.P;
    return (((int64_t)page * A.Hkv + h) * A.P + (slot - page * A.P)) * A.row_bytes + (int64_t)c * (int)sizeof(V);
  };
  constexpr int U = 8;
  if (small) {
    for (int it = tid; it < items; it += 256) {
      const int h = it / chunks, c = it - h * chunks;
      for (int j0 = 1; j0 < length; j0 += U) {
        V v[U];
        int64_t to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = j0 + u, node = j < length ? next[j] : j;
          const int64_t from = node != j ? place(node, h, c) : -1;
          to[u] = from >= 0 ? place(j, h, c) : -1;
          if (to[u] >= 0) v[u] = *(const V*)(cache + from);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (to[u] >= 0) *(V*)(cache + to[u]) = v[u];
      }
    }
  } else {
    // (one node at a time, found by all threads)
    int j = 1;
    for (int at = next_node(A, s0, n, 0, &low); at < n; at = next_node(A, s0, n, at, &low), ++j) {
      if (at == j) continue;
      for (int it = tid; it < items; it += 256) {
        const int h = it / chunks, c = it - h * chunks;
        const int64_t from = place(at, h, c), to = place(j, h, c);
        if (from >= 0 && to >= 0) *(V*)(cache + to) = *(const V*)(cache + from);
      }
    }
  }
}

}  // namespace

void launch_tree_accept(const TreeAcceptArgs& a, hipStream_t stream, hipEvent_t done) {
  if (a.n_caches < 0 || a.n_caches > kMaxTreeCaches || a.B < 0 || a.T < 0 || (a.n_caches && (a.row_bytes < 1 || a.Hkv < 1 || a.P < 1)))
    fail(PJRT_Error_Code_INTERNAL, "tree_accept of a shape the kernel does not take");
  if (a.B == 0 && a.T == 0) return record_done(done, stream);
  // (without a sequence, one workgroup marks every row)
  const dim3 grid((unsigned)(a.B > 0 ? a.B : 1), (unsigned)(a.n_caches > 0 ? a.n_caches : 1));
  auto go = [&](auto chunk) { launch_k(done, tree_accept_kernel<decltype(chunk)>, grid, dim3(256), 0, stream, a); };
  const int rb = a.row_bytes;
  if (rb % 16 == 0) go(uint4{});
  else if (rb % 8 == 0) go(uint2{});
  else if (rb % 4 == 0) go(uint32_t{});
  else go(uint16_t{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PJRT_Error_Code_INTERNAL, std::string("tree_accept launch failed: ") + hipGetErrorString(e));
}

}  // namespace ryft
