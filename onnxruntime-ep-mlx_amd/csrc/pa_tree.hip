// pa_tree.hip — what the attention of drafted trees reads besides its rows: every node's bits over the new rows
// (itself and its ancestors, those in the window) and how many rows it stands behind its place in the text.
//
// A workgroup holds the parents of one sequence in LDS; a thread walks up from its node, whose ancestors come in
// falling rows, so that it writes its words from the last to the first.  A parent that is not an earlier row makes
// its node a root.  Bound by its launch and the chain of LDS reads, two walks to every node: a random tree of 257 nodes 5 us,
// of 1024 31, of 4096 303; chains, whose walks are as long as the rows before them, 38, 295 and 4000.  The matrix-core
// kernel makes the bits of trees of at most 64 nodes itself (small_tree).
#include "pa_device.hpp"

namespace pa {
namespace {

__global__ __launch_bounds__(256) void tree_bits_kernel(const TreeParams p) {
  __shared__ int16_t parent[PA_MAX_TREE_NODES];
  const int b = blockIdx.x;
  const int s0 = min(max(p.cum[b], 0), p.num_tokens);
  const int rows = min(max(p.cum[b + 1], s0), p.num_tokens) - s0;
  const int n = min(rows, min(32 * p.words, PA_MAX_TREE_NODES));
  for (int r = threadIdx.x; r < n; r += 256) {
    const int up = p.parents[s0 + r];
    parent[r] = (int16_t)(up >= 0 && up < r ? up : -1);
  }
  __syncthreads();
  for (int r = threadIdx.x; r < n; r += 256) {
    uint32_t* dst = p.bits + (int64_t)(s0 + r) * p.words;
    int node = r, left = p.window > 0 ? p.window : INT32_MAX;
    for (int w = p.words - 1; w >= 0; --w) {
      uint32_t m = 0;
      while (node >= 0 && (node >> 5) == w) {
        m |= 1u << (node & 31);
        node = --left > 0 ? parent[node] : -1;
      }
      dst[w] = m;
    }
    int depth = 0;
    for (int up = parent[r]; up >= 0; up = parent[up]) ++depth;
    p.lag[s0 + r] = r - depth;
  }
  // (rows beyond the bound on the nodes: roots that see the keys before them)
  for (int r = n + threadIdx.x; r < rows; r += 256) {
    for (int w = 0; w < p.words; ++w) p.bits[(int64_t)(s0 + r) * p.words + w] = 0;
    p.lag[s0 + r] = r;
  }
}

}  // namespace

hipError_t launch_tree_bits(const TreeParams& p, hipStream_t s) {
  if (p.batch <= 0 || p.num_tokens <= 0) return hipSuccess;
  hipLaunchKernelGGL(tree_bits_kernel, dim3(p.batch), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace pa
