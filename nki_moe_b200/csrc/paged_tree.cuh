// Attention of trees of drafted tokens: what the store of their rows
// (paged_store.cu) works out for the attention (paged_tree.cu).
#pragma once

#include "paged_mma.cuh"

namespace nkimoe {

// Of a node, for the attention: the nodes of its line (its ancestors that it
// sees, and itself), its position.
struct __align__(16) TrRow {
  unsigned long long line;
  int pos;
  int pad;
};

struct TreeOut {
  const int* parents;   // [T]
  TrRow* rows;          // [T]
  __nv_bfloat16* q_lo;  // [T, nq * 128]: what the rounding of the queries leaves
  int window, sinks;
};

cudaError_t paged_tree_store_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                                    const int* cu_seqlens, const int* kv_lens, const PagedCache& cache,
                                    __nv_bfloat16* q_out, long long T, int B, int nq, float theta, float eps,
                                    const TreeOut& tree, int* status, cudaStream_t s);

// A warp: the line of node i of n whose parents are at `parents` (in the order of
// the rows), and its position.  A parent that does not come before its child
// counts as none (flagged).
__device__ __forceinline__ TrRow tree_line(const int* parents, int n, int i, int past, int window, int sinks, int lane,
                                           int* status) {
  const int p0 = lane < n ? parents[lane] : -1, p1 = lane + 32 < n ? parents[lane + 32] : -1;
  int depth = 0, cur = i;
  unsigned long long line = 1ull << i;
  for (;;) {  // every lane takes the same way
    const int a = __shfl_sync(0xffffffffu, p0, cur & 31), b = __shfl_sync(0xffffffffu, p1, cur & 31);
    const int par = cur < 32 ? a : b;
    if (par < 0 || par >= cur) {
      if (par != -1 && lane == 0) atomicOr(status, kDevErrBadIndex);
      break;
    }
    cur = par;
    ++depth;
    line |= 1ull << cur;
  }
  const int pos = past + depth;
  if (window > 0 && depth >= window) {
    // the ancestor k steps up stands at pos - k
    line = 1ull << i;
    cur = i;
    for (int k = 1; k <= depth; ++k) {
      const int a = __shfl_sync(0xffffffffu, p0, cur & 31), b = __shfl_sync(0xffffffffu, p1, cur & 31);
      cur = cur < 32 ? a : b;
      if (k < window || pos - k < sinks) line |= 1ull << cur;
    }
  }
  return TrRow{line, pos, 0};
}

}  // namespace nkimoe
