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

// Up to two tiles of a sequence's nodes, for each kv head.
struct __align__(16) TrUnit {
  int row0;    // first packed row
  int tokens;  // nodes (<= 2 tpt)
  int past;    // positions before the tree
  int kv;      // places with it
  int b;
  int lo, hi;  // range of the unit's key blocks
  int slot;    // of its partial result, or -1
};

struct TrList {  // in the workspace
  int units;
  int total;  // places of all units and kv heads: key blocks, and kTrItem for each item
  int share;  // a CTA's run of them
  int pad;
};

constexpr int kTrItem = 1;      // key blocks that beginning and ending an item costs
constexpr int kTrMinBlocks = 2;  // places of a CTA's run at least: a key block for each tile

struct TrPlan {
  __nv_bfloat16* q_lo;  // [T, nq * 128]: what the rounding of the queries of units of one tile leaves
  TrRow* rows;    // [T]
  TrList* list;
  TrUnit* units;  // [max_units]
  int* offs;      // [max_units + 1] places before each unit
  int window, sinks;
  int tpt, sms, max_units;
};

cudaError_t paged_tree_store_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                                    const int* parents, const int* cu_seqlens, const int* kv_lens,
                                    const PagedCache& cache, __nv_bfloat16* q_out, long long T, int B, int nq,
                                    float theta, float eps, const TrPlan& plan, int* status, cudaStream_t s);

// Exclusive scan over a CTA of kThreads; `total` gets the sum.
template <int kThreads>
__device__ __forceinline__ int plan_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int w = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += w;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  const int ws = lane < kThreads / 32 ? warp_sums[lane] : 0;
  int wi = ws;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int w = __shfl_up_sync(0xffffffffu, wi, o);
    if (lane >= o) wi += w;
  }
  total = __shfl_sync(0xffffffffu, wi, 31);
  const int base = __shfl_sync(0xffffffffu, wi - ws, warp);
  __syncthreads();
  return base + incl - v;
}

// One CTA: the list of units from the lengths.
template <int kThreads>
__device__ __forceinline__ void tree_plan(const TrPlan& p, const PagedCache& c, const int* cu, const int* kv_lens,
                                          long long T, int B, int* status) {
  __shared__ int warp_sums[32];
  const int per = 2 * p.tpt;
  int units = 0;
  long long places = 0;
  for (int b0 = 0; b0 < B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int n = 0, kv = 0, lo = 0;
    if (b < B) {
      lo = cu[b];
      n = cu[b + 1] - lo;
      kv = kv_lens[b];
      if (lo < 0 || n < 0 || lo + n > T || n > kTreeNodes || kv < n ||
          (n > 0 && kv > static_cast<long long>(c.max_pages) << c.page_shift)) {
        atomicOr(status, kDevErrBadIndex);
        n = 0;
      }
    }
    const int u = (n + per - 1) / per;
    const int blocks = n > 0 ? blocks_of(kv - n, kv - 1, p.window, p.sinks).n : 0;
    const int each = (blocks + kTrItem) * c.nkv;
    int total_u, total_p;
    const int before = units + plan_scan<kThreads>(u, warp_sums, total_u);
    const long long at = places + plan_scan<kThreads>(u * each, warp_sums, total_p);
    for (int i = 0; i < u; ++i) {
      if (before + i >= p.max_units) {  // sequences that overlap: more rows than there are
        atomicOr(status, kDevErrBadIndex);
        break;
      }
      TrUnit un;
      un.row0 = lo + i * per;
      un.tokens = min(per, n - i * per);
      un.past = kv - n;
      un.kv = kv;
      un.b = b;
      un.lo = 0;
      un.hi = blocks;
      un.slot = -1;
      p.units[before + i] = un;
      p.offs[before + i] = static_cast<int>(min(at + static_cast<long long>(i) * each, 0x7fffffffLL));
    }
    units += total_u;
    places += total_p;
  }
  if (units > p.max_units) {
    __syncthreads();  // the last unit's end is not known here: none is run
    units = 0;
    places = 0;
  }
  if (threadIdx.x == 0) {
    places = min(places, 0x7fffffffLL);
    p.offs[units] = static_cast<int>(places);
    const int share = static_cast<int>((places + p.sms - 1) / p.sms);
    *p.list = TrList{units, static_cast<int>(places), max(kTrMinBlocks + kTrItem, share), 0};
  }
}

// A warp: the line of node i of n whose parents are at `parents` (in the order of
// the rows), and its depth.  A parent that does not come before its child counts
// as none (flagged).
__device__ __forceinline__ TrRow tree_line(const int* parents, int n, int i, int past, int window, int sinks, int lane,
                                           int* status) {
  const int p0 = lane < n ? parents[lane] : -1, p1 = lane + 32 < n ? parents[lane + 32] : -1;
  int depth = 0, cur = i;
  unsigned long long line = 1ull << i;
  // every lane takes the same way
  for (;;) {
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
