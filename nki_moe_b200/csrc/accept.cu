// The end of a step with drafted tokens: which of a sequence's drafts the drawn
// tokens agree with, and those drafts' keys and values to where the sequence
// goes on.
//
//   cur = node 0;  while a child c of cur has tokens[c] == sampled[cur]: cur = the lowest such c
//
// The nodes passed are the path; what was drawn after each of them are the new
// tokens.  Node path[k] lies in place past + path[k] of the cache and belongs in
// place past + k, in every plane (layer, key or value) of the pool.  A path's
// nodes rise, so path[k] >= k, and a row that is written was read before by the
// thread that writes it: the moves need no second buffer.
//
// What bounds it: bytes where many rows move (64 trees of 31 nodes, 44 MB in 96 planes
// of 4 heads: 10 us from the L2, 19 from HBM, a kernel's start and the chain among it),
// else the chain lengths -> parents and tokens -> page ids -> rows (8 trees of 8: 3.5 us,
// cold 6).  A sequence's tree is
// walked by every CTA that moves its rows, as a path that another CTA would hand over
// takes a launch or a wait, which cost as much as the whole.
//
// Reference: the reference decodes one token a step; no kernel of its own.
#include "paged.cuh"

namespace nkimoe {

namespace {

constexpr int kAcThreads = 256;
constexpr int kAcAhead = 8;  // rows in flight per thread

struct AcParams {
  const long long* tokens;
  const long long* sampled;
  const int* parents;
  const int* cu;
  const int* kv_lens;
  char* pages;
  const int* table;
  int* counts;
  int* path;
  long long* new_tokens;
  int* status;
  long long table_stride, plane_bytes, page_bytes;
  long long T;
  int B, planes, per_cta, num_pages, max_pages, page_size, row16, units;  // units: 16-byte columns of a plane's row
};

// Nodes of sequence b, -1 where its lengths make no sense.
__device__ __forceinline__ int ac_nodes(const AcParams& p, int b) {
  const int lo = p.cu[b], hi = p.cu[b + 1], kv = p.kv_lens[b];
  if (lo < 0 || hi < lo || hi > p.T) return -1;  // (the difference of two that make no sense may pass 32 bits)
  const int n = hi - lo;
  return n <= kTreeNodes && kv >= n && kv <= static_cast<long long>(p.max_pages) * p.page_size ? n : -1;
}

// A warp: -1 for the rows [from, end), which no path is in.  Where starts do not rise they
// may lie in another sequence, whose own they are then.
__device__ __noinline__ void ac_none(const AcParams& p, long long from, long long end, int lane) {
  from = max(from, 0LL);
  end = min(end, p.T);
  if (from >= end) return;
  bool rise = true;
  for (int q = lane; q < p.B; q += 32) rise = rise && p.cu[q] <= p.cu[q + 1];
  rise = __all_sync(0xffffffffu, rise);
  for (long long i = from + lane; i < end; i += 32) {
    bool owned = false;
    for (int q = 0; !rise && q < p.B; ++q) owned = owned || (ac_nodes(p, q) > 0 && p.cu[q] <= i && i < p.cu[q + 1]);
    if (owned) continue;
    p.path[i] = -1;
    p.new_tokens[i] = -1;
  }
}

// CTA (group of planes, sequence); every CTA walks its sequence's tree itself,
// two nodes a lane, and then moves the path's rows, a thread a column of 16 bytes.
__global__ void __launch_bounds__(kAcThreads) accept_drafts_kernel(const __grid_constant__ AcParams p) {
  __shared__ long long from[kTreeNodes], to[kTreeNodes];  // bytes inside a plane; from < 0: stays
  __shared__ int s_count;
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  if (threadIdx.x < 32) {
    const int lo = p.cu[b], hi = p.cu[b + 1], kv = p.kv_lens[b], n = ac_nodes(p, b);
    int count = 0;
    if (n > 0) {
      int par[2];
      long long tok[2], sam[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = lane + 32 * e;
        par[e] = i < n ? p.parents[lo + i] : -2;
        tok[e] = i < n ? p.tokens[lo + i] : 0;
        sam[e] = i < n ? p.sampled[lo + i] : 0;
      }
      int mine[2] = {lane == 0 ? 0 : -1, -1};  // node of places lane, lane + 32 of the path
      count = 1;
      for (int cur = 0; count < n; ++count) {
        const long long a = __shfl_sync(0xffffffffu, sam[0], cur & 31), c = __shfl_sync(0xffffffffu, sam[1], cur & 31);
        const long long want = cur < 32 ? a : c;
        const unsigned m0 = __ballot_sync(0xffffffffu, par[0] == cur && lane > cur && tok[0] == want);
        const unsigned m1 = __ballot_sync(0xffffffffu, par[1] == cur && lane + 32 > cur && tok[1] == want);
        if (!(m0 | m1)) break;
        cur = m0 ? __ffs(m0) - 1 : 31 + __ffs(m1);
        if (count == lane) mine[0] = cur;
        if (count == lane + 32) mine[1] = cur;
      }
      const int past = kv - n;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = lane + 32 * e;
        from[k] = -1;
        if (k < count && mine[e] != k) {
          const int s = past + mine[e], d = past + k;
          const int* row = p.table + b * p.table_stride;
          const int sp = row[s / p.page_size], dp = row[d / p.page_size];
          const bool held = sp >= 0 && sp < p.num_pages && dp >= 0 && dp < p.num_pages;
          if (held) {
            from[k] = sp * p.page_bytes + (s % p.page_size) * p.row16 * 16LL;
            to[k] = dp * p.page_bytes + (d % p.page_size) * p.row16 * 16LL;
          } else {
            atomicOr(p.status, kDevErrBadIndex);
          }
        }
        if (blockIdx.x == 0 && k < n) {
          const int i = mine[e];
          p.path[lo + k] = i;
          p.new_tokens[lo + k] = i >= 0 ? p.sampled[lo + i] : -1;
        }
      }
    } else if (n < 0 && lane == 0) {
      atomicOr(p.status, kDevErrBadIndex);
    }
    if (lane == 0) {
      s_count = count;
      if (blockIdx.x == 0) p.counts[b] = count;
    }
  } else if (blockIdx.x == 0 && threadIdx.x < 64) {
    // rows without a path: of a refused sequence, of none before the first or behind the last
    if (ac_nodes(p, b) < 0) ac_none(p, p.cu[b], p.cu[b + 1], lane);
    if (b == 0) ac_none(p, 0, p.cu[0], lane);
    if (b == p.B - 1) ac_none(p, p.cu[p.B], p.T, lane);
  }
  __syncthreads();
  const int count = s_count;
  const int last_plane = min(p.planes, static_cast<int>(blockIdx.x + 1) * p.per_cta);
  const int total = (last_plane - static_cast<int>(blockIdx.x) * p.per_cta) * p.units;
  for (int u = threadIdx.x; u < total; u += kAcThreads) {
    const int plane = blockIdx.x * p.per_cta + u / p.units, column = u % p.units;
    const int head = column / p.row16, c = column % p.row16;
    char* base = p.pages + plane * p.plane_bytes + (static_cast<long long>(head) * p.page_size * p.row16 + c) * 16;
    for (int k0 = 1; k0 < count; k0 += kAcAhead) {
      uint4 v[kAcAhead];
#pragma unroll
      for (int e = 0; e < kAcAhead; ++e)
        if (k0 + e < count && from[k0 + e] >= 0) v[e] = *reinterpret_cast<const uint4*>(base + from[k0 + e]);
#pragma unroll
      for (int e = 0; e < kAcAhead; ++e)
        if (k0 + e < count && from[k0 + e] >= 0) *reinterpret_cast<uint4*>(base + to[k0 + e]) = v[e];
    }
  }
}

}  // namespace

cudaError_t accept_drafts_launch(const long long* tokens, const long long* sampled, const int* parents, const int* cu_seqlens,
                                 const int* kv_lens, void* pages, long long planes, long long num_pages, int n_heads,
                                 int page_size, int row_bytes, const int* table, long long table_stride, int max_pages,
                                 int* counts, int* path, long long* new_tokens, long long T, int B, int* status,
                                 cudaStream_t s) {
  AcParams p;
  p.tokens = tokens;
  p.sampled = sampled;
  p.parents = parents;
  p.cu = cu_seqlens;
  p.kv_lens = kv_lens;
  p.pages = static_cast<char*>(pages);
  p.table = table;
  p.counts = counts;
  p.path = path;
  p.new_tokens = new_tokens;
  p.status = status;
  p.table_stride = table_stride;
  p.page_bytes = static_cast<long long>(n_heads) * page_size * row_bytes;
  p.plane_bytes = p.page_bytes * num_pages;
  p.T = T;
  p.planes = static_cast<int>(planes);
  p.num_pages = static_cast<int>(num_pages);
  p.max_pages = max_pages;
  p.page_size = page_size;
  p.row16 = row_bytes / 16;
  p.units = n_heads * p.row16;
  p.per_cta = p.units >= kAcThreads ? 1 : kAcThreads / p.units;
  const unsigned groups = static_cast<unsigned>((planes + p.per_cta - 1) / p.per_cta);
  p.B = B;
  return launch_pdl(accept_drafts_kernel, dim3(groups, B), dim3(kAcThreads), 0, s, p);
}

}  // namespace nkimoe
