// The prompt rows of a batch into a paged cache: per-head q/k RMSNorm and
// rotate-half RoPE of packed QKV rows, the keys and values stored in the
// pages of their sequences, the queries written out for the attention.
//
// Reference: the q/k norms and RoPE of qwen_with_nki.py:330-350 before the
// attention; the reference's caches are the runtime's own (not vendored).
#include <math.h>

#include "paged.cuh"

namespace nkimoe {

namespace {

constexpr int kStoreThreads = 256;
constexpr int kStoreHalves = kStoreThreads / 16;

struct StoreParams {
  const __nv_bfloat16* qkv;  // [T, (nq + 2 nkv) * 128]
  const void* qw;
  const void* kw;
  const int* cu;       // [B + 1]
  const int* kv_lens;  // [B]
  __nv_bfloat16* q_out;  // [T, nq * 128]
  int* status;
  PagedCache c;
  RopeTurns turns;
  int w_dtype, B, nq;
  float eps;
};

// The sequence whose rows hold row t: the number of starts cu[1..B) that are
// <= t, found 32 candidates at a time (one load and one ballot per level).
__device__ __forceinline__ int sequence_of(const int* cu, int B, int t, int lane) {
  int lo = 0, n = B;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + lane * step;
    const bool starts = lane * step < n && (lane == 0 || cu[at] <= t);
    const int k = 31 - __clz(__ballot_sync(0xffffffffu, starts));
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

// One CTA per row; a half-warp per head (16-byte pieces).  The row's loads go
// out before the position is known, so the two latencies overlap.
//
// Bound by HBM: (nq + 2 nkv) * 256 bytes read and as many written per row.
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const __grid_constant__ StoreParams p) {
  constexpr int D = kHeadDim;
  constexpr int kAhead = 3;  // heads per half-warp in flight: 48 heads in one pass
  __shared__ float2 tab[D / 2];
  const int lane = threadIdx.x & 31, l = threadIdx.x & 15, half = threadIdx.x >> 4;
  const long long t = blockIdx.x;
  const int nh = p.nq + 2 * p.c.nkv;
  pdl_launch_dependents();
  pdl_wait();
  const uint4* row = reinterpret_cast<const uint4*>(p.qkv + t * nh * D);
  uint4 raw[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int h = half + i * kStoreHalves;
    if (h < nh) raw[i] = __ldcs(row + h * 16 + l);
  }
  if (t >= p.cu[p.B]) return;  // rows behind the last sequence
  const int b = sequence_of(p.cu, p.B, static_cast<int>(t), lane);
  const int start = p.cu[b], end = p.cu[b + 1];
  const int pos = p.kv_lens[b] - end + static_cast<int>(t);
  const int slot = pos >> p.c.page_shift;
  if (t < start || t >= end || pos < 0 || slot >= p.c.max_pages) {
    if (threadIdx.x == 0) atomicOr(p.status, kDevErrBadIndex);
    return;
  }
  const int page = p.c.table[b * p.c.table_stride + slot];
  const bool held = page >= 0 && page < p.c.num_pages;
  if (!held && page != -1 && threadIdx.x == 0) atomicOr(p.status, kDevErrBadIndex);
  if (threadIdx.x < D / 2) tab[threadIdx.x] = rope_cos_sin(p.turns.f[threadIdx.x], pos);
  float qw[8], kw[8];
  load_weight8(p.qw, p.w_dtype, l, qw);
  load_weight8(p.kw, p.w_dtype, l, kw);
  __syncthreads();
  const int in_page = pos & ((1 << p.c.page_shift) - 1);
  // a half-warp past the last head runs along with the other (the norm
  // shuffles within the whole warp) and stores nothing
  for (int h0 = 0; h0 < nh; h0 += kAhead * kStoreHalves) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + half + i * kStoreHalves;
      if ((h & ~1) >= nh) break;
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (h < nh) u = h0 == 0 ? raw[i] : __ldcs(row + h * 16 + l);
      const bool is_q = h < p.nq, is_k = !is_q && h < p.nq + p.c.nkv;
      float x[8], w[8], o[8];
      unpack8(u, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = is_q ? qw[e] : kw[e];
      norm_rope_half(x, w, tab, p.eps, l, o);
      if (h >= nh) continue;
      if (is_q) {
        *reinterpret_cast<uint4*>(p.q_out + (t * p.nq + h) * D + l * 8) = pack8(o);
      } else if (held) {
        const int j = is_k ? h - p.nq : h - p.nq - p.c.nkv;
        __nv_bfloat16* dst = is_k ? p.c.k + page * p.c.k_stride : p.c.v + page * p.c.v_stride;
        dst += ((static_cast<long long>(j) << p.c.page_shift) + in_page) * D + l * 8;
        *reinterpret_cast<uint4*>(dst) = is_k ? pack8(o) : u;  // the value bit for bit
      }
    }
  }
}

}  // namespace

RopeTurns rope_turns(float theta) {
  RopeTurns r;
  const double step = pow(static_cast<double>(theta), -1.0 / (kHeadDim / 2));
  double f = 0.15915494309189533577;  // 1 / (2 pi)
  for (int i = 0; i < kHeadDim / 2; ++i, f *= step) r.f[i] = f;
  return r;
}

cudaError_t paged_store_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                               const int* cu_seqlens, const int* kv_lens, const PagedCache& cache,
                               __nv_bfloat16* q_out, long long T, int B, int nq, float theta, float eps, int* status,
                               cudaStream_t s) {
  StoreParams p;
  p.qkv = qkv;
  p.qw = qw;
  p.kw = kw;
  p.cu = cu_seqlens;
  p.kv_lens = kv_lens;
  p.q_out = q_out;
  p.status = status;
  p.c = cache;
  p.turns = rope_turns(theta);
  p.w_dtype = w_dtype;
  p.B = B;
  p.nq = nq;
  p.eps = eps;
  return launch_pdl(paged_store_kernel, dim3(static_cast<unsigned>(T)), dim3(kStoreThreads), 0, s, p);
}

}  // namespace nkimoe
