// The prompt rows of a batch into a paged cache: per-head q/k RMSNorm and
// rotate-half RoPE of packed QKV rows, the keys and values stored in the
// pages of their sequences, the queries written out for the attention.
//
// Reference: the q/k norms and RoPE of qwen_with_nki.py:330-350 before the
// attention; the reference's caches are the runtime's own (not vendored).
#include <math.h>

#include <type_traits>

#include "paged_tree.cuh"

namespace nkimoe {

namespace {

constexpr int kStoreThreads = 256;

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
  long long T;
  int w_dtype, B, nq;
  float eps;
};

// The rows are nodes of trees: a row's place is where it is stored, its depth
// makes its position.
struct TreeStoreParams : StoreParams {
  TreeOut tree;
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

// kWarps warps share a row, a half-warp a head; a warp needs no other's work
// but the norm weights in shared memory.  Its first heads' loads go out before
// the row's position is known, so the two latencies overlap.
//
// (nq + 2 nkv) * 256 bytes are read and as many written per row.  Measured: 8192
// rows of 32 + 2 * 4 heads 41 us, 4.1 TB/s read and written = 0.63 of the measured
// copy, while the profile shows DRAM at 33 % (half of the traffic ends in L2) and
// issue at 64 %: neither is full, a row's chain of lookups, sines and packing is
// what it waits for.  15 rows 5.1 us.  Of that 4 us and 1.5 us are the keys formed
// again in 64 bits (their check alone 0.3 us).
template <int kWarps, typename Params>
__global__ void __launch_bounds__(kStoreThreads, kWarps == 1 ? 4 : 3) paged_store_kernel(const __grid_constant__ Params p) {
  constexpr bool kTree = std::is_same<Params, TreeStoreParams>::value;
  constexpr int D = kHeadDim;
  constexpr int kHalves = 2 * kWarps;                     // heads of a row at a time
  constexpr int kAhead = kWarps >= 4 ? 3 : 5;             // heads per half-warp in flight
  __shared__ __align__(16) float wtab[2][D];
  __shared__ __align__(16) float2 tab[kStoreThreads / 32][D / 2];
  const int lane = threadIdx.x & 31, l = threadIdx.x & 15, warp = threadIdx.x >> 5;
  const int half = (warp % kWarps) * 2 + (lane >> 4);
  const long long t = static_cast<long long>(blockIdx.x) * (kStoreThreads / 32 / kWarps) + warp / kWarps;
  const int nh = p.nq + 2 * p.c.nkv;
  // the attention of trees reads what lies before them at once: it may start only
  // when all that came before this kernel has ended
  if (!kTree) pdl_launch_dependents();
  pdl_wait();
  if (kTree) pdl_launch_dependents();
  const uint2* row = reinterpret_cast<const uint2*>(p.qkv + t * nh * D) + l;  // head h: row[32 h], row[32 h + 16]
  uint2 raw[kAhead][2];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int h = half + i * kHalves;
    if (h < nh && t < p.T) {
      raw[i][0] = __ldcs(row + h * 32);
      raw[i][1] = __ldcs(row + h * 32 + 16);
    }
  }
  wtab[threadIdx.x >> 7][threadIdx.x & 127] = head_wload(threadIdx.x < D ? p.qw : p.kw, p.w_dtype, threadIdx.x & 127);
  __syncthreads();
  if (t >= p.T) return;
  int b, start, end, kv;
  if (kTree && p.B <= 32) {  // a step's sequences: one look at all of them, a chain of loads less
    const int c = lane < p.B ? p.cu[lane] : 0, next = lane < p.B ? p.cu[lane + 1] : 0, len = lane < p.B ? p.kv_lens[lane] : 0;
    if (t >= __shfl_sync(0xffffffffu, next, p.B - 1)) return;  // behind the last sequence
    b = 31 - __clz(__ballot_sync(0xffffffffu, lane == 0 || (lane < p.B && c <= t)));
    start = __shfl_sync(0xffffffffu, c, b);
    end = __shfl_sync(0xffffffffu, next, b);
    kv = __shfl_sync(0xffffffffu, len, b);
  } else {
    if (t >= p.cu[p.B]) return;  // behind the last sequence
    b = sequence_of(p.cu, p.B, static_cast<int>(t), lane);
    start = p.cu[b];
    end = p.cu[b + 1];
    kv = p.kv_lens[b];
  }
  const int place = kv - end + static_cast<int>(t);
  const int slot = place >> p.c.page_shift;
  if (t < start || t >= end || place < 0 || slot >= p.c.max_pages) {
    if (lane == 0) atomicOr(p.status, kDevErrBadIndex);
    return;
  }
  const int page = p.c.table[b * p.c.table_stride + slot];
  int pos = place;
  if constexpr (kTree) {
    const int n = end - start, i = static_cast<int>(t) - start;
    if (start < 0 || end > p.T || n > kTreeNodes || place < i) {  // the attention leaves such a sequence out
      if (lane == 0) atomicOr(p.status, kDevErrBadIndex);
      return;
    }
    const TrRow line = tree_line(p.tree.parents + start, n, i, place - i, p.tree.window, p.tree.sinks, lane, p.status);
    pos = line.pos;
    if (lane == 0 && warp % kWarps == 0) p.tree.rows[t] = line;
  }
  const bool held = page >= 0 && page < p.c.num_pages;
  if (!held && page != -1 && lane == 0) atomicOr(p.status, kDevErrBadIndex);
  tab[warp][lane] = rope_cos_sin(p.turns.f[lane], pos);
  tab[warp][lane + 32] = rope_cos_sin(p.turns.f[lane + 32], pos);
  __syncwarp();
  const TurnPart turn = turn_part(tab[warp], l);
  // where the row's heads go, this lane's part
  const int in_page = place & ((1 << p.c.page_shift) - 1), head_shift = p.c.page_shift + 5;  // in 8-byte pieces
  uint2* const q_dst = reinterpret_cast<uint2*>(p.q_out + t * p.nq * D) + l;
  uint2* const k_dst = reinterpret_cast<uint2*>(p.c.k + (held ? page * p.c.k_stride + in_page * D : 0)) + l;
  uint2* const v_dst = reinterpret_cast<uint2*>(p.c.v + (held ? page * p.c.v_stride + in_page * D : 0)) + l;
  // a half-warp past the last head runs along with the other (the norm
  // shuffles within the whole warp) and stores nothing
  uint32_t again = 0;  // which pairs of keys to form again: four bits per turn (modulo 8)
  for (int h0 = 0; h0 < nh; h0 += kAhead * kHalves) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = h0 + half + i * kHalves;
      if ((h & ~1) >= nh) break;
      uint2 lo = raw[i][0], hi = raw[i][1];
      if (h + kAhead * kHalves < nh) {
        raw[i][0] = __ldcs(row + (h + kAhead * kHalves) * 32);
        raw[i][1] = __ldcs(row + (h + kAhead * kHalves) * 32 + 16);
      }
      const bool is_q = h < p.nq, is_v = h >= p.nq + p.c.nkv;
      if (!__all_sync(0xffffffffu, is_v)) {
        HeadPart w;
        const float* wt = wtab[is_q ? 0 : 1] + l * 4;
        *reinterpret_cast<ulonglong2*>(w.a) = *reinterpret_cast<const ulonglong2*>(wt);
        *reinterpret_cast<ulonglong2*>(w.b) = *reinterpret_cast<const ulonglong2*>(wt + 64);
        const HeadPart o = norm_rope_part(part_of_rows(lo, hi), w, turn, p.eps);
        if (!is_v) {  // a value goes bit for bit
          lo = row_of_pairs(o.a);
          hi = row_of_pairs(o.b);
          if constexpr (kTree) {
            if (is_q && h < nh) {
              const uint64_t minus = pair2(-1.f, -1.f);
              const HeadPart top = part_of_rows(lo, hi);
              const uint64_t ra[2] = {fma2(top.a[0], minus, o.a[0]), fma2(top.a[1], minus, o.a[1])};
              const uint64_t rb[2] = {fma2(top.b[0], minus, o.b[0]), fma2(top.b[1], minus, o.b[1])};
              uint2* const rest = reinterpret_cast<uint2*>(p.tree.q_lo + t * p.nq * D) + l + h * 32;
              rest[0] = row_of_pairs(ra);
              rest[16] = row_of_pairs(rb);
            }
          }
          if (!is_q) again |= key_near_tie(o) << (4 * ((h0 / kHalves + i) & 7));
        }
      }
      if (h < nh && (is_q || held)) {
        uint2* const dst = is_q ? q_dst + h * 32
                           : is_v ? v_dst + (static_cast<long long>(h - p.nq - p.c.nkv) << head_shift)
                                  : k_dst + (static_cast<long long>(h - p.nq) << head_shift);
        dst[0] = lo;
        dst[16] = hi;
      }
    }
  }
  again = __reduce_or_sync(0xffffffffu, again);
  if (again == 0 || !held) return;
  for (int turn_no = p.nq / kHalves; turn_no * kHalves < p.nq + p.c.nkv; ++turn_no) {
    const uint32_t which = again >> (4 * (turn_no & 7)) & 15u;
    if (which == 0) continue;
    const int h = half + turn_no * kHalves;
    const bool is_k = h >= p.nq && h < p.nq + p.c.nkv;
    uint2 lo = make_uint2(0u, 0u), hi = lo;
    if (is_k) {
      lo = row[h * 32];
      hi = row[h * 32 + 16];
    }
    uint2* const dst = k_dst + (static_cast<long long>(is_k ? h - p.nq : 0) << head_shift);
    uint2 klo = lo, khi = hi;
    if (is_k) {  // as this lane stored them
      klo = dst[0];
      khi = dst[16];
    }
    key_in_64_bits(which, lo, hi, wtab[1] + l * 4, p.turns.f, l, pos, p.eps, klo, khi);
    if (is_k) {
      dst[0] = klo;
      dst[16] = khi;
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

// Rows that get a CTA each.
static int store_few() { return 4 * device_sm_count(); }

static StoreParams store_params(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                                const int* cu_seqlens, const int* kv_lens, const PagedCache& cache,
                                __nv_bfloat16* q_out, long long T, int B, int nq, float theta, float eps, int* status) {
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
  p.T = T;
  p.B = B;
  p.nq = nq;
  p.eps = eps;
  return p;
}

cudaError_t paged_store_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                               const int* cu_seqlens, const int* kv_lens, const PagedCache& cache,
                               __nv_bfloat16* q_out, long long T, int B, int nq, float theta, float eps, int* status,
                               cudaStream_t s) {
  const StoreParams p =
      store_params(qkv, qw, kw, w_dtype, cu_seqlens, kv_lens, cache, q_out, T, B, nq, theta, eps, status);
  // few rows: a CTA's eight warps on each; many: a warp each, so that the lookups
  // and the sines of a row are done once (8192 rows of 32 + 2 * 4 heads, before keys
  // were formed again: 37 us, with two warps 46, with eight 42)
  if (T <= store_few())
    return launch_pdl(paged_store_kernel<8, StoreParams>, dim3(static_cast<unsigned>(T)), dim3(kStoreThreads), 0, s, p);
  return launch_pdl(paged_store_kernel<1, StoreParams>, dim3(static_cast<unsigned>((T + 7) / 8)), dim3(kStoreThreads), 0, s,
                    p);
}

cudaError_t paged_tree_store_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                                    const int* cu_seqlens, const int* kv_lens, const PagedCache& cache,
                                    __nv_bfloat16* q_out, long long T, int B, int nq, float theta, float eps,
                                    const TreeOut& tree, int* status, cudaStream_t s) {
  TreeStoreParams p;
  static_cast<StoreParams&>(p) =
      store_params(qkv, qw, kw, w_dtype, cu_seqlens, kv_lens, cache, q_out, T, B, nq, theta, eps, status);
  p.tree = tree;
  // steps are hundreds of rows: eight warps on each as long as all CTAs run at
  // once, then four (the whole step, 16 trees of 49 to 64 nodes = 913 rows: with
  // four 115 us, two 122, eight 120, one 127; 8 trees of 8: 20, 23, 19 us)
  if (T <= store_few() / 2)
    return launch_pdl(paged_store_kernel<8, TreeStoreParams>, dim3(static_cast<unsigned>(T)), dim3(kStoreThreads), 0, s, p);
  if (T <= 4 * store_few())
    return launch_pdl(paged_store_kernel<4, TreeStoreParams>, dim3(static_cast<unsigned>((T + 1) / 2)), dim3(kStoreThreads), 0,
                      s, p);
  return launch_pdl(paged_store_kernel<1, TreeStoreParams>, dim3(static_cast<unsigned>((T + 7) / 8)), dim3(kStoreThreads), 0,
                    s, p);
}

}  // namespace nkimoe
