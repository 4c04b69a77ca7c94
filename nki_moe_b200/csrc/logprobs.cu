// Log probabilities of given tokens, the entropy of each row's distribution
// and its most likely tokens, in one pass over the logits.
//
//   d_i = x_i - max x,  S = sum e^{d_i},  log p_i = d_i - log S,
//   entropy = log S - (sum e^{d_i} d_i) / S
//
// (the entropy from the shifted values: log S and the mean of d do not cancel
// the way lse and the mean of x would).  Sums are fp32 per thread over at most
// a few hundred elements and joined pairwise.
//
// Reference: the scoring of generated tokens compares full logits on the host
// (main.py:296-378); no kernel of its own.
#include <limits.h>

#include "paged.cuh"

namespace nkimoe {

namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpVecs = 4;                          // 16-byte vectors per thread and chunk
constexpr int kLpChunkBytes = kLpThreads * kLpVecs * 16;  // 16 KB: 8192 bf16 or 4096 fp32 logits
constexpr int kLpTopMax = 32;
constexpr int kLpSplits = 32;                       // CTAs per row at most
constexpr int kLpSplitRows = 4 * 148;               // rows from which on one CTA takes a whole row
static_assert(kLpSplits <= 32 && kLpSplitRows <= kPagedCounters, "one lane and one counter each");
// a CTA's part of a row in the workspace: m, s, t, count, then keys and ids
constexpr int kLpPart = 4 + 2 * kLpTopMax;

struct LpParams {
  const void* x;
  long long row_stride;
  const long long* tokens;
  float* logprob;
  float* entropy;
  float* top_lp;
  long long* top_ids;
  int* counters;  // [T], zero between calls
  float* part;    // [T, splits, kLpPart]
  int V, top, splits, per_split;  // per_split: elements of a split, whole chunks
};

// Integers that order as the values do: NaN above +inf, -0 equal to +0.
__device__ __forceinline__ int order_key(float x) {
  if (x != x) return 0x7fffffff;
  const int b = __float_as_int(x + 0.0f);
  return b < 0 ? b ^ 0x7fffffff : b;
}
__device__ __forceinline__ float key_value(int k) { return __int_as_float(k < 0 ? k ^ 0x7fffffff : k); }

__device__ __forceinline__ float ex2_ftz(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Running maximum, sum and shifted first moment of a set of logits.
struct Stat {
  float m, s, t;
};

__device__ __forceinline__ void stat_join(Stat& a, const Stat& b) {
  const float m = fmaxf(a.m, b.m);
  // a side without a finite value (m = -inf, s = 0) moves nothing; its shift
  // would be inf - inf
  const float da = a.m == m ? 0.f : a.m - m, db = b.m == m ? 0.f : b.m - m;
  const float fa = expf(da), fb = expf(db);
  // e^{d} is 0 from -200 on; d itself times a sum could overflow, and 0 * inf would not be 0
  const float ca = fmaxf(da, -200.f), cb = fmaxf(db, -200.f);
  a.t = fa * fmaf(ca, a.s, a.t) + fb * fmaf(cb, b.s, b.t);
  a.s = fa * a.s + fb * b.s;
  a.m = m;
}

template <typename T>
struct LpVec {
  static constexpr int VE = 16 / sizeof(T);                 // elements per vector
  static constexpr int NE = kLpVecs * VE;                   // per thread and chunk: 32 or 16
  static constexpr int Chunk = kLpThreads * NE;             // per CTA and chunk
};

__device__ __forceinline__ float lp_float(float v) { return v; }
__device__ __forceinline__ float lp_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// A thread's vectors of a chunk, as loaded: vector v of the thread covers 16
// bytes at element base + (v * threads + tid) * VE, the base being on a
// 16-byte boundary.  Whole vectors are loaded as such; a vector that crosses
// the row's ends is read element by element, and what lies outside is -inf.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, long long base, int lo, int hi, uint4 (&raw)[kLpVecs]) {
  constexpr int VE = LpVec<T>::VE;
#pragma unroll
  for (int v = 0; v < kLpVecs; ++v) {
    const long long e0 = base + static_cast<long long>(v * kLpThreads + threadIdx.x) * VE;
    if (e0 >= lo && e0 + VE <= hi) {
      raw[v] = __ldcs(reinterpret_cast<const uint4*>(row + e0));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
          const long long e = e0 + 2 * i;
          const float a = e >= lo && e < hi ? lp_float(row[e]) : -INFINITY;
          const float b = e + 1 >= lo && e + 1 < hi ? lp_float(row[e + 1]) : -INFINITY;
          w[i] = pack_bf16x2(a, b);
        } else {
          w[i] = __float_as_uint(e0 + i >= lo && e0 + i < hi ? lp_float(row[e0 + i]) : -INFINITY);
        }
      }
      raw[v] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// Vector v of a chunk as fp32.
template <typename T>
__device__ __forceinline__ void unpack_vec(const uint4& raw, float (&x)[LpVec<T>::VE]) {
  if constexpr (sizeof(T) == 2) {
    unpack8(raw, x);
  } else {
    x[0] = __uint_as_float(raw.x);
    x[1] = __uint_as_float(raw.y);
    x[2] = __uint_as_float(raw.z);
    x[3] = __uint_as_float(raw.w);
  }
}

// a before b: the greater key, equal ones by the lower id
__device__ __forceinline__ bool before(int ka, int ia, int kb, int ib) { return ka > kb || (ka == kb && ia < ib); }

// A warp's best 32 so far, the lane-th best in each lane (INT_MIN: none; the
// ids are all different, so no two entries are equal).
struct WarpTop {
  int key, id;

  __device__ __forceinline__ void clear(int lane) {
    key = INT_MIN;
    id = INT_MAX - lane;
  }

  // Of a pair of lanes, d apart, the one with the bit clear (`up`: set) takes
  // the entry that comes first.
  __device__ __forceinline__ void exchange(int d, bool up, int lane) {
    const int pk = __shfl_xor_sync(0xffffffffu, key, d), pi = __shfl_xor_sync(0xffffffffu, id, d);
    if (before(pk, pi, key, id) == (((lane & d) == 0) != up)) {
      key = pk;
      id = pi;
    }
  }

  // Sorts any 32 entries (bitonic).
  __device__ __forceinline__ void sort(int lane) {
#pragma unroll
    for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
      for (int d = n >> 1; d > 0; d >>= 1) exchange(d, n < 32 && (lane & n), lane);
  }

  // The first 32 of two sorted lists, sorted.
  __device__ __forceinline__ void merge(const WarpTop& o, int lane) {
    const int pk = __shfl_sync(0xffffffffu, o.key, 31 - lane), pi = __shfl_sync(0xffffffffu, o.id, 31 - lane);
    if (before(pk, pi, key, id)) {
      key = pk;
      id = pi;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) exchange(d, false, lane);
  }

  __device__ __forceinline__ void insert(int k, int i, int lane) {
    const int at = __popc(__ballot_sync(0xffffffffu, before(key, id, k, i)));
    const int pk = __shfl_up_sync(0xffffffffu, key, 1), pi = __shfl_up_sync(0xffffffffu, id, 1);
    if (lane > at) {
      key = pk;
      id = pi;
    } else if (lane == at) {
      key = k;
      id = i;
    }
  }
};

struct TopShared {
  int2 list[kLpWarps][32];
  int2 cand[kLpWarps][64];  // a warp's candidates that are not in its list yet
  uint4 spread[kLpWarps][kLpVecs];
  int floor;                // `top` elements of the row are known to be at or above this key
};

// The CTA's best 32 of the warps' lists, in warp 0.
__device__ __forceinline__ void join_warps(TopShared& sh, WarpTop& best, int warp, int lane) {
#pragma unroll
  for (int d = 1; d < kLpWarps; d <<= 1) {
    sh.list[warp][lane] = make_int2(best.key, best.id);
    __syncthreads();
    if ((warp & (2 * d - 1)) == 0) {
      const int2 o = sh.list[warp + d][lane];
      best.merge(WarpTop{o.x, o.y}, lane);
    }
    __syncthreads();
  }
}

// Joins a warp's part of a chunk (its lanes' vectors, their largest values mx)
// into the warp's best.  The warps do this each for itself; what one has found
// lets the others pass over more (sh.floor).  Most chunks of a row hold
// nothing: one comparison and one vote.
template <typename T>
__device__ __forceinline__ void warp_top(TopShared& sh, WarpTop& best, const uint4 (&raw)[kLpVecs], float mx, bool nan,
                                         long long base, int lo, int hi, int top, int lane) {
  constexpr int VE = LpVec<T>::VE;
  // the lane's greatest key (what lies outside the row counts as -inf here,
  // which only lowers the bound)
  const int mk = nan ? 0x7fffffff : order_key(mx);
  const int worst = __shfl_sync(0xffffffffu, best.key, top - 1);
  int least;  // keys from here on are candidates
  if (worst != INT_MIN) {
    least = worst == 0x7fffffff ? worst : worst + 1;  // later elements lose ties against the ones held
  } else {
    // the top-th largest of the lanes' maxima has `top` elements at or above it
    int place = 0;
#pragma unroll
    for (int o = 0; o < 32; ++o) {
      const int k = __shfl_sync(0xffffffffu, mk, o);
      place += k > mk || (k == mk && o < lane);
    }
    least = __shfl_sync(0xffffffffu, mk, __ffs(__ballot_sync(0xffffffffu, place == top - 1)) - 1);
  }
  least = max(least, *const_cast<volatile int*>(&sh.floor));
  unsigned lanes = __ballot_sync(0xffffffffu, mk >= least);
  if (lanes == 0) return;
  int2* const cand = sh.cand[threadIdx.x >> 5];
  uint4* const spread = sh.spread[threadIdx.x >> 5];
  int n = 0;
  while (lanes) {  // one lane's elements at a time, spread over the warp
    const int src = __ffs(lanes) - 1;
    lanes &= lanes - 1;
    if (lane == src) {
#pragma unroll
      for (int v = 0; v < kLpVecs; ++v) spread[v] = raw[v];
    }
    __syncwarp();
    float x = 0.f;
    if (lane < LpVec<T>::NE) x = lp_float(reinterpret_cast<const T*>(spread)[lane]);
    const int k = order_key(x);
    const int tid = (threadIdx.x & ~31) + src;
    const long long id = base + static_cast<long long>((lane / VE) * kLpThreads + tid) * VE + lane % VE;
    const bool in = lane < LpVec<T>::NE && id >= lo && id < hi && k >= least;
    const unsigned hit = __ballot_sync(0xffffffffu, in);
    if (in) cand[n + __popc(hit & ((1u << lane) - 1u))] = make_int2(k, static_cast<int>(id));
    n += __popc(hit);
    __syncwarp();
    if (n < 32 && lanes) continue;
    if (n <= 4) {  // a few: each to its place
      for (int i = 0; i < n; ++i) best.insert(cand[i].x, cand[i].y, lane);
      n = 0;
    }
    while (n >= 32 || (n > 0 && lanes == 0)) {  // many (the first chunk): sorted and merged, 32 at a time
      const int2 c = lane < n ? cand[lane] : make_int2(INT_MIN, INT_MAX - 32 - lane);
      WarpTop more{c.x, c.y};
      more.sort(lane);
      best.merge(more, lane);
      const int2 rest = cand[32 + lane];
      __syncwarp();
      cand[lane] = rest;
      __syncwarp();
      n = max(n - 32, 0);
    }
  }
  const int now = __shfl_sync(0xffffffffu, best.key, top - 1);
  if (lane == 0 && now > worst) atomicMax(&sh.floor, now);
}

// CTA (split, row): elements [split * per_split, ...) of the row in chunks of
// 16 KB held in registers, the next chunk in flight; the last CTA of a row joins the splits' parts.
//
// Bound by HBM over many rows (the logits read once).
template <typename T, bool kTop>
__global__ void __launch_bounds__(kLpThreads, 3) token_logprobs_kernel(const LpParams p) {
  __shared__ TopShared sh;
  __shared__ Stat warp_stat[kLpWarps];
  __shared__ int s_last;
  const int split = blockIdx.x % p.splits;
  const long long r = blockIdx.x / p.splits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (kTop && threadIdx.x == 0) sh.floor = INT_MIN;
  pdl_launch_dependents();
  pdl_wait();
  const T* row = static_cast<const T*>(p.x) + r * p.row_stride;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const long long first = static_cast<long long>(split) * p.per_split - mis;  // a 16-byte boundary
  const int lo = static_cast<int>(max(first, 0LL));
  const int hi = static_cast<int>(min(first + p.per_split, static_cast<long long>(p.V)));
  __syncthreads();

  Stat st{-INFINITY, 0.f, 0.f};
  WarpTop best;
  best.clear(lane);
  uint4 raw[kLpVecs], next[kLpVecs];
  if (first < hi) load_chunk<T>(row, first, lo, hi, next);
  for (long long base = first; base < hi; base += LpVec<T>::Chunk) {
#pragma unroll
    for (int v = 0; v < kLpVecs; ++v) raw[v] = next[v];
    // the next chunk is in flight while this one is worked on
    if (base + LpVec<T>::Chunk < hi) load_chunk<T>(row, base + LpVec<T>::Chunk, lo, hi, next);
    constexpr int VE = LpVec<T>::VE;
    float x[VE];
    float mx = -INFINITY;
#pragma unroll
    for (int v = 0; v < kLpVecs; ++v) {
      unpack_vec<T>(raw[v], x);
#pragma unroll
      for (int e = 0; e < VE; ++e) mx = fmaxf(mx, x[e]);
    }
    Stat c{mx, 0.f, 0.f};
    if (mx == -INFINITY) {  // nothing, or only -inf and NaN: a NaN has to show
#pragma unroll
      for (int v = 0; v < kLpVecs; ++v) {
        unpack_vec<T>(raw[v], x);
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (x[e] != x[e]) c.s = x[e];
      }
    } else {
      float s4[4] = {0.f, 0.f, 0.f, 0.f}, t4[4] = {0.f, 0.f, 0.f, 0.f};  // short chains
#pragma unroll
      for (int v = 0; v < kLpVecs; ++v) {
        unpack_vec<T>(raw[v], x);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float d = x[i] - mx;
          const float e = ex2_ftz(d * 1.4426950408889634f);
          s4[i & 3] += e;
          t4[i & 3] = fmaf(e, fmaxf(d, -200.f), t4[i & 3]);  // e is 0 there, and 0 * -inf would not be
        }
      }
      c.s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
      c.t = (t4[0] + t4[1]) + (t4[2] + t4[3]);
    }
    stat_join(st, c);
    if constexpr (kTop) warp_top<T>(sh, best, raw, mx, c.s != c.s, base, lo, hi, p.top, lane);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    b.t = __shfl_xor_sync(0xffffffffu, st.t, o);
    stat_join(st, b);
  }
  if (lane == 0) warp_stat[warp] = st;
  __syncthreads();
  if constexpr (kTop) join_warps(sh, best, warp, lane);
  if (warp == 0) {
    st = lane < kLpWarps ? warp_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Stat b;
      b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
      b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
      b.t = __shfl_xor_sync(0xffffffffu, st.t, o);
      stat_join(st, b);
    }
  }

  if (p.splits > 1) {
    float* part = p.part + (r * p.splits + split) * kLpPart;
    if (threadIdx.x == 0) __stcg(reinterpret_cast<float4*>(part), make_float4(st.m, st.s, st.t, 0.f));
    if (kTop && threadIdx.x < p.top) {  // lane < top of warp 0
      __stcg(reinterpret_cast<int*>(part) + 4 + lane, best.key);
      __stcg(reinterpret_cast<int*>(part) + 4 + kLpTopMax + lane, best.id);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      s_last = atomicAdd(p.counters + r, 1) == p.splits - 1;
      if (s_last) {
        __threadfence();
        p.counters[r] = 0;
      }
    }
    __syncthreads();
    if (!s_last) return;
    const float* parts = p.part + r * p.splits * kLpPart;
    if constexpr (kTop) {  // the splits' lists, spread over the warps
      best.clear(lane);
      for (int sp = warp; sp < p.splits; sp += kLpWarps) {
        const int* ip = reinterpret_cast<const int*>(parts + sp * kLpPart) + 4 + lane;
        WarpTop o;
        o.clear(lane);
        if (lane < p.top) o = WarpTop{__ldcg(ip), __ldcg(ip + kLpTopMax)};
        best.merge(o, lane);
      }
    }
    if (warp == 0) {
      st = Stat{-INFINITY, 0.f, 0.f};
      if (lane < p.splits) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(parts + lane * kLpPart));
        st = Stat{v.x, v.y, v.z};
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        Stat b;
        b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        b.t = __shfl_xor_sync(0xffffffffu, st.t, o);
        stat_join(st, b);
      }
    }
    if constexpr (kTop) join_warps(sh, best, warp, lane);
  }

  if (threadIdx.x == 0) {
    const float ls = logf(st.s);
    const long long tok = p.tokens[r];
    float lp = 0.f;  // a negative token: none is given
    if (tok >= p.V) lp = __int_as_float(0x7fc00000);
    else if (tok >= 0) lp = (lp_float(row[tok]) - st.m) - ls;
    p.logprob[r] = lp;
    p.entropy[r] = ls - st.t / st.s;
    warp_stat[0] = Stat{st.m, ls, 0.f};
  }
  if constexpr (kTop) {
    __syncthreads();
    if (threadIdx.x < p.top) {
      const int k = best.key;
      const float v = k == 0x7fffffff ? __int_as_float(0x7fc00000) : key_value(k);
      p.top_lp[r * p.top + threadIdx.x] = (v - warp_stat[0].m) - warp_stat[0].s;
      p.top_ids[r * p.top + threadIdx.x] = best.id;
    }
  }
}

// Chunks of a row: up to 7 places of the first lie before the row (it starts
// at the 16-byte boundary at or below the row's).
long long lp_chunks(long long V, int dtype) {
  const int chunk = kLpChunkBytes / (dtype == kF32 ? 4 : 2);
  return (V + 7 + chunk - 1) / chunk;
}

// CTAs per row: one wave of resident CTAs (4 per SM) in all, and no more than the
// row has chunks.
int lp_splits(long long T, long long V, int dtype) {
  const long long chunks = lp_chunks(V, dtype);
  long long n = (kLpSplitRows + T - 1) / T;
  if (n > chunks) n = chunks;
  if (n > kLpSplits) n = kLpSplits;
  return static_cast<int>(n < 1 ? 1 : n);
}

template <typename T>
cudaError_t lp_launch(const LpParams& p, long long rows, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(rows * p.splits));
  return p.top ? launch_pdl(token_logprobs_kernel<T, true>, grid, dim3(kLpThreads), 0, s, p)
               : launch_pdl(token_logprobs_kernel<T, false>, grid, dim3(kLpThreads), 0, s, p);
}

}  // namespace

size_t token_logprobs_workspace_bytes(long long T, long long V, int top_n) {
  (void)top_n;
  // the wider type has the more chunks
  const int splits = T > 0 ? lp_splits(T, V, kF32) : 1;
  return kPagedScratch + (splits > 1 ? sizeof(float) * T * splits * kLpPart : 0);
}

cudaError_t token_logprobs_launch(const void* logits, int dtype, long long row_stride, const long long* tokens,
                                  long long T, long long V, int top_n, float* logprob, float* entropy, float* top_lp,
                                  long long* top_ids, void* workspace, cudaStream_t s) {
  LpParams p;
  p.x = logits;
  p.row_stride = row_stride;
  p.tokens = tokens;
  p.logprob = logprob;
  p.entropy = entropy;
  p.top_lp = top_lp;
  p.top_ids = top_ids;
  char* ws = static_cast<char*>(workspace);
  p.counters = reinterpret_cast<int*>(ws + kPagedStatusBytes);
  p.part = reinterpret_cast<float*>(ws + kPagedScratch);
  p.V = static_cast<int>(V);
  p.top = top_n;
  const long long chunks = lp_chunks(V, dtype), most = lp_splits(T, V, dtype);
  const long long per = (chunks + most - 1) / most;
  p.splits = static_cast<int>((chunks + per - 1) / per);
  p.per_split = static_cast<int>(per * (kLpChunkBytes / (dtype == kF32 ? 4 : 2)));
  return dtype == kF32 ? lp_launch<float>(p, T, s) : lp_launch<__nv_bfloat16>(p, T, s);
}

}  // namespace nkimoe
