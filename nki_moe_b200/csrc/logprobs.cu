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

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpElems = 32;                        // elements per thread and chunk
constexpr int kLpChunk = kLpThreads * kLpElems;     // 16384
constexpr int kLpTopMax = 32;
constexpr int kLpCand = 1024;                       // candidates a chunk may add before the slow path
constexpr int kLpSplits = 32;                       // CTAs per row at most
static_assert(kLpSplits <= 32 && 4 * 148 <= kPagedCounters, "one lane and one counter each");
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
  int V, top, splits, per_split;  // per_split: elements of a split, a multiple of the chunk
};

// Integers that order as the values do: NaN above +inf, -0 equal to +0.
__device__ __forceinline__ int order_key(float x) {
  if (x != x) return 0x7fffffff;
  const int b = __float_as_int(x + 0.0f);
  return b < 0 ? b ^ 0x7fffffff : b;
}
__device__ __forceinline__ float key_value(int k) { return __int_as_float(k < 0 ? k ^ 0x7fffffff : k); }

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
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// A thread's elements of a chunk: vector v of the thread covers VE = 16 bytes
// at element base + (v * threads + tid) * VE, the base rounded down to a
// 16-byte boundary.  Whole vectors are loaded as such; a vector that crosses
// the row's ends is read element by element, and what lies outside is -inf.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, long long base, int lo, int hi, float (&x)[kLpElems]) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int NV = kLpElems / VE;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const long long e0 = base + static_cast<long long>(v * kLpThreads + threadIdx.x) * VE;
    if (e0 >= lo && e0 + VE <= hi) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(row + e0));
      if constexpr (sizeof(T) == 2) {
        float f[8];
        unpack8(u, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[v * VE + e] = f[e];
      } else {
        x[v * VE] = __uint_as_float(u.x);
        x[v * VE + 1] = __uint_as_float(u.y);
        x[v * VE + 2] = __uint_as_float(u.z);
        x[v * VE + 3] = __uint_as_float(u.w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        x[v * VE + e] = e0 + e >= lo && e0 + e < hi ? to_f<T>(row[e0 + e]) : -INFINITY;
    }
  }
}

struct TopShared {
  int key[kLpCand + kLpTopMax];  // candidates, then the best so far
  int id[kLpCand + kLpTopMax];
  int best_key[kLpTopMax];
  int best_id[kLpTopMax];
  int count, have;
  int red_key[kLpWarps], red_id[kLpWarps];
};

// a before b: the greater key, equal ones by the lower id
__device__ __forceinline__ bool before(int ka, int ia, int kb, int ib) { return ka > kb || (ka == kb && ia < ib); }

// The best `top` of the n entries in sh.key / sh.id, in order, into sh.best_*:
// an entry's place is the number of entries before it.
__device__ __forceinline__ void take_best(TopShared& sh, int n, int top) {
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const int k = sh.key[i], id = sh.id[i];
    int place = 0;
    for (int j = 0; j < n && place < top; ++j) place += before(sh.key[j], sh.id[j], k, id);
    if (place < top) {
      sh.best_key[place] = k;
      sh.best_id[place] = id;
    }
  }
  if (threadIdx.x == 0) sh.have = min(n, top);
  __syncthreads();
}

// Joins a chunk (this thread's x, first element ids as load_chunk lays them
// out) into the row's best `top`.  Called by the whole CTA.
template <typename T>
__device__ __forceinline__ void top_chunk(TopShared& sh, const float (&x)[kLpElems], long long base, int lo, int hi,
                                          int top) {
  constexpr int VE = 16 / sizeof(T);
  auto id_of = [&](int i) {
    return static_cast<int>(base + static_cast<long long>((i / VE) * kLpThreads + threadIdx.x) * VE + (i % VE));
  };
  int mk = INT_MIN;  // INT_MIN is no value's key: -inf has 0x807fffff
#pragma unroll
  for (int i = 0; i < kLpElems; ++i) {
    const int id = id_of(i);
    if (id >= lo && id < hi) mk = max(mk, order_key(x[i]));
  }
  const int have = sh.have;
  int least;  // keys from here on are candidates
  if (have == top) {
    // later elements lose ties against the ones already held
    least = sh.best_key[top - 1] == 0x7fffffff ? 0x7fffffff : sh.best_key[top - 1] + 1;
  } else {
    // the top-th largest of the threads' maxima has `top` elements at or above
    // it; its upper 16 bits, found bit by bit, serve as well
    unsigned v = 0;
    const unsigned u = static_cast<unsigned>(mk) ^ 0x80000000u;
    for (int bit = 31; bit >= 16; --bit) {
      const unsigned cand = v | (1u << bit);
      if (__syncthreads_count(u >= cand) >= top) v = cand;
    }
    least = static_cast<int>(v ^ 0x80000000u);
    if (least == INT_MIN) least = INT_MIN + 1;  // fewer than `top` threads have a value: all values
  }
  if (mk >= least) {
#pragma unroll
    for (int i = 0; i < kLpElems; ++i) {
      const int id = id_of(i), k = order_key(x[i]);
      if (id >= lo && id < hi && k >= least) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kLpCand) {
          sh.key[at] = k;
          sh.id[at] = id;
        }
      }
    }
  }
  __syncthreads();
  const int n = sh.count;
  __syncthreads();
  if (n == 0) return;
  if (threadIdx.x == 0) sh.count = 0;
  if (n <= kLpCand) {
    if (threadIdx.x < have) {
      sh.key[n + threadIdx.x] = sh.best_key[threadIdx.x];
      sh.id[n + threadIdx.x] = sh.best_id[threadIdx.x];
    }
    __syncthreads();
    take_best(sh, n + have, top);
    return;
  }
  // More candidates than fit (many equal values): the chunk's best one after
  // another, each the first that comes after the one before it.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int pk = INT_MAX, pid = -1;
  int got = 0;
  for (; got < top; ++got) {
    int bk = INT_MIN, bid = INT_MAX;
#pragma unroll
    for (int i = 0; i < kLpElems; ++i) {
      const int id = id_of(i), k = order_key(x[i]);
      if (id >= lo && id < hi && before(pk, pid, k, id) && before(k, id, bk, bid)) {
        bk = k;
        bid = id;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int ok = __shfl_xor_sync(0xffffffffu, bk, o), oid = __shfl_xor_sync(0xffffffffu, bid, o);
      if (before(ok, oid, bk, bid)) {
        bk = ok;
        bid = oid;
      }
    }
    if (lane == 0) {
      sh.red_key[warp] = bk;
      sh.red_id[warp] = bid;
    }
    __syncthreads();
    bk = INT_MIN;
    bid = INT_MAX;
    for (int w = 0; w < kLpWarps; ++w)
      if (before(sh.red_key[w], sh.red_id[w], bk, bid)) {
        bk = sh.red_key[w];
        bid = sh.red_id[w];
      }
    __syncthreads();
    if (bk == INT_MIN) break;
    if (threadIdx.x == 0) {
      sh.key[got] = bk;
      sh.id[got] = bid;
    }
    pk = bk;
    pid = bid;
  }
  if (threadIdx.x < have) {
    sh.key[got + threadIdx.x] = sh.best_key[threadIdx.x];
    sh.id[got + threadIdx.x] = sh.best_id[threadIdx.x];
  }
  __syncthreads();
  take_best(sh, got + have, top);
}

// CTA (split, row): elements [split * per_split, ...) of the row in chunks of
// 16384 held in registers; the last CTA of a row joins the splits' parts.
//
// Bound by HBM over many rows (the logits read once).
template <typename T, bool kTop>
__global__ void __launch_bounds__(kLpThreads, 2) token_logprobs_kernel(const LpParams p) {
  __shared__ TopShared sh;
  __shared__ Stat warp_stat[kLpWarps];
  __shared__ int s_last;
  const int split = blockIdx.x % p.splits;
  const long long r = blockIdx.x / p.splits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (kTop && threadIdx.x == 0) {
    sh.count = 0;
    sh.have = 0;
  }
  pdl_launch_dependents();
  pdl_wait();
  const T* row = static_cast<const T*>(p.x) + r * p.row_stride;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const long long first = static_cast<long long>(split) * p.per_split - mis;  // a 16-byte boundary
  const int lo = static_cast<int>(max(first, 0LL));
  const int hi = static_cast<int>(min(first + p.per_split, static_cast<long long>(p.V)));
  __syncthreads();

  Stat st{-INFINITY, 0.f, 0.f};
  for (long long base = first; base < hi; base += kLpChunk) {
    float x[kLpElems];
    load_chunk<T>(row, base, lo, hi, x);
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLpElems; ++i) mx = fmaxf(mx, x[i]);
    Stat c{mx, 0.f, 0.f};
    if (mx == -INFINITY) {  // nothing, or only -inf and NaN: a NaN has to show
#pragma unroll
      for (int i = 0; i < kLpElems; ++i)
        if (x[i] != x[i]) c.s = x[i];
    } else {
#pragma unroll
      for (int i = 0; i < kLpElems; ++i) {
        const float d = x[i] - mx;
        const float e = exp2f(d * 1.4426950408889634f);
        c.s += e;
        c.t = fmaf(e, fmaxf(d, -200.f), c.t);  // e is 0 there, and 0 * -inf would not be
      }
    }
    stat_join(st, c);
    if constexpr (kTop) top_chunk<T>(sh, x, base, lo, hi, p.top);
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
    const int have = kTop ? sh.have : 0;
    if (threadIdx.x == 0) __stcg(reinterpret_cast<float4*>(part), make_float4(st.m, st.s, st.t, __int_as_float(have)));
    if (kTop && threadIdx.x < have) {
      __stcg(reinterpret_cast<int*>(part) + 4 + threadIdx.x, sh.best_key[threadIdx.x]);
      __stcg(reinterpret_cast<int*>(part) + 4 + kLpTopMax + threadIdx.x, sh.best_id[threadIdx.x]);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      s_last = atomicAdd(p.counters + r, 1) == p.splits - 1;
      if (s_last) {
        __threadfence();
        p.counters[r] = 0;
        if (kTop) sh.count = 0;
      }
    }
    __syncthreads();
    if (!s_last) return;
    const float* parts = p.part + r * p.splits * kLpPart;
    if (warp == 0) {
      st = Stat{-INFINITY, 0.f, 0.f};
      int n = 0;
      if (lane < p.splits) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(parts + lane * kLpPart));
        st = Stat{v.x, v.y, v.z};
        n = __float_as_int(v.w);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        Stat b;
        b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        b.t = __shfl_xor_sync(0xffffffffu, st.t, o);
        stat_join(st, b);
      }
      if (kTop) {  // where each split's entries go
        int at = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += v;
        }
        if (lane == 31) sh.count = at;
        at -= n;
        const int* ip = reinterpret_cast<const int*>(parts + lane * kLpPart);
        for (int i = 0; i < n; ++i) {
          sh.key[at + i] = __ldcg(ip + 4 + i);
          sh.id[at + i] = __ldcg(ip + 4 + kLpTopMax + i);
        }
      }
    }
    if constexpr (kTop) {
      __syncthreads();
      take_best(sh, sh.count, p.top);
    }
  }

  if (threadIdx.x == 0) {
    const float ls = logf(st.s);
    const long long tok = p.tokens[r];
    float lp = 0.f;  // a negative token: none is given
    if (tok >= p.V) lp = __int_as_float(0x7fc00000);
    else if (tok >= 0) lp = (to_f<T>(row[tok]) - st.m) - ls;
    p.logprob[r] = lp;
    p.entropy[r] = ls - st.t / st.s;
    warp_stat[0] = Stat{st.m, ls, 0.f};
  }
  if constexpr (kTop) {
    __syncthreads();
    if (threadIdx.x < p.top) {
      const int k = sh.best_key[threadIdx.x];
      const float v = k == 0x7fffffff ? __int_as_float(0x7fc00000) : key_value(k);
      p.top_lp[r * p.top + threadIdx.x] = (v - warp_stat[0].m) - warp_stat[0].s;
      p.top_ids[r * p.top + threadIdx.x] = sh.best_id[threadIdx.x];
    }
  }
}

// Chunks of a row: up to 7 places of the first lie before the row (it starts
// at the 16-byte boundary at or below the row's).
long long lp_chunks(long long V) { return (V + 7 + kLpChunk - 1) / kLpChunk; }

// CTAs per row: enough for about two waves of resident CTAs, and no more than
// the row has chunks.
int lp_splits(long long T, long long V) {
  const long long chunks = lp_chunks(V);
  long long n = (4LL * 148 + T - 1) / T;
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
  const int splits = T > 0 ? lp_splits(T, V) : 1;
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
  const long long chunks = lp_chunks(V);
  const long long per = (chunks + lp_splits(T, V) - 1) / lp_splits(T, V);
  p.splits = static_cast<int>((chunks + per - 1) / per);
  p.per_split = static_cast<int>(per) * kLpChunk;
  return dtype == kF32 ? lp_launch<float>(p, T, s) : lp_launch<__nv_bfloat16>(p, T, s);
}

}  // namespace nkimoe
