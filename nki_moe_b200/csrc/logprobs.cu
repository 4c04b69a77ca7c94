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
  long long rows;
  int V, top, splits, per_split;  // per_split: elements of a split, whole chunks
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

// The factor that moves sums from maximum `from` to `to` (>= from), and the
// distance itself; a side without a finite value (m = -inf, s = 0) moves
// nothing where both are -inf, its distance would be inf - inf.
__device__ __forceinline__ void stat_move(Stat& a, float to) {
  const float d = a.m == to ? 0.f : a.m - to;
  const float f = ex2(d * 1.4426950408889634f);
  // f is 0 from -200 on; d itself times a sum could overflow, and 0 * inf would not be 0
  a.t = f * fmaf(fmaxf(d, -200.f), a.s, a.t);
  a.s *= f;
  a.m = to;
}

__device__ __forceinline__ void stat_join(Stat& a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  stat_move(a, m);
  stat_move(b, m);
  a.s += b.s;
  a.t += b.t;
}

// The stat of the whole warp, in every lane.
__device__ __forceinline__ Stat stat_warp(Stat a) {
  stat_move(a, warp_max(a.m));
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  return a;
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
  if (base >= lo && base + LpVec<T>::Chunk <= hi) {
    const uint4* at = reinterpret_cast<const uint4*>(row + base) + threadIdx.x;
#pragma unroll
    for (int v = 0; v < kLpVecs; ++v) raw[v] = __ldcs(at + v * kLpThreads);
    return;
  }
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

// Maxima that let a NaN through, of two bf16 or of fp32.
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The largest value of a thread's vectors (NaN if one is).
template <typename T>
__device__ __forceinline__ float max_of(const uint4 (&raw)[kLpVecs]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = max_nan_bf16x2(max_nan_bf16x2(raw[0].x, raw[0].y), max_nan_bf16x2(raw[0].z, raw[0].w));
#pragma unroll
    for (int v = 1; v < kLpVecs; ++v)
      m = max_nan_bf16x2(m, max_nan_bf16x2(max_nan_bf16x2(raw[v].x, raw[v].y), max_nan_bf16x2(raw[v].z, raw[v].w)));
    const float2 f = unpack_bf16x2(m);
    return max_nan(f.x, f.y);
  } else {
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < kLpVecs; ++v)
      m = max_nan(m, max_nan(max_nan(__uint_as_float(raw[v].x), __uint_as_float(raw[v].y)),
                             max_nan(__uint_as_float(raw[v].z), __uint_as_float(raw[v].w))));
    return m;
  }
}

// Maxima between -this and this take the short way through the sums, which
// raises -inf to the lowest finite value.  Above, that value's distance from the
// maximum would round to -inf (from 1.02e31 on in fp32, from 1.3e36 on in bf16),
// and 0 times that is NaN; below, it would come near the maximum itself and count.
constexpr float kLpFar = 1e30f;

// A pair of neighbouring elements as fp32, -inf raised to the type's lowest
// finite value (so that 0 times its distance from a maximum within kLpFar is 0).
template <typename T, int P>
__device__ __forceinline__ uint64_t pair_of(const uint4& u) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w = max_nan_bf16x2(P == 0 ? u.x : P == 1 ? u.y : P == 2 ? u.z : u.w, 0xff7fff7fu);
    return pair2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    const float low = __uint_as_float(0xff7fffffu);
    return pair2(max_nan(__uint_as_float(P == 0 ? u.x : u.z), low), max_nan(__uint_as_float(P == 0 ? u.y : u.w), low));
  }
}

// Adds a pair's e^d and e^d d to the sums.
__device__ __forceinline__ void add_pair(uint64_t x, uint64_t neg_max, uint64_t& s, uint64_t& t) {
  const uint64_t d = add2(x, neg_max);
  const float2 y = split2(mul2(d, pair2(1.4426950408889634f, 1.4426950408889634f)));
  const uint64_t e = pair2(ex2(y.x), ex2(y.y));
  s = add2(s, e);
  t = fma2(e, d, t);
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

constexpr int kLpShow = 32 / kLpWarps;  // keys that each warp shows the others

struct TopShared {
  int2 list[kLpWarps][32];
  int2 cand[kLpWarps][64];  // a warp's candidates that are not in its list yet
  int first[32];            // the first chunk's largest keys of eight lanes each
  int seen[32];             // keys of elements seen, kLpShow of each warp (INT_MIN: none yet)
  int4 copy[kLpWarps][8];
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

// The n-th largest of 32 keys that the warps show (`keys`: sh.first or sh.seen),
// as one warp finds them: `n` elements reach it.  The warps write sh.seen while
// others read it, so a reader may find any mix of older and newer keys; the
// keys of a mix are still those of different elements, since an element has one
// slot for good (show_best), and an older key only lowers the bound.
// A few places by one maximum each, more by the keys' ranks (8000 rows of 32000
// with 5 alternatives 145 us against 151, 2000 rows of 151936 with 20 155
// against 169).
__device__ __forceinline__ int nth_shown(TopShared& sh, const volatile int* keys, int n, int warp, int lane) {
  int mine = keys[lane];
  if (n <= 8) {
    for (;;) {
      const int v = __reduce_max_sync(0xffffffffu, mine);
      n -= __popc(__ballot_sync(0xffffffffu, mine == v));
      if (n <= 0) return v;
      if (mine == v) mine = INT_MIN;
    }
  }
  reinterpret_cast<int*>(sh.copy[warp])[lane] = mine;  // one state for all lanes
  __syncwarp();
  int above = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int4 o = sh.copy[warp][i];
    above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
  }
  return __reduce_min_sync(0xffffffffu, above < n ? mine : INT_MAX);
}

// Shows the keys of the warp's best kLpShow elements in its slots of sh.seen; lane
// i < kLpShow holds the id of what slot i shows (negative: nothing).  What is
// among the best stays in its slot, what has come in takes the slot of what has
// dropped out.  What has dropped out never comes back (the best only get better),
// so no element is ever in two slots, at whatever times they are read.
__device__ __forceinline__ void show_best(TopShared& sh, const WarpTop& best, int& shown, int warp, int lane) {
  bool stays = false, known = false;  // this lane's slot, this lane's place in the list
#pragma unroll
  for (int i = 0; i < kLpShow; ++i) {
    stays |= __shfl_sync(0xffffffffu, best.id, i) == shown;
    known |= __shfl_sync(0xffffffffu, shown, i) == best.id;
  }
  const unsigned slots = __ballot_sync(0xffffffffu, lane < kLpShow && !stays);
  unsigned places = __ballot_sync(0xffffffffu, lane < kLpShow && !known && best.key != INT_MIN);
  if (places == 0) return;
  // the i-th free slot takes the i-th new element
  const int turn = __popc(slots & ((1u << lane) - 1u));
#pragma unroll
  for (int i = 0; i + 1 < kLpShow; ++i)
    if (i < turn) places &= places - 1;
  const int from = places ? __ffs(places) - 1 : 0;
  const int key = __shfl_sync(0xffffffffu, best.key, from), id = __shfl_sync(0xffffffffu, best.id, from);
  if ((slots >> lane & 1u) && places) {
    shown = id;
    *static_cast<volatile int*>(&sh.seen[warp * kLpShow + lane]) = key;
  }
}

// Which of a thread's elements may reach the key `least`: bit i for word i
// (bf16: its low half, bit 16 + i its high half).  NaNs always may, and so may
// bf16 values right below a key that is not one of theirs.
template <typename T>
__device__ __forceinline__ unsigned may_reach(const uint4 (&raw)[kLpVecs], int least) {
  unsigned bits = 0;
  if constexpr (sizeof(T) == 2) {
    const unsigned h = (least >= 0 ? least : least ^ 0x7fff0000) >> 16 & 0xffff;
    const unsigned t = h << 16 | h;
#pragma unroll
    for (int v = 0; v < kLpVecs; ++v) {
      const uint32_t w[4] = {raw[v].x, raw[v].y, raw[v].z, raw[v].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t m;
        asm("set.geu.u32.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(w[i]), "r"(t));
        bits |= m & (0x00010001u << (4 * v + i));
      }
    }
  } else {
    const float t = key_value(least);
#pragma unroll
    for (int v = 0; v < kLpVecs; ++v) {
      const uint32_t w[4] = {raw[v].x, raw[v].y, raw[v].z, raw[v].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) bits |= __uint_as_float(w[i]) < t ? 0u : 1u << (4 * v + i);
    }
  }
  return bits;
}

// Word w (0 .. 15) of a thread's vectors, by selection.
__device__ __forceinline__ uint32_t word_of(const uint4 (&raw)[kLpVecs], int w) {
  const bool a = w & 8, b = w & 4, c = w & 2, d = w & 1;
  const uint32_t x = a ? (b ? raw[3].x : raw[2].x) : (b ? raw[1].x : raw[0].x);
  const uint32_t y = a ? (b ? raw[3].y : raw[2].y) : (b ? raw[1].y : raw[0].y);
  const uint32_t z = a ? (b ? raw[3].z : raw[2].z) : (b ? raw[1].z : raw[0].z);
  const uint32_t u = a ? (b ? raw[3].w : raw[2].w) : (b ? raw[1].w : raw[0].w);
  return c ? (d ? u : z) : (d ? y : x);
}

// Joins a warp's part of a chunk (its lanes' vectors, their largest values mx)
// into the warp's best.  Most chunks of a row hold nothing: one comparison and
// one vote.  Where one may, the bound is drawn up to what the CTA's warps have
// seen by then; elements of this warp's own come after all that its list holds,
// so they lose ties there.  In the row's first chunk the warps show the largest
// values of eight lanes each and wait for one another; that bound stays in `least`.
template <typename T>
__device__ __forceinline__ void warp_top(TopShared& sh, WarpTop& best, int& shown, const uint4 (&raw)[kLpVecs], float mx,
                                         int& least, long long base, bool first, int lo, int hi, int top, int warp,
                                         int lane) {
  constexpr int VE = LpVec<T>::VE;
  const int mk = order_key(mx);  // (what lies outside the row counts as -inf, which only lowers the bound)
  if (first) {
    int k = mk;
#pragma unroll
    for (int d = 1; d < 32 / kLpShow; d <<= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, d));
    if (lane % (32 / kLpShow) == 0) {
      sh.first[threadIdx.x / (32 / kLpShow)] = k;
      sh.seen[threadIdx.x / (32 / kLpShow)] = INT_MIN;
    }
    __syncthreads();
  } else if (!__any_sync(0xffffffffu, mk >= least)) {
    return;
  }
  const int worst = __shfl_sync(0xffffffffu, best.key, top - 1);
  least = max(max(least, nth_shown(sh, first ? sh.first : sh.seen, top, warp, lane)),
              worst == 0x7fffffff || worst == INT_MIN ? worst : worst + 1);
  unsigned mine = mk >= least ? may_reach<T>(raw, least) : 0;
  if (!__any_sync(0xffffffffu, mine != 0)) return;
  int2* const cand = sh.cand[warp];
  int n = 0;
  for (bool more = true; more;) {  // an element of every lane that has one left
    const int bit = __ffs(mine) - 1, w = bit & 15;
    const uint32_t word = word_of(raw, w);
    const float x = sizeof(T) == 4 ? __uint_as_float(word) : __uint_as_float(bit & 16 ? word & 0xffff0000u : word << 16);
    const int k = order_key(x);
    const int e = sizeof(T) == 4 ? w : 2 * w + (bit >> 4 & 1);
    const long long id = base + static_cast<long long>((e / VE) * kLpThreads + threadIdx.x) * VE + e % VE;
    const bool in = mine != 0 && id >= lo && id < hi && k >= least;
    const unsigned hit = __ballot_sync(0xffffffffu, in);
    if (in) cand[n + __popc(hit & ((1u << lane) - 1u))] = make_int2(k, static_cast<int>(id));
    n += __popc(hit);
    mine &= mine - 1;
    more = __any_sync(0xffffffffu, mine != 0);
    __syncwarp();
    if (n < 32 && more) continue;
    if (n <= 8) {  // a few: each to its place
      for (int i = 0; i < n; ++i) best.insert(cand[i].x, cand[i].y, lane);
      n = 0;
    }
    while (n >= 32 || (n > 0 && !more)) {  // many: sorted and merged, 32 at a time
      const int2 c = lane < n ? cand[lane] : make_int2(INT_MIN, INT_MAX - 32 - lane);
      WarpTop o{c.x, c.y};
      o.sort(lane);
      best.merge(o, lane);
      const int2 rest = cand[32 + lane];
      __syncwarp();
      cand[lane] = rest;
      __syncwarp();
      n = max(n - 32, 0);
    }
  }
  show_best(sh, best, shown, warp, lane);
}

// CTA (split, row): elements [split * per_split, ...) of the row in chunks of
// 16 KB held in registers, the next chunk in flight; the last CTA of a row
// joins the splits' parts.
//
// Bound by HBM over many rows (the logits read once), by the exponentials next
// to it: measured 2000 rows of 151936 bf16 99.5 us without alternatives (6.11
// TB/s = 0.93 of the measured copy), 124 us with 5 and 154 us with 20: a warp that
// finds a candidate keeps its next loads waiting.  Back to back for seconds, at
// the power cap, 5 alternatives take 135 us.  1000 rows in fp32: 92 us, with 5
// alternatives 104 us.  8 rows with 20 alternatives 8.8 us, in fp32 11 us (one
// chunk per CTA, then the join).
// What was slower with 5 alternatives (when they took 122 us, 8000 rows of 32000
// 140 us; that an element keeps its slot in what the warps show has added 2 and 5
// us): the CTA's best tokens kept in common, a barrier per chunk, 500 us; the
// warps' lists made one after 1, 2, 4, 8 ... chunks, 137 us; a lane's elements
// spread over its warp, one such lane at a time, 124 us (8000 rows: 158).  Chunks
// copied to shared memory two ahead: 121 us, but 108 without alternatives and 155
// for the shorter rows.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(const LpParams p) {
  __shared__ TopShared sh;
  __shared__ Stat warp_stat[kLpWarps];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int split = blockIdx.x % p.splits;
  const long long r = blockIdx.x / p.splits;
  pdl_launch_dependents();
  pdl_wait();
  const T* row = static_cast<const T*>(p.x) + r * p.row_stride;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const long long first = static_cast<long long>(split) * p.per_split - mis;  // a 16-byte boundary
  const int lo = static_cast<int>(max(first, 0LL));
  const int hi = static_cast<int>(min(first + p.per_split, static_cast<long long>(p.V)));
  uint4 raw[kLpVecs], next[kLpVecs];
  if (first < hi) load_chunk<T>(row, first, lo, hi, next);
  // the given token's logit, long before it is needed
  long long tok = -1;
  float x_tok = 0.f;
  if (threadIdx.x == 0) {
    tok = p.tokens[r];
    if (tok >= 0 && tok < p.V) x_tok = lp_float(row[tok]);
  }

  Stat st{-INFINITY, 0.f, 0.f};
  WarpTop best;
  best.clear(lane);
  int least = INT_MIN, shown = -1;
  for (long long base = first; base < hi; base += LpVec<T>::Chunk) {
#pragma unroll
    for (int v = 0; v < kLpVecs; ++v) raw[v] = next[v];
    if (base + LpVec<T>::Chunk < hi) load_chunk<T>(row, base + LpVec<T>::Chunk, lo, hi, next);
    const float mx = max_of<T>(raw);
    Stat c{mx, 0.f, 0.f};
    if (fabsf(mx) < kLpFar) {
      uint64_t s2[2] = {0, 0}, t2[2] = {0, 0};  // short chains
      const uint64_t nm = pair2(-mx, -mx);
#pragma unroll
      for (int v = 0; v < kLpVecs; ++v) {
        add_pair(pair_of<T, 0>(raw[v]), nm, s2[0], t2[0]);
        add_pair(pair_of<T, 1>(raw[v]), nm, s2[1], t2[1]);
        if constexpr (sizeof(T) == 2) {
          add_pair(pair_of<T, 2>(raw[v]), nm, s2[0], t2[0]);
          add_pair(pair_of<T, 3>(raw[v]), nm, s2[1], t2[1]);
        }
      }
      const float2 s = split2(add2(s2[0], s2[1])), t = split2(add2(t2[0], t2[1]));
      c.s = s.x + s.y;
      c.t = t.x + t.y;
    } else if (mx != -INFINITY) {
      // a NaN, +inf, or a maximum so far out that -inf has to stay what it is
#pragma unroll 1
      for (int v = 0; v < kLpVecs; ++v) {
        float x[LpVec<T>::VE];
        unpack_vec<T>(v == 0 ? raw[0] : v == 1 ? raw[1] : v == 2 ? raw[2] : raw[3], x);
#pragma unroll
        for (int i = 0; i < LpVec<T>::VE; ++i) {
          const float d = x[i] - mx;
          const float e = ex2(d * 1.4426950408889634f);
          c.s += e;
          c.t = fmaf(e, fmaxf(d, -200.f), c.t);  // e is 0 there
        }
      }
      if (mx != mx) c.m = -INFINITY;  // the sums hold the NaN
    }
    stat_join(st, c);
    if constexpr (kTop) {
      warp_top<T>(sh, best, shown, raw, mx, least, base, base == first, lo, hi, p.top, warp, lane);
    }
  }
  st = stat_warp(st);
  if (lane == 0) warp_stat[warp] = st;
  __syncthreads();
  if constexpr (kTop) join_warps(sh, best, warp, lane);
  if (warp == 0) st = stat_warp(lane < kLpWarps ? warp_stat[lane] : Stat{-INFINITY, 0.f, 0.f});

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
      st = stat_warp(st);
    }
    if constexpr (kTop) join_warps(sh, best, warp, lane);
  }

  if (warp == 0) {
    const float ls = logf(st.s);
    if (lane == 0) {
      float lp = 0.f;  // a negative token: none is given
      if (tok >= p.V) lp = __int_as_float(0x7fc00000);
      else if (tok >= 0) lp = (x_tok - st.m) - ls;
      p.logprob[r] = lp;
      p.entropy[r] = ls - st.t / st.s;
    }
    if (kTop && lane < p.top) {
      const float v = best.key == 0x7fffffff ? __int_as_float(0x7fc00000) : key_value(best.key);
      p.top_lp[r * p.top + lane] = (v - st.m) - ls;
      p.top_ids[r * p.top + lane] = best.id;
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
cudaError_t lp_launch(const LpParams& p, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.rows * p.splits));
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
  p.rows = T;
  p.V = static_cast<int>(V);
  p.top = top_n;
  const long long chunks = lp_chunks(V, dtype), most = lp_splits(T, V, dtype);
  const long long per = (chunks + most - 1) / most;
  p.splits = static_cast<int>((chunks + per - 1) / per);
  p.per_split = static_cast<int>(per * (kLpChunkBytes / (dtype == kF32 ? 4 : 2)));
  return dtype == kF32 ? lp_launch<float>(p, s) : lp_launch<__nv_bfloat16>(p, s);
}

}  // namespace nkimoe
