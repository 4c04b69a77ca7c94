// Draws a token from every row of logits: softmax of x / temperature,
// restricted to the first top_k tokens (in the order of falling logits, equal
// ones by the lower id), of those to the fewest that hold top_p of their sum,
// and to weights of at least min_p times the largest; then the first id whose
// running sum over the kept ids, in rising order, exceeds u times the whole.
//
//   d_i = x_i - max x,  w_i = 2^(d_i log2(e) / temperature)
//   token = min { i kept : sum_{j <= i, kept} w_j > u S },  log p = log w - log S
//
// The random number u is the caller's.  Which token comes out depends on sums
// over up to V weights next to a border, so the sums have to be better than
// fp32: a border lies within 2^-24 S of u S for one row in a hundred when 10^5
// tokens are kept.  Weights are formed in fp64.  The draw adds them up as whole
// numbers of 2^-44 of the largest, histograms of weights as whole numbers too, so
// that no order of addition, by threads or by atomics, changes a token.
//
// Few rows: a cluster of CTAs holds a row in shared memory, each a slice, so that
// all SMs work on them.  Rows whose slices do not all run at once stay in global
// memory (from the L2 after the first pass), with as many CTAs each as do.  What top_k and
// top_p keep is found from histograms:
//
//   bf16  of the values themselves.  Of each sign the 2048 values of the 16 binary
//         orders below the largest magnitude that matters have a bin, so counts
//         alone give every sum exactly (a weight per bin), and equal logits are
//         cut by counting them in order.  What lies nearer to zero is summed by
//         itself; a border among it is found as in fp32.
//   fp32  over 1024 distances from the maximum (1/32 of a binary order each), of
//         counts or of weights; the border's bin is sorted by the cluster's first
//         CTA, or, with more tokens than that takes, split further by its own
//         smallest and largest (logit, id).
//
// Bounds and figures (B200, 151936 logits a row, device time of replays, so from the L2
// as far as the rows fit; where they come from HBM 6 to 12 us more, a kernel's start and
// its instructions among it): 8 bf16 rows with top-k
// and top-p 20 us (cold 33), a chain of some 20 barriers of a cluster; 1024 rows with top-p 208 us
// (215; 1.5 TB/s of 6.5): an SM has two rows at a time and 3.46 rounds of them, of 60 us a
// row 25 go to the counting pass (7 operations and a shared atomic a logit, whose banks
// conflict 3.3 times), 12 to the borders and the table of weights, 16 to the sums and 6
// to the draw.  fp32 with top-p, 290 rows: 265 to 284 us, 14 operations in 64 bits per logit
// and pass; without filters 120, with min-p alone 62.
// At two CTAs per SM a thread has 64 registers, and the instances spill, of bytes of
// stack: bf16 slices 88, bf16 in global memory 288 (a whole row per CTA 216), fp32 in
// global memory 184 (128), fp32 slices 0; sm_values' bins of a thread are most of it.
//
// Reference: the sampling of the reference's runtime is not vendored; no
// kernel of its own.
#include <cooperative_groups.h>

#include <cstddef>

#include "paged.cuh"

namespace nkimoe {

namespace cg = cooperative_groups;

namespace {

constexpr int kSmThreads = 512;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kSmBins = 1024;
constexpr int kSmBinsPerOctave = 32;
constexpr int kSmList = 2048;        // tokens that the last sort takes
constexpr int kSmCluster = 8;        // CTAs per row at most
constexpr int kSmSlice = 75 * 1024;  // bytes of a row per CTA that two CTAs per SM leave room for
constexpr int kSmValues = 2048;      // values of a sign that have a bin
constexpr int kSmNear = 512;         // logits nearer to zero that a CTA sums
constexpr int kSmMaxVocab = 1 << 18;
constexpr int kSmGroups = 17;        // groups of vectors in a warp's part
constexpr int kSmFew = 48;           // kept logits of a warp's 32 vectors that are set aside
static_assert(2 * kSmThreads == kSmBins, "two bins per thread");
static_assert(2 * (kSmSlice + 39 * 1024) <= 228 * 1024, "two CTAs, with 39 KB of SmShared and the system's each");

using u64 = unsigned long long;

struct SmParams {
  const void* x;
  long long row_stride;
  const void* u;
  const float* temperature;  // per row, or null: the value below
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* tokens;
  float* logprob;
  double temperature_all, top_p_all, min_p_all;
  long long top_k_all;
  int V, slice;  // slice: elements per CTA, whole 16-byte vectors
  int u_f64;
};

struct SmShared {
  float max_of[kSmCluster], min_of[kSmCluster];
  u64 sum_of[kSmCluster];
  u64 lo_of[kSmCluster], hi_of[kSmCluster];
  int count_of[kSmCluster];
  double zone_of[kSmCluster];  // weight of the logits near zero, and how many they are
  int zones_of[kSmCluster];
  double mass_of[kSmCluster];
  // what the first CTA tells all
  int bin;        // -1: no border
  double above;   // counts or weights before the bin
  double target;
  u64 lo, hi;     // the range that is split, as (order, id)
  u64 border;     // the last kept (order, id)
  int listed;     // the first CTA's: tokens in its list
  int pick;
  // the borders of top_k and top_p among values: place in the list of values (-1:
  // none), how many of its tokens are kept, of how many
  int place_of[2], ties_of[2], held_of[2];
  double sum_k;
  int near;                 // logits nearer to zero than the window
  unsigned short near_of[kSmNear];
  double powers[64];  // 2^(j / 64)
  double warp_d[kSmWarps];
  u64 warp_lo[kSmWarps], warp_hi[kSmWarps];
  int warp_n[kSmWarps];
  float warp_f[kSmWarps], warp_g[kSmWarps];
  u64 group_sum[kSmWarps * kSmGroups];  // of kept weights, without equal logits that are cut
  int group_ties[kSmWarps * kSmGroups];  // those
  u64 part_before;
  int part_ties, part;
  union __align__(16) {
    struct {
      unsigned a[kSmBins];  // counts, or the lower words of weights
      unsigned b[kSmBins];  // the upper words
    } hist;
    u64 list[kSmList];
    unsigned values[2 * kSmValues];  // counts by magnitude, then of negative values
    uint2 weights[2 * kSmValues];    // as the counts: a weight's low 22 bits, and the others
    float kept[kSmWarps][32 + kSmFew];  // logits of each warp that wait for their weights
  };
};

static_assert(offsetof(SmShared, values) % 16 == 0, "cleared by vectors");

// Integers that rise as the values fall; -0 equal to +0.
__device__ __forceinline__ unsigned falling(float x) {
  const unsigned b = __float_as_uint(x + 0.0f);
  return ~(b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float falling_value(unsigned o) {
  const unsigned b = ~o;
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

// 2^t for t <= 1, 0 from -1022 on: t = n + f with |f| <= 1/2, 2^f by its Taylor
// series about 0 (the first term left out is 0.35^12 / 12! = 2^-47), 2^n by the exponent.
__device__ __forceinline__ double pow2(double t) {
  const double big = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is rint(t)
  const double s = t + big;
  const int n = __double2loint(s);
  const double f = (t - (s - big)) * 0.69314718055994530942;
  double y = 1.0 / 39916800.0;
  y = fma(y, f, 1.0 / 3628800.0);
  y = fma(y, f, 1.0 / 362880.0);
  y = fma(y, f, 1.0 / 40320.0);
  y = fma(y, f, 1.0 / 5040.0);
  y = fma(y, f, 1.0 / 720.0);
  y = fma(y, f, 1.0 / 120.0);
  y = fma(y, f, 1.0 / 24.0);
  y = fma(y, f, 1.0 / 6.0);
  y = fma(y, f, 0.5);
  y = fma(y, f, 1.0);
  y = fma(y, f, 1.0);
  return t < -1022.0 ? 0.0 : __hiloint2double(__double2hiint(y) + (n << 20), __double2loint(y));
}

// The same for many: t = n / 64 + f with |f| <= 1/128, 2^(n / 64) from a table of 64
// (2^(j / 64)) and the exponent, 2^f by four terms (the first left out is
// (0.0054)^5 / 120 = 2^-44.5); 0 below 2^-60.  11 operations in 64 bits, not 21 (an
// SM does 64 a cycle).
__device__ __forceinline__ double pow2_by(const double* table, double t) {
  const double big = 105553116266496.0;  // 1.5 * 2^46: the sum's low word is rint(64 t)
  const double s = t + big;
  const int n = __double2loint(s);
  const double f = t - (s - big);
  double y = 0.0096181291076284771619790715736589;  // ln(2)^k / k!
  y = fma(y, f, 0.055504108664821579953142263768622);
  y = fma(y, f, 0.24022650695910071233355126316333);
  y = fma(y, f, 0.69314718055994530941723212145818);
  const double w = table[n & 63];
  y = fma(w * y, f, w);
  return t < -60.0 ? 0.0 : __hiloint2double(__double2hiint(y) + ((n >> 6) << 20), __double2loint(y));
}

// Maxima that let a NaN through, and minima that pass one over.
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t min_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// All bits of the halves that are equal.
__device__ __forceinline__ uint32_t equal_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("set.eq.u32.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One row's settings and what is known of it.
struct SmRow {
  double c;    // log2(e) / temperature
  double max;  // the largest logit
  float maxf;
  float bins;  // bins per unit of x
  double min_weight;
  // what is kept so far: logits above `least`, and equal ones up to an id
  float least;
  int last_id;
  bool cut;  // of equal ones the first `ties` in the order of their ids
  int ties;

  __device__ __forceinline__ bool keeps(float x, int id) const { return x > least || (x == least && id <= last_id); }
  __device__ __forceinline__ void keep_all() {
    cut = false;
    least = -INFINITY;  // and no equal one: what lies before the row has negative ids
    last_id = -0x7fffffff - 1;
  }
  __device__ __forceinline__ void keep_to(u64 border) {
    least = falling_value(static_cast<unsigned>(border >> 32));
    last_id = static_cast<int>(border & 0xffffffffu);
  }
  // (rounded by itself: contracted with what follows it, differently where it is inlined,
  // the sums of a group and of its vectors might not be the same whole number)
  __device__ __forceinline__ double exponent(float x) const { return __dmul_rn(static_cast<double>(x) - max, c); }
  __device__ __forceinline__ int bin(float x) const {
    return __float2int_rn(fminf(fminf(maxf - x, 3e38f) * bins, kSmBins - 1.f));
  }
};

// The warp's sum, in every lane.
template <typename N>
__device__ __forceinline__ N sm_sum(N v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The shared memory of CTA r of a row, and their barrier; a whole row's CTA is alone.
template <bool kAlone>
__device__ __forceinline__ SmShared& sm_of(const cg::cluster_group& cl, SmShared& sh, int r) {
  if constexpr (kAlone) return sh;
  return *cl.map_shared_rank(&sh, r);
}
template <bool kAlone>
__device__ __forceinline__ void sm_sync(const cg::cluster_group& cl) {
  if constexpr (kAlone) __syncthreads();
  else cl.sync();
}

// The CTA's part of the row, in shared memory or (kStream) where it is; kOne: all of it.
template <typename T, bool kStream, bool kOne>
struct SmSlice {
  static constexpr int VE = 16 / sizeof(T);
  static constexpr bool kAlone = kOne;
  static constexpr int kAhead = kStream ? 4 : 1;  // vectors in flight per thread
  const uint4* data;
  int vecs;
  int id0;  // of the first element (a vector may begin before the row: -inf there)
  int V;
  int in_lo, in_n;  // the vectors [in_lo, in_lo + in_n) lie inside the row

  // A vector of the row in global memory; what lies outside of the row is -inf.
  static __device__ __forceinline__ uint4 fetch(const uint4* at, int id, int V) {
    if (id >= 0 && id + VE <= V) return __ldg(at);
    union {
      T e[VE];
      uint4 u;
    } x;
    const T* row = reinterpret_cast<const T*>(at);
#pragma unroll
    for (int i = 0; i < VE; ++i) x.e[i] = id + i >= 0 && id + i < V ? row[i] : static_cast<T>(-INFINITY);
    return x.u;
  }
  __device__ __forceinline__ uint4 raw(int v) const {
    if constexpr (kStream) {
      if (static_cast<unsigned>(v - in_lo) < static_cast<unsigned>(in_n)) return __ldg(data + v);
      return fetch(data + v, id0 + v * VE, V);
    }
    return data[v];
  }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[VE]) {
    if constexpr (sizeof(T) == 2) {
      unpack8(u, x);
    } else {
      x[0] = __uint_as_float(u.x);
      x[1] = __uint_as_float(u.y);
      x[2] = __uint_as_float(u.z);
      x[3] = __uint_as_float(u.w);
    }
  }
  // f(vector, its number) for the vectors lo + at, lo + at + step, ... below hi, at
  // being a thread's number in its warp or CTA.  (The warp comes together after each
  // vector: lanes that took a rare way would stay apart for many.)
  template <typename F>
  __device__ __forceinline__ void vectors(int lo, int hi, int at, int step, F f) const {
    int v = lo + at;
    const int lane = threadIdx.x & 31;
    for (; v - lane + 31 + (kAhead - 1) * step < hi; v += kAhead * step) {
      uint4 u[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) u[a] = raw(v + a * step);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        f(u[a], v + a * step);
        __syncwarp();
      }
    }
    for (; v < hi; v += kAhead * step) {
      uint4 u[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (v + a * step < hi) u[a] = raw(v + a * step);
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (v + a * step < hi) f(u[a], v + a * step);
    }
  }
  // f(logit, id) for every finite logit up to the row's border
  template <typename F>
  __device__ __forceinline__ void each(const SmRow& row, F f) const {
    vectors(0, vecs, threadIdx.x, kSmThreads, [&](const uint4& u, int v) {
      float x[VE];
      unpack(u, x);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int id = id0 + v * VE + i;
        if (row.keeps(x[i], id)) f(x[i], id);
      }
    });
  }
};

__device__ __forceinline__ u64 composite(float x, int id) {
  return (static_cast<u64>(falling(x)) << 32) | static_cast<unsigned>(id);
}

// Running sums over the CTA's threads in order, each thread's before it and with
// it (the one is bit for bit the other of the thread before); `total` gets the whole.
template <typename N>
struct SmSums {
  N before, upto;
};
template <typename N>
__device__ __forceinline__ SmSums<N> sm_scan(N v, N* warp_sum, N& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  N prev = __shfl_up_sync(0xffffffffu, v, 1);
  if (lane == 0) prev = 0;
  __syncthreads();  // warp_sum is free
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  N all = lane < kSmWarps ? warp_sum[lane] : N(0);
#pragma unroll
  for (int o = 1; o < kSmWarps; o <<= 1) {
    const N w = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += w;
  }
  total = __shfl_sync(0xffffffffu, all, kSmWarps - 1);
  N base = __shfl_sync(0xffffffffu, all, warp > 0 ? warp - 1 : 0);
  if (warp == 0) base = 0;
  N upto = base + v;
  const N at_end = __shfl_sync(0xffffffffu, all, warp);
  if (lane == 31) upto = at_end;  // as the next warp has it
  return SmSums<N>{base + prev, upto};
}

// Whether this thread is the first whose running sums pass `need` (0 < need <=
// the whole, so there is one).
__device__ __forceinline__ bool sm_passes(const SmSums<double>& s, double need, int* pick) {
  if (threadIdx.x == 0) *pick = kSmThreads;
  __syncthreads();
  if (s.before < need && need <= s.upto) atomicMin(pick, static_cast<int>(threadIdx.x));
  __syncthreads();
  return *pick == static_cast<int>(threadIdx.x);
}

// Finds the last (order, id) that is kept when tokens are taken in order until
// their count reaches k (kMass false; `limit` is k) or their weight reaches
// `limit` times the whole (kMass).  Only tokens that row keeps take part, and
// what it keeps is what comes out.  All CTAs of the cluster call it and take the
// same way through it.
template <bool kMass, typename Slice>
__device__ void sm_select(const cg::cluster_group& cl, SmShared& sh, const Slice& sl, SmRow& row, double limit) {
  const int tid = threadIdx.x, ranks = Slice::kAlone ? 1 : cl.num_blocks();
  const bool first = Slice::kAlone || cl.block_rank() == 0;
  SmShared& lead = sm_of<Slice::kAlone>(cl, sh, 0);
  bool split = false;  // the range is [lo, hi], not yet: one bin of distances
  u64 lo = 0, hi = 0, width = 0;
  double top = 0.0;  // split: exponent of the range's largest weight
  int bin = 0;

  auto member = [&](float x, u64 key) { return split ? key >= lo && key <= hi : row.bin(x) == bin; };

  for (int level = 0;; ++level) {
    // ---- histogram of the range
    for (int i = tid; i < kSmBins; i += kSmThreads) sh.hist.a[i] = sh.hist.b[i] = 0;
    if (first && tid == 0) sh.listed = 0;
    __syncthreads();
    sl.each(row, [&](float x, int id) {
      int at;
      double y = 0.0;  // exponent of the weight relative to the bin
      if (split) {
        const u64 key = composite(x, id);
        if (key < lo || key > hi) return;
        at = static_cast<int>((key - lo) / width);
        if (kMass) y = row.exponent(x) - top;
      } else {
        at = row.bin(x);
        if (kMass) y = row.exponent(x) + at * (1.0 / kSmBinsPerOctave);
      }
      if constexpr (kMass) {
        // in units of 2^-31, at most 2^32 - 1; whoever makes the lower word wrap carries
        const double q = pow2_by(sh.powers, y) * 2147483648.0;
        const unsigned w = q >= 4294967295.0 ? 0xffffffffu : __double2uint_rn(q);
        if (atomicAdd(&sh.hist.a[at], w) > 0xffffffffu - w) atomicAdd(&sh.hist.b[at], 1u);
      } else {
        atomicAdd(&sh.hist.a[at], 1u);
      }
    });
    sm_sync<Slice::kAlone>(cl);
    // ---- the first CTA joins the histograms and finds the bin
    if (first) {
      double v[2] = {0.0, 0.0};
      for (int r = 0; r < ranks; ++r) {
        const SmShared& o = sm_of<Slice::kAlone>(cl, sh, r);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * tid + e;
          v[e] += kMass ? fma(static_cast<double>(o.hist.b[i]), 4294967296.0, static_cast<double>(o.hist.a[i]))
                        : static_cast<double>(o.hist.a[i]);
        }
      }
      if constexpr (kMass) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          v[e] *= pow2(split ? top : (2 * tid + e) * (-1.0 / kSmBinsPerOctave)) * (1.0 / 2147483648.0);
      }
      double total;
      const SmSums<double> sums = sm_scan(v[0] + v[1], sh.warp_d, total);
      if (level == 0 && tid == 0) {
        sh.target = kMass ? fmax(limit * total, 1e-300) : limit;
        sh.above = 0.0;
        sh.bin = -1;
      }
      __syncthreads();
      const double above = sh.above;
      // what is left to reach; the sums of a split range differ from its bin's by their rounding
      double need = sh.target - above;
      const bool none = !kMass && level == 0 && total <= limit;
      if (level > 0) need = fmin(fmax(need, 1e-300), total * (1.0 - 0x1p-50));
      const bool here = sm_passes(sums, need, &sh.pick);
      if (!none && here) {
        const bool second = sums.before + v[0] < need && v[1] > 0.0;
        const int at = 2 * tid + second;
        const double ab = above + sums.before + (second ? v[0] : 0.0);
        for (int r = 0; r < ranks; ++r) {
          SmShared& o = sm_of<Slice::kAlone>(cl, sh, r);
          o.bin = at;
          o.above = ab;
        }
      } else if (none && tid == 0) {
        for (int r = 0; r < ranks; ++r) sm_of<Slice::kAlone>(cl, sh, r).bin = -1;
      }
    }
    sm_sync<Slice::kAlone>(cl);
    bin = sh.bin;
    if (bin < 0) return;  // fewer than k
    if (split) {
      lo += width * bin;
      hi = min(hi, lo + width - 1);
    }
    // ---- the bin's tokens to the first CTA
    sl.each(row, [&](float x, int id) {
      const u64 key = composite(x, id);
      if (!member(x, key)) return;
      const int at = atomicAdd(&lead.listed, 1);
      if (at < kSmList) lead.list[at] = key;
    });
    sm_sync<Slice::kAlone>(cl);
    const int n = lead.listed;
    if (n <= kSmList) {
      if (first) {
        int m = 32;
        while (m < n) m <<= 1;
        for (int i = n + tid; i < m; i += kSmThreads) sh.list[i] = ~0ull;
        __syncthreads();
        for (int size = 2; size <= m; size <<= 1)
          for (int d = size >> 1; d > 0; d >>= 1) {
            for (int i = tid; i < m / 2; i += kSmThreads) {
              const int a = 2 * i - (i & (d - 1)), b = a + d;
              const u64 ka = sh.list[a], kb = sh.list[b];
              if ((ka > kb) == ((a & size) == 0)) {
                sh.list[a] = kb;
                sh.list[b] = ka;
              }
            }
            __syncthreads();
          }
        // in order until the border is reached.  Weights are formed relative to the
        // list's largest, as the histogram's are to their bin's: pow2_by gives 0 below
        // 2^-60, where a top_p just below 1 may have its border
        constexpr int kEach = kSmList / kSmThreads;
        auto listed = [&](int i) { return row.exponent(falling_value(static_cast<unsigned>(sh.list[i] >> 32))); };
        const double most = kMass ? listed(0) : 0.0, unit = kMass ? pow2(most) : 1.0;
        double v[kEach], sum = 0.0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int i = tid * kEach + e;
          v[e] = i >= n ? 0.0 : kMass ? pow2_by(sh.powers, listed(i) - most) * unit : 1.0;
          sum += v[e];
        }
        double total;
        const SmSums<double> sums = sm_scan(sum, sh.warp_d, total);
        const double need = fmin(fmax(sh.target - sh.above, 1e-300), total * (1.0 - 0x1p-50));
        if (sm_passes(sums, need, &sh.pick)) {
          double before = sums.before;
          int at = tid * kEach;
#pragma unroll
          for (int e = 0; e + 1 < kEach; ++e)
            if (at == tid * kEach + e && before + v[e] < need) {
              before += v[e];
              ++at;
            }
          const u64 border = sh.list[min(at, n - 1)];
          for (int r = 0; r < ranks; ++r) sm_of<Slice::kAlone>(cl, sh, r).border = border;
        }
      }
      sm_sync<Slice::kAlone>(cl);
      row.keep_to(sh.border);
      return;
    }
    // ---- too many: the range from the smallest to the largest of them is split
    u64 least = ~0ull, most = 0;
    sl.each(row, [&](float x, int id) {
      const u64 key = composite(x, id);
      if (!member(x, key)) return;
      least = min(least, key);
      most = max(most, key);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    if ((tid & 31) == 0) {
      sh.warp_lo[tid >> 5] = least;
      sh.warp_hi[tid >> 5] = most;
    }
    __syncthreads();
    if (tid < ranks) {
      for (int w = 0; w < kSmWarps; ++w) {
        least = min(least, sh.warp_lo[w]);
        most = max(most, sh.warp_hi[w]);
      }
      SmShared& o = sm_of<Slice::kAlone>(cl, sh, tid);
      o.lo_of[cl.block_rank()] = least;
      o.hi_of[cl.block_rank()] = most;
    }
    sm_sync<Slice::kAlone>(cl);
    lo = ~0ull;
    hi = 0;
    for (int r = 0; r < ranks; ++r) {
      lo = min(lo, sh.lo_of[r]);
      hi = max(hi, sh.hi_of[r]);
    }
    width = (hi - lo) / kSmBins + 1;
    top = row.exponent(falling_value(static_cast<unsigned>(lo >> 32)));
    split = true;
  }
}

// The window of magnitudes that have a bin: [lo, lo + kSmValues).
struct SmWindow {
  int lo;
  __device__ __forceinline__ int place(unsigned b) const { return static_cast<int>(b & 0x7fffu) - lo; }
  __device__ __forceinline__ float value(int bin) const {
    return __uint_as_float(static_cast<unsigned>(lo + (bin & (kSmValues - 1))) << 16 | (bin & kSmValues ? 0x80000000u : 0u));
  }
  // Byte offsets of the bins (kBytes each) of a word's two logits, both halves at a
  // time.  What lies outside of the window, on either side, goes to its sign's last
  // bin; `least` takes the smallest magnitudes, for near().
  template <int kBytes>
  __device__ __forceinline__ void offsets(uint32_t w, unsigned& first, unsigned& second, uint32_t& least) const {
    static_assert(kSmValues * kBytes * 2 <= 1 << 16 && kSmValues == 1 << 11, "halves of 16 bits, the sign above the place");
    const uint32_t mags = w & 0x7fff7fffu;
    least = __vminu2(least, mags);
    const uint32_t minus = static_cast<uint32_t>(-lo & 0xffff) * 0x10001u;
    const uint32_t q = (__viaddmin_u16x2(mags, minus, (kSmValues - 1) * 0x10001u) | (w >> 4 & 0x08000800u)) * kBytes;
    first = q & 0xffffu;
    second = q >> 16;
  }
  // whether one of them lies nearer to zero than the window
  __device__ __forceinline__ bool near(uint32_t least) const { return static_cast<int>(min(least & 0xffffu, least >> 16)) < lo; }
};
// Bins in falling order of their values: the positive ones by falling magnitude,
// then the negative ones by rising magnitude.
__device__ __forceinline__ int sm_bin_at(int place) { return place < kSmValues ? kSmValues - 1 - place : place; }
constexpr int kSmZone = 2 * kSmValues;  // the place of what is nearer to zero than the window

// Counts the values of a vector.  -inf, and what is too far below the maximum to
// weigh anything, add to the last negative bin, which no other logit is in; what is
// nearer to zero than the window is listed (and counted in its sign's last bin).
__device__ __forceinline__ void sm_count(SmShared& sh, const SmWindow& win, const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  unsigned at[8];
  uint32_t least = 0x7fff7fffu;
#pragma unroll
  for (int i = 0; i < 4; ++i) win.offsets<4>(w[i], at[2 * i], at[2 * i + 1], least);
#pragma unroll
  for (int i = 0; i < 8; ++i) atomicAdd(reinterpret_cast<unsigned*>(reinterpret_cast<char*>(sh.values) + at[i]), 1u);
  if (win.near(least)) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = i < 2 ? u.x : i < 4 ? u.y : i < 6 ? u.z : u.w;
      const unsigned b = i & 1 ? x >> 16 : x & 0xffffu;
      if (win.place(b) < 0) {
        const int k = atomicAdd(&sh.near, 1);
        if (k < kSmNear) sh.near_of[k] = static_cast<unsigned short>(b);
      }
    }
  }
}
__device__ __forceinline__ void sm_clear(SmShared& sh) {
  for (int i = threadIdx.x; i < 2 * kSmValues / 4; i += kSmThreads)
    reinterpret_cast<uint4*>(sh.values)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (threadIdx.x == 0) sh.near = 0;
  __syncthreads();
}

// The border of top_k (0: none) and top_p (1: none) among bf16 logits, into what
// row keeps.  In order stand the positive values, the zone (what is nearer to zero
// than the window), the negative ones; each CTA of the cluster has a share of the
// bins.  Weights below 2^-60 count as 0 (pow2_by).  `counted`: sh.values holds the counts
// already.  All CTAs of the cluster call it and take the same way through it; false:
// the border lies in the zone and has to be searched.
template <typename Slice>
__device__ bool sm_values(const cg::cluster_group& cl, SmShared& sh, const Slice& sl, SmRow& row, const SmWindow& win,
                          bool counted, int top_k, double top_p) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ranks = Slice::kAlone ? 1 : cl.num_blocks(), rank = Slice::kAlone ? 0 : cl.block_rank();
  if (!counted) {
    sm_clear(sh);
    sl.vectors(0, sl.vecs, tid, kSmThreads, [&](const uint4& u, int) { sm_count(sh, win, u); });
  }
  __syncthreads();
  const int zones = sh.near;
  // (their sum is the same whatever order they were listed in: whole numbers of 2^-52)
  u64 near = 0;
  for (int k = tid; k < min(zones, kSmNear); k += kSmThreads) {
    const unsigned b = sh.near_of[k];
    near += static_cast<u64>(pow2_by(sh.powers, row.exponent(__uint_as_float(b << 16))) * 0x1p52);
    if (!(b & 0x8000u)) atomicSub(&sh.values[kSmValues - 1], 1u);  // it is not one of the largest
  }
  near = sm_sum(near);
  if (lane == 0) sh.warp_lo[warp] = near;
  if (tid < 2) sh.place_of[tid] = -1;
  __syncthreads();
  if (warp == 0) {
    near = sm_sum(lane < kSmWarps ? sh.warp_lo[lane] : 0ull);
    if (lane < ranks) {
      SmShared& o = sm_of<Slice::kAlone>(cl, sh, lane);
      o.zone_of[rank] = static_cast<double>(near) * 0x1p-52;
      o.zones_of[rank] = zones;
    }
  }
  sm_sync<Slice::kAlone>(cl);
  for (int r = 0; r < ranks; ++r)
    if (sh.zones_of[r] > kSmNear) return false;  // more than were listed
  // ---- this CTA's share of the bins: a thread's are neighbours in the order
  constexpr int kMost = 2 * kSmValues / kSmThreads;  // bins per thread of a whole row's CTA
  const int shift = Slice::kAlone ? 3 : __ffs(kMost / ranks) - 1, each = 1 << shift, share = 2 * kSmValues / ranks;  // (1, 2, 4 or 8 CTAs)
  static_assert(kMost == 8, "shift");
  const int place0 = rank * share + tid * each;
  int n[kMost + 1];
  double w[kMost + 1], mass[kMost + 1];
#pragma unroll
  for (int e = 0; e <= kMost; ++e) n[e] = 0;
  {
    unsigned got[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i)  // all loads in flight
      got[i] = sm_of<Slice::kAlone>(cl, sh, i >> shift).values[sm_bin_at(place0 + (i & (each - 1)))];
#pragma unroll
    for (int e = 0; e < kMost; ++e)
#pragma unroll
      for (int i = 0; i < kMost; ++i)
        if ((i & (each - 1)) == e) n[e] += static_cast<int>(got[i]);
  }
  if (place0 + each == 2 * kSmValues) {  // the last negative bin holds what does not count
#pragma unroll
    for (int e = 0; e < kMost; ++e)
      if (e == each - 1) n[e] = 0;
  }
  if (win.lo == 0) {  // -0 is 0: the first negative bin joins the last positive one
    const bool gets = place0 + each == kSmValues, gives = place0 == kSmValues;
    if (gets)
      for (int r = 0; r < ranks; ++r) {
        const int more = static_cast<int>(sm_of<Slice::kAlone>(cl, sh, r).values[kSmValues]);
#pragma unroll
        for (int e = 0; e < kMost; ++e)
          if (e == each - 1) n[e] += more;
      }
    if (gives) n[0] = 0;
  }
  int count = 0;
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < kMost; ++e) {
    w[e] = mass[e] = 0.0;
    count += n[e];
  }
  if (__any_sync(0xffffffffu, count != 0)) {  // most warps' bins are empty
#pragma unroll
    for (int e = 0; e < kMost; ++e) {
      if (e >= each) break;
      w[e] = pow2_by(sh.powers, row.exponent(fminf(win.value(sm_bin_at(place0 + e)), row.maxf)));
      mass[e] = n[e] * w[e];
      sum += mass[e];
    }
  }
  w[kMost] = mass[kMost] = 0.0;
  if (place0 + each == kSmValues) {  // the zone follows the last positive bin
    for (int r = 0; r < ranks; ++r) {
      mass[kMost] += sh.zone_of[r];
      n[kMost] += sh.zones_of[r];
    }
    count += n[kMost];
    sum += mass[kMost];
  }
  double mine;
  int held;
  SmSums<int> counts = sm_scan(count, sh.warp_n, held);
  SmSums<double> sums = sm_scan(sum, sh.warp_d, mine);
  if (tid < ranks) {
    SmShared& o = sm_of<Slice::kAlone>(cl, sh, tid);
    o.count_of[rank] = held;
    o.mass_of[rank] = mine;
  }
  sm_sync<Slice::kAlone>(cl);
  int all = 0, count_before = 0;
  double total = 0.0, mass_before = 0.0;
  for (int r = 0; r < ranks; ++r) {
    if (r == rank) {
      count_before = all;
      mass_before = total;
    }
    all += sh.count_of[r];
    total += sh.mass_of[r];
  }
  const double mass_after = mass_before + mine;
  counts.before += count_before;
  counts.upto += count_before;
  sums.before += mass_before;
  sums.upto += mass_before;
  // tells all CTAs border i: of a thread's bin e the first `ties` tokens are kept
  auto tell = [&](int i, int e, int ties, int of, double kept) {
    for (int r = 0; r < ranks; ++r) {
      SmShared& o = sm_of<Slice::kAlone>(cl, sh, r);
      o.place_of[i] = e == kMost ? kSmZone : place0 + e;
      o.ties_of[i] = ties;
      o.held_of[i] = of;
      o.sum_k = kept;
    }
  };
  double kept = total;
  if (top_k > 0 && top_k < all) {
    if (counts.before < top_k && top_k <= counts.upto) {  // one thread
      int c = counts.before;
      double m = sums.before;
      bool found = false;
#pragma unroll
      for (int e = 0; e <= kMost; ++e) {
        if (found) continue;
        found = c + n[e] >= top_k;
        if (found) tell(0, e, top_k - c, n[e], m + (top_k - c) * w[e]);
        c += n[e];
        m += mass[e];
      }
    }
    sm_sync<Slice::kAlone>(cl);
    if (sh.place_of[0] == kSmZone) return false;
    kept = sh.sum_k;
  }
  if (top_p < 1.0) {
    const double need = fmin(fmax(top_p * kept, 1e-300), total * (1.0 - 0x1p-50));
    if (mass_before < need && need <= mass_after && sm_passes(sums, need, &sh.pick)) {
      double m = sums.before;
      bool found = false;
#pragma unroll
      for (int e = 0; e <= kMost; ++e) {
        if (found || n[e] == 0) continue;
        found = m + mass[e] >= need;
        // (by rounding it may be none: then it is the thread's last)
        const double ties = w[e] > 0.0 ? fmin(fmax(ceil((need - m) / w[e]), 1.0), static_cast<double>(n[e])) : 1.0;
        tell(1, e, static_cast<int>(ties), n[e], kept);
        m += mass[e];
      }
    }
    sm_sync<Slice::kAlone>(cl);
    if (sh.place_of[1] == kSmZone) return false;
  }
  // ---- the first of the two
  const int pk = sh.place_of[0], pp = sh.place_of[1];
  if (pk < 0 && pp < 0) return true;
  const int i = pk < 0 || (pp >= 0 && pp < pk) ? 1 : 0;
  const int ties = pk == pp ? min(sh.ties_of[0], sh.ties_of[1]) : sh.ties_of[i];
  const float edge = win.value(sm_bin_at(sh.place_of[i]));
  row.least = edge;
  row.cut = ties < sh.held_of[i];
  row.ties = ties;
  row.last_id = row.cut ? -0x7fffffff - 1 : 0x7fffffff;
  return true;
}

// A weight (at most 1) in whole numbers of 2^-44, none below min_weight: the sum's
// low 52 bits.
__device__ __forceinline__ u64 sm_fixed(double w, double min_weight) {
  const u64 bits = static_cast<u64>(__double_as_longlong(fma(w, 0x1p44, 0x1p52))) & ((1ull << 52) - 1);
  return w >= min_weight ? bits : 0ull;
}

// The sum of a vector's kept weights, each formed for itself; id: of its first.
template <typename T>
__device__ __forceinline__ u64 sm_weigh_here(const uint4& d, int id, const SmRow& row, const double* powers) {
  constexpr int VE = 16 / sizeof(T);
  float e[VE];
  SmSlice<T, false, false>::unpack(d, e);
  u64 sum = 0;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const u64 x = sm_fixed(pow2_by(powers, row.exponent(e[i])), row.min_weight);
    sum += row.keeps(e[i], id + i) ? x : 0ull;
  }
  return sum;
}
__device__ __noinline__ u64 sm_weigh_rare(uint4 d, int id, SmRow row, const double* powers) {
  return sm_weigh_here<__nv_bfloat16>(d, id, row, powers);
}
template <typename T>
__device__ __forceinline__ u64 sm_weigh(const uint4& d, int id, const SmRow& row, const double* powers) {
  if constexpr (sizeof(T) == 2) return sm_weigh_rare(d, id, row, powers);  // near zero, or equal logits that are cut
  else return sm_weigh_here<T>(d, id, row, powers);
}

// Grid: a CTA (kAlone) or a cluster per row.
template <typename T, bool kStream, bool kAlone>
__global__ void __launch_bounds__(kSmThreads, 2) sample_tokens_kernel(const __grid_constant__ SmParams p) {
  using Slice = SmSlice<T, kStream, kAlone>;
  constexpr int VE = Slice::VE;
  extern __shared__ __align__(16) uint8_t sm_raw[];
  __shared__ __align__(16) SmShared sh;
  const cg::cluster_group cl = cg::this_cluster();
  const int ranks = kAlone ? 1 : cl.num_blocks(), rank = kAlone ? 0 : cl.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long r = blockIdx.x / ranks;
  if (!kAlone) cl.barrier_arrive();  // no CTA is written to before it runs
  if (tid < 64) sh.powers[tid] = pow2(tid * (1.0 / 64));
  pdl_launch_dependents();
  pdl_wait();

  // ---- the slice, from the 16-byte boundary at or below the row's first element on
  const T* const x = static_cast<const T*>(p.x) + r * p.row_stride;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const uint4* const row0 = reinterpret_cast<const uint4*>(x - mis);
  Slice sl;
  sl.V = p.V;
  sl.id0 = rank * p.slice - mis;
  sl.vecs = min(p.slice, max(0, p.V - sl.id0) + VE - 1) / VE;
  sl.in_lo = mis > 0;
  sl.in_n = max(0, (p.V - sl.id0) / VE - sl.in_lo);
  const uint4* const from = row0 + rank * (p.slice / VE);
  if constexpr (kStream) {
    sl.data = from;
  } else {
    uint4* const data = reinterpret_cast<uint4*>(sm_raw);
    sl.data = data;
    for (int v = tid; v < sl.vecs; v += kSmThreads) {
      const int id = sl.id0 + v * VE;
      if (id >= 0 && id + VE <= p.V) cp_async_16(smem_u32(data + v), from + v, 16);
      else data[v] = Slice::fetch(from + v, id, p.V);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const double temperature = p.temperature ? static_cast<double>(p.temperature[r]) : p.temperature_all;
  const long long top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const double top_p = p.top_p ? static_cast<double>(p.top_p[r]) : p.top_p_all;
  const double min_p = p.min_p ? static_cast<double>(p.min_p[r]) : p.min_p_all;
  const double u = p.u_f64 ? static_cast<const double*>(p.u)[r] : static_cast<double>(static_cast<const float*>(p.u)[r]);
  if constexpr (!kStream) asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- the largest logit (a NaN comes through), and of bf16 the smallest
  float mx = -INFINITY, mn = INFINITY;
  const bool by_k = top_k > 0 && top_k < p.V, by_p = top_p < 1.0;
  SmWindow win{0};
  bool counted = false;
  if constexpr (sizeof(T) == 2) {
    uint32_t high = 0xff80ff80u, low = 0x7f807f80u;
    auto look = [&](const uint4& d) {
      high = max_nan_bf16x2(high, max_nan_bf16x2(max_nan_bf16x2(d.x, d.y), max_nan_bf16x2(d.z, d.w)));
      low = min_bf16x2(low, min_bf16x2(min_bf16x2(d.x, d.y), min_bf16x2(d.z, d.w)));
    };
    if (kStream && (by_k || by_p) && temperature > 0.0 && top_k != 1) {
      // counts in the same pass, for magnitudes up to four times what a sample of the
      // row shows, and where it shows -inf for all that weigh something; where that was
      // too little they are counted again
      const int v = static_cast<int>(static_cast<long long>((p.V + mis + VE - 1) / VE) * tid / kSmThreads);
      const uint4 d = Slice::fetch(row0 + v, v * VE - mis, p.V);
      int most = 0;
      bool masked = false;
      const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int a = static_cast<int>(w[i >> 1] >> (16 * (i & 1)) & 0x7fffu);
        masked = masked || a == 0x7f80;
        if (a < 0x7f80) most = max(most, a);
      }
      if (masked) most = max(most, static_cast<int>(__float_as_uint(fminf(static_cast<float>(64.0 * temperature) * 0.6932f, 1e38f)) >> 16) - 255);
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) sh.warp_n[warp] = most;
      sm_clear(sh);
      most = __reduce_max_sync(0xffffffffu, lane < kSmWarps ? sh.warp_n[lane] : 0);
      win.lo = max(0, min(most + 256, 0x7f7f) - kSmValues + 1);
      sl.vectors(0, sl.vecs, tid, kSmThreads, [&](const uint4& u, int) {
        look(u);
        sm_count(sh, win, u);
      });
      counted = true;
    } else {
      sl.vectors(0, sl.vecs, tid, kSmThreads, [&](const uint4& u, int) { look(u); });  // what this thread copied
    }
    const float2 f = unpack_bf16x2(high), g = unpack_bf16x2(low);
    mx = max_nan(f.x, f.y);
    mn = fminf(g.x, g.y);
  } else {
    sl.vectors(0, sl.vecs, tid, kSmThreads, [&](const uint4& d, int) {
      float e[VE];
      Slice::unpack(d, e);
#pragma unroll
      for (int i = 0; i < VE; ++i) mx = max_nan(mx, e[i]);
    });
  }
  auto join = [&] {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (sizeof(T) == 2) mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
  };
  join();
  if (lane == 0) {
    sh.warp_f[warp] = mx;
    sh.warp_g[warp] = mn;
  }
  __syncthreads();
  if (!kAlone) cl.barrier_wait();
  if (warp == 0) {
    mx = lane < kSmWarps ? sh.warp_f[lane] : -INFINITY;
    mn = lane < kSmWarps ? sh.warp_g[lane] : INFINITY;
    join();
    if (lane < ranks) {
      SmShared& o = sm_of<kAlone>(cl, sh, lane);
      o.max_of[rank] = mx;
      o.min_of[rank] = mn;
    }
  }
  sm_sync<kAlone>(cl);
  mx = -INFINITY;
  mn = INFINITY;
  for (int q = 0; q < ranks; ++q) {
    mx = max_nan(mx, sh.max_of[q]);
    mn = fminf(mn, sh.min_of[q]);
  }
  if (!(fabsf(mx) < INFINITY) || !(temperature >= 0.0)) {  // no distribution
    if (rank == 0 && tid == 0) {
      p.tokens[r] = -1;
      p.logprob[r] = __int_as_float(0x7fc00000);
    }
    return;
  }

  if (temperature == 0.0 || top_k == 1) {  // the largest, the lowest id of equal ones
    int id = 0x7fffffff;
    sl.vectors(0, sl.vecs, tid, kSmThreads, [&](const uint4& d, int v) {
      float e[VE];
      Slice::unpack(d, e);
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (e[i] == mx) id = min(id, sl.id0 + v * VE + i);
    });
    id = __reduce_min_sync(0xffffffffu, id);
    if (lane == 0) sh.warp_n[warp] = id;
    __syncthreads();
    if (warp == 0) {
      id = __reduce_min_sync(0xffffffffu, lane < kSmWarps ? sh.warp_n[lane] : 0x7fffffff);
      if (lane == 0) sm_of<kAlone>(cl, sh, 0).count_of[rank] = id;
    }
    sm_sync<kAlone>(cl);
    if (rank == 0 && tid == 0) {
      for (int q = 0; q < ranks; ++q) id = min(id, sh.count_of[q]);
      p.tokens[r] = id;
      p.logprob[r] = 0.f;
    }
    return;
  }

  SmRow row;
  row.c = fmin(1.4426950408889634074 / temperature, 1e300);
  row.max = static_cast<double>(mx);
  row.maxf = mx;
  row.bins = static_cast<float>(fmin(row.c * kSmBinsPerOctave, 1e30));
  row.min_weight = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
  row.keep_all();
  bool search = by_k || by_p, plain = true;  // plain: the table holds all weights but the zone's
  if constexpr (sizeof(T) == 2) {
    // magnitudes up to beyond the largest of a negative logit that weighs 2^-64 or
    // more: the last negative bin is left to those that weigh nothing
    const float low = fmaxf(mn, static_cast<float>(row.max - fmin(64.0 / row.c, 1e38)));
    const int top = static_cast<int>((__float_as_uint(mx) & 0x7fffffffu) >> 16);
    const int down = low < 0.f ? static_cast<int>((__float_as_uint(low) & 0x7fffffffu) >> 16) + 1 : 0;
    plain = down <= 0x7f7f && 64.0 / row.c < 1e38;
    const int hi = min(max(top, down), 0x7f7f);
    counted = counted && hi <= win.lo + kSmValues - 1;
    if (!counted) win.lo = max(0, hi - kSmValues + 1);
    if (search && plain && sm_values(cl, sh, sl, row, win, counted, by_k ? static_cast<int>(top_k) : 0, top_p))
      search = false;
  }
  if (search) {
    row.keep_all();
    if (by_k) sm_select<false>(cl, sh, sl, row, static_cast<double>(top_k));
    if (by_p) sm_select<true>(cl, sh, sl, row, top_p);
  }

  // what weighs less than min_p need not be looked at: a bound a little below it, by
  // 2^-30 of a binary order and the rounding of the logit (the weights themselves decide)
  if (row.min_weight > 0.0) {
    float bound = static_cast<float>(row.max + (log2(row.min_weight) - 0x1p-30) / row.c);
    bound -= fabsf(bound) * 0x1p-22f + 1e-30f;
    if (bound > row.least) {
      row.least = bound;
      row.last_id = 0x7fffffff;
      row.cut = false;
      if (sizeof(T) == 2 && bound > 0.f) row.least = __uint_as_float(__float_as_uint(bound) & 0xffff0000u);
    }
  }

  // ---- the kept weights' sums, a warp's vectors being neighbours: whole numbers
  // of 2^-44 of the largest weight, so 2^18 of them fit 64 bits and add up alike
  // in any order.  bf16 weights come from a table.
  if constexpr (sizeof(T) == 2) {
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < 2 * kSmValues; i += kSmThreads) {  // (a warp's bins are neighbours: mostly all or none)
      const float x = win.value(i);
      u64 w = 0;
      if (x >= row.least && x <= mx && i != 2 * kSmValues - 1 && !(row.cut && x == row.least)) w = sm_fixed(pow2_by(sh.powers, row.exponent(x)), row.min_weight);
      sh.weights[i] = make_uint2(static_cast<unsigned>(w) & 0x3fffffu, static_cast<unsigned>(w >> 22));
    }
    __syncthreads();
  }
  auto some = [&](const uint4& d) {  // whether any of a vector may be kept
    if constexpr (sizeof(T) == 2) {
      const float2 f = unpack_bf16x2(max_nan_bf16x2(max_nan_bf16x2(d.x, d.y), max_nan_bf16x2(d.z, d.w)));
      return fmaxf(f.x, f.y) >= row.least;
    } else {
      return fmaxf(fmaxf(__uint_as_float(d.x), __uint_as_float(d.y)), fmaxf(__uint_as_float(d.z), __uint_as_float(d.w))) >= row.least;
    }
  };
  const uint32_t edge2 = pack_bf16x2(row.least, row.least);  // (bf16 only)
  auto sum_of = [&](const uint4& d, int v) {
    u64 sum = 0;
    if (!some(d)) return sum;
    if constexpr (sizeof(T) == 2) {
      const uint32_t x[4] = {d.x, d.y, d.z, d.w};
      unsigned at[8];
      uint32_t least = 0x7fff7fffu;
#pragma unroll
      for (int i = 0; i < 4; ++i) win.offsets<8>(x[i], at[2 * i], at[2 * i + 1], least);
      const int id = sl.id0 + v * VE;
      bool ties = false;  // cut within this vector
      if (!row.cut && id + VE - 1 > row.last_id && row.least > -INFINITY) {  // behind the last equal logit that is kept, if not before its vector's end
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t q;
          asm("set.eq.u32.bf16x2 %0, %1, %2;" : "=r"(q) : "r"(x[i]), "r"(edge2));
          m |= q;
        }
        ties = m != 0;
      }
      if (plain && !win.near(least) && !ties) {
        unsigned low = 0, high = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(sh.weights) + at[i]);
          low += w.x;
          high += w.y;
        }
        return low + (static_cast<u64>(high) << 22);
      }
    }
    return sm_weigh<T>(d, sl.id0 + v * VE, row, sh.powers);
  };
  // equal logits that are cut weigh nothing there and are counted (masks of 16 bits
  // are added: a equal ones in the words' low halves and c in the high ones give
  // (a - c) 2^16 - a)
  const u64 edge = row.cut ? sm_fixed(pow2_by(sh.powers, row.exponent(row.least)), row.min_weight) : 0ull;
  auto equal = [&](const uint4& d) {
    return equal_bf16x2(d.x, edge2) + equal_bf16x2(d.y, edge2) + equal_bf16x2(d.z, edge2) + equal_bf16x2(d.w, edge2);
  };
  auto equals = [](uint32_t masks) {
    const uint32_t a = -masks & 0xffffu;
    return static_cast<int>(a + ((a - ((masks + a) >> 16)) & 0xffffu));
  };
  constexpr int kGroup = kStream ? 32 / VE : 1;  // vectors of a lane in a group
  constexpr int kAtOnce = kStream ? 4 : 1;
  constexpr int kSliceVecs = kSmMaxVocab / VE / kSmCluster + 1 > kSmSlice / 16 ? kSmMaxVocab / VE / kSmCluster + 1 : kSmSlice / 16;
  constexpr int kMostVecs = kStream ? kSmMaxVocab / VE + 1 : kSliceVecs;
  static_assert((kMostVecs + kSmWarps - 1) / kSmWarps <= kSmGroups * 32 * kGroup && kSmWarps * kSmGroups <= kSmThreads, "groups");
  const int per = (sl.vecs + kSmWarps - 1) / kSmWarps;
  const int v_lo = min(sl.vecs, warp * per), v_hi = min(sl.vecs, v_lo + per);
  if (lane < kSmGroups) {
    sh.group_sum[warp * kSmGroups + lane] = 0;
    sh.group_ties[warp * kSmGroups + lane] = 0;
  }
  __syncwarp();
  // where only positive logits of the window are kept: as signed numbers, what is below
  // them reads the one bin before the border's, which holds 0, so lanes that keep
  // nothing share an access
  const int edge_place = win.place(__float_as_uint(row.least) >> 16);
  const bool high_only =
      sizeof(T) == 2 && plain && row.least > 0.f && edge_place > 0 && (row.cut || row.last_id == 0x7fffffff);
  const uint32_t low2 = static_cast<uint32_t>(win.lo + edge_place - 1) * 0x10001u, lo2 = static_cast<uint32_t>(win.lo) * 0x10001u;
  auto weigh = [&](float x) { return sm_fixed(pow2_by(sh.powers, row.exponent(x)), row.min_weight); };
  int waiting = 0;  // of this warp's logits in sh.kept (fp32 only)
  for (int g = 0, v0 = v_lo; v0 < v_hi; ++g, v0 += 32 * kGroup) {
    u64 sum = 0;
    uint32_t masks = 0;
#pragma unroll
    for (int a0 = 0; a0 < kGroup; a0 += kAtOnce) {
      uint4 d[kAtOnce];
      const int v = v0 + a0 * 32 + lane;
      if (v0 + (a0 + kAtOnce) * 32 <= v_hi) {
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a) d[a] = sl.raw(v + a * 32);
      } else {  // -inf behind the part
        const unsigned none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a) d[a] = v + a * 32 < v_hi ? sl.raw(v + a * 32) : make_uint4(none, none, none, none);
      }
      if (high_only) {
        unsigned low = 0, high = 0;
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a) {
          const uint32_t w[4] = {d[a].x, d[a].y, d[a].z, d[a].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t at = (__vmaxs2(w[i], low2) - lo2) * 8u;
            const uint2 e = *reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(sh.weights) + (at & 0xffffu));
            const uint2 f = *reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(sh.weights) + (at >> 16));
            low += e.x + f.x;
            high += e.y + f.y;
          }
        }
        sum += low + (static_cast<u64>(high) << 22);
      } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a) {
          sum += sum_of(d[a], v + a * 32);
          __syncwarp();
        }
      } else {
        // a weight is a chain of 600 cycles: where a warp's vectors keep few, 32 of
        // them are weighed at a time (257 rows with min-p 21 us, and 26 one vector at a time, the
        // row that keeps most being what the others wait for)
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a) {
          if (!__any_sync(0xffffffffu, some(d[a]))) continue;
          float e[VE];
          Slice::unpack(d[a], e);
          unsigned who[VE];
          int n = row.least > -INFINITY ? 0 : 32 * VE;  // (nothing is cut: hardly few)
          if (n == 0) {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
              who[i] = __ballot_sync(0xffffffffu, row.keeps(e[i], sl.id0 + (v + a * 32) * VE + i));
              n += __popc(who[i]);
            }
          }
          if (n > kSmFew) {
            sum += sm_weigh<T>(d[a], sl.id0 + (v + a * 32) * VE, row, sh.powers);
            continue;
          }
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            if (who[i] >> lane & 1u) sh.kept[warp][waiting + __popc(who[i] & ((1u << lane) - 1u))] = e[i];
            waiting += __popc(who[i]);
          }
          __syncwarp();
          while (waiting >= 32) {
            waiting -= 32;
            sum += weigh(sh.kept[warp][waiting + lane]);
          }
          __syncwarp();
        }
      }
      if (sizeof(T) == 2 && row.cut) {
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a) masks += equal(d[a]);
      }
    }
    if (sizeof(T) == 4 && waiting > 0) {
      if (lane < waiting) sum += weigh(sh.kept[warp][lane]);
      waiting = 0;
      __syncwarp();
    }
    // (a lane's weights, 32 or at most 48 in all lanes more: 50 bits)
    const u64 low = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(sum) & 0x3ffffffu);
    const u64 high = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(sum >> 26));
    if (lane == 0) sh.group_sum[warp * kSmGroups + g] = low + (high << 26);
    if (sizeof(T) == 2 && row.cut) {
      const int ties = __reduce_add_sync(0xffffffffu, equals(masks));
      if (lane == 0) sh.group_ties[warp * kSmGroups + g] = ties;
    }
  }
  __syncthreads();
  const u64 group = tid < kSmWarps * kSmGroups ? sh.group_sum[tid] : 0ull;
  const int group_ties = tid < kSmWarps * kSmGroups ? sh.group_ties[tid] : 0;
  u64 mine;
  int own = 0;
  SmSums<u64> sums = sm_scan(group, sh.warp_lo, mine);
  SmSums<int> ties{0, 0};
  if (row.cut) ties = sm_scan(group_ties, sh.warp_n, own);
  if (tid < ranks) {
    SmShared& o = sm_of<kAlone>(cl, sh, tid);
    o.sum_of[rank] = mine;
    o.zones_of[rank] = own;
  }
  sm_sync<kAlone>(cl);

  // ---- the CTA, the group, the vector and the token where the running sum passes
  // u S; for a u outside of [0, 1) the first or the last that is kept
  u64 whole = 0;
  int had = 0;  // equal logits before
  auto kept_ties = [&](int n, int before) { return row.cut ? max(0, min(n, row.ties - before)) : 0; };
  u64 before = 0;
  int before_ties = 0;
  for (int q = 0; q < ranks; ++q) {
    if (q == rank) {
      before = whole;
      before_ties = had;
    }
    whole += sh.sum_of[q] + edge * static_cast<u64>(kept_ties(sh.zones_of[q], had));
    had += sh.zones_of[q];
  }
  const double part = u * static_cast<double>(whole);
  const u64 goal = part >= static_cast<double>(whole) || part != part ? whole - 1 : part > 0.0 ? min(static_cast<u64>(part), whole - 1) : 0ull;
  const u64 here = mine + edge * static_cast<u64>(kept_ties(own, before_ties));
  if (goal < before || goal - before >= here) return;
  // of the threads' parts, in order, the one that holds the goal
  auto choose = [&](u64 part, int n, SmSums<u64> sums, SmSums<int> ties) {
    if (row.cut) {
      part += edge * static_cast<u64>(kept_ties(n, before_ties + ties.before));
      u64 all;
      sums = sm_scan(part, sh.warp_lo, all);
    }
    if (before + sums.before <= goal && goal < before + sums.upto) {
      sh.part = tid;
      sh.part_before = before + sums.before;
      sh.part_ties = before_ties + ties.before;
    }
    __syncthreads();
    before = sh.part_before;
    before_ties = sh.part_ties;
    return sh.part;
  };
  const int at = choose(group, group_ties, sums, ties);
  const int g_lo = min(sl.vecs, at / kSmGroups * per) + at % kSmGroups * 32 * kGroup;
  const int g_hi = min(min(sl.vecs, (at / kSmGroups + 1) * per), g_lo + 32 * kGroup);
  u64 vector = 0;
  int vector_ties = 0;
  if (g_lo + tid < g_hi) {
    const uint4 d = sl.raw(g_lo + tid);
    vector = sum_of(d, g_lo + tid);
    if (sizeof(T) == 2 && row.cut) vector_ties = equals(equal(d));
  }
  u64 all;
  int some_ties;
  if (row.cut) ties = sm_scan(vector_ties, sh.warp_n, some_ties);
  else sums = sm_scan(vector, sh.warp_lo, all);
  const int v = g_lo + choose(vector, vector_ties, sums, ties);
  if (warp == 1 && lane == 0) sh.warp_d[0] = log(static_cast<double>(whole) * 0x1p-44);
  if (warp == 0) {  // its logits, one a lane
    const int id = sl.id0 + v * VE + lane;
    float x = -INFINITY;
    if (lane < VE && id >= 0 && id < p.V) x = static_cast<float>(reinterpret_cast<const T*>(sl.data)[v * VE + lane]);
    u64 w = row.keeps(x, id) ? sm_fixed(pow2_by(sh.powers, row.exponent(x)), row.min_weight) : 0ull;
    const unsigned equal_ones = __ballot_sync(0xffffffffu, row.cut && x == row.least);
    if ((equal_ones >> lane & 1u) && before_ties + __popc(equal_ones & ((1u << lane) - 1u)) < row.ties) w = edge;
    u64 upto = w;
#pragma unroll
    for (int o = 1; o < VE; o <<= 1) {
      const u64 q = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += q;
    }
    if (lane < VE && before + upto - w <= goal && goal < before + upto) {
      p.tokens[r] = id;
      sh.warp_d[1] = row.exponent(x) * 0.69314718055994530942;  // the weight itself, not its whole number
    }
  }
  __syncthreads();
  if (tid == 0) p.logprob[r] = static_cast<float>(sh.warp_d[1] - sh.warp_d[0]);
}

template <typename T>
cudaError_t sm_launch(const SmParams& params, long long rows, cudaStream_t s) {
  constexpr int VE = 16 / sizeof(T);
  SmParams p = params;
  const long long vecs = (static_cast<long long>(p.V) + VE - 1 + VE - 1) / VE;  // a row may begin inside a vector
  // as few CTAs per row as hold it at two per SM; more where rows are few
  int ranks = 1;
  while (ranks < kSmCluster && ((vecs + ranks - 1) / ranks) * 16 > kSmSlice) ranks *= 2;
  while (ranks < kSmCluster && rows * ranks < device_sm_count() && vecs > 64 * ranks) ranks *= 2;
  // where they do not all run at once, rows stay where they are, with as many CTAs as do:
  // 100 rows of 151936 bf16 with top-p take 46 us so, as slices of four CTAs each, in two
  // rounds, 58; 70 rows, whose slices fit, 33 us as slices
  const long long room = 2 * device_sm_count();
  // (bf16 rows do from one per SM on even where slices would fit: of 18000 with filters, 150 of
  // them: 23.1 us, as slices 25.7; fp32 rows of 500: 11.3 and 6.6 us, of 18000 20.2 and 17.3)
  const bool stream = rows * ranks > room || (sizeof(T) == 2 && rows >= device_sm_count());
  if (stream) ranks = kSmCluster;
  while (stream && ranks > 1 && rows * ranks > room) ranks /= 2;
  const bool alone = stream && ranks == 1;
  p.slice = static_cast<int>((vecs + ranks - 1) / ranks) * VE;
  const size_t smem = stream ? 0 : static_cast<size_t>(p.slice) * sizeof(T);
  constexpr int kMost = kSmMaxVocab * sizeof(T) / kSmCluster;
  cudaError_t e = allow_smem<sample_tokens_kernel<T, false, false>>((kMost > kSmSlice ? kMost : kSmSlice) + 64);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ranks));
  cfg.blockDim = dim3(kSmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  if (alone) return cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T, true, true>, p);
  if (stream) return cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T, true, false>, p);
  return cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T, false, false>, p);
}

}  // namespace

cudaError_t sample_tokens_launch(const void* logits, int dtype, long long row_stride, const void* uniforms, bool u_f64,
                                 const SampleSettings& set, long long rows, long long V, long long* tokens,
                                 float* logprob, cudaStream_t s) {
  SmParams p{};
  p.x = logits;
  p.row_stride = row_stride;
  p.u = uniforms;
  p.u_f64 = u_f64;
  p.temperature = set.temperature;
  p.top_k = set.top_k;
  p.top_p = set.top_p;
  p.min_p = set.min_p;
  p.temperature_all = set.temperature_all;
  p.top_k_all = set.top_k_all;
  p.top_p_all = set.top_p_all;
  p.min_p_all = set.min_p_all;
  p.tokens = tokens;
  p.logprob = logprob;
  p.V = static_cast<int>(V);
  return dtype == kF32 ? sm_launch<float>(p, rows, s) : sm_launch<__nv_bfloat16>(p, rows, s);
}

}  // namespace nkimoe
