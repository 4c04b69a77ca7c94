// Shared by the kernels of the paged key-value cache: the cache's layout, the
// rotary angles taken in 64 bits, and the q/k norms of half-warp heads.
//
// A layer's cache is two pools [num_pages, nkv, page_size, 128] (bf16; a
// page's [nkv, page_size, 128] block is contiguous, the pages may be any
// 8-element multiple apart), and row b of the page table lists the pages of
// sequence b: position s lives in page table[b][s / page_size], row
// s % page_size.  -1 marks a page that is not held.
#pragma once

#include <atomic>

#include "kernels.h"
#include "rope.cuh"

namespace nkimoe {

// Workspace of these kernels: a status word, counters that are zero between
// calls, then scratch.  The first two have a fixed size, so calls of any of
// the kernels and any shape may share one workspace on a stream.
constexpr size_t kPagedStatusBytes = 256;
constexpr int kPagedCounters = 8192;
constexpr size_t kPagedScratch = kPagedStatusBytes + sizeof(int) * kPagedCounters;

struct PagedCache {
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  long long k_stride, v_stride;  // elements between pages
  const int* table;              // [B, max_pages]
  long long table_stride;
  int max_pages, num_pages, nkv;
  int page_shift;  // log2 of the page size
};

// theta^(-i/64) / (2 pi): turns per position of each rotary frequency.  The
// angle of a far position needs more bits than fp32 has (at position 10^5 an
// fp32 angle is off by up to 4e-3 rad), so it is formed and reduced to a
// fraction of a turn in 64 bits; the sine and cosine themselves are fp32.
struct RopeTurns {
  double f[kHeadDim / 2];
};

__device__ __forceinline__ float2 rope_cos_sin(double turns_per_pos, long long pos) {
  double t = turns_per_pos * static_cast<double>(pos);
  t -= rint(t);
  float sn, cs;
  sincospif(static_cast<float>(2.0 * t), &sn, &cs);
  return make_float2(cs, sn);
}

// Whether the query at position p sees the key at position s.
__device__ __forceinline__ bool key_visible(int s, int p, int window, int sinks) {
  return s <= p && (window == 0 || s > p - window || s < sinks);
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                    pack_bf16x2(v[6], v[7]));
}

// Two fp32 operations in one instruction (sm_100).
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x to 2 ulp, subnormal results as 0 (ex2 of the hardware).
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A head held by a half-warp: lane l of the sixteen owns elements [4l, 4l + 4)
// and their rotate-half partners [64 + 4l, 64 + 4l + 4), each as two pairs, so
// the rotation needs no other lane.
struct HeadPart {
  uint64_t a[2], b[2];
};

__device__ __forceinline__ uint64_t pair_of_bf16x2(uint32_t u) {
  return pair2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ HeadPart part_of_rows(const uint2& lo, const uint2& hi) {
  return HeadPart{{pair_of_bf16x2(lo.x), pair_of_bf16x2(lo.y)}, {pair_of_bf16x2(hi.x), pair_of_bf16x2(hi.y)}};
}
__device__ __forceinline__ uint32_t bf16x2_of_pair(uint64_t v) {
  const float2 f = split2(v);
  return pack_bf16x2(f.x, f.y);
}
__device__ __forceinline__ uint2 row_of_pairs(const uint64_t (&v)[2]) {
  return make_uint2(bf16x2_of_pair(v[0]), bf16x2_of_pair(v[1]));
}

// The lane's norm weights.
__device__ __forceinline__ HeadPart load_weight_part(const void* w, int w_dtype, int l) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[e] = head_wload(w, w_dtype, l * 4 + e);
    f[4 + e] = head_wload(w, w_dtype, 64 + l * 4 + e);
  }
  return HeadPart{{pair2(f[0], f[1]), pair2(f[2], f[3])}, {pair2(f[4], f[5]), pair2(f[6], f[7])}};
}

// cos, sin and -sin of frequencies 4l .. 4l + 3, as two pairs each.
struct TurnPart {
  uint64_t c[2], s[2], ms[2];
};
__device__ __forceinline__ TurnPart turn_part(const float2* tab, int l) {
  TurnPart t;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float2 x = tab[l * 4 + 2 * e], y = tab[l * 4 + 2 * e + 1];
    t.c[e] = pair2(x.x, y.x);
    t.s[e] = pair2(x.y, y.y);
    t.ms[e] = pair2(-x.y, -y.y);
  }
  return t;
}

// RMSNorm of the head times the weights, then rotate-half RoPE, times `scale`:
// the rotation is linear, so the norm's factor comes last.  All 32 lanes of
// the warp call it.
__device__ __forceinline__ HeadPart norm_rope_part(const HeadPart& x, const HeadPart& w, const TurnPart& t, float eps,
                                                   float scale = 1.f) {
  uint64_t sq = mul2(x.a[0], x.a[0]);
  sq = fma2(x.a[1], x.a[1], sq);
  sq = fma2(x.b[0], x.b[0], sq);
  sq = fma2(x.b[1], x.b[1], sq);
  const float2 q = split2(sq);
  float ss = q.x + q.y;
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
  const float r = rsqrtf(ss * (1.f / kHeadDim) + eps) * scale;
  const uint64_t r2 = pair2(r, r);
  HeadPart o;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint64_t a = mul2(x.a[e], w.a[e]), b = mul2(x.b[e], w.b[e]);
    o.a[e] = mul2(fma2(b, t.ms[e], mul2(a, t.c[e])), r2);
    o.b[e] = mul2(fma2(a, t.s[e], mul2(b, t.c[e])), r2);
  }
  return o;
}

// Keys are kept rounded, so a sum in fp32 that falls on the other side of the
// middle between two bf16 values stays one bf16 step off for good (more than half
// a step from the formula's value).  key_near_tie says which
// of the lane's rotated pairs (bit e: elements 4l + e and 64 + 4l + e) lie that
// near to a middle, by 2^-23 of the pair's length, which the rotation keeps: one
// head in 60 has one.  Those are formed again by key_in_64_bits.  Of 361 values in
// 12 million that fp32 alone rounds to the other side 2 are left (none with
// 2^-22, 61 with 2^-24).
__device__ __forceinline__ uint32_t key_near_tie(const HeadPart& o) {
  uint32_t near = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = split2(o.a[i]), b = split2(o.b[i]);
    const float av[2] = {a.x, a.y}, bv[2] = {b.x, b.y};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float e = (fabsf(av[k]) + fabsf(bv[k])) * 0x1p-23f;
      const float am = __uint_as_float((__float_as_uint(av[k]) & 0xffff0000u) | 0x8000u);
      const float bm = __uint_as_float((__float_as_uint(bv[k]) & 0xffff0000u) | 0x8000u);
      if (fabsf(av[k] - am) < e || fabsf(bv[k] - bm) < e) near |= 1u << (2 * i + k);
    }
  }
  return near;
}

// The pairs of `which` (any lane's) of a head, from its bf16 elements lo and hi
// into its rounded key klo and khi; a half-warp per head, all 32 lanes call it.
// w: the lane's first weight, of 128 in fp32.
__device__ __noinline__ static void key_in_64_bits(uint32_t which, uint2 lo, uint2 hi, const float* w,
                                                   const double* turns, int l, int pos, float eps, uint2& klo,
                                                   uint2& khi) {
  const uint32_t words[4] = {lo.x, lo.y, hi.x, hi.y};
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double x = __uint_as_float(words[i] << 16), y = __uint_as_float(words[i] & 0xffff0000u);
    ss += x * x + y * y;
  }
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
  const double r = rsqrt(ss * (1.0 / kHeadDim) + static_cast<double>(eps));
  which = __reduce_or_sync(0xffffffffu, which);
#pragma unroll 1
  for (int e = 0; e < 4; ++e) {
    if (!((which >> e) & 1u)) continue;
    const bool second = e & 2;
    const uint32_t sh = e & 1 ? 16 : 0, keep = e & 1 ? 0xffffu : 0xffff0000u;
    const uint32_t ua = second ? lo.y : lo.x, ub = second ? hi.y : hi.x;
    const double a = static_cast<double>(__uint_as_float(ua >> sh << 16)) * w[e];
    const double b = static_cast<double>(__uint_as_float(ub >> sh << 16)) * w[64 + e];
    double t = turns[4 * l + e] * static_cast<double>(pos), sn, cs;
    t -= rint(t);
    sincospi(2.0 * t, &sn, &cs);
    const uint32_t ra = __bfloat16_as_ushort(__float2bfloat16_rn(static_cast<float>((a * cs - b * sn) * r)));
    const uint32_t rb = __bfloat16_as_ushort(__float2bfloat16_rn(static_cast<float>((b * cs + a * sn) * r)));
    uint32_t& wa = second ? klo.y : klo.x;
    uint32_t& wb = second ? khi.y : khi.x;
    wa = (wa & keep) | ra << sh;
    wb = (wb & keep) | rb << sh;
  }
}

// Lets a kernel take `bytes` of dynamic shared memory, once per device.
template <auto kKernel>
cudaError_t allow_smem(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// ----------------------------------------------------------------- launches
RopeTurns rope_turns(float theta);

cudaError_t paged_store_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                               const int* cu_seqlens, const int* kv_lens, const PagedCache& cache,
                               __nv_bfloat16* q_out, long long T, int B, int nq, float theta, float eps, int* status,
                               cudaStream_t s);

cudaError_t copy_pages_launch(void* pages, long long planes, long long plane_bytes, long long page_bytes,
                              const int* src, const int* dst, long long n, cudaStream_t s);

size_t paged_decode_workspace_bytes(long long B, int nq, int nkv, long long max_pages, int page_size);
cudaError_t paged_decode_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                                const long long* positions, long long pos_stride, const PagedCache& cache,
                                __nv_bfloat16* out, int B, int nq, float theta, float eps, float scale, int window,
                                int sinks, void* workspace, cudaStream_t s);

size_t paged_prefill_workspace_bytes(long long T, long long B, int nq, int nkv, long long max_pages, int page_size);
cudaError_t paged_prefill_launch(const __nv_bfloat16* q, long long q_stride, const int* cu_seqlens,
                                 const int* kv_lens, const PagedCache& cache, __nv_bfloat16* out, long long T, int B,
                                 int nq, float scale, int window, int sinks, void* workspace, cudaStream_t s);

size_t token_logprobs_workspace_bytes(long long T, long long V, int top_n);
cudaError_t token_logprobs_launch(const void* logits, int dtype, long long row_stride, const long long* tokens,
                                  long long T, long long V, int top_n, float* logprob, float* entropy, float* top_lp,
                                  long long* top_ids, void* workspace, cudaStream_t s);

}  // namespace nkimoe
