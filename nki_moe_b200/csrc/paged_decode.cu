// Attention of one new token per sequence over a paged key-value cache
// (grouped-query attention, head_dim 128), fused with what feeds it: the q/k
// RMSNorm + rotate-half RoPE of the new token and the store of its key and
// value into its page.  Optionally a sliding window with a few first
// positions that stay visible.
//
//   out = sum_s softmax_s(q . k_s * scale) v_s  over the visible s
//
// Reference: nki_attention.py:252-373 (one query token against the cached
// keys/values, online softmax :333-359) and the attention block of
// qwen_with_nki.py:330-350 (per-head q/k norms, then RoPE).
//
// Split: the batch's visible positions, in granules of 64, form one list over
// (sequence, kv head, granule), each (sequence, kv head) preceded by places
// that stand for its own cost, and every CTA takes an equal run of it, so a
// batch of any mix of lengths loads all SMs alike and the launch needs no
// length on the host.  A (sequence, kv head) whose granules fall to several
// CTAs leaves one partial (m, l, o) per CTA; the last of them to finish
// (device-scope counter, no spinning) joins them in order.
//
// Arithmetic: S = Q K^T and O += P V as warp MMAs (m16n8k16, bf16 in, fp32
// accumulate), each warp on 16 positions of its own with its own ring of
// cp.async stages, so the loop has no CTA barrier.  Queries and weights enter
// the MMAs as a sum of two bf16 (hi + lo), which keeps their rounding (2^-17)
// below the output's (2^-8): up to 8 heads per kv head the lo parts take the
// MMA's 8 rows that would idle, at no cost.
//
// Bound by HBM where the cache is large, by the chain of latencies (positions,
// pages, keys, join) where it is small.  Measured (32 heads over 4): 48 ragged
// sequences of 1 to 32768 positions 64 us = 5.3 TB/s = 0.81 of the measured
// copy; 24 streams with a window of 2048 23.5 us = 4.2 TB/s; 8 sequences of 512
// to 639 positions 11.7 us.  With 16 heads per kv head (the lo parts are MMAs of
// their own): 70, 32 and 14.4 us.
#include "paged.cuh"

namespace nkimoe {

namespace {

constexpr int kPdWarps = 4;
constexpr int kPdThreads = kPdWarps * 32;
constexpr int kPdTile = 16;                     // positions per warp step
constexpr int kPdGran = kPdWarps * kPdTile;     // positions per granule
constexpr int kPdStages = 3;
constexpr int kPdRow = kHeadDim;                // elements per staged row (swizzled, unpadded)
constexpr int kPdStage = 2 * kPdTile * kPdRow;  // elements per stage: K and V
constexpr int kPdPart = 132;                    // floats per partial and head: o[128], m, l, pad
constexpr int kPdCtasPerSm = 2;
constexpr int kPdItem = 6;                      // granules that beginning and ending an item costs:
                                                // 48 ragged sequences 98 us at 0, 75 at 2, 64 at 6 and 8
constexpr float kPdLog2e = 1.4426950408889634f;
constexpr int kPdMaxBatch = 4096;
constexpr int kPdQRow = kHeadDim + 8;           // padded query row (conflict-free ldmatrix)

struct PdParams {
  const __nv_bfloat16* qkv;  // [B, (nq + 2 nkv) * 128]
  const void* qw;
  const void* kw;
  const long long* positions;
  __nv_bfloat16* out;  // [B, nq * 128]
  int* status;
  int* counters;
  float* part;  // [2 * grid, grp, kPdPart]
  PagedCache c;
  RopeTurns turns;
  long long pos_stride;
  int w_dtype, B, nq, grp, window, sinks;
  float eps, scale_log2;
};

__device__ __forceinline__ void pd_ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void pd_ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// D[16x8] += A[16x16] B[16x8], bf16 in, fp32 accumulate
__device__ __forceinline__ void pd_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The granules of a sequence whose query stands at pos: those of the first
// `sinks` positions, then those from the window's first on.
struct Granules {
  int sink;   // granules 0 .. sink - 1
  int first;  // then granule `first` and what follows
  int n;
};
__device__ __forceinline__ Granules granules_of(int pos, int window, int sinks) {
  Granules g;
  const int start = window && pos >= window ? pos - window + 1 : 0;  // the window's first position
  g.first = start / kPdGran;
  g.sink = start > 0 ? min((min(sinks, start) + kPdGran - 1) / kPdGran, g.first) : 0;
  g.n = g.sink + pos / kPdGran - g.first + 1;
  return g;
}

// A valid position of sequence b, or -1 for an idle row (a negative position,
// or one that the page table has no place for, which is flagged).
__device__ __forceinline__ int pd_position(const PdParams& p, int b, bool flag) {
  const long long pos = p.positions[b * p.pos_stride];
  if (pos < 0) return -1;
  if (pos >= (static_cast<long long>(p.c.max_pages) << p.c.page_shift)) {
    if (flag) atomicOr(p.status, kDevErrBadIndex);
    return -1;
  }
  return static_cast<int>(pos);
}

template <bool kWide>  // 9 to 16 heads per kv head
struct PdShared {
  __nv_bfloat16 stage[kPdWarps][kPdStages][kPdStage];
  __nv_bfloat16 q[kWide ? 2 : 1][16][kPdQRow];  // narrow: rows 0-7 hi, 8-15 lo; wide: hi, lo
  __align__(16) __nv_bfloat16 knew[kHeadDim], vnew[kHeadDim];
  float2 tab[kHeadDim / 2];
  float kw[kHeadDim];  // key norm weights, for a key that is done again
  float ml[kPdWarps][16][2];
  int warp_sum[kPdWarps];
  int last;
};

template <bool kWide>
__global__ void __launch_bounds__(kPdThreads, kPdCtasPerSm)
    paged_decode_kernel(const __grid_constant__ PdParams p) {
  constexpr int D = kHeadDim;
  extern __shared__ __align__(128) uint8_t pd_smem[];
  PdShared<kWide>& sh = *reinterpret_cast<PdShared<kWide>*>(pd_smem);
  int* const before = reinterpret_cast<int*>(pd_smem + sizeof(PdShared<kWide>));  // [B + 1] granules before b
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;  // MMA fragment row group / column pair
  const int nkv = p.c.nkv, grp = p.grp;
  const int page_mask = (1 << p.c.page_shift) - 1;
  pdl_launch_dependents();
  pdl_wait();

  // granules before each sequence (all its kv heads counted)
  int carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPdThreads) {
    const int b = b0 + tid;
    int n = 0;
    if (b < p.B) {
      const int pos = pd_position(p, b, blockIdx.x == 0);
      if (pos >= 0) n = (granules_of(pos, p.window, p.sinks).n + kPdItem) * nkv;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh.warp_sum[warp] = incl;
    __syncthreads();
    int base = carry;
    for (int w = 0; w < kPdWarps; ++w) {
      if (w < warp) base += sh.warp_sum[w];
      carry += sh.warp_sum[w];
    }
    if (b < p.B) before[b] = base + incl - n;
    __syncthreads();
  }
  if (tid == 0) before[p.B] = carry;
  __syncthreads();
  const int total = carry;
  const int share = max(1, (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));

  // idle rows come out as zeros
  for (int b = blockIdx.x; b < p.B; b += gridDim.x)
    if (before[b] == before[b + 1])
      for (int i = tid; i < p.nq * D / 8; i += kPdThreads)
        reinterpret_cast<uint4*>(p.out + static_cast<long long>(b) * p.nq * D)[i] = make_uint4(0u, 0u, 0u, 0u);

  const int run_lo = min(total, static_cast<int>(blockIdx.x) * share), run_hi = min(total, run_lo + share);
  const uint32_t stage0 = smem_u32(&sh.stage[warp][0][0]);

  for (int at = run_lo; at < run_hi;) {
    // the (sequence, kv head) of granule `at`, and this CTA's run of it
    int b = 0;
    for (int lo = 0, hi = p.B; hi - lo > 1;) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= at) lo = mid; else hi = mid;
      b = lo;
    }
    const int pos = pd_position(p, b, false);
    const Granules gr = granules_of(pos, p.window, p.sinks);
    const int j = (at - before[b]) / (gr.n + kPdItem);
    // the list's first granule of (b, j), behind the places that stand for its own cost
    const int item = before[b] + j * (gr.n + kPdItem) + kPdItem;
    const int g_lo = max(at - item, 0), g_hi = min(gr.n, run_hi - item);
    at = item + gr.n;
    if (g_hi <= 0) break;  // the run ends before the item's granules
    const int first_cta = item / share, parts = (item + gr.n - 1) / share - first_cta + 1;
    const int* table = p.c.table + b * p.c.table_stride;

    // this warp's tiles: 16 positions of each granule; lane i looks up the
    // page of the warp's tile i (of the next 32)
    const int tiles = g_hi - g_lo;
    const __nv_bfloat16* kbase = p.c.k + (static_cast<long long>(j) << p.c.page_shift) * D;
    const __nv_bfloat16* vbase = p.c.v + (static_cast<long long>(j) << p.c.page_shift) * D;
    auto tile_pos = [&](int i) {  // first position of the warp's tile i
      const int gi = g_lo + i;
      return (gi < gr.sink ? gi : gi - gr.sink + gr.first) * kPdGran + warp * kPdTile;
    };
    auto tile_live = [&](int s0) {  // whether the query sees any of its positions
      if (s0 > pos) return false;
      return p.window == 0 || s0 + kPdTile - 1 > pos - p.window || s0 < p.sinks;
    };
    int lane_page = -1;
    uint32_t held = 0;  // bit i % 32: tile i has its rows staged
    auto look_up = [&](int i0) {
      const int i = i0 + lane;
      lane_page = -1;
      if (i < tiles) {
        const int s0 = tile_pos(i);
        if (tile_live(s0)) {
          const int pg = table[s0 >> p.c.page_shift];
          if (pg >= 0 && pg < p.c.num_pages) lane_page = pg;
          else atomicOr(p.status, kDevErrBadIndex);  // a page that the query needs is not held
        }
      }
    };
    // issue(i): tile i's rows into its stage; invisible rows are zero-filled
    // (whatever their memory holds), the new token's row comes later
    const int r0 = lane >> 4, ch = lane & 15;
    auto issue = [&](int i) {
      if (i < tiles) {
        const int pg = __shfl_sync(0xffffffffu, lane_page, i & 31);
        held = (held & ~(1u << (i & 31))) | (static_cast<uint32_t>(pg >= 0) << (i & 31));
        if (pg >= 0) {
          const int s0 = tile_pos(i);
          const long long in_page = static_cast<long long>(s0 & page_mask) * D + ch * 8;
          const __nv_bfloat16* ks = kbase + pg * p.c.k_stride + in_page;
          const __nv_bfloat16* vs = vbase + pg * p.c.v_stride + in_page;
          const uint32_t dst = stage0 + (i % kPdStages) * (kPdStage * 2);
#pragma unroll
          for (int u = 0; u < kPdTile / 2; ++u) {
            const int r = u * 2 + r0, s = s0 + r;
            const uint32_t bytes = s != pos && key_visible(s, pos, p.window, p.sinks) ? 16u : 0u;
            const uint32_t off = r * 256 + ((ch ^ (r & 7)) << 4);
            cp_async_16(dst + off, ks + r * D, bytes);
            cp_async_16(dst + kPdTile * 256 + off, vs + r * D, bytes);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up(0);
#pragma unroll
    for (int i = 0; i < kPdStages - 1; ++i) issue(i);

    // queries of the group: normalised, rotated, scaled (base-2 softmax), as
    // hi + lo; a half-warp per head.  The CTA that holds the new token's
    // granule prepares its key and value row and stores them.
    const bool owns_new = g_hi == gr.n;
    if (tid < D / 2) sh.tab[tid] = rope_cos_sin(p.turns.f[tid], pos);
    __syncthreads();
    {
      const int l = lane & 15, half = tid >> 4;
      const __nv_bfloat16* row = p.qkv + static_cast<long long>(b) * (p.nq + 2 * nkv) * D;
      constexpr int kHalves = kPdThreads / 16;
      const TurnPart turn = turn_part(sh.tab, l);
      HeadPart w = load_weight_part(p.qw, p.w_dtype, l);
      for (int h0 = 0; h0 < (kWide ? 16 : 8); h0 += kHalves) {
        const int h = h0 + half;
        uint2 lo = make_uint2(0u, 0u), hi = lo;
        if (h < grp) {
          const uint2* from = reinterpret_cast<const uint2*>(row + static_cast<long long>(j * grp + h) * D) + l;
          lo = from[0];
          hi = from[16];
        }
        const HeadPart o = norm_rope_part(part_of_rows(lo, hi), w, turn, p.eps, p.scale_log2);  // 0 for no head
        const uint2 ha = row_of_pairs(o.a), hb = row_of_pairs(o.b);
        const uint64_t minus = pair2(-1.f, -1.f);
        const HeadPart top = part_of_rows(ha, hb);
        const HeadPart rest{{fma2(top.a[0], minus, o.a[0]), fma2(top.a[1], minus, o.a[1])},
                            {fma2(top.b[0], minus, o.b[0]), fma2(top.b[1], minus, o.b[1])}};
        uint2* q_hi = reinterpret_cast<uint2*>(&sh.q[0][h][0]);
        uint2* q_lo = reinterpret_cast<uint2*>(kWide ? &sh.q[kWide ? 1 : 0][h][0] : &sh.q[0][h + 8][0]);
        q_hi[l] = ha;
        q_hi[16 + l] = hb;
        q_lo[l] = row_of_pairs(rest.a);
        q_lo[16 + l] = row_of_pairs(rest.b);
      }
      if (owns_new && warp == kPdWarps - 1) {
        const uint2* from =
            reinterpret_cast<const uint2*>(row + static_cast<long long>(p.nq + (lane < 16 ? 0 : nkv) + j) * D) + l;
        uint2 lo = from[0], hi = from[16];
        w = load_weight_part(p.kw, p.w_dtype, l);
        const HeadPart o = norm_rope_part(part_of_rows(lo, hi), w, turn, p.eps);
        uint2 klo = row_of_pairs(o.a), khi = row_of_pairs(o.b);
        const uint32_t which = lane < 16 ? key_near_tie(o) : 0u;
        if (__any_sync(0xffffffffu, which != 0)) {
          for (int i = lane; i < D; i += 32) sh.kw[i] = head_wload(p.kw, p.w_dtype, i);
          __syncwarp();
          key_in_64_bits(which, lo, hi, sh.kw + 4 * l, p.turns.f, l, pos, p.eps, klo, khi);
        }
        if (lane < 16) {  // the value goes bit for bit
          lo = klo;
          hi = khi;
        }
        uint2* keep = reinterpret_cast<uint2*>(lane < 16 ? sh.knew : sh.vnew);
        keep[l] = lo;
        keep[16 + l] = hi;
        const int pg = table[pos >> p.c.page_shift];
        if (pg >= 0 && pg < p.c.num_pages) {
          const long long off = ((static_cast<long long>(j) << p.c.page_shift) + (pos & page_mask)) * D;
          uint2* dst = reinterpret_cast<uint2*>((lane < 16 ? p.c.k + pg * p.c.k_stride : p.c.v + pg * p.c.v_stride) + off);
          dst[l] = lo;
          dst[16 + l] = hi;
        }
      }
    }
    __syncthreads();
    const int ld_row = (lane & 7) + ((lane >> 3) & 1) * 8, ld_col = (lane >> 4) * 8;
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) pd_ldsm4(smem_u32(&sh.q[0][ld_row][kk * 16 + ld_col]), qf[kk]);

    // running softmax of heads g (and g + 8 when wide); l holds this thread's
    // positions only until the end
    constexpr int kH = kWide ? 2 : 1;
    float m_run[kH], l_run[kH];
#pragma unroll
    for (int h = 0; h < kH; ++h) {
      m_run[h] = -INFINITY;
      l_run[h] = 0.f;
    }
    float acc[16][4];
#pragma unroll
    for (int n = 0; n < 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;

    for (int i = 0; i < tiles; ++i) {
      if (i + kPdStages - 1 < tiles && ((i + kPdStages - 1) & 31) == 0) look_up(i + kPdStages - 1);
      issue(i + kPdStages - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kPdStages - 1) : "memory");
      const int s0 = tile_pos(i);
      const uint32_t ks = stage0 + (i % kPdStages) * (kPdStage * 2), vs = ks + kPdTile * 256;
      __syncwarp();  // every lane's copies have landed
      if (!((held >> (i & 31)) & 1u)) continue;
      if (pos >= s0 && pos < s0 + kPdTile) {
        const int r = pos - s0, l = lane & 15;
        const uint32_t off = r * 256 + ((l ^ (r & 7)) << 4);
        const uint4 u = *reinterpret_cast<const uint4*>((lane < 16 ? sh.knew : sh.vnew) + l * 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((lane < 16 ? ks : vs) + off), "r"(u.x), "r"(u.y),
                     "r"(u.z), "r"(u.w)
                     : "memory");
        __syncwarp();
      }

      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t bk[4];  // positions 0-7 (dims lo, hi), positions 8-15
        const int r = (lane & 7) + ((lane >> 4) << 3), c16 = kk * 2 + ((lane >> 3) & 1);
        pd_ldsm4(ks + r * 256 + ((c16 ^ (r & 7)) << 4), bk);
        pd_mma(sc[0], qf[kk], bk[0], bk[1]);
        pd_mma(sc[1], qf[kk], bk[2], bk[3]);
        if constexpr (kWide) {
          uint32_t ql[4];
          pd_ldsm4(smem_u32(&sh.q[1][ld_row][kk * 16 + ld_col]), ql);
          pd_mma(sc[0], ql, bk[0], bk[1]);
          pd_mma(sc[1], ql, bk[2], bk[3]);
        }
      }
      // scores of heads g (+ 8h), positions n * 8 + 2t + e
      float s[kH][2][2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool see = key_visible(s0 + n * 8 + 2 * t + e, pos, p.window, p.sinks);
          if constexpr (kWide) {
            s[0][n][e] = see ? sc[n][e] : -INFINITY;
            s[kH - 1][n][e] = see ? sc[n][2 + e] : -INFINITY;
          } else {
            s[0][n][e] = see ? sc[n][e] + sc[n][2 + e] : -INFINITY;
          }
        }
      float alpha[kH];
      uint32_t ph[2][4];  // A fragments of the weights: [narrow: one, wide: hi / lo]
#pragma unroll
      for (int h = 0; h < kH; ++h) {
        float mx = fmaxf(fmaxf(s[h][0][0], s[h][0][1]), fmaxf(s[h][1][0], s[h][1][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m_run[h], mx);
        const float ms = mn == -INFINITY ? 0.f : mn;  // scores of -inf all through
        alpha[h] = exp2f(m_run[h] - ms);
        m_run[h] = mn;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float e0 = exp2f(s[h][n][0] - ms), e1 = exp2f(s[h][n][1] - ms);
          sum += e0 + e1;
          const uint32_t hi = pack_bf16x2(e0, e1);
          const float2 hf = unpack_bf16x2(hi);
          const uint32_t lo = pack_bf16x2(e0 - hf.x, e1 - hf.y);
          if constexpr (kWide) {
            ph[0][n * 2 + h] = hi;
            ph[1][n * 2 + h] = lo;
          } else {
            ph[0][n * 2] = hi;
            ph[0][n * 2 + 1] = lo;
          }
        }
        l_run[h] = l_run[h] * alpha[h] + sum;
      }
      const bool same = kWide ? (alpha[0] == 1.f && alpha[kH - 1] == 1.f) : alpha[0] == 1.f;
      if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          acc[n][0] *= alpha[0];
          acc[n][1] *= alpha[0];
          acc[n][2] *= alpha[kH - 1];
          acc[n][3] *= alpha[kH - 1];
        }
      }
#pragma unroll
      for (int n = 0; n < 16; n += 2) {
        uint32_t bv[4];
        const int r = (lane & 7) + ((lane >> 3) & 1) * 8, c16 = n + (lane >> 4);
        pd_ldsm4t(vs + r * 256 + ((c16 ^ (r & 7)) << 4), bv);
        pd_mma(acc[n], ph[0], bv[0], bv[1]);
        pd_mma(acc[n + 1], ph[0], bv[2], bv[3]);
        if constexpr (kWide) {
          pd_mma(acc[n], ph[1], bv[0], bv[1]);
          pd_mma(acc[n + 1], ph[1], bv[2], bv[3]);
        }
      }
      __syncwarp();  // every lane has read the stage before it is filled again
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // join the four warps: each leaves (m, l) and its o rows over its own stages
    __syncthreads();
    float* const ow = reinterpret_cast<float*>(&sh.stage[warp][0][0]);  // [16][128]
#pragma unroll
    for (int h = 0; h < kH; ++h) {
      float l = l_run[h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t == 0) {
        sh.ml[warp][g + 8 * h][0] = m_run[h];
        sh.ml[warp][g + 8 * h][1] = l;
      }
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const float2 o = kWide ? make_float2(acc[n][2 * h], acc[n][2 * h + 1])
                               : make_float2(acc[n][0] + acc[n][2], acc[n][1] + acc[n][3]);
        *reinterpret_cast<float2*>(ow + (g + 8 * h) * D + n * 8 + 2 * t) = o;
      }
    }
    __syncthreads();
    const int slot = 2 * static_cast<int>(blockIdx.x) + (item < run_lo ? 0 : 1);
    for (int i = tid; i < grp * (D / 4); i += kPdThreads) {
      const int h = i >> 5, d = (i & 31) * 4;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kPdWarps; ++w) m = fmaxf(m, sh.ml[w][h][0]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kPdWarps; ++w) {
        const float f = m == -INFINITY ? 0.f : exp2f(sh.ml[w][h][0] - m);
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(&sh.stage[w][0][0]) + h * D + d);
        l = fmaf(f, sh.ml[w][h][1], l);
        o.x = fmaf(f, v.x, o.x);
        o.y = fmaf(f, v.y, o.y);
        o.z = fmaf(f, v.z, o.z);
        o.w = fmaf(f, v.w, o.w);
      }
      if (parts == 1) {
        const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
        const uint2 u = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        *reinterpret_cast<uint2*>(p.out + (static_cast<long long>(b) * p.nq + j * grp + h) * D + d) = u;
      } else {
        float* dst = p.part + (static_cast<long long>(slot) * grp + h) * kPdPart;
        __stcg(reinterpret_cast<float4*>(dst + d), o);
        if (d == 0) __stcg(reinterpret_cast<float2*>(dst + D), make_float2(m, l));
      }
    }
    __syncthreads();
    if (parts > 1) {
      if (tid == 0) {
        __threadfence();
        sh.last = atomicAdd(p.counters + first_cta, 1) == parts - 1;
        if (sh.last) {
          __threadfence();
          p.counters[first_cta] = 0;  // ready for the next call
        }
      }
      __syncthreads();
      if (sh.last) {
        // the item begins in its first CTA (slot 1) and goes on in the others (slot 0)
        const int slot_first = 2 * first_cta + 1;
        for (int h = warp; h < grp; h += kPdWarps) {
          float m = -INFINITY;
          for (int c = lane; c < parts; c += 32) {
            const int sl = c == 0 ? slot_first : 2 * (first_cta + c);
            m = fmaxf(m, __ldcg(p.part + (static_cast<long long>(sl) * grp + h) * kPdPart + D));
          }
          m = warp_max(m);
          float l = 0.f;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int c0 = 0; c0 < parts; c0 += 8) {
            float4 v[8];
            float2 ml[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int c = c0 + u;
              const int sl = c == 0 ? slot_first : 2 * (first_cta + c);
              const float* src = p.part + (static_cast<long long>(sl) * grp + h) * kPdPart;
              ml[u] = c < parts ? __ldcg(reinterpret_cast<const float2*>(src + D)) : make_float2(-INFINITY, 0.f);
              v[u] = c < parts ? __ldcg(reinterpret_cast<const float4*>(src + lane * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const float f = m == -INFINITY ? 0.f : exp2f(ml[u].x - m);
              l = fmaf(f, ml[u].y, l);
              o.x = fmaf(f, v[u].x, o.x);
              o.y = fmaf(f, v[u].y, o.y);
              o.z = fmaf(f, v[u].z, o.z);
              o.w = fmaf(f, v[u].w, o.w);
            }
          }
          const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
          const uint2 u = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
          *reinterpret_cast<uint2*>(p.out + (static_cast<long long>(b) * p.nq + j * grp + h) * D + lane * 4) = u;
        }
      }
    }
    __syncthreads();  // the next run overwrites the stages and the queries
  }
}

int pd_grid(long long B, int nkv, long long max_pages, int page_size) {
  const long long most = B * nkv * ((max_pages * page_size + kPdGran - 1) / kPdGran);
  const long long full = static_cast<long long>(kPdCtasPerSm) * device_sm_count();
  return static_cast<int>(most < full ? most : full);
}

template <bool kWide>
cudaError_t pd_launch(const PdParams& p, int grid, cudaStream_t s) {
  const size_t smem = sizeof(PdShared<kWide>) + sizeof(int) * (p.B + 1);
  const cudaError_t e = allow_smem<paged_decode_kernel<kWide>>(
      static_cast<int>(sizeof(PdShared<kWide>) + sizeof(int) * (kPdMaxBatch + 1)));
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_decode_kernel<kWide>, dim3(grid), dim3(kPdThreads), smem, s, p);
}

}  // namespace

size_t paged_decode_workspace_bytes(long long B, int nq, int nkv, long long max_pages, int page_size) {
  const size_t grid = pd_grid(B, nkv, max_pages, page_size);
  return kPagedScratch + sizeof(float) * 2 * grid * (nq / nkv) * kPdPart;
}

cudaError_t paged_decode_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                                const long long* positions, long long pos_stride, const PagedCache& cache,
                                __nv_bfloat16* out, int B, int nq, float theta, float eps, float scale, int window,
                                int sinks, void* workspace, cudaStream_t s) {
  PdParams p;
  p.qkv = qkv;
  p.qw = qw;
  p.kw = kw;
  p.positions = positions;
  p.out = out;
  char* ws = static_cast<char*>(workspace);
  p.status = reinterpret_cast<int*>(ws);
  p.counters = reinterpret_cast<int*>(ws + kPagedStatusBytes);
  p.part = reinterpret_cast<float*>(ws + kPagedScratch);
  p.c = cache;
  p.turns = rope_turns(theta);
  p.pos_stride = pos_stride;
  p.w_dtype = w_dtype;
  p.B = B;
  p.nq = nq;
  p.grp = nq / cache.nkv;
  p.window = window;
  p.sinks = sinks;
  p.eps = eps;
  p.scale_log2 = scale * kPdLog2e;
  const int grid = pd_grid(B, cache.nkv, cache.max_pages, 1 << cache.page_shift);
  return p.grp <= 8 ? pd_launch<false>(p, grid, s) : pd_launch<true>(p, grid, s);
}

}  // namespace nkimoe
