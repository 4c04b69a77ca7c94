// Attention of packed prompt rows over a paged key-value cache (grouped-query
// attention, head_dim 128, causal, optionally a sliding window with a few
// first positions that stay visible) on the 5th-generation tensor cores.
//
//   out_p = sum_s softmax_s(q_p . k_s * scale) v_s  over the visible s
//
// Reference: the attention of qwen_with_nki.py:330-350 (causal, GQA, scale
// head_dim^-0.5); nki_attention.py:333-359 for the online softmax.
//
// Tile: 128 MMA rows are floor(128 / group) tokens times the `group` query
// heads of one kv head, so a tile's rows share their keys, a short chunk
// still fills the rows, and the causal and window edges of a tile are a few
// tokens wide.  A CTA works on two such tiles at a time ("pair") against the
// same key blocks of 128 positions:
//
//   warp 0      one thread: takes work units, loads Q (TMA, rows gathered by
//               a 3-D box over heads and tokens) and the K / V blocks page by
//               page (4-D boxes, 128-byte swizzle) into a ring of 32 KB stages
//   warp 1      issues the MMAs: S = Q K^T into tensor memory, then
//               O += P V with P read from tensor memory and V as the
//               transposed (MN-major) operand
//   warps 4-7,  the softmax of tile 0 / tile 1, one thread per row: S from
//   8-11        tensor memory, running maximum and sum in registers, P as
//               bf16 over S's own columns, the final scaling of O
//
// While one tile's softmax runs, the tensor core works on the other tile.
// The running maximum is raised (and O rescaled) only when a block exceeds it
// by more than 2^8; P then is at most 256 times what it would be, which bf16
// and fp32 hold as exactly, and the last division cancels it.
// P is rounded to bf16 (relative 2^-9 at most, the size of the output's own
// rounding); sums and maxima are fp32.
//
// Work: a small kernel turns the lengths (device data) into a list of units,
// (sequence, pair, range of key blocks), the longest of a sequence first;
// CTAs take units from a counter.  A pair is cut into several ranges only
// when there are too few pairs for the SMs; the parts are joined by a third
// kernel.
#include <cudaTypedefs.h>

#include "paged.cuh"

namespace nkimoe {

namespace {

constexpr int kPfBlock = 128;                  // key positions per block
constexpr int kPfRows = 128;                   // MMA rows per tile
constexpr int kPfThreads = 384;
constexpr int kPfRing = 5;                     // stages of 32 KB
constexpr uint32_t kPfTileBytes = kPfRows * kHeadDim * 2;  // 32 KB: a Q tile, a K block or a V block
constexpr uint32_t kPfHalf = kPfTileBytes / 2;             // one 64-column half (128 rows x 128 bytes)
constexpr size_t kPfSmem = 1024 + 2 * kPfTileBytes + kPfRing * kPfTileBytes;
constexpr int kPfPartRow = 132;                // floats per partial row: o[128], m, l, pad
constexpr int kPfMinBlocks = 4;                // key blocks of a part at least
constexpr float kPfLog2e = 1.4426950408889634f;
constexpr float kPfSlack = 8.f;                // log2 by which a block may exceed the running maximum
// tensor memory columns: S (and P over its first half) of tile t at 128 t, O at 256 + 128 t
constexpr uint32_t kPfTmemO = 256;

struct PfUnit {
  int b, pair, split, nsplit;
};

struct PfList {  // in the workspace
  int count;     // entries; unit u is entry u / nkv, kv head u % nkv
  int next;      // the counter that CTAs take units from
  int splits;    // pairs that are cut into parts
  int pad;
};

// A pair that is cut: its rows and its parts' slots (slot + split) * nkv + j.
struct PfSplit {
  int b, pair, slot, nsplit;
};

struct PfParams {
  const int* cu;       // [B + 1]
  const int* kv_lens;  // [B]
  __nv_bfloat16* out;  // [T, nq * 128]
  int* status;
  PfList* list;
  PfUnit* units;
  int* slots;       // per unit entry: its first slot, or -1
  PfSplit* splits;  // [count of cut pairs]
  int* starts;      // [B + 1] pairs before each sequence
  float* part;      // [slots * nkv, 256, kPfPartRow]
  PagedCache c;
  int T, B, nq, grp, tpt;  // tpt: tokens per tile
  int window, sinks;
  int sms, max_pairs, max_entries, max_slots;
  float scale_log2;
};

// The key blocks of queries at positions [lo, hi]: those of the first `sinks`
// positions, then from the first block of lo's window on.
struct Blocks {
  int sink, first, n;
  __device__ __forceinline__ int at(int i) const { return i < sink ? i : i - sink + first; }
};
__device__ __forceinline__ Blocks blocks_of(int lo, int hi, int window, int sinks) {
  Blocks r;
  const int start = window && lo >= window ? lo - window + 1 : 0;
  r.first = start / kPfBlock;
  r.sink = start > 0 ? min((min(sinks, start) + kPfBlock - 1) / kPfBlock, r.first) : 0;
  r.n = r.sink + hi / kPfBlock - r.first + 1;
  return r;
}

// New rows of sequence b, 0 where its lengths make no sense (flagged).
__device__ __forceinline__ int pf_rows(const PfParams& p, int b, int& kv, bool flag) {
  const int lo = p.cu[b], hi = p.cu[b + 1];
  kv = p.kv_lens[b];
  if (lo == hi) return 0;
  if (lo < 0 || hi < lo || hi > p.T || kv < hi - lo || kv > static_cast<long long>(p.c.max_pages) << p.c.page_shift) {
    if (flag) atomicOr(p.status, kDevErrBadIndex);
    return 0;
  }
  return hi - lo;
}

constexpr int kPlanThreads = 1024;

// Exclusive scan over the CTA; `total` gets the sum.
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
  const int ws = warp_sums[lane];
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
__global__ void __launch_bounds__(kPlanThreads) paged_prefill_plan_kernel(const __grid_constant__ PfParams p) {
  __shared__ int warp_sums[32];
  __shared__ float warp_tot[32];
  const int tid = threadIdx.x;
  const int per_pair = 2 * p.tpt;
  pdl_launch_dependents();
  pdl_wait();
  int pairs = 0;
  float blocks = 0.f;  // all key blocks of all units, estimated from each sequence's first and last pair
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int n = 0, kv = 0;
    if (b < p.B) n = pf_rows(p, b, kv, true);
    const int np = (n + per_pair - 1) / per_pair;
    if (np > 0) {
      const int lo = kv - n;
      const int a = blocks_of(lo, min(lo + per_pair, kv) - 1, p.window, p.sinks).n;
      const int z = blocks_of(kv - 1 - (n - 1) % per_pair, kv - 1, p.window, p.sinks).n;
      blocks += 0.5f * np * (a + z) * p.c.nkv;
    }
    int total;
    const int before = plan_scan(np, warp_sums, total);
    if (b < p.B) p.starts[b] = pairs + before;
    pairs += total;
  }
  if (tid == 0) p.starts[p.B] = pairs;
  if (pairs > p.max_pairs) {  // sequences that overlap: more rows than there are
    if (tid == 0) atomicOr(p.status, kDevErrBadIndex);
    pairs = p.max_pairs;
  }
  blocks = warp_sum(blocks);
  if ((tid & 31) == 0) warp_tot[tid >> 5] = blocks;
  __syncthreads();
  blocks = 0.f;
  for (int w = 0; w < kPlanThreads / 32; ++w) blocks += warp_tot[w];
  const int most = max(kPfMinBlocks, static_cast<int>(blocks / p.sms) + 1);  // blocks of a unit

  int entries = 0, slots = 0, cut = 0;
  for (int i0 = 0; i0 < pairs; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int ns = 0, b = 0, pair = 0;
    if (i < pairs) {
      int hi = p.B;
      while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (p.starts[mid] <= i) b = mid; else hi = mid;
      }
      int kv;
      const int n = pf_rows(p, b, kv, false);
      pair = p.starts[b + 1] - 1 - i;  // the sequence's last pair, the longest, first
      const int lo = kv - n + pair * per_pair;
      ns = (blocks_of(lo, min(lo + per_pair, kv) - 1, p.window, p.sinks).n + most - 1) / most;
    }
    int total;
    // parts are given up where the list or the slots would not hold them
    int at = plan_scan(ns > 1 ? ns : 0, warp_sums, total);
    const int room = min((p.max_slots - slots), p.max_entries - entries - (pairs - i0));
    if (ns > 1 && at + ns > room) ns = 1;
    const int slot = plan_scan(ns > 1 ? ns : 0, warp_sums, total) + slots;
    slots += total;
    const int k = plan_scan(ns > 1, warp_sums, total) + cut;
    cut += total;
    const int e = plan_scan(ns, warp_sums, total) + entries;
    entries += total;
    for (int s = 0; s < ns; ++s) {
      p.units[e + s] = PfUnit{b, pair, s, ns};
      p.slots[e + s] = ns > 1 ? slot : -1;
    }
    if (ns > 1) p.splits[k] = PfSplit{b, pair, slot, ns};
  }
  if (tid == 0) *p.list = PfList{entries, 0, cut, 0};
}

// ------------------------------------------------------------------ tensor memory, MMA with A from tensor memory
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D += A B with A (bf16 pairs, one row per lane) in tensor memory
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// Descriptor of a 128-byte-swizzled MN-major operand: blocks of 64 columns
// (leading byte offset: the distance of two blocks), 8 rows of K every 1024 bytes.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t smem_addr, uint32_t block_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(block_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What the roles need to know of a unit.
struct PfWork {
  int row0;    // first packed row of the pair
  int pos0;    // its position
  int tokens;  // rows of the pair (<= 2 tpt), 0: no more units
  int j;       // kv head
  int kv;      // length of the sequence
  int b;
  int lo, hi;  // range of the pair's key blocks
  int slot;    // of the partial result, or -1
};

struct PfCtl {
  uint64_t q_full, q_empty;
  uint64_t kv_full[kPfRing], kv_empty[kPfRing];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t u_full[2], u_empty[2];
  uint64_t drain;
  PfWork work[2];
  uint32_t tmem_base;
  int abort_flag;
};

__global__ void __launch_bounds__(kPfThreads, 1)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                         const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PfParams p) {
  extern __shared__ uint8_t pf_raw[];
  __shared__ PfCtl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pf_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sq = smem;
  uint8_t* ring = smem + 2 * kPfTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, 1);
    mbar_init(&ctl.q_empty, 1);
    for (int s = 0; s < kPfRing; ++s) {
      mbar_init(&ctl.kv_full[s], 1);
      mbar_init(&ctl.kv_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctl.s_full[t], 1);
      mbar_init(&ctl.p_full[t], 4);  // one arrival per softmax warp
      mbar_init(&ctl.o_full[t], 1);
      mbar_init(&ctl.u_full[t], 1);
      mbar_init(&ctl.u_empty[t], 1 + 8);  // the MMA warp and the softmax warps
    }
    mbar_init(&ctl.drain, 1);
    ctl.abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  if (warp == 1) tmem_alloc(&ctl.tmem_base, 512);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = ctl.tmem_base;
  pdl_launch_dependents();
  pdl_wait();

  if (warp == 0) {
    // ---------------------------------------------------------------- units and loads (one thread)
    if (lane == 0) {
      const int page_rows = min(1 << p.c.page_shift, kPfBlock);  // rows per box
      const uint32_t q_bytes = 2u * p.grp * p.tpt * 128u;        // both halves of one tile's box
      int stage = 0, u = 0;
      uint32_t phase = 0, issued = 0, last_phase = 0;
      bool ok = true, q_issued = false;
      const int total = p.list->count * p.c.nkv;
      for (;; ++u) {
        const int us = u & 1;
        if (!mbar_wait(&ctl.u_empty[us], ((u >> 1) & 1) ^ 1u, &ctl.abort_flag, p.status)) {
          ok = false;
          break;
        }
        const int unit = atomicAdd(&p.list->next, 1);
        PfWork w{};
        Blocks bl{};
        if (unit < total) {
          const int e = unit / p.c.nkv;
          const PfUnit pu = p.units[e];
          const int per_pair = 2 * p.tpt;
          int kv;
          const int n = pf_rows(p, pu.b, kv, false);
          w.b = pu.b;
          w.kv = kv;
          w.j = unit - e * p.c.nkv;
          w.row0 = p.cu[pu.b] + pu.pair * per_pair;
          w.pos0 = kv - n + pu.pair * per_pair;
          w.tokens = min(per_pair, n - pu.pair * per_pair);
          bl = blocks_of(w.pos0, w.pos0 + w.tokens - 1, p.window, p.sinks);
          w.lo = static_cast<int>(static_cast<long long>(bl.n) * pu.split / pu.nsplit);
          w.hi = static_cast<int>(static_cast<long long>(bl.n) * (pu.split + 1) / pu.nsplit);
          w.slot = pu.nsplit > 1 ? (p.slots[e] + pu.split) * p.c.nkv + w.j : -1;
        }
        ctl.work[us] = w;
        mbar_arrive(&ctl.u_full[us]);
        if (w.tokens == 0) break;
        const bool two = w.tokens > p.tpt;
        if (!mbar_wait(&ctl.q_empty, (u & 1) ^ 1u, &ctl.abort_flag, p.status)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&ctl.q_full, two ? 2 * q_bytes : q_bytes);
        for (int t = 0; t < (two ? 2 : 1); ++t)
          for (int h = 0; h < 2; ++h)
            tma_load_3d(sq + t * kPfTileBytes + h * kPfHalf, &tmap_q, &ctl.q_full, h * 64, w.j * p.grp,
                        w.row0 + t * p.tpt);
        q_issued = true;
        // positions that some query of the pair sees; a page outside is read as zeros
        const int last = w.pos0 + w.tokens - 1;
        const int start = p.window && w.pos0 >= p.window ? w.pos0 - p.window + 1 : 0;
        const int* table = p.c.table + w.b * p.c.table_stride;
        for (int i = w.lo; ok && i < w.hi; ++i) {
          const int k0 = bl.at(i) * kPfBlock;
          int pages[8];
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const int s0 = k0 + g * page_rows;
            pages[g] = p.c.num_pages;  // past the last page: the load fills zeros
            if (g * page_rows < kPfBlock && s0 <= last && (s0 + page_rows > start || s0 < p.sinks)) {
              const int pg = table[s0 >> p.c.page_shift];
              if (pg >= 0 && pg < p.c.num_pages) pages[g] = pg;
              else atomicOr(p.status, kDevErrBadIndex);
            }
          }
          for (int kvsel = 0; kvsel < 2; ++kvsel) {
            if (!mbar_wait(&ctl.kv_empty[stage], phase ^ 1u, &ctl.abort_flag, p.status)) {
              ok = false;
              break;
            }
            uint8_t* dst = ring + stage * kPfTileBytes;
            mbar_arrive_expect_tx(&ctl.kv_full[stage], kPfTileBytes);
            const void* tm = kvsel ? static_cast<const void*>(&tmap_v) : static_cast<const void*>(&tmap_k);
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              if (g * page_rows < kPfBlock) {
                const int in_page = (k0 + g * page_rows) & ((1 << p.c.page_shift) - 1);
                tma_load_4d(dst + g * page_rows * 128, tm, &ctl.kv_full[stage], 0, in_page, w.j, pages[g]);
                tma_load_4d(dst + kPfHalf + g * page_rows * 128, tm, &ctl.kv_full[stage], 64, in_page, w.j, pages[g]);
              }
            }
            issued |= 1u << stage;
            last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
            if (++stage == kPfRing) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        if (!ok) break;
      }
      if (!ok) {  // let the copies in flight land before the CTA exits
        for (int s = 0; s < kPfRing; ++s)
          if ((issued >> s) & 1u) {
            const long long t0 = clock64();
            while (!mbar_try_wait(&ctl.kv_full[s], (last_phase >> s) & 1u) && clock64() - t0 < kWaitBudgetCycles / 8) {
            }
          }
        if (q_issued) {
          // the last unit whose Q was issued: u itself, or the one before it
          const long long t0 = clock64();
          while (clock64() - t0 < kWaitBudgetCycles / 64) {
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issue
    constexpr uint32_t idesc_s = umma_idesc_bf16_f32(kPfRows, kPfBlock);
    constexpr uint32_t idesc_o = umma_idesc_bf16_f32(kPfRows, kHeadDim) | (1u << 16);  // B is MN-major
    int stage = 0;
    uint32_t phase = 0, pphase[2] = {0, 0};  // pphase: of p_full, one phase per key block of the tile
    bool ok = true, any = false;
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      const bool got = mbar_wait(bar, ph, &ctl.abort_flag, p.status);
      return __all_sync(0xffffffffu, got);
    };
    // S of tile t against the K block in `st`
    auto issue_s = [&](int t, int st) {
      if (lane == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint64_t da = umma_desc_sw128(smem_u32(sq + t * kPfTileBytes + h * kPfHalf));
          const uint64_t db = umma_desc_sw128(smem_u32(ring + st * kPfTileBytes + h * kPfHalf));
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(tmem + t * 128, da + 2 * k, db + 2 * k, idesc_s, (h | k) != 0);
        }
        umma_commit(&ctl.s_full[t]);
      }
      any = true;
    };
    for (int u = 0; ok; ++u) {
      const int us = u & 1;
      if (!wait(&ctl.u_full[us], (u >> 1) & 1)) { ok = false; break; }
      const PfWork w = ctl.work[us];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.u_empty[us]);
      if (w.tokens == 0) break;
      const int tiles = w.tokens > p.tpt ? 2 : 1;
      const Blocks bl = blocks_of(w.pos0, w.pos0 + w.tokens - 1, p.window, p.sinks);
      if (!wait(&ctl.q_full, u & 1) || !wait(&ctl.kv_full[stage], phase)) { ok = false; break; }
      tcgen05_fence_after();
      for (int t = 0; t < tiles; ++t) issue_s(t, stage);
      if (lane == 0) {
        umma_commit(&ctl.kv_empty[stage]);
        if (w.hi - w.lo == 1) umma_commit(&ctl.q_empty);
      }
      if (++stage == kPfRing) { stage = 0; phase ^= 1u; }
      for (int i = w.lo; i < w.hi; ++i) {
        const int vs = stage;
        if (!wait(&ctl.kv_full[stage], phase)) { ok = false; break; }
        if (++stage == kPfRing) { stage = 0; phase ^= 1u; }
        // rows behind the sequence's end hold anything: their weights are 0,
        // and 0 times a NaN would not be
        const int live = w.kv - bl.at(i) * kPfBlock;
        if (live < kPfBlock) {
          uint8_t* v = ring + vs * kPfTileBytes;
          for (int x = live * 8 + lane; x < kPfBlock * 8; x += 32) {
            *reinterpret_cast<uint4*>(v + x * 16) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(v + kPfHalf + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_shared();
          __syncwarp();
        }
        const bool more = i + 1 < w.hi;
        for (int t = 0; t < tiles; ++t) {
          if (!wait(&ctl.p_full[t], pphase[t])) { ok = false; break; }
          pphase[t] ^= 1u;
          tcgen05_fence_after();
          if (lane == 0) {
            const uint64_t dv = umma_desc_sw128_mn(smem_u32(ring + vs * kPfTileBytes), kPfHalf);
#pragma unroll
            for (int k = 0; k < 8; ++k)  // 16 positions: 2048 bytes of V, 8 columns of P
              umma_bf16_ts(tmem + kPfTmemO + t * 128, tmem + t * 128 + 8 * k, dv + 128 * k, idesc_o,
                           i > w.lo || k != 0);
          }
          if (more) {
            if (t == 0 && !wait(&ctl.kv_full[stage], phase)) { ok = false; break; }
            issue_s(t, stage);
          } else if (lane == 0) {
            umma_commit(&ctl.o_full[t]);
          }
        }
        if (!ok) break;
        if (lane == 0) umma_commit(&ctl.kv_empty[vs]);
        if (more) {
          if (lane == 0) {
            umma_commit(&ctl.kv_empty[stage]);
            if (i + 2 == w.hi) umma_commit(&ctl.q_empty);
          }
          if (++stage == kPfRing) { stage = 0; phase ^= 1u; }
        }
      }
    }
    if (!ok && any && lane == 0) {  // issued MMAs end before tensor memory is released
      umma_commit(&ctl.drain);
      const long long t0 = clock64();
      while (!mbar_try_wait(&ctl.drain, 0) && clock64() - t0 < kWaitBudgetCycles / 8) {
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- softmax, one row per thread
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int token = row / p.grp, head = row - token * p.grp;
    const uint32_t ts = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + t * 128;
    const uint32_t to = ts + kPfTmemO;
    uint32_t sphase = 0, ophase = 0;
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      const bool got = mbar_wait(bar, ph, &ctl.abort_flag, p.status);
      return __all_sync(0xffffffffu, got);
    };
    for (int u = 0;; ++u) {
      const int us = u & 1;
      if (!wait(&ctl.u_full[us], (u >> 1) & 1)) break;
      const PfWork w = ctl.work[us];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.u_empty[us]);
      if (w.tokens == 0) break;
      if (t == 1 && w.tokens <= p.tpt) continue;
      const Blocks bl = blocks_of(w.pos0, w.pos0 + w.tokens - 1, p.window, p.sinks);
      const int tile_pos = w.pos0 + t * p.tpt;  // the tile's first position
      const int pos = tile_pos + token;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int i = w.lo; i < w.hi; ++i) {
        const int k0 = bl.at(i) * kPfBlock;
        if (!wait(&ctl.s_full[t], sphase)) { ok = false; break; }
        sphase ^= 1u;
        tcgen05_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(ts + c * 32, s[c]);
        tmem_ld_wait();
        if (k0 + kPfBlock - 1 > tile_pos || (p.window && k0 <= tile_pos + p.tpt - 1 - p.window)) {
          const int hi = pos - k0;                                       // columns up to hi,
          const int lo = p.window ? hi - p.window + 1 : 0, sk = p.sinks - k0;  // from lo on or below sk
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (!(c <= hi && (c >= lo || c < sk))) s[c >> 5][c & 31] = 0xff800000u;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 128; ++c) mx = fmaxf(mx, __uint_as_float(s[c >> 5][c & 31]));
        mx *= p.scale_log2;
        const bool raise = mx > m + kPfSlack;  // the first finite maximum too: m is -inf
        if (__any_sync(0xffffffffu, raise)) {
          const float mn = raise ? mx : m;
          if (i > w.lo) {
            // every lane takes part; lanes that keep their maximum multiply by 1
            const float f = raise ? ex2(m - mn) : 1.f;
            l *= f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(to + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st_32x32b_x32(to + c * 32, o);
            }
          }
          m = mn;
        }
        const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            const int c = h * 64 + 2 * x;
            const float a = ex2(fmaf(__uint_as_float(s[c >> 5][c & 31]), p.scale_log2, -ms));
            const float b = ex2(fmaf(__uint_as_float(s[c >> 5][(c & 31) + 1]), p.scale_log2, -ms));
            l += a + b;
            pk[x] = pack_bf16x2(a, b);
          }
          tmem_st_32x32b_x32(ts + h * 32, pk);
        }
        tmem_st_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.p_full[t]);
      }
      if (!ok || !wait(&ctl.o_full[t], ophase)) break;
      ophase ^= 1u;
      tcgen05_fence_after();
      const bool mine = token < p.tpt && t * p.tpt + token < w.tokens;
      const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
      const long long orow = w.row0 + t * p.tpt + token;
      __nv_bfloat16* dst = p.out + (orow * p.nq + w.j * p.grp + head) * kHeadDim;
      float* part = w.slot >= 0 ? p.part + (static_cast<long long>(w.slot) * 2 * kPfRows + t * kPfRows + row) * kPfPartRow : nullptr;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        __syncwarp();
        tmem_ld_32x32b_x32(to + c * 32, o);
        tmem_ld_wait();
        if (!mine) {
        } else if (part) {
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            __stcg(reinterpret_cast<uint4*>(part + c * 32 + x), make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]));
        } else {
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[x + e]) * inv;
            *reinterpret_cast<uint4*>(dst + c * 32 + x) = pack8(f);
          }
        }
      }
      if (part && mine) __stcg(reinterpret_cast<float2*>(part + kHeadDim), make_float2(m, l));
      tcgen05_fence_before();  // the next unit's MMAs follow this thread's next arrival
    }
  }

  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of cut pairs: one warp per (pair, kv head, row), a lane per
// four columns, the parts in order.
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const __grid_constant__ PfParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int rows = 2 * kPfRows;
  const long long total = static_cast<long long>(p.list->splits) * p.c.nkv * rows;
  for (long long i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < total; i += gridDim.x * 8ll) {
    const int r = static_cast<int>(i % rows), j = static_cast<int>(i / rows % p.c.nkv);
    const PfSplit sp = p.splits[i / rows / p.c.nkv];
    const int tile = r >> 7, token = (r & 127) / p.grp, head = (r & 127) - token * p.grp;
    const int at = sp.pair * 2 * p.tpt + tile * p.tpt + token;  // row of the sequence
    const int start = p.cu[sp.b];
    if (token >= p.tpt || at >= p.cu[sp.b + 1] - start) continue;
    const float* part = p.part + (static_cast<long long>(sp.slot * p.c.nkv + j) * rows + r) * kPfPartRow;
    const long long stride = static_cast<long long>(p.c.nkv) * rows * kPfPartRow;
    float m = -INFINITY;
    for (int s = lane; s < sp.nsplit; s += 32) m = fmaxf(m, __ldcg(part + s * stride + kHeadDim));
    m = warp_max(m);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < sp.nsplit; s0 += 4) {
      float4 v[4];
      float2 ml[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const bool in = s0 + x < sp.nsplit;
        ml[x] = in ? __ldcg(reinterpret_cast<const float2*>(part + (s0 + x) * stride + kHeadDim)) : make_float2(-INFINITY, 0.f);
        v[x] = in ? __ldcg(reinterpret_cast<const float4*>(part + (s0 + x) * stride + lane * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float f = m == -INFINITY ? 0.f : exp2f(ml[x].x - m);
        l = fmaf(f, ml[x].y, l);
        o.x = fmaf(f, v[x].x, o.x);
        o.y = fmaf(f, v[x].y, o.y);
        o.z = fmaf(f, v[x].z, o.z);
        o.w = fmaf(f, v[x].w, o.w);
      }
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    *reinterpret_cast<uint2*>(p.out + ((static_cast<long long>(start + at) * p.nq + j * p.grp + head) * kHeadDim + lane * 4)) =
        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
}

// Sizes that the host can bound without the lengths.
struct PfLayout {
  long long pairs, slots, entries;
  size_t list, units, slot_of, splits, starts, part, total;
};

PfLayout pf_layout(long long T, long long B, int nkv, int grp, long long max_pages, int page_size) {
  PfLayout L;
  const int tpt = kPfRows / grp;
  L.pairs = T / (2 * tpt) + B;
  const long long blocks = (max_pages * page_size + kPfBlock - 1) / kPfBlock;
  const long long sms = device_sm_count();
  // parts of all cut pairs: about one per SM and kv head share, twice that with the rounding
  long long slots = blocks > kPfMinBlocks ? 2 * sms / nkv + 16 : 0;
  const long long most = L.pairs * ((blocks + kPfMinBlocks - 1) / kPfMinBlocks);
  L.slots = slots < most ? slots : most;
  L.entries = L.pairs + L.slots;
  auto round = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
  size_t at = kPagedScratch;
  L.list = at;
  at += 256;
  L.units = at;
  at += round(sizeof(PfUnit) * L.entries);
  L.slot_of = at;
  at += round(sizeof(int) * L.entries);
  L.splits = at;
  at += round(sizeof(PfSplit) * (L.slots / 2 + 1));
  L.starts = at;
  at += round(sizeof(int) * (B + 1));
  L.part = at;
  at += sizeof(float) * L.slots * nkv * 2 * kPfRows * kPfPartRow;
  L.total = at;
  return L;
}

}  // namespace

size_t paged_prefill_workspace_bytes(long long T, long long B, int nq, int nkv, long long max_pages, int page_size) {
  return pf_layout(T, B, nkv, nq / nkv, max_pages, page_size).total;
}

cudaError_t paged_prefill_launch(const __nv_bfloat16* q, long long q_stride, const int* cu_seqlens,
                                 const int* kv_lens, const PagedCache& cache, __nv_bfloat16* out, long long T, int B,
                                 int nq, float scale, int window, int sinks, void* workspace, cudaStream_t s) {
  auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tmap_encode_fn());
  if (!encode) return cudaErrorNotSupported;
  const int nkv = cache.nkv, grp = nq / nkv, tpt = kPfRows / grp, page = 1 << cache.page_shift;
  CUtensorMap mq, mk, mv;
  {
    const cuuint64_t dims[3] = {kHeadDim, static_cast<cuuint64_t>(nq), static_cast<cuuint64_t>(T)};
    const cuuint64_t strides[2] = {kHeadDim * 2, static_cast<cuuint64_t>(q_stride) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(grp), static_cast<cuuint32_t>(tpt)};
    const cuuint32_t one[3] = {1, 1, 1};
    if (encode(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(q), dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  for (int i = 0; i < 2; ++i) {
    const cuuint64_t dims[4] = {kHeadDim, static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(nkv),
                                static_cast<cuuint64_t>(cache.num_pages)};
    const cuuint64_t strides[3] = {kHeadDim * 2, static_cast<cuuint64_t>(page) * kHeadDim * 2,
                                   static_cast<cuuint64_t>(i ? cache.v_stride : cache.k_stride) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(page < kPfBlock ? page : kPfBlock), 1, 1};
    const cuuint32_t one[4] = {1, 1, 1, 1};
    if (encode(i ? &mv : &mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, i ? cache.v : cache.k, dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  const PfLayout L = pf_layout(T, B, nkv, grp, cache.max_pages, page);
  char* ws = static_cast<char*>(workspace);
  PfParams p;
  p.cu = cu_seqlens;
  p.kv_lens = kv_lens;
  p.out = out;
  p.status = reinterpret_cast<int*>(ws);
  p.list = reinterpret_cast<PfList*>(ws + L.list);
  p.units = reinterpret_cast<PfUnit*>(ws + L.units);
  p.slots = reinterpret_cast<int*>(ws + L.slot_of);
  p.splits = reinterpret_cast<PfSplit*>(ws + L.splits);
  p.starts = reinterpret_cast<int*>(ws + L.starts);
  p.part = reinterpret_cast<float*>(ws + L.part);
  p.c = cache;
  p.T = static_cast<int>(T);
  p.B = B;
  p.nq = nq;
  p.grp = grp;
  p.tpt = tpt;
  p.window = window;
  p.sinks = sinks;
  p.sms = device_sm_count();
  p.max_pairs = static_cast<int>(L.pairs);
  p.max_entries = static_cast<int>(L.entries);
  p.max_slots = static_cast<int>(L.slots);
  p.scale_log2 = scale * kPfLog2e;
  cudaError_t e = launch_pdl(paged_prefill_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
  if (e != cudaSuccess) return e;
  e = allow_smem<paged_prefill_kernel>(static_cast<int>(kPfSmem));
  if (e != cudaSuccess) return e;
  const long long units = L.entries * nkv;
  const int grid = static_cast<int>(units < p.sms ? units : p.sms);
  e = launch_pdl(paged_prefill_kernel, dim3(grid), dim3(kPfThreads), kPfSmem, s, mq, mk, mv, p);
  if (e != cudaSuccess || L.slots == 0) return e;
  return launch_pdl(paged_prefill_join_kernel, dim3(2 * p.sms), dim3(256), 0, s, p);
}

}  // namespace nkimoe
