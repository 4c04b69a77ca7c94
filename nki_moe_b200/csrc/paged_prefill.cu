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
//   warp 0      takes work units, loads Q (TMA, rows gathered by a 3-D box over
//               heads and tokens) and the K blocks page by page (4-D boxes,
//               128-byte swizzle) into a ring of 32 KB stages
//   warp 2      loads the V blocks
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
// P is rounded to bf16 (relative 2^-8 at most, the size of the output's own
// rounding); sums and maxima are fp32.
//
// Bound by the tensor core and, more, by each tile's chain: scores -> softmax
// -> weights -> product -> next scores, about 3500 cycles per block and pair
// against 2100 of MMAs (P lies over S, so a tile's next scores wait for its
// product).  Measured: 8192 causal tokens, 32 heads over 4, 441 to 451 us in runs
// of some 40 ms at 1965 MHz = 1.22 to 1.25 PFLOP/s = 0.73 to 0.75 of the measured
// cuBLAS burst; back to back for seconds, 1670 MHz at the power cap, 511 us = 1.08
// PFLOP/s = 0.77 of the sustained one.  8 x 512 tokens 37 to 38 us either way; 945
// rows in four chunks over 9001 cached positions, window 4096: 83 to 88 us.
// Other shapes of the pipeline were slower (8192 tokens, short runs): key blocks of 64 with
// two score buffers per tile 891 us (an MMA of N = 64 takes as long as one of
// 128: it is bound by reading Q), one tile with two score buffers and its own
// P columns 581 us (twice the K / V traffic through shared memory), two softmax
// threads per row 500 us, a share of the exponentials as polynomials on the FMA
// pipe 500 us, weights handed over in two parts 450 us.  One score buffer that
// the tiles use in turn, P in columns of its own and a thread per tile for the
// MMAs: 415 us, but 8 x 512 tokens 39 us (with the unit's first scores in O's
// columns 426 and 42 us), and as much again in barriers to keep right.
//
// Work: a small kernel turns the lengths (device data) into the list of pairs,
// a sequence's longest first, with their counts of key blocks.  With pairs
// enough, CTAs take whole ones from a counter.  Where one pair would be longer
// than a CTA's share of all blocks (a chunk over a long cache), every CTA takes
// an equal run of the list of blocks instead, the pairs that are cut leave
// partial results, and a third kernel joins them.
#include "paged_mma.cuh"

namespace nkimoe {

namespace {

constexpr int kPfThreads = 384;
constexpr int kPfRing = 4;                     // stages of 32 KB
constexpr size_t kPfSmem = 1024 + 2 * kPfTileBytes + kPfRing * kPfBlockBytes;
// A part of a cut pair, per tile: o four columns at a time [32][128 rows][4],
// then the rows' m, then their l (a warp's rows are neighbours: coalesced)
constexpr int kPfPartTile = (kHeadDim + 2) * kPfRows;
constexpr int kPfMinBlocks = 4;                // key blocks of a part at least

// A unit, for each kv head.
struct __align__(16) PfUnit {
  int row0;    // first packed row of the pair
  int pos0;    // its position
  int tokens;  // rows of the pair (<= 2 tpt)
  int kv;      // length of the sequence
  int b;
  int lo, hi;  // range of the pair's key blocks
  int slot;    // of its partial result, or -1
};

struct PfList {  // in the workspace
  int pairs;
  int next;   // the counter that CTAs take pairs from, after one each
  int total;  // key blocks of all pairs and kv heads
  int share;  // a CTA's run of them, or 0: CTAs take whole pairs
};

// What a CTA began and others went on with: the pair of a kv head whose parts
// lie in slot 2 c + 1 of CTA c and the slots 0 of the CTAs after it.
struct PfSplit {
  int pair, j, parts, pad;
};

struct PfParams {
  const int* cu;       // [B + 1]
  const int* kv_lens;  // [B]
  __nv_bfloat16* out;  // [T, nq * 128]
  int* status;
  PfList* list;
  PfUnit* units;    // [pairs]
  int* offs;        // [pairs + 1] key blocks before each pair
  PfSplit* splits;  // [grid]
  int* starts;      // [B + 1] pairs before each sequence
  float* part;      // [2 grid, 2, kPfPartTile]
  PagedCache c;
  int T, B, nq, grp, tpt;  // tpt: tokens per tile
  int window, sinks;
  int sms, max_pairs;
  float scale_log2;
};

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

constexpr int kPlanThreads = 256;   // 1024: 0.4 us more (8 x 512, four chunks)
constexpr int kPlanStarts = 4096;  // sequences whose first pairs are also kept in shared memory

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
  const int ws = lane < kPlanThreads / 32 ? warp_sums[lane] : 0;
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
  __shared__ int near_starts[kPlanStarts + 1];
  __shared__ int longest;
  const int tid = threadIdx.x;
  const int per_pair = 2 * p.tpt;
  if (tid == 0) longest = 0;
  pdl_launch_dependents();
  pdl_wait();
  int pairs = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int n = 0, kv = 0;
    if (b < p.B) n = pf_rows(p, b, kv, true);
    int total;
    const int before = plan_scan((n + per_pair - 1) / per_pair, warp_sums, total);
    if (b < p.B) (b <= kPlanStarts ? near_starts : p.starts)[b] = min(pairs + before, p.max_pairs);
    pairs = min(pairs + total, p.max_pairs + 1);
  }
  if (pairs > p.max_pairs) {  // sequences that overlap: more rows than there are
    if (tid == 0) atomicOr(p.status, kDevErrBadIndex);
    pairs = p.max_pairs;
  }
  if (tid == 0) (p.B <= kPlanStarts ? near_starts : p.starts)[p.B] = pairs;
  __syncthreads();

  auto start_of = [&](int b) { return b <= kPlanStarts ? near_starts[b] : p.starts[b]; };
  long long blocks = 0;  // of the pairs so far
  for (int i0 = 0; i0 < pairs; i0 += kPlanThreads) {
    const int i = i0 + tid;
    PfUnit un{};
    if (i < pairs) {
      int b = 0, hi = p.B;
      while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (start_of(mid) <= i) b = mid; else hi = mid;
      }
      const int n = pf_rows(p, b, un.kv, false);
      const int pair = (n + per_pair - 1) / per_pair - 1 - (i - start_of(b));  // a sequence's longest pair first
      un.b = b;
      un.row0 = p.cu[b] + pair * per_pair;
      un.pos0 = un.kv - n + pair * per_pair;
      un.tokens = min(per_pair, n - pair * per_pair);
      un.hi = blocks_of(un.pos0, un.pos0 + un.tokens - 1, p.window, p.sinks).n;
      un.slot = -1;
      p.units[i] = un;
    }
    const int most = __reduce_max_sync(0xffffffffu, un.hi);
    if ((tid & 31) == 0) atomicMax(&longest, most);
    int total;
    const int before = plan_scan(un.hi, warp_sums, total);
    if (i < pairs) p.offs[i] = static_cast<int>(min(blocks + before, 0x7fffffffLL));
    blocks += total;
  }
  if (tid == 0) {
    p.offs[pairs] = static_cast<int>(min(blocks, 0x7fffffffLL));
    blocks *= p.c.nkv;
    // a pair is cut only where one is longer than a CTA's share of the work
    const long long share = max(static_cast<long long>(kPfMinBlocks), (blocks + p.sms - 1) / p.sms);
    const bool cut = longest > share && blocks < (1LL << 30);
    *p.list = PfList{pairs, 0, static_cast<int>(min(blocks, 1LL << 30)), cut ? static_cast<int>(share) : 0};
  }
}

// What the roles need to know of a unit; tokens 0: there are no more.
struct PfWork : PfUnit {
  int j;  // kv head
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
  __shared__ __align__(16) __nv_bfloat16 stg[8][32][40];  // per softmax warp: 32 output columns of its rows
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
      mbar_init(&ctl.u_empty[t], 2 + 8);  // the MMA warp, the warp that loads V, the softmax warps
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
  // 384 x 168 registers at launch = 128 x 88 + 256 x 208
  if (warp == 0 || warp == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ---------------------------------------------------------------- units and loads
    // Lane (h, g) loads half h of page g of a block.  A box takes its warp 110
    // cycles (a block of 16-position pages 1800), so K and V have a warp each and
    // the first queries go out before the page ids are there: 8 x 512 tokens 39.0
    // -> 37.8 us.
    const int v = warp >> 1;
    const int h_lane = (lane >> 3) & 1, g_lane = lane & 7;
    const int page_rows = min(1 << p.c.page_shift, kPfBlock);  // rows per box
    const bool loads = lane < 16 && g_lane * page_rows < kPfBlock;
    const void* const tm = v ? static_cast<const void*>(&tmap_v) : static_cast<const void*>(&tmap_k);
    const int box_at = h_lane * static_cast<int>(kPfBlockHalf) + g_lane * page_rows * 128;
    const uint32_t q_bytes = 2u * p.grp * p.tpt * 128u;  // both halves of one tile's box
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      const bool got = mbar_wait(bar, ph, &ctl.abort_flag, p.status);
      return __all_sync(0xffffffffu, got);
    };
    int stage = v;  // K blocks in the even stages, V blocks in the odd ones
    uint32_t phase = 0, issued = 0, last_phase = 0;
    bool ok = true, q_issued = false;
    const PfList list = *p.list;
    // a run of the list of key blocks (pair, kv head, block), or whole pairs
    const int run_lo = min(list.total, static_cast<int>(blockIdx.x) * list.share);
    const int run_hi = min(list.total, run_lo + list.share);
    int at = run_lo, pair = 0, unit = blockIdx.x;
    if (v == 0 && list.share) {
      if (lane == 0) p.splits[blockIdx.x].parts = 0;
      for (int hi = list.pairs; hi - pair > 1;) {
        const int mid = (pair + hi) >> 1;
        if (p.offs[mid] * p.c.nkv <= at) pair = mid; else hi = mid;
      }
    }
    auto load_q = [&](const PfWork& w, int u) {
      if (!wait(&ctl.q_empty, (u & 1) ^ 1u)) return false;
      const int tiles = w.tokens > p.tpt ? 2 : 1;
      if (lane == 0) mbar_arrive_expect_tx(&ctl.q_full, tiles * q_bytes);
      __syncwarp();
      if (lane < 2 * tiles)
        tma_load_3d(sq + (lane >> 1) * kPfTileBytes + (lane & 1) * kPfTileHalf, &tmap_q, &ctl.q_full, (lane & 1) * 64,
                    w.j * p.grp, w.row0 + (lane >> 1) * p.tpt);
      q_issued = true;
      return true;
    };
    for (int u = 0; ok; ++u) {
      const int us = u & 1;
      PfWork w{};
      if (v) {
        if (!wait(&ctl.u_full[us], (u >> 1) & 1)) { ok = false; break; }
        w = ctl.work[us];
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.u_empty[us]);
      } else {
        if (!wait(&ctl.u_empty[us], ((u >> 1) & 1) ^ 1u)) { ok = false; break; }
        if (list.share == 0) {
          if (unit < list.pairs * p.c.nkv) {
            static_cast<PfUnit&>(w) = p.units[unit / p.c.nkv];
            w.j = unit % p.c.nkv;
            // the one after it, long before it is needed
            if (lane == 0) unit = atomicAdd(&p.list->next, 1) + gridDim.x;
          }
        } else if (at < run_hi) {
          static_cast<PfUnit&>(w) = p.units[pair];
          const int base = p.offs[pair] * p.c.nkv, n = w.hi;
          w.j = (at - base) / n;
          const int item = base + w.j * n;  // the list's first block of (pair, kv head)
          w.lo = at - item;
          w.hi = min(n, run_hi - item);
          const int first = item / list.share, parts = (item + n - 1) / list.share - first + 1;
          if (parts > 1) w.slot = 2 * static_cast<int>(blockIdx.x) + (item < run_lo ? 0 : 1);
          if (parts > 1 && item >= run_lo && lane == 0) p.splits[blockIdx.x] = PfSplit{pair, w.j, parts, 0};
          at = item + w.hi;
          if (w.hi == n && w.j == p.c.nkv - 1) ++pair;
        }
        if (lane == 0) {
          ctl.work[us] = w;
          mbar_arrive(&ctl.u_full[us]);
        }
      }
      if (w.tokens == 0) break;
      const Blocks bl = blocks_of(w.pos0, w.pos0 + w.tokens - 1, p.window, p.sinks);
      // positions that some query of the pair sees; a page outside is read as zeros
      const int last = w.pos0 + w.tokens - 1;
      const int start = p.window && w.pos0 >= p.window ? w.pos0 - p.window + 1 : 0;
      const int* table = p.c.table + w.b * p.c.table_stride;
      auto look_up = [&](int i) {
        const int s0 = bl.at(i) * kPfBlock + g_lane * page_rows;
        const bool need = loads && s0 <= last && (s0 + page_rows > start || s0 < p.sinks);
        return need ? table[s0 >> p.c.page_shift] : -2;
      };
      if (v == 0 && u == 0 && !load_q(w, u)) { ok = false; break; }
      int next = look_up(w.lo);
      for (int i = w.lo; ok && i < w.hi; ++i) {
        const bool held = next >= 0 && next < p.c.num_pages;
        if (!held && next != -2) atomicOr(p.status, kDevErrBadIndex);
        const int page = held ? next : p.c.num_pages;  // past the last page: the load fills zeros
        const int in_page = (bl.at(i) * kPfBlock + g_lane * page_rows) & ((1 << p.c.page_shift) - 1);
        if (i + 1 < w.hi) next = look_up(i + 1);  // in flight while this block waits for its stage
        if (!wait(&ctl.kv_empty[stage], phase ^ 1u)) { ok = false; break; }
        if (lane == 0) mbar_arrive_expect_tx(&ctl.kv_full[stage], kPfBlockBytes);
        __syncwarp();
        if (loads) tma_load_4d(ring + stage * kPfBlockBytes + box_at, tm, &ctl.kv_full[stage], h_lane * 64, in_page, w.j, page);
        issued |= 1u << stage;
        last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
        stage += 2;
        if (stage >= kPfRing) {
          stage = v;
          phase ^= 1u;
        }
        // later units' queries after their first block, which goes out while the
        // unit before still reads its own
        if (v == 0 && u > 0 && i == w.lo && !load_q(w, u)) { ok = false; break; }
      }
      unit = __shfl_sync(0xffffffffu, unit, 0);
    }
    if (!ok && lane == 0) {  // let the copies in flight land before the CTA exits
      for (int s = 0; s < kPfRing; ++s)
        if ((issued >> s) & 1u) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&ctl.kv_full[s], (last_phase >> s) & 1u) && clock64() - t0 < kWaitBudgetCycles / 8) {
          }
        }
      if (q_issued) {
        const long long t0 = clock64();
        while (clock64() - t0 < kWaitBudgetCycles / 64) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ---------------------------------------------------------------- MMA issue (one thread)
    constexpr uint32_t idesc_s = umma_idesc_bf16_f32(kPfRows, kPfBlock);
    constexpr uint32_t idesc_o = umma_idesc_bf16_f32(kPfRows, kHeadDim) | (1u << 16);  // B is MN-major
    const int page_rows = min(1 << p.c.page_shift, kPfBlock);
    int stage = 0;
    uint32_t phase = 0, pphase = 0;  // pphase: bit t, of p_full
    bool ok = true, any = false;
    auto wait = [&](uint64_t* bar, uint32_t ph) { return mbar_wait(bar, ph, &ctl.abort_flag, p.status); };
    auto next_stage = [&] {
      if (++stage == kPfRing) {
        stage = 0;
        phase ^= 1u;
      }
    };
    // S of tile t against the K block in the current stage
    auto issue_s = [&](int t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t da = umma_desc_sw128(smem_u32(sq + t * kPfTileBytes + h * kPfTileHalf));
        const uint64_t db = umma_desc_sw128(smem_u32(ring + stage * kPfBlockBytes + h * kPfBlockHalf));
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16(tmem + t * 128, da + 2 * k, db + 2 * k, idesc_s, (h | k) != 0);
      }
      umma_commit(&ctl.s_full[t]);
      any = true;
    };
    // one thread alone: a loop with warp collectives around each step took 1000
    // cycles per tile and block for the hand-offs alone (8192 tokens 607 -> 484 us)
    for (int u = 0; lane == 0 && ok; ++u) {
      const int us = u & 1;
      if (!wait(&ctl.u_full[us], (u >> 1) & 1)) { ok = false; break; }
      const PfWork w = ctl.work[us];
      mbar_arrive(&ctl.u_empty[us]);
      if (w.tokens == 0) break;
      const int tiles = w.tokens > p.tpt ? 2 : 1;
      const Blocks bl = blocks_of(w.pos0, w.pos0 + w.tokens - 1, p.window, p.sinks);
      if (!wait(&ctl.q_full, u & 1) || !wait(&ctl.kv_full[stage], phase)) { ok = false; break; }
      for (int t = 0; t < tiles; ++t) issue_s(t);
      umma_commit(&ctl.kv_empty[stage]);
      if (w.hi - w.lo == 1) umma_commit(&ctl.q_empty);
      next_stage();
      for (int i = w.lo; i < w.hi; ++i) {
        const int vs = stage;
        if (!wait(&ctl.kv_full[stage], phase)) { ok = false; break; }
        next_stage();
        // rows behind the sequence's end in its last page hold anything: their
        // weights are 0, and 0 times a NaN would not be (further pages are
        // loaded as zeros)
        const int live = w.kv - bl.at(i) * kPfBlock;
        if (live < kPfBlock) {
          uint8_t* v = ring + vs * kPfBlockBytes;
          const int end = (live + page_rows - 1) & ~(page_rows - 1);
          for (int x = live * 8; x < end * 8; ++x) {
            *reinterpret_cast<uint4*>(v + x * 16) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(v + kPfBlockHalf + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_shared();
        }
        // O += P V of block i, then, over P, S of block i + 1
        const bool more = i + 1 < w.hi;
        for (int t = 0; t < tiles; ++t) {
          if (!wait(&ctl.p_full[t], (pphase >> t) & 1u)) { ok = false; break; }
          pphase ^= 1u << t;
          tcgen05_fence_after();
          const uint64_t dv = umma_desc_sw128_mn(smem_u32(ring + vs * kPfBlockBytes), kPfBlockHalf);
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 positions: 2048 bytes of V, 8 columns of P
            umma_bf16_ts(tmem + kPfTmemO + t * 128, tmem + t * 128 + 8 * k, dv + 128 * k, idesc_o, i > w.lo || k != 0);
          if (more) {
            if (t == 0 && !wait(&ctl.kv_full[stage], phase)) { ok = false; break; }
            issue_s(t);
          } else {
            umma_commit(&ctl.o_full[t]);
          }
        }
        if (!ok) break;
        umma_commit(&ctl.kv_empty[vs]);
        if (more) {
          umma_commit(&ctl.kv_empty[stage]);
          if (i + 2 == w.hi) umma_commit(&ctl.q_empty);
          next_stage();
        }
      }
    }
    if (!ok && any) {  // issued MMAs end before tensor memory is released
      umma_commit(&ctl.drain);
      const long long t0 = clock64();
      while (!mbar_try_wait(&ctl.drain, 0) && clock64() - t0 < kWaitBudgetCycles / 8) {
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
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
#pragma unroll 1
      for (int i = w.lo; i < w.hi; ++i) {
        const int k0 = bl.at(i) * kPfBlock;
        if (!wait(&ctl.s_full[t], sphase)) { ok = false; break; }
        sphase ^= 1u;
        tcgen05_fence_after();
        uint32_t s[4][32];
        bool half_only = false;  // no row of the tile sees the second 64 columns: their weights are 0
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(ts + c * 32, s[c]);
        tmem_ld_wait();
        if (k0 + kPfBlock - 1 > tile_pos || (p.window && k0 <= tile_pos + p.tpt - 1 - p.window)) {
          // visible columns of each 32: up to hi, from lo on or below sk
          const int hi = pos - k0 + 1, lo = p.window ? hi - p.window : 0, sk = p.sinks - k0;
          // the last block of a pair is half unseen on average
          half_only = tile_pos + p.tpt - k0 <= kPfBlock / 2;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t see = low_bits(hi - c * 32) & (~low_bits(lo - c * 32) | low_bits(sk - c * 32));
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (!((see >> x) & 1u)) s[c][x] = 0xff800000u;
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four short chains
#pragma unroll
        for (int c = 0; c < 128; c += 2)
          mx4[(c >> 1) & 3] = max3(mx4[(c >> 1) & 3], __uint_as_float(s[c >> 5][c & 31]), __uint_as_float(s[c >> 5][(c & 31) + 1]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
        const bool raise = mx > m + kPfSlack;  // the first finite maximum too: m is -inf
        if (__any_sync(0xffffffffu, raise)) {
          const float mn = raise ? mx : m;
          if (i > w.lo) {
            // every lane takes part; lanes that keep their maximum multiply by
            // 1.  All products so far are done: this block's S came after them.
            const float f = raise ? ex2(m - mn) : 1.f;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {  // rolled: rare
              uint32_t o[16];
              tmem_ld_32x32b_x16(to + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st_32x32b_x16(to + c * 16, o);
            }
          }
          m = mn;
        }
        const float ms = m == -INFINITY ? 0.f : m;
        const uint64_t sc2 = pair2(p.scale_log2, p.scale_log2), ms2 = pair2(-ms, -ms);
        uint64_t sum[4] = {0, 0, 0, 0};
        auto weigh = [&](int c) {
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const uint64_t y = fma2(pair2(__uint_as_float(s[c][2 * x]), __uint_as_float(s[c][2 * x + 1])), sc2, ms2);
            float2 e = split2(y);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[x & 3] = add2(sum[x & 3], pair2(e.x, e.y));
            pk[x] = pack_bf16x2(e.x, e.y);
          }
          tmem_st_32x32b_x16(ts + c * 16, pk);
        };
        weigh(0);
        weigh(1);
        if (half_only) {
          const uint32_t none[16] = {};
          tmem_st_32x32b_x16(ts + 32, none);
          tmem_st_32x32b_x16(ts + 48, none);
        } else {
          weigh(2);
          weigh(3);
        }
        const float2 sums = split2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
        l += sums.x + sums.y;
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
      const long long out_at =
          mine ? ((static_cast<long long>(w.row0) + t * p.tpt + token) * p.nq + w.j * p.grp + head) * kHeadDim : -1;
      float* part = w.slot >= 0 ? p.part + (static_cast<long long>(w.slot) * 2 + t) * kPfPartTile : nullptr;
      // where this lane stores: row 8 k + lane / 4, columns 8 (lane % 4) of each 32
      __nv_bfloat16* to_row[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long at = __shfl_sync(0xffffffffu, out_at, k * 8 + (lane >> 2));
        to_row[k] = at >= 0 ? p.out + at + (lane & 3) * 8 : nullptr;
      }
      uint32_t o[4][32];  // all at once: 8 x 512 tokens 37.8 -> 37.4 us against 32 columns at a time
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(to + c * 32, o[c]);
      tmem_ld_wait();
      if (part) {
#pragma unroll
        for (int x = 0; x < 128; x += 4)
          __stcg(reinterpret_cast<uint4*>(part) + (x / 4) * kPfRows + row,
                 make_uint4(o[x >> 5][x & 31], o[x >> 5][(x & 31) + 1], o[x >> 5][(x & 31) + 2], o[x >> 5][(x & 31) + 3]));
      } else {
        // through shared memory: eight rows of 64 bytes per store instead of
        // 32 rows of 16
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[c][x + e]) * inv;
            *reinterpret_cast<uint4*>(&stg[warp - 4][lane][x]) = pack8(f);
          }
          __syncwarp();
          uint4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const uint4*>(&stg[warp - 4][k * 8 + (lane >> 2)][(lane & 3) * 8]);
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (to_row[k]) *reinterpret_cast<uint4*>(to_row[k] + c * 32) = v[k];
        }
      }
      if (part) {
        __stcg(part + kHeadDim * kPfRows + row, m);
        __stcg(part + (kHeadDim + 1) * kPfRows + row, l);
      }
      tcgen05_fence_before();  // the next unit's MMAs follow this thread's next arrival
    }
  }

  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a cut pair, in order: a CTA per (pair and kv head, 32
// rows), a lane per row, a warp per 16 columns.
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const __grid_constant__ PfParams p) {
  pdl_launch_dependents();
  pdl_wait();
  if (p.list->share == 0) return;
  const int cta = blockIdx.x >> 3, tile = (blockIdx.x >> 2) & 1;
  const int lane = threadIdx.x & 31, col = (threadIdx.x >> 5) * 16, row = (blockIdx.x & 3) * 32 + lane;
  const PfSplit sp = p.splits[cta];
  if (sp.parts == 0) return;
  const PfUnit un = p.units[sp.pair];
  const int token = row / p.grp, head = row - token * p.grp;
  if (token >= p.tpt || tile * p.tpt + token >= un.tokens) return;
  auto part_of = [&](int s) {
    const int slot = 2 * (cta + s) + (s == 0);
    return p.part + (static_cast<long long>(slot) * 2 + tile) * kPfPartTile;
  };
  float m = -INFINITY;
  for (int s = 0; s < sp.parts; ++s) m = fmaxf(m, __ldcg(part_of(s) + kHeadDim * kPfRows + row));
  float l = 0.f, o[16];
#pragma unroll
  for (int x = 0; x < 16; ++x) o[x] = 0.f;
  for (int s = 0; s < sp.parts; ++s) {
    const float* from = part_of(s);
    float4 v[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = __ldcg(reinterpret_cast<const float4*>(from) + (col / 4 + x) * kPfRows + row);
    const float f = m == -INFINITY ? 0.f : exp2f(__ldcg(from + kHeadDim * kPfRows + row) - m);
    l = fmaf(f, __ldcg(from + (kHeadDim + 1) * kPfRows + row), l);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      o[4 * x] = fmaf(f, v[x].x, o[4 * x]);
      o[4 * x + 1] = fmaf(f, v[x].y, o[4 * x + 1]);
      o[4 * x + 2] = fmaf(f, v[x].z, o[4 * x + 2]);
      o[4 * x + 3] = fmaf(f, v[x].w, o[4 * x + 3]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  __nv_bfloat16* dst =
      p.out + ((static_cast<long long>(un.row0) + tile * p.tpt + token) * p.nq + sp.j * p.grp + head) * kHeadDim + col;
#pragma unroll
  for (int x = 0; x < 16; x += 8) {
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = o[x + e] * inv;
    *reinterpret_cast<uint4*>(dst + x) = pack8(h);
  }
}

// Sizes that the host can bound without the lengths.
struct PfLayout {
  long long pairs, grid;  // grid: of the main kernel
  bool may_cut;
  size_t list, units, offs, splits, starts, part, total;
};

PfLayout pf_layout(long long T, long long B, int nkv, int grp, long long max_pages, int page_size) {
  PfLayout L;
  const int tpt = kPfRows / grp;
  L.pairs = T / (2 * tpt) + B;
  const long long blocks = (max_pages * page_size + kPfBlock - 1) / kPfBlock;
  const long long most = L.pairs * nkv * ((blocks + kPfMinBlocks - 1) / kPfMinBlocks);  // runs at least
  L.grid = device_sm_count();
  if (most < L.grid) L.grid = most;
  L.may_cut = blocks > kPfMinBlocks;
  auto round = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
  size_t at = kPagedScratch;
  L.list = at;
  at += 256;
  L.units = at;
  at += round(sizeof(PfUnit) * L.pairs);
  L.offs = at;
  at += round(sizeof(int) * (L.pairs + 1));
  L.splits = at;
  at += round(sizeof(PfSplit) * L.grid);
  L.starts = at;
  at += round(sizeof(int) * (B + 1));
  L.part = at;
  if (L.may_cut) at += sizeof(float) * 2 * L.grid * 2 * kPfPartTile;
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
  if (!tmap_of_rows(encode, &mq, q, nq, T, q_stride, grp, tpt) || !tmap_of_pages(encode, &mk, cache, false) ||
      !tmap_of_pages(encode, &mv, cache, true))
    return cudaErrorInvalidValue;
  const PfLayout L = pf_layout(T, B, nkv, grp, cache.max_pages, page);
  char* ws = static_cast<char*>(workspace);
  PfParams p;
  p.cu = cu_seqlens;
  p.kv_lens = kv_lens;
  p.out = out;
  p.status = reinterpret_cast<int*>(ws);
  p.list = reinterpret_cast<PfList*>(ws + L.list);
  p.units = reinterpret_cast<PfUnit*>(ws + L.units);
  p.offs = reinterpret_cast<int*>(ws + L.offs);
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
  p.sms = static_cast<int>(L.grid);
  p.max_pairs = static_cast<int>(L.pairs);
  p.scale_log2 = scale * kPfLog2e;
  cudaError_t e = launch_pdl(paged_prefill_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
  if (e != cudaSuccess) return e;
  e = allow_smem<paged_prefill_kernel>(static_cast<int>(kPfSmem));
  if (e != cudaSuccess) return e;
  e = launch_pdl(paged_prefill_kernel, dim3(p.sms), dim3(kPfThreads), kPfSmem, s, mq, mk, mv, p);
  if (e != cudaSuccess || !L.may_cut) return e;
  return launch_pdl(paged_prefill_join_kernel, dim3(8 * p.sms), dim3(256), 0, s, p);
}

}  // namespace nkimoe
