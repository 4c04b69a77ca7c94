// Attention of trees of drafted tokens over a paged key-value cache (grouped-
// query attention, head_dim 128, optionally a sliding window with a few first
// positions that stay visible) on the 5th-generation tensor cores.
//
//   out_i = sum_s softmax_s(q_i . k_s * scale) v_s
//
// over the places s that node i sees: those before the tree (in the window),
// its ancestors and itself.  A node's place in the cache is where its row stands
// in the tree, its position the length before the tree and its depth.
//
// The store before it (paged_store.cu) norms and turns the rows, puts keys and
// values in their pages and the queries in the workspace, and works out every
// node's line of ancestors as 64 bits; a kernel after it joins what was cut.
//
// Tile: 128 MMA rows are floor(128 / group) nodes times the `group` query heads
// of one kv head, against key blocks of 128 places.  One warp loads Q and K, one
// V, one thread each issues the MMAs of scores and of products, and two warpgroups take S from tensor memory,
// a thread per row, and leave P there.  The warpgroups take a tile's blocks in
// turn, each with its own maximum, sum and O, which are joined at its end: a
// block's chain (scores, softmax, product, 4000 cycles) takes longer than its
// bytes take to come from HBM (2800), two chains at a time do not.
//
// Arithmetic: bf16 operands, sums, maxima and O in fp32.  Queries enter as a sum
// of two bf16 (hi + lo, 2^-17) by a second MMA into the same scores; weights are
// rounded to bf16 (2^-9 at most, random over the terms of a sum).  With the
// queries rounded too the output's error against 64 bits is 1.8 times that of its
// own rounding, so 1.4 times; weights as hi + lo bring it to 1.0, but take 2500
// cycles more per block (37 sequences of 16 nodes over 16 K: 290 us, so 228, and
// with rounded queries 201).  The attention of prompts rounds its weights the same way;
// the decode step, whose MMAs have idle rows for it, keeps them to 2^-17, so logits
// after a node are not bit for bit those of a decode step.
//
// Work: the blocks of all (sequence, kv head, tile) form one list, and every CTA
// takes an equal run of it, so sequences of any mix of lengths load all SMs alike
// and the launch needs no length on the host.  Each CTA finds its run from the
// lengths itself, and loads its first keys, while the store still runs: the
// store lets this kernel start only once all that came before it has ended, so
// what the store does not write may be read at once.
//
// Bounds and figures (B200, 32 heads over 4, all three kernels; replays, so from the L2
// as far as the cache fits, in brackets from HBM): trees of 13 over 30011
// places 29 us (36), 40 ragged ones over 1 to 32768 72 us (77, 3.8 TB/s of 6.5): 1.6 us per
// block of a CTA, beginnings and ends of items, and 2 to 2.5 us for each kernel's
// start.  8 trees of 8 over 512 to 639: 18 us (24), that chain with two blocks.  16 trees
// of 49 to 64 nodes: 111 us (119), two chains of scores, softmax and products per SM.
#include "paged_tree.cuh"

namespace nkimoe {

namespace {

constexpr int kTrThreads = 384;
constexpr int kTrK = 3, kTrV = 2;  // stages of 32 KB: K blocks, V blocks
constexpr int kTrItem = 2;         // key blocks that beginning and ending an item (sequence, kv head, tile) costs:
                                   // 40 ragged sequences 114 us at 0, 80 at 1, 71 at 2, 72 at 3, 73 at 4
constexpr int kTrMinRun = 3;       // places of a CTA's run at least
// A part of a cut item: o four columns at a time [32][128 rows][4], then the
// rows' m, then their l (a warp's rows are neighbours: coalesced)
constexpr int kTrPart = (kHeadDim + 2) * kPfRows;
constexpr int kTrJoinRows = 8;     // rows per CTA of the join

// What a CTA began and others went on with: the item whose parts lie in slot
// 2 c + 1 of CTA c and the slots 0 of the CTAs after it.
struct TrSplit {
  int row0, tokens, j, parts;
};

struct TrParams {
  const int* cu;       // [B + 1]
  const int* kv_lens;  // [B]
  __nv_bfloat16* out;  // [T, nq * 128]
  int* status;
  const TrRow* rows;  // [T]
  TrSplit* splits;    // [grid]
  float* part;        // [2 grid, kTrPart]
  PagedCache c;
  int T, B, nq, grp, tpt;  // tpt: nodes per tile
  int window, sinks;
  float scale_log2;
};

// What the roles need to know of an item; tokens 0: there are no more.
struct TrWork {
  int row0;    // first packed row of the tile
  int tokens;  // its nodes
  int past;    // places before the tree
  int kv;      // places with it
  int b, j;    // sequence, kv head
  int lo, hi;  // range of key blocks
  int slot;    // of the partial result, or -1
};

struct TrCtl {
  uint64_t q_full, q_empty;
  uint64_t k_full[kTrK], k_empty[kTrK];
  uint64_t v_full[kTrV], v_empty[kTrV];
  uint64_t s_full[2], p_full[2], pv_done[2], o_full[2];
  uint64_t u_full[2], u_empty[2];
  uint64_t ml_full, ml_empty;  // the softmax warps have left their maxima and sums; have read them and both O
  uint64_t tail, drain[2];
  TrWork work[2];
  uint32_t tmem_base;
  int abort_flag;
  float2 ml[2][kPfRows];  // maximum and sum of both warpgroups
};

struct TrShared {  // on a 1024-byte boundary: the tiles are swizzled
  uint8_t q[2][kPfTileBytes];  // hi, lo
  uint8_t k[kTrK][kPfBlockBytes];
  uint8_t v[kTrV][kPfBlockBytes];
  TrCtl ctl;
};
static_assert(sizeof(TrShared) <= 227 * 1024, "shared memory of an SM");

// A sequence's nodes and lengths; n 0: none, or they make no sense (flagged).
struct TrSeq {
  int row0, n, kv, blocks;
};
__device__ __forceinline__ TrSeq tr_sequence(const TrParams& p, int b, bool flag) {
  TrSeq s{0, 0, 0, 0};
  if (b >= p.B) return s;
  s.row0 = p.cu[b];
  s.kv = p.kv_lens[b];
  const int end = p.cu[b + 1];
  if (s.row0 == end) return s;
  // (the order first: the difference of two that make no sense may pass 32 bits)
  if (s.row0 < 0 || end < s.row0 || end > p.T || end - s.row0 > kTreeNodes || s.kv < end - s.row0 ||
      s.kv > static_cast<long long>(p.c.max_pages) << p.c.page_shift) {
    if (flag) atomicOr(p.status, kDevErrBadIndex);
    return s;
  }
  s.n = end - s.row0;
  s.blocks = blocks_of(s.kv - s.n, s.kv - 1, p.window, p.sinks).n;
  return s;
}

// The run of one CTA through the list of blocks (sequence, kv head, tile, block),
// each item preceded by places for its own cost; a warp walks it.  Where two blocks
// a CTA are enough for all, items begin at even places instead, so that no CTA
// has a block each of two items.
struct TrRun {
  bool pairs;
  int share, run_lo, run_hi;
  int at;    // place in the list
  int base;  // place of the first of sequence b
  int b;
  TrSeq mine;  // of sequence 32 * (b / 32) + lane

  __device__ __forceinline__ int tiles(const TrParams& p, const TrSeq& s) const { return (s.n + p.tpt - 1) / p.tpt; }
  __device__ __forceinline__ int cost() const { return pairs ? 0 : kTrItem; }
  __device__ __forceinline__ int span(const TrSeq& s) const {  // places of an item
    return pairs ? (s.blocks + 1) & ~1 : s.blocks + kTrItem;
  }
  __device__ __forceinline__ int places(const TrParams& p, const TrSeq& s) const {
    return tiles(p, s) * p.c.nkv * span(s);
  }
  __device__ __forceinline__ TrSeq of(int b) const {
    const int l = b & 31;
    return TrSeq{__shfl_sync(0xffffffffu, mine.row0, l), __shfl_sync(0xffffffffu, mine.n, l),
                 __shfl_sync(0xffffffffu, mine.kv, l), __shfl_sync(0xffffffffu, mine.blocks, l)};
  }

  __device__ __forceinline__ void begin(const TrParams& p, int lane) {
    int total = 0, even = 0;
    for (int c = 0; c < p.B; c += 32) {
      mine = tr_sequence(p, c + lane, blockIdx.x == 0);
      pairs = true;
      even += __reduce_add_sync(0xffffffffu, places(p, mine));
      pairs = false;
      total += __reduce_add_sync(0xffffffffu, places(p, mine));
    }
    const int ctas = gridDim.x;
    pairs = even <= 2 * ctas;
    if (pairs) total = even;
    share = pairs ? 2 : max(kTrMinRun, (total + ctas - 1) / ctas);
    run_lo = min(total, static_cast<int>(blockIdx.x) * share);
    run_hi = min(total, run_lo + share);
    at = run_lo;
    base = b = 0;
    if (at >= run_hi) return;
    // the sequence of place `at`
    for (int c = 0;; c += 32) {
      if (p.B > 32) mine = tr_sequence(p, c + lane, false);
      int incl = places(p, mine);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const int all = __shfl_sync(0xffffffffu, incl, 31);
      if (base + all <= at) {
        base += all;
        continue;
      }
      const int l = __ffs(__ballot_sync(0xffffffffu, base + incl > at)) - 1;
      b = c + l;
      const int before = __shfl_sync(0xffffffffu, incl, l > 0 ? l - 1 : 0);
      if (l > 0) base += before;
      return;
    }
  }

  // The run's next item, or one without nodes.
  __device__ __forceinline__ TrWork next(const TrParams& p, int lane) {
    TrWork w{};
    if (at >= run_hi) return w;
    TrSeq s = of(b);
    while (at >= base + places(p, s)) {  // (there is a next one: at < run_hi <= the whole list)
      base += places(p, s);
      ++b;
      if ((b & 31) == 0) mine = tr_sequence(p, b + lane, false);
      s = of(b);
    }
    const int n = s.blocks, tls = tiles(p, s);
    const int q = (at - base) / span(s);
    const int item = base + q * span(s) + cost();  // the list's first block of the item
    const int tile = q % tls;
    w.lo = max(at - item, 0);
    w.hi = min(n, run_hi - item);
    at = base + (q + 1) * span(s);
    if (w.hi <= 0) return TrWork{};  // the run ends before the item's blocks
    w.row0 = s.row0 + tile * p.tpt;
    w.tokens = min(p.tpt, s.n - tile * p.tpt);
    w.past = s.kv - s.n;
    w.kv = s.kv;
    w.b = b;
    w.j = q / tls;
    const int first = item / share, parts = (item + n - 1) / share - first + 1;
    w.slot = parts > 1 ? 2 * static_cast<int>(blockIdx.x) + (item < run_lo ? 0 : 1) : -1;
    if (parts > 1 && item >= run_lo && lane == 0) p.splits[blockIdx.x] = TrSplit{w.row0, w.tokens, w.j, parts};
    return w;
  }
};

__global__ void __launch_bounds__(kTrThreads, 1)
    paged_tree_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_lo,
                      const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                      const __grid_constant__ TrParams p) {
  extern __shared__ __align__(1024) uint8_t tr_raw[];
  TrShared& sh = *reinterpret_cast<TrShared*>(tr_raw);
  TrCtl& ctl = sh.ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(tr_raw) & 1023u) {  // never: the kernel has no other shared memory
    if (threadIdx.x == 0) atomicOr(p.status, kDevErrTmem);
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, 1);
    mbar_init(&ctl.q_empty, 1);
    for (int s = 0; s < kTrK; ++s) {
      mbar_init(&ctl.k_full[s], 1);
      mbar_init(&ctl.k_empty[s], 1);
    }
    for (int s = 0; s < kTrV; ++s) {
      mbar_init(&ctl.v_full[s], 1);
      mbar_init(&ctl.v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctl.s_full[t], 1);
      mbar_init(&ctl.p_full[t], 4);  // one arrival per softmax warp
      mbar_init(&ctl.pv_done[t], 1);
      mbar_init(&ctl.o_full[t], 1);
      mbar_init(&ctl.u_full[t], 1);
      mbar_init(&ctl.u_empty[t], 3 + 8);  // the MMA warps, the warp that loads V, the softmax warps
    }
    mbar_init(&ctl.ml_full, 8);
    mbar_init(&ctl.ml_empty, 8);
    mbar_init(&ctl.tail, 1);
    mbar_init(&ctl.drain[0], 1);
    mbar_init(&ctl.drain[1], 1);
    ctl.abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_lo);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  if (warp == 1) tmem_alloc(&ctl.tmem_base, 512);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = ctl.tmem_base;
  pdl_launch_dependents();
  // 384 x 168 registers at launch = 128 x 88 + 256 x 208
  if (warp == 0 || warp == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ---------------------------------------------------------------- items and loads
    // Lane (h, g) loads half h of page g of a block.
    const int v = warp >> 1;
    const int stages = v ? kTrV : kTrK;
    uint8_t* const ring = v ? &sh.v[0][0] : &sh.k[0][0];
    uint64_t* const full = v ? ctl.v_full : ctl.k_full;
    uint64_t* const empty = v ? ctl.v_empty : ctl.k_empty;
    const int h_lane = (lane >> 3) & 1, g_lane = lane & 7;
    const int page_rows = min(1 << p.c.page_shift, kPfBlock);  // rows per box
    const bool loads = lane < 16 && g_lane * page_rows < kPfBlock;
    const void* const tm = v ? static_cast<const void*>(&tmap_v) : static_cast<const void*>(&tmap_k);
    const int box_at = h_lane * static_cast<int>(kPfBlockHalf) + g_lane * page_rows * 128;
    const uint32_t q_bytes = 2u * p.grp * p.tpt * 128u;  // both halves of the tile's box
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      const bool got = mbar_wait(bar, ph, &ctl.abort_flag, p.status);
      return __all_sync(0xffffffffu, got);
    };
    int stage = 0;
    uint32_t phase = 0, issued = 0, last_phase = 0, tail_phase = 0;
    bool ok = true, q_issued = false;
    bool stored = false;  // the store before this kernel has ended
    auto after_store = [&] {
      if (!stored) pdl_wait();
      stored = true;
    };
    TrRun run;
    if (v == 0) {
      if (lane == 0) p.splits[blockIdx.x].parts = 0;
      run.begin(p, lane);
    }
    for (int u = 0; ok; ++u) {
      const int us = u & 1;
      TrWork w;
      if (v) {
        if (!wait(&ctl.u_full[us], (u >> 1) & 1)) { ok = false; break; }
        w = ctl.work[us];
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.u_empty[us]);
      } else {
        if (!wait(&ctl.u_empty[us], ((u >> 1) & 1) ^ 1u)) { ok = false; break; }
        w = run.next(p, lane);
        if (lane == 0) {
          ctl.work[us] = w;
          mbar_arrive(&ctl.u_full[us]);
        }
      }
      if (w.tokens == 0) break;
      const Blocks bl = blocks_of(w.past, w.kv - 1, p.window, p.sinks);
      // places that some node of the tree sees; a page outside is read as zeros
      const int last = w.kv - 1;
      const int start = p.window && w.past >= p.window ? w.past - p.window + 1 : 0;
      const int* table = p.c.table + w.b * p.c.table_stride;
      auto look_up = [&](int i) {
        const int s0 = bl.at(i) * kPfBlock + g_lane * page_rows;
        const bool need = loads && s0 <= last && (s0 + page_rows > start || s0 < p.sinks);
        return need ? table[s0 >> p.c.page_shift] : -2;
      };
      int next = look_up(w.lo);
      for (int i = w.lo; ok && i < w.hi; ++i) {
        const bool held = next >= 0 && next < p.c.num_pages;
        if (!held && next != -2) atomicOr(p.status, kDevErrBadIndex);
        const int page = held ? next : p.c.num_pages;  // past the last page: the load fills zeros
        const int k0 = bl.at(i) * kPfBlock;
        const int in_page = (k0 + g_lane * page_rows) & ((1 << p.c.page_shift) - 1);
        if (i + 1 < w.hi) next = look_up(i + 1);  // in flight while this block waits for its stage
        if (!wait(&empty[stage], phase ^ 1u)) { ok = false; break; }
        if (k0 + kPfBlock > w.past) after_store();  // the tree's own rows are in the block
        // rows behind the sequence's end in its last page hold anything: their
        // weights are 0, and 0 times a NaN would not be, so this warp clears
        // them once the block is there (further pages are loaded as zeros)
        const int live = w.kv - k0;
        const bool clear = v == 1 && live < kPfBlock && (live & (page_rows - 1)) != 0;
        uint64_t* const bar = clear ? &ctl.tail : &full[stage];
        if (lane == 0) mbar_arrive_expect_tx(bar, kPfBlockBytes);
        __syncwarp();
        uint8_t* const to = ring + stage * kPfBlockBytes;
        if (loads) tma_load_4d(to + box_at, tm, bar, h_lane * 64, in_page, w.j, page);
        if (clear) {
          if (!wait(&ctl.tail, tail_phase)) { ok = false; break; }
          tail_phase ^= 1u;
          const int end = (live + page_rows - 1) & ~(page_rows - 1);
          for (int x = live * 8 + lane; x < end * 8; x += 32) {
            *reinterpret_cast<uint4*>(to + x * 16) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(to + kPfBlockHalf + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[stage]);
        }
        issued |= 1u << stage;
        last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
        // the item's queries after its first keys, which may go out before the store
        // has ended, and while the item before still reads its own queries
        if (v == 0 && i == w.lo) {
          if (!wait(&ctl.q_empty, (u & 1) ^ 1u)) { ok = false; break; }
          after_store();
          if (lane == 0) mbar_arrive_expect_tx(&ctl.q_full, 2 * q_bytes);
          __syncwarp();
          if (lane < 4)
            tma_load_3d(sh.q[lane >> 1] + (lane & 1) * kPfTileHalf, lane < 2 ? &tmap_q : &tmap_lo, &ctl.q_full,
                        (lane & 1) * 64, w.j * p.grp, w.row0);
          q_issued = true;
        }
      }
    }
    after_store();
    if (!ok && lane == 0) {  // let the copies in flight land before the CTA exits
      for (int s = 0; s < stages; ++s)
        if ((issued >> s) & 1u) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&full[s], (last_phase >> s) & 1u) && clock64() - t0 < kWaitBudgetCycles / 8) {
          }
        }
      if (q_issued || v) {
        const long long t0 = clock64();
        while (clock64() - t0 < kWaitBudgetCycles / 64) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ---------------------------------------------------------------- scores (one thread)
    constexpr uint32_t idesc_s = umma_idesc_bf16_f32(kPfRows, kPfBlock);
    int ks = 0;
    uint32_t kphase = 0, dphase = 3;  // dphase: bit t, of pv_done (nothing to wait for at first)
    bool ok = true, any = false;
    auto wait = [&](uint64_t* bar, uint32_t ph) { return mbar_wait(bar, ph, &ctl.abort_flag, p.status); };
    for (int u = 0; lane == 0 && ok; ++u) {
      const int us = u & 1;
      if (!wait(&ctl.u_full[us], (u >> 1) & 1)) { ok = false; break; }
      const int tokens = ctl.work[us].tokens, n = ctl.work[us].hi - ctl.work[us].lo;
      mbar_arrive(&ctl.u_empty[us]);
      if (tokens == 0) break;
      if (!wait(&ctl.q_full, u & 1)) { ok = false; break; }
      for (int i = 0; i < n; ++i) {  // block i is warpgroup i % 2's
        const int t = i & 1;
        // over P, which the product of the warpgroup's block before has read
        if (!wait(&ctl.pv_done[t], (dphase >> t) & 1u) || !wait(&ctl.k_full[ks], kphase)) { ok = false; break; }
        dphase ^= 1u << t;
        tcgen05_fence_after();
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint64_t da = umma_desc_sw128(smem_u32(sh.q[q] + h * kPfTileHalf));
            const uint64_t db = umma_desc_sw128(smem_u32(sh.k[ks] + h * kPfBlockHalf));
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_bf16(tmem + t * 128, da + 2 * k, db + 2 * k, idesc_s, (q | h | k) != 0);
          }
        any = true;
        umma_commit(&ctl.s_full[t]);
        umma_commit(&ctl.k_empty[ks]);
        if (++ks == kTrK) {
          ks = 0;
          kphase ^= 1u;
        }
      }
      if (ok) umma_commit(&ctl.q_empty);
    }
    if (!ok && any) {  // issued MMAs end before tensor memory is released
      umma_commit(&ctl.drain[0]);
      const long long t0 = clock64();
      while (!mbar_try_wait(&ctl.drain[0], 0) && clock64() - t0 < kWaitBudgetCycles / 8) {
      }
    }
    __syncwarp();
    pdl_wait();
  } else if (warp == 3) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ---------------------------------------------------------------- products (one thread)
    constexpr uint32_t idesc_o = umma_idesc_bf16_f32(kPfRows, kHeadDim) | (1u << 16);  // B is MN-major
    int vs = 0;
    uint32_t vphase = 0, pphase = 0;  // pphase: bit t, of p_full
    bool ok = true, any = false;
    auto wait = [&](uint64_t* bar, uint32_t ph) { return mbar_wait(bar, ph, &ctl.abort_flag, p.status); };
    for (int u = 0; lane == 0 && ok; ++u) {
      const int us = u & 1;
      if (!wait(&ctl.u_full[us], (u >> 1) & 1)) { ok = false; break; }
      const int tokens = ctl.work[us].tokens, n = ctl.work[us].hi - ctl.work[us].lo;
      mbar_arrive(&ctl.u_empty[us]);
      if (tokens == 0) break;
      for (int i = 0; i < n; ++i) {
        const int t = i & 1;
        if (!wait(&ctl.v_full[vs], vphase) || !wait(&ctl.p_full[t], (pphase >> t) & 1u)) { ok = false; break; }
        pphase ^= 1u << t;
        tcgen05_fence_after();
        const uint64_t dv = umma_desc_sw128_mn(smem_u32(sh.v[vs]), kPfBlockHalf);
#pragma unroll
        for (int k = 0; k < 8; ++k)  // 16 positions: 2048 bytes of V, 8 columns of P
          umma_bf16_ts(tmem + kPfTmemO + t * 128, tmem + t * 128 + 8 * k, dv + 128 * k, idesc_o, i > 1 || k != 0);
        any = true;
        umma_commit(&ctl.pv_done[t]);
        umma_commit(&ctl.v_empty[vs]);
        if (i + 2 >= n) umma_commit(&ctl.o_full[t]);
        if (++vs == kTrV) {
          vs = 0;
          vphase ^= 1u;
        }
      }
    }
    if (!ok && any) {
      umma_commit(&ctl.drain[1]);
      const long long t0 = clock64();
      while (!mbar_try_wait(&ctl.drain[1], 0) && clock64() - t0 < kWaitBudgetCycles / 8) {
      }
    }
    __syncwarp();
    pdl_wait();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---------------------------------------------------------------- softmax, one row per thread
    const int g = (warp - 4) >> 2, quarter = warp & 3;  // warpgroup
    const int row = quarter * 32 + lane;
    const int token = row / p.grp, head = row - token * p.grp;
    const uint32_t ts = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + g * 128;
    const uint32_t to = ts + kPfTmemO;
    uint32_t sphase = 0, ophase = 0, jphase = 0;
    auto wait = [&](uint64_t* bar, uint32_t ph) {
      const bool got = mbar_wait(bar, ph, &ctl.abort_flag, p.status);
      return __all_sync(0xffffffffu, got);
    };
    pdl_wait();
    for (int u = 0;; ++u) {
      const int us = u & 1;
      if (!wait(&ctl.u_full[us], (u >> 1) & 1)) break;
      const TrWork w = ctl.work[us];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.u_empty[us]);
      if (w.tokens == 0) break;
      const bool mine = token < w.tokens;
      TrRow info{0, w.past, 0};
      if (mine) info = p.rows[w.row0 + token];
      const Blocks bl = blocks_of(w.past, w.kv - 1, p.window, p.sinks);
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      const int first = w.lo + g;
#pragma unroll 1
      for (int i = first; i < w.hi; i += 2) {
        const int k0 = bl.at(i) * kPfBlock;
        if (!wait(&ctl.s_full[g], sphase)) { ok = false; break; }
        sphase ^= 1u;
        tcgen05_fence_after();
        uint32_t s[4][32];
        const bool half_only = w.kv - k0 <= kPfBlock / 2;  // no row sees the second 64 columns: their weights are 0
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(ts + c * 32, s[c]);
        tmem_ld_wait();
        if (k0 + kPfBlock > w.past || (p.window && k0 <= w.past + kTreeNodes - p.window)) {
          // visible columns of each 32: places before the tree, from lo on or below sk; nodes of the row's line
          const int hi = w.past - k0, lo = p.window ? info.pos - k0 - p.window + 1 : 0, sk = p.sinks - k0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int d = c * 32 - hi;  // column 0 of these 32 is node d
            const uint32_t nodes = d >= 64 || d <= -32 ? 0u
                                   : d >= 0 ? static_cast<uint32_t>(info.line >> d)
                                            : static_cast<uint32_t>(info.line) << -d;
            const uint32_t see = (low_bits(hi - c * 32) & (~low_bits(lo - c * 32) | low_bits(sk - c * 32))) | nodes;
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
          if (i > first) {
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
        if (lane == 0) mbar_arrive(&ctl.p_full[g]);
      }
      if (!ok) break;
      if (first < w.hi) {
        if (!wait(&ctl.o_full[g], ophase)) break;
        ophase ^= 1u;
      }
      float own = 1.f, other = 0.f;  // what this warpgroup's O and the other's are multiplied by
      const bool joined = w.hi - w.lo > 1;
      if (joined) {
        ctl.ml[g][row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.ml_full);
        if (!wait(&ctl.ml_full, jphase)) break;
        const float2 o = ctl.ml[1 - g][row];
        const float mn = fmaxf(m, o.x);
        own = m == -INFINITY ? 0.f : ex2(m - mn);
        other = o.x == -INFINITY ? 0.f : ex2(o.x - mn);
        l = l * own + o.y * other;
        m = mn;
      }
      tcgen05_fence_after();
      float* const part = w.slot >= 0 ? p.part + static_cast<long long>(w.slot) * kTrPart : nullptr;
      if (!part) {
        const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
        own *= inv;
        other *= inv;
      }
      // columns [64 g, 64 g + 64) of both O, or all of the one
      const int c_lo = joined ? 2 * g : 0, c_hi = joined ? 2 * g + 2 : g ? 0 : 4;
      const uint32_t to_other = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (1 - g) * 128 + kPfTmemO;
      __nv_bfloat16* const dst =
          p.out + ((static_cast<long long>(w.row0) + token) * p.nq + w.j * p.grp + head) * kHeadDim;
      __syncwarp();
#pragma unroll 1
      for (int c = c_lo; c < c_hi; ++c) {
        uint32_t o[32], q[32];
        tmem_ld_32x32b_x32(to + c * 32, o);
        if (joined) tmem_ld_32x32b_x32(to_other + c * 32, q);
        tmem_ld_wait();
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          const float a = __uint_as_float(o[x]) * own;
          o[x] = __float_as_uint(joined ? fmaf(__uint_as_float(q[x]), other, a) : a);
        }
        if (mine && part) {
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            __stcg(reinterpret_cast<uint4*>(part) + (c * 8 + x / 4) * kPfRows + row, make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]));
        } else if (mine) {
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[x + e]);
            *reinterpret_cast<uint4*>(dst + c * 32 + x) = pack8(f);
          }
        }
        __syncwarp();  // before the next load from tensor memory
      }
      if (part && mine && c_lo == 0 && c_hi > 0) {
        __stcg(part + kHeadDim * kPfRows + row, m);
        __stcg(part + (kHeadDim + 1) * kPfRows + row, l);
      }
      __syncwarp();
      tcgen05_fence_before();  // the next item's MMAs follow this thread's next arrival
      if (joined) {  // they, and the next maxima, wait until both warpgroups have read both
        if (lane == 0) mbar_arrive(&ctl.ml_empty);
        if (!wait(&ctl.ml_empty, jphase)) break;
        jphase ^= 1u;
      }
    }
  }

  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a cut item, in order: a CTA per (item, 8 rows), a thread per
// row and four columns, 13 parts in flight (a third of the 37 that one sequence of 4 kv
// heads has on 148 SMs, whatever its length; more parts take more turns).  (With a few CTAs that take slices in
// turn the ragged batch takes 6 us more.)
__global__ void __launch_bounds__(32 * kTrJoinRows) paged_tree_join_kernel(const __grid_constant__ TrParams p) {
  constexpr int kSlices = kPfRows / kTrJoinRows, kAhead = 13, kFew = 4;
  extern __shared__ float2 factor[];  // [parts][rows]: maximum and sum, then the weight and the sum's share
  __shared__ float whole[kTrJoinRows];
  __shared__ unsigned most[kTrJoinRows];
  const int cta = blockIdx.x / kSlices, row0 = (blockIdx.x % kSlices) * kTrJoinRows;
  const int r = threadIdx.x % kTrJoinRows, col4 = threadIdx.x / kTrJoinRows, row = row0 + r;
  pdl_launch_dependents();
  pdl_wait();
  const TrSplit sp = p.splits[cta];
  if (sp.parts == 0 || row0 >= sp.tokens * p.grp) return;
  auto part_of = [&](int s) { return p.part + static_cast<long long>(2 * (cta + s) + (s == 0)) * kTrPart; };
  const int token = row / p.grp, head = row - token * p.grp;
  __nv_bfloat16* const dst =
      p.out + ((static_cast<long long>(sp.row0) + token) * p.nq + sp.j * p.grp + head) * kHeadDim + 4 * col4;
  if (sp.parts <= kFew) {  // all at once
    if (token >= sp.tokens) return;
    float4 v[kFew];
    float2 ml[kFew];
#pragma unroll
    for (int e = 0; e < kFew; ++e) {
      if (e >= sp.parts) break;
      const float* from = part_of(e);
      v[e] = __ldcg(reinterpret_cast<const float4*>(from) + col4 * kPfRows + row);
      ml[e] = make_float2(__ldcg(from + kHeadDim * kPfRows + row), __ldcg(from + (kHeadDim + 1) * kPfRows + row));
    }
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < kFew; ++e)
      if (e < sp.parts) m = fmaxf(m, ml[e].x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int e = 0; e < kFew; ++e) {
      if (e >= sp.parts) break;
      const float f = ml[e].x == -INFINITY ? 0.f : exp2f(ml[e].x - m);
      l = fmaf(f, ml[e].y, l);
      o.x = fmaf(f, v[e].x, o.x);
      o.y = fmaf(f, v[e].y, o.y);
      o.z = fmaf(f, v[e].z, o.z);
      o.w = fmaf(f, v[e].w, o.w);
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
    return;
  }
  if (threadIdx.x < kTrJoinRows) most[threadIdx.x] = 0u;
  // the first parts, long before their factors are known
  float4 v[kAhead];
  auto load = [&](int s0) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e)
      if (s0 + e < sp.parts) v[e] = __ldcg(reinterpret_cast<const float4*>(part_of(s0 + e)) + col4 * kPfRows + row);
  };
  load(0);
  __syncthreads();
  for (int s = col4; s < sp.parts; s += 32) {
    const float* from = part_of(s) + kHeadDim * kPfRows + row;
    const float2 ml = make_float2(__ldcg(from), __ldcg(from + kPfRows));
    factor[s * kTrJoinRows + r] = ml;
    const unsigned b = __float_as_uint(ml.x);  // integers that rise as the maxima do
    atomicMax(&most[r], b & 0x80000000u ? ~b : b | 0x80000000u);
  }
  __syncthreads();
  const float m = __uint_as_float(most[r] & 0x80000000u ? most[r] & 0x7fffffffu : ~most[r]);
  for (int s = col4; s < sp.parts; s += 32) {
    float2& f = factor[s * kTrJoinRows + r];
    f.x = f.x == -INFINITY ? 0.f : exp2f(f.x - m);
    f.y *= f.x;
  }
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < sp.parts; s0 += kAhead) {
    if (s0 > 0) load(s0);
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      if (s0 + e >= sp.parts) break;
      const float f = factor[(s0 + e) * kTrJoinRows + r].x;
      o.x = fmaf(f, v[e].x, o.x);
      o.y = fmaf(f, v[e].y, o.y);
      o.z = fmaf(f, v[e].z, o.z);
      o.w = fmaf(f, v[e].w, o.w);
    }
  }
  if (col4 == 0) {
    float l = 0.f;
    for (int s = 0; s < sp.parts; ++s) l += factor[s * kTrJoinRows + r].y;
    whole[r] = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  }
  __syncthreads();
  if (token >= sp.tokens) return;
  const float inv = whole[r];
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

// Sizes that the host can bound without the lengths.
struct TrLayout {
  long long grid;  // of the main kernel
  size_t rows, splits, q, q_lo, part, total;
};

TrLayout tr_layout(long long T, long long B, int nq, int nkv, long long max_pages, int page_size) {
  TrLayout L;
  const int tpt = kPfRows / (nq / nkv);
  const long long tiles = T / tpt + (B < T ? B : T);
  const long long blocks = (max_pages * page_size + kPfBlock - 1) / kPfBlock;
  // pairs of blocks at most
  const long long most = tiles * nkv * ((blocks + 2) / 2);
  L.grid = device_sm_count();
  if (most < L.grid) L.grid = most;
  auto round = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
  size_t at = kPagedScratch;
  L.rows = at;
  at += round(sizeof(TrRow) * T);
  L.splits = at;
  at += round(sizeof(TrSplit) * L.grid);
  L.q = at;
  at += round(sizeof(__nv_bfloat16) * T * nq * kHeadDim);
  L.q_lo = at;
  at += round(sizeof(__nv_bfloat16) * T * nq * kHeadDim);
  L.part = at;
  at += sizeof(float) * 2 * L.grid * kTrPart;
  L.total = at;
  return L;
}

}  // namespace

size_t paged_tree_workspace_bytes(long long T, long long B, int nq, int nkv, long long max_pages, int page_size) {
  return tr_layout(T, B, nq, nkv, max_pages, page_size).total;
}

cudaError_t paged_tree_launch(const __nv_bfloat16* qkv, const void* qw, const void* kw, int w_dtype,
                              const int* parents, const int* cu_seqlens, const int* kv_lens, const PagedCache& cache,
                              __nv_bfloat16* out, long long T, int B, int nq, float theta, float eps, float scale,
                              int window, int sinks, void* workspace, cudaStream_t s) {
  auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tmap_encode_fn());
  if (!encode) return cudaErrorNotSupported;
  const int nkv = cache.nkv, grp = nq / nkv, tpt = kPfRows / grp;
  const TrLayout L = tr_layout(T, B, nq, nkv, cache.max_pages, 1 << cache.page_shift);
  char* ws = static_cast<char*>(workspace);
  TrParams p;
  p.cu = cu_seqlens;
  p.kv_lens = kv_lens;
  p.out = out;
  p.status = reinterpret_cast<int*>(ws);
  p.rows = reinterpret_cast<TrRow*>(ws + L.rows);
  p.splits = reinterpret_cast<TrSplit*>(ws + L.splits);
  p.part = reinterpret_cast<float*>(ws + L.part);
  p.c = cache;
  p.T = static_cast<int>(T);
  p.B = B;
  p.nq = nq;
  p.grp = grp;
  p.tpt = tpt;
  p.window = window;
  p.sinks = sinks;
  p.scale_log2 = scale * kPfLog2e;
  TreeOut tree;
  tree.parents = parents;
  tree.rows = reinterpret_cast<TrRow*>(ws + L.rows);
  tree.q_lo = reinterpret_cast<__nv_bfloat16*>(ws + L.q_lo);
  tree.window = window;
  tree.sinks = sinks;
  __nv_bfloat16* q = reinterpret_cast<__nv_bfloat16*>(ws + L.q);
  const long long q_row = static_cast<long long>(nq) * kHeadDim;
  CUtensorMap mq, ml, mk, mv;
  if (!tmap_of_rows(encode, &mq, q, nq, T, q_row, grp, tpt) || !tmap_of_rows(encode, &ml, tree.q_lo, nq, T, q_row, grp, tpt) ||
      !tmap_of_pages(encode, &mk, cache, false) || !tmap_of_pages(encode, &mv, cache, true))
    return cudaErrorInvalidValue;
  cudaError_t e = paged_tree_store_launch(qkv, qw, kw, w_dtype, cu_seqlens, kv_lens, cache, q, T, B, nq, theta, eps,
                                          tree, p.status, s);
  if (e != cudaSuccess) return e;
  e = allow_smem<paged_tree_kernel>(static_cast<int>(sizeof(TrShared)));
  if (e != cudaSuccess) return e;
  e = launch_pdl(paged_tree_kernel, dim3(static_cast<unsigned>(L.grid)), dim3(kTrThreads), sizeof(TrShared), s, mq, ml,
                 mk, mv, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_tree_join_kernel, dim3(static_cast<unsigned>(L.grid * (kPfRows / kTrJoinRows))),
                    dim3(32 * kTrJoinRows), sizeof(float2) * kTrJoinRows * L.grid, s, p);
}

}  // namespace nkimoe
