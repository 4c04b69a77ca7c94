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
// Two launches come before: the store (paged_store.cu) norms and turns the rows,
// puts keys and values in their pages and the queries in the workspace, works out
// every node's line of ancestors as 64 bits, and one CTA of it makes the list of
// units; a kernel after it joins what was cut.
//
// Tile: 128 MMA rows are floor(128 / group) nodes times the `group` query heads
// of one kv head.  A unit is up to two tiles of a sequence's nodes, for one kv
// head, against key blocks of 128 places.  Warps as in paged_prefill.cu: one
// loads Q and K, one V, one thread issues the MMAs, and a warpgroup per tile
// takes S from tensor memory and leaves P there.  With two tiles both work on
// the same block; with one (trees of up to 128 / group nodes) the two warpgroups
// take the blocks in turn, each with its own maximum, sum and O, which are joined
// at the unit's end: a block's chain (scores, softmax, product) takes longer than
// its bytes take to come from HBM, two chains at a time do not.
//
// Arithmetic: bf16 operands, sums, maxima and O in fp32.  In a unit of one tile
// queries and weights enter the MMAs as a sum of two bf16 (hi + lo, 2^-17), as in
// the decode step: the second query tile and the columns of S beside P are free
// for the lo parts there, and their MMAs fit into the time that a block's bytes
// take.  In a unit of two tiles both are rounded to bf16 (2^-9, random over the
// terms of a sum), as in the prompt attention.
//
// Work: the blocks of all (unit, kv head) form one list, and every CTA takes an
// equal run of it, so sequences of any mix of lengths load all SMs alike and the
// launch needs no length on the host.
#include "paged_tree.cuh"

namespace nkimoe {

namespace {

constexpr int kTrThreads = 384;
constexpr int kTrRing = 4;  // stages of 32 KB: K blocks in the even ones, V blocks in the odd ones
constexpr size_t kTrSmem = 1024 + 2 * kPfTileBytes + kTrRing * kPfBlockBytes;
// A part of a cut unit, per tile: o four columns at a time [32][128 rows][4],
// then the rows' m, then their l (a warp's rows are neighbours: coalesced)
constexpr int kTrPartTile = (kHeadDim + 2) * kPfRows;

// What a CTA began and others went on with: the unit of a kv head whose parts
// lie in slot 2 c + 1 of CTA c and the slots 0 of the CTAs after it.
struct TrSplit {
  int unit, j, parts, pad;
};

struct TrParams {
  __nv_bfloat16* out;  // [T, nq * 128]
  int* status;
  const TrRow* rows;    // [T]
  const TrList* list;
  const TrUnit* units;
  const int* offs;
  TrSplit* splits;  // [grid]
  float* part;      // [2 grid, 2, kTrPartTile]
  PagedCache c;
  int nq, grp, tpt;  // tpt: nodes per tile
  int window, sinks;
  float scale_log2;
};

// What the roles need to know of a unit; tokens 0: there are no more.
struct TrWork : TrUnit {
  int j;  // kv head
};

struct TrCtl {
  uint64_t q_full, q_empty;
  uint64_t kv_full[kTrRing], kv_empty[kTrRing];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t u_full[2], u_empty[2];
  uint64_t ml_full, ml_empty;  // the softmax warps have left their maxima and sums; have read them and both O
  uint64_t tail, drain;
  TrWork work[2];
  uint32_t tmem_base;
  int abort_flag;
  float2 ml[2][kPfRows];  // one tile: maximum and sum of both warpgroups
};

__global__ void __launch_bounds__(kTrThreads, 1)
    paged_tree_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_lo,
                      const __grid_constant__ TrParams p) {
  extern __shared__ uint8_t tr_raw[];
  __shared__ TrCtl ctl;
  __shared__ __align__(16) __nv_bfloat16 stg[8][32][40];  // per softmax warp: 32 output columns of its rows
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tr_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sq = smem;
  uint8_t* ring = smem + 2 * kPfTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&ctl.q_full, 1);
    mbar_init(&ctl.q_empty, 1);
    for (int s = 0; s < kTrRing; ++s) {
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
    mbar_init(&ctl.ml_full, 8);
    mbar_init(&ctl.ml_empty, 8);
    mbar_init(&ctl.tail, 1);
    mbar_init(&ctl.drain, 1);
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
  pdl_wait();
  // 384 x 168 registers at launch = 128 x 88 + 256 x 208
  if (warp == 0 || warp == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ---------------------------------------------------------------- units and loads
    // Lane (h, g) loads half h of page g of a block.
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
    int stage = v;
    uint32_t phase = 0, issued = 0, last_phase = 0, tail_phase = 0;
    bool ok = true, q_issued = false;
    const TrList list = *p.list;
    const int run_lo = min(list.total, static_cast<int>(blockIdx.x) * list.share);
    const int run_hi = min(list.total, run_lo + list.share);
    int at = run_lo, unit = 0;
    if (v == 0) {
      if (lane == 0) p.splits[blockIdx.x].parts = 0;
      for (int hi = list.units; hi - unit > 1;) {
        const int mid = (unit + hi) >> 1;
        if (p.offs[mid] <= at) unit = mid; else hi = mid;
      }
    }
    for (int u = 0; ok; ++u) {
      const int us = u & 1;
      TrWork w{};
      if (v) {
        if (!wait(&ctl.u_full[us], (u >> 1) & 1)) { ok = false; break; }
        w = ctl.work[us];
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.u_empty[us]);
      } else {
        if (!wait(&ctl.u_empty[us], ((u >> 1) & 1) ^ 1u)) { ok = false; break; }
        if (at < run_hi) {
          static_cast<TrUnit&>(w) = p.units[unit];
          const int n = w.hi, base = p.offs[unit];
          w.j = (at - base) / (n + kTrItem);
          // the list's first block of (unit, kv head), behind the places for its own cost
          const int item = base + w.j * (n + kTrItem) + kTrItem;
          w.lo = max(at - item, 0);
          w.hi = min(n, run_hi - item);
          const int first = item / list.share, parts = (item + n - 1) / list.share - first + 1;
          if (w.hi <= 0) {
            w.tokens = 0;  // the run ends before the item's blocks
          } else {
            if (parts > 1) w.slot = 2 * static_cast<int>(blockIdx.x) + (item < run_lo ? 0 : 1);
            if (parts > 1 && item >= run_lo && lane == 0) p.splits[blockIdx.x] = TrSplit{unit, w.j, parts, 0};
          }
          at = item + w.hi;
          if (w.hi == n && w.j == p.c.nkv - 1) ++unit;
        }
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
      if (v == 0) {
        if (!wait(&ctl.q_empty, (u & 1) ^ 1u)) { ok = false; break; }
        // two tiles, or one tile's hi and lo parts
        const bool lo = w.tokens <= p.tpt && lane > 1;
        if (lane == 0) mbar_arrive_expect_tx(&ctl.q_full, 2 * q_bytes);
        __syncwarp();
        if (lane < 4)
          tma_load_3d(sq + (lane >> 1) * kPfTileBytes + (lane & 1) * kPfTileHalf, lo ? &tmap_lo : &tmap_q, &ctl.q_full,
                      (lane & 1) * 64, w.j * p.grp, w.row0 + (lo ? 0 : (lane >> 1) * p.tpt));
        q_issued = true;
      }
      for (int i = w.lo; ok && i < w.hi; ++i) {
        const bool held = next >= 0 && next < p.c.num_pages;
        if (!held && next != -2) atomicOr(p.status, kDevErrBadIndex);
        const int page = held ? next : p.c.num_pages;  // past the last page: the load fills zeros
        const int k0 = bl.at(i) * kPfBlock;
        const int in_page = (k0 + g_lane * page_rows) & ((1 << p.c.page_shift) - 1);
        if (i + 1 < w.hi) next = look_up(i + 1);  // in flight while this block waits for its stage
        if (!wait(&ctl.kv_empty[stage], phase ^ 1u)) { ok = false; break; }
        // rows behind the sequence's end in its last page hold anything: their
        // weights are 0, and 0 times a NaN would not be, so this warp clears
        // them once the block is there (further pages are loaded as zeros)
        const int live = w.kv - k0;
        const bool clear = v == 1 && live < kPfBlock && (live & (page_rows - 1)) != 0;
        uint64_t* const bar = clear ? &ctl.tail : &ctl.kv_full[stage];
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
          if (lane == 0) mbar_arrive(&ctl.kv_full[stage]);
        }
        issued |= 1u << stage;
        last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
        stage += 2;
        if (stage >= kTrRing) {
          stage = v;
          phase ^= 1u;
        }
      }
    }
    if (!ok && lane == 0) {  // let the copies in flight land before the CTA exits
      for (int s = 0; s < kTrRing; ++s)
        if ((issued >> s) & 1u) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&ctl.kv_full[s], (last_phase >> s) & 1u) && clock64() - t0 < kWaitBudgetCycles / 8) {
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
    // ---------------------------------------------------------------- MMA issue (one thread)
    constexpr uint32_t idesc_s = umma_idesc_bf16_f32(kPfRows, kPfBlock);
    constexpr uint32_t idesc_o = umma_idesc_bf16_f32(kPfRows, kHeadDim) | (1u << 16);  // B is MN-major
    uint32_t ks = 0, vs = 0, pphase = 0;  // K and V blocks taken so far; pphase: bit t, of p_full
    bool ok = true, any = false;
    auto wait = [&](uint64_t* bar, uint32_t ph) { return mbar_wait(bar, ph, &ctl.abort_flag, p.status); };
    auto k_stage = [&] { return 2 * (ks & 1); };
    auto v_stage = [&] { return 2 * (vs & 1) + 1; };
    auto k_here = [&] { return wait(&ctl.kv_full[k_stage()], (ks >> 1) & 1); };
    auto v_here = [&] { return wait(&ctl.kv_full[v_stage()], (vs >> 1) & 1); };
    // S of tile t against the K block in the current stage, with the queries of slots q_lo .. q_hi
    auto issue_s = [&](int t, int q_lo, int q_hi) {
      for (int q = q_lo; q <= q_hi; ++q) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint64_t da = umma_desc_sw128(smem_u32(sq + q * kPfTileBytes + h * kPfTileHalf));
          const uint64_t db = umma_desc_sw128(smem_u32(ring + k_stage() * kPfBlockBytes + h * kPfBlockHalf));
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(tmem + t * 128, da + 2 * k, db + 2 * k, idesc_s, q > q_lo || (h | k) != 0);
        }
      }
      umma_commit(&ctl.s_full[t]);
      any = true;
    };
    auto k_done = [&] {
      umma_commit(&ctl.kv_empty[k_stage()]);
      ++ks;
    };
    // O += P V of tile t; lo: P's lo part lies behind it
    auto issue_o = [&](int t, bool more, bool lo) {
      const uint64_t dv = umma_desc_sw128_mn(smem_u32(ring + v_stage() * kPfBlockBytes), kPfBlockHalf);
#pragma unroll
      for (int k = 0; k < 8; ++k)  // 16 positions: 2048 bytes of V, 8 columns of P
        umma_bf16_ts(tmem + kPfTmemO + t * 128, tmem + t * 128 + 8 * k, dv + 128 * k, idesc_o, more || k != 0);
      if (lo)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_bf16_ts(tmem + kPfTmemO + t * 128, tmem + t * 128 + 64 + 8 * k, dv + 128 * k, idesc_o, 1);
    };
    auto p_here = [&](int t) {
      if (!wait(&ctl.p_full[t], (pphase >> t) & 1u)) return false;
      pphase ^= 1u << t;
      tcgen05_fence_after();
      return true;
    };
    for (int u = 0; lane == 0 && ok; ++u) {
      const int us = u & 1;
      if (!wait(&ctl.u_full[us], (u >> 1) & 1)) { ok = false; break; }
      const int tokens = ctl.work[us].tokens, n = ctl.work[us].hi - ctl.work[us].lo;
      mbar_arrive(&ctl.u_empty[us]);
      if (tokens == 0) break;
      if (!wait(&ctl.q_full, u & 1) || !k_here()) { ok = false; break; }
      if (tokens <= p.tpt) {
        // one tile: block i is warpgroup i % 2's
        issue_s(0, 0, 1);
        k_done();
        if (n > 1) {
          if (!k_here()) { ok = false; break; }
          issue_s(1, 0, 1);
          k_done();
        }
        if (n <= 2) umma_commit(&ctl.q_empty);
        for (int i = 0; i < n; ++i) {
          const int t = i & 1;
          if (!v_here() || !p_here(t)) { ok = false; break; }
          issue_o(t, i > 1, true);
          umma_commit(&ctl.kv_empty[v_stage()]);
          ++vs;
          if (i + 2 < n) {  // over P, which the product before it has read
            if (!k_here()) { ok = false; break; }
            issue_s(t, 0, 1);
            k_done();
            if (i + 3 == n) umma_commit(&ctl.q_empty);
          } else {
            umma_commit(&ctl.o_full[t]);
          }
        }
        continue;
      }
      for (int t = 0; t < 2; ++t) issue_s(t, t, t);
      k_done();
      if (n == 1) umma_commit(&ctl.q_empty);
      for (int i = 0; ok && i < n; ++i) {
        if (!v_here()) { ok = false; break; }
        const bool more = i + 1 < n;
        for (int t = 0; t < 2; ++t) {
          if (!p_here(t)) { ok = false; break; }
          issue_o(t, i > 0, false);
          if (more) {
            if (t == 0 && !k_here()) { ok = false; break; }
            issue_s(t, t, t);
          } else {
            umma_commit(&ctl.o_full[t]);
          }
        }
        if (!ok) break;
        umma_commit(&ctl.kv_empty[v_stage()]);
        ++vs;
        if (more) {
          k_done();
          if (i + 2 == n) umma_commit(&ctl.q_empty);
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
    for (int u = 0;; ++u) {
      const int us = u & 1;
      if (!wait(&ctl.u_full[us], (u >> 1) & 1)) break;
      const TrWork w = ctl.work[us];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.u_empty[us]);
      if (w.tokens == 0) break;
      const bool single = w.tokens <= p.tpt;  // one tile, whose blocks the warpgroups share
      const int node = (single ? 0 : g * p.tpt) + token;
      const bool mine = token < p.tpt && node < w.tokens;
      TrRow info{0, w.past, 0};
      if (mine) info = p.rows[w.row0 + node];
      const Blocks bl = blocks_of(w.past, w.kv - 1, p.window, p.sinks);
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      const int first = w.lo + (single ? g : 0), step = single ? 2 : 1;
#pragma unroll 1
      for (int i = first; i < w.hi; i += step) {
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
        auto weigh = [&](int c) {  // 16 columns at a time: registers
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk[8], lo[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const uint64_t y = fma2(pair2(__uint_as_float(s[c][16 * h + 2 * x]), __uint_as_float(s[c][16 * h + 2 * x + 1])), sc2, ms2);
              float2 e = split2(y);
              e.x = ex2(e.x);
              e.y = ex2(e.y);
              const uint64_t w2 = pair2(e.x, e.y);
              sum[x & 3] = add2(sum[x & 3], w2);
              pk[x] = pack_bf16x2(e.x, e.y);
              if (single) lo[x] = bf16x2_of_pair(fma2(pair_of_bf16x2(pk[x]), pair2(-1.f, -1.f), w2));
            }
            tmem_st_32x32b_x8(ts + c * 16 + h * 8, pk);
            if (single) tmem_st_32x32b_x8(ts + 64 + c * 16 + h * 8, lo);
          }
        };
        weigh(0);
        weigh(1);
        if (half_only) {
          const uint32_t none[16] = {};
          tmem_st_32x32b_x16(ts + 32, none);
          tmem_st_32x32b_x16(ts + 48, none);
          if (single) {
            tmem_st_32x32b_x16(ts + 96, none);
            tmem_st_32x32b_x16(ts + 112, none);
          }
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
      // where this lane stores: row 8 k + lane / 4, columns 8 (lane % 4) of each 32
      const long long out_at =
          mine ? ((static_cast<long long>(w.row0) + node) * p.nq + w.j * p.grp + head) * kHeadDim : -1;
      __nv_bfloat16* to_row[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long at = __shfl_sync(0xffffffffu, out_at, k * 8 + (lane >> 2));
        to_row[k] = at >= 0 ? p.out + at + (lane & 3) * 8 : nullptr;
      }
      float* part = w.slot >= 0 ? p.part + (static_cast<long long>(w.slot) * 2 + (single ? 0 : g)) * kTrPartTile : nullptr;
      float own = 1.f, other = 0.f;  // what this warpgroup's O and the other's are multiplied by
      const bool joined = single && w.hi - w.lo > 1;
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
      const float inv = part ? 1.f : l > 0.f ? 1.f / l : (l == l ? 0.f : l);
      own *= inv;
      other *= inv;
      // columns [64 g, 64 g + 64) of a joined tile, all of a tile of its own; nothing for the second warpgroup of one block
      const int c_lo = joined ? 2 * g : 0, c_hi = joined ? 2 * g + 2 : single && g ? 0 : 4;
      const uint32_t to_other = joined ? tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (1 - g) * 128 + kPfTmemO : to;
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
        if (part) {
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            __stcg(reinterpret_cast<uint4*>(part) + (c * 8 + x / 4) * kPfRows + row, make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]));
        } else {
          // through shared memory: eight rows of 64 bytes per store instead of 32 rows of 16
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[x + e]);
            *reinterpret_cast<uint4*>(&stg[warp - 4][lane][x]) = pack8(f);
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint4 v = *reinterpret_cast<const uint4*>(&stg[warp - 4][k * 8 + (lane >> 2)][(lane & 3) * 8]);
            if (to_row[k]) *reinterpret_cast<uint4*>(to_row[k] + c * 32) = v;
          }
          __syncwarp();
        }
      }
      if (part && c_lo == 0 && c_hi > 0) {
        __stcg(part + kHeadDim * kPfRows + row, m);
        __stcg(part + (kHeadDim + 1) * kPfRows + row, l);
      }
      tcgen05_fence_before();  // the next unit's MMAs follow this thread's next arrival
      if (joined) {  // the next unit's MMAs and maxima wait until both warpgroups have read both
        __syncwarp();
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

// Joins the parts of a cut unit, in order: a CTA per (unit and kv head, 32
// rows), a lane per row, a warp per 16 columns.
__global__ void __launch_bounds__(256) paged_tree_join_kernel(const __grid_constant__ TrParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int cta = blockIdx.x >> 3, tile = (blockIdx.x >> 2) & 1;
  const int lane = threadIdx.x & 31, col = (threadIdx.x >> 5) * 16, row = (blockIdx.x & 3) * 32 + lane;
  const TrSplit sp = p.splits[cta];
  if (sp.parts == 0) return;
  const TrUnit un = p.units[sp.unit];
  const int token = row / p.grp, head = row - token * p.grp;
  if (token >= p.tpt || tile * p.tpt + token >= un.tokens) return;
  auto part_of = [&](int s) {
    const int slot = 2 * (cta + s) + (s == 0);
    return p.part + (static_cast<long long>(slot) * 2 + tile) * kTrPartTile;
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
struct TrLayout {
  long long units, grid;  // grid: of the main kernel
  size_t rows, list, units_at, offs, splits, q, q_lo, part, total;
};

TrLayout tr_layout(long long T, long long B, int nq, int nkv, long long max_pages, int page_size) {
  TrLayout L;
  const int tpt = kPfRows / (nq / nkv);
  L.units = T / (2 * tpt) + (B < T ? B : T);
  const long long blocks = (max_pages * page_size + kPfBlock - 1) / kPfBlock;
  // places at most, and so runs at most
  const long long most = (L.units * nkv * (blocks + 1 + kTrItem) + kTrMinBlocks + kTrItem - 1) / (kTrMinBlocks + kTrItem);
  L.grid = device_sm_count();
  if (most < L.grid) L.grid = most;
  auto round = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
  size_t at = kPagedScratch;
  L.list = at;
  at += 256;
  L.rows = at;
  at += round(sizeof(TrRow) * T);
  L.units_at = at;
  at += round(sizeof(TrUnit) * L.units);
  L.offs = at;
  at += round(sizeof(int) * (L.units + 1));
  L.splits = at;
  at += round(sizeof(TrSplit) * L.grid);
  L.q = at;
  at += round(sizeof(__nv_bfloat16) * T * nq * kHeadDim);
  L.q_lo = at;
  at += round(sizeof(__nv_bfloat16) * T * nq * kHeadDim);
  L.part = at;
  at += sizeof(float) * 2 * L.grid * 2 * kTrPartTile;
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
  int* status = reinterpret_cast<int*>(ws);
  __nv_bfloat16* q = reinterpret_cast<__nv_bfloat16*>(ws + L.q);
  __nv_bfloat16* q_lo = reinterpret_cast<__nv_bfloat16*>(ws + L.q_lo);
  CUtensorMap mq, mk, mv, ml;
  if (!tmap_of_rows(encode, &mq, q, nq, T, static_cast<long long>(nq) * kHeadDim, grp, tpt) ||
      !tmap_of_rows(encode, &ml, q_lo, nq, T, static_cast<long long>(nq) * kHeadDim, grp, tpt) ||
      !tmap_of_pages(encode, &mk, cache, false) || !tmap_of_pages(encode, &mv, cache, true))
    return cudaErrorInvalidValue;
  TrPlan plan;
  plan.q_lo = q_lo;
  plan.rows = reinterpret_cast<TrRow*>(ws + L.rows);
  plan.list = reinterpret_cast<TrList*>(ws + L.list);
  plan.units = reinterpret_cast<TrUnit*>(ws + L.units_at);
  plan.offs = reinterpret_cast<int*>(ws + L.offs);
  plan.window = window;
  plan.sinks = sinks;
  plan.tpt = tpt;
  plan.sms = static_cast<int>(L.grid);
  plan.max_units = static_cast<int>(L.units);
  cudaError_t e = paged_tree_store_launch(qkv, qw, kw, w_dtype, parents, cu_seqlens, kv_lens, cache, q, T, B, nq, theta,
                                          eps, plan, status, s);
  if (e != cudaSuccess) return e;
  TrParams p;
  p.out = out;
  p.status = status;
  p.rows = plan.rows;
  p.list = plan.list;
  p.units = plan.units;
  p.offs = plan.offs;
  p.splits = reinterpret_cast<TrSplit*>(ws + L.splits);
  p.part = reinterpret_cast<float*>(ws + L.part);
  p.c = cache;
  p.nq = nq;
  p.grp = grp;
  p.tpt = tpt;
  p.window = window;
  p.sinks = sinks;
  p.scale_log2 = scale * kPfLog2e;
  e = allow_smem<paged_tree_kernel>(static_cast<int>(kTrSmem));
  if (e != cudaSuccess) return e;
  e = launch_pdl(paged_tree_kernel, dim3(static_cast<unsigned>(L.grid)), dim3(kTrThreads), kTrSmem, s, mq, mk, mv, ml, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_tree_join_kernel, dim3(static_cast<unsigned>(8 * L.grid)), dim3(256), 0, s, p);
}

}  // namespace nkimoe
