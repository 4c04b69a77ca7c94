"""The paged key-value cache on the GPU: store, decode attention and page
copies against the formulas in 64 bits.

Bars.  An output is one rounding to bf16 (at most 2^-8 of the value) of what
fp32 arithmetic gives.  Scores carry the split of the queries (2^-17) and 128
fp32 additions (2^-17), relative to |q| |k| scale <= 11.4 w^2 with the norm
weights w <= 1.6: at most 2^-16 * 11.4 * 2.6 = 2^-11.1 on the exponent, twice
that on a normalised weight, so 2^-10 of the largest value at most on the sum.
The stored keys are one rounding of fp32 arithmetic (2^-8, and 2^-16 for the
norm, sine and cosine in fp32, absolute on values up to 8); the stored values
are copies.
"""

import math

import pytest
import torch

from nki_moe_b200 import ops
from nki_moe_b200._lib import NKIMoEError

pytestmark = pytest.mark.gpu

HD = 128
THETA = 1e6
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def turned(x, w, pos):
    """RMSNorm over heads x [rows, heads, 128] and rotate-half, in 64 bits."""
    x = x.double()
    x = x / ((x * x).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    ang = pos.double()[:, None, None] * THETA ** (-torch.arange(64, dtype=torch.float64) / 64)
    a, b = x[..., :64], x[..., 64:]
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)


def visible(p, n, window, sinks):
    s = torch.arange(n)
    see = s <= p
    if window:
        see &= (s > p - window) | (s < sinks)
    return see


def attend(q, p, k, v, scale, window, sinks):
    """q [heads, 128] at position p over k, v [kv heads, keys, 128] (64 bits);
    a query that sees nothing gives 0."""
    see = visible(p, k.shape[1], window, sinks)
    if not see.any():
        return torch.zeros_like(q)
    grp = q.shape[0] // k.shape[0]
    out = torch.empty_like(q)
    for h in range(q.shape[0]):
        s = (k[h // grp][see] @ q[h]) * scale
        out[h] = torch.softmax(s, 0) @ v[h // grp][see]
    return out


class Cache:
    """A pool on the CPU with sequences in shuffled pages.  Rows that hold no
    token of any sequence are NaN, and so are pages that no sequence needs."""

    def __init__(self, lens, nkv, ps, seed, needed=None, extra=3):
        g = torch.Generator().manual_seed(seed)
        B = len(lens)
        need = [(n + ps - 1) // ps for n in lens]
        P = max(1, sum(need)) + extra
        ids = torch.randperm(P, generator=g)[:sum(need)].to(torch.int32)
        self.k = torch.full((P, nkv, ps, HD), math.nan, dtype=torch.bfloat16)
        self.v = torch.full((P, nkv, ps, HD), math.nan, dtype=torch.bfloat16)
        self.table = torch.full((B, max(1, max(need, default=1))), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = ids[at:at + need[b]]
            at += need[b]
            for i in range(need[b]):
                held = needed is None or needed(b, i * ps, min((i + 1) * ps, n))
                pg = int(self.table[b, i])
                rows = min(ps, n - i * ps)
                if held:
                    self.k[pg, :, :rows] = torch.randn(nkv, rows, HD, generator=g).bfloat16()
                    self.v[pg, :, :rows] = torch.randn(nkv, rows, HD, generator=g).bfloat16()
                else:
                    self.table[b, i] = -1
        self.ps, self.nkv = ps, nkv

    def rows(self, pages, b, n):
        out = torch.full((self.nkv, n, HD), math.nan, dtype=torch.float64)
        for s in range(n):
            pg = int(self.table[b, s // self.ps])
            if pg >= 0:
                out[:, s] = pages[pg, :, s % self.ps].double()
        return out


def weights(seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return tuple((1 + 0.6 * torch.rand(HD, generator=g)).to(dtype) for _ in range(2))


def near(out, ref, vmax, rtol=2 ** -8, atol=2 ** -10):
    out = out.double().cpu()
    assert torch.isfinite(out).all()
    over = (out - ref).abs() - (rtol * ref.abs() + atol * vmax)
    assert over.max() <= 0, f"off by {float(over.max()):.3e} more than allowed (values to {vmax:.2f})"


def decode_case(lens, nq, nkv, ps, window=0, sinks=0, seed=0, w_dtype=torch.bfloat16, idle=(), interleaved=False,
                scale=None, broadcast=False):
    """Runs one decode step and checks output and cache; lens[b] counts the new token."""
    B = len(lens)

    def needed(b, lo, hi):
        see = visible(lens[b] - 1, lens[b], window, sinks)
        return bool(see[lo:hi].any())

    c = Cache(lens, nkv, ps, seed, needed if window else None)
    g = torch.Generator().manual_seed(seed + 1)
    qkv = torch.randn(B, (nq + 2 * nkv) * HD, generator=g).bfloat16()
    qw, kw = weights(seed + 2, w_dtype)
    pos = torch.tensor([n - 1 for n in lens])
    for b in idle:
        pos[b] = -1 - b
    rows = qkv.view(B, nq + 2 * nkv, HD)
    q = turned(rows[:, :nq], qw, pos)
    k_new = turned(rows[:, nq:nq + nkv], kw, pos)
    k_ref, v_ref = c.k.clone(), c.v.clone()
    ref = torch.zeros(B, nq, HD, dtype=torch.float64)
    vmax = 1.0
    for b in range(B):
        if b in idle:
            continue
        p = int(pos[b])
        pg = int(c.table[b, p // ps])
        k_ref[pg, :, p % ps] = k_new[b].bfloat16()
        v_ref[pg, :, p % ps] = rows[b, nq + nkv:]
        k, v = c.rows(k_ref, b, p + 1), c.rows(v_ref, b, p + 1)
        vmax = max(vmax, float(v.nan_to_num().abs().max()))
        ref[b] = attend(q[b], p, k, v, scale or HD ** -0.5, window, sinks)
    if interleaved:
        pool = torch.stack([c.k, c.v], 1).cuda()
        kd, vd = pool[:, 0], pool[:, 1]
    else:
        kd, vd = c.k.cuda(), c.v.cuda()
    table = c.table.cuda()
    before_k, before_v = kd.clone(), vd.clone()
    out = ops.paged_decode_attention(qkv.cuda(), qw.cuda(), kw.cuda(), (pos[:1] if broadcast else pos).cuda(), kd, vd,
                                     table, nq, nkv, window=window, sinks=sinks, scale=scale)
    ops.read_paged_status()
    near(out.view(B, nq, HD), ref, vmax)
    for b in idle:
        assert torch.count_nonzero(out[b]) == 0
    # the new rows, and nothing else
    for new, old, want, exact in ((kd, before_k, k_ref, False), (vd, before_v, v_ref, True)):
        new, old = new.cpu(), old.cpu()
        for b in range(B):
            if b in idle:
                continue
            p = int(pos[b])
            pg = int(c.table[b, p // ps])
            got, ref_row = new[pg, :, p % ps].double(), want[pg, :, p % ps].double()
            if exact:
                assert torch.equal(got, ref_row)
            else:
                assert ((got - ref_row).abs() <= 2 ** -7 * ref_row.abs() + 2 ** -13).all()
            new[pg, :, p % ps] = old[pg, :, p % ps]
        assert torch.equal(new.view(torch.int16), old.view(torch.int16))
    return out


@pytest.mark.parametrize("nq,nkv", [(32, 4), (8, 8), (16, 1), (12, 4), (7, 1), (40, 8), (18, 2)])
@pytest.mark.parametrize("ps", [16, 64])
def test_decode_heads_and_odd_lengths(nq, nkv, ps):
    decode_case([1, 2, 15, 16, 17, 63, 64, 65, 200], nq, nkv, ps, seed=nq + ps)


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
def test_decode_page_sizes(ps):
    decode_case([ps - 1, ps, ps + 1, 3 * ps + 7, 700], 32, 4, ps, seed=ps)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 0), (16, 4), (64, 4), (100, 65), (17, 300), (1000, 4),
                                          (700, 0), (701, 3)])
def test_decode_window_and_sinks(window, sinks):
    decode_case([1, 3, 64, 65, 100, 333, 700], 32, 4, 16, window, sinks, seed=window + sinks)


@pytest.mark.parametrize("window,sinks", [(33, 2), (130, 1)])
def test_decode_window_in_larger_pages(window, sinks):
    decode_case([1, 3, 64, 257, 700], 8, 2, 64, window, sinks, seed=window)
    decode_case([300, 900], 16, 1, 256, window, sinks, seed=window + 1)


def test_decode_one_long_sequence_is_split_over_the_gpu():
    decode_case([20011], 32, 4, 64, seed=5)
    decode_case([9000], 16, 1, 128, seed=6)


def test_decode_ragged_batch():
    decode_case([1, 5000, 40, 2, 1200, 64, 1, 3000], 16, 2, 32, seed=7)


def test_decode_idle_rows_fp32_weights_and_interleaved_pools():
    decode_case([5, 70, 9, 130], 32, 4, 16, idle=(1, 3), seed=8, w_dtype=torch.float32, interleaved=True)
    decode_case([5, 70], 8, 4, 16, idle=(0, 1), seed=9)


def test_decode_scale_and_one_position_for_all():
    decode_case([40, 40, 40], 8, 2, 16, seed=10, scale=0.3, broadcast=True)


def test_decode_calls_of_many_shapes_share_a_workspace():
    """Counters and partials of one call must not disturb the next."""
    for i, (lens, nq, nkv) in enumerate([([3000], 32, 4), ([70] * 40, 32, 4), ([5000, 1], 16, 1), ([65] * 100, 8, 8),
                                         ([3000], 32, 4)]):
        decode_case(lens, nq, nkv, 64, seed=20 + i)


def step_inputs(lens, nq, nkv, ps, seed):
    c = Cache(lens, nkv, ps, seed)
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(len(lens), (nq + 2 * nkv) * HD, generator=g).bfloat16()
    qw, kw = weights(seed)
    pos = torch.tensor([n - 1 for n in lens])
    return [t.cuda() for t in (qkv, qw, kw, pos, c.k, c.v, c.table)] + [nq, nkv]


def test_decode_is_deterministic_and_follows_its_stream():
    args = step_inputs([2000, 37, 800, 1], 32, 4, 16, 30)
    want = ops.paged_decode_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [ops.paged_decode_attention(*args) for _ in range(5)]
    here = [ops.paged_decode_attention(*args) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs + here)


def test_decode_graphs_replay_at_the_same_time():
    """Two graphs captured on one stream and replayed on two: each has its own
    workspace.  The positions are device data, so a replay serves the next step."""
    side = torch.cuda.Stream()
    graphs = []
    for seed in (31, 32):
        args = step_inputs([4000, 900, 65, 2500], 32, 4, 64, seed)
        want = ops.paged_decode_attention(*args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = ops.paged_decode_attention(*args)
        graphs.append((g, args, out, want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (g, _, out, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        ops.paged_decode_attention(*graphs[0][1])
    torch.cuda.synchronize()
    for _, _, out, want in graphs:
        assert torch.equal(out, want)
    g, args, out, _ = graphs[0]
    args[3].fill_(64)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.paged_decode_attention(*args))
    ops.read_paged_status()


def test_decode_reports_positions_and_pages_out_of_range(monkeypatch):
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    args = step_inputs([70, 33, 50], 8, 2, 16, 33)
    good = ops.paged_decode_attention(*args)
    ops.read_paged_status()
    args[3][0] = 10_000  # past the page table
    out = ops.paged_decode_attention(*args)
    with pytest.raises(NKIMoEError):
        ops.read_paged_status()
    ops.read_paged_status()  # cleared
    assert torch.count_nonzero(out[0]) == 0 and torch.equal(out[1:], good[1:])
    args[3][0] = 69
    for bad in (-1, -7, 10_000):  # a page that the second sequence needs
        keep = int(args[6][1, 0])
        args[6][1, 0] = bad
        out = ops.paged_decode_attention(*args)
        with pytest.raises(NKIMoEError):
            ops.read_paged_status()
        args[6][1, 0] = keep
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2]) and torch.isfinite(out[1]).all()


def test_decode_pool_past_32_bit_offsets():
    """The last pages of a pool of more than 2^31 elements."""
    nq, nkv, ps = 8, 4, 256
    P = 2 ** 31 // (nkv * ps * HD) + 40
    k = torch.zeros(P, nkv, ps, HD, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    c = Cache([600, 300], nkv, ps, 40, extra=0)
    first = P - c.k.shape[0]
    k[first:], v[first:] = c.k.cuda(), c.v.cuda()
    args = step_inputs([600, 300], nq, nkv, ps, 40)
    small = ops.paged_decode_attention(*args[:4], c.k.cuda(), c.v.cuda(), c.table.cuda(), nq, nkv)
    table = torch.where(c.table >= 0, c.table + first, c.table).cuda()
    big = ops.paged_decode_attention(*args[:4], k, v, table, nq, nkv)
    ops.read_paged_status()
    assert torch.isfinite(big).all() and torch.equal(big, small)
    ops.copy_pages(k, [P - 1], [0])
    torch.cuda.synchronize()
    assert torch.equal(k[0].view(torch.int16), k[P - 1].view(torch.int16))


# ------------------------------------------------------------------ store
def store_case(news, pasts, nq, nkv, ps, seed, w_dtype=torch.bfloat16, behind=0, drop=()):
    B = len(news)
    total = [n + p for n, p in zip(news, pasts)]
    c = Cache(total, nkv, ps, seed)
    for b, i in drop:
        c.table[b, i] = -1
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(news).cumsum(0)
    T = int(cu[-1]) + behind
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (nq + 2 * nkv) * HD, generator=g).bfloat16()
    qw, kw = weights(seed, w_dtype)
    kd, vd = c.k.cuda(), c.v.cuda()
    out = torch.full((T, nq, HD), 7.0, dtype=torch.bfloat16, device="cuda")
    got = ops.qk_norm_rope_store(qkv.cuda(), qw.cuda(), kw.cuda(), cu.cuda(), torch.tensor(total, dtype=torch.int32).cuda(),
                                 kd, vd, c.table.cuda(), nq, nkv, out=out)
    ops.read_paged_status()
    assert got.data_ptr() == out.data_ptr()
    rows = qkv.view(T, nq + 2 * nkv, HD)
    k_new, v_new, out = kd.cpu(), vd.cpu(), out.cpu().double()
    assert (out[int(cu[-1]):] == 7).all()
    for b in range(B):
        r = slice(int(cu[b]), int(cu[b + 1]))
        pos = torch.arange(pasts[b], total[b])
        q, k = turned(rows[r, :nq], qw, pos), turned(rows[r, nq:nq + nkv], kw, pos)
        assert ((out[r] - q).abs() <= 2 ** -8 * q.abs() + 2 ** -13).all()
        for i, s in enumerate(pos.tolist()):
            pg = int(c.table[b, s // ps])
            if pg < 0:
                continue
            got_k = k_new[pg, :, s % ps].double()
            assert ((got_k - k[i]).abs() <= 2 ** -8 * k[i].abs() + 2 ** -13).all()
            assert torch.equal(v_new[pg, :, s % ps], rows[r, nq + nkv:][i])
            k_new[pg, :, s % ps], v_new[pg, :, s % ps] = c.k[pg, :, s % ps], c.v[pg, :, s % ps]
    assert torch.equal(k_new.view(torch.int16), c.k.view(torch.int16))
    assert torch.equal(v_new.view(torch.int16), c.v.view(torch.int16))


@pytest.mark.parametrize("nq,nkv", [(32, 4), (8, 8), (7, 1), (16, 1), (64, 8), (1, 1)])
def test_store_heads(nq, nkv):
    store_case([1, 5, 33], [0, 20, 3], nq, nkv, 16, seed=nq)


def test_store_many_sequences_some_without_rows():
    news = [(i * 7) % 5 for i in range(70)]
    news[0] = news[-1] = 0
    store_case(news, [(i * 3) % 40 for i in range(70)], 4, 2, 16, seed=50)


def test_store_far_positions_rows_behind_and_pages_not_kept():
    store_case([40, 3], [100_000, 0], 8, 2, 256, seed=51, w_dtype=torch.float32, behind=9)
    store_case([100], [0], 8, 2, 16, seed=52, drop=[(0, 0), (0, 3)])


def test_store_reports_rows_out_of_range(monkeypatch):
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    nq, nkv = 4, 2
    k = torch.zeros(4, nkv, 16, HD, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    qkv = torch.randn(8, (nq + 2 * nkv) * HD, device="cuda").bfloat16()
    w = torch.ones(HD, dtype=torch.bfloat16, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for cu, lens, table in ((i32(0, 8), i32(40), i32(0, 1).view(1, 2)), (i32(0, 8), i32(5), i32(0, 1).view(1, 2)),
                            (i32(0, 8), i32(8), i32(4, 1).view(1, 2)), (i32(0, 8), i32(8), i32(-2, 1).view(1, 2)),
                            (i32(0, 6, 3, 8), i32(1, 1, 1), i32(0, 1, 2).view(3, 1))):
        ops.qk_norm_rope_store(qkv, w, w, cu, lens, k, v, table, nq, nkv)
        with pytest.raises(NKIMoEError):
            ops.read_paged_status()


# ------------------------------------------------------------------ copies
@pytest.mark.parametrize("shape,n", [((3, 2, 40, 4, 16, 128), 5), ((9, 2, 16, 8), 4), ((1, 1200, 1, 16, 128), 590),
                                     ((2, 9000, 1, 1, 8), 4400), ((2, 7, 8, 256, 128), 3)])
def test_copy_pages(shape, n):
    pages = torch.randn(shape, device="cuda").bfloat16()
    P = shape[-4]
    ids = torch.randperm(P, generator=torch.Generator().manual_seed(n))
    src, dst = ids[:n], ids[n:2 * n]
    want = pages.clone()
    want.view(-1, *shape[-4:])[:, dst.cuda()] = want.view(-1, *shape[-4:])[:, src.cuda()]
    got = ops.copy_pages(pages, src, dst.to(torch.int32))
    assert got is pages and torch.equal(pages, want)
    # one page to several others, by lists; nothing for no pairs
    ops.copy_pages(pages, [int(src[0])] * 2, dst[:2].tolist())
    want.view(-1, *shape[-4:])[:, dst[1].item()] = want.view(-1, *shape[-4:])[:, src[0].item()]
    ops.copy_pages(pages, [], [])
    assert torch.equal(pages, want)


def test_copy_pages_other_types_and_a_captured_copy():
    pages = torch.arange(6 * 4 * 8 * 8, device="cuda").view(1, 6, 4, 8, 8).to(torch.uint8)
    want = pages.clone()
    want[:, 5] = want[:, 0]
    assert torch.equal(ops.copy_pages(pages, [0], [5]), want)
    pool = torch.randn(2, 6, 2, 16, HD, device="cuda").bfloat16()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.copy_pages(pool, [1], [2])
    ops.copy_pages(pool, [3], [4])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(pool[:, 1], pool[:, 2]) and torch.equal(pool[:, 3], pool[:, 4])


def test_copy_pages_refusals_copy_nothing():
    pages = torch.randn(2, 6, 2, 16, HD, device="cuda").bfloat16()
    before = pages.clone()
    for src, dst in (([0], [6]), ([-1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]), ([2 ** 31 + 1], [0])):
        with pytest.raises((NKIMoEError, ValueError)):
            ops.copy_pages(pages, src, dst)
    for src, dst in (([0], [1, 2]), (torch.tensor([0], device="cuda"), [1]), ([0.5], [1]), ([[0]], [[1]])):
        with pytest.raises(ValueError):
            ops.copy_pages(pages, src, dst)
    with pytest.raises(ValueError):
        ops.copy_pages(pages[:, ::2], [0], [1])
    assert torch.equal(pages, before)


# ------------------------------------------------------------------ prompt attention
def prefill_case(news, pasts, nq, nkv, ps, window=0, sinks=0, seed=0, behind=0, scale=None, strided=False, sharp=1.0):
    """P enters its product as bf16 (2^-8 of each weight), so the sum may be off
    by 2^-8 of the largest value, beside the bars of the decode step."""
    B = len(news)
    total = [n + p for n, p in zip(news, pasts)]

    def needed(b, lo, hi):
        if news[b] == 0:
            return False
        see = visible(total[b] - 1, total[b], 0, 0)
        if window:
            first = pasts[b]
            s = torch.arange(total[b])
            see = (s > first - window) | (s < sinks)
        return bool(see[lo:hi].any())

    c = Cache(total, nkv, ps, seed, needed)
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(news).cumsum(0)
    T = int(cu[-1]) + behind
    g = torch.Generator().manual_seed(seed + 1)
    q = (sharp * 1.3 * torch.randn(T, nq + (2 * nkv if strided else 0), HD, generator=g)).bfloat16()
    qd = q.cuda()[:, :nq]
    q = q[:, :nq]
    out = torch.full((T, nq * HD), 7.0, dtype=torch.bfloat16, device="cuda")
    kd, vd = c.k.cuda(), c.v.cuda()
    ops.paged_prefill_attention(qd, kd, vd, c.table.cuda(), cu.cuda(), torch.tensor(total, dtype=torch.int32).cuda(),
                                window=window, sinks=sinks, scale=scale, out=out)
    ops.read_paged_status()
    assert (out[int(cu[-1]):] == 7).all()
    grp = nq // nkv
    for b in range(B):
        if not news[b]:
            continue
        r = slice(int(cu[b]), int(cu[b + 1]))
        k, v = c.rows(c.k, b, total[b]).nan_to_num(), c.rows(c.v, b, total[b]).nan_to_num()
        qb = q[r].double().transpose(0, 1)
        s = qb @ k.repeat_interleave(grp, 0).transpose(1, 2) * (scale or HD ** -0.5)
        p = torch.arange(pasts[b], total[b])[:, None]
        t = torch.arange(total[b])
        see = t <= p
        if window:
            see &= (t > p - window) | (t < sinks)
        s.masked_fill_(~see, -math.inf)
        ref = (torch.softmax(s, -1) @ v.repeat_interleave(grp, 0)).transpose(0, 1)
        near(out[r].view(-1, nq, HD), ref, float(v.abs().max()), atol=2 ** -8 + 2 ** -10 * max(1.0, sharp))
        rel = (out[r].view(-1, nq, HD).double().cpu() - ref).norm() / ref.norm()
        assert rel < 2 ** -8, f"sequence {b}: {rel:.2e}"
    return out


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
def test_prefill_page_sizes_and_odd_lengths(ps):
    prefill_case([1, 2, 16, 17, 33, 129, 300], [0] * 7, 32, 4, ps, seed=ps)


@pytest.mark.parametrize("nq,nkv", [(8, 8), (16, 1), (12, 4), (7, 1), (40, 8), (18, 2), (1, 1), (28, 4)])
def test_prefill_heads(nq, nkv):
    prefill_case([5, 140, 261], [3, 0, 200], nq, nkv, 16, seed=nq)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (128, 0), (129, 5), (200, 130), (500, 4),
                                          (5000, 9), (40, 1000)])
def test_prefill_window_and_sinks(window, sinks):
    prefill_case([300, 5, 64], [0, 777, 400], 16, 2, 16, window, sinks, seed=window)
    prefill_case([130], [1000], 32, 4, 64, window, sinks, seed=window + 1)


def test_prefill_chunk_over_a_long_cache_is_cut_into_parts():
    prefill_case([16], [9000], 32, 4, 64, seed=60)
    prefill_case([1, 40, 3], [5000, 3000, 10], 16, 2, 128, seed=61)
    prefill_case([33], [6000], 8, 1, 16, 3000, 200, seed=62)


def test_prefill_sequences_without_rows_rows_behind_and_strided_queries():
    prefill_case([0, 5, 0, 0, 33, 0], [10, 0, 0, 40, 7, 0], 16, 2, 32, seed=63, behind=11, strided=True)
    prefill_case([20], [0], 8, 2, 16, seed=64, scale=0.5)


def test_prefill_many_short_sequences():
    prefill_case([1 + (7 * i) % 11 for i in range(60)], [(13 * i) % 90 for i in range(60)], 8, 2, 16, seed=65)


def test_prefill_scores_that_rise_along_the_keys():
    """The running maximum has to be raised often, by much."""
    prefill_case([260], [300], 8, 2, 16, seed=66, sharp=6.0)
    nq, nkv, ps, n = 8, 1, 64, 700
    c = Cache([n], nkv, ps, 67)
    ramp = torch.arange(n).float()
    for s in range(n):
        c.k[int(c.table[0, s // ps]), :, s % ps] = 0
        c.k[int(c.table[0, s // ps]), :, s % ps, 0] = ramp[s] * 0.5
    q = torch.zeros(n, nq, HD).bfloat16()
    q[:, :, 0] = 4.0
    out = ops.paged_prefill_attention(q.cuda(), c.k.cuda(), c.v.cuda(), c.table.cuda(),
                                      torch.tensor([0, n], dtype=torch.int32).cuda(),
                                      torch.tensor([n], dtype=torch.int32).cuda())
    k, v = c.rows(c.k, 0, n), c.rows(c.v, 0, n)
    s = torch.einsum("thd,xd->htx", q.double(), k[0]) * HD ** -0.5
    s.masked_fill_(torch.ones(n, n).triu(1).bool(), -math.inf)
    ref = torch.einsum("htx,xd->thd", torch.softmax(s, -1), v[0])
    near(out.view(n, nq, HD), ref, float(v.abs().max()), atol=2 ** -8 + 2 ** -9)


def test_prefill_equals_decode_of_the_last_token():
    """The two kernels on the same cache, the store between them."""
    nq, nkv, ps, lens = 32, 4, 16, [1, 37, 400]
    c = Cache(lens, nkv, ps, 68)
    g = torch.Generator().manual_seed(68)
    qkv = torch.randn(sum(lens), (nq + 2 * nkv) * HD, generator=g).bfloat16().cuda()
    qw, kw = (w.cuda() for w in weights(68))
    k, v, table = c.k.cuda(), c.v.cuda(), c.table.cuda()
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    kv = torch.tensor(lens, dtype=torch.int32).cuda()
    q = ops.qk_norm_rope_store(qkv, qw, kw, cu, kv, k, v, table, nq, nkv)
    o = ops.paged_prefill_attention(q, k, v, table, cu, kv)
    last = (cu[1:] - 1).long()
    k2, v2 = k.clone(), v.clone()
    d = ops.paged_decode_attention(qkv[last], qw, kw, (kv - 1).long(), k2, v2, table, nq, nkv)
    ops.read_paged_status()
    assert torch.equal(k.view(torch.int16), k2.view(torch.int16)) and torch.equal(v.view(torch.int16), v2.view(torch.int16))
    assert (o[last].float() - d.float()).abs().max() <= 2 ** -5


def test_prefill_two_streams_and_graphs():
    nq, nkv, ps = 16, 2, 64
    cases = []
    for seed in (70, 71):
        c = Cache([3000, 50], nkv, ps, seed)
        g = torch.Generator().manual_seed(seed)
        q = torch.randn(40, nq, HD, generator=g).bfloat16().cuda()
        cu = torch.tensor([0, 30, 40], dtype=torch.int32).cuda()
        args = (q, c.k.cuda(), c.v.cuda(), c.table.cuda(), cu, torch.tensor([3000, 50], dtype=torch.int32).cuda())
        cases.append((args, ops.paged_prefill_attention(*args)))
    torch.cuda.synchronize()
    side, graphs = torch.cuda.Stream(), []
    for args, want in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = ops.paged_prefill_attention(*args)
        graphs.append((g, out, want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        here = ops.paged_prefill_attention(*cases[0][0])
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, want in graphs) and torch.equal(here, cases[0][1])
    ops.read_paged_status()


def test_prefill_reports_lengths_and_pages(monkeypatch):
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    nq, nkv, ps = 8, 2, 16
    c = Cache([40, 30], nkv, ps, 72)
    q = torch.randn(70, nq, HD).bfloat16().cuda()
    k, v, table = c.k.cuda(), c.v.cuda(), c.table.cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    good = ops.paged_prefill_attention(q, k, v, table, i32(0, 40, 70), i32(40, 30))
    ops.read_paged_status()
    for cu, kv in ((i32(0, 40, 71), i32(40, 31)), (i32(0, 40, 30), i32(40, 30)), (i32(-3, 40, 70), i32(43, 30)),
                   (i32(0, 40, 70), i32(39, 30)), (i32(0, 40, 70), i32(40, 3000)), (i32(0, 0, 70), i32(-5, 70))):
        ops.paged_prefill_attention(q, k, v, table, cu, kv)
        with pytest.raises(NKIMoEError):
            ops.read_paged_status()
    wide = torch.cat([table, table[:, :1], table[:, :1]], 1)
    ops.paged_prefill_attention(q, k, v, wide[[0, 0, 0]], i32(0, 70, 0, 70), i32(70, 0, 70))  # overlapping
    with pytest.raises(NKIMoEError):
        ops.read_paged_status()
    for bad in (-1, 1000):
        t2 = table.clone()
        t2[1, 0] = bad
        out = ops.paged_prefill_attention(q, k, v, t2, i32(0, 40, 70), i32(40, 30))
        with pytest.raises(NKIMoEError):
            ops.read_paged_status()
        assert torch.equal(out[:40], good[:40])


def test_kept_keys_are_the_rounded_ones():
    """Keys against the formula in 64 bits, rounded once: fp32 alone puts about 3 of 10^5
    values on the other side of the middle between two bf16 values; those near one are
    formed again, so at most 1 of 10^6 may differ (and 2, so that one value is no failure)."""
    for B, new, past, nq, nkv, ps, seed in ((3, 701, 20000, 12, 4, 64, 1), (2, 150, 5, 24, 8, 16, 2), (1, 4001, 0, 6, 2, 256, 3)):
        total = [past + new + b for b in range(B)]
        c = Cache(total, nkv, ps, seed)
        g = torch.Generator().manual_seed(seed)
        T = B * new
        qkv = torch.randn(T, (nq + 2 * nkv) * HD, generator=g).bfloat16()
        w = (1 + 0.2 * torch.randn(HD, generator=g)).bfloat16()
        kd, vd = c.k.cuda(), c.v.cuda()
        cu = torch.arange(B + 1, dtype=torch.int32) * new
        ops.qk_norm_rope_store(qkv.cuda(), w.cuda(), w.cuda(), cu.cuda(), torch.tensor(total, dtype=torch.int32).cuda(),
                               kd, vd, c.table.cuda(), nq, nkv)
        x = qkv.view(T, -1, HD)[:, nq:nq + nkv].double()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
        pos = torch.cat([torch.arange(t - new, t) for t in total]).double()
        ang = pos[:, None, None] * 1e6 ** (-torch.arange(HD // 2, dtype=torch.float64) / (HD // 2))
        a, b = x[..., :HD // 2], x[..., HD // 2:]
        ref = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1).float().bfloat16()
        got = torch.cat([c.rows(kd.cpu(), i, t)[:, t - new:].transpose(0, 1) for i, t in enumerate(total)])
        bad = int((got.double() != ref.double()).sum())
        assert bad <= 2 + 1e-6 * ref.numel(), f"{bad} of {ref.numel()}"


@pytest.mark.parametrize("pool,n", [(2000, 900), (70000, 3)])
def test_copy_pages_takes_lists_tuples_and_vectors(pool, n):
    g = torch.Generator().manual_seed(n)
    at = torch.randperm(pool, generator=g)[:2 * n]
    want = torch.randn(pool, 1, 16, 8, generator=g).bfloat16().cuda()
    start = want.clone()
    want[at[n:].cuda()] = want[at[:n].cuda()]
    for form in (list, tuple, torch.tensor, lambda x: torch.tensor(x, dtype=torch.int32)):
        got = start.clone()
        ops.copy_pages(got, form(at[:n].tolist()), form(at[n:].tolist()))
        assert torch.equal(got, want)
    ops.copy_pages(got, [], ())
    assert torch.equal(got, want)


# ------------------------------------------------------------------ status
def test_reports_survive_a_larger_workspace(monkeypatch):
    """A bad row is reported after a later, larger call of the stream too, in a captured graph as well."""
    monkeypatch.setenv("NKIMOE_SYNC_CHECK", "0")
    nq, nkv = 4, 2
    pages = torch.zeros(64, nkv, 256, HD, dtype=torch.bfloat16, device="cuda")
    qkv = torch.randn(8, (nq + 2 * nkv) * HD, device="cuda").bfloat16()
    w = torch.ones(HD, dtype=torch.bfloat16, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, table = i32(0, 8), torch.arange(64, dtype=torch.int32, device="cuda")[None]
    logits, tokens = torch.randn(8, 60000, device="cuda"), torch.zeros(8, dtype=torch.int64, device="cuda")
    lens, far = i32(9000), i32(100_000)

    def calls(kv):
        q = ops.qk_norm_rope_store(qkv, w, w, cu, kv, pages, pages, table, nq, nkv)  # 100000 has no place
        ops.paged_prefill_attention(q, pages, pages, table, cu, lens)
        ops.token_logprobs(logits, tokens, 5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    fresh = [k for k in ops._paged_ws if k[1] == side.cuda_stream]
    for k in fresh:  # as on a stream that no call has used
        del ops._paged_ws[k]
    with torch.cuda.stream(side):
        calls(far)
    with pytest.raises(NKIMoEError):
        ops.read_paged_status()
    ops.read_paged_status()
    with torch.cuda.stream(side):
        calls(lens)
    ops.read_paged_status()
    kv = lens.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        calls(kv)
    g.replay()
    ops.read_paged_status()
    kv.copy_(far)
    g.replay()
    with pytest.raises(NKIMoEError):
        ops.read_paged_status()


def test_outputs_lie_apart_from_what_is_read():
    nq, nkv, B = 8, 2, 5
    args = step_inputs([70, 33, 50, 1, 17], nq, nkv, 16, 33)
    qkv, qw, kw, pos, k, v, table = args[:7]
    want = ops.paged_decode_attention(*args)
    row = (nq + 2 * nkv) * HD
    buf = torch.empty(B * row + B * nq * HD, dtype=torch.bfloat16, device="cuda")
    buf[:B * row] = qkv.reshape(-1)
    rows = buf[:B * row].view(B, row)
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    kv = (pos + 1).int()
    for at in (0, 64, 2 * row, B * row - 8):
        out = buf[at:at + B * nq * HD].view(B, nq * HD)
        with pytest.raises(ValueError):
            ops.paged_decode_attention(rows, *args[1:], out=out)
        with pytest.raises(ValueError):
            ops.qk_norm_rope_store(rows, qw, kw, cu, kv, k, v, table, nq, nkv, out=out.view(B, nq, HD))
    out = buf[B * row:].view(B, nq * HD)  # right behind
    assert ops.paged_decode_attention(rows, *args[1:], out=out) is out and torch.equal(out, want)
    q = ops.qk_norm_rope_store(rows, qw, kw, cu, kv, k, v, table, nq, nkv, out=out.view(B, nq, HD))
    want = ops.paged_prefill_attention(q, k, v, table, cu, kv)
    for at in (8, nq * HD):
        with pytest.raises(ValueError):
            ops.paged_prefill_attention(buf[:B * nq * HD].view(B, nq, HD), k, v, table, cu, kv,
                                        out=buf[at:at + B * nq * HD].view(B, nq * HD))
    apart = torch.empty(B, 2 * nq, HD, dtype=torch.bfloat16, device="cuda")
    apart[:, :nq] = q
    with pytest.raises(ValueError):  # rows with gaps cannot be written in place
        ops.paged_prefill_attention(apart[:, :nq], k, v, table, cu, kv,
                                    out=apart.view(-1)[:B * nq * HD].view(B, nq * HD))
    got = ops.paged_prefill_attention(q, k, v, table, cu, kv, out=q.view(B, nq * HD))
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    ops.read_paged_status()


@pytest.mark.parametrize("new,past,window", [(700, 0, 0), (45, 9000, 0), (300, 4000, 600)])
def test_prefill_over_its_own_queries(new, past, window):
    """Whole pairs and cut ones, into the queries' own rows."""
    nq, nkv, ps = 16, 2, 64
    c = Cache([past + new, past + new + 7], nkv, ps, 90)
    g = torch.Generator().manual_seed(new)
    q = torch.randn(2 * new, nq, HD, generator=g).bfloat16().cuda()
    args = (c.k.cuda(), c.v.cuda(), c.table.cuda(), torch.tensor([0, new, 2 * new], dtype=torch.int32).cuda(),
            torch.tensor([past + new, past + new + 7], dtype=torch.int32).cuda())
    want = ops.paged_prefill_attention(q, *args, window=window, sinks=4 if window else 0)
    ops.paged_prefill_attention(q, *args, window=window, sinks=4 if window else 0, out=q.view(2 * new, nq * HD))
    assert torch.equal(q.view(2 * new, nq * HD), want)
    ops.read_paged_status()
