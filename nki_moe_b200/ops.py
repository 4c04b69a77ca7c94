"""Tensor-level entry points over the C ABI.

PyTorch is used here only as plumbing: device memory, the current CUDA
stream and dtype conversions at the boundary.  Every computation runs in
``libnkimoe.so``; CPU tensors are rejected (no CPU fallback), except as the
host buffers of :func:`moe_block_host`, whose block runs on the GPU.
"""

from __future__ import annotations

import array
import ctypes
import functools
import os
import threading
import weakref
from collections import OrderedDict

import torch

from . import _lib
from ._lib import BF16, F32, F64, I32, I64, LAYOUT_HF, LAYOUT_NXD, call, size_call

__all__ = [
    "rmsnorm", "add_rmsnorm", "qk_norm_rope", "router_logits", "topk_softmax", "permute",
    "pack_gate_up", "pack_down", "PackedExperts", "packed_experts", "moe_experts", "moe_block",
    "grouped_gemm", "swiglu", "aggregate", "read_status", "workspace", "sync_check_enabled", "router_split",
    "route", "dispatch", "segment_experts", "combine", "ep_dispatch", "decode_attention", "skinny_linear",
    "moe_block_add_rmsnorm", "moe_block_host", "kmajor_weights",
    "release_captured_workspaces", "moe_block_rmsnorm", "qk_norm_rope_store", "paged_decode_attention",
    "paged_prefill_attention", "copy_pages", "token_logprobs", "read_paged_status",
    "paged_tree_attention", "accept_drafts", "sample_tokens",
]

_DT = {torch.float32: F32, torch.bfloat16: BF16, torch.int32: I32, torch.int64: I64}


def sync_check_enabled() -> bool:
    """When NKIMOE_SYNC_CHECK=1, every block call synchronises and raises on a
    device-flagged fault (timeout, expert id out of range) -- except while a
    CUDA graph is being captured, where a synchronisation is not allowed."""
    return os.environ.get("NKIMOE_SYNC_CHECK", "0") == "1" and not torch.cuda.is_current_stream_capturing()


def _cuda(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this package has no CPU path)")
    return t


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None and t.numel() > 0 else ctypes.c_void_p(0)


def _s(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _contig(t: torch.Tensor, dtype=None) -> torch.Tensor:
    if dtype is not None and t.dtype != dtype:
        t = t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


# ---------------------------------------------------------------- workspace
_ws_lock = threading.Lock()
_ws: dict = {}
# Buffers that a CUDA graph captured and that a later, larger call replaced:
# the graph still writes them on every replay, so they stay alive until the
# caller says its graphs are gone (release_captured_workspaces).
_ws_retired: list = []


def _grow(table: dict, key, device: torch.device, nbytes: int, zero: bool) -> torch.Tensor:
    """The buffer of ``table[key]``, replaced by a larger one when it is
    smaller than ``nbytes``.  A buffer handed out while the current stream
    is being captured is marked, and a marked buffer that gets replaced is
    kept in ``_ws_retired`` instead of going back to the allocator."""
    capturing = torch.cuda.is_current_stream_capturing()
    with _ws_lock:
        buf = table.get(key)
        if buf is None or buf.numel() < nbytes:
            if buf is not None and getattr(buf, "_nkimoe_captured", False):
                _ws_retired.append(buf)
            n = max(nbytes, 1 << 20 if not zero else 1 << 16)
            buf = torch.zeros(n, dtype=torch.uint8, device=device) if zero else \
                torch.empty(n, dtype=torch.uint8, device=device)
            table[key] = buf
        if capturing:
            buf._nkimoe_captured = True
        return buf


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """A per-(device, stream) scratch buffer from the torch caching allocator,
    grown on demand and reused by later calls on the same stream.  A buffer
    that a CUDA graph captured outlives its replacement by a larger call
    (streams from torch's pool reuse their handles), until
    :func:`release_captured_workspaces`."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    return _grow(_ws, key, device, nbytes, zero=False)


def release_captured_workspaces() -> int:
    """Drop the replaced workspaces kept for captured CUDA graphs (call after
    those graphs are destroyed), and what the paged calls hold of the last
    graph's memory.  Returns how many replaced ones were released."""
    with _ws_lock:
        n = len(_ws_retired)
        _ws_retired.clear()
        for key in [k for k in _paged_ws if k[2]]:
            del _paged_ws[key]
    return n


def read_status(ws: torch.Tensor) -> int:
    st = ctypes.c_int(0)
    call("nkimoe_read_status", _p(ws), _s(ws), ctypes.byref(st))
    return st.value


# ---------------------------------------------------------------- norms
def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, out_dtype=None) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last axis (K1)."""
    _cuda(x, "x")
    _cuda(weight, "weight")
    if x.dtype not in (torch.float32, torch.bfloat16):
        x = x.to(torch.bfloat16)
    if weight.dtype not in (torch.float32, torch.bfloat16):
        weight = weight.float()
    x = _contig(x)
    weight = _contig(weight)
    out_dtype = out_dtype or x.dtype
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    H = x.shape[-1]
    rows = x.numel() // H if H else 0
    call("nkimoe_rmsnorm", _p(x), _DT[x.dtype], _p(weight), _DT[weight.dtype], _p(out), _DT[out_dtype],
         rows, H, float(eps), _s(x))
    return out


def add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                residual_out: torch.Tensor | None = None):
    """``r = x + residual``; returns ``(rmsnorm(r), r)`` (bf16)."""
    x = _contig(_cuda(x, "x"), torch.bfloat16)
    residual = _contig(_cuda(residual, "residual"), torch.bfloat16)
    weight = _contig(_cuda(weight, "weight"))
    if weight.dtype not in (torch.float32, torch.bfloat16):
        weight = weight.float()
    if residual_out is None:
        residual_out = torch.empty_like(x)
    out = torch.empty_like(x)
    H = x.shape[-1]
    call("nkimoe_add_rmsnorm", _p(x), _p(residual), _p(residual_out), _p(weight), _DT[weight.dtype], _p(out),
         x.numel() // H, H, float(eps), _s(x))
    return out, residual_out


def qk_norm_rope(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                 n_heads: int, n_kv_heads: int, head_dim: int = 128, theta: float = 1e6, eps: float = 1e-6,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Per-head q/k RMSNorm + rotate-half RoPE on a fused ``[T, (nh+2nkv)*d]``
    bf16 QKV row (K6).  ``out`` may be ``qkv`` (in place)."""
    qkv = _contig(_cuda(qkv, "qkv"), torch.bfloat16)
    T = qkv.numel() // ((n_heads + 2 * n_kv_heads) * head_dim)
    wdt = torch.float32 if q_weight.dtype == torch.float32 else torch.bfloat16
    qw = _contig(_cuda(q_weight, "q_weight"), wdt)
    kw = _contig(_cuda(k_weight, "k_weight"), wdt)
    pos = _contig(_cuda(positions, "positions").reshape(-1), torch.int64)
    if pos.numel() != T:
        raise ValueError(f"positions has {pos.numel()} entries for {T} tokens")
    if out is None:
        out = torch.empty_like(qkv)
    call("nkimoe_qk_norm_rope", _p(qkv), _p(out), _p(qw), _p(kw), _DT[wdt], _p(pos), T, n_heads, n_kv_heads,
         head_dim, float(theta), float(eps), _s(qkv))
    return out


_attn_ws: dict = {}


def _attention_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Zero-filled per-(device, stream) workspace of the decode attention
    (its split counters must start at zero; every call leaves them at zero).
    Kept for captured graphs as :func:`workspace` is."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    return _grow(_attn_ws, key, device, nbytes, zero=True)


def decode_attention(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                     k_cache: torch.Tensor, v_cache: torch.Tensor, n_heads: int, n_kv_heads: int,
                     theta: float = 1e6, eps: float = 1e-6, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """One decode step of grouped-query attention over a KV cache, fused with
    the q/k RMSNorm + RoPE of the step's token and the store of its key and
    value at its position.

    ``qkv``: ``[B, (n_heads + 2*n_kv_heads) * 128]`` bf16, the QKV projection
    before the norms; ``positions``: int64 ``[B]`` or ``[1]`` (one position for
    every sequence); ``k_cache``/``v_cache``: one layer's ``[B', n_kv_heads,
    max_seq, 128]`` bf16 caches (B' >= B, updated in place).  Returns
    ``[B, n_heads * 128]`` bf16."""
    hd = 128
    qkv = _cuda(qkv, "qkv")
    if qkv.dtype != torch.bfloat16 or not qkv.is_contiguous():
        raise ValueError("qkv must be a contiguous bf16 tensor")
    B = qkv.numel() // ((n_heads + 2 * n_kv_heads) * hd)
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        _cuda(c, name)
        if c.dtype != torch.bfloat16 or c.dim() != 4 or c.shape[1] != n_kv_heads or c.shape[3] != hd:
            raise ValueError(f"{name} must be bf16 [B, {n_kv_heads}, max_seq, {hd}]")
        if c.shape[0] < B or not c[:B].is_contiguous():
            raise ValueError(f"{name} must hold {B} contiguous sequences")
    max_seq = k_cache.shape[2]
    if v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache differ in shape")
    wdt = torch.float32 if q_weight.dtype == torch.float32 else torch.bfloat16
    qw = _contig(_cuda(q_weight, "q_weight"), wdt)
    kw = _contig(_cuda(k_weight, "k_weight"), wdt)
    pos = _cuda(positions, "positions").reshape(-1)
    if pos.dtype != torch.int64 or not pos.is_contiguous():
        raise ValueError("positions must be a contiguous int64 tensor")
    if pos.numel() not in (1, B):
        raise ValueError(f"positions has {pos.numel()} entries for {B} sequences")
    if out is None:
        out = torch.empty(B, n_heads * hd, dtype=torch.bfloat16, device=qkv.device)
    nbytes = size_call("nkimoe_decode_attention_workspace_bytes", B, n_heads, n_kv_heads, hd, max_seq)
    ws = _attention_workspace(qkv.device, nbytes)
    call("nkimoe_decode_attention", _p(qkv), _p(qw), _p(kw), _DT[wdt], _p(pos), 0 if pos.numel() == 1 else 1,
         _p(k_cache), _p(v_cache), _p(out), B, n_heads, n_kv_heads, hd, max_seq, float(theta), float(eps),
         float(scale if scale is not None else hd ** -0.5), _p(ws), ws.numel(), _s(qkv))
    if sync_check_enabled():
        read_status(ws)
    return out


def skinny_linear(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ w.T`` for at most 16 rows of ``x`` (bf16, fp32 accumulation):
    the decode step's projections, streaming ``w`` [N, K] once."""
    x = _cuda(x, "x")
    w = _cuda(w, "w")
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        raise ValueError("skinny_linear takes bf16 x and w")
    x = _contig(x)
    w = _contig(w)
    K = x.shape[-1]
    M = x.numel() // K if K else 0
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"w is {tuple(w.shape)}, x has {K} columns")
    if out is None:
        out = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=x.device)
    call("nkimoe_skinny_linear", _p(x), _p(w), _p(out), M, N, K, _s(x))
    return out


# ---------------------------------------------------------------- paged cache, token scores
_paged_ws: dict = {}
_paged_sinks: list = []  # weak references to status words of graphs' owners
_raw_stream = torch._C._cuda_getCurrentRawStream
_PAGE_SIZES = (16, 32, 64, 128, 256)
_STATUS_BYTES = 4  # the status word at the head of a workspace


@functools.lru_cache(maxsize=512)
def _paged_ws_bytes(device_index: int, name: str, *args) -> int:
    """A workspace size (a function of the sizes and the device's SM count)."""
    return size_call(name, *args)


def _paged_workspace(dev: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """Zero-filled workspace of the paged-cache and token-score calls, one per
    (device, stream).  A stream that is being captured gets one per capture,
    allocated (and zeroed, as a node of the graph) in the graph's own memory,
    so graphs that replay at the same time share none; only the latest
    capture's is held here, the graph keeps the memory.  A larger workspace
    takes over the status of the one that it replaces."""
    capture = 0
    if torch.cuda.is_current_stream_capturing():
        cid = ctypes.c_ulonglong(0)
        call("nkimoe_stream_capture_id", stream, ctypes.byref(cid))
        capture = cid.value
    key = (dev.index, stream, capture != 0)
    held = _paged_ws.get(key)
    if held is not None and held[0] == capture and held[1].numel() >= nbytes:
        return held[1]
    with _ws_lock:
        held = _paged_ws.get(key)  # again: another thread may have been here
        if held is not None and held[0] == capture and held[1].numel() >= nbytes:
            return held[1]
        ws = torch.zeros(max(nbytes, 1 << 16), dtype=torch.uint8, device=dev)
        if held is not None and held[0] == capture:  # a smaller one: what it has reported goes on
            ws[:_STATUS_BYTES].copy_(held[1][:_STATUS_BYTES])
        _paged_ws[key] = (capture, ws)
        return ws


def _status_sink(device: torch.device) -> torch.Tensor:
    """A status word that collects what the replays of its owner's graphs report
    (:func:`_end_of_capture`); :func:`read_paged_status` reads it while it lives."""
    sink = torch.zeros(1, dtype=torch.int32, device=device)
    with _ws_lock:
        _paged_sinks[:] = [r for r in _paged_sinks if r() is not None] + [weakref.ref(sink)]
    return sink


def _end_of_capture(sink: torch.Tensor) -> list:
    """Called last in a capture on the current stream, by the owner of the
    graph: each replay ends by adding its paged calls' status to ``sink``.
    Returns the workspaces that the capture uses, which the owner holds as long
    as the graph."""
    key = (sink.device.index, torch.cuda.current_stream(sink.device).cuda_stream)
    with _ws_lock:
        held = [table[key] for table in (_ws, _attn_ws) if key in table]
        paged = _paged_ws.pop(key + (True,), None)
    if paged is not None:
        sink.bitwise_or_(paged[1][:_STATUS_BYTES].view(torch.int32))
        held.append(paged[1])
    return held


def read_paged_status(device=None) -> None:
    """Synchronises ``device`` and raises if a paged-cache call on it met a
    position or page id out of range, or a page that it needed and that was
    not held (the status is cleared).  Of calls in a caller's own CUDA graphs it
    sees the last replay of the graph captured last on each stream: a replay
    begins by clearing its own status.  The decoder stack's captured steps
    collect theirs, and every one is seen."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    torch.cuda.synchronize(index)
    with _ws_lock:
        held = [v[1] for k, v in _paged_ws.items() if k[0] == index]
        sinks = [r() for r in _paged_sinks]
        held += [t for t in sinks if t is not None and t.get_device() == index]
    bad = None
    with torch.cuda.device(index):
        for ws in held:
            try:
                call("nkimoe_read_status", ws.data_ptr(), _raw_stream(index), None)
            except _lib.NKIMoEError as e:
                bad = e
    if bad is not None:
        raise bad


def _on_its_device(fn):
    """Runs ``fn`` with the device of its first CUDA tensor as the current one (its
    kernels launch there, on that device's current stream)."""
    @functools.wraps(fn)
    def run(*args, **kw):
        t = args[0] if args else next((v for v in kw.values() if isinstance(v, torch.Tensor) and v.is_cuda), None)
        if isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() != torch._C._cuda_getDevice():
            with torch.cuda.device(t.device):
                return fn(*args, **kw)
        return fn(*args, **kw)
    return run


def _same_device(index: int, names: str, *tensors: torch.Tensor) -> None:
    for i, t in enumerate(tensors):
        if t.get_device() != index:
            raise ValueError(f"{names.split()[i]} is on {t.device}, expected cuda:{index}")


def _norm_weights(q_weight: torch.Tensor, k_weight: torch.Tensor):
    wdt = q_weight.dtype
    if wdt != torch.bfloat16 or k_weight.dtype != wdt or not q_weight.is_contiguous() or not k_weight.is_contiguous():
        wdt = torch.float32 if wdt == torch.float32 else torch.bfloat16
        q_weight, k_weight = _contig(_cuda(q_weight, "q_weight"), wdt), _contig(_cuda(k_weight, "k_weight"), wdt)
    if q_weight.numel() != 128 or k_weight.numel() != 128:
        raise ValueError("q_weight and k_weight must have 128 elements")
    return q_weight, k_weight, _DT[wdt]


def _page_stride(c: torch.Tensor, name: str, n_kv_heads: int) -> int:
    """Checks one pool and returns the elements between its pages."""
    shape = c.shape
    if not c.is_cuda or c.dtype != torch.bfloat16 or len(shape) != 4 or shape[1] != n_kv_heads or shape[3] != 128:
        raise ValueError(f"{name} must be CUDA bf16 [pages, {n_kv_heads}, page_size, 128]")
    if shape[2] not in _PAGE_SIZES:
        raise ValueError(f"page size {shape[2]} (one of {_PAGE_SIZES})")
    if shape[0] == 0:
        raise ValueError(f"{name} has no pages")
    page = n_kv_heads * shape[2] * 128
    if c.is_contiguous():
        return page
    st = c.stride()
    if st[3] != 1 or st[2] != 128 or (n_kv_heads > 1 and st[1] != 128 * shape[2]):
        raise ValueError(f"{name}: the pages themselves must be contiguous")
    return st[0] if shape[0] > 1 else page


def _paged_cache(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, n_kv_heads: int,
                 batch: int):
    """Checks one layer's pools and the page table of ``batch`` sequences and
    returns their C arguments."""
    shape = k_pages.shape
    if len(shape) == 4 and shape == v_pages.shape and shape[1] == n_kv_heads and shape[3] == 128 and shape[0] \
            and shape[2] in _PAGE_SIZES and k_pages.dtype == v_pages.dtype == torch.bfloat16 \
            and k_pages.is_contiguous() and v_pages.is_contiguous():
        kst = vst = n_kv_heads * shape[2] * 128
    else:
        kst, vst = _page_stride(k_pages, "k_pages", n_kv_heads), _page_stride(v_pages, "v_pages", n_kv_heads)
        if v_pages.shape != shape:
            raise ValueError("k_pages and v_pages differ in shape")
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise ValueError("page_table must be CUDA int32 [sequences, pages per sequence]")
    rows, width = page_table.shape
    if rows < batch or width == 0 or (width > 1 and page_table.stride(1) != 1):
        raise ValueError(f"page_table must have contiguous rows for {batch} sequences")
    return (k_pages.data_ptr(), v_pages.data_ptr(), kst, vst, shape[0], shape[2], page_table.data_ptr(),
            page_table.stride(0) if rows > 1 else width, width)


def _lengths(cu_seqlens: torch.Tensor, kv_lens: torch.Tensor) -> int:
    for name, t in (("cu_seqlens", cu_seqlens), ("kv_lens", kv_lens)):
        if not t.is_cuda or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous CUDA int32 vector")
    if cu_seqlens.shape[0] != kv_lens.shape[0] + 1:
        raise ValueError(f"cu_seqlens has {cu_seqlens.shape[0]} entries for {kv_lens.shape[0]} sequences")
    return kv_lens.shape[0]


def _rows_out(out: torch.Tensor | None, shape: tuple, like: torch.Tensor, in_place: bool = False) -> torch.Tensor:
    """``out`` checked against the rows ``like`` (bf16) that the call reads, or
    a new tensor on their device.  A call writes some rows while it still
    reads others, so the two must lie apart, or with ``in_place`` be the same."""
    if out is None:
        return like.new_empty(shape)
    dev = like.device
    if out.dtype != torch.bfloat16 or out.shape != shape or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out must be a contiguous bf16 {list(shape)} tensor on {dev}")
    if out.numel() and like.numel():
        a, b = out.data_ptr(), like.data_ptr()
        last = sum((n - 1) * st for n, st in zip(like.shape, like.stride()))
        if a < b + 2 * (last + 1) and b < a + 2 * out.numel() and not (in_place and a == b and like.is_contiguous()):
            raise ValueError("out must not overlap the rows that the call reads")
    return out


@_on_its_device
def qk_norm_rope_store(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cu_seqlens: torch.Tensor,
                       kv_lens: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                       n_heads: int, n_kv_heads: int, theta: float = 1e6, eps: float = 1e-6,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Prompt rows into a paged cache: per-head q/k RMSNorm + rotate-half RoPE
    of the packed QKV rows, keys and values stored in their pages, queries
    returned.

    ``qkv``: ``[T, (n_heads + 2*n_kv_heads) * 128]`` bf16; ``cu_seqlens``:
    int32 ``[B + 1]``, the first row of each sequence; ``kv_lens``: int32
    ``[B]``, its length with the new rows (row ``i`` of ``n`` stands at
    ``kv_len - n + i``); ``k_pages``/``v_pages``: one layer's ``[pages,
    n_kv_heads, page_size, 128]`` bf16 pools, updated in place;
    ``page_table``: int32 ``[B, pages per sequence]`` (-1: not kept).  Returns
    the queries ``[T, n_heads, 128]`` bf16 (``out``, contiguous and apart from
    ``qkv``, if given); rows from ``cu_seqlens[B]`` on are left as they were."""
    _cuda(qkv, "qkv")
    row = (n_heads + 2 * n_kv_heads) * 128
    if qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or qkv.shape[1] != row or not qkv.is_contiguous():
        raise ValueError(f"qkv must be a contiguous bf16 [T, {row}] tensor")
    T, dev = qkv.shape[0], qkv.device
    B = _lengths(cu_seqlens, kv_lens)
    qw, kw, wdt = _norm_weights(q_weight, k_weight)
    cache = _paged_cache(k_pages, v_pages, page_table, n_kv_heads, B)
    _same_device(dev.index, "q_weight k_weight cu_seqlens kv_lens k_pages v_pages page_table", qw, kw, cu_seqlens,
                 kv_lens, k_pages, v_pages, page_table)
    out = _rows_out(out, (T, n_heads, 128), qkv)
    s = _raw_stream(dev.index)
    ws = _paged_workspace(dev, s, 0)
    call("nkimoe_qk_norm_rope_store", qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), wdt,
             cu_seqlens.data_ptr(), kv_lens.data_ptr(), *cache, out.data_ptr(), T, B, n_heads, n_kv_heads, 128,
             theta, eps, ws.data_ptr(), s)
    if "NKIMOE_SYNC_CHECK" in os.environ and sync_check_enabled():
        read_status(ws)
    return out


@_on_its_device
def paged_decode_attention(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                           positions: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           page_table: torch.Tensor, n_heads: int, n_kv_heads: int, theta: float = 1e6,
                           eps: float = 1e-6, scale: float | None = None, window: int = 0, sinks: int = 0,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """One decode step of grouped-query attention over a paged cache, fused
    with the q/k RMSNorm + RoPE of the step's token and the store of its key
    and value in its page (:func:`decode_attention` on pages).

    ``qkv``: ``[B, (n_heads + 2*n_kv_heads) * 128]`` bf16 before the norms;
    ``positions``: int64 ``[B]`` or ``[1]``, a negative one marks an idle row
    (nothing is stored, its output is zero); ``k_pages``/``v_pages``/
    ``page_table`` as in :func:`qk_norm_rope_store`.  With ``window > 0`` the
    query at ``p`` sees the last ``window`` positions up to ``p`` and the first
    ``sinks`` ones; pages that lie outside both need not be held.  Returns
    ``[B, n_heads * 128]`` bf16 (``out``, contiguous and apart from ``qkv``, if
    given)."""
    _cuda(qkv, "qkv")
    row = (n_heads + 2 * n_kv_heads) * 128
    if qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or qkv.shape[1] != row or not qkv.is_contiguous():
        raise ValueError(f"qkv must be a contiguous bf16 [B, {row}] tensor")
    B, dev = qkv.shape[0], qkv.device
    if not positions.is_cuda or positions.dtype != torch.int64 or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous CUDA int64 tensor")
    n_pos = positions.numel()
    if n_pos != B and n_pos != 1:
        raise ValueError(f"positions has {n_pos} entries for {B} sequences")
    qw, kw, wdt = _norm_weights(q_weight, k_weight)
    cache = _paged_cache(k_pages, v_pages, page_table, n_kv_heads, B)
    _same_device(dev.index, "q_weight k_weight positions k_pages v_pages page_table", qw, kw, positions, k_pages,
                 v_pages, page_table)
    out = _rows_out(out, (B, n_heads * 128), qkv)
    s = _raw_stream(dev.index)
    nbytes = _paged_ws_bytes(dev.index, "nkimoe_paged_decode_attention_workspace_bytes", B, n_heads, n_kv_heads,
                             cache[8], cache[5])
    ws = _paged_workspace(dev, s, nbytes)
    call("nkimoe_paged_decode_attention", qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), wdt,
             positions.data_ptr(), 0 if n_pos == 1 else 1, *cache, out.data_ptr(), B, n_heads, n_kv_heads, 128, theta,
             eps, 128 ** -0.5 if scale is None else scale, window, sinks, ws.data_ptr(), ws.numel(), s)
    if "NKIMOE_SYNC_CHECK" in os.environ and sync_check_enabled():
        read_status(ws)
    return out


@_on_its_device
def paged_prefill_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                            cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, scale: float | None = None,
                            window: int = 0, sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompt rows over a paged cache that already
    holds their keys and values: whole prompts, or chunks of prompts over what
    the cache holds of them.

    ``q``: ``[T, n_heads, 128]`` bf16, normed and rotated (what
    :func:`qk_norm_rope_store` returns), rows at any stride that is a multiple
    of 8; ``cu_seqlens``, ``kv_lens``, ``k_pages``, ``v_pages``,
    ``page_table`` as there; ``window``, ``sinks`` as in
    :func:`paged_decode_attention`.  Cached rows below ``kv_lens`` must be
    finite.  Returns ``[T, n_heads * 128]`` bf16; rows from ``cu_seqlens[B]``
    on are left as they were in ``out`` (apart from ``q``, or a contiguous ``q``
    itself in its place)."""
    _cuda(q, "q")
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[2] != 128 or q.stride(2) != 1 \
            or (q.shape[1] > 1 and q.stride(1) != 128):
        raise ValueError("q must be bf16 [T, n_heads, 128] with contiguous rows")
    T, nq, _ = q.shape
    dev = q.device
    B = _lengths(cu_seqlens, kv_lens)
    nkv = k_pages.shape[1] if k_pages.dim() == 4 else 0
    cache = _paged_cache(k_pages, v_pages, page_table, nkv, B)
    _same_device(dev.index, "cu_seqlens kv_lens k_pages v_pages page_table", cu_seqlens, kv_lens, k_pages, v_pages,
                 page_table)
    out = _rows_out(out, (T, nq * 128), q, in_place=True)
    s = _raw_stream(dev.index)
    nbytes = _paged_ws_bytes(dev.index, "nkimoe_paged_prefill_attention_workspace_bytes", T, B, nq, nkv, cache[8],
                             cache[5])
    ws = _paged_workspace(dev, s, nbytes)
    call("nkimoe_paged_prefill_attention", q.data_ptr(), q.stride(0) if T > 1 else nq * 128, *cache,
         cu_seqlens.data_ptr(), kv_lens.data_ptr(), out.data_ptr(), T, B, nq, nkv, 128,
         128 ** -0.5 if scale is None else scale, window, sinks, ws.data_ptr(), ws.numel(), s)
    if "NKIMOE_SYNC_CHECK" in os.environ and sync_check_enabled():
        read_status(ws)
    return out


@_on_its_device
def paged_tree_attention(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, parents: torch.Tensor,
                         cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, k_pages: torch.Tensor,
                         v_pages: torch.Tensor, page_table: torch.Tensor, n_heads: int, n_kv_heads: int,
                         theta: float = 1e6, eps: float = 1e-6, scale: float | None = None, window: int = 0,
                         sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """One step of grouped-query attention for a tree of drafted tokens per
    sequence over a paged cache, fused with the q/k RMSNorm + RoPE of the nodes
    and the store of their keys and values (:func:`paged_decode_attention` for
    more than one token).

    ``qkv``: ``[T, (n_heads + 2*n_kv_heads) * 128]`` bf16 before the norms, the
    sequences' nodes packed; ``cu_seqlens``, ``kv_lens``, ``k_pages``,
    ``v_pages``, ``page_table`` as in :func:`qk_norm_rope_store`: node ``i`` of
    ``n`` (at most 64) lies in place ``kv_len - n + i`` of the cache.
    ``parents``: int32 ``[T]``, the index of a node's parent among its
    sequence's nodes (below its own) or -1; a node's position, for RoPE and the
    window, is ``kv_len - n`` and its depth.  A node sees what was in the cache
    before the tree, its ancestors and itself, within ``window`` and ``sinks``
    as in :func:`paged_decode_attention`.  Cached rows below ``kv_lens`` and the
    nodes' own must be finite.  Returns ``[T, n_heads * 128]`` bf16 (``out``,
    contiguous and apart from ``qkv``, if given); rows from ``cu_seqlens[B]`` on
    are left as they were.  :func:`accept_drafts` keeps the path that is agreed
    with."""
    _cuda(qkv, "qkv")
    row = (n_heads + 2 * n_kv_heads) * 128
    if qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or qkv.shape[1] != row or not qkv.is_contiguous():
        raise ValueError(f"qkv must be a contiguous bf16 [T, {row}] tensor")
    T, dev = qkv.shape[0], qkv.get_device()
    _node_ids(parents, "parents", torch.int32, T, dev)
    B = _lengths(cu_seqlens, kv_lens)
    qw, kw, wdt = _norm_weights(q_weight, k_weight)
    cache = _paged_cache(k_pages, v_pages, page_table, n_kv_heads, B)
    if not (dev == qw.get_device() == kw.get_device() == cu_seqlens.get_device() == kv_lens.get_device()
            == k_pages.get_device() == v_pages.get_device() == page_table.get_device()):
        _same_device(dev, "q_weight k_weight cu_seqlens kv_lens k_pages v_pages page_table", qw, kw, cu_seqlens,
                     kv_lens, k_pages, v_pages, page_table)
    out = qkv.new_empty((T, n_heads * 128)) if out is None else _rows_out(out, (T, n_heads * 128), qkv)
    s = _raw_stream(dev)
    nbytes = _paged_ws_bytes(dev, "nkimoe_paged_tree_attention_workspace_bytes", T, B, n_heads, n_kv_heads,
                             cache[8], cache[5])
    ws = _paged_workspace(qkv.device, s, nbytes)
    call("nkimoe_paged_tree_attention", qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), wdt, parents.data_ptr(),
         cu_seqlens.data_ptr(), kv_lens.data_ptr(), *cache, out.data_ptr(), T, B, n_heads, n_kv_heads, 128, theta, eps,
         128 ** -0.5 if scale is None else scale, window, sinks, ws.data_ptr(), ws.numel(), s)
    if "NKIMOE_SYNC_CHECK" in os.environ and sync_check_enabled():
        read_status(ws)
    return out


def _page_ids(ids, name: str) -> torch.Tensor:
    if isinstance(ids, (list, tuple)):
        try:
            ids = array.array("i", ids)
        except (TypeError, OverflowError) as e:
            raise ValueError(f"{name} holds what is no page id: {e}") from None
        return torch.frombuffer(ids, dtype=torch.int32) if len(ids) else torch.empty(0, dtype=torch.int32)
    t = torch.as_tensor(ids)
    if t.is_cuda or t.dim() != 1 or (t.numel() and t.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"{name} must be a list or CPU vector of page ids (page bookkeeping is host data)")
    if t.dtype == torch.int64 and t.numel() and (int(t.max()) > 0x7fffffff or int(t.min()) < -0x80000000):
        raise ValueError(f"{name} holds ids that are not page ids")
    return _contig(t, torch.int32)


@_on_its_device
def copy_pages(pages: torch.Tensor, src, dst) -> torch.Tensor:
    """Copies page ``src[i]`` to page ``dst[i]`` in every plane of a pool, in
    place: forks (the last page of a sequence that two continue) and
    compactions, all layers' keys and values in one launch.

    ``pages``: contiguous CUDA tensor ``[..., pages, n_kv_heads, page_size,
    head_dim]`` of any type (a stack's pool is ``[layers, 2, pages, ...]``);
    ``src``/``dst``: lists or CPU vectors.  Ids out of range, a page written
    twice, or one that is both read and written are refused before anything
    is copied.  Returns ``pages``."""
    _cuda(pages, "pages")
    if pages.dim() < 4 or not pages.is_contiguous():
        raise ValueError("pages must be contiguous [..., pages, n_kv_heads, page_size, head_dim]")
    src, dst = _page_ids(src, "src"), _page_ids(dst, "dst")
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} source pages for {dst.numel()} destinations")
    if src.numel() == 0:
        return pages
    shape, dev = pages.shape, pages.device
    page_bytes = shape[-1] * shape[-2] * shape[-3] * pages.element_size()
    if pages.numel() == 0:
        raise ValueError("pages is empty")
    call("nkimoe_copy_pages", pages.data_ptr(), pages.numel() // (shape[-1] * shape[-2] * shape[-3] * shape[-4]),
             shape[-4], page_bytes, src.data_ptr(), dst.data_ptr(), src.numel(), _raw_stream(dev.index))
    return pages


@_on_its_device
def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_n: int = 0):
    """Scores of given tokens under rows of logits, in one pass over them:
    ``(logprob [T], entropy [T], top_logprobs [T, top_n], top_ids [T,
    top_n])``, fp32 and int64.

    ``logits``: ``[T, V]`` bf16 or fp32, rows at any stride; ``tokens``: int64
    ``[T]`` (negative: none given, its logprob is 0; ``>= V``: NaN).  The
    ``top_n`` (at most 32) most likely tokens come in order, equal logits by
    the lower id.  -inf logits have probability zero; a row with a NaN, a +inf
    or only -inf has no distribution and gives NaN."""
    _cuda(logits, "logits")
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("logits must be fp32 or bf16 [T, V]")
    T, V = logits.shape
    if V == 0 or (V > 1 and logits.stride(1) != 1):
        raise ValueError("logits must have contiguous, non-empty rows")
    if not tokens.is_cuda or tokens.dtype != torch.int64 or tokens.shape != (T,) or not tokens.is_contiguous():
        raise ValueError(f"tokens must be a contiguous CUDA int64 [{T}] tensor")
    if not 0 <= top_n <= min(32, V):
        raise ValueError(f"top_n {top_n} is not in [0, min(32, {V})]")
    dev = logits.device
    _same_device(dev.index, "tokens", tokens)
    lp = torch.empty(T, dtype=torch.float32, device=dev)
    ent = torch.empty_like(lp)
    top_lp = lp.new_empty((T, top_n))
    top_ids = tokens.new_empty((T, top_n))
    if T == 0:
        return lp, ent, top_lp, top_ids
    s = _raw_stream(dev.index)
    ws = _paged_workspace(dev, s, _paged_ws_bytes(dev.index, "nkimoe_token_logprobs_workspace_bytes", T, V, top_n))
    call("nkimoe_token_logprobs", logits.data_ptr(), _DT[logits.dtype], logits.stride(0) if T > 1 else V,
             tokens.data_ptr(), T, V, top_n, lp.data_ptr(), ent.data_ptr(), top_lp.data_ptr(), top_ids.data_ptr(),
             ws.data_ptr(), ws.numel(), s)
    return lp, ent, top_lp, top_ids


def _setting(value, name: str, dtype: torch.dtype, rows: int, dev: int):
    """A sampling setting as the C pair (array of a value per row, value for all)."""
    if not isinstance(value, torch.Tensor):
        return None, value
    if value.dtype != dtype or value.shape != (rows,) or not value.is_contiguous() or value.get_device() != dev:
        raise ValueError(f"{name} must be a number or a contiguous {dtype} [{rows}] tensor on cuda:{dev}")
    return value.data_ptr(), 0


@_on_its_device
def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """A token from every row of logits, and the logarithm of its probability:
    ``(tokens [T] int64, logprob [T] fp32)``.

    ``logits``: ``[T, V]`` bf16 or fp32, rows at any stride, V at most 2^18;
    ``uniforms``: ``[T]`` fp32 or fp64, a random number of [0, 1) per row.  The
    distribution is ``softmax(logits / temperature)`` restricted, in the order of
    falling logits (equal ones by the lower id), to the first ``top_k`` tokens (0:
    all), of those to the fewest that hold ``top_p`` of their sum (at least one),
    and to probabilities of at least ``min_p`` times the largest.  The token is
    the first id whose running sum over the kept ids, in rising order, exceeds
    ``uniforms`` times the whole.  ``temperature`` 0: the largest logit, the
    lowest id of equal ones, logprob 0.

    Each setting is a number or a tensor ``[T]`` with one per row (fp32; ``top_k``
    int32), in which ``top_k < 1``, ``top_p >= 1`` and ``min_p <= 0`` restrict
    nothing.  -inf logits are never drawn; a row with a NaN, a +inf or only -inf,
    or with a negative or NaN temperature, has no distribution and gives -1 and
    NaN."""
    _cuda(logits, "logits")
    shape, dt, udt, dev = logits.shape, logits.dtype, uniforms.dtype, logits.get_device()
    if len(shape) != 2 or (dt != torch.bfloat16 and dt != torch.float32):
        raise ValueError("logits must be fp32 or bf16 [T, V]")
    T, V = shape
    row, step = logits.stride()
    if V == 0 or (V > 1 and step != 1):
        raise ValueError("logits must have contiguous, non-empty rows")
    if uniforms.get_device() != dev or (udt != torch.float32 and udt != torch.float64) or uniforms.shape != (T,) \
            or not uniforms.is_contiguous():
        raise ValueError(f"uniforms must be a contiguous fp32 or fp64 [{T}] tensor on cuda:{dev}")
    t_rows, t_all = _setting(temperature, "temperature", torch.float32, T, dev)
    k_rows, k_all = _setting(top_k, "top_k", torch.int32, T, dev)
    if k_all > V:  # any number, as all
        k_all = 0
    p_rows, p_all = _setting(top_p, "top_p", torch.float32, T, dev)
    m_rows, m_all = _setting(min_p, "min_p", torch.float32, T, dev)
    tokens = uniforms.new_empty((T,), dtype=torch.int64)
    lp = torch.empty_like(uniforms) if udt == torch.float32 else uniforms.new_empty((T,), dtype=torch.float32)
    call("nkimoe_sample_tokens", logits.data_ptr(), _DT[dt], row if T > 1 else V, uniforms.data_ptr(),
         F32 if udt == torch.float32 else F64, t_rows, t_all, k_rows, k_all, p_rows, p_all, m_rows, m_all, T, V,
         tokens.data_ptr(), lp.data_ptr(), _raw_stream(dev))
    return tokens, lp


def _node_ids(t: torch.Tensor, name: str, dtype: torch.dtype, T: int, dev: int) -> None:
    if t.get_device() != dev or t.dtype != dtype or t.shape != (T,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} [{T}] tensor on cuda:{dev}")


@_on_its_device
def accept_drafts(tokens: torch.Tensor, sampled: torch.Tensor, parents: torch.Tensor, cu_seqlens: torch.Tensor,
                  kv_lens: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor):
    """The end of a step with drafted tokens: ``(counts [B] int32, path [T] int32,
    new_tokens [T] int64)``, and the kept drafts' keys and values in place.

    Packed trees (see :func:`paged_tree_attention`): ``tokens`` int64 ``[T]``, node
    0 of a sequence being its current token, ``sampled`` int64 ``[T]`` what was
    drawn after every node, ``parents``, ``cu_seqlens``, ``kv_lens`` as there.  The
    path begins at node 0 and goes on to the lowest child whose token is what was
    drawn, until there is none; of a sequence's rows in ``path`` and ``new_tokens``
    the first ``counts[b]`` hold its nodes and what was drawn after them, the
    others -1.  In ``pages`` (a pool ``[..., pages, n_kv_heads, page_size,
    head_dim]``, contiguous, any type) the rows of the path's nodes move to the
    places right behind what the cache held before, so that the sequence goes on
    from ``kv_len - n + counts[b]`` positions."""
    _cuda(tokens, "tokens")
    T, dev = tokens.numel(), tokens.get_device()
    _node_ids(tokens, "tokens", torch.int64, T, dev)
    _node_ids(sampled, "sampled", torch.int64, T, dev)
    _node_ids(parents, "parents", torch.int32, T, dev)
    B, width, shape = _lengths(cu_seqlens, kv_lens), page_table.shape, pages.shape
    if pages.get_device() != dev or len(shape) < 4 or not pages.is_contiguous() or 0 in shape:
        raise ValueError(f"pages must be contiguous [..., pages, n_kv_heads, page_size, head_dim] on cuda:{dev}")
    if page_table.get_device() != dev or page_table.dtype != torch.int32 or len(width) != 2:
        raise ValueError(f"page_table must be int32 [sequences, pages per sequence] on cuda:{dev}")
    rows, width = width
    row_step, step = page_table.stride()
    if rows < B or width == 0 or (width > 1 and step != 1):
        raise ValueError(f"page_table must have contiguous rows for {B} sequences")
    if cu_seqlens.get_device() != dev or kv_lens.get_device() != dev:
        raise ValueError(f"cu_seqlens and kv_lens must be on cuda:{dev}")
    counts, path, new = torch.empty_like(kv_lens), torch.empty_like(parents), torch.empty_like(tokens)
    if B == 0 or T == 0:
        return counts.zero_(), path.fill_(-1), new.fill_(-1)
    s = _raw_stream(dev)
    ws = _paged_workspace(tokens.device, s, 0)
    n_pages, heads, size, dim = shape[-4:]
    call("nkimoe_accept_drafts", tokens.data_ptr(), sampled.data_ptr(), parents.data_ptr(), cu_seqlens.data_ptr(),
         kv_lens.data_ptr(), pages.data_ptr(), pages.numel() // (n_pages * heads * size * dim), n_pages, heads, size,
         dim * pages.element_size(), page_table.data_ptr(), row_step if rows > 1 else width, width, counts.data_ptr(),
         path.data_ptr(), new.data_ptr(), T, B, ws.data_ptr(), s)
    if "NKIMOE_SYNC_CHECK" in os.environ and sync_check_enabled():
        read_status(ws)
    return counts, path, new


# ---------------------------------------------------------------- router
def router_logits(x: torch.Tensor, router_w: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    x = _contig(_cuda(x, "x"), torch.bfloat16)
    rw = _contig(_cuda(router_w, "router_w"), torch.float32)
    b = _contig(bias, torch.float32) if bias is not None else None
    T, H = x.shape
    E = rw.shape[0]
    out = torch.empty(T, E, dtype=torch.float32, device=x.device)
    call("nkimoe_router_logits", _p(x), _p(rw), _p(b), _p(out), T, H, E, _s(x))
    return out


def topk_softmax(logits: torch.Tensor, top_k: int):
    lg = _contig(_cuda(logits, "logits"), torch.float32)
    T, E = lg.shape
    idx = torch.empty(T, top_k, dtype=torch.int32, device=lg.device)
    w = torch.empty(T, top_k, dtype=torch.float32, device=lg.device)
    call("nkimoe_topk_softmax", _p(lg), T, E, top_k, _p(idx), _p(w), _s(lg))
    return idx, w


# ---------------------------------------------------------------- permutation
def permute(idx: torch.Tensor, num_experts: int):
    """Returns ``(row_token, row_slot, slot_row, expert_offsets)`` (int32)."""
    idx = _contig(_cuda(idx, "idx"))
    if idx.dtype not in (torch.int32, torch.int64):
        idx = idx.to(torch.int64)
    T, K = idx.shape
    dev = idx.device
    rt = torch.empty(T * K, dtype=torch.int32, device=dev)
    rs = torch.empty(T * K, dtype=torch.int32, device=dev)
    sr = torch.empty(T * K, dtype=torch.int32, device=dev)
    off = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    nbytes = size_call("nkimoe_permute_workspace_bytes", T, K, num_experts)
    ws = workspace(dev, nbytes)
    call("nkimoe_permute", _p(idx), _DT[idx.dtype], T, K, num_experts, _p(rt), _p(rs), _p(sr), _p(off), _p(ws),
         ws.numel(), _s(idx))
    if sync_check_enabled():
        read_status(ws)
    return rt, rs, sr, off


# ---------------------------------------------------------------- weights
class PackedExperts:
    """Expert weights in the GEMM layout: ``w13 [E, 2I, H]`` (K-major, 128-row
    blocks of [gate 64 | up 64]) and ``w2 [E, H, I]`` (K-major), bf16."""

    def __init__(self, w13: torch.Tensor, w2: torch.Tensor, num_experts: int, hidden: int, inter: int):
        self.w13, self.w2 = w13, w2
        self.num_experts, self.hidden, self.inter = num_experts, hidden, inter


def pack_gate_up(gate_up: torch.Tensor, layout: str = "nxd") -> torch.Tensor:
    g = _contig(_cuda(gate_up, "gate_up"), torch.bfloat16)
    if layout == "nxd":
        E, H, I2 = g.shape
        code = LAYOUT_NXD
    elif layout == "hf":
        E, I2, H = g.shape
        code = LAYOUT_HF
    else:
        raise ValueError(f"unknown layout {layout}")
    out = torch.empty(E, I2, H, dtype=torch.bfloat16, device=g.device)
    call("nkimoe_pack_gate_up", _p(g), code, _p(out), E, H, I2 // 2, _s(g))
    return out


def pack_down(down: torch.Tensor, layout: str = "nxd") -> torch.Tensor:
    d = _contig(_cuda(down, "down"), torch.bfloat16)
    if layout == "nxd":
        E, I, H = d.shape
        code = LAYOUT_NXD
    elif layout == "hf":
        E, H, I = d.shape
        code = LAYOUT_HF
    else:
        raise ValueError(f"unknown layout {layout}")
    out = torch.empty(E, H, I, dtype=torch.bfloat16, device=d.device)
    call("nkimoe_pack_down", _p(d), code, _p(out), E, H, I, _s(d))
    return out


_pack_lock = threading.Lock()
_pack_cache: "OrderedDict[tuple, tuple]" = OrderedDict()
_PACK_CACHE_MAX = int(os.environ.get("NKIMOE_PACK_CACHE", "4"))


def _stamp(t: torch.Tensor):
    return (t.data_ptr(), t._version, tuple(t.shape), t.dtype, t.device.index)


def packed_experts(gate_up: torch.Tensor, down: torch.Tensor, layout: str = "nxd") -> PackedExperts:
    """Pack (once) and cache.  An entry is reused only while the very same
    source tensors are alive and unmodified (weak references + pointer,
    version and shape stamps), so freed-and-reused memory never hits a stale
    entry."""
    key = (id(gate_up), id(down), layout)
    with _pack_lock:
        hit = _pack_cache.get(key)
        if hit is not None:
            wg, wd, sg, sd, pe = hit
            if wg() is gate_up and wd() is down and sg == _stamp(gate_up) and sd == _stamp(down):
                _pack_cache.move_to_end(key)
                return pe
            del _pack_cache[key]
    w13 = pack_gate_up(gate_up.detach(), layout)
    w2 = pack_down(down.detach(), layout)
    E, I2, H = w13.shape
    pe = PackedExperts(w13, w2, E, H, I2 // 2)
    with _pack_lock:
        for k in [k for k, v in _pack_cache.items() if v[0]() is None or v[1]() is None]:
            del _pack_cache[k]
        _pack_cache[key] = (weakref.ref(gate_up), weakref.ref(down), _stamp(gate_up), _stamp(down), pe)
        while len(_pack_cache) > _PACK_CACHE_MAX:
            _pack_cache.popitem(last=False)
    return pe


_kmajor_cache: "OrderedDict[int, tuple]" = OrderedDict()


def kmajor_weights(w: torch.Tensor, k_multiple: int = 64, n_multiple: int = 128) -> torch.Tensor:
    """Weights ``w [E, K, N]`` (or ``[K, N]``, taken as one expert) as the
    grouped GEMM's K-major bf16 operand ``[E, N', K']``, K and N zero-padded to
    the given multiples.  The transpose runs in the library (``nkimoe_pack_down``)
    once per weight tensor and is cached while ``w`` lives unmodified (weak
    reference + pointer/version stamp, as :func:`packed_experts`)."""
    key = id(w)
    with _pack_lock:
        hit = _kmajor_cache.get(key)
        if hit is not None and hit[0]() is w and hit[1] == _stamp(w) and hit[2] == (k_multiple, n_multiple):
            _kmajor_cache.move_to_end(key)
            return hit[3]
    src = _contig(_cuda(w, "w").detach(), torch.bfloat16)
    if src.dim() == 2:
        src = src.unsqueeze(0)
    E, K, N = src.shape
    Kp, Np = -(-K // k_multiple) * k_multiple, -(-N // n_multiple) * n_multiple
    if (Kp, Np) != (K, N):
        src = torch.nn.functional.pad(src, (0, Np - N, 0, Kp - K)).contiguous()
    out = torch.empty(E, Np, Kp, dtype=torch.bfloat16, device=src.device)
    # pack_down's plain transpose: [E, I, H] -> [E, H, I] with I = K', H = N'
    call("nkimoe_pack_down", _p(src), LAYOUT_NXD, _p(out), E, Np, Kp, _s(src))
    with _pack_lock:
        for k in [k for k, v in _kmajor_cache.items() if v[0]() is None]:
            del _kmajor_cache[k]
        _kmajor_cache[key] = (weakref.ref(w), _stamp(w), (k_multiple, n_multiple), out)
        while len(_kmajor_cache) > _PACK_CACHE_MAX:
            _kmajor_cache.popitem(last=False)
    return out


# ---------------------------------------------------------------- MoE block
def moe_experts(x: torch.Tensor, experts: PackedExperts, idx: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
    """``out[t] = sum_k w[t,k] * FFN_{idx[t,k]}(x[t])`` (bf16 in/out)."""
    x = _contig(_cuda(x, "x"), torch.bfloat16)
    idx = _contig(_cuda(idx, "idx"))
    if idx.dtype not in (torch.int32, torch.int64):
        idx = idx.to(torch.int64)
    w = _contig(_cuda(weights, "weights"), torch.float32)
    T, H = x.shape
    K = idx.shape[1]
    E, I = experts.num_experts, experts.inter
    if H != experts.hidden or idx.shape[0] != T or w.shape != idx.shape:
        raise ValueError("shape mismatch between hidden states, routing and expert weights")
    out = torch.empty(T, H, dtype=torch.bfloat16, device=x.device)
    nbytes = size_call("nkimoe_moe_workspace_bytes", T, H, I, E, K)
    ws = workspace(x.device, nbytes)
    call("nkimoe_moe_experts", _p(x), _p(experts.w13), _p(experts.w2), _p(idx), _DT[idx.dtype], _p(w), _p(out),
         T, H, I, E, K, _p(ws), ws.numel(), _s(x))
    if sync_check_enabled():
        read_status(ws)
    return out


_router_lock = threading.Lock()
_router_cache: "OrderedDict[int, tuple]" = OrderedDict()


def router_split(router_w: torch.Tensor) -> torch.Tensor:
    """fp32 router weights [E, H] -> bf16 planes [3, E, H] (hi, mid, lo; exact
    sum) for the tensor-core router; cached while the source tensor lives
    unmodified."""
    key = id(router_w)
    with _router_lock:
        hit = _router_cache.get(key)
        if hit is not None and hit[0]() is router_w and hit[1] == _stamp(router_w):
            return hit[2]
    rw = _contig(_cuda(router_w, "router_w").detach(), torch.float32)
    E, H = rw.shape
    out = torch.empty(3, E, H, dtype=torch.bfloat16, device=rw.device)
    call("nkimoe_router_split", _p(rw), _p(out), E, H, _s(rw))
    with _router_lock:
        for k in [k for k, v in _router_cache.items() if v[0]() is None]:
            del _router_cache[k]
        _router_cache[key] = (weakref.ref(router_w), _stamp(router_w), out)
        while len(_router_cache) > _PACK_CACHE_MAX:
            _router_cache.popitem(last=False)
    return out


def moe_block(x: torch.Tensor, router_w: torch.Tensor, experts: PackedExperts, top_k: int,
              bias: torch.Tensor | None = None, return_routing: bool = False, tensor_router: bool = True,
              router_w_split: torch.Tensor | None = None):
    """Router (fp32) + softmax/top-k/renormalise + experts (K2..K7).

    With ``tensor_router`` the fp32 router GEMM of large batches runs on the
    tensor cores over the exact three-plane bf16 split of ``router_w``
    (``router_w_split``, [3, E, H] from :func:`router_split`, when the caller
    keeps it; otherwise taken from a small cache)."""
    x = _contig(_cuda(x, "x"), torch.bfloat16)
    rsplit = None
    if tensor_router and router_w.shape[0] % 128 == 0:
        rsplit = router_w_split if router_w_split is not None else router_split(router_w)
    rw = _contig(_cuda(router_w, "router_w"), torch.float32)
    b = _contig(bias, torch.float32) if bias is not None else None
    T, H = x.shape
    E, I = experts.num_experts, experts.inter
    out = torch.empty(T, H, dtype=torch.bfloat16, device=x.device)
    idx = w = None
    if return_routing:
        idx = torch.empty(T, top_k, dtype=torch.int32, device=x.device)
        w = torch.empty(T, top_k, dtype=torch.float32, device=x.device)
    nbytes = size_call("nkimoe_moe_workspace_bytes", T, H, I, E, top_k)
    ws = workspace(x.device, nbytes)
    call("nkimoe_moe_block", _p(x), _p(rw), _p(b), _p(rsplit), _p(experts.w13), _p(experts.w2), _p(out), _p(idx),
         _p(w), T, H, I, E, top_k, _p(ws), ws.numel(), _s(x))
    if sync_check_enabled():
        read_status(ws)
    return (out, idx, w) if return_routing else out


_host_ws: dict = {}


def _host_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Per-(device, stream) workspace of the host-batch block, kept apart from
    :func:`workspace`: with a completion event, the library's copy back still
    reads a call's staging rows after the stream has moved on, so no device
    entry point may write them meanwhile."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    with _ws_lock:
        buf = _host_ws.get(key)
        if buf is not None and buf.numel() >= nbytes:
            return buf
    # the copy streams may still use the buffer being replaced (its memory
    # goes back to this stream's pool)
    torch.cuda.synchronize(device)
    buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
    with _ws_lock:
        _host_ws[key] = buf
    return buf


def moe_block_host(x: torch.Tensor, router_w: torch.Tensor, experts: PackedExperts, top_k: int,
                   bias: torch.Tensor | None = None, out: torch.Tensor | None = None, chunk_tokens: int = 0,
                   return_routing: bool = False, router_w_split: torch.Tensor | None = None,
                   non_blocking: bool = False, done: torch.cuda.Event | None = None):
    """:func:`moe_block` on a HOST batch ``x [T, H]`` (bf16; page-locked for
    the copies to overlap): the tokens cross to the weights' GPU in chunks
    whose copies overlap the block on the chunk before, and the result comes
    back to ``out`` (a new page-locked host tensor when None).  Equal to
    :func:`moe_block` on the whole batch bit for bit (chunks are cut only where
    each takes the whole batch's router and GEMM paths).  Routing outputs, when
    asked for, stay on the GPU.  The work runs on the current stream of the
    weights' device.

    ``done`` None: the stream completes with the copy back, and the call
    synchronises it unless ``non_blocking``.  ``done`` an event: the copy
    back's completion is recorded on it and the stream goes on without it, so
    the next call's block overlaps this call's copy back (and this call's copy
    in overlaps the previous call's block); ``out`` is ready after
    ``done.synchronize()``.  Until then ``x`` and ``out`` must stay alive and
    untouched."""
    if x.is_cuda:
        raise ValueError("x must be a host tensor (moe_block takes device tensors)")
    dev = _cuda(router_w, "router_w").device
    x = _contig(x, torch.bfloat16)
    T, H = x.shape
    if out is None:
        out = torch.empty(T, H, dtype=torch.bfloat16, pin_memory=True)
    elif out.is_cuda or out.dtype != torch.bfloat16 or tuple(out.shape) != (T, H) or not out.is_contiguous():
        raise ValueError("out must be a contiguous bf16 host tensor shaped like x")
    rsplit = None
    if router_w.shape[0] % 128 == 0:
        rsplit = router_w_split if router_w_split is not None else router_split(router_w)
    rw = _contig(router_w, torch.float32)
    b = _contig(_cuda(bias, "bias"), torch.float32) if bias is not None else None
    E, I = experts.num_experts, experts.inter
    idx = w = None
    if return_routing:
        idx = torch.empty(T, top_k, dtype=torch.int32, device=dev)
        w = torch.empty(T, top_k, dtype=torch.float32, device=dev)
    nbytes = size_call("nkimoe_moe_block_host_workspace_bytes", T, H, I, E, top_k)
    with torch.cuda.device(dev):
        ws = _host_workspace(dev, nbytes)
        ev = None
        if done is not None:
            done.record(torch.cuda.current_stream(dev))  # creates the CUDA event on this device
            ev = ctypes.c_void_p(done.cuda_event)
        call("nkimoe_moe_block_host", _p(x), _p(rw), _p(b), _p(rsplit), _p(experts.w13), _p(experts.w2), _p(out),
             _p(idx), _p(w), T, H, I, E, top_k, int(chunk_tokens), _p(ws), ws.numel(), ev, _s(rw))
        if sync_check_enabled():
            read_status(ws)
            if done is not None:
                done.synchronize()
        elif not non_blocking and done is None:
            torch.cuda.current_stream(dev).synchronize()
    return (out, idx, w) if return_routing else out


def moe_block_rmsnorm(h: torch.Tensor, norm_weight: torch.Tensor, router_w: torch.Tensor, experts: PackedExperts,
                      top_k: int, eps: float = 1e-6, bias: torch.Tensor | None = None, return_x: bool = False,
                      return_routing: bool = False, router_w_split: torch.Tensor | None = None):
    """The block with the RMSNorm in front of it inside the call:
    ``moe_block(rmsnorm(h) * norm_weight)``, equal bit for bit to
    :func:`rmsnorm` + :func:`moe_block`.  For prefill batches (more than 512
    tokens, 128 experts) the norm and the router logits are one tensor-core
    kernel that writes the normalised rows once.  With
    ``return_x`` also returns the normalised rows (bf16)."""
    h = _contig(_cuda(h, "h"), torch.bfloat16)
    rsplit = None
    if router_w.shape[0] % 128 == 0:
        rsplit = router_w_split if router_w_split is not None else router_split(router_w)
    rw = _contig(_cuda(router_w, "router_w"), torch.float32)
    wdt = torch.float32 if norm_weight.dtype == torch.float32 else torch.bfloat16
    nw = _contig(_cuda(norm_weight, "norm_weight"), wdt)
    b = _contig(bias, torch.float32) if bias is not None else None
    T, H = h.shape
    E, I = experts.num_experts, experts.inter
    out = torch.empty(T, H, dtype=torch.bfloat16, device=h.device)
    x = torch.empty_like(h) if return_x else None
    idx = w = None
    if return_routing:
        idx = torch.empty(T, top_k, dtype=torch.int32, device=h.device)
        w = torch.empty(T, top_k, dtype=torch.float32, device=h.device)
    nbytes = size_call("nkimoe_moe_block_rmsnorm_workspace_bytes", T, H, I, E, top_k)
    ws = workspace(h.device, nbytes)
    call("nkimoe_moe_block_rmsnorm", _p(h), _p(nw), _DT[wdt], float(eps), _p(x), _p(rw), _p(b), _p(rsplit),
         _p(experts.w13), _p(experts.w2), _p(out), _p(idx), _p(w), T, H, I, E, top_k, _p(ws), ws.numel(), _s(h))
    if sync_check_enabled():
        read_status(ws)
    res = (out,)
    if return_x:
        res += (x,)
    if return_routing:
        res += (idx, w)
    return res if len(res) > 1 else out


def moe_block_add_rmsnorm(x: torch.Tensor, router_w: torch.Tensor, experts: PackedExperts, top_k: int,
                          residual: torch.Tensor, norm_weight: torch.Tensor, eps: float = 1e-6,
                          residual_out: torch.Tensor | None = None, router_w_split: torch.Tensor | None = None):
    """The MoE block on ``x`` followed by the decoder's residual add and the
    next RMSNorm: returns ``(rmsnorm(r) * norm_weight, r)`` with
    ``r = residual + moe(x)`` (bf16).  ``residual_out`` may be ``residual``
    (in place).  Equal bit for bit to :func:`moe_block` + :func:`add_rmsnorm`;
    up to 512 tokens the block's combine and the norm are one kernel."""
    x = _contig(_cuda(x, "x"), torch.bfloat16)
    residual = _contig(_cuda(residual, "residual"), torch.bfloat16)
    rsplit = None
    if router_w.shape[0] % 128 == 0:
        rsplit = router_w_split if router_w_split is not None else router_split(router_w)
    rw = _contig(_cuda(router_w, "router_w"), torch.float32)
    wdt = torch.float32 if norm_weight.dtype == torch.float32 else torch.bfloat16
    nw = _contig(_cuda(norm_weight, "norm_weight"), wdt)
    T, H = x.shape
    if residual.shape != x.shape:
        raise ValueError(f"residual {tuple(residual.shape)} does not match x {tuple(x.shape)}")
    if residual_out is None:
        residual_out = torch.empty_like(residual)
    out = torch.empty_like(x)
    E, I = experts.num_experts, experts.inter
    nbytes = size_call("nkimoe_moe_workspace_bytes", T, H, I, E, top_k)
    ws = workspace(x.device, nbytes)
    call("nkimoe_moe_block_add_rmsnorm", _p(x), _p(rw), None, _p(rsplit), _p(experts.w13), _p(experts.w2),
         _p(residual), _p(residual_out), _p(nw), _DT[wdt], float(eps), _p(out), None, None, T, H, I, E, top_k,
         _p(ws), ws.numel(), _s(x))
    if sync_check_enabled():
        read_status(ws)
    return out, residual_out


# ---------------------------------------------------------------- pieces
def grouped_gemm(a: torch.Tensor, w_packed: torch.Tensor, offsets: torch.Tensor,
                 out_row_map: torch.Tensor | None = None, out_rows: int | None = None) -> torch.Tensor:
    """``out[r] = a[r] @ w_packed[e]^T`` for rows r of expert segment e."""
    a = _contig(_cuda(a, "a"), torch.bfloat16)
    w = _contig(_cuda(w_packed, "w_packed"), torch.bfloat16)
    off = _contig(_cuda(offsets, "offsets"), torch.int32)
    M, Kd = a.shape
    E, N, Kw = w.shape
    if Kw != Kd:
        raise ValueError("inner dimensions differ")
    rows = M if out_rows is None else out_rows
    out = torch.empty(rows, N, dtype=torch.bfloat16, device=a.device)
    rm = _contig(out_row_map, torch.int32) if out_row_map is not None else None
    st = workspace(a.device, 256)
    call("nkimoe_grouped_gemm", _p(a), _p(w), _p(off), _p(rm), _p(out), M, N, Kd, E, _p(st), _s(a))
    return out


def swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    g = _contig(_cuda(gate_up, "gate_up"), torch.bfloat16)
    M, N2 = g.shape
    out = torch.empty(M, N2 // 2, dtype=torch.bfloat16, device=g.device)
    call("nkimoe_swiglu", _p(g), _p(out), M, N2 // 2, _s(g))
    return out


def aggregate(expert_outputs: torch.Tensor) -> torch.Tensor:
    eo = _contig(_cuda(expert_outputs, "expert_outputs"), torch.bfloat16)
    K, T, H = eo.shape
    out = torch.empty(T, H, dtype=torch.bfloat16, device=eo.device)
    call("nkimoe_aggregate", _p(eo), _p(out), K, T, H, _s(eo))
    return out


# ---------------------------------------------------------------- expert-parallel pieces
def route(x: torch.Tensor, router_w: torch.Tensor, top_k: int, bias: torch.Tensor | None = None,
          tensor_router: bool = True):
    """Router + softmax/top-k/renormalise: ``(idx int32 [T,K], w fp32 [T,K])``."""
    x = _contig(_cuda(x, "x"), torch.bfloat16)
    rsplit = router_split(router_w) if tensor_router and router_w.shape[0] % 128 == 0 else None
    rw = _contig(_cuda(router_w, "router_w"), torch.float32)
    b = _contig(bias, torch.float32) if bias is not None else None
    T, H = x.shape
    E = rw.shape[0]
    idx = torch.empty(T, top_k, dtype=torch.int32, device=x.device)
    w = torch.empty(T, top_k, dtype=torch.float32, device=x.device)
    ws = workspace(x.device, size_call("nkimoe_route_workspace_bytes", T, H, E, top_k))
    call("nkimoe_route", _p(x), _p(rw), _p(b), _p(rsplit), _p(idx), _p(w), T, H, E, top_k, _p(ws), ws.numel(), _s(x))
    return idx, w


def dispatch(x: torch.Tensor, idx: torch.Tensor, weights: torch.Tensor, num_experts: int):
    """Group the (token, slot) rows by global expert: returns ``(x_perm [T*K, H],
    row_weight [T*K], slot_row [T*K], expert_counts [E])``."""
    x = _contig(_cuda(x, "x"), torch.bfloat16)
    idx = _contig(_cuda(idx, "idx"))
    if idx.dtype not in (torch.int32, torch.int64):
        idx = idx.to(torch.int64)
    w = _contig(_cuda(weights, "weights"), torch.float32)
    T, H = x.shape
    K = idx.shape[1]
    dev = x.device
    x_perm = torch.empty(T * K, H, dtype=torch.bfloat16, device=dev)
    row_weight = torch.empty(T * K, dtype=torch.float32, device=dev)
    slot_row = torch.empty(T * K, dtype=torch.int32, device=dev)
    counts = torch.empty(num_experts, dtype=torch.int32, device=dev)
    ws = workspace(dev, size_call("nkimoe_dispatch_workspace_bytes", T, K, num_experts))
    call("nkimoe_dispatch", _p(x), _p(idx), _DT[idx.dtype], _p(w), T, H, num_experts, K, _p(x_perm), _p(row_weight),
         _p(slot_row), _p(counts), _p(ws), ws.numel(), _s(x))
    if sync_check_enabled():
        read_status(ws)
    return x_perm, row_weight, slot_row, counts


def segment_experts(a: torch.Tensor, row_weight: torch.Tensor, segment_counts: torch.Tensor,
                    experts: PackedExperts) -> torch.Tensor:
    """``y[r] = row_weight[r] * FFN_{s % E_local}(a[r])`` for rows r of segment s."""
    a = _contig(_cuda(a, "a"), torch.bfloat16)
    rw = _contig(_cuda(row_weight, "row_weight"), torch.float32)
    sc = _contig(_cuda(segment_counts, "segment_counts").reshape(-1), torch.int32)
    R, H = a.shape
    S = sc.numel()
    y = torch.empty(R, H, dtype=torch.bfloat16, device=a.device)
    ws = workspace(a.device, size_call("nkimoe_segment_experts_workspace_bytes", R, experts.inter, S))
    call("nkimoe_segment_experts", _p(a), _p(rw), _p(sc), S, experts.num_experts, _p(experts.w13), _p(experts.w2),
         _p(y), R, H, experts.inter, _p(ws), ws.numel(), _s(a))
    if sync_check_enabled():
        read_status(ws)
    return y


def combine(y: torch.Tensor, slot_row: torch.Tensor, tokens: int, top_k: int,
            slot_weight: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = sum_k (w[t,k]) * y[slot_row[t*K+k]]`` (fp32 sum, k ascending)."""
    y = _contig(_cuda(y, "y"), torch.bfloat16)
    sr = _contig(_cuda(slot_row, "slot_row"), torch.int32)
    sw = _contig(slot_weight, torch.float32) if slot_weight is not None else None
    H = y.shape[1]
    out = torch.empty(tokens, H, dtype=torch.bfloat16, device=y.device)
    call("nkimoe_combine", _p(y), _p(sr), _p(sw), _p(out), tokens, top_k, H, _s(y))
    return out


def ep_dispatch(x: torch.Tensor, idx: torch.Tensor, weights: torch.Tensor, num_ranks: int, experts_per_rank: int):
    """De-duplicated expert-parallel dispatch: one send row per (token, rank).

    Returns ``(x_send [R, H], slots [R, K] int32, wts [R, K] fp32, rank_counts [P]
    int32, slot_row [T, P] int32)``; the buffers hold ``T*min(P, K)`` rows, of
    which ``rank_counts.sum()`` are valid.
    """
    x = _contig(_cuda(x, "x"), torch.bfloat16)
    idx = _contig(_cuda(idx, "idx"), torch.int32)
    w = _contig(_cuda(weights, "weights"), torch.float32)
    T, H = x.shape
    K = idx.shape[1]
    P = num_ranks
    dev = x.device
    cap = T * min(P, K)
    x_send = torch.empty(cap, H, dtype=torch.bfloat16, device=dev)
    slots = torch.empty(cap, K, dtype=torch.int32, device=dev)
    wts = torch.empty(cap, K, dtype=torch.float32, device=dev)
    counts = torch.empty(P, dtype=torch.int32, device=dev)
    slot_row = torch.empty(T, P, dtype=torch.int32, device=dev)
    ws = workspace(dev, size_call("nkimoe_ep_dispatch_workspace_bytes", T, P))
    call("nkimoe_ep_dispatch", _p(x), _p(idx), _p(w), T, H, K, P, experts_per_rank, _p(x_send), _p(slots), _p(wts),
         _p(counts), _p(slot_row), _p(ws), ws.numel(), _s(x))
    if sync_check_enabled():
        read_status(ws)
    return x_send, slots, wts, counts, slot_row
