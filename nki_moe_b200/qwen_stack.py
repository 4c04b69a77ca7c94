"""Qwen3-MoE decoder stack on this library's kernels, for end-to-end latency.

The decoder wiring of the reference's model file (``qwen_with_nki.py:402-460``,
``NeuronQwen3MoeDecoderLayer.forward``): per layer

    r = h;  h = attn(rmsnorm(h));  h = r + h
    r = h;  h = moe(rmsnorm(h));   h = r + h

with the attention of ``qwen_with_nki.py:330-350`` (fused QKV projection,
per-head q/k RMSNorm, rotate-half RoPE with theta 1e6, GQA, scale
head_dim^-0.5) and a final RMSNorm + LM head (``qwen_with_nki.py:495``).

Library kernels on the path: RMSNorm and the fused residual-add + RMSNorm
(``nkimoe_rmsnorm`` / ``nkimoe_add_rmsnorm``), q/k RMSNorm + RoPE on the fused
QKV rows (``nkimoe_qk_norm_rope``, prefill), the decode step's attention fused
with its q/k norms, RoPE and KV-cache store (``nkimoe_decode_attention``) and
the whole MoE block (``nkimoe_moe_block``).  The dense projections (QKV, O,
LM head) are plain cuBLAS GEMMs through torch and prefill attention is torch's
scaled-dot-product attention; neither is part of the MoE hot path.

Serving from a paged cache (:mod:`nki_moe_b200.paged`; sequences of their own
lengths, shared prompts, windows): :meth:`Qwen3MoEStack.prefill_paged`,
:meth:`~Qwen3MoEStack.decode_paged`, :meth:`~Qwen3MoEStack.generate_paged` and
:meth:`~Qwen3MoEStack.score` run the library's own attention for prompts too
(``nkimoe_qk_norm_rope_store``, ``nkimoe_paged_prefill_attention``,
``nkimoe_paged_decode_attention``, ``nkimoe_token_logprobs``), draw from
restricted distributions (``nkimoe_sample_tokens``), and check trees of drafted
tokens in one step (:meth:`~Qwen3MoEStack.draft_paged`,
:meth:`~Qwen3MoEStack.accept_paged`: ``nkimoe_paged_tree_attention``,
``nkimoe_accept_drafts``).

Decode keeps every shape static (a KV cache of ``max_seq`` positions, the
current position in a device tensor that the attention kernel reads), so one
decode step over all layers is captured into a single CUDA graph.
"""

from __future__ import annotations

import contextlib
import math
import time
import weakref
from collections import OrderedDict
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import ops
from .drafts import LookupDrafts
from .paged import CacheFull, PagedKVCache


@contextlib.contextmanager
def _appending(cache: PagedKVCache, seqs, counts):
    """Extends the sequences; where what follows fails, they get their lengths back."""
    seqs = list(seqs)
    lengths = [cache.length(q) for q in seqs]
    cache.extend(seqs, counts)
    try:
        yield
    except BaseException:
        cache.take_back(seqs, lengths)
        raise


def _token_ids(t: torch.Tensor, vocab: int) -> torch.Tensor:
    """``t`` as a vector, checked: its type, and on the host its range (on the
    device that would wait for it)."""
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise ValueError(f"token ids must be whole numbers, not {t.dtype}")
    t = t.reshape(-1)
    if not t.is_cuda and t.numel() and not (0 <= int(t.min()) and int(t.max()) < vocab):
        raise ValueError(f"token ids must be in [0, {vocab})")
    return t


@dataclass
class DraftStep:
    """A step with drafted tokens that waits for :meth:`Qwen3MoEStack.accept_paged`."""

    cache: PagedKVCache
    seqs: list
    marks: list  # of the sequences with its nodes
    lengths: list  # of the sequences before it
    nodes: list  # of each tree
    tokens: torch.Tensor  # packed, as ops.accept_drafts takes them
    parents: torch.Tensor
    cu_seqlens: torch.Tensor
    kv_lens: torch.Tensor
    ended: bool = False


@dataclass
class Qwen3MoEConfig:
    """Qwen3-30B-A3B shape (the defaults) or any smaller one of the same kind."""

    vocab_size: int = 151936
    hidden_size: int = 2048
    num_hidden_layers: int = 48
    num_attention_heads: int = 32
    num_key_value_heads: int = 4
    head_dim: int = 128
    moe_intermediate_size: int = 768
    num_experts: int = 128
    num_experts_per_tok: int = 8
    rope_theta: float = 1e6
    rms_norm_eps: float = 1e-6

    @classmethod
    def from_hf(cls, c) -> "Qwen3MoEConfig":
        theta = getattr(c, "rope_theta", None)
        if theta is None:
            theta = (getattr(c, "rope_parameters", None) or {}).get("rope_theta", 1e6)
        return cls(vocab_size=c.vocab_size, hidden_size=c.hidden_size, num_hidden_layers=c.num_hidden_layers,
                   num_attention_heads=c.num_attention_heads, num_key_value_heads=c.num_key_value_heads,
                   head_dim=getattr(c, "head_dim", c.hidden_size // c.num_attention_heads),
                   moe_intermediate_size=c.moe_intermediate_size, num_experts=c.num_experts,
                   num_experts_per_tok=c.num_experts_per_tok, rope_theta=float(theta), rms_norm_eps=c.rms_norm_eps)


class _Layer:
    """One decoder layer's weights in the layouts the kernels take.  With
    ``ep`` (an expert-parallel block holding this rank's experts) the MoE runs
    through it; otherwise ``experts`` holds all experts."""

    def __init__(self, in_norm, qkv_w, q_norm, k_norm, o_w, post_norm, router_w, experts: ops.PackedExperts,
                 ep=None, ep_decode=None):
        self.in_norm, self.qkv_w, self.q_norm, self.k_norm = in_norm, qkv_w, q_norm, k_norm
        self.o_w, self.post_norm, self.router_w, self.experts = o_w, post_norm, router_w, experts
        # expert parallel: one exchange sized for prefill batches, one for a
        # decode step (the receiver's kernels cover every source's whole region)
        self.ep, self.ep_decode = ep, ep_decode
        self.router_split = (ops.router_split(router_w) if ep is None and router_w.shape[0] % 128 == 0 else None)


class Qwen3MoEStack:
    """bf16 Qwen3-MoE causal LM: prefill, static-shape decode, greedy generate."""

    PAGED_STEPS = 32  # captured paged steps (batch sizes) that are kept of each cache

    def __init__(self, cfg: Qwen3MoEConfig, embed: torch.Tensor, layers: list[_Layer], final_norm: torch.Tensor,
                 lm_head: torch.Tensor, max_batch: int, max_seq: int):
        self.cfg = cfg
        self.embed, self.layers, self.final_norm, self.lm_head = embed, layers, final_norm, lm_head
        self.device = embed.device
        self.max_batch, self.max_seq = max_batch, max_seq
        kv = (cfg.num_hidden_layers, max_batch, cfg.num_key_value_heads, max_seq, cfg.head_dim)
        self.k_cache = torch.zeros(kv, dtype=torch.bfloat16, device=self.device)
        self.v_cache = torch.zeros(kv, dtype=torch.bfloat16, device=self.device)
        self.length = 0
        # decode-step state (static for graph capture)
        self._pos = torch.zeros(1, dtype=torch.int64, device=self.device)
        self._tokens = torch.zeros(max_batch, dtype=torch.int64, device=self.device)
        self._graph = None
        self._graph_batch = None
        self._graph_out = None
        # the captured paged decode steps: of each cache in use, its buffers and graph by batch size, the
        # last used last (a cache that is gone takes its steps along); and which was used last
        self._paged_steps: weakref.WeakKeyDictionary[PagedKVCache, OrderedDict] = weakref.WeakKeyDictionary()
        self._paged_last = None
        # the steps share their capture stream's workspaces, so one begins when the one before has ended
        self._paged_stream = self._paged_done = self._paged_status = None
        # the skinny linear kernel takes N % 16 == 0 and K % 32 == 0
        H, hd = cfg.hidden_size, cfg.head_dim
        nq, nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        self._skinny_ok = (H % 32 == 0 and (nq * hd) % 32 == 0 and ((nq + 2 * nkv) * hd) % 16 == 0
                           and H % 16 == 0 and cfg.vocab_size % 16 == 0)

    # ------------------------------------------------------------ construction
    @classmethod
    def random_init(cls, cfg: Qwen3MoEConfig, seed: int = 0, device="cuda", max_batch: int = 8,
                    max_seq: int = 640, std: float = 0.02, expert_parallel: bool = False,
                    group=None) -> "Qwen3MoEStack":
        """Random N(0, std) weights (norm weights 1, router fp32), expert weights
        drawn in the reference's ``[E, H, 2I]`` / ``[E, I, H]`` layout and
        packed once.

        ``expert_parallel``: one rank of an expert-parallel stack over the
        initialised process group (``group``, default WORLD): every rank draws
        the same weights (same generator sequence as the single-GPU stack),
        keeps the attention, norms, router and embeddings whole and only its
        ``E / P`` experts, and runs each layer's MoE as a peer-memory
        expert-parallel block over its own sequences (``max_batch`` of them,
        up to ``max_seq`` tokens each).  Every rank must run the same calls
        (prefill, decode steps) in the same order; the batches of the paged
        calls may differ."""
        dev = torch.device(device)
        g = torch.Generator(device=dev).manual_seed(seed)
        H, hd = cfg.hidden_size, cfg.head_dim
        nq, nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        E, I = cfg.num_experts, cfg.moe_intermediate_size
        P, r = 1, 0
        if expert_parallel:
            import torch.distributed as dist

            from .ep_peer import PeerExpertParallelMoE
            P, r = dist.get_world_size(group), dist.get_rank(group)
            if E % P:
                raise ValueError(f"{E} experts do not split over {P} ranks")
        El = E // P

        def rnd(*shape, dtype=torch.bfloat16):
            return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * std).to(dtype)

        ones = lambda n: torch.ones(n, dtype=torch.bfloat16, device=dev)  # noqa: E731
        layers = []
        for _ in range(cfg.num_hidden_layers):
            gate_up = rnd(E, H, 2 * I)
            w13 = ops.pack_gate_up(gate_up[r * El:(r + 1) * El].contiguous(), "nxd")
            del gate_up
            down = rnd(E, I, H)
            w2 = ops.pack_down(down[r * El:(r + 1) * El].contiguous(), "nxd")
            del down
            experts = ops.PackedExperts(w13, w2, El, H, I)
            attn = (ones(H), rnd((nq + 2 * nkv) * hd, H), ones(hd), ones(hd), rnd(H, nq * hd), ones(H))
            router_w = rnd(E, H, dtype=torch.float32)
            ep = ep_decode = None
            if expert_parallel:
                ep = PeerExpertParallelMoE(router_w, None, None, E, cfg.num_experts_per_tok, max_batch * max_seq,
                                           group=group, device_epochs=True, packed=experts)
                ep_decode = PeerExpertParallelMoE(router_w, None, None, E, cfg.num_experts_per_tok, max_batch,
                                                  group=group, device_epochs=True, packed=experts)
            layers.append(_Layer(*attn, router_w, experts, ep=ep, ep_decode=ep_decode))
        return cls(cfg, rnd(cfg.vocab_size, H), layers, ones(H), rnd(cfg.vocab_size, H), max_batch, max_seq)

    def close(self):
        """Release the expert-parallel exchange buffers (every rank together)."""
        self.release_graph()
        for lyr in self.layers:
            for blk in (lyr.ep, lyr.ep_decode):
                if blk is not None:
                    blk.close()

    @classmethod
    def from_hf(cls, model, device="cuda", max_batch: int = 8, max_seq: int = 640) -> "Qwen3MoEStack":
        """Copy the weights of an HF ``Qwen3MoeForCausalLM`` (bf16 on the GPU,
        router fp32), expert weights from the HF ``[E, 2I, H]`` / ``[E, H, I]``
        layout."""
        cfg = Qwen3MoEConfig.from_hf(model.config)
        dev = torch.device(device)
        bf = lambda t: t.detach().to(dev, torch.bfloat16).contiguous()  # noqa: E731
        layers = []
        for lyr in model.model.layers:
            a, m = lyr.self_attn, lyr.mlp
            qkv = torch.cat([a.q_proj.weight, a.k_proj.weight, a.v_proj.weight], 0)
            w13 = ops.pack_gate_up(bf(m.experts.gate_up_proj), "hf")
            w2 = ops.pack_down(bf(m.experts.down_proj), "hf")
            layers.append(_Layer(bf(lyr.input_layernorm.weight), bf(qkv), bf(a.q_norm.weight), bf(a.k_norm.weight),
                                 bf(a.o_proj.weight), bf(lyr.post_attention_layernorm.weight),
                                 m.gate.weight.detach().to(dev, torch.float32).contiguous(),
                                 ops.PackedExperts(w13, w2, cfg.num_experts, cfg.hidden_size,
                                                   cfg.moe_intermediate_size)))
        return cls(cfg, bf(model.model.embed_tokens.weight), layers, bf(model.model.norm.weight),
                   bf(model.lm_head.weight), max_batch, max_seq)

    @classmethod
    def from_safetensors(cls, path: str, device="cuda", max_batch: int = 8,
                         max_seq: int = 640) -> "Qwen3MoEStack":
        """Load an HF Qwen3-MoE checkpoint directory (hub format, bf16 or FP8
        with block scales) tensor by tensor: each layer's experts are read in
        the HF fused layout and packed on the device (``hf_loader``)."""
        from .hf_loader import Qwen3MoECheckpoint

        ck = Qwen3MoECheckpoint(path, device=device)
        cfg = Qwen3MoEConfig.from_hf(ck.hf_config)
        pre = ck.reader.prefix
        layers = []
        for l in range(cfg.num_hidden_layers):  # noqa: E741
            t = lambda rest, dtype=None: ck.layer_tensor(l, rest, dtype)  # noqa: E731
            qkv = torch.cat([t("self_attn.q_proj.weight"), t("self_attn.k_proj.weight"),
                             t("self_attn.v_proj.weight")], 0).contiguous()
            gate_up, down = ck.experts(l)
            I = gate_up.shape[1] // 2
            experts = ops.PackedExperts(ops.pack_gate_up(gate_up, "hf"), ops.pack_down(down, "hf"),
                                        cfg.num_experts, cfg.hidden_size, I)
            del gate_up, down
            layers.append(_Layer(t("input_layernorm.weight"), qkv, t("self_attn.q_norm.weight"),
                                 t("self_attn.k_norm.weight"), t("self_attn.o_proj.weight"),
                                 t("post_attention_layernorm.weight"),
                                 t("mlp.gate.weight", torch.float32).contiguous(), experts))
        lm = "lm_head.weight"
        lm_head = ck.tensor(lm) if ck.reader.has(lm) else ck.tensor(f"{pre}embed_tokens.weight")
        return cls(cfg, ck.tensor(f"{pre}embed_tokens.weight"), layers, ck.tensor(f"{pre}norm.weight"), lm_head,
                   max_batch, max_seq)

    # ------------------------------------------------------------ layers
    def _moe_add_norm(self, lyr: _Layer, x: torch.Tensor, res: torch.Tensor, norm_w: torch.Tensor,
                      decode: bool):
        """The layer's MoE block on ``x``, then the residual add and the next
        RMSNorm (the next layer's input norm, or the final norm): returns
        ``(normed, residual)``."""
        eps = self.cfg.rms_norm_eps
        if lyr.ep is not None:
            h = lyr.ep_decode(x) if decode else lyr.ep(x)
            return ops.add_rmsnorm(h, res, norm_w, eps)
        return ops.moe_block_add_rmsnorm(x, lyr.router_w, lyr.experts, self.cfg.num_experts_per_tok, res, norm_w,
                                         eps, router_w_split=lyr.router_split)

    def _qkv(self, lyr: _Layer, xn: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        c = self.cfg
        qkv = F.linear(xn, lyr.qkv_w)
        return ops.qk_norm_rope(qkv, lyr.q_norm, lyr.k_norm, positions, c.num_attention_heads,
                                c.num_key_value_heads, c.head_dim, c.rope_theta, c.rms_norm_eps, out=qkv)

    def _split(self, qkv: torch.Tensor, B: int, S: int):
        c = self.cfg
        nq, nkv, hd = c.num_attention_heads, c.num_key_value_heads, c.head_dim
        q = qkv[:, : nq * hd].view(B, S, nq, hd).transpose(1, 2)
        k = qkv[:, nq * hd:(nq + nkv) * hd].view(B, S, nkv, hd).transpose(1, 2)
        v = qkv[:, (nq + nkv) * hd:].view(B, S, nkv, hd).transpose(1, 2)
        return q, k, v

    def _layers(self, h: torch.Tensor, attention, linear=F.linear, decode: bool = False):
        """Run every layer on h [T, H]; ``attention(li, lyr, xn)`` returns the
        attention output [T, nq*hd] before the O projection (``linear``).
        Returns the final norm of the residual stream."""
        eps = self.cfg.rms_norm_eps
        res = h
        xn = ops.rmsnorm(h, self.layers[0].in_norm, eps)
        for li, lyr in enumerate(self.layers):
            a = linear(attention(li, lyr, xn), lyr.o_w)
            xn, res = ops.add_rmsnorm(a, res, lyr.post_norm, eps)
            # the MoE output joins the residual and feeds the next norm
            nxt = self.layers[li + 1].in_norm if li + 1 < len(self.layers) else self.final_norm
            xn, res = self._moe_add_norm(lyr, xn, res, nxt, decode)
        return xn

    # ------------------------------------------------------------ prefill
    @torch.inference_mode()
    def prefill(self, input_ids: torch.Tensor, all_logits: bool = False) -> torch.Tensor:
        """Causal forward over ``input_ids [B, S]`` from position 0; fills the KV
        cache.  Returns the last position's logits ``[B, V]`` (or all
        positions' ``[B, S, V]`` with ``all_logits``)."""
        B, S = input_ids.shape
        if B > self.max_batch or S > self.max_seq:
            raise ValueError(f"batch {B} x {S} exceeds the cache ({self.max_batch} x {self.max_seq})")
        ids = input_ids.to(self.device)
        h = F.embedding(ids.reshape(-1), self.embed)
        positions = torch.arange(S, device=self.device, dtype=torch.int64).repeat(B)
        c = self.cfg

        def attention(li, lyr, xn):
            q, k, v = self._split(self._qkv(lyr, xn, positions), B, S)
            self.k_cache[li, :B, :, :S].copy_(k)
            self.v_cache[li, :B, :, :S].copy_(v)
            o = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)  # [B, nq, S, hd]
            return o.transpose(1, 2).reshape(B * S, c.num_attention_heads * c.head_dim)

        hn = self._layers(h, attention)
        self.length = S
        if all_logits:
            return F.linear(hn, self.lm_head).view(B, S, -1)
        last = hn.view(B, S, -1)[:, -1]
        return F.linear(last, self.lm_head)

    # ------------------------------------------------------------ decode
    def _decode_body(self, B: int) -> torch.Tensor:
        """One decode step for ``self._tokens[:B]`` at position ``self._pos``:
        per layer the QKV projection, then one library kernel for the q/k
        norms + RoPE, the KV-cache store and the attention over the cache
        (``ops.decode_attention``)."""
        c = self.cfg
        h = F.embedding(self._tokens[:B], self.embed)
        # the projections of a decode batch (<= 16 rows) stream their weights
        # through the library's skinny linear kernel
        linear = ops.skinny_linear if B <= 16 and self._skinny_ok else F.linear

        def attention(li, lyr, xn):
            qkv = linear(xn, lyr.qkv_w)
            return ops.decode_attention(qkv, lyr.q_norm, lyr.k_norm, self._pos, self.k_cache[li], self.v_cache[li],
                                        c.num_attention_heads, c.num_key_value_heads, c.rope_theta, c.rms_norm_eps)

        hn = self._layers(h, attention, linear, decode=True)
        return linear(hn, self.lm_head)

    @torch.inference_mode()
    def decode(self, tokens: torch.Tensor, graph: bool = True) -> torch.Tensor:
        """One decode step: ``tokens [B]`` at position ``self.length``; returns
        logits ``[B, V]`` (a tensor of its own) and advances the position."""
        out = self._step(tokens, graph)
        return out.clone() if graph else out

    def _step(self, tokens: torch.Tensor, graph: bool) -> torch.Tensor:
        """Decode step returning, with ``graph``, the captured graph's output
        buffer itself (overwritten by the next step)."""
        B = tokens.shape[0]
        if self.length >= self.max_seq:
            raise ValueError("KV cache full")
        self._tokens[:B].copy_(tokens.to(self.device).reshape(-1))
        self._pos.fill_(self.length)
        if graph:
            if self._graph is None or self._graph_batch != B:
                self._capture(B)
            self._graph.replay()
            out = self._graph_out
        else:
            out = self._decode_body(B)
        self.length += 1
        return out

    def _capture(self, B: int):
        s = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        # warm up on the capture stream (workspaces sized outside the capture);
        # the cache slot written here is rewritten by every replay
        with torch.cuda.stream(s):
            self._decode_body(B)
        torch.cuda.current_stream(self.device).wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = self._decode_body(B)
        self._graph, self._graph_batch, self._graph_out = g, B, out

    def release_graph(self):
        self._graph = self._graph_out = None
        for cache in list(self._paged_steps):
            self._drop_steps(cache)

    def _drop_steps(self, cache: PagedKVCache):
        """Ends the captured steps of a cache."""
        self._paged_steps.pop(cache, None)

    @property
    def _paged(self):
        """The captured paged step that was used last and its cache, or None."""
        if self._paged_last is None:
            return None
        cache, B = self._paged_last[0](), self._paged_last[1]
        step = None if cache is None else self._paged_steps.get(cache, {}).get(B)
        return None if step is None else {"cache": cache, "B": B, **step}

    # ------------------------------------------------------------ paged cache
    def paged_cache(self, num_pages: int, page_size: int = 64, max_seq: int | None = None, window: int = 0,
                    sinks: int = 0) -> PagedKVCache:
        """A paged cache of this stack's layers (``max_seq``: the longest
        sequence, the stack's by default)."""
        c = self.cfg
        return PagedKVCache(c.num_hidden_layers, c.num_key_value_heads, num_pages, page_size, max_seq or self.max_seq,
                            window, sinks, self.device)

    def _prompt_hidden(self, cache: PagedKVCache, seqs, prompts) -> torch.Tensor:
        """Runs the layers on new tokens of the sequences, which the cache has
        been extended by, packed, and returns the final norm's rows ``[T, H]``."""
        c = self.cfg
        cu = torch.zeros(len(seqs) + 1, dtype=torch.int32)
        cu[1:] = torch.tensor([p.numel() for p in prompts]).cumsum(0)
        cu = cu.to(self.device)
        kv = torch.tensor([cache.length(q) for q in seqs], dtype=torch.int32).to(self.device)
        table = cache.table(seqs).to(self.device)
        ids = torch.cat([p.reshape(-1).to(self.device, torch.int64) for p in prompts])
        h = F.embedding(ids, self.embed)

        def attention(li, lyr, xn):
            k, v = cache.layer(li)
            q = ops.qk_norm_rope_store(F.linear(xn, lyr.qkv_w), lyr.q_norm, lyr.k_norm, cu, kv, k, v, table,
                                       c.num_attention_heads, c.num_key_value_heads, c.rope_theta, c.rms_norm_eps)
            return ops.paged_prefill_attention(q, k, v, table, cu, kv, window=cache.window, sinks=cache.sinks)

        return self._layers(h, attention)

    def _prompt_lengths(self, seqs, prompts) -> list[int]:
        """The prompts' lengths, checked."""
        lens = [int(_token_ids(p, self.cfg.vocab_size).numel()) for p in prompts]
        if len(prompts) != len(seqs) or not seqs or min(lens) == 0:
            raise ValueError("one prompt, not empty, for each sequence")
        if any(lyr.ep is not None for lyr in self.layers) and sum(lens) > self.max_batch * self.max_seq:
            raise ValueError(f"{sum(lens)} tokens exceed the expert-parallel exchange "
                             f"({self.max_batch} x {self.max_seq})")
        return lens

    @torch.inference_mode()
    def prefill_paged(self, cache: PagedKVCache, seqs, prompts) -> torch.Tensor:
        """Appends ``prompts[i]`` (token ids, any lengths) to sequence
        ``seqs[i]`` of the cache, which may hold the beginning already (a
        prompt in chunks, or one that continues a fork).  Returns the logits
        of each prompt's last token ``[len(seqs), V]``.  Where the call fails,
        the sequences keep their lengths."""
        lens = self._prompt_lengths(seqs, prompts)
        with _appending(cache, seqs, lens):
            hn = self._prompt_hidden(cache, seqs, prompts)
            last = torch.tensor(lens).cumsum(0) - 1
            logits = F.linear(hn[last.to(self.device)], self.lm_head)
        for q in seqs:
            cache.trim(q)
        return logits

    def _paged_body(self, cache: PagedKVCache, tokens, positions, table) -> torch.Tensor:
        c = self.cfg
        B = tokens.shape[0]
        linear = ops.skinny_linear if B <= 16 and self._skinny_ok else F.linear

        def attention(li, lyr, xn):
            k, v = cache.layer(li)
            return ops.paged_decode_attention(linear(xn, lyr.qkv_w), lyr.q_norm, lyr.k_norm, positions, k, v, table,
                                              c.num_attention_heads, c.num_key_value_heads, c.rope_theta,
                                              c.rms_norm_eps, window=cache.window, sinks=cache.sinks)

        hn = self._layers(F.embedding(tokens, self.embed), attention, linear, decode=True)
        return linear(hn, self.lm_head)

    @torch.inference_mode()
    def decode_paged(self, cache: PagedKVCache, seqs, tokens: torch.Tensor, graph: bool = True) -> torch.Tensor:
        """One decode step: ``tokens[i]`` appended to sequence ``seqs[i]``.
        Returns logits ``[len(seqs), V]`` (a tensor of its own).  With
        ``graph`` the step is captured once per cache and batch size (the
        ``PAGED_STEPS`` sizes used last are kept); lengths and pages are device
        data.  The call that captures runs the step
        itself and the capture runs nothing, so that every call runs each
        layer's expert-parallel exchange once, whatever a rank's batch does.
        Where the call fails, the sequences keep their lengths."""
        B = len(seqs)
        if tokens.numel() != B:
            raise ValueError(f"{tokens.numel()} tokens for {B} sequences")
        if any(lyr.ep is not None for lyr in self.layers) and B > self.max_batch:
            raise ValueError(f"batch {B} exceeds the expert-parallel exchange ({self.max_batch})")
        tokens = _token_ids(tokens, self.cfg.vocab_size)
        with _appending(cache, seqs, [1] * B):
            positions = torch.tensor([cache.length(q) - 1 for q in seqs], dtype=torch.int64)
            table = cache.table(seqs)
            if graph:
                out = self._paged_step(cache, tokens, positions, table)
            else:
                out = self._paged_body(cache, tokens.to(self.device, torch.int64), positions.to(self.device),
                                       table.to(self.device))
        for q in seqs:
            cache.trim(q)
        return out

    def _paged_step(self, cache: PagedKVCache, tokens, positions, table) -> torch.Tensor:
        """The step's replay, or the step itself and its capture."""
        B = tokens.numel()
        here = torch.cuda.current_stream(self.device)
        if self._paged_done is None:
            self._paged_stream, self._paged_done = torch.cuda.Stream(device=self.device), torch.cuda.Event()
            self._paged_status = ops._status_sink(self.device)
        here.wait_event(self._paged_done)
        steps = self._paged_steps.setdefault(cache, OrderedDict())
        step = steps.get(B)
        if step is None:
            step = {"tokens": torch.zeros(B, dtype=torch.int64, device=self.device),
                    "positions": torch.zeros(B, dtype=torch.int64, device=self.device),
                    "table": torch.zeros(B, cache.max_pages, dtype=torch.int32, device=self.device)}
        step["tokens"].copy_(tokens)
        step["positions"].copy_(positions)
        step["table"].copy_(table)
        if "graph" in step:
            step["graph"].replay()
            out = step["out"].clone()
            steps.move_to_end(B)
        else:
            s = self._paged_stream
            s.wait_stream(here)
            # this call's step, on the capture stream (workspaces are sized outside the capture)
            try:
                with torch.cuda.stream(s):
                    out = self._paged_body(cache, step["tokens"], step["positions"], step["table"])
            finally:
                here.wait_stream(s)
            out = out.clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step["out"] = self._paged_body(cache, step["tokens"], step["positions"], step["table"])
                step["workspaces"] = ops._end_of_capture(self._paged_status)
            step["graph"] = g
            steps[B] = step
            if len(steps) > self.PAGED_STEPS:
                steps.popitem(last=False)
        self._paged_done.record(here)
        self._paged_last = (weakref.ref(cache), B)
        return out

    # ------------------------------------------------------------ drafted tokens
    @torch.inference_mode()
    def draft_paged(self, cache: PagedKVCache, seqs, tokens, parents=None) -> tuple[torch.Tensor, DraftStep]:
        """One step for a tree of tokens per sequence: ``tokens[i]`` (at most 64
        token ids, the first being what comes next in sequence ``seqs[i]``, the
        others drafts of what may follow) and ``parents[i]`` (for each the index
        of its parent, below its own, -1 for the first; None: each follows the one
        before).  Returns the logits after every node ``[sum of nodes, V]``, packed,
        and the step, which :meth:`accept_paged` ends: until then the sequences
        hold all nodes and are not forked.  Where the call fails, they keep their
        lengths."""
        if any(lyr.ep is not None for lyr in self.layers):
            raise ValueError("drafted tokens are for stacks on one GPU: ranks would take different numbers of steps")
        seqs, c = list(seqs), self.cfg
        nodes = self._prompt_lengths(seqs, tokens)
        if max(nodes) > 64:
            raise ValueError(f"trees of at most 64 nodes, not {max(nodes)}")
        if parents is None:
            parents = [range(-1, n - 1) for n in nodes]
        parents = [[int(x) for x in p] for p in parents]
        if len(parents) != len(seqs) or [len(p) for p in parents] != nodes:
            raise ValueError("one parent for each node")
        for p in parents:
            if p[0] != -1 or any(not 0 <= x < i for i, x in enumerate(p) if i):
                raise ValueError("the first node's parent is -1, the others' are nodes before them")
        lengths = [cache.length(q) for q in seqs]
        with _appending(cache, seqs, nodes):
            cu = torch.zeros(len(seqs) + 1, dtype=torch.int32)
            cu[1:] = torch.tensor(nodes).cumsum(0)
            step = DraftStep(cache, seqs, [cache.mark(q) for q in seqs], lengths, nodes,
                             torch.cat([t.reshape(-1).to(self.device, torch.int64) for t in tokens]),
                             torch.tensor([x for p in parents for x in p], dtype=torch.int32).to(self.device),
                             cu.to(self.device),
                             torch.tensor([n + m for n, m in zip(lengths, nodes)], dtype=torch.int32).to(self.device))
            table = cache.table(seqs).to(self.device)
            T = step.tokens.numel()
            linear = ops.skinny_linear if T <= 16 and self._skinny_ok else F.linear

            def attention(li, lyr, xn):
                k, v = cache.layer(li)
                return ops.paged_tree_attention(linear(xn, lyr.qkv_w), lyr.q_norm, lyr.k_norm, step.parents,
                                                step.cu_seqlens, step.kv_lens, k, v, table, c.num_attention_heads,
                                                c.num_key_value_heads, c.rope_theta, c.rms_norm_eps,
                                                window=cache.window, sinks=cache.sinks)

            hn = self._layers(F.embedding(step.tokens, self.embed), attention, linear, decode=True)
            return linear(hn, self.lm_head), step

    @torch.inference_mode()
    def accept_paged(self, cache: PagedKVCache, step: DraftStep, sampled: torch.Tensor) -> list[torch.Tensor]:
        """Ends a step with drafted tokens: ``sampled`` (int64 on the device) is the
        token drawn after each of its nodes, from the logits of :meth:`draft_paged`.
        Of each tree the path that the drawn tokens agree with stays in the
        sequence, the other nodes leave it.  Returns for each sequence the rows of
        its path: ``sampled[rows[i]]`` are its new tokens, of which the last is not
        in the cache yet."""
        if cache is not step.cache:
            raise ValueError("the step is of another cache")
        if step.ended or not all(cache.kept(q, m) for q, m in zip(step.seqs, step.marks)):
            raise ValueError("the sequences are not as the step left them")
        if not all(cache.alone(q, n) for q, n in zip(step.seqs, step.lengths)):
            raise ValueError("a sequence was forked between its step and the step's end")
        counts, path, _ = ops.accept_drafts(step.tokens, sampled, step.parents, step.cu_seqlens, step.kv_lens, cache.pool,
                                            cache.table(step.seqs).to(self.device))
        counts = counts.tolist()
        step.ended = True
        for q, m in zip(step.seqs, step.marks):
            cache.unmark(q, m)
        cache.take_back(step.seqs, [n + k for n, k in zip(step.lengths, counts)])
        for q in step.seqs:
            cache.trim(q)
        starts = torch.tensor(step.nodes).cumsum(0) - torch.tensor(step.nodes)
        return [path[a:a + k].long() + a for a, k in zip(starts.tolist(), counts)]

    def _draw(self, logits, temperature, top_k, top_p, min_p, generator):
        """Tokens from rows of logits, by a random number each; -1 for a row that has no
        distribution (a NaN, or nothing that is finite)."""
        if temperature == 0:
            most, tok = logits.max(-1)  # a NaN comes through; the first of equal logits
            return torch.where(most.abs() < math.inf, tok, -1)
        u = torch.rand(logits.shape[0], dtype=torch.float64, device=self.device, generator=generator)
        return ops.sample_tokens(logits, u, temperature, top_k, top_p, min_p)[0]

    def _generate_drafted(self, cache, seqs, tok, prompts, max_new, drafts, draw, top_logprobs, scores):
        """The loop of :meth:`generate_paged` with drafts, from each sequence's first
        new token on; appends to ``scores`` (one list per sequence)."""
        new = [[int(t)] for t in tok.tolist()]
        texts = [LookupDrafts(p + n) for p, n in zip(prompts, new)]
        live = [i for i in range(len(seqs)) if max_new > 1]
        while live:
            trees = []
            for i in live:
                room = cache.max_pages * cache.page_size - cache.length(seqs[i])
                most = max(0, min(drafts, max_new - len(new[i]) - 1, 63, room - 1))
                tokens, parents = texts[i].tree(most)
                trees.append(([new[i][-1]] + tokens, [-1] + [x + 1 for x in parents]))
            for attempt in (trees, [(t[:1], p[:1]) for t, p in trees]):  # pages may be short of drafts
                try:
                    logits, step = self.draft_paged(cache, [seqs[i] for i in live], [torch.tensor(t) for t, _ in attempt],
                                                    [p for _, p in attempt])
                    break
                except CacheFull:
                    if attempt is not trees:
                        raise
            sampled = draw(logits)
            rows = self.accept_paged(cache, step, sampled)
            kept = torch.cat(rows)
            if top_logprobs is not None:
                parts = ops.token_logprobs(logits[kept], sampled[kept], top_logprobs)
                at = 0
                for i, r in zip(live, rows):
                    scores[i].append(tuple(x[at:at + len(r)] for x in parts))
                    at += len(r)
            drawn = sampled[kept].tolist()
            if min(drawn) < 0:
                raise RuntimeError("logits without a distribution")
            for i, r in zip(live, rows):
                new[i] += drawn[:len(r)]
                texts[i].extend(drawn[:len(r)])
                drawn = drawn[len(r):]
            live = [i for i in live if len(new[i]) < max_new]
        return new

    @torch.inference_mode()
    def generate_paged(self, prompts, max_new_tokens: int, samples: int = 1, temperature: float = 0.0,
                       top_logprobs: int | None = None, page_size: int = 64, window: int = 0, sinks: int = 0,
                       generator: torch.Generator | None = None, cache: PagedKVCache | None = None,
                       graph: bool = True, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, drafts: int = 0):
        """Generation for prompts of any lengths, ``samples`` continuations of
        each from one prefill (the prompt's pages are shared).

        Greedy with ``temperature`` 0, else sampled (``generator`` on the
        stack's device), with ``top_k``, ``top_p`` and ``min_p`` from the
        distribution that they restrict (:func:`nki_moe_b200.ops.sample_tokens`).
        With ``drafts`` each step checks up to so many tokens (at most 63) that the
        text itself suggests (:class:`nki_moe_b200.drafts.LookupDrafts`) and keeps
        those that the model agrees with: every token is drawn from the model's own
        logits for the text before it, in fewer steps where texts repeat (near ties
        between logits may fall the other way than without drafts, whose steps round
        elsewhere); steps are not captured then.  With ``window`` the model attends to the last
        ``window`` tokens and the first ``sinks`` ones; a ``cache`` that is given
        brings its own page size and window.  Returns ``(tokens
        [len(prompts), samples, max_new_tokens], scores)``; ``scores`` is None
        or, with ``top_logprobs`` alternatives, a dict of ``logprob`` and
        ``entropy`` ``[.., max_new_tokens]`` and ``top_logprobs``/``top_ids``
        ``[.., max_new_tokens, top_logprobs]``."""
        if samples < 1 or max_new_tokens < 1:
            raise ValueError("samples and max_new_tokens must be positive")
        if not (0 <= top_p <= 1 and 0 <= min_p <= 1 and top_k >= 0 and 0 <= drafts <= 63):
            raise ValueError("top_k must not be negative, top_p and min_p must be in [0, 1], drafts in [0, 63]")
        if drafts and any(lyr.ep is not None for lyr in self.layers):
            raise ValueError("drafts are for stacks on one GPU")
        restricted = top_k > 0 or top_p < 1 or min_p > 0
        if (restricted or drafts) and not temperature >= 0:
            raise ValueError("temperature must not be negative")
        n, ends, own = len(prompts), [int(p.numel()) + max_new_tokens + drafts for p in prompts], cache is None
        if n == 0:
            raise ValueError("no prompts")
        if cache is None:
            pages = sum(-(-e // max(page_size, 1)) * samples for e in ends)
            cache = self.paged_cache(pages, page_size, max(ends), window, sinks)
        elif (window or sinks) and (window, sinks) != (cache.window, cache.sinks):
            raise ValueError(f"the cache has window {cache.window} and sinks {cache.sinks}, not {window} and {sinks}")
        seqs = [cache.add() for _ in prompts]
        try:
            logits = self.prefill_paged(cache, seqs, prompts)
            seqs = [q for first in seqs for q in [first] + [cache.fork(first) for _ in range(samples - 1)]]
            logits = logits.repeat_interleave(samples, 0)
            out, scores = [], []

            def draw(rows):
                return self._draw(rows, temperature, top_k, top_p, min_p, generator)

            if drafts:
                tok = draw(logits)
                if int(tok.min()) < 0:
                    raise RuntimeError("logits without a distribution")
                if top_logprobs is not None:
                    scores = [[tuple(x[i:i + 1] for x in ops.token_logprobs(logits, tok, top_logprobs))]
                              for i in range(len(seqs))]
                texts = [p.reshape(-1).tolist() for p in prompts for _ in range(samples)]
                out = self._generate_drafted(cache, seqs, tok, texts, max_new_tokens, drafts, draw, top_logprobs, scores)
            for i in range(0 if drafts else max_new_tokens):
                if restricted:
                    tok = draw(logits)
                elif temperature > 0:
                    # the largest of logits + Gumbel noise is a sample of the softmax
                    noise = torch.empty_like(logits, dtype=torch.float32).exponential_(generator=generator).log()
                    tok = (logits.float() / temperature - noise).argmax(-1)
                else:
                    tok = logits.argmax(-1)
                out.append(tok)
                if top_logprobs is not None:
                    scores.append(ops.token_logprobs(logits, tok, top_logprobs))
                if i + 1 < max_new_tokens:
                    # (a row without a distribution goes on with any token: it is refused at the end)
                    logits = self.decode_paged(cache, seqs, tok.clamp(min=0) if restricted else tok, graph)
        finally:
            for q in seqs:
                if q in cache:
                    cache.free(q)
            if own:
                self._drop_steps(cache)  # nobody else can use this cache
        tokens = torch.tensor(out, device=self.device) if drafts else torch.stack(out, 1)
        tokens = tokens.view(n, samples, max_new_tokens)
        if restricted and not drafts and int(tokens.min()) < 0:
            raise RuntimeError("logits without a distribution")
        if top_logprobs is None:
            return tokens, None
        if drafts:
            lp, ent, tlp, tid = (torch.stack([torch.cat(x) for x in part]) for part in
                                 zip(*([[s[k] for s in seq] for k in range(4)] for seq in scores)))
        else:
            lp, ent, tlp, tid = (torch.stack(x, 1) for x in zip(*scores))
        shape = (n, samples, max_new_tokens)
        return tokens, {"logprob": lp.view(shape), "entropy": ent.view(shape), "top_logprobs": tlp.view(*shape, -1),
                        "top_ids": tid.view(*shape, -1)}

    @torch.inference_mode()
    def score(self, prompts, top_n: int = 0, page_size: int = 64, window: int = 0, sinks: int = 0,
              chunk: int = 2048):
        """Scores of given texts: for each prompt a tuple ``(logprob [n - 1],
        entropy [n - 1], top_logprobs [n - 1, top_n], top_ids)`` of its tokens
        from the second on, each under what comes before it.  The logits are
        formed ``chunk`` rows at a time."""
        lens = [int(p.numel()) for p in prompts]
        if not lens or min(lens) == 0:
            raise ValueError("prompts must not be empty")
        if chunk < 1:
            raise ValueError(f"chunk {chunk} is not positive")
        cache = self.paged_cache(sum(-(-n // max(page_size, 1)) for n in lens), page_size, max(lens), window, sinks)
        seqs = [cache.add() for _ in prompts]
        cache.extend(seqs, self._prompt_lengths(seqs, prompts))
        hn = self._prompt_hidden(cache, seqs, prompts)
        # a prompt's last row predicts nothing that is given
        given = torch.cat([torch.cat([p.reshape(-1)[1:].to(self.device), p.new_full((1,), -1).to(self.device)])
                           for p in prompts]).to(torch.int64)
        parts = [ops.token_logprobs(F.linear(hn[r:r + chunk], self.lm_head), given[r:r + chunk], top_n)
                 for r in range(0, hn.shape[0], chunk)]
        whole = [torch.cat(x) for x in zip(*parts)]
        return [tuple(t[:n - 1] for t in rows) for n, rows in zip(lens, zip(*(w.split(lens) for w in whole)))]

    # ------------------------------------------------------------ generate
    @torch.inference_mode()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, graph: bool = True):
        """Greedy generation.  Returns ``(tokens [B, max_new_tokens], timing)``
        with timing = {"ttft_ms", "decode_ms", "decode_tok_s"} measured with
        CUDA events (TTFT = prefill through the first token's argmax)."""
        B = input_ids.shape[0]
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        torch.cuda.synchronize(self.device)
        ev[0].record()
        logits = self.prefill(input_ids)
        tok = logits.argmax(-1)
        ev[1].record()
        out = [tok]
        for _ in range(max_new_tokens - 1):
            tok = self._step(tok, graph).argmax(-1)
            out.append(tok)
        ev[2].record()
        torch.cuda.synchronize(self.device)
        ttft = ev[0].elapsed_time(ev[1])
        dec = ev[1].elapsed_time(ev[2])
        n = max_new_tokens - 1
        timing = {"ttft_ms": ttft, "decode_ms": dec, "decode_steps": n,
                  "decode_tok_s": (B * n) / (dec * 1e-3) if n and dec > 0 else math.nan}
        return torch.stack(out, 1), timing


def wall_ms(fn) -> float:
    torch.cuda.synchronize()
    t = time.perf_counter()
    fn()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) * 1e3
