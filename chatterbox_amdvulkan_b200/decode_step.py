"""Batched multi-stream T3 decode step, caller side.

The engine decodes one stream at a time (chatterbox-cpp/src/t3.cpp:297-328:
append_speech -> forward_impl per token).  This module runs one decode step
for B independent streams at once: each stream contributes one new token at
its own position, with its own KV-cache slab.  The per-layer order follows
forward_impl (t3.cpp:459-546):

    LN1 -> QKV GEMM -> qkv bias + Q + KV-cache append -> attention over the
    stream's cache -> out GEMM (+ bias) -> attn_residual = out + h -> LN2 ->
    fc GEMM -> fc bias + GELU -> proj GEMM (+ bias) -> h = proj + attn_residual

and ends with the final LayerNorm.  The elementwise steps are libcbx_ops
kernels (called through the C ABI), with each residual add fused into the
next LayerNorm.  The GEMMs are cuBLAS (torch.mm / torch.addmm) and the
attention is torch's scaled_dot_product_attention: both are outside this
library.  Everything is enqueued on the current CUDA stream and allocates
from torch's caching allocator, so a whole step can be captured in one CUDA
graph and replayed with new positions.

A stream whose position is outside [0, max_context) gets no K / V write; the
kernel raises a flag in the model's device error word instead.  ``step``
reads that word after an eager step and raises ``PositionOutOfRange``; when
the step is captured in a CUDA graph the caller calls ``check_errors()``
after each replay.

``T3PagedDecode`` is the form for a server: requests of unequal length on a
paged cache, attention and the answer's log probabilities in libcbx_ops too.

Weights are random (this repository ships no checkpoints); shapes follow
T3's GPT-2-style blocks (hidden 1024, 16 heads, FFN 4096).
"""
from __future__ import annotations

import torch

from . import ops


class PositionOutOfRange(RuntimeError):
    """A stream's position was outside [0, max_context): its K / V row was not
    written, so the step's attention ran over a stale cache."""


def _random_layers(n_layers, D, F, device, seed):
    """(blocks, final LN weight and bias, the generator behind them)."""
    g = torch.Generator(device=device).manual_seed(seed)

    def w(*shape, std=0.02):
        return torch.randn(*shape, generator=g, device=device) * std

    def ln():
        return 1.0 + 0.1 * torch.randn(D, generator=g, device=device), w(D, std=0.1)

    layers = []
    for _ in range(n_layers):
        ln1_w, ln1_b = ln()
        ln2_w, ln2_b = ln()
        layers.append(dict(
            ln1_w=ln1_w, ln1_b=ln1_b, qkv_w=w(D, 3 * D), qkv_b=w(3 * D, std=0.1),
            out_w=w(D, D), out_b=w(D, std=0.1), ln2_w=ln2_w, ln2_b=ln2_b,
            fc_w=w(D, F), fc_b=w(F, std=0.1), proj_w=w(F, D), proj_b=w(D, std=0.1)))
    return (layers, *ln(), g)


class T3BatchedDecode:
    """B streams, n_layers blocks, KV cache [n_layers][B][max_context][D]."""

    def __init__(self, n_layers: int, B: int, max_context: int, D: int = 1024, H: int = 16,
                 F: int = 4096, cache_dtype=torch.float32, device="cuda", seed: int = 0,
                 eps: float = 1e-5):
        if D % H:
            raise ValueError("D must be a multiple of H")
        self.L, self.B, self.ctx, self.D, self.H, self.F = n_layers, B, max_context, D, H, F
        self.eps = eps
        self.layers, self.lnf_w, self.lnf_b = _random_layers(n_layers, D, F, device, seed)[:3]
        self.cache_k = torch.zeros(n_layers, B, max_context, D, dtype=cache_dtype, device=device)
        self.cache_v = torch.zeros_like(self.cache_k)
        self.err = torch.zeros(1, dtype=torch.int32, device=device)

    # -- attention over each stream's cache, keys 0..positions[b] -------------
    def _attend(self, q: torch.Tensor, layer: int, positions: torch.Tensor) -> torch.Tensor:
        B, D, H = self.B, self.D, self.H
        hd = D // H
        k = self.cache_k[layer].view(B, self.ctx, H, hd).transpose(1, 2)
        v = self.cache_v[layer].view(B, self.ctx, H, hd).transpose(1, 2)
        qh = q.view(B, H, 1, hd).to(k.dtype)
        keys = torch.arange(self.ctx, device=q.device)
        mask = (keys[None, :] <= positions[:, None].long()).view(B, 1, 1, self.ctx)
        a = torch.nn.functional.scaled_dot_product_attention(qh, k, v, attn_mask=mask)
        return a.reshape(B, D).float()

    def check_errors(self) -> None:
        """Read and clear the device error word (synchronises with the stream);
        raise PositionOutOfRange when a step since the last check saw a
        position outside [0, max_context)."""
        from ._lib import EFLAG_POS_OOB
        flags = int(self.err.item())
        if flags:
            self.err.zero_()
            if flags & EFLAG_POS_OOB:
                raise PositionOutOfRange(
                    f"a stream's position was outside [0, {self.ctx}): its K / V row was not "
                    "written and the step's output is invalid")
            raise RuntimeError(f"decode step device error flags 0x{flags:x}")

    def step(self, x: torch.Tensor, positions: torch.Tensor, check: bool = True) -> torch.Tensor:
        """x: f32 [B, D] token + position embeddings of each stream's new token;
        positions: int32 [B] (each stream's n_past).  Writes the caches and
        returns the final-LN hidden state f32 [B, D].

        With ``check`` (the default) an eager step reads the device error word
        afterwards (one synchronisation) and raises PositionOutOfRange if a
        position was out of range.  Inside CUDA graph capture, or with
        ``check=False``, the caller calls ``check_errors()`` itself."""
        if positions.dtype != torch.int32:
            raise TypeError("positions must be int32")
        out = self._step(x, positions)
        if check and not torch.cuda.is_current_stream_capturing():
            self.check_errors()
        return out

    def _step(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        h = x
        mlp_out = resid = None
        for li, P in enumerate(self.layers):
            if li == 0:
                y1 = ops.layer_norm(h, P["ln1_w"], P["ln1_b"], self.eps)
            else:  # h = proj + attn_residual, fused into LN1 (t3.cpp:545, :465-466)
                y1, h = ops.add_layernorm(mlp_out, resid, P["ln1_w"], P["ln1_b"], self.eps,
                                          return_sum=True)
            qkv = torch.mm(y1, P["qkv_w"])
            q, _ = ops.qkv_kv_append(qkv, P["qkv_b"], self.cache_k[li], self.cache_v[li],
                                     positions=positions, slab_stride=self.ctx * self.D,
                                     max_context=self.ctx, err=self.err)
            a = self._attend(q, li, positions)
            o = torch.addmm(P["out_b"], a, P["out_w"])
            # attn_residual = o + h (t3.cpp:528), fused into LN2
            y2, resid = ops.add_layernorm(o, h, P["ln2_w"], P["ln2_b"], self.eps,
                                          return_sum=True)
            m = ops.bias_act(torch.mm(y2, P["fc_w"]), P["fc_b"], "gelu")
            mlp_out = torch.addmm(P["proj_b"], m, P["proj_w"])
        return ops.add_layernorm(mlp_out, resid, self.lnf_w, self.lnf_b, self.eps)

    # -- the same step with plain torch elementwise ops (the check) -----------
    def step_reference(self, x: torch.Tensor, positions: torch.Tensor, cache_k, cache_v):
        """The step in plain torch fp32 (F.layer_norm, tanh GELU, index writes)
        on separate caches: the reference the library-backed step is tested
        against."""
        B, D = self.B, self.D
        ln = torch.nn.functional.layer_norm
        h = x
        rows = torch.arange(B, device=x.device)
        pos = positions.long()
        for li, P in enumerate(self.layers):
            y1 = ln(h, (D,), P["ln1_w"], P["ln1_b"], self.eps)
            qkv = torch.mm(y1, P["qkv_w"]) + P["qkv_b"]
            q, k, v = qkv[:, :D], qkv[:, D:2 * D], qkv[:, 2 * D:]
            cache_k[li][rows, pos] = k.to(cache_k.dtype)
            cache_v[li][rows, pos] = v.to(cache_v.dtype)
            hd = D // self.H
            kk = cache_k[li].view(B, self.ctx, self.H, hd).transpose(1, 2)
            vv = cache_v[li].view(B, self.ctx, self.H, hd).transpose(1, 2)
            keys = torch.arange(self.ctx, device=x.device)
            mask = (keys[None, :] <= pos[:, None]).view(B, 1, 1, self.ctx)
            a = torch.nn.functional.scaled_dot_product_attention(
                q.reshape(B, self.H, 1, hd).to(kk.dtype), kk, vv, attn_mask=mask)
            a = a.reshape(B, D).float()
            o = torch.addmm(P["out_b"], a, P["out_w"])
            resid = o + h
            y2 = ln(resid, (D,), P["ln2_w"], P["ln2_b"], self.eps)
            m = torch.nn.functional.gelu(torch.mm(y2, P["fc_w"]) + P["fc_b"], approximate="tanh")
            h = torch.addmm(P["proj_b"], m, P["proj_w"]) + resid
        return ln(h, (D,), self.lnf_w, self.lnf_b, self.eps)


class PagedCacheFull(RuntimeError):
    """A request's tokens found no page (the pool is empty, or its row of the
    block table full) or its length was out of range: its new K / V rows are
    missing or mean nothing, and the step's output for it is invalid."""


class T3PagedDecode:
    """T3 serving on a paged KV cache: up to ``max_reqs`` requests of unequal
    length share ``n_pages`` pages of ``page_size`` tokens (all layers use one
    block table), and one step feeds any number of new tokens per request: a
    whole prompt, a speculated run or the next token.

        plan -> embedding gather-add -> per layer [LN1 -> QKV GEMM -> bias, Q and
        K / V into the pages -> attention over the pages -> out GEMM -> LN2 -> fc
        GEMM -> bias + GELU -> proj GEMM] -> final LN -> head GEMM -> log
        probabilities

    The GEMMs are cuBLAS, everything else is libcbx_ops.  All per-step state
    (block table, free pages, lengths) is on the device, so a step of fixed row
    count can be captured in one CUDA graph and replayed with new lengths and
    ids; rows behind the last token are padding.  Weights are random."""

    def __init__(self, n_layers: int, max_reqs: int, n_pages: int, page_size: int = 16,
                 max_context: int = 2048, D: int = 1024, H: int = 16, F: int = 4096,
                 vocab: int = 6563, cache_dtype=torch.float32, device="cuda", seed: int = 0,
                 eps: float = 1e-5):
        if D % H:
            raise ValueError("D must be a multiple of H")
        self.L, self.D, self.H, self.F, self.eps = n_layers, D, H, F, eps
        self.page_size, self.ctx = page_size, max_context
        self.layers, self.lnf_w, self.lnf_b, g = _random_layers(n_layers, D, F, device, seed)

        def w(*shape, std=0.02):
            return torch.randn(*shape, generator=g, device=device) * std

        self.tok_emb, self.pos_emb, self.head_w = w(vocab, D), w(max_context, D), w(D, vocab)
        shape = (n_layers, n_pages, page_size, H, D // H)
        self.cache_k = torch.zeros(shape, dtype=cache_dtype, device=device)
        self.cache_v = torch.zeros_like(self.cache_k)

        def ints(*shape, fill=0):
            return torch.full(shape, fill, dtype=torch.int32, device=device)

        self.block_table = ints(max_reqs, -(-max_context // page_size), fill=-1)
        self.n_blocks = ints(max_reqs)
        self.free_list = torch.arange(n_pages, dtype=torch.int32, device=device)
        self.n_free = ints(1, fill=n_pages)
        self.err = ints(1)

    def plan(self, seq_lens: torch.Tensor, n_new: torch.Tensor | None = None,
             max_rows: int | None = None) -> ops.PagedPlan:
        """Brings the block table to these lengths (int32 [max_reqs]; 0 ends a
        request and frees its pages) and lays out the rows of the last n_new
        tokens of each (None: one)."""
        return ops.paged_plan(seq_lens, self.block_table, self.n_blocks, self.free_list,
                              self.n_free, self.page_size, n_new=n_new, max_rows=max_rows,
                              in_place=True, err=self.err)

    def forward(self, ids: torch.Tensor, plan: ops.PagedPlan) -> torch.Tensor:
        """ids: int32 [rows], the token of each row of the plan (any valid id in
        padding rows).  Returns the final-LN hidden states f32 [rows, D]."""
        h = ops.embed_gather_add(self.tok_emb, ids, self.pos_emb, pos_ids=plan.positions,
                                 err_word=self.err)
        rows, mlp_out, resid = ids.numel(), None, None
        for li, P in enumerate(self.layers):
            if li == 0:
                y1 = ops.layer_norm(h, P["ln1_w"], P["ln1_b"], self.eps)
            else:
                y1, h = ops.add_layernorm(mlp_out, resid, P["ln1_w"], P["ln1_b"], self.eps,
                                          return_sum=True)
            ck, cv = self.cache_k[li], self.cache_v[li]
            q, _ = ops.qkv_kv_append_paged(torch.mm(y1, P["qkv_w"]), P["qkv_b"], ck, cv,
                                           plan.slots, err=self.err)
            a = ops.paged_decode_attention(q.view(rows, self.H, self.D // self.H), ck, cv,
                                           plan.block_table, plan.row_lens,
                                           row_reqs=plan.row_reqs, err=self.err)
            o = torch.addmm(P["out_b"], a.view(rows, self.D), P["out_w"])
            y2, resid = ops.add_layernorm(o, h, P["ln2_w"], P["ln2_b"], self.eps, return_sum=True)
            m = ops.bias_act(torch.mm(y2, P["fc_w"]), P["fc_b"], "gelu")
            mlp_out = torch.addmm(P["proj_b"], m, P["proj_w"])
        return ops.add_layernorm(mlp_out, resid, self.lnf_w, self.lnf_b, self.eps)

    def step(self, ids: torch.Tensor, seq_lens: torch.Tensor, n_new: torch.Tensor | None = None,
             targets: torch.Tensor | None = None, top_k: int = 1,
             check: bool = True) -> tuple[torch.Tensor, ops.TokenLogprobs]:
        """One step over ids.numel() rows (request by request, token by token):
        (hidden states, log probabilities of ``targets`` with entropy and the
        top_k next tokens of every row).  ``check`` as in T3BatchedDecode."""
        h = self.forward(ids, self.plan(seq_lens, n_new, ids.numel()))
        out = ops.token_logprobs(torch.mm(h, self.head_w), targets, top_k=top_k, err=self.err)
        if check and not torch.cuda.is_current_stream_capturing():
            self.check_errors()
        return h, out

    def check_errors(self) -> None:
        """Read and clear the device error word (synchronises with the stream)."""
        from ._lib import EFLAG_LENGTH, EFLAG_NO_PAGE, EFLAG_POS_OOB
        flags = int(self.err.item())
        if flags:
            self.err.zero_()
            # a length between max_context and the end of its last page has a page, but no position
            if flags & (EFLAG_NO_PAGE | EFLAG_LENGTH | EFLAG_POS_OOB):
                raise PagedCacheFull(
                    "a request found no page for its new tokens, or its length is outside "
                    f"[0, {self.ctx}] (device error flags 0x{flags:x})")
            raise RuntimeError(f"paged decode step device error flags 0x{flags:x}")


def rel_err(a: torch.Tensor, b: torch.Tensor) -> float:
    return float((a - b).abs().max() / b.abs().max().clamp_min(1e-30))


__all__ = ["PagedCacheFull", "PositionOutOfRange", "T3BatchedDecode", "T3PagedDecode", "rel_err"]
