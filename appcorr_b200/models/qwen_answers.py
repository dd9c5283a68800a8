"""Answers of many requests at once on the sm_100a VLM engine (models/qwen_engine.py).

A `PackedAnswers` serves up to `max_requests` requests in packed steps: one step takes any number of
new tokens of each of them (a whole question first, then one token at a time) as consecutive rows
of one batch. With a `session` (an image and its instructions after `QwenVLEngine.approx` or
`correct`), every request continues that prompt: its keys and values are copied once per layer into
this object's page pool and read once per step for all the requests.

    layout     packed_layout: pages, cache rows and positions of the step from the new lengths
    per layer  RMSNorm -> qkv GEMM [bias] -> qk_norm_rope [M-RoPE by position axes, K / V into their
               pages] -> shared_prefix_attention (packed_attention without a session) -> o GEMM
               [+ residual] -> RMSNorm -> SwiGLU GEMM -> down GEMM [+ residual]
    head       RMSNorm of every request's last row -> LM head GEMM

The reference answers only with the first token of one request (offload/server/model/
qwen25vl_executor.py:252-286) and leaves the rest to a library's generate().
"""
from __future__ import annotations

from typing import List, Optional

import torch

from ..ops import kernels as K
from ..ops import packed as P
from ..ops.native import check_errors
from .qwen_engine import BF16, QwenSession, QwenVLEngine, _pad_to


class PackedAnswers:
    """max_own: own tokens a request may hold (question and answer); max_step: tokens of one step."""

    def __init__(self, engine: QwenVLEngine, max_requests: int, max_own: int, max_step: int,
                 session: Optional[QwenSession] = None):
        c, dev = engine.cfg, engine.device
        if engine.nh != c.heads or engine.nkv != c.kv_heads:
            raise ValueError("PackedAnswers runs on an engine that holds all the heads (no tensor parallelism)")
        if session is not None and not session.approx_done:
            raise ValueError("the session's prompt has not been run (approx)")
        self.engine, self.max_requests, self.max_step = engine, max_requests, max_step
        own_blocks = (max_own + P.PAGE - 1) // P.PAGE
        self.prefix_len = session.N if session is not None else 0
        shared = (self.prefix_len + P.PAGE - 1) // P.PAGE
        pages = shared + max_requests * own_blocks
        kvd = c.kv_heads * c.head_dim
        i32 = lambda *s: torch.zeros(*s, device=dev, dtype=torch.int32)  # noqa: E731
        e = lambda *s, dtype=BF16: torch.empty(*s, device=dev, dtype=dtype)  # noqa: E731
        self.k = [e(pages * P.PAGE, kvd) for _ in range(c.depth)]
        self.v = [e(pages * P.PAGE, kvd) for _ in range(c.depth)]
        self.prefix_table = torch.arange(shared, device=dev, dtype=torch.int32)
        self.free_pages = torch.arange(shared, pages, device=dev, dtype=torch.int32)
        self.table = torch.full((max_requests, own_blocks), -1, device=dev, dtype=torch.int32)
        # rotary frequencies and the position axis (temporal / height / width) of each pair
        half = c.head_dim // 2
        self.inv_freq = (1.0 / c.rope_theta ** (torch.arange(half, dtype=torch.float64) / half)).float().to(dev)
        a, b, _ = c.mrope_section
        self.axis = ((torch.arange(half) >= a).int() + (torch.arange(half) >= a + b).int()).to(dev)
        self.first_pos = 0
        if session is not None:
            side = [s // c.patch // c.merge for s in session.img_hw]
            self.first_pos = session.n_before + max(side) + session.n_after  # text goes on after the prompt's last position
            rows = session.tensors["phys"].long()
            for l in range(c.depth):
                self.k[l][:self.prefix_len] = session.tensors["kc"][l][rows]
                self.v[l][:self.prefix_len] = session.tensors["vc"][l][rows]
        D = c.hidden
        self.t = dict(x=e(max_step, D), xn=e(max_step, D), qkv=e(max_step, (c.heads + 2 * c.kv_heads) * c.head_dim),
                      q=e(max_step, c.heads * c.head_dim), o=e(max_step, c.heads * c.head_dim), h=e(max_step, engine.nffn),
                      rows=i32(max_step), req=i32(max_step), pos=i32(max_step), q_start=i32(max_requests + 1),
                      logits=e(max_requests, _pad_to(c.vocab, 32), dtype=torch.float32), last=e(max_requests, D))
        if engine.fp8:
            self.t["a8"] = torch.empty(max_step, max(D, engine.nffn), device=dev, dtype=torch.float8_e4m3fn)
            self.t["a8s"] = torch.empty(max_step, device=dev, dtype=torch.float32)
        self.zero = torch.zeros(1, device=dev, dtype=torch.int64)
        self.reset()

    def reset(self) -> None:
        """Forget all requests (the shared prompt stays)."""
        z = lambda n: torch.zeros(n, device=self.engine.device, dtype=torch.int32)  # noqa: E731
        self.held = z(self.max_requests)          # own tokens of each request so far
        self.free_at = z(2)                       # next free page, blocks that went without one
        self.t["last"].zero_()                    # normalised last row of each request
        self.asked = torch.zeros_like(self.zero)  # tokens that q_len has named

    def step(self, ids: torch.Tensor, q_len: torch.Tensor) -> torch.Tensor:
        """ids int32 (N values): the new tokens, request by request; q_len int32 [B] how many each brings.
        Both lie on the engine's device; ids are rows of the embedding and not checked against it here.
        -> fp32 logits [B, vocab] after each request's last token (valid until the next step). A request
        that brings none (an answer that has ended) keeps those of its last step, zeros before its first.
        Tokens that q_len names and ids does not hold are not taken, ids past the sum of q_len are padding.
        Does not synchronise; `tokens_missing` tells whether ids were too few, `pages_missing` whether the
        pool was too small."""
        eng, c, t = self.engine, self.engine.cfg, self.t
        for name, x, fits in (("ids", ids, ids.is_contiguous()), ("q_len", q_len, q_len.dim() == 1)):
            if x.dtype != torch.int32 or x.device != t["x"].device or not fits:
                raise ValueError(f"{name} must be int32 on {t['x'].device}, ids contiguous, q_len of one dimension")
        N, B = ids.numel(), q_len.numel()
        if N > self.max_step or B > self.max_requests:
            raise ValueError(f"{N} tokens of {B} requests: this batch holds {self.max_step} of {self.max_requests}")
        if B:
            ends = q_len.clamp(min=0).cumsum(0)
            self.asked += ends[-1]
        if B and N:  # of each request, the tokens that are there
            self._layers(ids, torch.diff(ends.clamp_(max=N), prepend=self.zero).to(torch.int32))
        logits = t["logits"][:B]
        if B:
            K.gemm(t["last"][:B], eng.lm_head, logits, epi=K.EPI_F32)
        return logits[:, :c.vocab]

    def _layers(self, ids: torch.Tensor, q_len: torch.Tensor) -> None:
        """The new tokens through every layer; `last` takes the last one of each request that brings any."""
        eng, c, t = self.engine, self.engine.cfg, self.t
        N, B = ids.numel(), q_len.numel()
        rows, req, pos, q_start = t["rows"][:N], t["req"][:N], t["pos"][:N], t["q_start"][:B + 1]
        kv_len, free_at = torch.empty_like(q_len), torch.empty_like(self.free_at)
        table = self.table[:B]
        P.packed_layout(q_len, self.held[:B], table, self.free_pages, self.free_at[:1], q_start=q_start, kv_len=kv_len, rows=rows,
                        req=req, pos=pos, free_next=free_at)
        free_at[1:] += self.free_at[1:]
        at = (pos + self.first_pos)[None].expand(3, N)  # text: all axes together
        heads = dict(heads=c.heads, kv_heads=c.kv_heads, head_dim=c.head_dim)
        x, xn, qkv, q, o, h = (t[n][:N] for n in ("x", "xn", "qkv", "q", "o", "h"))
        K.gather_rows(eng.embed, ids, x)
        for l, w in enumerate(eng.llm):
            a, sa = eng._norm(t, x, w.norm1, xn)
            wq, sw = eng._wt(l, "qkv_w")
            K.gemm(a, wq, qkv, bias=w.qkv_b, a_scale=sa, b_scale=sw)
            P.qk_norm_rope(qkv, at, self.inv_freq, self.axis, q, self.k[l], self.v[l], rows=rows, **heads)
            if self.prefix_len:
                P.shared_prefix_attention(q, self.k[l], self.v[l], o, q_start=q_start, kv_len=kv_len, table=table,
                                          prefix_table=self.prefix_table, prefix_len=self.prefix_len, **heads)
            else:
                P.packed_attention(q, self.k[l], self.v[l], o, q_start=q_start, kv_len=kv_len, table=table, **heads)
            a, sa = eng._act(t, o)
            wq, sw = eng._wt(l, "o_w")
            K.gemm(a, wq, x, epi=K.EPI_RESID, gamma=eng.ones, resid=x, a_scale=sa, b_scale=sw)
            a, sa = eng._norm(t, x, w.norm2, xn)
            wq, sw = eng._wt(l, "w12")
            K.gemm(a, wq, h, epi=K.EPI_SWIGLU, a_scale=sa, b_scale=sw)
            a, sa = eng._act(t, h)
            wq, sw = eng._wt(l, "w3")
            K.gemm(a, wq, x, epi=K.EPI_RESID, gamma=eng.ones, resid=x, a_scale=sa, b_scale=sw)
        self.held = torch.cat([kv_len, self.held[B:]])
        self.free_at = free_at
        last = t["last"][:B]
        ends = torch.empty_like(last)
        K.rmsnorm(x, eng.norm, c.rms_eps, ends, rows=q_start[1:].clamp(min=1).sub_(1))
        torch.where(q_len[:, None] > 0, ends, last, out=last)

    @property
    def pages_missing(self) -> int:
        """Blocks that went without a page so far (synchronises); above zero the answers are not valid."""
        return int(self.free_at[1])

    @property
    def tokens_missing(self) -> int:
        """Tokens named by q_len that ids did not hold so far (synchronises)."""
        return int(self.asked - self.held.sum())

    def generate(self, questions: List[torch.Tensor], n: int) -> torch.Tensor:
        """Greedy answers of n tokens to the questions (int32 token ids each) -> int32 [B, n]. Raises where
        a kernel has recorded an error or the pages did not do (synchronises)."""
        dev = self.engine.device
        if not questions or any(q.numel() == 0 for q in questions):
            raise ValueError("every request needs at least one token")
        if n < 0:
            raise ValueError(f"answers of {n} tokens")
        ids = torch.cat([q.to(device=dev, dtype=torch.int64).reshape(-1) for q in questions])
        lo, hi = (int(v) for v in torch.stack(ids.aminmax()))
        if lo < 0 or hi >= self.engine.cfg.vocab:
            raise ValueError(f"token ids from {lo} to {hi}: the vocabulary has {self.engine.cfg.vocab}")
        ids = ids.to(torch.int32)
        self.reset()
        q_len = torch.tensor([q.numel() for q in questions], dtype=torch.int32, device=dev)
        one = torch.ones_like(q_len)
        out = []
        for _ in range(n):
            ids = self.step(ids, q_len).argmax(1).to(torch.int32)
            out.append(ids)
            q_len = one
        check_errors(dev)
        if self.pages_missing:
            raise RuntimeError("PackedAnswers: the requests outgrew the page pool (max_own)")
        return torch.stack(out, 1) if out else ids.new_empty(len(questions), 0)
