"""Generation over a paged key/value cache: a prompt's forward once, then one token a step for several answers.

``PagedDecoder`` runs the model of a (forward-only) ``TrainEngine`` on its weights. ``prefill`` computes a
prompt and leaves its keys and values in pages; ``branch(n)`` makes those pages the shared prefix of n answers;
``step`` adds one token to each of them; ``check`` says whether the GPU could do it all. Lengths, page tables, slots
and the attention's work list are made on the GPU each step (``ops.paged``); per layer the QKV GEMM is followed by the
append (bias, rotation, K and V to their slots) and the attention, in which the prompt's keys are read once for all
answers.

The reference re-runs the whole forward for every new token (node/cli/src/main.rs:1416-1548); this computes the logits
from the new tokens alone. They are those of the re-run forward (``serve.EngineLM``) up to roundings, of which there are
more here: the QKV product is rounded to bf16 before bias and rotation (there, for heads of 64 and 128, the GEMM's
epilogue adds and rotates its fp32 sums, which for this path would be a GEMM that knows the cache), and the logits are a
product with the bf16 embedding on the framework's own GEMM (there with the fp32 one). Against the fp32 oracle, with
random weights, they are 9.1e-3 of their norm off for the 12-layer preset (there 7.9e-3) and 2.0e-2 for the 24-layer one
(1.7e-2).
"""
from __future__ import annotations

import contextlib
import functools
from typing import List, Sequence

import torch

from .. import ops
from ..ops import paged
from .oracle import rope_tables

ROWS = 128  # rows of an activation buffer: whole GEMM tiles


def _pad(n: int, a: int) -> int:
    return (n + a - 1) // a * a


def on_device(dev: torch.device):
    """``dev`` as the current device, where kernels are launched. (Which device is current belongs to the calling
    thread, and a server's handlers have threads of their own.)"""
    return torch.cuda.device(dev) if dev.type == "cuda" else contextlib.nullcontext()


def _on_its_device(method):
    @functools.wraps(method)
    def run(self, *args, **kw):
        with on_device(self.dev):
            return method(self, *args, **kw)
    return run


class PagedDecoder:
    """Room for prompts of ``max_prompt`` tokens and ``max_batch`` answers of ``max_new`` tokens each."""

    def __init__(self, eng, max_prompt: int, max_new: int, max_batch: int = 1, page_size: int = 64):
        if eng.tp is not None and eng.tp.size > 1:
            raise NotImplementedError("PagedDecoder runs on engines without tensor parallelism")
        if eng.d not in (16, 32, 64, 128) or eng.nh // eng.nkv > paged.MAX_GROUP_HEADS:
            raise ValueError(f"no paged attention for head dim {eng.d} with {eng.nh // eng.nkv} query heads a kv head")
        self.eng, self.P, self.dev = eng, page_size, eng.device
        self.max_prompt, self.max_new, self.max_batch = int(max_prompt), int(max_new), int(max_batch)
        self.prompt_pages, self.answer_pages = -(-self.max_prompt // self.P), max(1, -(-self.max_new // self.P))
        pages = self.prompt_pages + self.max_batch * self.answer_pages
        shape = (eng.cfg.num_layers, pages, eng.nkv, self.P, eng.d)
        self.k, self.v = (torch.zeros(shape, dtype=torch.bfloat16, device=self.dev) for _ in range(2))
        self.dev = self.k.device  # (with its index)
        self.free = torch.arange(pages, dtype=torch.int32, device=self.dev)
        cos, sin = rope_tables(eng.cfg, self.max_prompt + self.max_new)
        self.cos, self.sin = cos.to(self.dev).contiguous(), sin.to(self.dev).contiguous()
        self.ldv = _pad(eng.V, 8)
        self._bufs = {}
        self.taken = 0  # pages in use
        self.used = self._ints(self.max_new + 1, 2)  # what page_tables said of the prompt (row 0) and of each step
        self.prompt_len = self.n = self.length = 0

    def _ints(self, *shape):
        return torch.zeros(*shape, dtype=torch.int32, device=self.dev)

    def _buffers(self, M: int):
        """Activations of ``M`` rows, made on first use."""
        if M not in self._bufs:
            e, b16, dev = self.eng, torch.bfloat16, self.dev
            new = lambda *s, dtype=b16: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
            f32 = torch.float32
            self._bufs = {M: dict(ids=self._ints(M), slots=self._ints(M), positions=self._ints(M), x=new(M, e.H, dtype=f32),
                                  mid=new(M, e.H, dtype=f32), xn=new(M, e.H), rstd=new(M, dtype=f32), br=new(M, e.H),
                                  qkv=new(M, e.W), q=new(M, e.nh * e.d), attn=new(M, e.nh * e.d), gu=new(M, 2 * e.F),
                                  h=new(M, e.F))}
        return self._bufs[M]

    def _tables(self, b, cached, new, tables, cu, total, start, pages, row):
        """Page tables of a step whose requests take ``pages`` pages together (the host knows all lengths)."""
        paged.page_tables(cached, new, self.free[self.taken:], tables, b["slots"], b["positions"], cu, total,
                          self.used[row], page_size=self.P, start=start)
        self.taken += pages

    def _forward(self, b, M: int, plan):
        """Hidden rows (final norm times output scale) of the ``M`` rows of ``b``."""
        e, cfg = self.eng, self.eng.cfg
        H, Lr, eps = e.H, cfg.num_layers, cfg.norm_eps
        ops.add_rmsnorm_fwd(emb=e.E, ids=b["ids"], T=M, S=M, w=e.pv[0]["attn_norm"], out_resid=b["x"], y=b["xn"],
                            rstd=b["rstd"], eps=eps, M=M, H=H)
        for l in range(Lr):
            pv, wv = e.pv[l], e.wv[l]
            ops.linear_fwd(b["xn"], wv["qkv_w"], b["qkv"])
            paged.kv_append(b["qkv"], pv["qkv_b"], self.cos, self.sin, b["slots"], b["positions"], b["q"], self.k[l],
                            self.v[l])
            paged.paged_attention(b["q"], self.k[l], self.v[l], b["attn"], plan)
            ops.linear_fwd(b["attn"], wv["o_w"], b["br"])
            ops.add_rmsnorm_fwd(x=b["x"], br=b["br"], w=pv["ffn_norm"], out_resid=b["mid"], y=b["xn"], rstd=b["rstd"],
                                eps=eps, M=M, H=H)
            if e.fused_swiglu:
                ops.gemm_swiglu_fwd(b["xn"], wv["gu_w"], b["gu"], b["h"])
            else:
                ops.linear_fwd(b["xn"], wv["gu_w"], b["gu"])
                ops.swiglu_fwd(b["gu"], b["h"], M=M, F=e.F)
            ops.linear_fwd(b["h"], wv["down_w"], b["br"])
            last = l + 1 == Lr
            ops.add_rmsnorm_fwd(x=b["mid"], br=b["br"], w=e.fnorm if last else e.pv[l + 1]["attn_norm"],
                                scale=e.oscale if last else None, out_resid=b["x"], y=b["xn"], rstd=b["rstd"], eps=eps,
                                M=M, H=H)
        return b["xn"]

    def _logits(self, rows: torch.Tensor) -> torch.Tensor:
        """fp32 logits [n, V] (a view of padded rows) of ``rows`` [n, H] hidden rows."""
        n, e = rows.shape[0], self.eng
        M = _pad(n, ROWS)
        a = torch.zeros(M, e.H, dtype=torch.bfloat16, device=self.dev)
        a[:n] = rows
        out = torch.empty(M, self.ldv, dtype=torch.float32, device=self.dev)
        ops.gemm(a, e.E16, out, M=M, N=e.V, K=e.H, ldc=self.ldv)
        return out[:n, :e.V]

    def _known(self, ids: Sequence[int]):
        """Refuses what is no token id: the embedding's rows are read without a bound."""
        for t in ids:
            if not 0 <= t < self.eng.V:
                raise ValueError(f"token id {t} outside the vocabulary of {self.eng.V}")

    @_on_its_device
    def prefill(self, ids: Sequence[int]) -> torch.Tensor:
        """Forward of a prompt into fresh pages; fp32 logits [1, V] of the token after it."""
        T = len(ids)
        if not 1 <= T <= self.max_prompt:
            raise ValueError(f"prompt of {T} tokens: 1 to {self.max_prompt}")
        self._known(ids)
        self.prompt_len = self.n = self.length = 0  # (the pages change from here on: a failure leaves no prompt to continue)
        e, M = self.eng, _pad(T, ROWS)
        b = self._buffers(M)
        b["ids"].zero_()
        b["ids"][:T] = torch.tensor(list(ids), dtype=torch.int32)
        self.taken = 0
        self.prefix = torch.full((1, self.prompt_pages), -1, dtype=torch.int32, device=self.dev)
        cu, total = self._ints(2), self._ints(1)
        self._tables(b, self._ints(1), torch.full_like(total, T), self.prefix, cu, total, None, -(-T // self.P), 0)
        plan = paged.AttentionPlan(M, 1, nh=e.nh, nkv=e.nkv, d=e.d, page_size=self.P, device=self.dev)
        plan.build(cu, total, self.prefix)
        hidden = self._forward(b, M, plan)
        self.prompt_len = T
        return self._logits(hidden[T - 1:T])

    @_on_its_device
    def branch(self, n: int):
        """n answers that continue the prompt; their tokens come with ``step``."""
        if not self.prompt_len:
            raise RuntimeError("prefill a prompt first")
        if not 1 <= n <= self.max_batch:
            raise ValueError(f"{n} answers: 1 to {self.max_batch}")
        e = self.eng
        self.n = self.length = 0  # (until the buffers below are those of n answers)
        self.taken = -(-self.prompt_len // self.P)
        self.tables = torch.full((n, self.answer_pages), -1, dtype=torch.int32, device=self.dev)
        self.cached, self.one = self._ints(n), torch.ones(n, dtype=torch.int32, device=self.dev)
        self.total, self.cu = self._ints(n), self._ints(n + 1)
        self.start = torch.full((n,), self.prompt_len, dtype=torch.int32, device=self.dev)
        self.group = (self.prefix, torch.full((1,), self.prompt_len, dtype=torch.int32, device=self.dev),
                      torch.tensor([0, n], dtype=torch.int32, device=self.dev))
        self.rows = _pad(n, ROWS)
        self.plan = paged.AttentionPlan(self.rows, n, 1, nh=e.nh, nkv=e.nkv, d=e.d, page_size=self.P, device=self.dev)
        self.n = n

    @_on_its_device
    def check(self):
        """Raises if the GPU could not do what the steps since ``prefill`` asked for; their logits are worth nothing then.
        Waits for the GPU: once at the end of an answer is enough. The library's error state is clear afterwards."""
        code, site = ops.device_error()
        if code:
            ops.clear_device_error()
            raise RuntimeError(f"generation failed on the GPU: error {code} at site {site}")
        refused = self.used[:self.length + 1, 1].amax().item()
        if refused:
            raise RuntimeError(f"generation failed on the GPU: page tables refused a step ({refused})")

    @_on_its_device
    def step(self, tokens: List[int]) -> torch.Tensor:
        """Adds ``tokens[i]`` to answer i; fp32 logits [n, V] of the tokens after them."""
        if len(tokens) != self.n or self.n == 0:
            raise ValueError(f"{len(tokens)} tokens for {self.n} answers")
        if self.length >= self.max_new:
            raise ValueError(f"answers have {self.max_new} tokens, the most there is room for")
        self._known(tokens)
        b = self._buffers(self.rows)
        b["ids"][:self.n] = torch.tensor(tokens, dtype=torch.int32)
        self._tables(b, self.cached, self.one, self.tables, self.cu, self.total, self.start,
                     self.n if self.length % self.P == 0 else 0, self.length + 1)
        self.plan.build(self.cu, self.total, self.tables, prefix=self.group)
        hidden = self._forward(b, self.rows, self.plan)
        self.cached.add_(self.one)
        self.length += 1
        return self._logits(hidden[:self.n])
