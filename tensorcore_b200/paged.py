"""Llama-shaped layers over the paged 4-bit cache: prompts and single tokens of several sequences in one step.

A step takes the hidden rows of some tokens of each sequence - a whole prompt, a piece of one, a single token, none - and runs, a
layer at a time and without a wait on the host,

    q, k, v = RMSNorm(x) Wq, Wk, Wv          tcx_raw_fused_rmsnorm_gemv_quantized
    turn q and k, append k and v             tcx_raw_kv_append (the rotary tables: tcx_raw_rope_table)
    a = attention(q, the sequence's cache)   tcx_raw_attention_paged
    x = x + a Wo                             tcx_raw_gemv_quantized
    x = x + (silu(g) u) Wdown,  g, u = RMSNorm(x) Wgate, Wup

`PageBook` hands out pages on the host; `python -m tensorcore_b200.paged` runs a batch of prompts and then tokens, the same
prompts token by token, and prints the times and how far the two are apart.  Weights are seeded numbers of the shapes of
`decode.LlamaShape`; torch supplies device memory, the residual sums and the activation.
"""
from __future__ import annotations

import argparse
from dataclasses import dataclass

import numpy as np

import tensorcore_b200 as tc
from tensorcore_b200 import decode as D


class OutOfPages(RuntimeError):
    """The free pages, or a sequence's row of the table, do not hold the tokens asked for."""


@dataclass
class Plan:
    positions: np.ndarray     # of each token of the step
    sequences: np.ndarray
    starts: np.ndarray        # where each sequence's tokens begin, and their number
    lengths: np.ndarray       # keys of each sequence with this step's


class PageBook:
    """Which pages of a cache belong to which of `slots` sequences, and how long those are."""

    def __init__(self, n_pages: int, page_tokens: int, slots: int, max_pages: int):
        self.page_tokens = page_tokens
        self.table = np.full((slots, max_pages), -1, np.int32)
        self.lengths = np.zeros(slots, np.int32)
        self._free = list(range(n_pages - 1, -1, -1))

    def free_pages(self) -> int:
        return len(self._free)

    def plan(self, counts) -> Plan:
        """Places for counts[s] more tokens of each sequence; all of them or, with OutOfPages, none."""
        counts = np.asarray(counts, np.int64)
        if counts.shape != self.lengths.shape or (counts < 0).any():
            raise ValueError("a number of tokens, zero or more, for every slot")
        lengths = self.lengths + counts
        have, need = -(-self.lengths // self.page_tokens), -(-lengths // self.page_tokens)
        if (need > self.table.shape[1]).any() or (need - have).sum() > len(self._free):
            raise OutOfPages(f"{int((need - have).sum())} pages asked for, {len(self._free)} free, {self.table.shape[1]} to a sequence")
        for s in np.nonzero(need > have)[0]:
            for i in range(have[s], need[s]):
                self.table[s, i] = self._free.pop()
        positions = np.concatenate([np.arange(a, b) for a, b in zip(self.lengths, lengths)]).astype(np.int32)
        sequences = np.repeat(np.arange(len(counts)), counts).astype(np.int32)
        self.lengths = lengths.astype(np.int32)
        return Plan(positions, sequences, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), self.lengths.copy())

    def release(self, slot: int) -> None:
        """The sequence is done: its pages are free, the slot empty."""
        used = -(-int(self.lengths[slot]) // self.page_tokens)
        self._free.extend(int(p) for p in self.table[slot, :used][::-1])
        self.table[slot] = -1
        self.lengths[slot] = 0


class PagedDecoder:
    """`slots` sequences over one cache of n_pages pages a layer; everything on torch's current device and stream."""

    def __init__(self, ctx: tc.Context, shape: D.LlamaShape, slots: int, n_pages: int, page_tokens: int = 64, max_pages: int | None = None, freq_base: float = 10000.0,
                 scaling: str = "plain", factor: float = 1.0, original_context: float = 0.0, layout: str = "half", fmt: int = 0):
        import torch
        self.torch, self.ctx, self.shape, self.fmt, self.layout = torch, ctx, shape, fmt, layout
        self.head_dim = shape.d_model // shape.n_heads
        max_pages = max_pages or n_pages
        self.book = PageBook(n_pages, page_tokens, slots, max_pages)
        self.kv = tc.kv_desc(n_pages, page_tokens, shape.n_kv_heads, self.head_dim)
        self.pages = torch.zeros((shape.n_layers, n_pages, tc.kv_page_bytes(self.kv)), dtype=torch.uint8, device="cuda")
        self.table_rows = max_pages * page_tokens
        self.cos, self.sin = (torch.empty((self.table_rows, self.head_dim // 2), dtype=torch.float32, device="cuda") for _ in range(2))
        tc.raw_rope_table(ctx, tc.rope_table_desc(self.table_rows, self.head_dim, freq_base=freq_base, scaling=scaling, factor=factor, original_context=original_context),
                          self.cos.data_ptr(), self.sin.data_ptr(), torch.cuda.current_stream().cuda_stream)
        self.weights = []
        for l in range(shape.n_layers):
            w = {p: D.quantize_into(ctx, D.device_weights_fp16(*shape.proj_shape(p), D.tensor_seed(l, t)), fmt) for t, p in enumerate(D.PROJ)}
            for i, n in enumerate(("attn_norm", "ffn_norm")):
                w[n] = torch.from_numpy(D.gamma_fp16(shape.d_model, 0x7CB000 + 0x1000 * i + l)).cuda()
            self.weights.append(w)

    def _project(self, x, which, w, gamma=None):
        N, K = self.shape.proj_shape(which)
        y = self.torch.empty((x.shape[0], N), dtype=self.torch.float16, device="cuda")
        stream = self.torch.cuda.current_stream().cuda_stream
        if gamma is None:
            tc.raw_gemv_quantized(self.ctx, x.data_ptr(), w[which].device_ptr(), y.data_ptr(), self.fmt, x.shape[0], N, K, cuda_stream=stream)
        else:
            tc.raw_fused_rmsnorm_gemv_quantized(self.ctx, x.data_ptr(), gamma.data_ptr(), w[which].device_ptr(), y.data_ptr(), self.fmt, x.shape[0], N, K, cuda_stream=stream)
        return y

    def step(self, x, counts):
        """x [tokens, d_model] fp16 on the GPU: counts[s] more tokens of each sequence, in the slots' order.  Returns their rows behind the last layer."""
        torch, s = self.torch, self.shape
        T = int(np.sum(counts))
        if x.shape != (T, s.d_model) or x.dtype != torch.float16 or not x.is_cuda:
            raise ValueError(f"fp16 rows [{T}, {s.d_model}] on the GPU")
        plan = self.book.plan(counts)
        if T == 0:
            return x
        x = x.contiguous()                       # the calls below take its address
        slots, max_pages = self.book.table.shape
        parts = (plan.positions, plan.sequences, plan.starts, plan.lengths, self.book.table)
        ints = torch.from_numpy(np.concatenate([p.reshape(-1) for p in parts])).cuda(non_blocking=True)      # one copy
        at, places = 0, []
        for p in parts:
            places.append(ints[at:].data_ptr())
            at += p.size
        positions, sequences, starts, lengths, table = places
        append = tc.kv_append_desc(T, slots, max_pages, q_heads=s.n_heads, layout=self.layout, rot_dim=self.head_dim, table_rows=self.table_rows)
        attend = tc.attention_paged_desc(T, slots, max_pages, s.n_heads, max_q=int(np.max(counts)))
        stream = torch.cuda.current_stream().cuda_stream
        a = torch.empty((T, s.d_model), dtype=torch.float16, device="cuda")
        for w, pages in zip(self.weights, self.pages):
            q, k, v = (self._project(x, p, w, w["attn_norm"]) for p in ("attn_q", "attn_k", "attn_v"))
            tc.raw_kv_append(self.ctx, self.kv, append, pages.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr(), q.data_ptr(), self.cos.data_ptr(), self.sin.data_ptr(),
                             positions, sequences, table, stream)
            tc.raw_attention_paged(self.ctx, self.kv, attend, pages.data_ptr(), q.data_ptr(), table, lengths, starts, a.data_ptr(), 0, stream)
            x = x + self._project(a, "attn_output", w)
            g, u = (self._project(x, p, w, w["ffn_norm"]) for p in ("ffn_gate", "ffn_up"))
            x = x + self._project(torch.nn.functional.silu(g).mul_(u), "ffn_down", w)
        return x

    def release(self, slot: int) -> None:
        self.book.release(slot)


def rows(n: int, d_model: int, seed: int):
    import torch
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((n, d_model)).astype(np.float16)).cuda()


def main(argv=None) -> int:
    import torch
    p = argparse.ArgumentParser(description="prompts, then single tokens, over the paged 4-bit cache")
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--slots", type=int, default=4)
    p.add_argument("--prompt", type=int, default=200)
    p.add_argument("--tokens", type=int, default=32)
    a = p.parse_args(argv)
    shape = D.LlamaShape("example", a.layers, 4096, 11008, 32, 8, 32000)
    lens = [max(1, a.prompt - 37 * i) for i in range(a.slots)]
    per = -(-(max(lens) + a.tokens) // 64)
    with tc.Context() as ctx:
        d = PagedDecoder(ctx, shape, a.slots, n_pages=per * a.slots, max_pages=per)
        xs = [rows(n + a.tokens, shape.d_model, i) for i, n in enumerate(lens)]

        def prompts():
            return d.step(torch.cat([x[:n] for x, n in zip(xs, lens)]), lens)

        def tokens(first, n):
            return [d.step(torch.stack([x[first[i] + t] for i, x in enumerate(xs)]), [1] * a.slots) for t in range(n)]
        out = {}
        for what in ("warm up", "timed"):
            for s in range(a.slots):
                d.release(s)
            ev = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
            ev[0].record()
            last = prompts()
            ev[1].record()
            got = tokens(lens, a.tokens)
            ev[2].record()
            torch.cuda.synchronize()
            out = {"prompts_ms": ev[0].elapsed_time(ev[1]), "token_ms": ev[1].elapsed_time(ev[2]) / max(1, a.tokens)}
        # the shortest prompt once more, token by token
        s = int(np.argmin(lens))
        at = int(np.sum(lens[:s]))
        d.release(s)
        one = [0] * a.slots
        one[s] = 1
        by_one = torch.cat([d.step(xs[s][t:t + 1], one) for t in range(lens[s])])
        apart = ((by_one - last[at:at + lens[s]]).float().norm() / (last[at:at + lens[s]] - xs[s][:lens[s]]).float().norm()).item()
        err = tc.take_device_error(ctx)
    print(f"{a.slots} prompts, {sum(lens)} tokens, {a.layers} layers: {out['prompts_ms']:.2f} ms; a token of each: {out['token_ms']:.3f} ms; cache {d.pages.nbytes / 2**20:.0f} MiB; "
          f"prompt at once and token by token: {apart:.1e} of what the layers add; finite {bool(torch.isfinite(got[-1]).all()) if got else True}; device error {err}")
    return 0 if err == 0 else 1


if __name__ == "__main__":
    raise SystemExit(main())
