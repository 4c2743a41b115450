"""Serving from a paged KV cache: pages shared and copied on write, steps that mix
pieces of prompts with decoding sequences, and sampling.

The reference serves one sequence from one contiguous cache
(python/kudacuda_static_decode.py:80-147) and takes the argmax of its logits.
Here a :class:`PagedKVCache` hands out pages of a pool to any number of
sequences, a :class:`PagedGenerator` runs a ragged batch of new tokens through
the model - the batched path's NF4 GEMMs, ``rope_append_paged``,
``paged_attention`` - and draws every sequence's next token with ``sample``.

    python -m kudacuda_b200.paged_serving --random --prompt-ids 1,2,3 --answers 4 --temperature 0.8 --json
"""

from __future__ import annotations

import argparse
import contextlib
import heapq
import json
import math
import random
import sys
import time
from dataclasses import dataclass, field
from typing import Any, Mapping, Optional, Sequence

from .decode_engine import ModelWeights, retile_nf4
from .kudacuda_sidecar import KudaCudaBridge, NativeCudaError

MAX_ROWS = 64  # new tokens of a step: the batched GEMM's columns


class PagedCacheFull(RuntimeError):
    """The pool has no page left; nothing was changed."""


@dataclass
class PagedSequence:
    pages: list[int] = field(default_factory=list)
    length: int = 0  # tokens whose keys are (or, within a step, are about to be) in the cache


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` tokens for every layer: K and V tensors
    [layers, num_pages, kv_heads, page_size, head_dim], a free list and a
    reference count a page.  A fork shares its parent's pages; a page that is
    shared and only partly filled is copied when one of its owners grows into it.
    Copies and moves run on the given stream through ``bridge``."""

    def __init__(self, bridge: Any, *, layers: int, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: Any = None, device: Any = "cuda:0", torch_module: Any = None) -> None:
        if torch_module is None:
            import torch as torch_module
        if page_size not in (16, 32, 64, 128):
            raise ValueError("page_size must be 16, 32, 64 or 128")
        if num_pages < 1 or layers < 1:
            raise ValueError("a cache needs layers and pages")
        self.torch, self.bridge, self.device = torch_module, bridge, device
        self.page_size, self.num_pages = int(page_size), int(num_pages)
        dtype = dtype if dtype is not None else torch_module.bfloat16
        shape = (int(layers), self.num_pages, int(kv_heads), self.page_size, int(head_dim))
        self.k = torch_module.zeros(shape, dtype=dtype, device=device)
        self.v = torch_module.zeros(shape, dtype=dtype, device=device)
        self._free = list(range(self.num_pages))  # a heap: the lowest page first
        self._refs = [0] * self.num_pages

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def _copy(self, pairs: list[tuple[int, int]], stream_ptr: int, block_table: Any = None) -> None:
        """Copies the pages and, with ``block_table``, points its entries at the copies."""

        torch = self.torch
        # The lists are dropped once the copy is launched: memory of its own stream is not handed out
        # to anyone who would write it earlier.
        on_stream = contextlib.nullcontext()
        if torch.device(self.device).type == "cuda":
            on_stream = torch.cuda.stream(torch.cuda.ExternalStream(stream_ptr, device=self.device))
        with on_stream:
            i32 = dict(dtype=torch.int32, device=self.device)
            tables = {}
            if block_table is not None:
                page_map = list(range(self.num_pages))
                for old, new in pairs:
                    page_map[old] = new
                tables = {"block_table": block_table, "page_map": torch.tensor(page_map, **i32)}
            self.bridge.dispatch_kv_pages_copy(self.k, self.v, torch.tensor(pairs, **i32).view(-1, 2),
                                               stream_ptr=stream_ptr, **tables)

    def reserve(self, growth: Sequence[tuple[PagedSequence, int]], stream_ptr: int) -> None:
        """Room for each sequence's new tokens, whose lengths grow by them; all of them or none."""

        if len({id(seq) for seq, _ in growth}) != len(growth):
            raise ValueError("a sequence grows once in a step: its tokens come together")
        need, copies, owners = 0, [], {}
        for seq, tokens in growth:
            if tokens < 0:
                raise ValueError("a sequence grows by zero or more tokens")
            need += -(-(seq.length + tokens) // self.page_size) - len(seq.pages)
            if tokens > 0 and seq.length % self.page_size != 0:
                old = seq.pages[-1]
                owners[old] = owners.get(old, self._refs[old])
                if owners[old] > 1:  # (the last owner keeps the original)
                    owners[old] -= 1
                    copies.append(seq)
                    need += 1
        if need > len(self._free):
            raise PagedCacheFull(f"{need} pages are needed, {len(self._free)} are free")
        pairs = [(seq.pages[-1], self._take()) for seq in copies]
        if pairs:
            try:
                self._copy(pairs, stream_ptr)
            except BaseException:
                for _, new in pairs:
                    self._drop(new)
                raise
        for seq, (old, new) in zip(copies, pairs):
            seq.pages[-1] = new
            self._refs[old] -= 1
        for seq, tokens in growth:
            seq.length += tokens
            while len(seq.pages) * self.page_size < seq.length:
                seq.pages.append(self._take())

    def fork(self, seq: PagedSequence) -> PagedSequence:
        """Another sequence with the same tokens; no page is copied yet."""

        for page in seq.pages:
            self._refs[page] += 1
        return PagedSequence(list(seq.pages), seq.length)

    def truncate(self, seq: PagedSequence, length: int) -> None:
        """Forget the tokens from ``length`` on."""

        if not 0 <= length <= seq.length:
            raise ValueError("a sequence is cut to a length it has")
        keep = -(-length // self.page_size)
        for page in seq.pages[keep:]:
            self._drop(page)
        del seq.pages[keep:]
        seq.length = length

    def free(self, seq: PagedSequence) -> None:
        self.truncate(seq, 0)

    def compact(self, sequences: Sequence[PagedSequence], stream_ptr: int, block_table: Any = None) -> int:
        """Move every page in use below the number of pages in use; ``sequences`` are all of the cache's
        (a fork's pages are moved once), ``block_table`` a device table to rewrite too.  Returns the
        number of pages moved."""

        used = [p for p in range(self.num_pages) if self._refs[p] > 0]
        sequences = list({id(s): s for s in sequences}.values())
        owners = [0] * self.num_pages
        for s in sequences:
            for p in s.pages:
                owners[p] += 1
        if owners != self._refs:  # (a fork left out would keep pages that have moved)
            raise ValueError("compact needs all of the cache's sequences")
        low = [p for p in range(len(used)) if self._refs[p] == 0]
        pairs = list(zip([p for p in used if p >= len(used)], low))
        if not pairs:
            return 0
        to = dict(pairs)
        self._copy(pairs, stream_ptr, block_table)
        for seq in sequences:
            seq.pages = [to.get(p, p) for p in seq.pages]
        for old, new in pairs:
            self._refs[new], self._refs[old] = self._refs[old], 0
        self._free = [p for p in range(self.num_pages) if self._refs[p] == 0]
        return len(pairs)

    def table(self, sequences: Sequence[PagedSequence]) -> list[list[int]]:
        """Block-table rows, -1 past a sequence's pages."""

        width = max([len(s.pages) for s in sequences] + [1])
        return [s.pages + [-1] * (width - len(s.pages)) for s in sequences]


def paged_rope_tables(max_pos: int, rotary_dim: int, theta: float, scaling: Optional[Mapping[str, Any]] = None,
                      *, device: Any = "cpu", torch_module: Any = None) -> tuple[Any, Any]:
    """cos and sin, float32 [max_pos, rotary_dim / 2], computed in 64 bits.

    ``scaling["type"]`` (contexts longer than the model was trained for, by ``factor``):
    "linear" divides every frequency; "ntk" raises theta by factor^(d / (d - 2)); "llama3" divides the
    frequencies whose wavelength exceeds ``original`` / ``low_freq_factor`` tokens, keeps those below
    ``original`` / ``high_freq_factor`` and interpolates between; "yarn" interpolates between dividing and
    keeping over the pairs that turn ``beta_slow`` to ``beta_fast`` times within ``original`` tokens, and
    multiplies cos and sin by 0.1 ln(factor) + 1."""

    if torch_module is None:
        import torch as torch_module
    torch = torch_module
    d = int(rotary_dim)
    if d < 2 or d % 2:
        raise ValueError("rotary_dim must be even")
    kind = (scaling or {}).get("type", "none")
    factor = float((scaling or {}).get("factor", 1.0))
    if kind == "ntk":
        theta = theta * factor ** (d / (d - 2))
    inv = theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    gain = 1.0
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = float(scaling["original"]) * inv / (2 * math.pi)  # within the original context
        share = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        inv = inv / factor * (1 - share) + inv * share
    elif kind == "yarn":
        original = float(scaling["original"])
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

        def pair_of(turns: float) -> float:
            return d * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

        first, last = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), d - 1)
        ramp = ((torch.arange(d // 2, dtype=torch.float64) - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        inv = inv / factor * ramp + inv * (1 - ramp)
        gain = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif kind not in ("none", "ntk"):
        raise ValueError(f"unknown rope scaling {kind!r}")
    angle = torch.arange(int(max_pos), dtype=torch.float64)[:, None] * inv
    return ((angle.cos() * gain).float().contiguous().to(device), (angle.sin() * gain).float().contiguous().to(device))


@dataclass(frozen=True)
class Sampling:
    """How a sequence's next token is drawn; the defaults take the most likely one."""

    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0


class PagedGenerator:
    """Steps of a model over a :class:`PagedKVCache`: each takes up to 64 new tokens of any
    sequences - pieces of prompts and single tokens alike - and returns one drawn token per sequence."""

    def __init__(self, bridge: KudaCudaBridge, weights: ModelWeights, *, num_pages: int, page_size: int = 64,
                 max_position: int = 8192, rope_scaling: Optional[Mapping[str, Any]] = None, device: Any = "cuda:0",
                 torch_module: Any = None) -> None:
        if torch_module is None:
            import torch as torch_module
        self.torch = torch = torch_module
        self.bridge, self.weights, self.device = bridge, weights, device
        self.config = c = weights.config
        self.cache = PagedKVCache(bridge, layers=c.layers, num_pages=num_pages, kv_heads=c.kv_heads,
                                  head_dim=c.head_dim, page_size=page_size, device=device, torch_module=torch)
        sp = int(torch.cuda.current_stream(device).cuda_stream)
        self.qkv = [retile_nf4(bridge, torch, [L.q, L.k, L.v], sp) for L in weights.layers]
        self.gu = [retile_nf4(bridge, torch, [L.gate, L.up], sp) for L in weights.layers]
        self.o = [retile_nf4(bridge, torch, [L.o], sp) for L in weights.layers]
        self.down = [retile_nf4(bridge, torch, [L.down], sp) for L in weights.layers]
        self.lm = retile_nf4(bridge, torch, [weights.lm_head], sp) if weights.lm_head is not None else None
        self.vocab = self.lm.rows if self.lm is not None else c.vocab
        self.bias = [torch.cat([L.q_bias, L.k_bias, L.v_bias]) if L.q_bias is not None else None
                     for L in weights.layers]
        self.cos, self.sin = paged_rope_tables(max_position, c.head_dim, c.rope_theta, rope_scaling, device=device,
                                               torch_module=torch)
        bf16, f32, R = torch.bfloat16, torch.float32, MAX_ROWS
        ks = bridge.batch_gemm_ksplit
        self.ks_qkv, self.ks_o = ks(self.qkv[0].rows, c.hidden), ks(c.hidden, self.o[0].k)
        self.ks_gu, self.ks_dn = ks(2 * c.intermediate, c.hidden), ks(c.hidden, c.intermediate)
        self.ks_lm = ks(self.vocab, c.hidden)
        rows = max(self.ks_qkv * self.qkv[0].rows, self.ks_o * c.hidden, self.ks_gu * 2 * c.intermediate,
                   self.ks_dn * c.hidden, self.ks_lm * self.vocab)
        self.partials = torch.empty(rows * R, dtype=f32, device=device)
        self.x = torch.zeros((R, c.hidden), dtype=bf16, device=device)
        self.xn = torch.zeros((R, c.hidden), dtype=bf16, device=device)
        self.qkv_out = torch.zeros((R, self.qkv[0].rows), dtype=bf16, device=device)
        self.q = torch.zeros((R, c.q_heads, c.head_dim), dtype=bf16, device=device)
        self.attn = torch.zeros((R, c.q_heads, c.head_dim), dtype=bf16, device=device)
        self.h = torch.zeros((R, c.intermediate), dtype=bf16, device=device)
        self.logits = torch.zeros((R, self.vocab), dtype=bf16, device=device)
        self.tokens = torch.zeros((R,), dtype=torch.int32, device=device)
        self.logprobs = torch.zeros((R,), dtype=f32, device=device)
        # one workspace for steps of single tokens and of longer pieces
        widest = torch.empty((1, num_pages), dtype=torch.int32, device=device)
        self.workspace = max((bridge.paged_attention_workspace(self.q, self.cache.k[0], widest, max_query=m)
                              for m in (1, R)), key=lambda t: t.nbytes)
        torch.cuda.synchronize(device)

    @staticmethod
    def _n_pad(rows: int) -> int:
        return 16 if rows <= 16 else 32 if rows <= 32 else 64

    def _rows(self, lin: Any, x: Any, ksplit: int, out: Any, rows: int, sp: int, weight_type: int = 2,
              weight: Any = None, k: Optional[int] = None) -> None:
        """out[:rows] = the projection of x's rows, bf16 (the GEMM's splits summed onto zeros)."""

        n_pad = self._n_pad(rows)
        n, kk = out.shape[1], lin.k if lin is not None else k
        self.bridge.dispatch_batch_gemm(lin.data if lin is not None else weight, None, x[:n_pad], self.partials,
                                        weight_type=weight_type, rows=n, k=kk, n_pad=n_pad, ksplit=ksplit,
                                        stream_ptr=sp)
        out[:rows].zero_()
        self.bridge.dispatch_batch_residual(self.partials, out, ksplit=ksplit, rows=n, n_pad=n_pad, batch=rows,
                                            stream_ptr=sp)

    def _residual(self, lin: Any, x: Any, ksplit: int, rows: int, sp: int) -> None:
        n_pad = self._n_pad(rows)
        self.bridge.dispatch_batch_gemm(lin.data, None, x[:n_pad], self.partials, weight_type=2, rows=lin.rows,
                                        k=lin.k, n_pad=n_pad, ksplit=ksplit, stream_ptr=sp)
        self.bridge.dispatch_batch_residual(self.partials, self.x, ksplit=ksplit, rows=lin.rows, n_pad=n_pad,
                                            batch=rows, stream_ptr=sp)

    def step(self, entries: Sequence[tuple[PagedSequence, Sequence[int]]], sampling: Sequence[Sampling],
             uniform: Sequence[float], stream: Any = None) -> tuple[list[int], list[float]]:
        """Append each entry's tokens to its sequence and draw the token after its last one.

        ``sampling`` and ``uniform`` (numbers in [0, 1)) have one element per entry.  Returns the drawn
        tokens and their log-probabilities in the distribution they were drawn from.  A step that raises
        leaves the sequences at the lengths that they had."""

        torch = self.torch
        rows = sum(len(t) for _, t in entries)
        if not entries or any(len(t) == 0 for _, t in entries) or rows > MAX_ROWS:
            raise ValueError(f"a step takes 1 to {MAX_ROWS} tokens, at least one of each of its sequences")
        if len(sampling) != len(entries) or len(uniform) != len(entries):
            raise ValueError("one sampling setting and one uniform number per entry")
        if any(s.length + len(t) > self.cos.shape[0] for s, t in entries):
            raise ValueError("a sequence grows past max_position")
        stream = stream if stream is not None else torch.cuda.current_stream(self.device)
        sp = int(stream.cuda_stream)
        before = [s.length for s, _ in entries]
        with torch.cuda.stream(stream):
            self.cache.reserve([(s, len(t)) for s, t in entries], sp)
        try:
            return self._run(entries, sampling, uniform, stream)
        except BaseException:
            with contextlib.suppress(Exception):  # what was launched ends before its pages are given back
                stream.synchronize()
            for (s, _), length in zip(entries, before):
                self.cache.truncate(s, length)
            raise

    def _run(self, entries: Sequence[tuple[PagedSequence, Sequence[int]]], sampling: Sequence[Sampling],
             uniform: Sequence[float], stream: Any) -> tuple[list[int], list[float]]:
        """The step's work, the sequences grown by their tokens."""

        torch, br, c, w = self.torch, self.bridge, self.config, self.weights
        rows, sp = sum(len(t) for _, t in entries), int(stream.cuda_stream)
        with torch.cuda.stream(stream):
            i32 = dict(dtype=torch.int32, device=self.device)
            flat = [tok for _, t in entries for tok in t]
            state = torch.tensor([[tok, 0, 0, 0] for tok in flat], **i32)
            ends = [0]
            for _, t in entries:
                ends.append(ends[-1] + len(t))
            start = torch.tensor(ends, **i32)
            kv_len = torch.tensor([s.length for s, _ in entries], **i32)
            table = torch.tensor(self.cache.table([s for s, _ in entries]), **i32)
            longest = max(len(t) for _, t in entries)
            q, attn, qkv = self.q[:rows], self.attn[:rows], self.qkv_out[:rows]
            br.dispatch_batch_embedding(w.embedding, state, self.x, batch=rows, hidden=c.hidden, vocab=c.vocab,
                                        stream_ptr=sp)
            for i, L in enumerate(w.layers):
                br.dispatch_batch_rmsnorm(self.x, L.in_norm, self.xn, batch=rows, hidden=c.hidden, epsilon=c.eps,
                                          stream_ptr=sp)
                self._rows(self.qkv[i], self.xn, self.ks_qkv, self.qkv_out, rows, sp)
                br.dispatch_rope_append_paged(qkv, q, self.cache.k[i], self.cache.v[i], self.cos, self.sin, start,
                                              kv_len, table, bias=self.bias[i], stream_ptr=sp)
                br.dispatch_paged_attention(q, self.cache.k[i], self.cache.v[i], attn, start, kv_len, table,
                                            self.workspace, max_query=longest, stream_ptr=sp)
                self._residual(self.o[i], self.attn.view(MAX_ROWS, -1), self.ks_o, rows, sp)
                br.dispatch_batch_rmsnorm(self.x, L.post_norm, self.xn, batch=rows, hidden=c.hidden, epsilon=c.eps,
                                          stream_ptr=sp)
                n_pad = self._n_pad(rows)
                br.dispatch_batch_gemm(self.gu[i].data, None, self.xn[:n_pad], self.partials, weight_type=2,
                                       rows=self.gu[i].rows, k=self.gu[i].k, n_pad=n_pad, ksplit=self.ks_gu,
                                       stream_ptr=sp)
                br.dispatch_batch_swiglu(self.partials, self.h, ksplit=self.ks_gu, intermediate=c.intermediate,
                                         n_pad=n_pad, batch=rows, stream_ptr=sp)
                self._residual(self.down[i], self.h, self.ks_dn, rows, sp)
            # the last row of every entry
            n = len(entries)
            last = self.x.index_select(0, start[1:].long() - 1).contiguous()
            br.dispatch_batch_rmsnorm(last, w.final_norm, self.xn, batch=n, hidden=c.hidden, epsilon=c.eps,
                                      stream_ptr=sp)
            if self.lm is not None:
                self._rows(self.lm, self.xn, self.ks_lm, self.logits, n, sp)
            else:
                self._rows(None, self.xn, self.ks_lm, self.logits, n, sp, weight_type=1, weight=w.embedding,
                           k=c.hidden)
            f32 = dict(dtype=torch.float32, device=self.device)
            br.dispatch_sample(self.logits[:n], self.tokens[:n], torch.tensor(list(uniform), **f32),
                               temperature=torch.tensor([s.temperature for s in sampling], **f32),
                               top_k=torch.tensor([s.top_k for s in sampling], **i32),
                               top_p=torch.tensor([s.top_p for s in sampling], **f32),
                               min_p=torch.tensor([s.min_p for s in sampling], **f32), logprobs=self.logprobs[:n],
                               stream_ptr=sp)
            tokens, logprobs = self.tokens[:n].tolist(), self.logprobs[:n].tolist()
        word = br.error_word(clear=True)
        if word:
            raise NativeCudaError(f"paged step raised device error word {word:#x}")
        return tokens, logprobs

    def _most_pages(self, prompt: int, new_tokens: int, answers: int) -> int:
        """Pages of a prompt and its answers when all are finished: the first answer has all of its own, the
        others share the whole pages before the prompt's last token.  (The last token drawn is not fed.)"""

        size = self.cache.page_size
        whole = -(-(prompt + new_tokens - 1) // size)
        return whole + (answers - 1) * (whole - (prompt - 1) // size)

    def generate(self, prompts: Sequence[Sequence[int]], new_tokens: int, sampling: Sampling = Sampling(), *,
                 answers: int = 1, seed: int = 0, stream: Any = None) -> list[list[list[int]]]:
        """``answers`` continuations of every prompt: each prompt is fed once, in pieces that share steps with
        the sequences that already decode, and then forked.  A prompt waits until the pages that it and its
        answers will need are free.  Returns tokens [prompt][answer]."""

        if new_tokens < 1 or answers < 1 or any(len(p) == 0 for p in prompts):
            raise ValueError("prompts have tokens, and at least one new token and one answer are asked for")
        if answers > MAX_ROWS:
            raise ValueError(f"at most {MAX_ROWS} answers of a prompt")
        rng = random.Random(seed)
        waiting = [(i, PagedSequence(), list(p)) for i, p in enumerate(prompts)][::-1]  # the next one last
        decoding: list[tuple[int, list[int], PagedSequence]] = []
        out: list[list[list[int]]] = [[] for _ in prompts]
        live: list[PagedSequence] = []
        budget = self.cache.free_pages
        claims: dict[int, int] = {}  # pages of the prompts that have begun, at their most
        unfinished = [answers] * len(prompts)

        def done(i: int, seq: PagedSequence) -> None:
            self.cache.free(seq)
            live.remove(seq)
            unfinished[i] -= 1
            if unfinished[i] == 0:
                del claims[i]

        try:
            while waiting or decoding:
                room = MAX_ROWS
                batch: list[tuple[Any, PagedSequence, list[int]]] = []
                for _, got, seq in decoding[:room]:
                    batch.append((got, seq, [got[-1]]))
                room -= len(batch)
                fed = []
                while waiting and room > 0:
                    i, seq, left = waiting[-1]
                    if i not in claims:
                        pages = self._most_pages(len(left), new_tokens, answers)
                        if claims and sum(claims.values()) + pages > budget:
                            break
                        claims[i] = pages
                        live.append(seq)
                    waiting.pop()
                    batch.append((i, seq, left[:room]))
                    room -= len(left[:room])
                    fed.append((i, seq, left[len(batch[-1][2]):]))
                draws = [(sampling, rng.random()) for _ in batch]
                tokens, _ = self.step([(s, t) for _, s, t in batch], [d[0] for d in draws], [d[1] for d in draws],
                                      stream)
                still = []
                for (i, got, seq), token in zip(decoding[:MAX_ROWS], tokens):
                    got.append(token)
                    if len(got) < new_tokens:
                        still.append((i, got, seq))
                    else:
                        done(i, seq)
                decoding = decoding[MAX_ROWS:] + still
                for (i, seq, left), token in zip(fed, tokens[len(batch) - len(fed):]):
                    if left:
                        waiting.append((i, seq, left))
                        continue
                    # the prompt is in the cache: one answer goes on from the token drawn with it, the others
                    # feed its last token again from a shorter fork and draw their own
                    owners = [seq] + [self.cache.fork(seq) for _ in range(answers - 1)]
                    live.extend(owners[1:])
                    firsts = [token]
                    if answers > 1:
                        for fork in owners[1:]:
                            self.cache.truncate(fork, fork.length - 1)
                        more, _ = self.step([(f, [prompts[i][-1]]) for f in owners[1:]], [sampling] * (answers - 1),
                                            [rng.random() for _ in owners[1:]], stream)
                        firsts += more
                    for owner, first in zip(owners, firsts):
                        got = [first]
                        out[i].append(got)
                        if new_tokens > 1:
                            decoding.append((i, got, owner))
                        else:
                            done(i, owner)
        finally:
            for seq in live:
                self.cache.free(seq)
        return out


def main(argv: Optional[Sequence[str]] = None) -> int:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--random", action="store_true", required=True, help="Qwen2.5-3B architecture, random-init weights")
    p.add_argument("--prompt-ids", action="append", required=True, help="comma-separated token ids; may be repeated")
    p.add_argument("--new-tokens", type=int, default=32)
    p.add_argument("--answers", type=int, default=1, help="continuations of every prompt, from one copy of it")
    p.add_argument("--temperature", type=float, default=0.0)
    p.add_argument("--top-k", type=int, default=0)
    p.add_argument("--top-p", type=float, default=1.0)
    p.add_argument("--min-p", type=float, default=0.0)
    p.add_argument("--num-pages", type=int, default=512)
    p.add_argument("--page-size", type=int, default=64)
    p.add_argument("--layers", type=int, default=36)
    p.add_argument("--device", default="cuda:0")
    p.add_argument("--seed", type=int, default=20260824)
    p.add_argument("--json", action="store_true")
    args = p.parse_args(argv)
    from dataclasses import replace

    import torch

    from .decode_engine import QWEN25_3B, random_weights

    torch.cuda.set_device(torch.device(args.device))
    with KudaCudaBridge(device_id=torch.device(args.device).index or 0) as bridge:
        weights = random_weights(bridge, replace(QWEN25_3B, layers=args.layers), seed=args.seed, device=args.device)
        gen = PagedGenerator(bridge, weights, num_pages=args.num_pages, page_size=args.page_size, device=args.device)
        prompts = [[int(v) for v in ids.split(",") if v.strip()] for ids in args.prompt_ids]
        t0 = time.perf_counter()
        out = gen.generate(prompts, args.new_tokens, Sampling(args.temperature, args.top_k, args.top_p, args.min_p),
                           answers=args.answers, seed=args.seed)
        stats = {"seconds": time.perf_counter() - t0, "free_pages": gen.cache.free_pages}
    print(json.dumps({"tokens": out, **stats}) if args.json else f"{out}\n{stats}", flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
