"""The paged 4-bit KV cache (fmd_pkv_*) and greedy generation over it.

A ``PagedKvCache`` is a pool of pages of 64 tokens that sequences of any length
share; keys and values are held in 4 bits (4.25 with their scales), a quarter of
what ``KvCache`` takes.  Sequences are numbers: ``open`` makes one, ``fork``
another with the same tokens (shared pages, copied when written to), ``free``
gives its pages back.  With ``window`` a query sees the last ``window`` tokens
and the first ``sinks`` ones.

``step`` runs the decoder over new tokens of several sequences at once -- whole
prompts, pieces of prompts, single tokens; ``generate_paged`` is the greedy loop
of ``Engine::generate_batch`` (engine.rs:493-541) on it, with each token's log
probability.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import Sequence

import numpy as np

from .decoder import DEFAULT_EOS, FinishReason, FmdError, Qwen3, _as_src, _check, _data_ptr, _ptr, lib

PAGE_TOKENS = 64


def _i32(x) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(x, dtype=np.int32).reshape(-1))


class _Pool:
    """The pool's device memory for torch.as_tensor (which keeps this object)."""

    def __init__(self, cache, ptr, shape):
        self.cache = cache
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "|u1", "data": (ptr, False),
                                         "version": 2, "strides": None}


class PagedKvCache:
    """All layers' K/V in pages of 64 tokens and 4 bits a value."""

    def __init__(self, model: Qwen3, pages: int, max_seqs: int, max_rows: int, window: int = 0,
                 sinks: int = 0):
        self.model = model
        self.max_seqs, self.max_rows, self.window, self.sinks = max_seqs, max_rows, window, sinks
        h = ctypes.c_void_p()
        _check(lib().fmd_pkv_create(model.handle, pages, max_seqs, max_rows, window, sinks,
                                    ctypes.byref(h)))
        self.handle = h
        self.num_pages = pages

    def __del__(self):
        if getattr(self, "handle", None):
            lib().fmd_pkv_destroy(self.handle)
            self.handle = None

    @staticmethod
    def bytes(model: Qwen3, pages: int) -> int:
        return int(lib().fmd_pkv_bytes(model.handle, pages))

    # -- sequences -----------------------------------------------------------
    def _new(self, fn, *args) -> int:
        out = ctypes.c_int32()
        _check(fn(self.handle, *args, ctypes.byref(out)))
        return out.value

    def open(self) -> int:
        return self._new(lib().fmd_pkv_open)

    def fork(self, seq: int) -> int:
        """A new sequence on the same pages."""
        return self._new(lib().fmd_pkv_fork, seq)

    def copy(self, seq: int) -> int:
        """A new sequence on copies of the pages."""
        return self._new(lib().fmd_pkv_copy, seq)

    def free(self, seq: int) -> None:
        _check(lib().fmd_pkv_free(self.handle, seq))

    def truncate(self, seq: int, length: int) -> None:
        _check(lib().fmd_pkv_truncate(self.handle, seq, length))

    def resize(self, pages: int) -> None:
        """Compact the pages in use into a pool of `pages` pages."""
        _check(lib().fmd_pkv_resize(self.handle, pages))
        self.num_pages = pages

    def len(self, seq: int) -> int:
        n = lib().fmd_pkv_len(self.handle, seq)
        if n < 0:
            _check(-1)
        return n

    def free_pages(self) -> int:
        return lib().fmd_pkv_free_pages(self.handle)

    def pages(self, seq: int) -> list[int]:
        """The sequence's page ids, -1 where a page behind the window was given back."""
        n = ctypes.c_int32()
        _check(lib().fmd_pkv_pages(self.handle, seq, None, 0, ctypes.byref(n)))
        out = np.empty(max(n.value, 1), dtype=np.int32)
        _check(lib().fmd_pkv_pages(self.handle, seq, _ptr(out), n.value, ctypes.byref(n)))
        return out[: n.value].tolist()

    def pool(self):
        """The pool as a uint8 device tensor (layers, pages, bytes of a page);
        ``resize`` moves the pool, and the tensor is then no longer it."""
        import torch

        ptr, size = ctypes.c_void_p(), ctypes.c_size_t()
        _check(lib().fmd_pkv_pool(self.handle, ctypes.byref(ptr), ctypes.byref(size)))
        layers = self.model.cfg.num_hidden_layers
        shape = (layers, self.num_pages, size.value // (layers * self.num_pages))
        return torch.as_tensor(_Pool(self, ptr.value, shape), device=torch.device("cuda", self.model.device))

    # -- a plan and what runs on it (device pointers) --------------------------
    def plan(self, seqs: Sequence[int], counts: Sequence[int]) -> None:
        """counts[i] new tokens for sequence seqs[i]."""
        s, c = _i32(seqs), _i32(counts)
        if s.size != c.size:
            raise FmdError(-1, "one count per sequence")
        _check(lib().fmd_pkv_plan(self.handle, s.size, _ptr(s), _ptr(c)))

    def append(self, layer: int, qkv_ptr: int, q_ptr: int) -> None:
        """q/k norm and rotation of the raw projection's rows: q out, K and V into the pages."""
        _check(lib().fmd_op_pkv_append(self.model.handle, self.handle, layer, qkv_ptr, q_ptr))

    def write(self, layer: int, k_ptr: int, v_ptr: int) -> None:
        """K (rotated) and V rows (rows, kv_heads, 128) into the pages."""
        _check(lib().fmd_op_pkv_write(self.model.handle, self.handle, layer, k_ptr, v_ptr))

    def read(self, layer: int, k_ptr: int | None, v_ptr: int | None) -> None:
        """The plan's K and V rows as the values they stand for."""
        _check(lib().fmd_op_pkv_read(self.model.handle, self.handle, layer, k_ptr, v_ptr))

    def attention(self, layer: int, q_ptr: int, ctx_ptr: int) -> None:
        """Context of the plan's rows over everything they see."""
        _check(lib().fmd_op_pkv_attention(self.model.handle, self.handle, layer, q_ptr, ctx_ptr))

    def copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Page src[i] to page dst[i] in every layer."""
        s, t = _i32(src), _i32(dst)
        if s.size != t.size:
            raise FmdError(-1, "one destination per source")
        _check(lib().fmd_op_pkv_copy_pages(self.handle, s.size, _ptr(s), _ptr(t)))

    # -- the decoder -----------------------------------------------------------
    def step(self, seqs: Sequence[int], tokens: Sequence[Sequence[int]] | None = None, embeds=None,
             counts: Sequence[int] | None = None, logits: bool = True) -> np.ndarray | None:
        """Run the decoder over new tokens: ``tokens[i]`` of sequence seqs[i], or
        ``embeds`` (all rows, hidden; numpy storage or a torch tensor in the
        activation dtype) with ``counts``.  Returns f32 logits (n, vocab) of each
        sequence's last token (None with ``logits=False``; they stay on the
        device for ``logprobs`` and ``greedy``)."""
        m, s = self.model, _i32(seqs)
        if (tokens is None) == (embeds is None):
            raise FmdError(-1, "a step takes tokens or embeds")
        ids, keep, on_dev = None, None, 0
        if tokens is not None:
            c = _i32([len(t) for t in tokens])
            ids = (np.ascontiguousarray(np.concatenate([np.asarray(t, dtype=np.uint32).reshape(-1)
                                                        for t in tokens])) if len(tokens) else None)
        else:
            if counts is None:
                raise FmdError(-1, "embeds need counts")
            c = _i32(counts)
            code, on_dev, shape, keep = _as_src(embeds)
            if code != {"f32": 0, "f16": 1, "bf16": 2}[m.precision.activation_dtype()]:
                raise FmdError(-1, "embeds must be in the activation dtype")
            if shape != (int(c.sum()), m.cfg.hidden_size):
                raise FmdError(-1, "embeds must be (all rows, hidden)")
        if c.size != s.size:
            raise FmdError(-1, "one token list or count per sequence")
        out = np.empty((s.size, m.cfg.vocab_size), dtype=np.float32) if logits else None
        _check(lib().fmd_dec_step(m.handle, self.handle, s.size, _ptr(s), _ptr(c), _ptr(ids),
                                  None if keep is None else _data_ptr(keep), on_dev, _ptr(out)))
        return out

    def prefill(self, seqs: Sequence[int], prompts: Sequence[Sequence[int]]) -> None:
        """``step`` over prompts of any length, as many tokens at a time as the
        cache takes; under a window, pages that fall behind it are reused in
        between."""
        at = [0] * len(prompts)
        while True:
            room, which, pieces = self.max_rows, [], []
            for i, p in enumerate(prompts):
                piece = p[at[i]:at[i] + room]
                if len(piece):
                    which.append(seqs[i])
                    pieces.append(piece)
                    at[i] += len(piece)
                    room -= len(piece)
            if not which:
                return
            self.step(which, pieces, logits=False)


@dataclass
class Scored:
    """A generated sequence: its tokens, their log probabilities, the entropy of
    the distribution each was taken from and, with ``top``, the alternatives
    (id, log probability) of each."""

    tokens: list[int] = field(default_factory=list)
    finish_reason: FinishReason = FinishReason.LENGTH
    logp: list[float] = field(default_factory=list)
    entropy: list[float] = field(default_factory=list)
    alternatives: list[list[tuple[int, float]]] = field(default_factory=list)


def generate_paged(cache: PagedKvCache, prompts: Sequence[Sequence[int]], budget: int,
                   eos: int = DEFAULT_EOS, top: int = 0) -> list[Scored]:
    """Greedy generation (ties to the smallest id, eos ends a row and is not
    kept; engine.rs:493-541) for up to ``cache.max_seqs`` prompts over the paged
    cache.  Rows leave the batch when they end; the sequences are freed."""
    if budget < 1:
        raise FmdError(-1, "budget must be >= 1")
    if any(len(p) == 0 for p in prompts):
        raise FmdError(-1, "empty prompt")
    model = cache.model
    out = [Scored() for _ in prompts]
    seqs: list[int] = []
    try:
        for _ in prompts:
            seqs.append(cache.open())
        live = list(range(len(prompts)))
        # all but the last tokens, so that the first step has every row's logits
        cache.prefill(seqs, [list(p[:-1]) for p in prompts])
        feed = [[p[-1]] for p in prompts]
        for step in range(budget):
            if not live:
                break
            cache.step([seqs[i] for i in live], feed, logits=False)
            s = model.logprobs(len(live), top=max(top, 1))
            stay, feed = [], []
            for r, i in enumerate(live):
                tok = int(s.top_ids[r, 0])
                if tok == eos:
                    out[i].finish_reason = FinishReason.STOP
                    continue
                out[i].tokens.append(tok)
                out[i].logp.append(float(s.top_logp[r, 0]))
                out[i].entropy.append(float(s.entropy[r]))
                if top:
                    out[i].alternatives.append([(int(a), float(b)) for a, b in
                                                zip(s.top_ids[r], s.top_logp[r])])
                stay.append(i)
                feed.append([tok])
            live = stay
    finally:
        for i in seqs:
            cache.free(i)
    return out
