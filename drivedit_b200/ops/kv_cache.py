"""Paged key/value cache in 8 bits for streaming generation.

A page holds 64 consecutive tokens of one sequence, for every layer and head, as e4m3
codes with one power-of-two scale for each (layer, page, head), keys and values apart:
half a bf16 cache's memory and reads. Sequences are lists of pages of one pool, so the
oldest tokens are dropped by giving pages back (:meth:`PagedKVCache.trim`), one sequence
becomes several by sharing pages (:meth:`PagedKVCache.fork`), and the pool is packed
without touching any sequence's contents (:meth:`PagedKVCache.compact`).

Use::

    cache = PagedKVCache(n_layers, n_heads, n_pages, device="cuda")
    seqs = cache.add(batch)
    step = cache.begin(seqs, n_new)            # room for n_new tokens of each sequence
    for layer in range(n_layers):
        step.write(layer, k, v)                # [B, n_new, n_heads, 64]
        o = step.attend(layer, q, causal="frame", tokens_per_frame=512, window=36, sinks=4)
    step.commit()                              # the tokens stay; without it they are redone

What a cached block stands for: ``code * scale``, ``scale = 2^e`` with the smallest ``e``
for which the block's largest finite magnitude is at most ``448 * 2^e`` (``e`` in
[-100, 119]), codes rounded to nearest even, infinities saturated, NaN kept. Writing into an
unfinished page re-codes the tokens it already holds when its scale changes: exactly, but
for codes that become subnormal, so tokens of far larger magnitude in the same page (also
ones that are never committed) leave small values coarser.

CUDA caches run the sm_100a kernels (``csrc/kvcache``); CPU caches the PyTorch statements
below, which are also the kernels' oracle. Calls run on the current stream. A step may
be used on another stream than the one it was begun on (its table is waited for); the
order of writes and reads of the cache itself between streams is the caller's, as for
any tensor. Bookkeeping (``csrc/kvcache/book.cpp``) is on the host: calls on one cache come
from one thread, and none that changes it can be captured into a graph. ``write`` and ``attend`` can (on another
stream than the step's, the host waits for its table); a graph that holds them is replayed
behind the refill of its step (``begin(..., out=step)``) for the sequences as they are then,
as long as the step lives, and not after :meth:`PagedKVCache.resize`.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Union

import numpy as np
import torch

from ..data.native import native
from ._ext import ext
from .window_attention import _check_mask

PAGE = 64       # tokens of a page
_INFO = 4       # words of a step's row before its page ids
_MAX_TOKENS = 1 << 30


def _pages(tokens: int) -> int:
    return (tokens + PAGE - 1) // PAGE


def _two_to(e: torch.Tensor) -> torch.Tensor:
    """``2^e`` of whole ``e`` in [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def quantize_block(x: torch.Tensor):
    """Codes and scales of blocks ``x [..., tokens, channels]`` (fp32): ``(e4m3, fp32 [...])``."""
    amax = torch.where(x.isfinite(), x, 0.0).abs().amax((-1, -2))
    mant, exp = torch.frexp(amax)
    e = torch.where(mant <= 0.875, exp - 9, exp - 8)
    e = torch.where(amax > 0, e, -100).clamp(-100, 119)
    y = x * _two_to(-e)[..., None, None]
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), _two_to(e)


class CacheStep:
    """Room for new tokens of some sequences (:meth:`PagedKVCache.begin`).

    ``write`` / ``attend`` may run any number of times, for any layers, before ``commit``.
    Once a sequence of the step has changed otherwise (commit, trim, fork, free, a later
    ``begin``, compaction) the step is stale and its calls raise."""

    def __init__(self, cache: "PagedKVCache", seqs, n_new, versions, max_tokens, table, handle):
        self.cache = cache
        self.seqs, self.n_new = seqs, n_new
        self.max_tokens = max_tokens  # launches are shaped for sequences up to this length
        self._versions, self._epoch = versions, cache._book.epoch
        self._rows, self._h = table, handle

    @property
    def table(self) -> torch.Tensor:
        """Page ids by sequence, int32 ``[B, max_pages_per_seq]`` (-1: none)."""
        return (self._rows if self._h is None else self._h.rows)[:, _INFO:]

    def _check(self):
        book = self.cache._book
        if self._epoch != book.epoch:  # something of the cache has changed
            if not book.fresh(self.seqs, self._versions):
                raise RuntimeError("stale step: a sequence has changed since it was begun; begin a new one")
            self._epoch = book.epoch

    @property
    def _states(self):
        return [self.cache._book.seq(i) for i in self.seqs]

    def _tokens(self, x: torch.Tensor, name: str, heads: Optional[int]):
        """The extension's checks, for the PyTorch form."""
        c = self.cache
        if x.dim() != 4 or x.shape[0] != len(self.seqs) or x.shape[3] != 64:
            raise ValueError(f"{name} must be [{len(self.seqs)}, T, heads, 64], got {tuple(x.shape)}")
        if heads is not None and x.shape[2] != heads or x.shape[2] == 0 or x.shape[2] % c.n_heads:
            raise ValueError(f"{name} has {x.shape[2]} heads, the cache {c.n_heads}")
        if x.shape[1] < max(self.n_new, default=0):
            raise ValueError(f"{name} holds {x.shape[1]} tokens, the step {max(self.n_new)}")
        if x.device != c.device:
            raise ValueError(f"{name} is on {x.device}, the cache on {c.device}")

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Cache the new tokens' ``k``, ``v`` ``[B, T, n_heads, 64]`` (any strides; sequence
        ``i`` has the first ``n_new[i]`` rows, the others are not read)."""
        self._check()
        if self._h is not None:
            ext().kv_step_write(self._h, layer, k, v)
            return
        c = self.cache
        c._layer(layer)
        self._tokens(k, "k", c.n_heads), self._tokens(v, "v", c.n_heads)
        if k.shape != v.shape:
            raise ValueError("k and v differ in shape")
        self._write_torch(layer, k, v)

    def attend(self, layer: int, q: torch.Tensor, causal: str = "frame", tokens_per_frame: int = 1,
               window: int = 0, sinks: int = 0, scale: Optional[float] = None, return_lse: bool = False):
        """Attention of the new tokens ``q [B, T, heads, 64]`` over their sequences, the new
        tokens (written before) among them; ``heads`` is a multiple of the cache's, head
        ``h`` reading cached head ``h // (heads / n_heads)``.

        ``causal``: "frame" (a query sees its whole frame and earlier ones), "token" or
        "none". ``window`` (frames, for "token" tokens; 0: no limit) keeps the newest ones
        visible, the query's own counted, and ``sinks`` the sequence's first ones beside
        them. Of a trimmed sequence what :meth:`PagedKVCache.trim` kept is visible at most.
        Returns ``o [B, T, heads, 64]`` (and ``lse [B, heads, T]``, log2 domain), without
        gradient; rows behind a sequence's ``n_new`` and rows that see no key are zero (-inf)."""
        self._check()
        if self._h is not None:
            out = ext().kv_step_attend(self._h, layer, q, causal, tokens_per_frame, window, sinks, scale, return_lse)
            return tuple(out) if return_lse else out[0]
        c = self.cache
        c._layer(layer)
        self._tokens(q, "q", None)
        scale = 1.0 / math.sqrt(64) if scale is None else float(scale)
        _check_mask(causal, tokens_per_frame, window, sinks, 0, 0, scale, 0, 0)
        unit = tokens_per_frame if causal == "frame" else 1
        n_sink = min(sinks * unit, _MAX_TOKENS)
        if (window or sinks) and any(s.trimmed and s.sinks != n_sink for s in self._states):
            raise ValueError(f"a trimmed sequence keeps the first tokens it was trimmed to; the call names {n_sink} sinks")
        return self._attend_torch(layer, q, causal, unit, window, n_sink, scale, return_lse)

    def commit(self) -> None:
        """Keep the step's tokens: its sequences grow by ``n_new``."""
        self._check()
        self.cache._book.commit(self.seqs, self.n_new)

    # ------------------------------------------------------------------ PyTorch form
    @torch.no_grad()
    def _write_torch(self, layer, k, v):
        c = self.cache
        for i, (s, n) in enumerate(zip(self._states, self.n_new)):
            for j in range(s.length // PAGE, _pages(s.length + n)) if n else ():
                lo, hi = max(s.length, j * PAGE), min(s.length + n, (j + 1) * PAGE)
                kept = max(0, s.length - j * PAGE)
                for codes, scales, new, last in ((c.k, c.k_scale, k, False), (c.v, c.v_scale, v, True)):
                    held = codes[layer, s.pages[j]].float() * scales[layer, s.pages[j]][:, None, None]
                    x = torch.zeros(c.n_heads, PAGE, 64, device=c.device)
                    x[:, :kept] = (held.mT if last else held)[:, :kept]
                    x[:, lo - j * PAGE:hi - j * PAGE] = new[i, lo - s.length:hi - s.length].transpose(0, 1).float()
                    y, sc = quantize_block(x)
                    codes[layer, s.pages[j]] = y.mT if last else y
                    scales[layer, s.pages[j]] = sc

    @torch.no_grad()
    def _attend_torch(self, layer, q, causal, unit, window, n_sink, scale, return_lse):
        c = self.cache
        o = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), -math.inf, device=q.device)
        G = q.shape[2] // c.n_heads
        for i, (s, n) in enumerate(zip(self._states, self.n_new)):
            if not n:
                continue
            total = s.length + n
            k, v = c._values(layer, s, total)                                  # [total, heads, 64]
            k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
            sc = torch.einsum("thd,shd->hts", q[i, :n].float(), k) * scale
            qf = (torch.arange(s.length, total, device=q.device) // unit)[:, None]
            pos = torch.arange(total, device=q.device)
            kf = (pos // unit)[None]
            seen = kf <= qf if causal != "none" else torch.ones(n, total, dtype=torch.bool, device=q.device)
            if window:
                seen = seen & ((kf > qf - window) | (pos < n_sink))
            if s.trimmed:
                seen = seen & ((pos >= s.first) | (pos < s.sinks))
            sc = sc.masked_fill(~seen, -math.inf)
            ls = torch.logsumexp(sc, -1)
            p = torch.where(seen, torch.exp(sc - ls[..., None]), 0.0)
            o[i, :n] = torch.einsum("hts,shd->thd", p, torch.where(seen.any(0)[:, None, None], v, 0.0)).to(q.dtype)
            lse[i, :, :n] = ls / math.log(2)
        return (o, lse) if return_lse else o


class PagedKVCache:
    """A pool of ``n_pages`` pages of 64 tokens for ``n_layers`` x ``n_heads`` (cached heads,
    64 channels each) and the sequences that own them.

    ``k`` / ``v``: float8_e4m3fn ``[layers, pages, heads, 64, 64]``, keys by (token, channel),
    values by (channel, token); ``k_scale`` / ``v_scale``: float32 ``[layers, pages, heads]``.
    ``max_pages_per_seq`` bounds a sequence (default: the pool, at the largest that it has
    been). Free pages are taken in
    the order of their ids. Every call that does not fit raises before it changes anything."""

    def __init__(self, n_layers: int, n_heads: int, n_pages: int, device=None,
                 max_pages_per_seq: Optional[int] = None):
        if n_layers < 1 or n_heads < 1 or n_pages < 1:
            raise ValueError("layers, heads and pages must be positive")
        device = torch.device(device if device is not None else ("cuda" if torch.cuda.is_available() else "cpu"))
        if device.type == "cuda":
            if device.index is None:
                device = torch.device("cuda", torch.cuda.current_device())
            with torch.cuda.device(device):
                ext().read_status()  # the status word exists before any capture
        self.device = device
        self.n_layers, self.n_heads, self.n_pages = n_layers, n_heads, n_pages
        self.max_pages_per_seq = n_pages if max_pages_per_seq is None else max_pages_per_seq
        self._bound_by_pool = max_pages_per_seq is None
        if not 1 <= self.max_pages_per_seq <= _MAX_TOKENS // PAGE:
            raise ValueError("max_pages_per_seq out of range")
        self.k, self.v, self.k_scale, self.v_scale = self._pool(n_pages)
        self._book = native().KvBook(n_pages, self.max_pages_per_seq)

    def _pool(self, n):
        shape = (self.n_layers, n, self.n_heads)
        codes = [torch.zeros(*shape, PAGE, 64, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn) for _ in "kv"]
        return (*codes, *(torch.ones(*shape, device=self.device) for _ in "kv"))

    # ------------------------------------------------------------------ bookkeeping
    def _layer(self, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of a cache of {self.n_layers}")

    @property
    def _seqs(self) -> dict:
        return self._book.seqs()

    @property
    def _refs(self) -> np.ndarray:
        """Sequences that hold each page."""
        return self._book.refs()

    def _copy(self, src: torch.Tensor, dst: torch.Tensor):
        if not src.numel():
            return
        if self.device.type == "cuda":
            ext().kv_cache_copy_pages(self.k, self.v, self.k_scale, self.v_scale, src, dst)
        else:
            for t in (self.k.view(torch.uint8), self.v.view(torch.uint8), self.k_scale, self.v_scale):
                t[:, dst.long()] = t[:, src.long()]

    def _not_capturing(self, what):
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} changes the cache's tables on the host and cannot be captured")

    @property
    def free_pages(self) -> int:
        return self._book.free_pages

    @property
    def sequences(self) -> List[int]:
        return list(self._book.seqs())

    def length(self, seq: int) -> int:
        """Committed tokens of a sequence (its next position), dropped ones counted."""
        return self._book.seq(seq).length

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale))

    def table(self, seqs: Sequence[int]) -> torch.Tensor:
        """Page ids of the sequences, int32 ``[n, max_pages_per_seq]`` (-1: none)."""
        rows = self._book.table(list(seqs))
        return rows.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else rows

    # ------------------------------------------------------------------ sequences
    def add(self, n: int = 1) -> List[int]:
        """``n`` new empty sequences; returns their ids."""
        return self._book.add(n)

    def begin(self, seqs: Sequence[int], n_new: Union[int, Sequence[int]], max_tokens: Optional[int] = None,
              out: Optional[CacheStep] = None) -> CacheStep:
        """Make room for ``n_new`` tokens (one number, or one for each sequence) behind each
        sequence's committed ones. A shared unfinished page that they go into is copied first.

        ``max_tokens``: the longest sequence (its new tokens counted) that the step's launches
        are shaped for, for steps whose calls are captured into a graph; default: the
        longest of now. ``out``: a step of as many sequences to refill in place (on the current
        stream, behind the calls that still read it), so that a graph captured with it runs
        on the new tables; its ``max_tokens`` must suffice, ``n_new`` fit the rows of its captured
        calls, and the sinks of windowed ones be those that the sequences were trimmed to."""
        self._not_capturing("begin")
        seqs = list(seqs)
        n_new = [int(n) for n in n_new] if isinstance(n_new, (list, tuple)) else [int(n_new)] * len(seqs)
        if out is not None:
            if out.cache is not self or len(out.seqs) != len(seqs):
                raise ValueError("out is a step of another cache or number of sequences")
            if out._rows.shape[1] != _INFO + self.max_pages_per_seq:
                raise ValueError("out was begun before the cache grew")
            max_tokens = out.max_tokens if max_tokens is None else max_tokens
            if max_tokens != out.max_tokens:
                raise ValueError("out keeps its max_tokens")
            if out._h is not None:
                ext().kv_step_check_refill(out._h, max(n_new, default=0), self._book.trim_sinks(seqs))
        if max_tokens is not None and max_tokens < 0:
            raise ValueError("max_tokens must not be negative")
        rows, src, dst, longest, trim, versions = self._book.begin(seqs, n_new, -1 if max_tokens is None else int(max_tokens))
        max_tokens = longest if max_tokens is None else int(max_tokens)
        self._copy(src, dst)
        handle = None
        if self.device.type == "cuda":
            handle = ext().kv_step_begin(self.k, self.v, self.k_scale, self.v_scale, rows, max_tokens, max(n_new, default=0),
                                         trim, None if out is None else out._h)
        if out is None:
            return CacheStep(self, seqs, n_new, versions, max_tokens, rows, handle)
        out.__init__(self, seqs, n_new, versions, max_tokens, rows, handle)
        return out

    def fork(self, seqs: Sequence[int], copies: int = 1) -> List[int]:
        """``copies`` new sequences from each of ``seqs`` (all copies of the first, then of the
        next), sharing its pages; an unfinished page is copied when one of them is written."""
        return self._book.fork(list(seqs), copies)

    def copy(self, seqs: Sequence[int]) -> List[int]:
        """New sequences with the committed tokens of ``seqs`` in pages of their own."""
        self._not_capturing("copy")
        out, src, dst = self._book.copy(list(seqs))
        self._copy(src, dst)
        return out

    def free(self, seqs: Sequence[int]) -> None:
        """Drop sequences; pages that no other sequence shares become free."""
        self._book.free(list(seqs))

    def trim(self, seqs: Sequence[int], keep: int, sinks: int = 0) -> None:
        """Drop each sequence's tokens but its first ``sinks`` and its newest ``keep`` ones:
        no query sees them any more, and pages that held nothing else become free."""
        self._book.trim(list(seqs), keep, sinks)

    def compact(self) -> int:
        """Move the pages in use to the front of the pool; returns how many there are."""
        self._not_capturing("compact")
        self._copy(*self._book.compact())
        return self.n_pages - self.free_pages

    def resize(self, n_pages: int) -> None:
        """Change the pool to ``n_pages`` pages (compacted first when it shrinks below a page
        in use); the pages in use keep their contents. The pool's tensors are new ones."""
        self._not_capturing("resize")
        used = self.n_pages - self.free_pages
        if n_pages < max(used, 1):
            raise ValueError(f"{used} pages are in use, {n_pages} asked for")
        if self._bound_by_pool and n_pages > _MAX_TOKENS // PAGE:
            raise ValueError("max_pages_per_seq out of range")
        if self._book.used_end() > n_pages:
            self.compact()
        old, n = (self.k, self.v, self.k_scale, self.v_scale), min(n_pages, self.n_pages)
        self.k, self.v, self.k_scale, self.v_scale = self._pool(n_pages)
        for a, b in zip((self.k, self.v, self.k_scale, self.v_scale), old):
            a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
            a[:, :n].copy_(b[:, :n])
        if self._bound_by_pool:
            self.max_pages_per_seq = max(self.max_pages_per_seq, n_pages)
        self._book.resize(n_pages, self.max_pages_per_seq)
        self.n_pages = n_pages

    def _values(self, layer, s, n: int):
        ids = torch.from_numpy(np.maximum(s.pages[:_pages(n)], 0)).long().to(self.device)
        out = []
        for codes, scales, last in ((self.k, self.k_scale, False), (self.v, self.v_scale, True)):
            x = codes[layer].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * scales[layer, ids][..., None, None]
            x = (x.mT if last else x).transpose(1, 2).reshape(-1, self.n_heads, 64)[:n]
            if s.trimmed:
                x = x.clone()
                x[s.sinks:s.first] = 0
            out.append(x)
        return out

    def read(self, layer: int, seq: int):
        """The committed keys and values of a sequence as they are held, fp32
        ``[length, n_heads, 64]`` each (dropped tokens zero)."""
        self._layer(layer)
        s = self._book.seq(seq)
        return tuple(self._values(layer, s, s.length))
