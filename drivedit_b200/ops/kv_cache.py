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
any tensor. Bookkeeping is on the host: calls on one cache come from one thread, and none
that changes it can be captured into a graph. ``write`` and ``attend`` can; a graph that
holds them is replayed after its step was refilled (``begin(..., out=step)``) for the
sequences as they are then, and not after :meth:`PagedKVCache.resize`.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Union

import numpy as np
import torch

from ._ext import ext
from .window_attention import _check_mask

PAGE = 64       # tokens of a page
_INFO = 4       # words of a step's row before its page ids
_MAX_TOKENS = 1 << 30


def _pages(tokens: int) -> int:
    return (tokens + PAGE - 1) // PAGE


class _Seq:
    __slots__ = ("pages", "length", "first", "sinks", "version")

    def __init__(self, pages, length=0, first=0, sinks=0):
        self.pages = pages          # int32 ids by page of the sequence; -1: given back
        self.length = length        # committed tokens
        self.first = first          # tokens in [sinks, first) are gone
        self.sinks = sinks
        self.version = 0            # a step begun at another version is stale

    @property
    def trimmed(self):
        return self.first > self.sinks


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

    def __init__(self, cache: "PagedKVCache", seqs, n_new, max_tokens, table, handle):
        self.cache = cache
        self.seqs, self.n_new = seqs, n_new
        self.max_tokens = max_tokens  # launches are shaped for sequences up to this length
        self._states = [cache._seqs[i] for i in seqs]
        self._versions = [s.version for s in self._states]
        self._epoch = cache._epoch
        self._rows, self._h = table, handle

    @property
    def table(self) -> torch.Tensor:
        """Page ids by sequence, int32 ``[B, max_pages_per_seq]`` (-1: none)."""
        return (self._rows if self._h is None else self._h.rows)[:, _INFO:]

    def _check(self):
        if self._epoch != self.cache._epoch:  # something of the cache has changed
            if any(s.version != v for s, v in zip(self._states, self._versions)):
                raise RuntimeError("stale step: a sequence has changed since it was begun; begin a new one")
            self._epoch = self.cache._epoch

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
        Returns ``o [B, T, heads, 64]`` (and ``lse [B, heads, T]``, log2 domain); rows
        behind a sequence's ``n_new`` and rows that see no key are zero (-inf)."""
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
        self.cache._epoch += 1
        for s, n in zip(self._states, self.n_new):
            s.length += n
            s.version += 1

    # ------------------------------------------------------------------ PyTorch form
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
    ``max_pages_per_seq`` bounds a sequence (default: the pool). Free pages are taken in
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
        if not 1 <= self.max_pages_per_seq <= _MAX_TOKENS // PAGE:
            raise ValueError("max_pages_per_seq out of range")
        self.k, self.v, self.k_scale, self.v_scale = self._pool(n_pages)
        self._refs = np.zeros(n_pages, np.int32)  # sequences that hold a page
        self._n_free, self._low = n_pages, 0      # no page below _low is free
        self._seqs: dict = {}
        self._next = 0
        self._epoch = 0                           # counts changes of any sequence

    def _pool(self, n):
        shape = (self.n_layers, n, self.n_heads)
        codes = [torch.zeros(*shape, PAGE, 64, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn) for _ in "kv"]
        return (*codes, *(torch.ones(*shape, device=self.device) for _ in "kv"))

    # ------------------------------------------------------------------ bookkeeping
    def _layer(self, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of a cache of {self.n_layers}")

    def _get(self, seqs) -> List[_Seq]:
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        missing = [i for i in seqs if i not in self._seqs]
        if missing:
            raise ValueError(f"no sequence {missing[0]} in this cache")
        return [self._seqs[i] for i in seqs]

    def _need(self, n):
        if n > self._n_free:
            raise RuntimeError(f"out of cache pages: {n} needed, {self._n_free} of {self.n_pages} free")

    def _take(self, n: int) -> np.ndarray:
        """The ``n`` lowest free pages (there are as many)."""
        ids = np.flatnonzero(self._refs[self._low:self._low + 4 * n + 256] == 0)
        if len(ids) < n:
            ids = np.flatnonzero(self._refs[self._low:] == 0)
        ids = (ids[:n] + self._low).astype(np.int32)
        if n:
            self._refs[ids] = 1
            self._n_free -= n
            self._low = int(ids[-1]) + 1
        return ids

    def _give(self, pages: np.ndarray) -> None:
        """A hold of each of these pages ends (a page named twice has two)."""
        held = np.bincount(pages[pages >= 0])
        refs = self._refs[:len(held)]
        refs -= held.astype(np.int32)
        freed = np.flatnonzero((refs == 0) & (held > 0))
        if len(freed):
            self._n_free += len(freed)
            self._low = min(self._low, int(freed[0]))

    def _copy(self, src, dst):
        if not len(src):
            return
        if self.device.type == "cuda":
            ids = [torch.from_numpy(np.ascontiguousarray(x, np.int32)) for x in (src, dst)]
            ext().kv_cache_copy_pages(self.k, self.v, self.k_scale, self.v_scale, *ids)
        else:
            for t in (self.k.view(torch.uint8), self.v.view(torch.uint8), self.k_scale, self.v_scale):
                t[:, list(dst)] = t[:, list(src)]

    def _not_capturing(self, what):
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} changes the cache's tables on the host and cannot be captured")

    @property
    def free_pages(self) -> int:
        return self._n_free

    @property
    def sequences(self) -> List[int]:
        return list(self._seqs)

    def length(self, seq: int) -> int:
        """Committed tokens of a sequence (its next position), dropped ones counted."""
        return self._get([seq])[0].length

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale))

    def table(self, seqs: Sequence[int]) -> torch.Tensor:
        """Page ids of the sequences, int32 ``[n, max_pages_per_seq]`` (-1: none)."""
        rows = np.full((len(seqs), self.max_pages_per_seq), -1, np.int32)
        for i, s in enumerate(self._get(seqs)):
            rows[i, :len(s.pages)] = s.pages
        rows = torch.from_numpy(rows)
        return rows.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else rows

    # ------------------------------------------------------------------ sequences
    def add(self, n: int = 1) -> List[int]:
        """``n`` new empty sequences; returns their ids."""
        if n < 0:
            raise ValueError("n must not be negative")
        ids = list(range(self._next, self._next + n))
        self._next += n
        for i in ids:
            self._seqs[i] = _Seq(np.empty(0, np.int32))
        return ids

    def begin(self, seqs: Sequence[int], n_new: Union[int, Sequence[int]], max_tokens: Optional[int] = None,
              out: Optional[CacheStep] = None) -> CacheStep:
        """Make room for ``n_new`` tokens (one number, or one for each sequence) behind each
        sequence's committed ones. A shared unfinished page that they go into is copied first.

        ``max_tokens``: the longest sequence (its new tokens counted) that the step's launches
        are shaped for, for steps whose calls are captured into a graph; default: the
        longest of now. ``out``: a step of as many sequences to refill in place (on the current
        stream, behind the calls that still read it), so that a graph captured with it runs
        on the new tables; its ``max_tokens`` must suffice."""
        self._not_capturing("begin")
        states = self._get(seqs)
        n_new = [int(n_new)] * len(states) if not isinstance(n_new, (list, tuple)) else [int(n) for n in n_new]
        if len(n_new) != len(states) or any(n < 0 for n in n_new):
            raise ValueError("n_new must be one number, or one for each sequence, none negative")
        longest = max((s.length + n for s, n in zip(states, n_new)), default=0)
        if longest > self.max_pages_per_seq * PAGE:
            raise ValueError(f"{longest} tokens do not fit a sequence's {self.max_pages_per_seq} pages")
        if out is not None:
            if out.cache is not self or len(out.seqs) != len(states):
                raise ValueError("out is a step of another cache or number of sequences")
            max_tokens = out.max_tokens if max_tokens is None else max_tokens
            if max_tokens != out.max_tokens:
                raise ValueError("out keeps its max_tokens")
        max_tokens = longest if max_tokens is None else int(max_tokens)
        if max_tokens < longest:
            raise ValueError(f"sequences of {longest} tokens in a step for {max_tokens}")
        # Pages to take: behind the present ones, and for shared pages that get new tokens (of
        # a page shared within this call the last one to write keeps it). Pages behind the
        # new tokens are the room of an abandoned step.
        refs = self._refs
        need, spare, shared, todo = 0, 0, {}, []
        for i, (s, n) in enumerate(zip(states, n_new)):
            have, upto = len(s.pages), (s.length + n + PAGE - 1) // PAGE
            if upto > have:
                need += upto - have
                todo.append(i)
            elif upto < have:
                spare += have - upto
            for j in range(s.length // PAGE, min(upto, have)) if n else ():
                p = int(s.pages[j])
                if refs[p] > 1:
                    shared[p] = shared.get(p, int(refs[p])) - 1
                    if shared[p] > 0:
                        need += 1
                        todo.append(i)
        self._need(need - spare)
        self._epoch += 1
        if spare:
            for s, n in zip(states, n_new):
                upto = _pages(s.length + n)
                if len(s.pages) > upto:
                    self._give(s.pages[upto:])
                    s.pages = s.pages[:upto]
        if todo:
            fresh = iter(self._take(need).tolist())
            src, dst = [], []
            for i in dict.fromkeys(todo):
                s = states[i]
                have, upto = len(s.pages), _pages(s.length + n_new[i])
                for j in range(s.length // PAGE, min(upto, have)) if shared and n_new[i] else ():
                    p = int(s.pages[j])
                    if refs[p] > 1:
                        s.pages = s.pages.copy()
                        s.pages[j] = to = next(fresh)
                        if j * PAGE < s.length:
                            src.append(p)
                            dst.append(to)
                        refs[p] -= 1
                if upto > have:
                    s.pages = np.append(s.pages, np.fromiter(fresh, np.int32, upto - have))
            self._copy(src, dst)
        rows = np.full((len(states), _INFO + self.max_pages_per_seq), -1, np.int32)
        trim, heads = -1, []
        for i, (s, n) in enumerate(zip(states, n_new)):
            s.version += 1
            if s.first > s.sinks:
                heads.append((s.length + n, n, s.first, s.sinks))
                trim = s.sinks if trim in (-1, s.sinks) else -2
            else:
                heads.append((s.length + n, n, 0, -1))
            rows[i, _INFO:_INFO + len(s.pages)] = s.pages
        if heads:
            rows[:, :_INFO] = heads
        rows, handle = torch.from_numpy(rows), None
        if self.device.type == "cuda":
            handle = ext().kv_step_begin(self.k, self.v, self.k_scale, self.v_scale, rows, max_tokens, max(n_new, default=0),
                                         trim, None if out is None else out._h)
        if out is None:
            return CacheStep(self, list(seqs), n_new, max_tokens, rows, handle)
        out.__init__(self, list(seqs), n_new, max_tokens, rows, handle)
        return out

    def fork(self, seqs: Sequence[int], copies: int = 1) -> List[int]:
        """``copies`` new sequences from each of ``seqs`` (all copies of the first, then of the
        next), sharing its pages; an unfinished page is copied when one of them is written."""
        states = self._get(seqs)
        if copies < 0:
            raise ValueError("copies must not be negative")
        self._epoch += 1
        out = self.add(copies * len(states))
        for i, s in enumerate(states):
            s.version += 1
            pages = s.pages[:_pages(s.length)].copy()
            self._refs[pages[pages >= 0] if s.trimmed else pages] += copies
            for k in out[i * copies:(i + 1) * copies]:
                # a sequence's page list is replaced, never written in place
                self._seqs[k] = _Seq(pages, s.length, s.first, s.sinks)
        return out

    def copy(self, seqs: Sequence[int]) -> List[int]:
        """New sequences with the committed tokens of ``seqs`` in pages of their own."""
        self._not_capturing("copy")
        states = self._get(seqs)
        kept = [s.pages[:_pages(s.length)] for s in states]
        src = np.concatenate([p[p >= 0] for p in kept]) if kept else np.empty(0, np.int32)
        self._need(len(src))
        dst = self._take(len(src))
        out, at = self.add(len(states)), 0
        for i, s, p in zip(out, states, kept):
            pages, n = p.copy(), int((p >= 0).sum())
            pages[p >= 0] = dst[at:at + n]
            at += n
            self._seqs[i] = _Seq(pages, s.length, s.first, s.sinks)
        self._copy(src, dst)
        return out

    def free(self, seqs: Sequence[int]) -> None:
        """Drop sequences; pages that no other sequence shares become free."""
        states = self._get(seqs)
        if not states:
            return
        self._epoch += 1
        self._give(np.concatenate([s.pages for s in states]))
        for i, s in zip(seqs, states):
            s.version += 1
            del self._seqs[i]

    def trim(self, seqs: Sequence[int], keep: int, sinks: int = 0) -> None:
        """Drop each sequence's tokens but its first ``sinks`` and its newest ``keep`` ones:
        no query sees them any more, and pages that held nothing else become free."""
        states = self._get(seqs)
        if keep < 0 or sinks < 0:
            raise ValueError("keep and sinks must not be negative")
        if any(s.trimmed and s.sinks != sinks for s in states):
            raise ValueError("a sequence that was trimmed keeps its number of sinks")
        self._epoch += 1
        for s in states:
            first = max(s.first, s.length - keep)
            if first <= sinks:
                continue
            s.first, s.sinks = first, sinks
            lo, hi = _pages(sinks), min(first // PAGE, len(s.pages))
            if hi > lo:
                self._give(s.pages[lo:hi])
                s.pages = s.pages.copy()
                s.pages[lo:hi] = -1
            s.version += 1

    def compact(self) -> int:
        """Move the pages in use to the front of the pool; returns how many there are."""
        self._not_capturing("compact")
        used = self._refs > 0
        n = self.n_pages - self._n_free
        src, dst = np.flatnonzero(used[n:]) + n, np.flatnonzero(~used[:n])
        if len(src):
            self._epoch += 1
            self._copy(src, dst)
            to = np.arange(self.n_pages, dtype=np.int32)
            to[src] = dst
            for s in self._seqs.values():
                moved = np.where(s.pages >= 0, to[s.pages], -1).astype(np.int32)
                if not np.array_equal(moved, s.pages):
                    s.pages = moved
                    s.version += 1
            self._refs[dst] = self._refs[src]
            self._refs[src] = 0
            self._low = n
        return n

    def resize(self, n_pages: int) -> None:
        """Change the pool to ``n_pages`` pages (compacted first when it shrinks below a page
        in use); the pages in use keep their contents. The pool's tensors are new ones."""
        self._not_capturing("resize")
        used = self.n_pages - self._n_free
        if n_pages < max(used, 1):
            raise ValueError(f"{used} pages are in use, {n_pages} asked for")
        if self._refs[n_pages:].any():
            self.compact()
        old, n = (self.k, self.v, self.k_scale, self.v_scale), min(n_pages, self.n_pages)
        self.k, self.v, self.k_scale, self.v_scale = self._pool(n_pages)
        for a, b in zip((self.k, self.v, self.k_scale, self.v_scale), old):
            a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
            a[:, :n].copy_(b[:, :n])
        self._refs = np.concatenate([self._refs[:n], np.zeros(n_pages - n, np.int32)])
        self._n_free, self._low, self.n_pages = n_pages - used, 0, n_pages
        self._epoch += 1
        for s in self._seqs.values():
            s.version += 1

    def _values(self, layer, s: _Seq, n: int):
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
        s = self._get([seq])[0]
        return tuple(self._values(layer, s, s.length))
