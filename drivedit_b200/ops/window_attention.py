"""Attention over a sliding window and the first tokens, forward and backward.

A query of frame ``f`` sees the frames ``f - window + 1 .. f`` and the first ``sinks`` frames
(the context a rollout starts from): the mask under which a rollout with a rolling
key/value window runs, for training with it and for chunks over a contiguous buffer.
The 8-bit paged cache (:mod:`drivedit_b200.ops.kv_cache`) applies the same mask.

CUDA tensors run the tcgen05 kernels (``csrc/attn``, windowed mode): a tile of queries
reads only key tiles with a visible key, so time goes with the window, not the length.
CPU tensors run the PyTorch statement.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from ..layers.attention import window_mask
from ._ext import ext

_LIMIT = 1 << 30  # positions stay below


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """``x`` as the kernels read it: contiguous channels, strides of 16 bytes (a copy if not)."""
    ok = x.stride(3) == 1 and x.data_ptr() % 16 == 0 and all(
        n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(x.shape[:3], x.stride()[:3]))
    if ok:
        return x
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def window_forward(q, k, v, mask):
    """``(o, lse)`` on CUDA tensors; ``mask`` as :func:`mask_args` gives it. ``lse`` (log2
    domain) is ``[B, H, T]`` with T rounded up to 128, the backward's layout."""
    B, T, H, _ = q.shape
    o = torch.empty(B, T, H, 64, device=q.device, dtype=torch.bfloat16)
    lse = torch.empty(B, H, (T + 127) // 128 * 128, device=q.device, dtype=torch.float32)
    ext().attn_window_fwd(q, k, v, o, lse, *mask)
    return o, lse


def window_backward(q, k, v, o, lse, do, mask, dq, dk, dv):
    """Gradients into the bf16 views ``dq``, ``dk``, ``dv`` (rows of contiguous heads)."""
    B, T, H, _ = q.shape
    do = do.contiguous()
    do = do if do.data_ptr() % 16 == 0 else do.clone()
    delta = torch.empty_like(lse)
    # dQ is summed over the key tiles in fp32; the order of the sums is not fixed, so equal
    # calls may differ in dQ's last fp32 bits before the rounding to bf16
    acc = torch.zeros(B * T, H * 64, device=q.device, dtype=torch.float32)
    ext().attn_window_bwd(q, k, v, o, do, lse, delta, acc, dk, dv, *mask)
    rows = dq.as_strided((B * T, H * 64), (dq.stride(1) if T > 1 else dq.stride(0) if B > 1 else H * 64, 1))
    ext().attn_dq_finalize(acc, rows, 0, H, None, T, 0)


_STREAM = "drivedit_b200.stream"


def _leaf_nodes(*tensors):
    """The accumulation nodes of the leaves among ``tensors``."""
    return [x.view_as(x).grad_fn.next_functions[0][0] for x in tensors if x.requires_grad and x.is_leaf]


def _apply(q, k, v, mask):
    """A backward pass that is captured while an eager graph of the same leaf is alive ends
    the process inside autograd: the leaf's accumulation node belongs to the default
    stream. So the nodes that a graph made here keeps alive are marked with their stream,
    and a capture that meets a node of the default stream is refused."""
    leaves = torch.is_grad_enabled() and any(x.requires_grad and x.is_leaf for x in (q, k, v))
    if leaves and torch.cuda.is_current_stream_capturing():
        if any(n.metadata.get(_STREAM) == 0 for n in _leaf_nodes(q, k, v)):
            raise RuntimeError("an autograd graph made on the default stream still uses this leaf: drop it before "
                               "capturing a backward pass, or warm up on another stream")
    out = _WindowAttention.apply(q, k, v, mask)
    if leaves:
        stream = torch.cuda.current_stream(q.device).cuda_stream
        for n in _leaf_nodes(q, k, v):
            n.metadata.setdefault(_STREAM, stream)
    return out


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask):
        q, k, v = _aligned(q), _aligned(k), _aligned(v)
        o, lse = window_forward(q, k, v, mask)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.mask = mask
        lse = lse[:, :, :q.shape[1]]
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, _):
        q, k, v, o, lse = ctx.saved_tensors
        dq, dk, dv = (torch.empty(x.shape, device=x.device, dtype=x.dtype) for x in (q, k, v))
        window_backward(q, k, v, o, lse, do.to(torch.bfloat16), ctx.mask, dq, dk, dv)
        return dq, dk, dv, None


def mask_args(causal: str, tokens_per_frame: int, window: int, sinks: int, q_pos_offset: int, kv_pos_offset: int,
              scale: float, T: int, S: int):
    """The kernels' mask arguments (checked): causal code, unit, window, sink tokens, positions, scale."""
    if causal not in ("frame", "token", "none"):
        raise ValueError(f"causal must be frame, token or none, got {causal!r}")
    if tokens_per_frame < 1 or window < 0 or sinks < 0 or q_pos_offset < 0 or kv_pos_offset < 0:
        raise ValueError("tokens_per_frame must be positive; window, sinks and offsets not negative")
    if causal == "none" and (window or sinks):
        raise ValueError("a window needs causal frame or token")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if max(q_pos_offset + T, kv_pos_offset + S) > _LIMIT:
        raise ValueError(f"positions must stay below {_LIMIT}")
    if T > 65536 * 64:
        raise ValueError(f"at most {65536 * 64} queries per sample")
    unit = tokens_per_frame if causal == "frame" else 1
    if unit > 1 << 24:
        raise ValueError("at most 2^24 tokens per frame")
    # positions stay below 2^30: a longer window or run of sinks is the same as all of them
    return (int(causal != "none"), unit, window if window * unit <= _LIMIT else 0, min(sinks * unit, _LIMIT),
            q_pos_offset, kv_pos_offset, scale)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: str = "frame",
                     tokens_per_frame: int = 1, window: int = 0, sinks: int = 0, q_pos_offset: int = 0,
                     kv_pos_offset: int = 0, scale: Optional[float] = None, return_lse: bool = False):
    """Softmax attention ``q [B, T, H, 64]`` over ``k``, ``v`` ``[B, S, H, 64]`` (bf16 on CUDA, any
    strides), differentiable in q, k and v.

    ``causal`` "frame": a query at position p (its index plus ``q_pos_offset``) belongs to
    frame ``p // tokens_per_frame`` and sees that whole frame and earlier ones, of those
    the newest ``window`` (its own counted; 0: all) and the first ``sinks``; "token" counts
    tokens instead of frames; "none" sees every key. Keys sit at their index plus
    ``kv_pos_offset``. Rows that see no key are zero and get no gradient; keys that no
    query sees get zero gradients, and their values have no effect. Returns ``o`` (and, if
    asked, ``lse [B, H, T]``, log2 domain of the scaled scores, without gradient)."""
    if q.dim() != 4 or k.dim() != 4 or q.shape[3] != 64 or k.shape != v.shape or \
            (q.shape[0], *q.shape[2:]) != (k.shape[0], *k.shape[2:]):
        raise ValueError(f"q must be [B, T, H, 64], k and v [B, S, H, 64]: got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        raise ValueError("q, k and v must be of one type and on one device")
    B, T, H, _ = q.shape
    S = k.shape[1]
    scale = 1.0 / math.sqrt(64) if scale is None else float(scale)
    mask = mask_args(causal, tokens_per_frame, window, sinks, q_pos_offset, kv_pos_offset, scale, T, S)
    if q.is_cuda and q.dtype != torch.bfloat16:
        raise ValueError(f"window_attention takes bfloat16 on CUDA, got {q.dtype}")
    if q.numel() == 0 or S == 0:  # no key or no query: zeros that depend on nothing
        yes = torch.ones((), dtype=torch.bool, device=q.device)
        o = q.masked_fill(yes, 0) + (k.sum() + v.sum()).masked_fill(yes, 0)
        lse = torch.full((B, H, T), -math.inf, device=q.device)
    elif q.is_cuda:
        o, lse = _apply(q, k, v, mask)
    else:
        seen = window_mask(T, S, causal, tokens_per_frame, window, sinks, q_pos_offset, kv_pos_offset, q.device)
        f = torch.promote_types(q.dtype, torch.float32)
        s = torch.einsum("bthd,bshd->bhts", q.to(f), k.to(f)) * scale
        s = torch.where(seen, s, -math.inf)
        some = seen.any(1)[:, None]
        p = torch.softmax(torch.where(some, s, 0.0), -1) * some
        o = torch.einsum("bhts,bshd->bthd", p, torch.where(seen.any(0)[:, None, None], v.to(f), 0.0)).to(q.dtype)
        lse = torch.logsumexp(s, -1).float().detach() / math.log(2)
    return (o, lse) if return_lse else o
