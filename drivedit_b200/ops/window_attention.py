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
from ._ext import ext, sync_check

_LIMIT = 1 << 30  # positions stay below


def _check_mask(causal, tokens_per_frame, window, sinks, q_pos_offset, kv_pos_offset, scale, T, S):
    """The extension's checks, for the PyTorch statement."""
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
    if causal == "frame" and tokens_per_frame > 1 << 24:
        raise ValueError("at most 2^24 tokens per frame")


class _SyncChecked(torch.autograd.Function):
    """The operator for the sync-check mode, which brackets entry points called from Python: the
    extension's own autograd node calls its backward behind it."""

    @staticmethod
    def forward(ctx, q, k, v, *args):
        o, lse, rest = ext().attn_window_fwd(q, k, v, *args)
        ctx.save_for_backward(q, k, v, o, rest, lse)
        ctx.args = args
        ctx.set_materialize_grads(False)
        lse = lse[..., :q.shape[1]]
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * (3 + len(ctx.args))
        q, k, v, o, rest, lse = ctx.saved_tensors
        out = [torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v)]
        ext().attn_window_bwd(q, k, v, o, rest, lse, grad, *ctx.args[:5], *out, *ctx.args[5:])
        return (*out, *(None for _ in ctx.args))


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: str = "frame",
                     tokens_per_frame: int = 1, window: int = 0, sinks: int = 0, q_pos_offset: int = 0,
                     kv_pos_offset: int = 0, scale: Optional[float] = None, return_lse: bool = False):
    """Softmax attention ``q [B, T, H, 64]`` over ``k``, ``v`` ``[B, S, H, 64]`` (bf16 on CUDA, any
    strides), differentiable in q, k and v.

    ``causal`` "frame": a query at position p (its index plus ``q_pos_offset``) belongs to
    frame ``p // tokens_per_frame`` and sees that whole frame and earlier ones, of those
    the newest ``window`` (its own counted; 0: all) and the first ``sinks``; "token" counts
    tokens instead of frames; "none" sees every key. Keys sit at their index plus
    ``kv_pos_offset``. Rows that see no key are zero and keys that no query sees are
    left out; both get zero gradients, and what they hold has no effect on the others.
    Returns ``o`` (and, if asked, ``lse [B, H, T]``, log2 domain of the scaled scores, without
    gradient). On CUDA scaled scores are fp32 and have to stay below 2^30 in magnitude, or
    rows become NaN; the backward pass makes each weight from its score and ``lse``, so that
    scores of magnitude M leave it a relative error of M * 2^-24. dQ is summed in fp32 in no
    fixed order: equal backward passes may differ in dq by a rounding of bf16. A second
    derivative raises on CUDA. A backward pass is captured into a graph only when no autograd
    graph of the same leaves made on the default stream is alive (refused otherwise)."""
    if q.is_cuda and q.numel() and k.numel():
        if sync_check() and torch.is_grad_enabled() and any(x.requires_grad for x in (q, k, v)):
            o, lse = _SyncChecked.apply(q, k, v, causal, tokens_per_frame, window, sinks, scale, q_pos_offset, kv_pos_offset)
            return (o, lse) if return_lse else o
        o, lse = ext().window_attention(q, k, v, causal, tokens_per_frame, window, sinks, q_pos_offset, kv_pos_offset, scale)
        return (o, lse) if return_lse else o
    if q.dim() != 4 or k.dim() != 4 or q.shape[3] != 64 or k.shape != v.shape or \
            (q.shape[0], *q.shape[2:]) != (k.shape[0], *k.shape[2:]):
        raise ValueError(f"q must be [B, T, H, 64], k and v [B, S, H, 64]: got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        raise ValueError("q, k and v must be of one type and on one device")
    B, T, H, _ = q.shape
    S = k.shape[1]
    scale = 1.0 / math.sqrt(64) if scale is None else float(scale)
    _check_mask(causal, tokens_per_frame, window, sinks, q_pos_offset, kv_pos_offset, scale, T, S)
    if q.numel() == 0 or S == 0:  # no key or no query: zeros that depend on nothing
        yes = torch.ones((), dtype=torch.bool, device=q.device)
        o = q.masked_fill(yes, 0) + (k.sum() + v.sum()).masked_fill(yes, 0)
        lse = torch.full((B, H, T), -math.inf, device=q.device)
    else:
        seen = window_mask(T, S, causal, tokens_per_frame, window, sinks, q_pos_offset, kv_pos_offset, q.device)
        f = torch.promote_types(q.dtype, torch.float32)
        some, used = seen.any(1)[:, None, None], seen.any(0)[:, None, None]  # by query, by key
        # what hidden rows hold stays out of the products, and of the gradients' (0 * NaN)
        qf, kf, vf = torch.where(some, q.to(f), 0.0), torch.where(used, k.to(f), 0.0), torch.where(used, v.to(f), 0.0)
        s = torch.where(seen, torch.einsum("bthd,bshd->bhts", qf, kf) * scale, -math.inf)
        p = torch.softmax(torch.where(some[..., 0], s, 0.0), -1)
        o = torch.where(some, torch.einsum("bhts,bshd->bthd", p, vf), 0.0).to(q.dtype)
        lse = torch.logsumexp(s, -1).float().detach() / math.log(2)
    return (o, lse) if return_lse else o
