"""The paged cache and rollouts over it at their edges, on the CPU."""
import subprocess
import sys

import pytest
import torch

from drivedit_b200.config import get_config
from drivedit_b200.inference.rollout import StreamingRollout
from drivedit_b200.models.world_dit import PagedKVCacheSet, WorldDiT, make_kv_cache
from drivedit_b200.ops.kv_cache import PagedKVCache


def _model(*over):
    torch.manual_seed(0)
    cfg = get_config("tiny", ["model.n_layers=1", *over])
    return cfg, WorldDiT(cfg.model).eval()


@pytest.mark.parametrize("context,sinks,window,chunk,branches", [
    (1, 8, 4, 1, 16), (1, 16, 8, 4, 8), (2, 5, 1, 2, 9), (3, 3, 2, 1, 7), (4, 2, 2, 3, 5), (1, 3, 1, 1, 2),
])
def test_branched_streams_fit_their_pool(context, sinks, window, chunk, branches):
    """Streams that branch before, at and after the end of their sinks, past sinks + window."""
    _, m = _model()
    total = context + sinks + 2 * window + 4 * chunk
    cache = make_kv_cache(m, 2, window, chunk, "cpu", torch.float32, "fp8", sinks, total, branches, context)
    for f0 in range(0, context, chunk):
        cache.step(min(chunk, context - f0) * cache.tpf)
        cache.commit(min(chunk, context - f0))
    cache.branch(branches)
    while cache.frames < total:
        n = min(chunk, total - cache.frames)
        cache.step(n * cache.tpf)
        cache.commit(n)
    assert len(cache.seqs) == 2 * branches
    assert all(cache.cache.length(s) == total * cache.tpf for s in cache.seqs)


def test_branched_rollout_with_sinks_behind_the_context():
    cfg, m = _model()
    r = cfg.rollout
    r.chunk_frames, r.flow_steps, r.window_frames, r.kv_cache, r.sink_frames = 1, 1, 2, "fp8", 8
    roll = StreamingRollout(m, r)
    res = roll.run_branches(torch.randn(1, 1, 16, 16, 16), torch.zeros(1, 16, 14, 2), total_frames=14)
    assert res.frames.shape[:2] == (16, 14) and torch.isfinite(res.frames).all()


def test_types_the_cuda_cache_does_not_hold_are_refused_when_it_is_made():
    _, m = _model()
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(ValueError, match="bfloat16"):
            make_kv_cache(m, 1, 2, 1, torch.device("cuda"), dtype, "fp8")
    assert isinstance(make_kv_cache(m, 1, 2, 1, "cpu", torch.float32, "fp8"), PagedKVCacheSet)


def test_cpu_cache_needs_no_cuda_extension():
    code = """
import sys
sys.modules["drivedit_b200._C"] = None  # its import fails
import torch
from drivedit_b200.ops.kv_cache import PagedKVCache
c = PagedKVCache(1, 1, 8, device="cpu")
s = c.add(2)
step = c.begin(s, [70, 3])
x = torch.randn(2, 70, 1, 64)
step.write(0, x, x)
assert torch.isfinite(step.attend(0, x, causal="token")).all()
step.commit()
kids = c.fork(s, 2)
c.trim(kids, keep=4)
c.free(s), c.compact(), c.resize(16), c.copy(kids)
print(c.table(kids).tolist(), c.length(kids[0]))
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("70"), run.stderr[-2000:]


def test_cache_calls_take_no_gradients():
    """The cache holds codes: what is read from it has no gradient, on either device."""
    c = PagedKVCache(1, 1, 4, device="cpu")
    step = c.begin(c.add(1), 5)
    x = torch.randn(1, 5, 1, 64, requires_grad=True)
    step.write(0, x, x)
    o, lse = step.attend(0, x, causal="token", return_lse=True)
    assert not o.requires_grad and not lse.requires_grad
    assert not any(t.requires_grad for t in (c.k_scale, c.v_scale, *c.read(0, step.seqs[0])))


def test_sequences_grow_with_the_pool():
    """Without a bound of its own a sequence may take the pages that the pool has gained."""
    c = PagedKVCache(1, 1, 4, device="cpu")
    (s,) = c.add(1)
    old = c.begin([s], 256)
    old.commit()
    with pytest.raises(ValueError):
        c.begin([s], 1)
    c.resize(7)
    free = c.free_pages
    with pytest.raises(ValueError):
        c.begin([s], 1, max_tokens=old.max_tokens, out=old)  # its table is of the old size
    assert c.free_pages == free and c.length(s) == 256
    step = c.begin([s], 192)
    assert step.table.shape == (1, 7) and (step.table >= 0).all()
    step.commit()
    c.trim([s], keep=64)
    c.resize(4)
    assert c.table([s]).shape == (1, 7) and c.length(s) == 448
    with pytest.raises(ValueError):
        c.begin([s], 1)
    fixed = PagedKVCache(1, 1, 4, device="cpu", max_pages_per_seq=2)
    fixed.resize(8)
    with pytest.raises(ValueError):
        fixed.begin(fixed.add(1), 129)
