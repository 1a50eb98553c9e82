"""Windowed attention, the 8-bit paged cache and rollouts over it, in their PyTorch form."""
import math
import random

import pytest
import torch

from drivedit_b200.config import get_config
from drivedit_b200.inference.rollout import StreamingRollout
from drivedit_b200.layers.attention import window_mask
from drivedit_b200.models.world_dit import KVCacheSet, PagedKVCacheSet, WorldDiT, forward_cached
from drivedit_b200.ops.kv_cache import PagedKVCache, quantize_block
from drivedit_b200.ops.window_attention import window_attention


def _brute(q, k, v, causal, unit, window, sinks, q_off, kv_off):
    """One query at a time, by the definition, in fp64."""
    o = torch.zeros_like(q, dtype=torch.float64)
    for b in range(q.shape[0]):
        for t in range(q.shape[1]):
            f = (t + q_off) // unit
            see = [j for j in range(k.shape[1]) if causal == "none" or (
                (j + kv_off) // unit <= f and (not window or f - (j + kv_off) // unit < window or (j + kv_off) // unit < sinks))]
            if see:
                w = torch.softmax(torch.einsum("hd,shd->hs", q[b, t].double(), k[b, see].double()) / 8, -1)
                o[b, t] = torch.einsum("hs,shd->hd", w, v[b, see].double())
    return o


@pytest.mark.parametrize("T,S,causal,unit,window,sinks,q_off,kv_off", [
    (9, 9, "token", 1, 3, 2, 0, 0), (8, 20, "frame", 4, 2, 1, 12, 0), (7, 11, "token", 1, 2, 0, 1, 4),
    (5, 6, "none", 1, 0, 0, 0, 0), (6, 6, "frame", 100, 1, 0, 0, 0), (12, 12, "token", 1, 0, 0, 0, 0),
])
def test_window_attention_definition_and_gradients(T, S, causal, unit, window, sinks, q_off, kv_off):
    q = torch.randn(2, T, 2, 64, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(2, S, 2, 64, dtype=torch.float64, requires_grad=True) for _ in "kv")
    args = (causal, unit, window, sinks, q_off, kv_off)
    o, lse = window_attention(q, k, v, *args, return_lse=True)
    assert torch.allclose(o, _brute(q.detach(), k.detach(), v.detach(), *args), atol=1e-12)
    assert lse.shape == (2, 2, T)
    small = [x[:1, :, :1].detach().clone().requires_grad_(True) for x in (q, k, v)]
    assert torch.autograd.gradcheck(lambda *x: window_attention(*x, *args), small, fast_mode=True)


@pytest.mark.parametrize("q_off,kv_off", [(250, 0), (0, 50), (0, 400)])
def test_window_attention_hidden_rows(q_off, kv_off):
    """What queries without a key and keys without a query hold reaches nothing else."""
    args = ("token", 1, 60, 0, q_off, kv_off)
    q, k, v = (torch.randn(1, n, 2, 64, requires_grad=True) for n in (200, 300, 300))
    do = torch.randn(1, 200, 2, 64)
    seen = window_mask(200, 300, *args)
    rows, keys = ~seen.any(1), ~seen.any(0)
    o = window_attention(q, k, v, *args)
    want = (o, *torch.autograd.grad(o, (q, k, v), do))
    do[:, rows] = math.nan
    with torch.no_grad():
        q[:, rows] = math.nan
        k[:, keys] = math.nan
        v[:, keys] = math.nan
    o = window_attention(q, k, v, *args)
    assert all(torch.equal(a, b) for a, b in zip((o, *torch.autograd.grad(o, (q, k, v), do)), want))


def test_window_attention_refusals():
    q, k = torch.randn(1, 4, 2, 64), torch.randn(1, 6, 2, 64)
    for bad in (lambda: window_attention(q[..., :32], k[..., :32], k[..., :32]),
                lambda: window_attention(q, k[:, :, :1], k[:, :, :1]),
                lambda: window_attention(q, k, k[:, :5]),
                lambda: window_attention(q, k.double(), k.double()),
                lambda: window_attention(q, k, k, "block"),
                lambda: window_attention(q, k, k, "none", window=2),
                lambda: window_attention(q, k, k, "frame", 0),
                lambda: window_attention(q, k, k, "token", window=-1),
                lambda: window_attention(q, k, k, "token", sinks=-1),
                lambda: window_attention(q, k, k, q_pos_offset=-1),
                lambda: window_attention(q, k, k, q_pos_offset=1 << 30),
                lambda: window_attention(q, k, k, scale=0.0),
                lambda: window_attention(q, k, k, scale=math.inf)):
        with pytest.raises(ValueError):
            bad()


def test_extension_errors_name_numbers():
    """Errors of the extension that print numbers reach Python (its C++ library is the one that
    torch uses)."""
    from drivedit_b200.ops import _ext
    if not _ext.available():
        pytest.skip("extension not built")
    q = torch.randn(1, 4, 1, 64).bfloat16()
    for args, text in ((("token", 1, 0, 0, 1 << 30, 0, None), "1073741824"), (("token", 1, 0, 0, 0, 0, math.inf), "finite"),
                       (("frame", 1 << 25, 0, 0, 0, 0, None), "2\\^24"), (("block", 1, 0, 0, 0, 0, None), "block")):
        with pytest.raises(ValueError, match=text):
            _ext.ext().window_attention(q, q, q, *args)
    with pytest.raises(ValueError, match=r"\[1, 4, 1, 32\]"):
        _ext.ext().window_attention(q[..., :32], q, q, "token", 1, 0, 0, 0, 0, None)


def test_quantize_block_definition():
    torch.manual_seed(0)
    x = torch.randn(7, 64, 64) * torch.logspace(-12, 12, 7)[:, None, None]
    x[3, 0, 0] = 448 * 2.0 ** 5
    x[5] = 0
    codes, scale = quantize_block(x)
    for i in range(7):
        top = float(x[i].abs().max())
        e = -100 if top == 0 else math.ceil(math.log2(top / 448))
        assert float(scale[i]) == 2.0 ** e
        held, want = codes[i].double() * float(scale[i]), x[i].double()
        # half a step of 3 stored bits, or of the smallest step
        assert ((held - want).abs() <= (2.0 ** -4 * want.abs()).clamp_min(2.0 ** (e - 10))).all()
    x = torch.tensor([[math.inf, -math.inf, math.nan, 1.0]])
    codes, scale = quantize_block(x)
    assert float(scale) == 2.0 ** -8 and codes.float().tolist()[0][:2] == [448.0, -448.0] and codes.float()[0, 2].isnan()


def _write(c, seqs, n, commit=True, seed=None):
    g = torch.Generator().manual_seed(seed) if seed is not None else None
    T = max(n) if isinstance(n, list) else n
    step = c.begin(seqs, n)
    k, v = (torch.randn(len(seqs), T, c.n_heads, 64, generator=g) for _ in "kv")
    for layer in range(c.n_layers):
        step.write(layer, k, v)
    if commit:
        step.commit()
    return step, k, v


def test_cache_holds_what_is_written_and_unfinished_pages_are_kept():
    c = PagedKVCache(1, 2, 12, device="cpu")
    seqs = c.add(2)
    _, k1, v1 = _write(c, seqs, [70, 3])
    before = [c.read(0, s) for s in seqs]
    _write(c, seqs, [9, 64], commit=False)   # abandoned
    _, k2, v2 = _write(c, seqs, [1, 64])
    for i, (a, b) in enumerate(([70, 1], [3, 64])):
        k, v = c.read(0, seqs[i])
        assert k.shape == (a + b, 2, 64)
        for got, old, new, new1 in ((k, before[i][0], k2, k1), (v, before[i][1], v2, v1)):
            step = got[:a].abs().clamp_min(2.0 ** -9 * 0.02)
            # re-coded once more at most: two half steps of the input's own coding
            assert ((got[:a] - new1[i, :a]).abs() <= 2 * 2.0 ** -4 * step + 2e-4).all()
            assert ((got[a:] - new[i, :b]).abs() <= 2.0 ** -4 * new[i, :b].abs() + 2e-4).all()


def test_fork_shares_pages_and_writes_apart():
    c = PagedKVCache(2, 1, 14, device="cpu")
    (s,) = c.add(1)
    _write(c, [s], 100)
    kids = c.fork([s], 3)
    assert c.free_pages == 12 and c.length(kids[0]) == 100
    old = c.read(1, s)
    _, k, _ = _write(c, kids, [1, 40, 0])
    # the unfinished page is copied for the two that write (the parent holds it too), one
    # page more for the 140 tokens
    assert c.free_pages == 12 - 3
    assert all(torch.equal(a, b) for a, b in zip(c.read(1, s), old))
    assert torch.equal(c.read(1, kids[1])[0][:64], old[0][:64])
    assert c.length(kids[1]) == 140 and c.length(kids[2]) == 100
    t = c.table([s] + kids)
    assert t[0, 0] == t[1, 0] == t[2, 0] == t[3, 0] and len({int(x) for x in t[:3, 1]}) == 3 and t[3, 1] == t[0, 1]
    c.free([s])
    _write(c, [kids[2]], 1)      # the last owner writes in place
    assert int(c.table([kids[2]])[0, 1]) == int(t[0, 1])
    c.free(kids)
    assert c.free_pages == 14 and c.sequences == []


def test_two_of_one_fork_in_one_step_keep_one_page():
    c = PagedKVCache(1, 1, 3, device="cpu")
    (s,) = c.add(1)
    _write(c, [s], 10)
    kids = c.fork([s], 2)
    c.free([s])
    _write(c, kids, 1)           # one copy, the other keeps the page
    assert c.free_pages == 1


def test_copy_compact_resize():
    c = PagedKVCache(2, 2, 20, device="cpu")
    seqs = c.add(3)
    for n in (65, 100, 30):
        _write(c, seqs, n)
    want = {s: [c.read(l, s) for l in range(2)] for s in seqs}
    more = c.copy(seqs[1:])
    c.free(seqs[:2])
    want.update({m: want[s] for m, s in zip(more, seqs[1:])})
    live = [seqs[2]] + more
    used = c.compact()
    assert used == 12 and sorted(int(p) for p in c.table(live).flatten() if p >= 0) == list(range(12))
    c.resize(12)
    assert c.n_pages == 12 and c.free_pages == 0 and c.k.shape[1] == 12
    with pytest.raises(ValueError):
        c.resize(11)
    c.resize(13)
    for s in live:
        for l in range(2):
            assert all(torch.equal(a, b) for a, b in zip(c.read(l, s), want[s][l]))
    _write(c, [live[0]], 2)


def test_trim_frees_pages_and_hides_tokens():
    c = PagedKVCache(1, 1, 10, device="cpu")
    (s,) = c.add(1)
    _write(c, [s], 400)
    k, v = c.read(0, s)
    c.trim([s], keep=100, sinks=10)      # tokens 10..299 go: pages 1-3 whole, parts of 0 and 4
    assert c.free_pages == 3 + 3
    step, nk, nv = _write(c, [s], 5, commit=False)
    q = torch.randn(1, 5, 2, 64)
    o = step.attend(0, q, causal="token")
    keep = torch.cat([torch.arange(10), torch.arange(300, 405)])
    kk, vv = c._values(0, c._seqs[s], 405)
    ref = _brute(q, kk[keep][None].repeat_interleave(2, 2), vv[keep][None].repeat_interleave(2, 2), "token", 1, 0, 0, 110, 0)
    assert torch.allclose(o.double(), ref, atol=1e-5)
    for call in (lambda: c.trim([s], 50, 11), lambda: step.attend(0, q, causal="token", window=20, sinks=4)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("seed", range(4))
def test_random_bookkeeping_keeps_every_sequence(seed):
    """Random calls against plain lists of tokens (whole numbers up to 15, exact in 8 bits);
    every page is held by as many sequences as the count says, a free one by none."""
    rng = random.Random(seed)
    c = PagedKVCache(1, 1, 60, device="cpu", max_pages_per_seq=12)
    held = {}  # sequence: (tokens, first, sinks)

    def check():
        counts = [0] * c.n_pages
        for i, (tokens, first, sinks) in held.items():
            assert c.length(i) == len(tokens)
            k, v = c.read(0, i)
            want = torch.tensor(tokens, dtype=torch.float32)
            if first > sinks:
                want[sinks:first] = 0
            assert torch.equal(k[:, 0, 0], want) and torch.equal(v[:, 0, 63], -want)
            s = c._seqs[i]
            for p in s.pages:
                if p >= 0:
                    counts[p] += 1
        assert c._refs.tolist() == counts and c.free_pages == counts.count(0) and c.sequences == sorted(held)

    for _ in range(150):
        some = rng.sample(sorted(held), rng.randint(0, min(3, len(held))))
        what = rng.choice(["add", "step", "step", "step", "step", "fork", "copy", "free", "trim", "compact", "resize"])
        try:
            if what == "add" and len(held) < 6:
                held.update((i, ([], 0, 0)) for i in c.add(rng.randint(1, 2)))
            elif what == "step":
                new = [rng.choice([0, 1, 1, 5, 64, 130]) for _ in some]
                step = c.begin(some, new)
                x = torch.zeros(len(some), max(new, default=0), 1, 64)
                for r, n in enumerate(new):
                    x[r, :n] = torch.randint(1, 16, (n, 1, 1)).float()
                step.write(0, x, -x)
                if rng.random() < 0.7:
                    step.commit()
                    held.update((i, (held[i][0] + x[r, :n, 0, 0].int().tolist(), *held[i][1:])) for r, (i, n) in enumerate(zip(some, new)))
            elif what == "fork" and len(held) < 8:
                held.update(zip(c.fork(some, 2), [held[i] for i in some for _ in "12"]))
            elif what == "copy" and len(held) < 8:
                held.update(zip(c.copy(some), [held[i] for i in some]))
            elif what == "free":
                c.free(some)
                for i in some:
                    del held[i]
            elif what == "trim":
                c.trim(some, keep := rng.choice([0, 30, 100, 200]), sinks := rng.choice([0, 10]))
                held.update((i, (t, f, sinks) if (f := max(first, len(t) - keep)) > sinks else (t, first, old))
                            for i, (t, first, old) in [(i, held[i]) for i in some])
            elif what == "compact":
                assert c.compact() == c.n_pages - c.free_pages
                assert not c._refs[c.n_pages - c.free_pages:].any()
            elif what == "resize":
                c.resize(rng.choice([50, 60, 70]))
        except (RuntimeError, ValueError):  # no room, or other sinks than before: nothing has changed
            pass
        check()


def test_cache_refusals_change_nothing():
    c = PagedKVCache(1, 2, 4, device="cpu", max_pages_per_seq=3)
    a, b = c.add(2)
    step, k, v = _write(c, [a], 100)
    state = lambda: (c.free_pages, [(s.pages.tolist(), s.length, s.version) for s in c._seqs.values()], c._refs.tolist())  # noqa: E731
    was = state()
    q = torch.randn(1, 100, 2, 64)
    for error, call in (
            (RuntimeError, lambda: step.write(0, k, v)),                   # stale
            (RuntimeError, lambda: step.attend(0, q)),
            (RuntimeError, lambda: step.commit()),
            (RuntimeError, lambda: c.begin([a, b], [1, 190])),             # out of pages
            (RuntimeError, lambda: c.copy([a, b]) and c.copy([a, b])),
            (ValueError, lambda: c.begin([a], 100)),                       # past max_pages_per_seq
            (ValueError, lambda: c.begin([a, a], 1)),
            (ValueError, lambda: c.begin([a, b], [1])),
            (ValueError, lambda: c.begin([a], -1)),
            (ValueError, lambda: c.begin([77], 1)),
            (ValueError, lambda: c.begin([a], 1, max_tokens=100)),
            (ValueError, lambda: c.free([a, a])),
            (ValueError, lambda: c.free([a, 9])),
            (ValueError, lambda: c.fork([a], -1)),
            (ValueError, lambda: c.trim([a], -1)),
            (ValueError, lambda: c.read(1, a)),
            (ValueError, lambda: c.resize(1)),
            (ValueError, lambda: PagedKVCache(1, 1, 0, device="cpu"))):
        with pytest.raises(error):
            call()
        if c.sequences != [a, b]:
            c.free([s for s in c.sequences if s not in (a, b)])
        assert state() == was
    step = c.begin([a, b], [2, 3])
    k, v = torch.randn(2, 3, 2, 64), torch.randn(2, 3, 2, 64)
    for call in (lambda: step.write(1, k, v), lambda: step.write(0, k[:1], v[:1]), lambda: step.write(0, k[:, :2], v[:, :2]),
                 lambda: step.write(0, k[:, :, :1], v[:, :, :1]), lambda: step.write(0, k, v[:, :, :, :32]),
                 lambda: step.attend(0, torch.randn(2, 3, 3, 64)), lambda: step.attend(0, k, causal="x"),
                 lambda: step.attend(0, k, causal="none", window=3), lambda: step.attend(0, k, tokens_per_frame=0),
                 lambda: step.attend(0, k, scale=-1.0), lambda: c.begin([a], 1, out=step),
                 lambda: c.begin([a, b], [9, 9], max_tokens=500, out=step)):
        with pytest.raises(ValueError):
            call()


def _model(*over, layers=2):
    torch.manual_seed(0)
    cfg = get_config("tiny", [f"model.n_layers={layers}", *over])
    m = WorldDiT(cfg.model)
    with torch.no_grad():
        for p in m.parameters():
            if p.abs().sum() == 0:
                p.normal_(0, 0.02)
    return cfg, m


def _data(B, F):
    return torch.randn(B, F, 16, 16, 16), torch.rand(B), torch.rand(B, F, 2)


def test_windowed_model_chunks_equal_full_forward():
    """A model trained with a window and no sinks streams through the rolling buffers with the
    same outputs; a window as long as the clip changes nothing."""
    _, m = _model("model.window_frames=2")
    x, t, a = _data(2, 6)
    full = m(x, t, a)
    cache = KVCacheSet(m, 2, window_frames=4, chunk_frames=2, device="cpu", dtype=torch.float32)
    outs = [forward_cached(m, x[:, f:f + 2], t, a[:, f:f + 2], cache, commit=True) for f in (0, 2, 4)]
    assert torch.allclose(torch.cat(outs, 1), full, atol=1e-4)
    _, wide = _model("model.window_frames=6")
    _, plain = _model()
    assert torch.allclose(wide(x, t, a), plain(x, t, a), atol=1e-5)
    assert not torch.allclose(full, plain(x, t, a), atol=1e-4)


@pytest.mark.parametrize("over", [("model.window_frames=2", "model.sink_frames=1"), ()])
def test_paged_stream_near_full_forward(over):
    """The paged window with sinks against the model's own full forward: what differs is the
    8-bit cache's rounding (2^-4 of a key's or value's element, averaged over a head)."""
    _, m = _model(*over)
    x, t, a = _data(2, 6)
    full = m(x, t, a)
    cache = PagedKVCacheSet(m, 2, window_frames=6, chunk_frames=2, device="cpu", sink_frames=m.cfg.sink_frames, max_frames=6)
    outs = [forward_cached(m, x[:, f:f + 2], t, a[:, f:f + 2], cache, commit=True) for f in (0, 2, 4)]
    got = torch.cat(outs, 1)
    assert (got - full).norm() / full.norm() < 2.0 ** -4
    trimmed = PagedKVCacheSet(m, 2, window_frames=2, chunk_frames=2, device="cpu", sink_frames=m.cfg.sink_frames, max_frames=6)
    again = torch.cat([forward_cached(m, x[:, f:f + 2], t, a[:, f:f + 2], trimmed, commit=True) for f in (0, 2, 4)], 1)
    if over:  # what trimming drops, the model's window hides
        assert torch.equal(again, got)


def test_rollout_of_a_context_longer_than_asked():
    cfg, m = _model()
    r = cfg.rollout
    r.total_frames, r.chunk_frames, r.flow_steps, r.window_frames, r.kv_cache = 2, 2, 1, 3, "fp8"
    ctx = torch.randn(1, 14, 16, 16, 16)
    assert torch.equal(StreamingRollout(m, r).run(ctx, torch.rand(1, 14, 2)).frames, ctx)


def test_rollout_over_the_paged_cache_and_branches():
    cfg, m = _model()
    r = cfg.rollout
    r.total_frames, r.chunk_frames, r.flow_steps, r.window_frames, r.kv_cache, r.sink_frames = 8, 2, 2, 3, "fp8", 1
    ctx, act = torch.randn(2, 2, 16, 16, 16), torch.rand(2, 3, 8, 2)
    act[:, :, :2] = act[:, :1, :2]
    roll = StreamingRollout(m, r)
    res = roll.run_branches(ctx, act, generator=torch.Generator().manual_seed(1))
    assert res.frames.shape == (6, 8, 16, 16, 16) and torch.equal(res.frames[1, :2], ctx[0])
    # the same streams, each with a context of its own
    one = roll.run(ctx.repeat_interleave(3, 0), act.flatten(0, 1), generator=torch.Generator().manual_seed(1))
    assert torch.allclose(one.frames, res.frames, atol=1e-4)
    r.kv_cache = "bf16"
    for call in (lambda: roll.run_branches(ctx, act), lambda: roll.run(ctx, act[:, 0])):
        with pytest.raises(ValueError):
            call()
    r.sink_frames, r.kv_cache = 0, "int4"
    with pytest.raises(ValueError):
        roll.run(ctx, act[:, 0])


def test_model_refusals():
    for over in (("model.sink_frames=1",), ("model.window_frames=-1",), ("model.window_frames=2", "model.causal=none"),
                 ("model.window_frames=2", "model.attention=sla")):
        with pytest.raises(ValueError):
            _model(*over)
    _, m = _model("model.window_frames=2", "model.sink_frames=1")
    with pytest.raises(ValueError):
        KVCacheSet(m, 1, 4, 2, "cpu", torch.float32)
    with pytest.raises(ValueError):
        PagedKVCacheSet(m, 1, 4, 2, "cpu", sink_frames=2)


def test_closed_loop_and_pipeline_over_the_paged_cache():
    from drivedit_b200.evaluation.closed_loop import ClosedLoopEvaluator, EvaluationConfig
    from drivedit_b200.inference.pipeline import InferencePipeline, PipelineConfig
    _, m = _model("model.window_frames=3", "model.sink_frames=1")
    ev = ClosedLoopEvaluator(m, EvaluationConfig(flow_steps=1, window_frames=4, kv_cache="fp8", max_episode_steps=8), device="cpu")
    ev._initialize_context(torch.randn(2, 16, 16, 16))
    for _ in range(7):
        frame = ev._predict_next(torch.zeros(2))
        assert torch.isfinite(frame).all()
    assert ev.cache.frames >= 2 and ev.cache.cache.length(ev.cache.seqs[0]) == 9 * 64
    with pytest.raises(ValueError):
        ClosedLoopEvaluator(m, EvaluationConfig(), device="cpu")._initialize_context(torch.randn(16, 16, 16))
    pipe = InferencePipeline(PipelineConfig(device="cpu", model_preset="tiny", model_overrides=["model.n_layers=1"], use_vae=False,
                                            chunk_frames=2, flow_steps=1, window_frames=2, kv_cache="fp8", sink_frames=1))
    res = pipe.rollout.run(torch.randn(1, 1, 16, 16, 16), torch.zeros(1, 7, 2), total_frames=7)
    assert res.frames.shape[1] == 7 and torch.isfinite(res.frames).all()
