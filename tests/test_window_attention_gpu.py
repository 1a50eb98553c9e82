"""Windowed attention (window and first tokens) on the GPU, forward and backward, against the
formula in 64 bits and against differences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _bits(*shape, scale=1.0):
    return (torch.randn(*shape, device="cuda") * scale).bfloat16()


def _seen(T, S, causal, unit, window, sinks, q_off, kv_off):
    q = torch.arange(q_off, q_off + T, device="cuda")[:, None] // unit
    k = torch.arange(kv_off, kv_off + S, device="cuda")[None] // unit
    if causal == "none":
        return torch.ones(T, S, dtype=torch.bool, device="cuda")
    seen = k <= q
    return seen & ((q - k < window) | (k < sinks)) if window else seen


def _formula(q, k, v, do, seen, scale):
    """o, lse (log2), dq, dk, dv in 64 bits, and a bound on each one's error.

    The kernels round the weights P and the score gradients dS to bf16 (half a step is
    2^-8 of the value), sum in fp32, subtract delta = sum(dO * O) with O rounded to bf16
    (2^-8), and round the results to bf16 (2^-8). fp32 sums and exponentials: under
    2^-12 of the magnitudes summed. So, with |.| the products of magnitudes:
      o:  2^-8 |o| + (2^-8 + 2^-12) P |v|
      dv: 2^-8 |dv| + (2^-8 + 2^-12) P^T |dO|
      dS: P (2^-12 |dO||V|^T + 2^-8 |dO|.|O|) + 2^-8 |dS|, and dq, dk take it through |K|, |Q|."""
    q, k, v, do = (x.double().transpose(1, 2) for x in (q, k, v, do))
    s = (q @ k.mT * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - lse[..., None]), 0.0)
    o = p @ v
    dp = do @ v.mT
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    # a seen score off by a little moves P by as much, relatively
    off = 2.0 ** -12 * (1 + (q.abs() @ k.abs().mT).amax() * scale * 2.0 ** -5)
    r = 2.0 ** -8
    e_p = p * (r + off)
    e_ds = p * scale * (2.0 ** -12 * (do.abs() @ v.abs().mT) + r * (do.abs() * o.abs()).sum(-1, keepdim=True)
                        + off * (dp - delta).abs()) + r * ds.abs()
    out = {"o": (o, r * o.abs() + e_p @ v.abs()), "dq": (ds @ k, e_ds @ k.abs()), "dk": (ds.mT @ q, e_ds.mT @ q.abs()),
           "dv": (p.mT @ do, e_p.mT @ do.abs())}
    return {n: (x.transpose(1, 2), (b + (r * x.abs() if n != "o" else 0) + 1e-30).transpose(1, 2)) for n, (x, b) in out.items()}, lse / math.log(2)


CASES = [
    # B, T, S, H, causal, unit, window, sinks, q_off, kv_off
    (1, 1, 1, 1, "token", 1, 1, 0, 0, 0),
    (2, 130, 130, 3, "token", 1, 0, 0, 0, 0),
    (2, 257, 257, 2, "token", 1, 1, 0, 0, 0),
    (1, 1003, 1003, 2, "token", 1, 257, 4, 0, 0),
    (2, 320, 320, 2, "token", 1, 128, 128, 0, 0),
    (1, 700, 700, 1, "token", 1, 100, 300, 0, 0),
    (2, 490, 490, 2, "frame", 49, 3, 1, 0, 0),
    (1, 1024, 1024, 2, "frame", 128, 2, 1, 0, 0),
    (1, 768, 768, 1, "frame", 256, 1, 0, 0, 0),
    (3, 100, 300, 2, "none", 1, 0, 0, 0, 0),
    (2, 64, 900, 2, "token", 1, 200, 7, 836, 0),
    (1, 200, 500, 2, "frame", 64, 2, 1, 300, 0),
    (1, 50, 70, 2, "token", 1, 5, 0, 10, 30),       # the first rows see nothing, many keys are seen by none
    (1, 300, 200, 1, "token", 1, 60, 20, 0, 0),     # the last rows see the sinks only
    (1, 300, 200, 1, "token", 1, 60, 0, 0, 0),      # the last rows see nothing
    (2, 33, 40, 1, "frame", 1000, 1, 1, 0, 0),
    (1, 2048, 2048, 1, "frame", 512, 1, 1, 0, 0),
    (1, 140, 2000, 2, "token", 1, 1700, 3, 1860, 0),
    (1, 200, 400, 1, "token", 1, 3, 9, 500, 100),   # sinks before the first key
]


def _inputs(B, T, S, H, packed):
    if packed and T == S:
        return _bits(B, T, 3, H, 64).unbind(2)
    if packed:  # heads before tokens, and rows further apart
        return (_bits(B, H, T, 64).transpose(1, 2), *_bits(B, S, H, 2, 72)[..., :64].unbind(3))
    return _bits(B, T, H, 64), _bits(B, S, H, 64), _bits(B, S, H, 64)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_matches_formula(case, packed):
    from drivedit_b200.ops.window_attention import window_attention
    B, T, S, H, causal, unit, window, sinks, q_off, kv_off = case
    q, k, v = (x.detach().requires_grad_(True) for x in _inputs(B, T, S, H, packed))
    do = _bits(B, H, T, 64).transpose(1, 2) if packed else _bits(B, T, H, 64)
    o, lse = window_attention(q, k, v, causal, unit, window, sinks, q_off, kv_off, return_lse=True)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)), o=o.detach())
    seen = _seen(T, S, causal, unit, window, sinks, q_off, kv_off)
    want, rlse = _formula(q.detach(), k.detach(), v.detach(), do, seen, 0.125)
    for n, (x, bound) in want.items():
        assert got[n].dtype == torch.bfloat16 and got[n].shape == x.shape
        err = (got[n].double() - x).abs()
        assert (err <= bound).all(), (n, float((err / bound).max()))
    assert torch.equal(torch.isfinite(rlse), torch.isfinite(lse))
    mag = float((q.detach().double().transpose(1, 2).abs() @ k.detach().double().transpose(1, 2).abs().mT).amax()) * 0.125
    fin = torch.isfinite(rlse)
    if fin.any():  # fp32 products of 64 terms, exponential and logarithm, times log2(e)
        assert (lse.double() - rlse)[fin].abs().max() <= 1.45 * (mag * 2.0 ** -18 + 2.0 ** -19)


@pytest.mark.parametrize("splits", [2, 3, 5, 8])
def test_split_keys(splits):
    from drivedit_b200.ops._ext import ext
    from drivedit_b200.ops.window_attention import window_attention
    q, k, v = _bits(1, 150, 2, 64), _bits(1, 2100, 2, 64), _bits(1, 2100, 2, 64)
    args = ("token", 1, 1500, 130, 1950)
    want, wl = window_attention(q, k, v, *args, return_lse=True)
    prev = ext().attn_fwd_set_kv_splits(splits)
    try:
        o, lse = window_attention(q, k, v, *args, return_lse=True)
    finally:
        ext().attn_fwd_set_kv_splits(prev)
    ref, _ = _formula(q, k, v, torch.zeros_like(q), _seen(150, 2100, "token", 1, 1500, 130, 1950, 0), 0.125)
    assert ((o.double() - ref["o"][0]).abs() <= ref["o"][1]).all()
    assert (lse - wl).abs().max() < 1e-4


def test_hidden_keys_do_not_matter():
    """NaN in keys and values that no query sees (before the window, between sinks and window,
    behind the last query), in the same tiles as visible ones; the samples next to them."""
    from drivedit_b200.ops.window_attention import window_attention
    B, T, S, H = 3, 100, 1000, 2
    q, k, v = (x.requires_grad_(True) for x in (_bits(B, T, H, 64), _bits(B, S, H, 64), _bits(B, S, H, 64)))
    do = _bits(B, T, H, 64)
    args = ("token", 1, 150, 5, 850)
    hidden = ~_seen(T, S, "token", 1, 150, 5, 850, 0).any(0)
    assert 0 < hidden.sum() < S
    o = window_attention(q, k, v, *args)
    want = (o, *torch.autograd.grad(o, (q, k, v), do))
    with torch.no_grad():
        k[:, hidden] = math.nan
        v[:, hidden] = math.nan
    o = window_attention(q, k, v, *args)
    got = (o, *torch.autograd.grad(o, (q, k, v), do))
    assert torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):
        # dq is summed in another order: one rounding of bf16 apart at most
        assert torch.isfinite(a).all() and ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-5).all()
    assert not got[2][:, hidden].any() and not got[3][:, hidden].any()


@pytest.mark.parametrize("q_off,kv_off,unit", [(0, 50, 1), (0, 130, 1), (250, 0, 1), (40, 100, 20), (1000, 0, 1), (0, 400, 1)])
def test_hidden_queries_do_not_matter(q_off, kv_off, unit):
    """NaN in queries that see no key (before the first key, behind the window of the last),
    in the same tiles as others, and in the gradients of their outputs."""
    from drivedit_b200.ops.window_attention import window_attention
    B, T, S, H = 2, 200, 300, 2
    q, k, v = (x.requires_grad_(True) for x in (_bits(B, T, H, 64), _bits(B, S, H, 64), _bits(B, S, H, 64)))
    do = _bits(B, T, H, 64)
    args = ("frame", unit, 60 // unit, 0, q_off, kv_off)
    hidden = ~_seen(T, S, "frame", unit, 60 // unit, 0, q_off, kv_off).any(1)
    assert hidden.any()
    o = window_attention(q, k, v, *args)
    want = (o, *torch.autograd.grad(o, (q, k, v), do))
    do[:, hidden] = math.nan
    with torch.no_grad():
        q[:, hidden] = math.nan
    o = window_attention(q, k, v, *args)
    got = (o, *torch.autograd.grad(o, (q, k, v), do))
    assert torch.equal(got[0], want[0]) and not got[0][:, hidden].any() and not got[1][:, hidden].any()
    for a, b in zip(got[1:], want[1:]):
        # dq is summed in another order: one rounding of bf16 apart at most
        assert torch.isfinite(a).all() and ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-5).all()


@pytest.mark.parametrize("window", [0, 300])
def test_equal_backward_passes_agree(window):
    """Many launches over many CTAs: dK and dV are summed in a fixed order, so each pass gives
    the same bits (a race for a barrier or for TMEM would not), and the status stays clean."""
    from drivedit_b200.ops._ext import check_device_status
    from drivedit_b200.ops.window_attention import window_attention
    q, k, v = (_bits(2, 2048, 12, 64).requires_grad_(True) for _ in "qkv")
    do = _bits(2, 2048, 12, 64)
    o = window_attention(q, k, v, "token", window=window, sinks=64 if window else 0)
    _, dk, dv = torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
    for _ in range(300):
        _, dk2, dv2 = torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
        assert torch.equal(dk, dk2) and torch.equal(dv, dv2)
    check_device_status()


def test_gradient_against_differences():
    """Directional differences of the forward kernel's own output, in a direction along which
    it is smooth: bf16 inputs moved by whole steps."""
    from drivedit_b200.ops.window_attention import window_attention
    torch.manual_seed(2)
    args = ("frame", 32, 2, 1)
    x = [_bits(1, 320, 2, 64) for _ in range(3)]
    do = _bits(1, 320, 2, 64)
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(window_attention(*leaves, *args), leaves, do)
    for i in range(3):
        d = torch.randn(1, 320, 2, 64, device="cuda")
        h = 2.0 ** -4
        moved = [[t + (s * h * d).bfloat16() if j == i else t for j, t in enumerate(x)] for s in (1, -1)]
        step = (moved[0][i].double() - moved[1][i].double())
        f = [(window_attention(*m, *args).double() * do.double()).sum() for m in moved]
        want = (grads[i].double() * step).sum()
        # outputs are rounded at random: 2^-9 of |o do| a term, over 40960 terms of unit size,
        # root sum of squares 0.4 a side; the third derivative leaves less than that
        noise = 2.0 ** -9 * math.sqrt(320 * 2 * 64) * 4
        assert abs(f[0] - f[1] - want) <= noise + 0.02 * (grads[i].double() * step).abs().pow(2).sum().sqrt() * 10


def test_only_some_inputs_need_gradients_and_shared_input():
    from drivedit_b200.ops.window_attention import window_attention
    q, kv = _bits(1, 90, 2, 64), _bits(1, 90, 2, 64).requires_grad_(True)
    do = _bits(1, 90, 2, 64)
    (both,) = torch.autograd.grad(window_attention(q, kv, kv, "token", window=9), kv, do)
    k, v = kv.detach().clone().requires_grad_(True), kv.detach().clone().requires_grad_(True)
    gk, gv = torch.autograd.grad(window_attention(q, k, v, "token", window=9), (k, v), do)
    assert torch.equal(both, gk + gv)
    one = _bits(1, 90, 1, 64).requires_grad_(True)  # one head broadcast to all
    (g,) = torch.autograd.grad(window_attention(q, one.expand(1, 90, 2, 64), v, "token", window=9), one, do)
    (gx,) = torch.autograd.grad(window_attention(q, e := one.detach().expand(1, 90, 2, 64).clone().requires_grad_(True), v, "token", window=9), e, do)
    assert torch.equal(g, gx.sum(2, keepdim=True))


def test_captured_forward_and_backward():
    from drivedit_b200.ops.window_attention import window_attention
    x = [_bits(2, 200, 2, 64).requires_grad_(True) for _ in range(3)]
    do = _bits(2, 200, 2, 64)

    def run():
        o = window_attention(*x, "token", window=70, sinks=3)
        return (o, *torch.autograd.grad(o, x, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs share no workspace
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    with torch.no_grad():
        for t in (*x, do):
            t.copy_(_bits(2, 200, 2, 64))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    want = run()
    for out in outs:
        assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2]) and torch.equal(out[3], want[3])
        assert (out[1].float() - want[1].float()).abs().max() <= 2.0 ** -7 * want[1].float().abs().max()


def test_capture_beside_an_eager_graph_is_refused():
    from drivedit_b200.ops.window_attention import window_attention
    x = _bits(1, 64, 1, 64).requires_grad_(True)
    alive = window_attention(x, x, x, "token")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="default stream"):
            window_attention(x, x, x, "token")
        window_attention(x.detach(), x.detach(), x.detach(), "token")
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (g,) = torch.autograd.grad(window_attention(x, x, x, "token"), x, torch.ones_like(x))
    graph.replay()
    torch.cuda.synchronize()
    (w,) = torch.autograd.grad(window_attention(x, x, x, "token"), x, torch.ones_like(x))
    assert (g.float() - w.float()).abs().max() <= 2.0 ** -7 * w.float().abs().max()


def test_empty_inputs():
    from drivedit_b200.ops.window_attention import window_attention
    q, k = _bits(2, 5, 1, 64).requires_grad_(True), _bits(2, 0, 1, 64).requires_grad_(True)
    o, lse = window_attention(q, k, k, "token", return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    gq, gk = torch.autograd.grad(o, (q, k), torch.ones_like(o))
    assert not gq.any() and gk.shape == k.shape
    assert window_attention(q[:, :0], _bits(2, 4, 1, 64), _bits(2, 4, 1, 64)).shape == (2, 0, 1, 64)
    assert window_attention(q[:0], _bits(0, 4, 1, 64), _bits(0, 4, 1, 64)).shape == (0, 5, 1, 64)


def test_status_clean():
    from drivedit_b200.ops._ext import device_status
    torch.cuda.synchronize()
    assert device_status() == 0


def _world(*over, frames=4):
    from drivedit_b200.config import get_config
    from drivedit_b200.models.world_dit import WorldDiT
    torch.manual_seed(0)
    cfg = get_config("tiny", ["model.n_layers=2", f"train.frames={frames}", *over])
    m = WorldDiT(cfg.model)
    with torch.no_grad():
        for p in m.parameters():
            if p.abs().sum() == 0:
                p.normal_(0, 0.02)
    return cfg, m


@pytest.mark.parametrize("over", [("model.window_frames=2", "model.sink_frames=1"),
                                  ("model.window_frames=2", "model.causal=token")])
def test_windowed_model_trains_on_the_kernels(over):
    """The flagship's fused forward and backward with a window against its PyTorch path."""
    cfg, m = _world(*over, frames=6)
    m = m.cuda()
    x, t, a = torch.randn(2, 6, 16, 16, 16, device="cuda"), torch.rand(2, device="cuda"), torch.rand(2, 6, 2, device="cuda")
    w = torch.randn(2, 6, 16, 16, 16, device="cuda")
    ref = m(x, t, a)
    (ref * w).sum().backward()
    names = ["blocks.0.attn.qkv.weight", "blocks.1.attn.qkv.weight", "blocks.0.attn.proj.weight"]
    want = {n: p.grad.clone() for n, p in m.named_parameters() if n in names}
    m.zero_grad(set_to_none=True)
    m.enable_fused()
    m.fused.group.grad.zero_()
    got = m(x, t, a)
    # bf16 activations (2^-8 a rounding, about 20 in a row in two blocks) against fp32
    assert (got.float() - ref).norm() / ref.norm() < 20 * 2.0 ** -9
    (got.float() * w).sum().backward()
    for n, p in m.named_parameters():
        if n in names:
            assert (p.grad - want[n]).norm() / want[n].norm() < 40 * 2.0 ** -9, n


def test_streams_on_the_kernels_match_the_pytorch_form():
    """A chunked stream on the GPU, bf16 buffers and 8-bit pages, with a window and sinks."""
    from drivedit_b200.models.world_dit import KVCacheSet, PagedKVCacheSet, forward_cached
    x, t, a = torch.randn(2, 6, 16, 16, 16), torch.rand(2), torch.rand(2, 6, 2)
    for over, sinks in ((("model.window_frames=2",), 0), (("model.window_frames=2", "model.sink_frames=1"), 1), ((), 1)):
        outs = []
        for dev, dt in (("cpu", torch.float32), ("cuda", torch.bfloat16)):
            cfg, m = _world(*over)
            m = m.to(dev)
            if dev == "cuda":
                m.enable_fused()
            caches = [PagedKVCacheSet(m, 2, 2, 2, torch.device(dev), sinks, 6)]
            if not m.cfg.sink_frames:
                caches.append(KVCacheSet(m, 2, 4, 2, dev, dt))
            outs.append([torch.cat([forward_cached(m, x[:, f:f + 2].to(dev, dt), t.to(dev), a[:, f:f + 2].to(dev), c, commit=True)
                                    .float().cpu() for f in (0, 2, 4)], 1) for c in caches])
        for got, want in zip(outs[1], outs[0]):
            # bf16 activations, and codes that fall to the other side of an e4m3 step for it
            assert (got - want).norm() / want.norm() < 20 * 2.0 ** -9 + 2.0 ** -5


def test_rollout_branches_on_the_kernels():
    from drivedit_b200.inference.rollout import StreamingRollout
    cfg, m = _world()
    m = m.cuda().eval()
    m.enable_fused()
    r = cfg.rollout
    r.chunk_frames, r.flow_steps, r.window_frames, r.kv_cache, r.sink_frames = 2, 2, 2, "fp8", 1
    ctx, act = torch.randn(2, 2, 16, 16, 16, device="cuda"), torch.rand(2, 3, 10, 2, device="cuda")
    act[:, :, :2] = act[:, :1, :2]
    roll = StreamingRollout(m, r)
    g = lambda: torch.Generator(device="cuda").manual_seed(4)  # noqa: E731
    res = roll.run_branches(ctx, act, total_frames=10, generator=g())
    one = roll.run(ctx.repeat_interleave(3, 0), act.flatten(0, 1), total_frames=10, generator=g())
    assert res.frames.shape == (6, 10, 16, 16, 16) and torch.isfinite(res.frames).all()
    # the same pages' contents and the same kernels: equal but for the context's batch shape
    assert (res.frames - one.frames).norm() / one.frames.norm() < 2.0 ** -6


def test_refusals():
    from drivedit_b200.ops.window_attention import window_attention
    q, k = _bits(1, 4, 2, 64), _bits(1, 6, 2, 64)
    for bad in (lambda: window_attention(q[..., :32], k[..., :32], k[..., :32]),
                lambda: window_attention(q, k[:, :, :1], k[:, :, :1]),
                lambda: window_attention(q, k, k[:, :5]),
                lambda: window_attention(q.float(), k.float(), k.float()),
                lambda: window_attention(q, k.float(), k.float()),
                lambda: window_attention(q, k.cpu(), k.cpu()),
                lambda: window_attention(q, k, k, "block"),
                lambda: window_attention(q, k, k, "none", window=2),
                lambda: window_attention(q, k, k, "frame", 0),
                lambda: window_attention(q, k, k, "frame", (1 << 24) + 1),
                lambda: window_attention(q, k, k, "token", window=-1),
                lambda: window_attention(q, k, k, "token", sinks=-1),
                lambda: window_attention(q, k, k, q_pos_offset=1 << 30),
                lambda: window_attention(q, k, k, scale=0.0),
                lambda: window_attention(q, k, k, scale=math.inf)):
        with pytest.raises(ValueError):
            bad()
    # a window and sinks past every position are all of them
    want = window_attention(q, k, k, "token", q_pos_offset=2)
    assert torch.equal(window_attention(q, k, k, "token", window=1 << 40, sinks=1 << 40, q_pos_offset=2), want)
    assert torch.equal(window_attention(q, k, k, "frame", 1 << 24), window_attention(q, k, k, "none"))
    torch.cuda.synchronize()


def test_no_second_derivative():
    from drivedit_b200.ops.window_attention import window_attention
    q = _bits(1, 8, 1, 64).requires_grad_(True)
    (g,) = torch.autograd.grad(window_attention(q, q, q, "token").sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)
