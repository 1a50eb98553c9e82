"""Windowed attention and the 8-bit paged cache on the GPU, at the edges of their numerics and of
captured calls."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(*shape, scale=1.0):
    return (torch.randn(*shape, device="cuda") * scale).bfloat16()


# ------------------------------------------------------------------ windowed attention
@pytest.mark.parametrize("splits", [1, 2, 3, 8])
def test_rows_that_meet_nan_are_nan_however_the_keys_are_split(splits):
    """A NaN in a query, or in a key that it sees, makes the row and its lse NaN; the other
    rows are as without it."""
    from drivedit_b200.ops._ext import ext
    from drivedit_b200.ops.window_attention import window_attention
    q, k, v = _randn(1, 150, 2, 64), _randn(1, 2100, 2, 64), _randn(1, 2100, 2, 64)
    args = ("token", 1, 1500, 130, 1950)
    prev = ext().attn_fwd_set_kv_splits(splits)
    try:
        want, wl = window_attention(q, k, v, *args, return_lse=True)
        q2, k2 = q.clone(), k.clone()
        q2[0, 37, 1, 5] = math.nan
        k2[0, 2000, 0, 3] = math.nan     # seen by the queries from 2000 on
        k2[0, 470, 1, 9] = math.nan      # seen by the queries before 1970
        o, lse = window_attention(q2, k2, v, *args, return_lse=True)
    finally:
        ext().attn_fwd_set_kv_splits(prev)
    pos = torch.arange(1950, 2100, device="cuda")
    bad = torch.stack([pos >= 2000, (pos < 1970) | (pos == 1987)], 1)  # [T, H]
    assert bad.any(0).all() and not bad.all(0).any()
    assert o[0][bad].isnan().all() and lse[0].T[bad].isnan().all()
    assert torch.equal(o[0][~bad], want[0][~bad]) and torch.equal(lse[0].T[~bad], wl[0].T[~bad])


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("far", [2.0 ** 12, 2.0 ** 20, 2.0 ** 24])
def test_large_scores_give_finite_rows(far, splits):
    """Scores up to 2^28, past what fp32 tells apart: rows are means of values."""
    from drivedit_b200.ops._ext import ext
    from drivedit_b200.ops.window_attention import window_attention
    q, k, v = _randn(1, 150, 2, 64).clamp(-1, 1), _randn(1, 1100, 2, 64).clamp(-1, 1) * far, _randn(1, 1100, 2, 64)
    prev = ext().attn_fwd_set_kv_splits(splits)
    try:
        o, lse = window_attention(q, k, v, "token", 1, 700, 3, 950, return_lse=True)
    finally:
        ext().attn_fwd_set_kv_splits(prev)
    assert torch.isfinite(lse).all() and torch.isfinite(o).all()
    # weights and output in bf16 (half a step, 2^-8, each), fp32 sums under 2^-12
    assert (o.abs().amax((0, 1)) <= v.abs().amax((0, 1)).float() * (1 + 2.0 ** -8) ** 2 * (1 + 2.0 ** -12)).all()


def test_second_derivative_in_a_sum_is_refused():
    """A second derivative through the operator raises, also where other terms have one."""
    from drivedit_b200.ops.window_attention import window_attention
    q = _randn(1, 8, 1, 64).requires_grad_(True)
    loss = window_attention(q, q, q, "token").float().sum() + q.float().pow(3).sum()
    (g,) = torch.autograd.grad(loss, q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), q)


def test_sync_check_names_both_passes():
    from drivedit_b200.ops import debug
    from drivedit_b200.ops._ext import ext
    from drivedit_b200.ops.window_attention import window_attention
    q, k, v = (_randn(2, 70, 2, 64).requires_grad_(True) for _ in "qkv")
    do = _randn(2, 70, 2, 64)
    args = ("token", 1, 30, 2, 5, 5)
    want = window_attention(q, k, v, *args, return_lse=True)
    wg = torch.autograd.grad(want[0], (q, k, v), do)
    debug.set_sync_check(True)
    try:
        got = window_attention(q, k, v, *args, return_lse=True)
        gg = torch.autograd.grad(got[0], (q, k, v), do)
        with torch.no_grad():
            plain = window_attention(q, k, v, *args)
        names = [d.split()[1].split("(")[0] for d in ext().recent]
    finally:
        debug.set_sync_check(False)
    assert names.count("attn_window_bwd") == 1 and any(n in ("attn_window_fwd", "window_attention") for n in names), names
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(plain, want[0])
    assert torch.equal(gg[1], wg[1]) and torch.equal(gg[2], wg[2])
    assert (gg[0].float() - wg[0].float()).abs().max() <= 2.0 ** -7 * wg[0].float().abs().max()  # dq: no fixed order


# ------------------------------------------------------------------ paged cache
def _cache(L=1, H=2, P=64, **kw):
    from drivedit_b200.ops.kv_cache import PagedKVCache
    return PagedKVCache(L, H, P, device="cuda", **kw)


def _check_rows(c, seq, o, lse, q, window=0, sinks=0):
    """Each row against 64 bits, its bound from the keys that it sees alone.

    bf16 output: half a step, 2^-8 of the computed value, which is off itself. Weights in fp16:
    half a step, 2^-11 of each, or half the smallest number, 2^-25, where 2^7 stands for a
    weight as large as the largest (or for one whose product with its page's scale is); a
    weight that becomes zero is off by itself. fp32 scores of 64 products, exponentials and
    sums: 2^-12 in all at score magnitudes up to 2^6, in proportion above."""
    n, G, st = q.shape[0], q.shape[1] // c.n_heads, c._seqs[seq]
    S = st.length + n
    k, v = (x.double().repeat_interleave(G, 1) for x in c._values(0, st, S))
    vs = c.v_scale[0, torch.from_numpy(st.pages).long().cuda()].double().repeat_interleave(64, 0)[:S].repeat_interleave(G, 1)
    q = q.double()
    pos = torch.arange(S, device="cuda")
    qp = torch.arange(S - n, S, device="cuda")[:, None]
    seen = pos[None] <= qp
    if window:
        seen = seen & ((qp - pos < window) | (pos < sinks))
    s = (torch.einsum("thd,shd->hts", q, k) * 0.125).masked_fill(~seen, -math.inf)
    mag = (torch.einsum("thd,shd->hts", q.abs(), k.abs()) * 0.125).masked_fill(~seen, 0.0).amax(-1)   # [H, T]
    rl = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - rl[..., None]), 0.0)
    ref = torch.einsum("hts,shd->thd", p, v)
    mean = torch.einsum("hts,shd->thd", p, v.abs())
    # least step of a weight, in units of its own: by the largest weight, or by weight times scale
    step = torch.maximum(p.amax(-1, keepdim=True), (p * vs.T[:, None]).amax(-1, keepdim=True) / vs.T[:, None])
    lost = torch.einsum("hts,shd->thd", torch.minimum(p, 2.0 ** -32 * step), v.abs())
    rel = (2.0 ** -11 + 2.0 ** -12 * (mag.T * 2.0 ** -6).clamp(min=1.0))[..., None]
    off = rel * mean + lost
    bound = 2.0 ** -8 * (ref.abs() + off) + off + 1e-37
    err = (o.double() - ref).abs()
    assert torch.isfinite(o).all() and (err <= bound).all(), (float((err / bound).max()), (err / bound).amax((1, 2)).argmax().item())
    lerr = (lse.double() - rl / math.log(2)).abs()
    assert (lerr <= 1.45 * (mag * 2.0 ** -18 + 2.0 ** -19)).all(), float(lerr.max())


def _prompt(c, T, change):
    """A sequence of 100 tokens and ``T`` more, whose keys and values ``change`` has altered."""
    (s,) = c.add(1)
    k, v = _randn(1, 100 + T, c.n_heads, 64), _randn(1, 100 + T, c.n_heads, 64)
    change(k, v)
    step = c.begin([s], 100)
    step.write(0, k[:, :100], v[:, :100])
    step.commit()
    step = c.begin([s], T)
    step.write(0, k[:, 100:], v[:, 100:])
    return s, step


@pytest.mark.parametrize("T,G", [(3, 1), (28, 1), (7, 3)])
@pytest.mark.parametrize("far", [2.0 ** e for e in (12, 20, 24, 30, 60)])
def test_large_scores_few_rows(T, G, far):
    """Scores past what fp32 tells apart: the largest one takes the weight, nothing overflows."""
    c = _cache(1, 2, 32)

    def change(k, v):
        k[:, 64:] *= far
    s, step = _prompt(c, T, change)
    q = _randn(1, T, 2 * G, 64)
    for window in (0, 50):
        o, lse = step.attend(0, q, causal="token", window=window, return_lse=True)
        _check_rows(c, s, o[0], lse[0], q[0], window)


@pytest.mark.parametrize("what,far", [("k", 2.0 ** e) for e in (12, 17, 20, 23, 26, 60, -30)] + [("v", 2.0 ** e) for e in (12, 17, 26, 60, -30)])
@pytest.mark.parametrize("T,G", [(28, 1), (200, 1), (300, 2), (700, 1)])
def test_pages_that_a_row_does_not_see_do_not_touch_it(T, G, what, far):
    """Pages of far larger (or smaller) keys or values, behind the causal edge of the earlier
    rows and out of the window of the later ones: each row is as exact as its own keys allow."""
    c = _cache(1, 2, 32)

    def change(k, v):
        x = k if what == "k" else v
        for lo in (64, 192, 512):  # whole pages, of the first part and of the second
            x[:, lo:lo + 64] *= far
    s, step = _prompt(c, T, change)
    q = _randn(1, T, 2 * G, 64)
    for window, sinks in ((0, 0), (50, 3)):
        o, lse = step.attend(0, q, causal="token", window=window, sinks=sinks, return_lse=True)
        _check_rows(c, s, o[0], lse[0], q[0], window, sinks)


@pytest.mark.parametrize("T,G", [(3, 1), (28, 1), (200, 1), (300, 2), (2000, 1)])
@pytest.mark.parametrize("far,gap", [(2.0 ** 26, -40.0), (2.0 ** 40, -60.0), (0.0, 8.0), (2.0 ** -40, 9.0)])
def test_weights_and_page_scales_far_apart(T, G, far, gap):
    """A visible page whose values are far larger but hardly weigh, and one that takes most of
    the weight but holds zeros (or next to nothing): the other pages' part is as exact."""
    c = _cache(1, 2, 40)

    def change(k, v):
        k[..., 0] = 0
        k[:, :64, :, 0] = gap   # times 8 * 0.125: the scores' distance in nats
        v[:, :64] *= far
    s, step = _prompt(c, T, change)
    q = _randn(1, T, 2 * G, 64, scale=0.5)
    q[..., 0] = 8
    o, lse = step.attend(0, q, causal="token", return_lse=True)
    _check_rows(c, s, o[0], lse[0], q[0])


@pytest.mark.parametrize("T", [1, 5, 200])
@pytest.mark.parametrize("gap", [18.7, 12.0])
def test_a_long_tail_of_small_weights_counts(T, gap):
    """One key takes the weight, its value zero; what is left is 20,000 weights of 2^-27 (or
    2^-17) each."""
    c = _cache(1, 1, 330)
    (s,) = c.add(1)
    n = 20000
    k, v = _randn(1, n, 1, 64, scale=0.01), _randn(1, n, 1, 64) + 2
    k[..., 0] = 0
    k[:, 0, :, 0] = gap
    v[:, 0] = 0
    step = c.begin([s], n)
    step.write(0, k, v)
    step.commit()
    step = c.begin([s], T)
    step.write(0, k[:, 1:T + 1], v[:, 1:T + 1])
    q = _randn(1, T, 1, 64)
    q[..., 0] = 8
    o, lse = step.attend(0, q, causal="token", return_lse=True)
    _check_rows(c, s, o[0], lse[0], q[0])


def test_refill_beyond_the_captured_rows_is_refused():
    """A step whose calls were captured with T rows takes no refill for more, and the refused
    refill changes nothing."""
    c = _cache(1, 2, 16)
    seqs = c.add(2)
    k, v, q = (_randn(2, 3, 2, 64) for _ in "kvq")
    step = c.begin(seqs, 3, max_tokens=600)
    step.write(0, k, v)
    step.attend(0, q, causal="token")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.write(0, k, v)
        o = step.attend(0, q[:, :3], causal="token")
    step.commit()
    free, lengths = c.free_pages, [c.length(s) for s in seqs]
    for n in (4, [1, 200]):
        with pytest.raises(ValueError):
            c.begin(seqs, n, out=step)
    assert c.free_pages == free and [c.length(s) for s in seqs] == lengths
    c.begin(seqs, [3, 2], out=step)
    graph.replay()
    assert torch.equal(o, step.attend(0, q, causal="token"))


def test_refill_with_other_sinks_than_captured_is_refused():
    """A captured windowed call names its sinks; sequences trimmed to others are refused at the
    refill, as the call itself would refuse them."""
    c = _cache(1, 2, 32)
    seqs = c.add(1)
    k, v, q = (_randn(1, 300, 2, 64) for _ in "kvq")
    step = c.begin(seqs, 300)
    step.write(0, k, v)
    step.commit()
    step = c.begin(seqs, 1, max_tokens=600)
    step.attend(0, q[:, :1], causal="token", window=90, sinks=2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.attend(0, q[:, :1], causal="token", window=90, sinks=2)
    c.trim(seqs, keep=150, sinks=70)
    length, free = c.length(seqs[0]), c.free_pages
    with pytest.raises(ValueError):
        c.begin(seqs, 1, out=step)
    assert c.length(seqs[0]) == length and c.free_pages == free
    other = c.add(1)
    c.begin(other, 1, out=step)  # not trimmed: as captured
    graph.replay()
    torch.cuda.synchronize()


def test_step_begun_on_another_stream_than_it_is_captured_on():
    """The table is on the device before a captured call can be replayed."""
    c = _cache(1, 2, 64)
    seqs = c.add(2)
    k, v, q = (_randn(2, 200, 2, 64) for _ in "kvq")
    warm = c.begin(seqs, 200)
    warm.write(0, k, v)
    warm.attend(0, q, causal="token")
    side = torch.cuda.Stream()
    busy = torch.randn(8192, 8192, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy @ busy
        step = c.begin(seqs, 200)  # its upload waits behind the products
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(other):  # not torch.cuda.graph, which waits for the device first
        graph.capture_begin()
        step.write(0, k, v)
        o = step.attend(0, q, causal="token")
        graph.capture_end()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, step.attend(0, q, causal="token"))


def test_status_clean():
    from drivedit_b200.ops._ext import check_device_status
    torch.cuda.synchronize()
    check_device_status()
