"""8-bit paged key/value cache on the GPU: writing, attention and page moves against the
definition in 64 bits and the PyTorch form."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(L=1, H=2, P=64, **kw):
    from drivedit_b200.ops.kv_cache import PagedKVCache
    return PagedKVCache(L, H, P, device="cuda", **kw)


def _randn(*shape, scale=1.0):
    return (torch.randn(*shape, device="cuda") * scale).bfloat16()


def _fill(cache, lens, layer=0, scale=1.0):
    """Sequences of these lengths, written in two pieces."""
    seqs = cache.add(len(lens))
    for part in ([n // 3 for n in lens], [n - n // 3 for n in lens]):
        T = max(max(part), 1)
        step = cache.begin(seqs, part)
        step.write(layer, _randn(len(lens), T, cache.n_heads, 64, scale=scale), _randn(len(lens), T, cache.n_heads, 64, scale=scale))
        step.commit()
    return seqs


def _oracle(k, v, q, n, causal, unit, window, sinks, first=0, first_sinks=0, scale=0.125):
    """fp64 attention of ``q [n, H, 64]``, the newest of ``k``, ``v [S, KH, 64]``; also the mean
    magnitude of the values and the largest score magnitude, which the bounds use."""
    S, G = k.shape[0], q.shape[1] // k.shape[1]
    k, v, q = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1), q.double()
    s = torch.einsum("thd,shd->hts", q, k) * scale
    mag = (torch.einsum("thd,shd->hts", q.abs(), k.abs()) * scale).amax() if S and n else torch.zeros((), device="cuda")
    qf = (torch.arange(S - n, S, device="cuda") // unit)[:, None]
    pos = torch.arange(S, device="cuda")
    kf = (pos // unit)[None]
    seen = (kf <= qf) if causal != "none" else torch.ones(n, S, dtype=torch.bool, device="cuda")
    if window:
        seen = seen & ((qf - kf < window) | (pos < sinks * unit))
    if first:
        seen = seen & ((pos >= first) | (pos < first_sinks))
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - lse[..., None]), 0.0)
    return torch.einsum("hts,shd->thd", p, v), torch.einsum("hts,shd->thd", p, v.abs()), lse / math.log(2), float(mag)


def _check(o, lse, ref, mean, rlse, mag):
    # bf16 output: half a step, 2^-8 of the value. P in fp16: half a step, 2^-11 of each
    # weight, so 2^-11 of the mean magnitude; fp32 sums and exponentials: under 2^-12 of it.
    err = (o.double() - ref).abs()
    bound = 2.0 ** -8 * ref.abs() + (2.0 ** -11 + 2.0 ** -12) * mean + 1e-30
    assert torch.isfinite(o).all() and (err <= bound).all(), float((err / bound).max())
    if lse is not None:
        # fp32 products of 64 terms (64 * 2^-24 of the magnitudes), exponential and
        # logarithm of 2^-22, each times log2(e)
        fin = torch.isfinite(rlse)
        assert torch.equal(fin, torch.isfinite(lse))
        assert (lse.double() - rlse)[fin].abs().max().item() <= 1.45 * (mag * 2.0 ** -18 + 2.0 ** -19) if fin.any() else True


@pytest.mark.parametrize("lens,T,own", [
    ([0, 1, 63, 64, 65, 200], 1, None), ([0, 5, 130], 70, [70, 1, 0]), ([17], 128, None), ([64, 3], 64, [64, 61]),
])
@pytest.mark.parametrize("H", [1, 3])
def test_write_matches_definition(lens, T, own, H):
    """Codes and scales bit for bit as the PyTorch form has them, strided inputs, outliers,
    an infinity and zeros among the tokens; other pages stay as they were."""
    from drivedit_b200.ops.kv_cache import PagedKVCache
    gpu, cpu = _cache(2, H, 40), PagedKVCache(2, H, 40, device="cpu")
    own = own or [T] * len(lens)
    seqs = gpu.add(len(lens)), cpu.add(len(lens))
    for c in (gpu, cpu):  # what the pages held before
        for t in (c.k, c.v):
            t.view(torch.uint8).fill_(0x35)
    for n, layer, factor in ((lens, 1, 1.0), (own, 1, 30.0), (own, 1, 2.0 ** -20)):
        t = max(max(n), 1)
        kv = _randn(len(lens), t, 2, H + 1, 64, scale=factor)[:, :, :, :H]
        kv[0, t // 2, 0, 0, 5] = math.inf
        kv[-1, 0, 1] = 0
        kv[0, 0, 0, 0, 0] = 3e38
        steps = gpu.begin(seqs[0], n), cpu.begin(seqs[1], n)
        steps[0].write(layer, kv[:, :, 0], kv[:, :, 1])
        steps[1].write(layer, kv[:, :, 0].cpu(), kv[:, :, 1].cpu())
        if n is lens:
            for s in steps:
                s.commit()
        for name in ("k", "v", "k_scale", "v_scale"):
            a, b = getattr(gpu, name).cpu(), getattr(cpu, name)
            if a.dtype == torch.float8_e4m3fn:
                a, b = a.view(torch.uint8), b.view(torch.uint8)
            assert torch.equal(a, b), name


def test_write_keeps_nan_and_every_exponent():
    """A NaN stays one; a block's scale follows its magnitude over the exponents of bf16."""
    c = _cache(1, 1, 260)
    seqs = c.add(254)
    k = torch.zeros(254, 1, 1, 64, device="cuda", dtype=torch.bfloat16)
    k[:, 0, 0, 0] = torch.ldexp(torch.full((254,), 1.7578125, device="cuda"), torch.arange(-126, 128, device="cuda")).bfloat16()
    v = k.clone()
    v[:, 0, 0, 1] = math.nan
    step = c.begin(seqs, 1)
    step.write(0, k, v)
    page = step.table[:, 0].long()
    e = (torch.arange(-126, 128, device="cuda") - 7).clamp(-100, 119).float()
    assert torch.equal(c.k_scale[0, page, 0].log2(), e) and torch.equal(c.v_scale[0, page, 0].log2(), e)
    assert c.v[0, page, 0, 1, 0].float().isnan().all()
    held = c.k[0, page, 0, 0, 0].double() * c.k_scale[0, page, 0].double()
    ok = e > -100
    want = k[:, 0, 0, 0].double()
    assert ((held - want).abs() <= 2.0 ** -4 * want.abs())[ok].all()


CASES = [
    # lens before, own tokens, cached heads, group, causal, unit, window, sinks
    ([0], [1], 1, 1, "token", 1, 0, 0),
    ([63, 64, 0, 500], [1, 1, 1, 1], 3, 1, "token", 1, 0, 0),
    ([1000, 37, 640], [1, 1, 1], 2, 4, "token", 1, 100, 3),
    ([700, 129], [5, 2], 2, 4, "token", 1, 65, 64),
    ([300, 5], [40, 0], 2, 1, "token", 1, 0, 0),
    ([257], [200], 1, 2, "token", 1, 64, 70),
    ([490, 98], [98, 49], 2, 1, "frame", 49, 3, 1),
    ([256, 0], [256, 128], 2, 1, "frame", 128, 2, 1),
    ([1024], [512], 1, 1, "frame", 256, 0, 0),
    ([130, 70], [33, 7], 2, 2, "none", 1, 0, 0),
    ([2000], [1], 1, 8, "token", 1, 1, 0),
    ([3000], [3], 12, 1, "token", 1, 1500, 2000),
    ([4000, 10], [1, 1], 1, 16, "token", 1, 0, 0),
    ([100], [1], 2, 1, "frame", 1000, 5, 5),
    ([900, 77], [300, 128], 1, 3, "frame", 64, 4, 2),
    ([0, 3, 100], [257, 129, 65], 2, 1, "token", 1, 0, 0),
    ([5000], [130], 1, 2, "token", 1, 0, 0),
    ([6000, 40], [200, 3], 1, 1, "token", 1, 4500, 130),
    ([4100], [700], 2, 4, "frame", 100, 7, 1),
    ([8000], [65], 1, 1, "token", 1, 64, 1),
]


def test_blocks_of_zeros_and_far_scales():
    """Pages of zero keys, and pages whose scales lie far apart: zero keys still weigh."""
    for T in (1, 100):
        c = _cache(1, 1, 16)
        seqs = c.add(1)
        step = c.begin(seqs, 256)
        k, v = _randn(1, 256, 1, 64), _randn(1, 256, 1, 64)
        k[:, 64:128] = 0
        v[:, 128:192] *= 2.0 ** -40
        k[:, 192:] *= 2.0 ** 20
        k[:, 192:, :, 1:] = 0
        step.write(0, k, v)
        step.commit()
        step = c.begin(seqs, T)
        step.write(0, _randn(1, T, 1, 64), _randn(1, T, 1, 64))
        q = _randn(1, T, 1, 64)
        q[..., 0] = 0
        o, lse = step.attend(0, q, causal="token", return_lse=True)
        kk, vv = c._values(0, c._seqs[seqs[0]], 256 + T)
        ref, mean, rlse, mag = _oracle(kk, vv, q[0], T, "token", 1, 0, 0)
        _check(o[0], lse[0], ref, mean, rlse, mag)


@pytest.mark.parametrize("case", CASES)
def test_attend_matches_definition(case):
    lens, own, KH, G, causal, unit, window, sinks = case
    c = _cache(1, KH, sum(-(-(a + b) // 64) for a, b in zip(lens, own)) + 3)
    junk = c.add(1)
    c.begin(junk, 65)
    c.k.view(torch.uint8).fill_(0x7f)  # NaN wherever nothing is written
    c.v.view(torch.uint8).fill_(0x7f)
    seqs = _fill(c, lens)
    T = max(own) + 2
    k, v = (_randn(len(lens), T, KH, 64) for _ in "kv")
    q = _randn(len(lens), T, 2, KH * G, 64, scale=2.0)[:, :, 1]
    step = c.begin(seqs, own)
    step.write(0, k, v)
    o, lse = step.attend(0, q, causal=causal, tokens_per_frame=unit, window=window, sinks=sinks, return_lse=True)
    again = step.attend(0, q, causal=causal, tokens_per_frame=unit, window=window, sinks=sinks)
    assert torch.equal(o, again)
    step.commit()
    for i, (s, n) in enumerate(zip(seqs, own)):
        kk, vv = c.read(0, s)
        ref, mean, rlse, mag = _oracle(kk, vv, q[i, :n], n, causal, unit, window, sinks)
        _check(o[i, :n], lse[i, :, :n], ref, mean, rlse, mag)
        assert not o[i, n:].any() and (lse[i, :, n:] == -math.inf).all()


@pytest.mark.parametrize("lens,own,KH,G,window,sinks", [
    ([4200, 4100, 3900, 64, 0, 4000, 4150], [130, 100, 1, 130, 77, 0, 64], 7, 1, 0, 0),
    ([6000, 5000, 70, 6100, 5900, 0, 300], [120, 128, 128, 50, 3, 100, 0], 7, 2, 4000, 100),
    ([5000], [2048], 6, 1, 0, 0),  # several row blocks of a sequence
])
def test_row_blocks_that_meet_in_scratch(lens, own, KH, G, window, sinks):
    """Numbers of row blocks at which clusters would leave SMs idle: the CTAs' results are added
    up by a second launch, alone and replayed from a graph on another stream."""
    from drivedit_b200.ops._ext import ext
    c = _cache(1, KH, sum(-(-(a + b) // 64) for a, b in zip(lens, own)) + 3)
    seqs = _fill(c, lens)
    T = max(own)
    step = c.begin(seqs, own)
    step.write(0, *(_randn(len(lens), T, KH, 64) for _ in "kv"))
    q = _randn(len(lens), T, KH * G, 64, scale=2.0)
    call = lambda: step.attend(0, q, causal="token", window=window, sinks=sinks, return_lse=True)  # noqa: E731
    before = ext().launch_count()
    o, lse = call()
    assert ext().launch_count() - before == 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2, lse2 = call()
    for _ in range(2):
        o2.zero_(), lse2.zero_()
        graph.replay()
        call()
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
    step.commit()
    for i, (s, n) in enumerate(zip(seqs, own)):
        kk, vv = c.read(0, s)
        ref, mean, rlse, mag = _oracle(kk, vv, q[i, :n], n, "token", 1, window, sinks)
        _check(o[i, :n], lse[i, :, :n], ref, mean, rlse, mag)
        assert not o[i, n:].any() and (lse[i, :, n:] == -math.inf).all()


@pytest.mark.parametrize("T", [1, 20, 300])
def test_hidden_tokens_do_not_matter(T):
    """NaN, infinities' codes and huge values at tokens that no query sees, inside visible
    pages too; a window whose every key is another query's."""
    c = _cache(1, 2, 40)
    seqs = _fill(c, [1000])
    step = c.begin(seqs, T)
    step.write(0, _randn(1, T, 2, 64), _randn(1, T, 2, 64))
    q = _randn(1, T, 4, 64)
    args = dict(causal="token", window=100, sinks=10)
    want = step.attend(0, q, **args)
    ids = step.table[0].tolist()
    for pos in [*range(10, 1000 + 1 - 100), *range(1000 + T, -(-(1000 + T) // 64) * 64)]:
        page = ids[pos // 64]
        c.k.view(torch.uint8)[0, page, :, pos % 64] = 0x7f
        c.v.view(torch.uint8)[0, page, :, :, pos % 64] = 0x7f
    assert torch.equal(step.attend(0, q, **args), want)


@pytest.mark.parametrize("T", [1, 90])
def test_trimmed_sequence(T):
    """Dropped tokens are gone for every call, their pages are free, the sinks stay."""
    c = _cache(1, 2, 64)
    seqs = _fill(c, [1000, 1300])
    full = [c.read(0, s) for s in seqs]
    c.trim([seqs[0]], keep=300, sinks=70)
    free = c.free_pages
    c.trim([seqs[0]], keep=200, sinks=70)
    assert c.free_pages == free + 2  # the pages of tokens 704-767 and, partly kept before, none else
    step = c.begin(seqs, T)
    k, v, q = _randn(2, T, 2, 64), _randn(2, T, 2, 64), _randn(2, T, 2, 64)
    step.write(0, k, v)
    for window, sinks in ((0, 0), (150, 70), (900, 70)):
        o, lse = step.attend(0, q, causal="token", window=window, sinks=sinks, return_lse=True)
        for i in range(2):
            n = full[i][0].shape[0]
            kk, vv = c._values(0, c._seqs[seqs[i]], n + T)
            ref, mean, rlse, mag = _oracle(kk, vv, q[i], T, "token", 1, window, sinks, first=800 if i == 0 else 0, first_sinks=70)
            _check(o[i], lse[i], ref, mean, rlse, mag)
    with pytest.raises(ValueError):
        step.attend(0, q, causal="token", window=150, sinks=3)


@pytest.mark.parametrize("T", [4, 100])
@pytest.mark.parametrize("magnitude", [2.0 ** -60, 2.0 ** 40])
def test_attend_scales_exactly(magnitude, T):
    """Queries, keys and values of very small and very large magnitude: powers of two change
    nothing but the result's own."""
    lens, outs = [200], []
    for f in (1.0, magnitude):
        torch.manual_seed(3)
        c = _cache(1, 1, 8)
        seqs = _fill(c, lens, scale=f)
        step = c.begin(seqs, T)
        step.write(0, _randn(1, T, 1, 64, scale=f), _randn(1, T, 1, 64, scale=f))
        outs.append(step.attend(0, _randn(1, T, 2, 64, scale=1 / f), causal="token"))
    assert torch.equal(outs[0].float() * magnitude, outs[1].float())


def test_generation_run_matches_cpu_form():
    """A run as a user makes it, two layers: prompt, fork, tokens, trim, free, compact, copy."""
    from drivedit_b200.ops.kv_cache import PagedKVCache
    torch.manual_seed(1)
    caches = [_cache(2, 2, 30), PagedKVCache(2, 2, 30, device="cpu")]
    outs = []
    for c in caches:
        g = torch.Generator().manual_seed(5)
        r = lambda *s: torch.randn(*s, generator=g).bfloat16().to(c.device)  # noqa: E731
        got, seqs = [], c.add(2)

        def run(seqs, n):
            step = c.begin(seqs, n)
            T = max(n) if isinstance(n, list) else n
            for layer in range(2):
                step.write(layer, r(len(seqs), T, 2, 64), r(len(seqs), T, 2, 64))
                got.append(step.attend(layer, r(len(seqs), T, 4, 64), causal="token", window=120, sinks=5).cpu())
            step.commit()

        run(seqs, [150, 70])
        kids = c.fork(seqs, 3)
        run(kids, 1)
        run(seqs, 2)
        c.trim(kids, 120, 5)
        c.free([seqs[0], kids[1]])
        got.append(torch.tensor(c.compact()))
        rest = [seqs[1]] + kids[:1] + kids[2:]
        run(rest, 66)
        more = c.copy(rest[1:3])
        c.free(rest[1:3])
        run(more, 1)
        c.resize(c.compact())
        got.append(c.table(more).cpu())
        outs.append(got)
    for a, b in zip(*outs):
        if a.dtype == torch.bfloat16:
            # the same cache: P in fp16 and the order of fp32 sums, then a bf16 rounding each
            assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -10 * b.float().abs().max()).all()
        else:
            assert torch.equal(a, b)
    for name in ("k", "v", "k_scale", "v_scale"):
        a, b = getattr(caches[0], name).cpu(), getattr(caches[1], name)
        ids = sorted({p for s in caches[1]._seqs.values() for p in s.pages if p >= 0})
        assert torch.equal(a.float()[:, ids], b.float()[:, ids]), name


def test_capture_and_refilled_step():
    """A captured write and attend, replayed on the tables of later steps."""
    c = _cache(1, 2, 64)
    seqs = _fill(c, [100, 250])
    k, v, q = (_randn(2, 1, 2, 64) for _ in "kvq")
    step = c.begin(seqs, 1, max_tokens=600)
    step.write(0, k, v)
    step.attend(0, q, causal="token", window=90, sinks=2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.write(0, k, v)
        o = step.attend(0, q, causal="token", window=90, sinks=2)
        with pytest.raises(RuntimeError):
            c.begin(seqs, 1)
    for i in range(70):
        for t in (k, v, q):
            t.copy_(_randn(2, 1, 2, 64))
        c.begin(seqs, 1, out=step)
        graph.replay()
        want = step.attend(0, q, causal="token", window=90, sinks=2)
        assert torch.equal(o, want)
        if i % 23 == 0:
            for j, s in enumerate(seqs):
                kk, vv = c._values(0, c._seqs[s], c.length(s) + 1)
                _check(o[j], None, *_oracle(kk, vv, q[j], 1, "token", 1, 90, 2))
        step.commit()


def test_other_stream_waits_for_the_table():
    c = _cache(1, 2, 64)
    seqs = _fill(c, [900, 40])
    k, v, q = (_randn(2, 3, 2, 64) for _ in "kvq")
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    step = c.begin(seqs, 3)
    with torch.cuda.stream(other):
        step.write(0, k, v)
        o = step.attend(0, q, causal="token")
    torch.cuda.synchronize()
    assert torch.equal(o, step.attend(0, q, causal="token"))


def test_pool_past_32_bit_offsets():
    """Pages behind 4 GB of codes."""
    c = _cache(1, 32, 33500, max_pages_per_seq=33000)
    c.begin(c.add(1), 32900 * 64)
    seqs = _fill(c, [300])
    kid = c.copy(seqs)
    step = c.begin(kid, 2)
    step.write(0, _randn(1, 2, 32, 64), _randn(1, 2, 32, 64))
    q = _randn(1, 2, 32, 64)
    o, lse = step.attend(0, q, causal="token", return_lse=True)
    step.commit()
    assert min(c._seqs[kid[0]].pages) > 32768
    assert all(torch.equal(a[:300], b) for a, b in zip(c.read(0, kid[0]), c.read(0, seqs[0])))
    kk, vv = c.read(0, kid[0])
    ref, mean, rlse, mag = _oracle(kk, vv, q[0], 2, "token", 1, 0, 0)
    _check(o[0], lse[0], ref, mean, rlse, mag)


def test_refusals():
    c = _cache(2, 2, 8, max_pages_per_seq=4)
    a, b = c.add(2)
    step = c.begin([a, b], [3, 1])
    k = _randn(2, 3, 2, 64)
    for call in (lambda: step.write(2, k, k), lambda: step.write(-1, k, k), lambda: step.write(0, k[:1], k[:1]),
                 lambda: step.write(0, k[:, :2], k[:, :2]), lambda: step.write(0, k[:, :, :1], k[:, :, :1]),
                 lambda: step.write(0, k, k[:, :, :, :32]), lambda: step.write(0, k.float(), k.float()),
                 lambda: step.write(0, k.cpu(), k.cpu()), lambda: step.attend(0, _randn(2, 3, 3, 64)),
                 lambda: step.attend(5, k), lambda: step.attend(0, k.half()), lambda: step.attend(0, k, causal="x"),
                 lambda: step.attend(0, k, causal="none", window=3), lambda: step.attend(0, k, tokens_per_frame=0),
                 lambda: step.attend(0, k, window=-1), lambda: step.attend(0, k, scale=0.0), lambda: c.begin([a], 1, out=step),
                 lambda: c.begin([a, b], [9, 9], max_tokens=500, out=step), lambda: c.begin([a], 1000)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        c.begin([a, b], 256) and c.begin(c.add(1), 64)
    with pytest.raises(RuntimeError):  # stale by then
        step.write(0, k, k)
    for bad in ([0, 0], [0, 99], [1, 0]):  # a page twice, outside, read and written
        with pytest.raises(RuntimeError):
            from drivedit_b200.ops._ext import ext
            ext().kv_cache_copy_pages(c.k, c.v, c.k_scale, c.v_scale, torch.tensor([1, 2], dtype=torch.int32),
                                      torch.tensor(bad, dtype=torch.int32))
    torch.cuda.synchronize()


def test_empty_calls():
    c = _cache(1, 2, 8)
    step = c.begin([], 0)
    assert step.attend(0, _randn(0, 3, 4, 64)).shape == (0, 3, 4, 64)
    seqs = c.add(2)
    step = c.begin(seqs, 0)
    step.write(0, _randn(2, 0, 2, 64), _randn(2, 0, 2, 64))
    assert step.attend(0, _randn(2, 0, 2, 64)).shape == (2, 0, 2, 64)
    o, lse = step.attend(0, _randn(2, 5, 2, 64), return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    c.free([])
    assert c.fork([], 3) == [] and c.copy([]) == [] and c.compact() == 0


@pytest.mark.parametrize("T", [1, 40, 300])
def test_two_streams_at_once(T):
    """The same call on two streams at a time, many times: no shared workspace."""
    c = _cache(1, 2, 200)
    seqs = _fill(c, [5000, 3000])
    step = c.begin(seqs, T)
    step.write(0, _randn(2, T, 2, 64), _randn(2, T, 2, 64))
    qs = [_randn(2, T, 4, 64) for _ in range(2)]
    want = [step.attend(0, q, causal="token", window=4000, sinks=9) for q in qs]
    torch.cuda.synchronize()
    outs, streams = [[], []], [torch.cuda.Stream() for _ in qs]
    for _ in range(10):
        for q, s, o in zip(qs, streams, outs):
            with torch.cuda.stream(s):
                o.append(step.attend(0, q, causal="token", window=4000, sinks=9))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)


def test_status_clean():
    from drivedit_b200.ops._ext import device_status
    torch.cuda.synchronize()
    assert device_status() == 0
