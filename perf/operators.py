"""The attention operators with a sliding window and the 8-bit paged key/value cache, as
measured cases: what each computes in plain torch, the framework's own call, and the
same from its definition in 64 bits.

Kinds of case:
  window   softmax attention whose queries see the newest ``window`` frames (or tokens)
           and the first ``sinks`` ones; forward, or forward and backward
  write    new keys and values into 64-token pages of e4m3 codes, one power-of-two scale
           for each (page, head), keys and values apart
  attend   attention of a sequence's newest tokens over such a cache, same masks
  pages    branching a sequence (pages shared, the unfinished page copied), or copying
           sequences, freeing the old ones and compacting the pool
"""
import math

import numpy as np
import torch

own = False

PAGE = 64   # tokens of a page, and of a scale
DIM = 64    # channels of a head


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # the tiny preset's training step: 4 frames of 64 tokens; latency counts
        dict(name="train_tiny", kind="window", B=2, T=256, S=256, H=4, unit=64, window=2, sinks=1, grad=True),
        # the dit_b preset's 16 frames of 512 tokens, trained with the mask it streams with
        dict(name="train_dit_b", kind="window", B=2, T=8192, S=8192, H=12, unit=512, window=4, sinks=1, grad=True),
        # token-causal training, odd length, a window that ends inside tiles
        dict(name="train_tokens_odd", kind="window", B=3, T=1003, S=1003, H=5, unit=1, window=257, sinks=4, grad=True),
        # forward only: two new frames against a long buffer of earlier keys
        dict(name="chunk_over_buffer", kind="window", B=2, T=1024, S=12288, H=12, unit=512, window=17, sinks=1, grad=False),
        # one generated token of each of 64 streams, pages at every fill
        dict(name="write_one_token", kind="write", B=64, T=1, H=12, len=700, ragged=True),
        # a rollout's 4-frame chunk of 512 tokens a frame, 4 streams
        dict(name="write_chunk", kind="write", B=4, T=2048, H=12, len=1024, ragged=False),
        # one token of one stream: the smallest call
        dict(name="one_token_one_stream", kind="attend", B=1, T=1, H=12, KH=12, len=1500, unit=1, window=0, sinks=0, ragged=False),
        # many long streams: the cache's bytes are the work
        dict(name="one_token_many_streams", kind="attend", B=64, T=1, H=16, KH=16, len=16384, unit=1, window=0, sinks=0, ragged=True),
        # a few tokens each, query heads in groups over fewer cached heads, window and sinks
        dict(name="few_tokens_grouped", kind="attend", B=16, T=5, H=16, KH=4, len=8191, unit=1, window=2048, sinks=4, ragged=True),
        # the rollout preset: a 4-frame chunk against its 32-frame window and 4 context frames
        dict(name="rollout_chunk", kind="attend", B=1, T=2048, H=12, KH=12, len=22528, unit=512, window=36, sinks=4, ragged=False),
        # eight futures of one stream: shared pages, the unfinished page copied in every layer
        dict(name="branch", kind="pages", L=12, H=12, B=1, len=4127, copies=8, compact=False),
        # streams copied, the old ones freed, the pool compacted
        dict(name="copy_and_compact", kind="pages", L=12, H=12, B=4, len=8150, copies=1, compact=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "write", "attend", "attend", "attend", "pages"])
    if kind == "window":
        unit = rng.choice([1, 1, 16, 49, 64, 256])
        grad = rng.random() < 0.7
        T = _log(rng, 1, 4096)
        S = T if grad or rng.random() < 0.3 else T + _log(rng, 1, 6000)
        B, H = rng.randint(1, 3), rng.randint(1, 8)
        return dict(kind=kind, B=B, T=T, S=S, H=H, unit=unit, window=max(1, _log(rng, 1, max(2, S // unit + 1))),
                    sinks=rng.choice([0, 1, 1, 3, 5]), grad=grad)
    if kind == "write":
        T = _log(rng, 1, 2048)
        return dict(kind=kind, B=rng.randint(1, 64 if T < 64 else 4), T=T, H=rng.randint(1, 16), len=_log(rng, 1, 1500),
                    ragged=rng.random() < 0.6)
    if kind == "attend":
        KH = rng.randint(1, 8)
        unit = rng.choice([1, 1, 1, 49, 64, 128])
        T = _log(rng, 1, 1500)
        n = T + _log(rng, 1, 12000)
        return dict(kind=kind, B=rng.randint(1, 24 if T < 33 else 3), T=T, H=KH * rng.choice([1, 1, 2, 4]), KH=KH, len=n, unit=unit,
                    window=rng.choice([0, max(1, _log(rng, 1, n // unit + 1))]), sinks=rng.choice([0, 1, 4]), ragged=rng.random() < 0.6)
    return dict(kind=kind, L=rng.randint(1, 12), H=rng.randint(1, 12), B=rng.randint(1, 4), len=_log(rng, 1, 8000),
                copies=rng.randint(1, 8), compact=rng.random() < 0.5)


# ---------------------------------------------------------------------------- inputs
def _lens(case, rs):
    """Tokens of each sequence before the call's own."""
    most = case["len"] - (case["T"] if case["kind"] == "attend" else 0)
    if not case.get("ragged"):
        return [most] * case["B"]
    return [int(n) for n in rs.randint(most // 2, most + 1, case["B"])]


def _tables(lens, more):
    """Each sequence's pages, the lowest free ones first: for half of each sequence's
    tokens in turn, then for the rest, then for ``more`` new ones."""
    free = iter(range(1 << 30))
    fill = lambda t, n: t + [next(free) for _ in range(-(-n // PAGE) - len(t))]  # noqa: E731
    tables = [fill([], n // 2) for n in lens]
    tables = [fill(t, n) for t, n in zip(tables, lens)]
    return [fill(t, n + more) for t, n in zip(tables, lens)]


def _codes(g, *shape):
    """e4m3 codes as a cache holds them: values of a normal distribution."""
    return (torch.randn(*shape, generator=g, device="cuda") * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(g, *shape):
    return 0.5 ** torch.randint(7, 10, shape, generator=g, device="cuda").float()


def _own_cache(state, lens, more):
    """The framework's cache with this state's pages, lengths and tables."""
    from drivedit_b200.ops.kv_cache import PagedKVCache

    L, P, H = state["k"].shape[:3]
    cache = PagedKVCache(L, H, P, device="cuda", max_pages_per_seq=state["table"].shape[1])
    seqs = cache.add(len(lens))
    cache.begin(seqs, [n // 2 for n in lens]).commit()
    cache.begin(seqs, [n - n // 2 for n in lens]).commit()
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(cache, name).copy_(state[name])
    return cache, seqs, cache.begin(seqs, more) if more else None


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 31))
    kind = case["kind"]
    state = dict(case=case)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").bfloat16()

    if kind == "window":
        B, T, S, H = (case[n] for n in "BTSH")
        # queries, keys and values as columns of one projection, as the blocks make them
        if T == S:
            packed = normal(B, T, 3, H, DIM)
            state["q"], state["k"], state["v"] = packed.unbind(2)
        else:
            state["q"] = normal(B, T, H, DIM)
            state["k"], state["v"] = normal(B, S, 2, H, DIM).unbind(2)
        if case["grad"]:
            state["do"] = normal(B, T, H, DIM)
            for n in "qkv":
                state[n] = state[n].detach().requires_grad_(own)
        return state
    lens = _lens(case, rs)
    B, H = case["B"], case.get("KH", case["H"])
    L = case.get("L", 1)
    more = case["T"] if kind in ("write", "attend") else 0
    tables = _tables(lens, more)
    # the pool's and the tables' sizes go by the case alone, not by the lengths drawn
    width = -(-(case["len"] + (more if kind == "write" else 0)) // PAGE) + 1
    pages = B * (width - 1) + 1
    if kind == "pages":
        pages += sum(map(len, tables)) if case["compact"] else case["copies"] * B
    state["k"], state["v"] = _codes(g, L, pages, H, PAGE, DIM), _codes(g, L, pages, H, DIM, PAGE)
    state["k_scale"], state["v_scale"] = _scales(g, L, pages, H), _scales(g, L, pages, H)
    state["lists"], state["lens"], state["pages"] = tables, lens, pages
    state["table"] = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32, device="cuda")
    state["len"] = torch.tensor(lens, device="cuda")
    if kind == "write":
        state["new_k"], state["new_v"] = normal(B, case["T"], 2, H, DIM).unbind(2)
        if case["T"] > 1:  # a token far above the others
            state["new_k"][:, case["T"] // 2] *= 9
    if kind == "attend":
        state["q"] = normal(B, case["T"], case["H"], DIM)
    if own:
        state["cache"], state["seqs"], state["step"] = _own_cache(state, lens, more)
    return state


# ---------------------------------------------------------------------------- plain forms
def _visible(case, q_pos, k_pos, upper):
    """Whether a query at ``q_pos`` sees a key at ``k_pos``: no later frame, and a frame of
    the window or one of the first ones; ``upper``: the sequence's length."""
    qf, kf = q_pos // case["unit"], k_pos // case["unit"]
    near = (kf > qf - case["window"]) | (kf < case["sinks"]) if case["window"] else torch.ones_like(kf <= qf)
    return (kf <= qf) & near & (k_pos < upper)


def _softmax(s, seen):
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    return p / p.sum(-1, keepdim=True).clamp_min(torch.finfo(p.dtype).tiny)


def _plain_window(state):
    case = state["case"]
    q, k, v = (state[n].detach().float().transpose(1, 2) for n in "qkv")
    T, S, scale = case["T"], case["S"], DIM ** -0.5
    seen = _visible(case, torch.arange(S - T, S, device="cuda")[:, None], torch.arange(S, device="cuda"), S)
    p = _softmax(q @ k.mT * scale, seen)
    o = p @ v
    out = lambda x: x.transpose(1, 2).bfloat16().contiguous()  # noqa: E731
    if not case["grad"]:
        return {"o": out(o)}
    do = state["do"].float().transpose(1, 2)
    ds = p * (do @ v.mT - (do * o).sum(-1, keepdim=True)) * scale
    return {"o": out(o), "dq": out(ds @ k), "dk": out(ds.mT @ q), "dv": out(p.mT @ do)}


def _two_to(e):
    """2^e of whole e in [-126, 127], exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _power(amax):
    """The smallest e with amax <= 448 * 2^e, kept in [-100, 119]."""
    mant, exp = torch.frexp(amax)
    e = torch.where(mant <= 0.875, exp - 9, exp - 8)
    return torch.where(amax > 0, e, -100).clamp(-100, 119)


def _plain_write(state):
    case = state["case"]
    B, T, H = case["B"], case["T"], case["H"]
    new, old = T, state["len"][:, None]
    # the pages that the new tokens touch, and each of their slots' place in the sequence
    n_pages = (new + PAGE - 2) // PAGE + 1
    at = old // PAGE + torch.arange(n_pages, device="cuda")                                     # [B, n]
    slot = (at[..., None] * PAGE + torch.arange(PAGE, device="cuda")).unsqueeze(-1).unsqueeze(-1)   # [B, n, 64, 1, 1]
    first = old[:, :, None, None, None]
    is_old, is_new = slot < first, (slot >= first) & (slot < first + new)
    there = (at * PAGE < old + new)
    page = torch.where(there, state["table"].gather(1, at.clamp(max=state["table"].shape[1] - 1)), state["pages"] - 1).long()
    seq = torch.arange(B, device="cuda")[:, None, None]
    tok = (slot[..., 0, 0] - old[..., None]).clamp(0, T - 1)

    def put(codes, scales, fresh, token_last):
        held = codes.view(torch.uint8)[0, page].view(codes.dtype).float()  # [B, n, H, 64, 64]
        held = (held.mT if token_last else held) * scales[0, page][..., None, None]
        x = torch.where(is_new, fresh[seq, tok].float(), torch.where(is_old, held.transpose(2, 3), 0.0)).transpose(2, 3)
        e = _power(torch.where(x.isfinite(), x, 0.0).abs().amax((-1, -2)))
        y = (x * _two_to(-e)[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        keep = there.nonzero(as_tuple=True)
        # 8-bit codes are stored by their bits
        codes[0].view(torch.uint8)[page[keep]] = (y.mT if token_last else y)[keep].contiguous().view(torch.uint8)
        scales[0, page[keep]] = _two_to(e[keep])

    put(state["k"], state["k_scale"], state["new_k"], False)
    put(state["v"], state["v_scale"], state["new_v"], True)
    return {n: state[n] for n in ("k", "v", "k_scale", "v_scale")}


def _plain_attend(state):
    case = state["case"]
    B, T, H, KH = (case[n] for n in ("B", "T", "H", "KH"))
    page = state["table"].clamp_min(0).long()
    k = state["k"][0].view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * state["k_scale"][0, page][..., None, None]
    v = state["v"][0].view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * state["v_scale"][0, page][..., None, None]
    k = k.transpose(1, 2).reshape(B, KH, 1, -1, DIM)
    v = v.mT.transpose(1, 2).reshape(B, KH, 1, -1, DIM)
    q = state["q"].float().view(B, T, KH, H // KH, DIM).permute(0, 2, 3, 1, 4)
    total = state["len"][:, None, None] + T
    seen = _visible(case, total - T + torch.arange(T, device="cuda")[:, None], torch.arange(k.shape[3], device="cuda"), total)
    p = _softmax(q @ k.mT * DIM ** -0.5, seen[:, None, None])
    return {"o": (p @ v).permute(0, 3, 1, 2, 4).reshape(B, T, H, DIM).bfloat16()}


def _move(state, src, dst):
    src, dst = (torch.tensor(x, device="cuda") for x in (src, dst))
    put = lambda t: t.index_copy_(1, dst, t.index_select(1, src))  # noqa: E731
    put(state["k"].view(torch.uint8)), put(state["v"].view(torch.uint8)), put(state["k_scale"]), put(state["v_scale"])


def _plain_pages(state):
    case, lists = state["case"], state["lists"]
    used = sum(map(len, lists))
    width = state["table"].shape[1]
    if case["compact"]:
        # the copies take the pages behind the old ones, then move to the pool's front
        flat = [p for t in lists for p in t]
        _move(state, flat, list(range(used, 2 * used)))
        _move(state, list(range(used, 2 * used)), list(range(used)))
        ends = np.cumsum([0] + [len(t) for t in lists]).tolist()
        state["lists"] = [list(range(a, b)) for a, b in zip(ends, ends[1:])]
        tables = state["lists"]
    else:
        # each branch gets its own copy of the unfinished page, then pages for its new token
        free = iter(range(used, state["pages"]))
        part = [n % PAGE != 0 for n in state["lens"] for _ in range(case["copies"])]
        kin = [t for t in lists for _ in range(case["copies"])]
        last = [next(free) for _ in part]
        tables = [t[:-1] + [x] if cut else t + [x] for t, x, cut in zip(kin, last, part)]
        moves = [(t[-1], x) for t, x, cut in zip(kin, last, part) if cut]
        if moves:
            _move(state, [a for a, _ in moves], [b for _, b in moves])
    table = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32).cuda()
    return {"table": table, **{n: state[n] for n in ("k", "v", "k_scale", "v_scale")}}


# ---------------------------------------------------------------------------- the framework's calls
def _own(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "window":
        from drivedit_b200.ops.window_attention import window_attention

        q, k, v = (state[n] for n in "qkv")
        o = window_attention(q, k, v, causal="frame" if case["unit"] > 1 else "token", tokens_per_frame=case["unit"],
                             window=case["window"], sinks=case["sinks"], q_pos_offset=case["S"] - case["T"])
        if not case["grad"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    cache = state["cache"]
    if kind == "write":
        state["step"].write(0, state["new_k"], state["new_v"])
    elif kind == "attend":
        return {"o": state["step"].attend(0, state["q"], causal="frame" if case["unit"] > 1 else "token",
                                          tokens_per_frame=case["unit"], window=case["window"], sinks=case["sinks"])}
    elif case["compact"]:
        old, state["seqs"] = state["seqs"], cache.copy(state["seqs"])
        cache.free(old)
        cache.compact()
    else:
        kids = cache.fork(state["seqs"], case["copies"])
        step = cache.begin(kids, 1)
        cache.free(kids)
        return {"table": step.table, **{n: getattr(cache, n) for n in ("k", "v", "k_scale", "v_scale")}}
    out = {n: getattr(cache, n) for n in ("k", "v", "k_scale", "v_scale")}
    return {"table": cache.table(state["seqs"]), **out} if kind == "pages" else out


def run(state):
    if own:
        return _own(state)
    return {"window": _plain_window, "write": _plain_write, "attend": _plain_attend, "pages": _plain_pages}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------- work
def _pairs(case, total, T):
    """Query-key pairs that the mask leaves, of one head, the queries being the newest T."""
    q = np.arange(total - T, total, dtype=np.int64) // case["unit"]
    hi = np.minimum((q + 1) * case["unit"], total)
    if not case["window"]:
        return int(hi.sum()), total
    lo = np.maximum(q - case["window"] + 1, 0) * case["unit"]
    first = np.minimum(np.minimum(case["sinks"] * case["unit"], lo), hi)
    return int((hi - lo + first).sum()), int(total - lo.min() + first.max())


def work(case):
    kind, B, H = case["kind"], case["B"], case["H"]
    if kind == "window":
        pairs, keys = _pairs(case, case["S"], case["T"])
        q, kv = 2 * B * case["T"] * H * DIM, 2 * B * keys * H * DIM
        grad = case["grad"]
        return {"bytes": (4 * q + 4 * kv) if grad else 2 * q + 2 * kv, "flops": (14 if grad else 4) * DIM * pairs * B * H}
    if kind == "pages":
        page = case["L"] * H * (2 * PAGE * DIM + 8)
        pages = -(-case["len"] // PAGE)
        if case["compact"]:
            return {"bytes": 4 * B * pages * page, "flops": 0}
        return {"bytes": (2 * B * case["copies"] * page if case["len"] % PAGE else 0) + 4 * B * case["copies"] * pages, "flops": 0}
    lens = _lens(case, np.random.RandomState(0))
    T = case["T"]
    if kind == "write":
        pages = sum(-(-(n + T) // PAGE) - n // PAGE for n in lens)
        held = sum(n % PAGE for n in lens)  # the unfinished pages' tokens are read
        return {"bytes": H * (2 * 2 * B * T * DIM + 2 * held * DIM + 2 * pages * PAGE * DIM + 8 * pages), "flops": 4 * B * T * H * DIM}
    KH = case["KH"]
    both = [_pairs(case, n + T, T) for n in lens]
    keys, pairs = sum(b for _, b in both), sum(a for a, _ in both)
    return {"bytes": KH * keys * 2 * DIM + 8 * KH * keys // PAGE + 4 * B * T * H * DIM, "flops": 4 * DIM * pairs * H}


# ---------------------------------------------------------------------------- in 64 bits
def _attention64(q, k, v, seen, scale, do=None):
    """One head's attention by its definition: q [T, D], k and v [S, D], seen [T, S]."""
    w = torch.zeros(seen.shape, dtype=torch.float64, device="cuda")
    s = (q @ k.T) * scale
    s[~seen] = -math.inf
    some = seen.any(1)
    w[some] = torch.softmax(s[some], 1)
    o = w @ v
    if do is None:
        return (o,)
    g = do @ v.T
    ds = w * (g - (w * g).sum(1, keepdim=True))
    return o, ds @ k * scale, ds.T @ q * scale, w.T @ do


def exact(case, seed):
    kind = case["kind"]
    if kind == "pages":
        return None
    state = prepare(case, seed)
    B = case["B"]
    if kind == "window":
        names = ("o", "dq", "dk", "dv") if case["grad"] else ("o",)
        T, S, u = case["T"], case["S"], case["unit"]
        at = {"o": T, "dq": T, "dk": S, "dv": S}
        out = {n: torch.zeros(B, at[n], case["H"], DIM, dtype=torch.float64, device="cuda") for n in names}
        tq, tk = (torch.arange(S - T, S, device="cuda") // u)[:, None], (torch.arange(S, device="cuda") // u)[None]
        seen = (tk <= tq) & ((tq - tk < case["window"]) | (tk < case["sinks"]))
        for b in range(B):
            for h in range(case["H"]):
                q, k, v = (state[n].detach()[b, :, h].double() for n in "qkv")
                got = _attention64(q, k, v, seen, DIM ** -0.5, state["do"][b, :, h].double() if case["grad"] else None)
                for n, x in zip(names, got):
                    out[n][b, :, h] = x
        return out
    if kind == "attend":
        T, H, KH, u = case["T"], case["H"], case["KH"], case["unit"]
        out = torch.zeros(B, T, H, DIM, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = state["lens"][b] + T
            pages = torch.tensor(state["lists"][b][:-(-n // PAGE)], device="cuda")
            tq, tk = (torch.arange(n - T, n, device="cuda") // u)[:, None], (torch.arange(n, device="cuda") // u)[None]
            seen = tk <= tq
            if case["window"]:
                seen = seen & ((tq - tk < case["window"]) | (tk < case["sinks"]))
            for h in range(H):
                c = h // (H // KH)
                k = state["k"][0][:, c].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * state["k_scale"][0, pages, c].double()[:, None, None]
                v = state["v"][0][:, c].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * state["v_scale"][0, pages, c].double()[:, None, None]
                out[b, :, h] = _attention64(state["q"][b, :, h].double(), k.reshape(-1, DIM)[:n], v.mT.reshape(-1, DIM)[:n], seen, DIM ** -0.5)[0]
        return {"o": out}
    # write: the codes' values and the scales, page by page
    codes = {n: state[n].double() for n in ("k", "v")}
    scales = {n: state[n + "_scale"].double() for n in ("k", "v")}
    for b in range(B):
        n, T = state["lens"][b], case["T"]
        for j in range(n // PAGE, -(-(n + T) // PAGE)):
            page, lo, hi = state["lists"][b][j], max(n, j * PAGE), min(n + T, (j + 1) * PAGE)
            for name in ("k", "v"):
                x = torch.zeros(case["H"], PAGE, DIM, dtype=torch.float64, device="cuda")
                was = codes[name][0, page] * scales[name][0, page][:, None, None]
                old = max(0, n - j * PAGE)
                x[:, :old] = (was if name == "k" else was.mT)[:, :old]
                x[:, lo - j * PAGE:hi - j * PAGE] = state["new_" + name][b, lo - n:hi - n].transpose(0, 1).double()
                amax = x.abs().amax((1, 2))
                e = torch.ceil(torch.log2(amax / 448)).clamp(-100, 119)
                y = x / torch.exp2(e)[:, None, None]
                # nearest value of 4 significant bits (steps of 2^-9 below 2^-6), ties to even
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
                y = torch.round(y / step) * step
                codes[name][0, page], scales[name][0, page] = (y if name == "k" else y.mT), torch.exp2(e)
    return {"k": codes["k"], "v": codes["v"], "k_scale": scales["k"], "v_scale": scales["v"]}
