"""Rotary positions, norms of queries and keys, and attention of branches that share their
past, as measured cases: what each computes in plain torch, the framework's own call,
and the same from its definition in 64 bits.

Kinds of case:
  rotary   channel pairs of each head rotated by the angles of their token's position:
           pairs side by side, as two halves, or read side by side and written as halves;
           all channels or the first ones; forward, or forward and backward
  qk       queries and keys divided by their head's root mean square, times a weight for
           each channel, and rotated; forward, or forward and backward
  branch   attention of the newest tokens of sequences that branched from a common past,
           over an 8-bit paged cache in which they share that past's pages
"""
import math

import numpy as np
import torch

own = False

PAGE = 64   # tokens of a page of the cache, and of a scale
DIM = 64    # channels of a cached head
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of each of 16 streams, at positions of their own: the smallest call
        dict(name="rotary_token", kind="rotary", dtype="bf16", layout="interleaved", B=16, T=1, H=12, D=64, R=64, places=4096, scattered=True, packed=False, grad=False),
        # a long context past the trained one: half of each head's channels, frequencies interpolated
        dict(name="rotary_long_half", kind="rotary", dtype="bf16", layout="half", B=1, T=32768, H=8, D=128, R=64, places=32768, scattered=False, packed=False, grad=True),
        # 32-bit training of an odd length; pairs that no wide load holds
        dict(name="rotary_odd", kind="rotary", dtype="fp32", layout="half", B=3, T=1003, H=5, D=72, R=40, places=1003, scattered=False, packed=False, grad=True),
        # packed sequences that each begin at position zero, written as halves as the reference lays them out
        dict(name="rotary_packed", kind="rotary", dtype="fp16", layout="split", B=1, T=20011, H=12, D=64, R=64, places=8192, scattered=True, packed=True, grad=False),
        # one new token of each of 64 streams, query heads in groups over fewer keys
        dict(name="qk_token", kind="qk", dtype="bf16", layout="half", B=64, T=1, H=16, KH=4, D=128, R=128, places=16384, scattered=True, grad=False),
        # the dit_b preset's training step: 2 samples of 16 frames of 512 tokens
        dict(name="qk_train_dit_b", kind="qk", dtype="bf16", layout="interleaved", B=2, T=8192, H=12, KH=12, D=64, R=64, places=8192, scattered=False, grad=True),
        # half-precision training, odd length, one key head for all queries, half the head rotated
        dict(name="qk_train_odd", kind="qk", dtype="fp16", layout="half", B=3, T=1003, H=5, KH=1, D=96, R=48, places=2048, scattered=True, grad=True),
        # eight futures of one stream, one token each, a short past
        dict(name="branch_token", kind="branch", B=1, n=8, T=1, H=12, KH=12, ctx=1500, more=40, unit=1, window=0, sinks=0),
        # 64 samples of one long context
        dict(name="branch_long", kind="branch", B=1, n=64, T=1, H=16, KH=16, ctx=16384, more=700, unit=1, window=0, sinks=0),
        # four contexts, eight futures of each, a few tokens at once, query heads in groups, window and sinks
        dict(name="branch_grouped", kind="branch", B=4, n=8, T=5, H=16, KH=4, ctx=8191, more=300, unit=1, window=4096, sinks=4),
        # many samples of one context, query heads in groups: many rows to a cached head
        dict(name="branch_many", kind="branch", B=1, n=48, T=1, H=16, KH=2, ctx=12007, more=200, unit=1, window=0, sinks=0),
        # eight futures of a small world model: a frame of 64 tokens each, 200 frames of context
        dict(name="branch_frames", kind="branch", B=1, n=8, T=64, H=12, KH=12, ctx=12800, more=256, unit=64, window=0, sinks=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "qk", "qk", "qk", "branch", "branch", "branch"])
    if kind == "branch":
        B, n, KH = rng.randint(1, 3), _log(rng, 2, 64), rng.randint(1, 12)
        unit = rng.choice([1, 1, 1, 1, 16, 49, 64])
        T, n = (unit, min(n, 8)) if unit > 1 else (_log(rng, 1, 12), n)
        H = KH * rng.choice([1, 1, 2, 4])
        ctx = min(_log(rng, 64, 14000), 70_000_000 // (B * n * T * H))
        return dict(kind=kind, B=B, n=n, T=T, H=H, KH=KH, ctx=ctx, more=_log(rng, 1, 400), unit=unit,
                    window=rng.choice([0, 0, max(1, _log(rng, 1, ctx // unit + 1))]), sinks=rng.choice([0, 1, 4]))
    D = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 256])
    if rng.random() < 0.15:
        D += rng.choice([2, 4, 8])
    D = min(D, 256)
    layout = rng.choice(["interleaved", "half", "split"])
    R = rng.choice([D, D, D, D // 4 * 2, max(2, D // 3 // 2 * 2)])
    B = rng.randint(1, 4)
    H = rng.randint(1, 16)
    T = _log(rng, 1, 12_000_000 // (B * H * D * 2))
    case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), layout=layout, B=B, T=T, H=H, D=D, R=R,
                places=T + _log(rng, 1, 20000), scattered=rng.random() < 0.5, grad=rng.random() < 0.6)
    if kind == "rotary":
        case["packed"] = B == 1 and rng.random() < 0.4
    else:
        case["KH"] = rng.choice([d for d in range(1, H + 1) if H % d == 0])
    return case


# ---------------------------------------------------------------------------- inputs
def _angles(case):
    """Angles of every position, in 64 bits: frequencies 10000^(-2i/R), the slow ones
    interpolated where the table goes past 8192 positions."""
    R, places = case["R"], case["places"]
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    if places > 8192:
        turns = 8192 * inv / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        inv = inv * (keep + (1 - keep) * 8192 / places)
    return torch.outer(torch.arange(places, dtype=torch.float64, device="cuda"), inv)


def _rotary_state(case, g, rs):
    B, T, H, D = (case[n] for n in "BTHD")
    dtype = TYPES[case["dtype"]]
    KH = case.get("KH", 0)
    ang = _angles(case)
    state = dict(case=case, table=torch.stack([ang.cos(), ang.sin()], -1).float())
    # queries, keys and values as columns of one projection
    rows = (torch.randn(B, T, H + 2 * KH, D, generator=g, device="cuda") * 1.5).to(dtype)
    if case.get("packed"):
        lens, left = [], T
        while left:
            lens.append(min(left, int(rs.randint(1, min(case["places"], T // 2 + 2) + 1))))
            left -= lens[-1]
        state["positions"] = torch.cat([torch.arange(n) for n in lens]).cuda()
    elif case["scattered"]:
        first = torch.randint(0, case["places"] - T + 1, (B, 1), generator=g, device="cuda")
        state["positions"] = first + torch.arange(T, device="cuda")
    else:
        state["positions"] = None
    names = ["x"] if not KH else ["q", "k"]
    parts = [rows] if not KH else [rows[:, :, :H], rows[:, :, H:H + KH]]
    for n, x in zip(names, parts):
        state[n] = x.detach().requires_grad_(own and case["grad"])
        if case["grad"]:
            state["d" + n] = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
    for n in names if KH else ():
        w = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
        state["w" + n] = w.requires_grad_(own and case["grad"])
    return state


def _codes(g, *shape):
    """e4m3 codes as a cache holds them: values of a normal distribution."""
    return (torch.randn(*shape, generator=g, device="cuda") * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(g, *shape):
    return 0.5 ** torch.randint(7, 10, shape, generator=g, device="cuda").float()


def _mores(case, rs):
    """Tokens that each branch has of its own before the call's."""
    return [int(m) for m in rs.randint(0, case["more"] + 1, case["B"] * case["n"])]


def _branch_state(case, g, rs):
    B, n, T, KH, ctx = (case[x] for x in ("B", "n", "T", "KH", "ctx"))
    mores = _mores(case, rs)
    shared = ctx // PAGE                                       # whole pages of the common past
    rest = -(-(ctx + case["more"] + T) // PAGE) - shared       # pages of a branch's own, from the unfinished one on
    state = dict(case=case, mores=mores)
    # the common past's pages, then every branch's own: keys by (token, channel), values by (channel, token)
    for part, shape in (("past", (B, shared)), ("own", (B * n, rest))):
        state["k_" + part], state["v_" + part] = _codes(g, *shape, KH, PAGE, DIM), _codes(g, *shape, KH, DIM, PAGE)
        state["ks_" + part], state["vs_" + part] = _scales(g, *shape, KH), _scales(g, *shape, KH)
    state["len"] = torch.tensor([ctx + m for m in mores], device="cuda")
    state["q"] = torch.randn(B * n, T, case["H"], DIM, generator=g, device="cuda").bfloat16()
    if own:
        from drivedit_b200.ops.kv_cache import PagedKVCache

        pages = B * (shared + 1) + B * n * rest
        cache = PagedKVCache(1, KH, pages, device="cuda", max_pages_per_seq=shared + rest)
        roots = cache.add(B)
        cache.begin(roots, ctx).commit()
        kids = cache.fork(roots, n)
        cache.free(roots)
        cache.begin(kids, mores).commit()
        step = cache.begin(kids, T, branches=n)
        table = step.table.long()
        for b in range(B):
            at = table[b * n, :shared]
            for name in ("k", "v"):
                getattr(cache, name)[0].view(torch.uint8)[at] = state[name + "_past"][b].view(torch.uint8)
                getattr(cache, name + "_scale")[0][at] = state[name + "s_past"][b]
        for i in range(B * n):
            used = -(-(ctx + mores[i] + T) // PAGE) - shared
            at = table[i, shared:shared + used]
            for name in ("k", "v"):
                getattr(cache, name)[0].view(torch.uint8)[at] = state[name + "_own"][i, :used].view(torch.uint8)
                getattr(cache, name + "_scale")[0][at] = state[name + "s_own"][i, :used]
        state["cache"], state["step"] = cache, step
    return state


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 31))
    return (_branch_state if case["kind"] == "branch" else _rotary_state)(case, g, rs)


# ---------------------------------------------------------------------------- plain forms
def _rotate(x, cs, layout, R):
    """``x [B, T, H, D]`` in 32 bits with its first ``R`` channels rotated; ``cs [.., T, 1, R/2, 2]``."""
    a, b = (x[..., :R // 2], x[..., R // 2:R]) if layout == "half" else (x[..., 0:R:2], x[..., 1:R:2])
    c, s = cs[..., 0], cs[..., 1]
    y, z = a * c - b * s, a * s + b * c
    y = torch.stack([y, z], -1).flatten(-2) if layout == "interleaved" else torch.cat([y, z], -1)
    return torch.cat([y, x[..., R:]], -1)


def _rotate_back(g, cs, layout, R):
    """The transposed rotation: gradients of the rotated channels to those of the channels."""
    a, b = (g[..., 0:R:2], g[..., 1:R:2]) if layout == "interleaved" else (g[..., :R // 2], g[..., R // 2:R])
    c, s = cs[..., 0], cs[..., 1]
    y, z = a * c + b * s, b * c - a * s
    y = torch.cat([y, z], -1) if layout == "half" else torch.stack([y, z], -1).flatten(-2)
    return torch.cat([y, g[..., R:]], -1)


def _rows_of(state):
    """(cos, sin) of each token, for all heads: ``[1 or B, T, 1, R/2, 2]``."""
    T = state["case"]["T"]
    p = state["positions"]
    cs = state["table"][:T] if p is None else state["table"][p]
    return (cs if cs.dim() == 4 else cs[None]).unsqueeze(-3)


def _plain_rotary(state):
    case = state["case"]
    cs = _rows_of(state)
    x = state["x"].detach()
    out = {"y": _rotate(x.float(), cs, case["layout"], case["R"]).to(x.dtype)}
    if case["grad"]:
        out["dx"] = _rotate_back(state["dx"].float(), cs, case["layout"], case["R"]).to(x.dtype)
    return out


def _plain_qk(state):
    case = state["case"]
    cs = _rows_of(state)
    out = {}
    for n in "qk":
        x, w = state[n].detach().float(), state["w" + n].detach()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        h = x * r
        out[n] = _rotate(h * w, cs, case["layout"], case["R"]).to(state[n].dtype)
        if case["grad"]:
            g = _rotate_back(state["d" + n].float(), cs, case["layout"], case["R"])
            # a long sum of terms of both signs
            out["dw" + n] = (g.double() * h.double()).sum((0, 1, 2)).float()
            g = g * w
            out["d" + n] = (r * (g - h * (g * h).mean(-1, keepdim=True))).to(state[n].dtype)
    return out


def _visible(case, q_pos, k_pos, upper):
    """Whether a query at ``q_pos`` sees a key at ``k_pos``: no later frame, and a frame of
    the window or one of the first ones; ``upper``: the sequence's length."""
    qf, kf = q_pos // case["unit"], k_pos // case["unit"]
    near = (kf > qf - case["window"]) | (kf < case["sinks"]) if case["window"] else torch.ones_like(kf <= qf)
    return (kf <= qf) & near & (k_pos < upper)


def _held(state, name, part):
    """What codes and scales stand for, ``[sequences, heads, tokens, 64]`` in 32 bits."""
    x = state[f"{name}_{part}"].float() * state[f"{name}s_{part}"][..., None, None]
    x = (x if name == "k" else x.mT).transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, DIM)


def _plain_branch(state):
    case = state["case"]
    B, n, T, H, KH = (case[x] for x in ("B", "n", "T", "H", "KH"))
    G, past = H // KH, case["ctx"] // PAGE * PAGE
    q = state["q"].float().view(B, n, T, KH, G, DIM).permute(0, 3, 1, 2, 4, 5).reshape(B, KH, n * T * G, DIM) * DIM ** -0.5
    kp, vp, ko, vo = (_held(state, name, part) for part in ("past", "own") for name in "kv")
    # all branches' rows against the common past at once, each branch's against its own keys
    s_past = q @ kp.mT
    per = lambda x: x.view(B, KH, n, T * G, -1).transpose(1, 2).reshape(B * n, KH, T * G, -1)  # noqa: E731
    s_own = per(q) @ ko.mT
    at = state["len"][:, None] + torch.arange(T, device="cuda")                                # [B n, T]
    at = at.repeat_interleave(G, 1)[:, None, :, None]                                         # [B n, 1, T G, 1]
    total = (state["len"] + T)[:, None, None, None]
    s = torch.cat([per(s_past), s_own], -1)
    keys = torch.arange(s.shape[-1], device="cuda")
    s = torch.where(_visible(case, at, keys, total), s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    back = p[..., :past].reshape(B, n, KH, T * G, past).transpose(1, 2).reshape(B, KH, n * T * G, past)
    o = per(back @ vp) + p[..., past:] @ vo                                                   # [B n, KH, T G, 64]
    return {"o": o.view(B * n, KH, T, G, DIM).permute(0, 2, 1, 3, 4).reshape(B * n, T, H, DIM).bfloat16()}


# ---------------------------------------------------------------------------- the framework's calls
def _own(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "branch":
        return {"o": state["step"].attend(0, state["q"], causal="frame" if case["unit"] > 1 else "token",
                                          tokens_per_frame=case["unit"], window=case["window"], sinks=case["sinks"])}
    from drivedit_b200.ops.rotary import qk_norm_rotary, rotary

    if kind == "rotary":
        y = rotary(state["x"], state["table"], state["positions"], layout=case["layout"])
        if not case["grad"]:
            return {"y": y}
        return {"y": y.detach(), "dx": torch.autograd.grad(y, state["x"], state["dx"])[0]}
    q, k = qk_norm_rotary(state["q"], state["k"], state["wq"], state["wk"], state["table"], state["positions"],
                          layout=case["layout"], eps=EPS)
    if not case["grad"]:
        return {"q": q, "k": k}
    names = ("q", "k", "wq", "wk")
    got = torch.autograd.grad((q, k), [state[n] for n in names], (state["dq"], state["dk"]))
    return {"q": q.detach(), "k": k.detach(), **{"d" + n: x for n, x in zip(names, got)}}


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "qk": _plain_qk, "branch": _plain_branch}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------- work
def work(case):
    B, T, H, kind = case["B"], case["T"], case["H"], case["kind"]
    if kind != "branch":
        size = torch.finfo(TYPES[case["dtype"]]).bits // 8
        D, R, KH = case["D"], case["R"], case.get("KH", 0)
        values = B * T * (H + KH) * D
        # the table's rows that some token is at: at most one a token, at most all
        rows = min(case["places"], B * T if case["scattered"] else T)
        table = rows * R * 4 + (8 * B * T if case["scattered"] or case.get("packed") else 0)
        one = 6 * values * R // D // 2 * 2 // 2 + (4 * values if KH else 0)
        if not case["grad"]:
            return {"bytes": 2 * size * values + table + 8 * D * bool(KH), "flops": one}
        # forward: read x, write y; backward: read dy (and x, for the norm), write dx
        return {"bytes": (5 if KH else 4) * size * values + table + 16 * D * bool(KH), "flops": 3 * one}
    n, KH = case["n"], case["KH"]
    pairs, shared, alone = 0, [0] * B, 0
    past = case["ctx"] // PAGE * PAGE
    u, w = case["unit"], case["window"]
    least = [past] * B
    for i, m in enumerate(_mores(case, np.random.RandomState(0))):
        total = case["ctx"] + m + T
        f = np.arange(total - T, total, dtype=np.int64) // u
        hi = np.minimum((f + 1) * u, total)
        lo = np.maximum(f - w + 1, 0) * u if w else np.zeros_like(f)
        first = np.minimum(np.minimum(case["sinks"] * u, lo), hi) if w else np.zeros_like(f)
        pairs += int((hi - lo + first).sum())
        alone += total - max(int(lo.min()), past)
        least[i // n] = min(least[i // n], int(lo.min()))
        shared[i // n] = max(shared[i // n], min(int(first.max()), past))
    keys = alone + sum(past - lo + min(s, lo) for lo, s in zip(least, shared))
    return {"bytes": KH * keys * 2 * DIM + 8 * KH * keys // PAGE + 4 * B * n * T * H * DIM, "flops": 4 * DIM * pairs * H}


# ---------------------------------------------------------------------------- in 64 bits
def _turned(x, case, cs):
    """Each pair as a complex number times e^(i angle), in the place where the layout keeps it."""
    R, n = case["R"], case["R"] // 2
    i = torch.arange(n, device="cuda")
    re_in, im_in = (i, i + n) if case["layout"] == "half" else (2 * i, 2 * i + 1)
    re_out, im_out = (2 * i, 2 * i + 1) if case["layout"] == "interleaved" else (i, i + n)
    z = torch.complex(x[..., re_in], x[..., im_in]) * torch.complex(cs[..., 0], cs[..., 1])
    y = x.clone()
    y[..., re_out], y[..., im_out] = z.real, z.imag
    return y


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] != "branch":
        B, T = case["B"], case["T"]
        p = state["positions"]
        p = torch.arange(T, device="cuda").expand(B, T) if p is None else p.reshape(-1, T).expand(B, T)
        cs = state["table"].double()[p][:, :, None]
        out = {}
        for n in ("x",) if case["kind"] == "rotary" else ("q", "k"):
            leaves = [state[n].detach().double().requires_grad_(case["grad"])]
            h = leaves[0]
            if n != "x":
                leaves.append(state["w" + n].detach().double().requires_grad_(case["grad"]))
                h = leaves[0] / torch.sqrt((leaves[0] ** 2).sum(-1, keepdim=True) / case["D"] + EPS) * leaves[1]
            y = _turned(h, case, cs)
            out["y" if n == "x" else n] = y.detach()
            if case["grad"]:
                got = torch.autograd.grad(y, leaves, state["d" + n].double())
                out.update(zip(("d" + n, "dw" + n), got))
        return out
    n, T, H, KH, u = (case[x] for x in ("n", "T", "H", "KH", "unit"))
    out = torch.zeros(case["B"] * n, T, H, DIM, dtype=torch.float64, device="cuda")
    for i, m in enumerate(state["mores"]):
        total = case["ctx"] + m + T
        tq = (torch.arange(total - T, total, device="cuda") // u)[:, None]
        tk = (torch.arange(total, device="cuda") // u)[None]
        seen = tk <= tq
        if case["window"]:
            seen = seen & ((tq - tk < case["window"]) | (tk < case["sinks"]))
        kv = []
        for name in "kv":
            codes = torch.cat([state[name + "_past"][i // n].double(), state[name + "_own"][i].double()])
            codes = codes * torch.cat([state[name + "s_past"][i // n], state[name + "s_own"][i]]).double()[..., None, None]
            codes = codes if name == "k" else codes.mT
            kv.append(codes.transpose(1, 2).reshape(-1, KH, DIM)[:total])
        for c in range(KH):
            k, v = (x[:, c] for x in kv)
            for h in range(c * (H // KH), (c + 1) * (H // KH)):
                s = state["q"][i, :, h].double() @ k.T / 8
                s[~seen] = -math.inf
                out[i, :, h] = torch.softmax(s, 1) @ v
    return {"o": out}
