"""Timed cases of the operators for drafted tokens over a paged cache.

Three operators, as one step of a server calls them:

* ``pages``: block tables, slots and positions from request lengths;
* ``rope``: rotary positions of the step's q and k rows, with k and v written
  to their pages;
* ``tree``: attention of each request's drafted nodes over its pages.

``run`` with ``own`` false is the plain form: elementary torch operations in
32 bits, rounded once at the end.  With ``own`` true it calls the package.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of the eight sessions that are stepped together
        {"name": "pages decode 8", "op": "pages", "req": 8, "ctx": 4096, "new": 1, "page": 16,
         "tree": False, "short": False},
        # prompts of many requests admitted at once: about a million tokens, ragged
        {"name": "pages admit 1500", "op": "pages", "req": 1500, "ctx": 2048, "new": 1400,
         "page": 32, "tree": False, "short": False},
        # one token of a 32/8 head layer: the smallest call
        {"name": "rope one token bf16", "op": "rope", "dtype": "bf16", "tokens": 1, "heads": 32,
         "kv": 8, "dim": 128, "rot": 128, "layout": "half", "scaling": "none", "theta": 1e6,
         "ctx": 32768, "page": 16, "fused": True},
        # odd row count, interleaved pairs over part of the head, stretched context
        {"name": "rope part f16", "op": "rope", "dtype": "f16", "tokens": 1003, "heads": 8,
         "kv": 4, "dim": 256, "rot": 64, "layout": "interleaved", "scaling": "yarn",
         "theta": 1e4, "ctx": 131072, "page": 16, "fused": False},
        # a 4096-token prompt of the 16/8 head model in the framework's own type
        {"name": "rope prompt f32", "op": "rope", "dtype": "f32", "tokens": 4096, "heads": 16,
         "kv": 8, "dim": 128, "rot": 128, "layout": "half", "scaling": "none", "theta": 1e6,
         "ctx": 8192, "page": 64, "fused": True},
        # prompts of several requests in one batch, banded frequencies
        {"name": "rope batch bf16", "op": "rope", "dtype": "bf16", "tokens": 32768, "heads": 32,
         "kv": 8, "dim": 128, "rot": 128, "layout": "half", "scaling": "banded", "theta": 5e5,
         "ctx": 131072, "page": 32, "fused": True},
        # one session, one token, in the framework's own type
        {"name": "tree one token f32", "op": "tree", "dtype": "f32", "req": 1, "nodes": 1,
         "ctx": 1037, "ragged": False, "heads": 16, "kv": 8, "dim": 128, "page": 16,
         "window": 0, "softcap": 0.0},
        # eight sessions with small trees, in the framework's own type
        {"name": "tree sessions f32", "op": "tree", "dtype": "f32", "req": 8, "nodes": 24,
         "ctx": 4500, "ragged": True, "heads": 16, "kv": 8, "dim": 128, "page": 16,
         "window": 0, "softcap": 0.0},
        # soft-capped, windowed layer with 256-wide heads and odd trees
        {"name": "tree window f16", "op": "tree", "dtype": "f16", "req": 5, "nodes": 13,
         "ctx": 7777, "ragged": True, "heads": 8, "kv": 4, "dim": 256, "page": 64,
         "window": 4096, "softcap": 50.0},
        # a server's ordinary verification step
        {"name": "tree batch bf16", "op": "tree", "dtype": "bf16", "req": 32, "nodes": 16,
         "ctx": 8192, "ragged": True, "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "window": 0, "softcap": 0.0},
        # many short requests, one token each, narrow heads
        {"name": "tree decode 256 f16", "op": "tree", "dtype": "f16", "req": 256, "nodes": 1,
         "ctx": 3001, "ragged": True, "heads": 16, "kv": 8, "dim": 64, "page": 32,
         "window": 0, "softcap": 0.0},
        # wide trees over very long contexts
        {"name": "tree long bf16", "op": "tree", "dtype": "bf16", "req": 2, "nodes": 64,
         "ctx": 131000, "ragged": True, "heads": 32, "kv": 8, "dim": 128, "page": 64,
         "window": 0, "softcap": 0.0},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    heads, kv, dim = rng.choice([(16, 8, 128), (32, 8, 128), (8, 4, 256), (8, 4, 64), (16, 8, 64),
                                 (16, 4, 32), (12, 4, 96), (24, 8, 80), (7, 7, 128)])
    dtype = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    op = rng.choice(["pages", "rope", "rope", "tree", "tree", "tree"])
    if op == "pages":
        req = log(1, 2000)
        return {"op": op, "req": req, "ctx": log(1, 30000), "new": log(1, max(1, 2000000 // req // 2)),
                "page": rng.choice([1, 5, 8, 16, 32, 64]), "tree": rng.random() < 0.5,
                "short": rng.random() < 0.25}
    if op == "rope":
        top = 32768 * 48 * 128 * 2 // ((heads + 2 * kv) * dim * (4 if dtype == "f32" else 2))
        return {"op": op, "dtype": dtype, "tokens": log(1, min(top, 40000)), "heads": heads,
                "kv": kv, "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4 * 3 // 2 * 2]),
                "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "banded", "yarn"]),
                "theta": rng.choice([1e4, 5e5, 1e6]), "ctx": log(16, 131072), "page": page,
                "fused": rng.random() < 0.5}
    req = log(1, 256)
    nodes = log(1, 64)
    room = 200_000_000 // (kv * dim * (2 if dtype == "f32" else 1)) // req
    ctx = log(1, max(2, min(131072, room)))
    return {"op": op, "dtype": dtype, "req": req, "nodes": nodes, "ctx": ctx,
            "ragged": rng.random() < 0.8, "heads": heads, "kv": kv, "dim": dim, "page": page,
            "window": rng.choice([0, 0, 0, 1 + ctx // 2]), "softcap": rng.choice([0.0, 0.0, 30.0])}


def lengths(case, seed):
    """The host's copy of the request lengths: what a scheduler decides from.
    A case has its lengths; the seed puts the requests in another order."""
    r = np.random.default_rng([case["req"], case["ctx"]])
    n = case["req"]
    if case["op"] == "pages":
        ctx = r.integers(0, case["ctx"] + 1, n)
        new = np.full(n, 1) if case["new"] == 1 else r.integers(0, case["new"] + 1, n)
        if n > 2:
            ctx[0] = 0
    elif case["ragged"] and n > 1:
        ctx = r.integers(case["ctx"] // 4, case["ctx"] + 1, n)
        new = r.integers(max(1, case["nodes"] // 2), case["nodes"] + 1, n)
        ctx[0], new[-1] = case["ctx"], case["nodes"]
    else:
        ctx, new = np.full(n, case["ctx"]), np.full(n, case["nodes"])
    order = np.random.default_rng(seed).permutation(n)
    return ctx[order].astype(np.int32), new[order].astype(np.int32)


def frequencies(case):
    """Turns per position of each rotated pair, and the amplitude, in 64 bits."""
    i = np.arange(case["rot"] // 2, dtype=np.float64)
    f = case["theta"] ** (-2.0 * i / case["rot"])
    amp = 1.0
    if case["scaling"] == "linear":
        f = f / 4.0
    elif case["scaling"] == "banded":  # factor 8, bands 1 and 4 turns, first trained at 8192
        blend = np.clip((8192.0 * f / (2 * np.pi) - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        f = f / 8.0 * (1.0 - blend) + f * blend
    elif case["scaling"] == "yarn":    # factor 4, ramp 32 to 1 turns, first trained at 32768
        def at(turns):
            return case["rot"] * np.log(32768.0 / (turns * 2 * np.pi)) / (2 * np.log(case["theta"]))
        lo = max(np.floor(at(32.0)), 0.0)
        hi = min(np.ceil(at(1.0)), case["rot"] - 1.0)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        f = f / 4.0 * ramp + f * (1.0 - ramp)
        amp = 0.1 * np.log(4.0) + 1.0
    return f / (2 * np.pi), float(amp)


SCALING = {"none": dict(), "linear": dict(kind="linear", factor=4.0),
           "banded": dict(kind="banded", factor=8.0, low=1.0, high=4.0, trained=8192),
           "yarn": dict(kind="yarn", factor=4.0, low=1.0, high=32.0, trained=32768)}


# ---------------------------------------------------------------- a state
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = np.random.default_rng(seed + 1)
    s = {"case": case}
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    if case["op"] == "pages":
        ctx, new = lengths(case, seed)
        P, n = case["page"], case["req"]
        have, want = -(-ctx // P), -(-(ctx + new) // P)
        s["max_pages"] = max(1, int(want.max()) + 3)
        need = int((want - have).sum())
        free = max(1, need * 2 // 3 if case["short"] else need + 17)
        ids = r.permutation(int(have.sum()) + free).astype(np.int32)
        table = np.full((n, s["max_pages"]), -1, np.int32)
        table[np.arange(s["max_pages"])[None, :] < have[:, None]] = ids[:int(have.sum())]
        total = int(new.sum())
        s["max_tokens"] = max(1, total + total // 16 + 3)
        s["lens"], s["news"], s["table"] = dev(ctx), dev(new), dev(table)
        s["free"] = dev(ids[int(have.sum()):])
        s["depths"] = None
        if case["tree"]:
            s["depths"] = torch.randint(0, 9, (s["max_tokens"],), generator=g, device=DEV,
                                        dtype=torch.int32)
        new_i32 = lambda k: torch.empty(k, dtype=torch.int32, device=DEV)  # noqa: E731
        s["out"] = {"table": s["table"], "starts": new_i32(n + 1), "used": new_i32(1),
                    "positions": new_i32(s["max_tokens"]), "slots": new_i32(s["max_tokens"]),
                    "owners": new_i32(s["max_tokens"])}
    elif case["op"] == "rope":
        dt, T, H, K, D, P = (case[k] for k in ("dtype", "tokens", "heads", "kv", "dim", "page"))
        dt = DTYPES[dt]
        rnd = lambda *sh: torch.randn(*sh, generator=g, device=DEV).to(dt)  # noqa: E731
        if case["fused"]:  # one projection's rows hold q, k and v
            rows = rnd(T, (H + 2 * K) * D)
            s["q"], s["k"], s["v"] = rows.split([H * D, K * D, K * D], dim=1)
        else:
            s["q"], s["k"], s["v"] = rnd(T, H * D), rnd(T, K * D), rnd(T, K * D)
        s["n_pages"] = -(-T // P) + 8
        slots = r.permutation(s["n_pages"] * P)[:T].astype(np.int32)
        if T > 40:  # padding rows of a captured step
            slots[r.integers(0, T, 3)] = -1
        s["slots"] = dev(slots)
        s["positions"] = dev(r.integers(0, case["ctx"], T).astype(np.int32))
        f, s["amp"] = frequencies(case)
        s["steps"] = dev(np.round(np.ldexp(f, 64)).astype(np.uint64).view(np.int64))
        s["k_cache"], s["v_cache"] = rnd(s["n_pages"], K, P, D), rnd(s["n_pages"], K, P, D)
        s["q_out"] = torch.empty(T, H * D, dtype=dt, device=DEV)
    else:
        dt, H, K, D, P, n = (case[k] for k in ("dtype", "heads", "kv", "dim", "page", "req"))
        dt = DTYPES[dt]
        ctx, new = lengths(case, seed)
        used = -(-(ctx + new) // P)
        s["max_pages"], s["n_pages"] = int(used.max()), int(used.sum()) + 5
        table = np.full((n, s["max_pages"]), -1, np.int32)
        table[np.arange(s["max_pages"])[None, :] < used[:, None]] = \
            r.permutation(s["n_pages"])[:int(used.sum())]
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        T, N = int(starts[-1]), int(new.max())
        # each node's parent is one of the nodes before it; it sees its ancestors and itself
        parent = (r.random((n, N)) * np.arange(N)[None, :]).astype(np.int64)
        see = np.zeros((n, N, N), bool)
        depth = np.zeros((n, N), np.int32)
        for i in range(N):
            if i:
                see[:, i] = see[np.arange(n), parent[:, i]]
                depth[:, i] = depth[np.arange(n), parent[:, i]] + 1
            see[:, i, i] = True
        words = -(-N // 32)
        bits = np.zeros((n, N, words * 32), np.uint8)
        bits[:, :, :N] = see
        mask = np.packbits(bits, axis=2, bitorder="little").view(np.uint32)
        live = np.arange(N)[None, :] < new[:, None]
        s["words"] = words
        s["mask"] = dev(mask[live].view(np.int32))
        s["positions"] = dev((ctx[:, None] + depth)[live].astype(np.int32))
        s["lens"], s["starts"], s["table"] = dev(ctx), dev(starts), dev(table)
        s["L"], s["N"], s["T"] = int((ctx + new).max()), N, T
        s["q"] = (2.0 * torch.randn(T, H * D, generator=g, device=DEV)).to(dt)
        s["k_cache"] = torch.randn(s["n_pages"], K, P, D, generator=g, device=DEV, dtype=dt)
        s["v_cache"] = torch.randn(s["n_pages"], K, P, D, generator=g, device=DEV, dtype=dt)
        s["o"] = torch.empty(T, H * D, dtype=dt, device=DEV)
    if own:
        s["call"] = _calls(s)
    return s


def _calls(s):
    """The prepared call that a user's program keeps for this step's buffers."""
    from chat_wgpu_b200 import GpuContext
    from chat_wgpu_b200.kernels import pages, rope, tree

    c = s["case"]
    ctx = s["ctx"] = GpuContext(0, stream=torch.cuda.current_stream().cuda_stream)
    w = lambda x: None if x is None else ctx.wrap(x)  # noqa: E731
    if c["op"] == "pages":
        o = s["out"]
        return pages.PagePlan(
            ctx, lens=w(s["lens"]), news=w(s["news"]), free_pages=w(s["free"]), table=w(s["table"]),
            depths=w(s["depths"]), starts=w(o["starts"]), positions=w(o["positions"]),
            slots=w(o["slots"]), owners=w(o["owners"]), used=w(o["used"]), n_req=c["req"],
            page_size=c["page"], max_pages=s["max_pages"], n_free=s["free"].numel(),
            max_tokens=s["max_tokens"])
    if c["op"] == "rope":
        plan = rope.rope_plan(ctx, c["rot"], c["theta"], **SCALING[c["scaling"]])
        return rope.RopeAppend(
            ctx, plan=plan, positions=w(s["positions"]), dtype=c["dtype"], layout=c["layout"],
            n_tokens=c["tokens"], n_heads=c["heads"], n_kv=c["kv"], head_dim=c["dim"],
            q=w(s["q"]), q_stride=s["q"].stride(0), q_out=w(s["q_out"]), k=w(s["k"]),
            k_stride=s["k"].stride(0), v=w(s["v"]), v_stride=s["v"].stride(0), slots=w(s["slots"]),
            k_cache=w(s["k_cache"]), v_cache=w(s["v_cache"]), page_size=c["page"],
            n_pages=s["n_pages"])
    return tree.TreeAttention(
        ctx, q=w(s["q"]), k_cache=w(s["k_cache"]), v_cache=w(s["v_cache"]), table=w(s["table"]),
        lens=w(s["lens"]), starts=w(s["starts"]), mask=w(s["mask"]), positions=w(s["positions"]),
        out=w(s["o"]), dtype=c["dtype"], n_req=c["req"], n_rows=s["T"], max_nodes=s["N"],
        n_heads=c["heads"], n_kv=c["kv"], head_dim=c["dim"], page_size=c["page"],
        n_pages=s["n_pages"], max_pages=s["max_pages"], window=c["window"], softcap=c["softcap"])


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        s["call"]()
        if c["op"] == "pages":
            return s["out"]
        if c["op"] == "rope":
            return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return {"out": s["o"]}
    return {"pages": _plain_pages, "rope": _plain_rope, "tree": _plain_tree}[c["op"]](s)


def _owners(starts, n, count):
    """Which range [starts[i], starts[i+1]) each of 0..count-1 lies in (n past the last)."""
    marks = torch.zeros(count + 1, dtype=torch.int32, device=DEV)
    at = starts[1:].clamp(max=count)
    marks.index_add_(0, at, torch.ones_like(at))
    return marks.cumsum(0)[:count]


def _plain_pages(s):
    P, n, M = s["case"]["page"], s["case"]["req"], s["max_pages"]
    lens, news, T, F = s["lens"], s["news"], s["max_tokens"], s["free"].numel()
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    have = ((lens + P - 1) // P).clamp(max=M)
    want = ((lens + news + P - 1) // P).clamp(max=M)
    ends = (want - have).cumsum(0).to(torch.int32)
    first = ends - (want - have)
    starts = torch.cat([zero, news.cumsum(0).to(torch.int32)])
    p = torch.arange(M, device=DEV, dtype=torch.int32)[None, :]
    take = first[:, None] + p - have[:, None]
    fresh = (p >= have[:, None]) & (p < want[:, None]) & (take < F)
    table = torch.where(fresh, s["free"][take.clamp(0, F - 1).long()], s["table"])
    t = torch.arange(T, device=DEV, dtype=torch.int32)
    who = _owners(starts, n, T)
    live = who < n
    who = who.clamp(max=n - 1)
    at = lens[who] + t - starts[who]
    pos = at if s["depths"] is None else lens[who] + s["depths"]
    page = at // P
    short = (page >= have[who]) & (first[who] + page - have[who] >= F)
    held = table[who, page.clamp(max=M - 1).long()]
    ok = live & (page < M) & (held >= 0) & ~short
    none = torch.full_like(t, -1)
    return {"table": table, "starts": starts, "used": ends[-1:].clone(),
            "positions": torch.where(live, pos, torch.zeros_like(t)),
            "slots": torch.where(ok, held * P + at % P, none),
            "owners": torch.where(live, who.to(torch.int32), none)}


def _plain_rope(s):
    c = s["case"]
    T, H, K, D, P, R = (c[k] for k in ("tokens", "heads", "kv", "dim", "page", "rot"))
    # turns modulo one as 64-bit whole numbers: no angle grows past half a turn
    turns = (s["positions"].long()[:, None] * s["steps"][None, :]).float() * 2.0 ** -64
    cos = (torch.cos(turns * (2 * math.pi)) * s["amp"])[:, None]
    sin = (torch.sin(turns * (2 * math.pi)) * s["amp"])[:, None]

    def turn(x, heads):
        x = x.reshape(T, heads, D).float()
        if c["layout"] == "half":
            a, b = x[..., :R // 2], x[..., R // 2:R]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., R:]], dim=-1)
        else:
            a, b = x[..., 0:R:2], x[..., 1:R:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
            y = torch.cat([y, x[..., R:]], dim=-1)
        return y.to(s["q"].dtype)

    live = s["slots"] >= 0
    to = s["slots"][live].long()
    s["k_cache"][to // P, :, to % P] = turn(s["k"], K)[live]
    s["v_cache"][to // P, :, to % P] = s["v"].reshape(T, K, D)[live]
    return {"q": turn(s["q"], H).reshape(T, H * D), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_tree(s):
    c = s["case"]
    n, H, K, D, P = (c[k] for k in ("req", "heads", "kv", "dim", "page"))
    L, N, T, G = s["L"], s["N"], s["T"], H // K
    first, lens = s["starts"][:-1].long(), s["lens"].long()
    news = s["starts"][1:].long() - first
    row = (first[:, None] + torch.arange(N, device=DEV)).clamp(max=T - 1)
    q = s["q"].reshape(T, K, G, D)[row].float()
    at = torch.arange(L, device=DEV)
    page = s["table"][:, at // P].long().clamp(min=0)
    off = (at % P).expand(n, L)
    k = s["k_cache"][page, :, off].float()
    v = s["v_cache"][page, :, off].float()
    x = torch.einsum("rnhgd,rlhd->rhgnl", q, k) * D ** -0.5
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    j = at[None, None, :] - lens[:, None, None]              # node index of a key, or below 0
    inside = j.clamp(0, N - 1).expand(n, N, L)
    bit = (s["mask"][row].gather(2, inside // 32) >> (inside % 32)) & 1
    see = (j < 0) | ((j < news[:, None, None]) & (bit == 1))
    if c["window"]:
        pos = s["positions"].long()[row]
        key = torch.where(j < 0, at[None, None, :].expand(n, N, L),
                          pos[:, None, :].expand(n, N, N).gather(2, inside))
        see = see & (pos[:, :, None] - key < c["window"])
    see = see[:, None, None]
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(x - top)
    o = torch.einsum("rhgnl,rlhd->rnhgd", e, v)
    o = o / e.sum(-1).clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
    t = torch.arange(T, device=DEV)
    who = _owners(s["starts"], n, T)
    return {"out": o[who, t - first[who]].reshape(T, H * D).to(s["q"].dtype)}


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["op"] == "pages":  # whole numbers only
        return None
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "rope":
        T, H, K, D, P, R = (case[k] for k in ("tokens", "heads", "kv", "dim", "page", "rot"))
        f, amp = frequencies(case)
        f = torch.from_numpy(f).to(DEV)
        z = torch.polar(torch.full((T, R // 2), amp, dtype=torch.float64, device=DEV),
                        2 * math.pi * torch.frac(s["positions"].double()[:, None] * f))

        def turned(x, heads):
            x = x.double().reshape(T, heads, D).clone()
            if case["layout"] == "half":
                w = torch.complex(x[:, :, :R // 2], x[:, :, R // 2:R]) * z[:, None]
                x[:, :, :R // 2], x[:, :, R // 2:R] = w.real, w.imag
            else:
                w = torch.complex(x[:, :, 0:R:2], x[:, :, 1:R:2]) * z[:, None]
                x[:, :, 0:R:2], x[:, :, 1:R:2] = w.real, w.imag
            return x

        kc = s["k_cache"].double().transpose(1, 2).reshape(-1, K, D)
        vc = s["v_cache"].double().transpose(1, 2).reshape(-1, K, D)
        live = torch.nonzero(s["slots"] >= 0)[:, 0]
        kc[s["slots"][live].long()] = turned(s["k"], K)[live]
        vc[s["slots"][live].long()] = s["v"].double().reshape(T, K, D)[live]
        back = lambda x: x.reshape(s["n_pages"], P, K, D).transpose(1, 2).contiguous()  # noqa: E731
        return {"q": turned(s["q"], H).reshape(T, H * D), "k_cache": back(kc), "v_cache": back(vc)}
    H, K, D, P = (case[k] for k in ("heads", "kv", "dim", "page"))
    out = torch.zeros(s["T"], H, D, dtype=torch.float64, device=DEV)
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for i in range(case["req"]):
        a, b, c0 = starts[i], starts[i + 1], lens[i]
        m, n_keys = b - a, lens[i] + b - a
        ids = s["table"][i, :-(-n_keys // P)].long()
        words = s["mask"][a:b].long() & 0xFFFFFFFF
        shifts = torch.arange(32, device=DEV)
        bits = ((words[:, :, None] >> shifts) & 1).reshape(m, -1)[:, :m].bool()
        see = torch.cat([torch.ones(m, c0, dtype=torch.bool, device=DEV), bits], dim=1)
        if case["window"]:
            mine = s["positions"][a:b].long()
            keys = torch.cat([torch.arange(c0, device=DEV), mine])
            see &= mine[:, None] < keys[None, :] + case["window"]
        for h in range(K):
            k = s["k_cache"][ids, h].reshape(-1, D)[:n_keys].double()
            v = s["v_cache"][ids, h].reshape(-1, D)[:n_keys].double()
            q = s["q"][a:b].reshape(m, K, H // K, D)[:, h].double()
            x = q.transpose(0, 1) @ k.T / math.sqrt(D)
            if case["softcap"]:
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            w = torch.softmax(x.masked_fill(~see, -math.inf), dim=-1)
            out[a:b].view(m, K, H // K, D)[:, h] = (w @ v).transpose(0, 1)
    return {"out": out.reshape(s["T"], H * D)}


# ---------------------------------------------------------------- the floor
def work(case):
    """What one pass cannot do without, for the mean lengths of the case."""
    if case["op"] == "pages":
        ctx, new = lengths(case, 0)
        P = case["page"]
        fresh = int((-(-(ctx + new) // P) + ctx // -P).sum())
        held = int(((ctx % P != 0) & (new > 0)).sum())
        return {"bytes": 4 * (3 * case["req"] + 2 * fresh + held + 1
                              + (4 if case["tree"] else 3) * int(new.sum())), "flops": 0}
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        rows = case["tokens"] * (case["heads"] + 2 * case["kv"]) * case["dim"]
        return {"bytes": 2 * rows * es + 8 * case["tokens"],
                "flops": 3 * case["tokens"] * (case["heads"] + case["kv"]) * case["rot"]}
    ctx, new = (x.astype(np.int64) for x in lengths(case, 0))
    seen = np.minimum(ctx, case["window"]) if case["window"] else ctx
    wide = case["kv"] * case["dim"]
    return {"bytes": int(2 * wide * es * (seen + new).sum()
                         + 2 * case["heads"] * case["dim"] * es * new.sum()),
            "flops": int(4 * case["heads"] * case["dim"] * (new * (seen + new)).sum())}
