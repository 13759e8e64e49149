"""Timed cases of the operators that take prompts in and choose from their logits.

Three operators, as one step of a server calls them:

* ``heads``: norms of each q and k head and their rotary positions in one pass, with k and v
  written to a paged cache;
* ``prompt``: causal attention of packed prompts, or of later pieces of prompts;
* ``logits``: penalties, biases and grammar masks on rows of logits, and their argmax.

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
        # one decode token of the 16/8 head model in the framework's own type: the smallest call
        {"name": "heads one token f32", "op": "heads", "dtype": "f32", "tokens": 1, "heads": 16,
         "kv": 8, "dim": 128, "rot": 128, "layout": "half", "theta": 1e6, "ctx": 32768,
         "page": 16, "fused": True, "shift": False, "rows": False},
        # odd row count, interleaved pairs over a quarter of wide heads, weights as 1 + w
        {"name": "heads part f16", "op": "heads", "dtype": "f16", "tokens": 1003, "heads": 8,
         "kv": 4, "dim": 256, "rot": 64, "layout": "interleaved", "theta": 1e4, "ctx": 131072,
         "page": 16, "fused": False, "shift": True, "rows": True},
        # prompts of several requests admitted in one batch of a 32/8 head layer
        {"name": "heads batch bf16", "op": "heads", "dtype": "bf16", "tokens": 32768, "heads": 32,
         "kv": 8, "dim": 128, "rot": 128, "layout": "half", "theta": 1e6, "ctx": 131072,
         "page": 32, "fused": True, "shift": False, "rows": True},
        # a chat line of one session in the framework's own type
        {"name": "prompt line f32", "op": "prompt", "dtype": "f32", "req": 1, "rows": 17,
         "past": 0, "ragged": False, "heads": 16, "kv": 8, "dim": 128, "window": 0,
         "softcap": 0.0, "fused": True},
        # the framework's own prefill: a 4096-token prompt of the 16/8 head model
        {"name": "prompt 4096 f32", "op": "prompt", "dtype": "f32", "req": 1, "rows": 4096,
         "past": 0, "ragged": False, "heads": 16, "kv": 8, "dim": 128, "window": 0,
         "softcap": 0.0, "fused": True},
        # soft-capped, windowed layer with 256-wide heads, odd lengths
        {"name": "prompt window f16", "op": "prompt", "dtype": "f16", "req": 3, "rows": 7001,
         "past": 0, "ragged": True, "heads": 8, "kv": 4, "dim": 256, "window": 4096,
         "softcap": 50.0, "fused": False},
        # prompts of a server's batch, all lengths up to 2048
        {"name": "prompt batch bf16", "op": "prompt", "dtype": "bf16", "req": 32, "rows": 2048,
         "past": 0, "ragged": True, "heads": 32, "kv": 8, "dim": 128, "window": 0,
         "softcap": 0.0, "fused": True},
        # the next pieces of four prompts after thousands of tokens
        {"name": "prompt piece bf16", "op": "prompt", "dtype": "bf16", "req": 4, "rows": 509,
         "past": 8192, "ragged": True, "heads": 32, "kv": 8, "dim": 128, "window": 0,
         "softcap": 0.0, "fused": False},
        # one long document
        {"name": "prompt long bf16", "op": "prompt", "dtype": "bf16", "req": 1, "rows": 16384,
         "past": 0, "ragged": False, "heads": 32, "kv": 8, "dim": 128, "window": 0,
         "softcap": 0.0, "fused": True},
        # one session's next token, with the text so far as history
        {"name": "logits one row f32", "op": "logits", "dtype": "f32", "rows": 1, "vocab": 151936,
         "history": 300, "bias": 5, "masks": 0},
        # eight sessions under a grammar, long histories, the larger vocabulary
        {"name": "logits grammar f32", "op": "logits", "dtype": "f32", "rows": 8, "vocab": 256000,
         "history": 8000, "bias": 0, "masks": 3},
        # a server's batch: every row has its own history, biases and one of a few grammars
        {"name": "logits batch bf16", "op": "logits", "dtype": "bf16", "rows": 256,
         "vocab": 151936, "history": 2000, "bias": 40, "masks": 7},
    ]


def draw(rng):
    def log(lo, hi):
        hi = max(lo, hi)
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    dtype = rng.choice(["f32", "f16", "bf16"])
    es = 4 if dtype == "f32" else 2
    heads, kv, dim = rng.choice([(16, 8, 128), (32, 8, 128), (8, 4, 256), (8, 4, 64), (16, 8, 64),
                                 (16, 4, 32), (12, 4, 96), (24, 8, 80), (7, 7, 128), (14, 2, 64)])
    op = rng.choice(["heads", "prompt", "prompt", "prompt", "logits"])
    if op == "heads":
        top = 32768 * 48 * 128 * 2 // ((heads + 2 * kv) * dim * es)
        return {"op": op, "dtype": dtype, "tokens": log(1, min(top, 40000)), "heads": heads,
                "kv": kv, "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4 * 3 // 2 * 2]),
                "layout": rng.choice(["half", "interleaved"]),
                "theta": rng.choice([1e4, 5e5, 1e6]), "ctx": log(16, 131072),
                "page": rng.choice([8, 16, 16, 32, 64, 128]), "fused": rng.random() < 0.5,
                "shift": rng.random() < 0.3, "rows": rng.random() < 0.5}
    if op == "logits":
        vocab = rng.choice([32000, 32003, 49152, 128256, 151936, 151936, 256000])
        rows = log(1, 256 * 151936 * 2 // (vocab * es))
        return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab,
                "history": log(1, min(8000, 600000 // rows)), "bias": rng.choice([0, 1, 40, 300]),
                "masks": rng.choice([0, 0, 1, 5])}
    # pairs of rows and keys that the largest listed case of the type affords
    room = (4096 ** 2 // 2 * 16 if dtype == "f32" else 16384 ** 2 // 2 * 32) * 128 // (heads * dim)
    req = log(1, 64)
    past = log(1, 16384) if rng.random() < 0.3 else 0
    most = room // req
    rows = log(1, min(16384, 40000 // req, int(math.sqrt(past * past + 2 * most)) - past))
    keys = past + rows
    return {"op": op, "dtype": dtype, "req": req, "rows": rows, "past": past,
            "ragged": rng.random() < 0.8, "heads": heads, "kv": kv, "dim": dim,
            "window": rng.choice([0, 0, 0, 1 + keys // 2]), "softcap": rng.choice([0.0, 0.0, 30.0]),
            "fused": past == 0 and rng.random() < 0.5}


def lengths(case, seed):
    """The host's copy of the requests' rows and keys: what a scheduler knows.
    A case has its lengths; the seed puts the requests in another order."""
    r = np.random.default_rng([case["req"], case["rows"], case["past"]])
    n = case["req"]
    rows, past = np.full(n, case["rows"]), np.full(n, case["past"])
    if case["ragged"] and n > 1:
        rows = r.integers(max(1, case["rows"] // 16), case["rows"] + 1, n)
        past = r.integers(case["past"] // 2, case["past"] + 1, n)
        rows[0], past[-1] = case["rows"], case["past"]
    order = np.random.default_rng(seed).permutation(n)
    return rows[order].astype(np.int64), (rows + past)[order].astype(np.int64)


def ragged(r, rows, most):
    """Sizes of rows' lists, up to `most` entries each, and where each list starts."""
    n = r.integers(most // 4, most + 1, rows) if rows > 1 else np.full(rows, most)
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


# ---------------------------------------------------------------- a state
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = np.random.default_rng(seed + 1)
    s = {"case": case}
    dt = DTYPES[case["dtype"]]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    rnd = lambda *sh: torch.randn(*sh, generator=g, device=DEV)  # noqa: E731
    if case["op"] == "heads":
        T, H, K, D, P = (case[k] for k in ("tokens", "heads", "kv", "dim", "page"))
        if case["fused"]:  # one projection's rows hold q, k and v
            rows = (3.0 * rnd(T, (H + 2 * K) * D)).to(dt)
            s["q"], s["k"], s["v"] = rows.split([H * D, K * D, K * D], dim=1)
        else:
            s["q"], s["k"] = (3.0 * rnd(T, H * D)).to(dt), (3.0 * rnd(T, K * D)).to(dt)
            s["v"] = rnd(T, K * D).to(dt)
        # trained norm weights lie around one, or around zero where one is added to them
        base = 0.0 if case["shift"] else 1.0
        s["q_norm"], s["k_norm"] = base + 0.2 * rnd(D), base + 0.2 * rnd(D)
        s["n_pages"] = -(-T // P) + 8
        slots = r.permutation(s["n_pages"] * P)[:T].astype(np.int32)
        if T > 40:  # padding rows of a captured step
            slots[r.integers(0, T, 3)] = -1
        s["slots"] = dev(slots)
        s["positions"] = dev(r.integers(0, case["ctx"], T).astype(np.int32))
        s["steps"] = dev(np.round(np.ldexp(turns_per_position(case), 64)).astype(np.uint64)
                         .view(np.int64))
        s["k_cache"], s["v_cache"] = rnd(s["n_pages"], K, P, D).to(dt), rnd(s["n_pages"], K, P, D).to(dt)
        s["q_out"] = torch.empty(T, H * D, dtype=dt, device=DEV)
        # rows for an attention over the prompt itself, besides the cache
        s["k_out"] = torch.empty(T, K * D, dtype=dt, device=DEV) if case["rows"] else None
    elif case["op"] == "prompt":
        H, K, D = (case[k] for k in ("heads", "kv", "dim"))
        rows, keys = s["lengths"] = lengths(case, seed)
        T, L = int(rows.sum()), int(keys.sum())
        if case["fused"]:  # v stays in the projection's rows
            s["q"], s["k"] = (1.5 * rnd(T, H * D)).to(dt), (1.5 * rnd(T, K * D)).to(dt)
            s["v"] = rnd(T, (H + 2 * K) * D).to(dt)[:, (H + K) * D:]
        else:
            s["q"], s["k"] = (1.5 * rnd(T, H * D)).to(dt), (1.5 * rnd(L, K * D)).to(dt)
            s["v"] = rnd(L, K * D).to(dt)
        s["starts"] = dev(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
        s["key_starts"] = None
        if case["past"]:
            s["key_starts"] = dev(np.concatenate([[0], np.cumsum(keys)]).astype(np.int32))
        s["o"] = torch.empty(T, H * D, dtype=dt, device=DEV)
    else:
        n, V = case["rows"], case["vocab"]
        s["logits"] = (4.0 * rnd(n, V)).to(dt)
        s["starts_host"] = ragged(r, n, case["history"])
        m = int(s["starts_host"][-1])
        # words of a text: few are frequent, most are rare
        words = np.minimum(V * r.random(max(m, 1)) ** 4, V - 1).astype(np.int32)
        s["starts"], s["tokens"] = dev(s["starts_host"]), dev(words)
        size = np.diff(s["starts_host"])
        s["prompts"] = dev((size * r.random(n)).astype(np.int32))
        p = np.stack([r.choice([1.0, 1.05, 1.1, 1.3], n), r.choice([0.0, 0.1, 0.5], n),
                      r.choice([0.0, 0.2, 0.6], n)], axis=1)
        if n == 1:
            p[:] = [1.1, 0.1, 0.2]
        s["penalties"] = dev(p.astype(np.float32))
        s["bias_starts"] = None
        if case["bias"]:
            s["bias_host"] = ragged(r, n, case["bias"])
            b = int(s["bias_host"][-1])
            s["bias_starts"] = dev(s["bias_host"])
            s["bias_tokens"] = dev(r.integers(0, V, max(b, 1)).astype(np.int32))
            s["bias_values"] = dev(r.choice([-100.0, -2.0, 1.5, 5.0], max(b, 1)).astype(np.float32))
        s["masks"] = None
        if case["masks"]:  # a grammar allows a handful of tokens, or nearly all
            words = -(-V // 32)
            share = r.choice([16, 3, 0.5], (case["masks"], 1))
            on = r.random((case["masks"], words, 32), np.float32) < np.exp2(-share)[:, :, None]
            bits = np.packbits(on.reshape(case["masks"], -1), axis=1, bitorder="little")
            s["masks"] = dev(bits.view(np.uint32).view(np.int32))
            s["mask_rows"] = dev(r.integers(-1, case["masks"], n).astype(np.int32))
        s["out"] = torch.empty(n, V, dtype=dt, device=DEV)
        s["best"] = torch.empty(n, dtype=torch.int32, device=DEV)
    if own:
        s["call"] = _calls(s)
    return s


def turns_per_position(case):
    i = np.arange(case["rot"] // 2, dtype=np.float64)
    return case["theta"] ** (-2.0 * i / case["rot"]) / (2 * np.pi)


def _calls(s):
    """The prepared call that a user's program keeps for this step's buffers."""
    from chat_wgpu_b200 import GpuContext
    from chat_wgpu_b200.kernels import logits, prompt, rope

    c = s["case"]
    ctx = s["ctx"] = GpuContext(0, stream=torch.cuda.current_stream().cuda_stream)
    w = lambda x: None if x is None else ctx.wrap(x)  # noqa: E731
    if c["op"] == "heads":
        plan = rope.rope_plan(ctx, c["rot"], c["theta"])
        return rope.NormRope(
            ctx, plan=plan, positions=w(s["positions"]), dtype=c["dtype"], layout=c["layout"],
            n_tokens=c["tokens"], n_heads=c["heads"], n_kv=c["kv"], head_dim=c["dim"], eps=1e-6,
            unit_shift=c["shift"], q=w(s["q"]), q_stride=s["q"].stride(0), q_norm=w(s["q_norm"]),
            q_out=w(s["q_out"]), k=w(s["k"]), k_stride=s["k"].stride(0), k_norm=w(s["k_norm"]),
            k_out=w(s["k_out"]), v=w(s["v"]), v_stride=s["v"].stride(0), slots=w(s["slots"]),
            k_cache=w(s["k_cache"]), v_cache=w(s["v_cache"]), page_size=c["page"],
            n_pages=s["n_pages"])
    if c["op"] == "prompt":
        return prompt.PromptAttention(
            ctx, q=w(s["q"]), k=w(s["k"]), v=w(s["v"]), starts=w(s["starts"]),
            key_starts=w(s["key_starts"]), out=w(s["o"]), dtype=c["dtype"], n_req=c["req"],
            n_rows=s["q"].shape[0], n_keys=s["k"].shape[0], n_heads=c["heads"], n_kv=c["kv"],
            head_dim=c["dim"], v_stride=s["v"].stride(0), window=c["window"],
            softcap=c["softcap"])
    more = {}
    if c["bias"]:
        more.update(bias_tokens=w(s["bias_tokens"]), bias_values=w(s["bias_values"]),
                    bias_starts=w(s["bias_starts"]), n_bias=s["bias_tokens"].numel())
    if c["masks"]:
        more.update(masks=w(s["masks"]), mask_rows=w(s["mask_rows"]), n_masks=c["masks"])
    return logits.AdjustLogits(
        ctx, logits=w(s["logits"]), out=w(s["out"]), best=w(s["best"]), dtype=c["dtype"],
        n_rows=c["rows"], vocab=c["vocab"], penalties=w(s["penalties"]), tokens=w(s["tokens"]),
        starts=w(s["starts"]), prompts=w(s["prompts"]), n_tokens=s["tokens"].numel(), **more)


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        s["call"]()
        if c["op"] == "heads":
            y = {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
            return {**y, "k": s["k_out"]} if c["rows"] else y
        if c["op"] == "prompt":
            return {"out": s["o"]}
        return {"out": s["out"], "best": s["best"]}
    return {"heads": _plain_heads, "prompt": _plain_prompt, "logits": _plain_logits}[c["op"]](s)


def _plain_heads(s):
    c = s["case"]
    T, H, K, D, P, R = (c[k] for k in ("tokens", "heads", "kv", "dim", "page", "rot"))
    # turns modulo one as 64-bit whole numbers: no angle grows past half a turn
    turns = (s["positions"].long()[:, None] * s["steps"][None, :]).float() * 2.0 ** -64
    cos = torch.cos(turns * (2 * math.pi))[:, None]
    sin = torch.sin(turns * (2 * math.pi))[:, None]

    def head(x, heads, w):
        x = x.reshape(T, heads, D).float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (w + 1.0 if c["shift"] else w)
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
    k = head(s["k"], K, s["k_norm"])
    s["k_cache"][to // P, :, to % P] = k[live]
    s["v_cache"][to // P, :, to % P] = s["v"].reshape(T, K, D)[live]
    y = {"q": head(s["q"], H, s["q_norm"]).reshape(T, H * D), "k_cache": s["k_cache"],
         "v_cache": s["v_cache"]}
    return {**y, "k": k.reshape(T, K * D)} if c["rows"] else y


def _plain_prompt(s):
    c = s["case"]
    H, K, D = (c[k] for k in ("heads", "kv", "dim"))
    out = torch.empty_like(s["q"])
    row = key = 0
    for nq, nk in zip(*(x.tolist() for x in s["lengths"])):
        k = s["k"][key:key + nk].reshape(nk, K, D).permute(1, 2, 0).float()
        v = s["v"][key:key + nk].reshape(nk, K, D).transpose(0, 1).float()
        step = max(1, min(nq, (1 << 28) // (H * nk)))  # rows at a time: a gigabyte of scores
        for a in range(0, nq, step):
            b = min(nq, a + step)
            end = b + nk - nq  # keys that these rows may see
            q = s["q"][row + a:row + b].reshape(b - a, K, H // K, D).permute(1, 2, 0, 3).float()
            x = (q.reshape(K, -1, D) @ k[:, :, :end]).reshape(K, H // K, b - a, end) * D ** -0.5
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            i = torch.arange(a, b, device=DEV)[:, None] + (nk - nq)
            j = torch.arange(end, device=DEV)[None, :]
            hide = j > i
            if c["window"]:
                hide = hide | (i - j >= c["window"])
            x = x.masked_fill_(hide, -math.inf)
            e = torch.exp_(x - x.amax(-1, keepdim=True))
            o = (e.reshape(K, -1, end) @ v[:, :end]).reshape(K, H // K, b - a, D)
            o = o / e.sum(-1, keepdim=True)
            out[row + a:row + b] = o.permute(2, 0, 1, 3).reshape(b - a, H * D).to(out.dtype)
        row, key = row + nq, key + nk
    return {"out": out}


def _plain_logits(s):
    c = s["case"]
    n, V = c["rows"], c["vocab"]
    y = s["logits"].float()
    m = s["tokens"].numel()
    at = torch.arange(m, device=DEV, dtype=torch.int32)
    row = torch.searchsorted(s["starts"][1:].contiguous(), at, right=True)
    live = row < n
    row = row.clamp(max=n - 1)
    cell = row * V + s["tokens"]
    made = live & (at - s["starts"][row] >= s["prompts"][row])
    seen = torch.zeros(n * V, dtype=torch.int32, device=DEV)
    seen.index_add_(0, cell, live.to(torch.int32))
    count = torch.zeros(n * V, dtype=torch.int32, device=DEV)
    count.index_add_(0, cell, made.to(torch.int32))
    seen, count = seen.view(n, V) > 0, count.view(n, V)
    rep, freq, pres = (s["penalties"][:, i:i + 1] for i in range(3))
    y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
    y = torch.where(count > 0, y - freq * count.float() - pres, y)
    if c["bias"]:
        b = s["bias_tokens"].numel()
        at = torch.arange(b, device=DEV, dtype=torch.int32)
        row = torch.searchsorted(s["bias_starts"][1:].contiguous(), at, right=True)
        row = row.clamp(max=n - 1)
        last = torch.full((n * V,), -1, dtype=torch.int32, device=DEV)
        last.scatter_reduce_(0, row * V + s["bias_tokens"],
                             torch.where(at < s["bias_starts"][-1], at, -1), "amax")
        last = last.view(n, V)
        y = torch.where(last >= 0, y + s["bias_values"][last.clamp(min=0).long()], y)
    if c["masks"]:
        v = torch.arange(V, device=DEV)
        bit = (s["masks"][s["mask_rows"].clamp(min=0).long()][:, v // 32] >> (v % 32)) & 1
        y = torch.where((bit == 1) | (s["mask_rows"] < 0)[:, None], y, torch.full_like(y, -math.inf))
    y = y.to(s["logits"].dtype)
    v = torch.arange(V, device=DEV, dtype=torch.int32)
    best = torch.where(y == y.amax(-1, keepdim=True), v, torch.full_like(v, V)).amin(-1)
    return {"out": y, "best": best}


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "heads":
        T, H, K, D, P, R = (case[k] for k in ("tokens", "heads", "kv", "dim", "page", "rot"))
        f = torch.from_numpy(turns_per_position(case)).to(DEV)
        z = torch.exp(2j * math.pi * torch.frac(s["positions"].double()[:, None] * f))[:, None]

        def turned(x, heads, w):
            x = x.double().reshape(T, heads, D)
            x = x / (x.square().sum(-1, keepdim=True) / D + 1e-6).sqrt()
            x = x * (w.double() + int(case["shift"]))
            if case["layout"] == "half":
                y = torch.complex(x[:, :, :R // 2], x[:, :, R // 2:R]) * z
                x[:, :, :R // 2], x[:, :, R // 2:R] = y.real, y.imag
            else:
                y = torch.complex(x[:, :, 0:R:2], x[:, :, 1:R:2]) * z
                x[:, :, 0:R:2], x[:, :, 1:R:2] = y.real, y.imag
            return x

        kc = s["k_cache"].double().transpose(1, 2).reshape(-1, K, D)
        vc = s["v_cache"].double().transpose(1, 2).reshape(-1, K, D)
        live = torch.nonzero(s["slots"] >= 0)[:, 0]
        k = turned(s["k"], K, s["k_norm"])
        kc[s["slots"][live].long()] = k[live]
        vc[s["slots"][live].long()] = s["v"].double().reshape(T, K, D)[live]
        back = lambda x: x.reshape(s["n_pages"], P, K, D).transpose(1, 2).contiguous()  # noqa: E731
        y = {"q": turned(s["q"], H, s["q_norm"]).reshape(T, H * D), "k_cache": back(kc),
             "v_cache": back(vc)}
        return {**y, "k": k.reshape(T, K * D)} if case["rows"] else y
    if case["op"] == "prompt":
        H, K, D = (case[k] for k in ("heads", "kv", "dim"))
        out = torch.zeros_like(s["q"], dtype=torch.float64).view(-1, K, H // K, D)
        starts = s["starts"].tolist()
        keys = starts if s["key_starts"] is None else s["key_starts"].tolist()
        for r in range(case["req"]):
            nq, nk = starts[r + 1] - starts[r], keys[r + 1] - keys[r]
            for h in range(K):
                k = s["k"][keys[r]:keys[r + 1], h * D:(h + 1) * D].double()
                v = s["v"][keys[r]:keys[r + 1], h * D:(h + 1) * D].double()
                for a in range(0, nq, 1024):
                    b = min(a + 1024, nq)
                    first, last = a + nk - nq, b - 1 + nk - nq
                    low = max(0, first + 1 - case["window"]) if case["window"] else 0
                    q = s["q"][starts[r] + a:starts[r] + b].view(b - a, K, H // K, D)[:, h].double()
                    x = torch.einsum("tgd,kd->tgk", q, k[low:last + 1]) / math.sqrt(D)
                    if case["softcap"]:
                        x = torch.tanh(x / case["softcap"]) * case["softcap"]
                    dist = (first + torch.arange(b - a, device=DEV)[:, None]
                            - torch.arange(low, last + 1, device=DEV)[None, :])
                    see = dist >= 0
                    if case["window"]:
                        see &= dist < case["window"]
                    w = torch.softmax(x.masked_fill(~see[:, None], -math.inf), dim=-1)
                    out[starts[r] + a:starts[r] + b, h] = torch.einsum("tgk,kd->tgd", w,
                                                                       v[low:last + 1])
        return {"out": out.reshape(-1, H * D)}
    out = s["logits"].double()
    words, p = s["tokens"].tolist(), s["penalties"].double().tolist()
    lead = s["prompts"].tolist()
    for r in range(case["rows"]):
        a, b = int(s["starts_host"][r]), int(s["starts_host"][r + 1])
        if b > a:
            ids = torch.tensor(sorted(set(words[a:b])), device=DEV)
            x = out[r, ids]
            out[r, ids] = torch.where(x > 0, x / p[r][0], x * p[r][0])
        if b > a + lead[r]:
            ids, many = np.unique(np.array(words[a + lead[r]:b]), return_counts=True)
            out[r, torch.from_numpy(ids).to(DEV)] -= \
                torch.from_numpy(many).to(DEV).double() * p[r][1] + p[r][2]
        if case["bias"]:
            a, b = int(s["bias_host"][r]), int(s["bias_host"][r + 1])
            add = dict(zip(s["bias_tokens"][a:b].tolist(), s["bias_values"][a:b].tolist()))
            if add:
                out[r, torch.tensor(list(add), device=DEV)] += \
                    torch.tensor(list(add.values()), device=DEV, dtype=torch.float64)
        if case["masks"] and int(s["mask_rows"][r]) >= 0:
            word = s["masks"][int(s["mask_rows"][r])].cpu().numpy().view(np.uint8)
            on = np.unpackbits(word, bitorder="little")[:case["vocab"]].astype(bool)
            out[r, torch.from_numpy(~on).to(DEV)] = -math.inf
    return {"out": out, "best": None}


# ---------------------------------------------------------------- the floor
def work(case):
    """What one pass cannot do without, for the mean lengths of the case."""
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "heads":
        T, H, K, D = (case[k] for k in ("tokens", "heads", "kv", "dim"))
        written = H + 2 * K + (K if case["rows"] else 0)
        return {"bytes": T * (H + 2 * K + written) * D * es + 8 * T + 8 * D,
                "flops": T * (H + K) * (4 * D + 3 * case["rot"])}
    if case["op"] == "prompt":
        nq, nk = lengths(case, 0)
        H, K, D = (case[k] for k in ("heads", "kv", "dim"))
        pairs, seen = 0, 0
        for a, b in zip(nq.tolist(), nk.tolist()):
            w = min(case["window"], b) if case["window"] else b
            short = max(0, min(a, w - 1 - (b - a)))  # rows that the window does not cut
            pairs += short * (b - a) + short * (short + 1) // 2 + (a - short) * w
            seen += min(b, a + w - 1)
        return {"bytes": es * D * (2 * H * int(nq.sum()) + 2 * K * seen),
                "flops": 4 * H * D * pairs}
    n, V = case["rows"], case["vocab"]
    mean = lambda most: most if n == 1 else (most // 4 + most) / 2  # noqa: E731
    return {"bytes": int(2 * n * V * es + 4 * n * mean(case["history"]) + 8 * n * mean(case["bias"])
                         + case["masks"] * -(-V // 32) * 4 + 32 * n),
            "flops": 4 * int(n * mean(case["history"]))}
