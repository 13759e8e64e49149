"""Plain 64-bit forms of the paged operators, and 16-bit types on the host."""
import math

import numpy as np

UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # rounding of one value
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def to_bits(x, dtype):
    """f32 array -> the stored values' bytes (round to nearest even)."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, dtype, shape):
    """The values of stored bytes, as f64."""
    raw = np.ascontiguousarray(b).view(np.uint8)
    if dtype == "f32":
        return raw.view(np.float32)[:int(np.prod(shape))].reshape(shape).astype(np.float64)
    if dtype == "f16":
        return raw.view(np.float16)[:int(np.prod(shape))].reshape(shape).astype(np.float64)
    w = raw.view(np.uint16)[:int(np.prod(shape))].astype(np.uint32) << 16
    return w.view(np.float32).reshape(shape).astype(np.float64)


def rounded(x, dtype):
    """x after one rounding to the type, as f64."""
    b = to_bits(x, dtype)
    return from_bits(b, dtype, np.shape(x))


def read(ctx, buf, dtype, shape):
    n = int(np.prod(shape)) * SIZE[dtype]
    return from_bits(ctx.read_u32(buf, (n + 3) // 4), dtype, shape)


def upload(ctx, x, dtype):
    """x in the type on the device, padded to whole words."""
    b = to_bits(x, dtype).view(np.uint8).ravel()
    return ctx.storage_bytes(np.concatenate([b, np.zeros(-b.size % 4, np.uint8)]))


def plan(lens, news, free, table, page, max_tokens, depths=None):
    """cw_page_plan on the host, one token at a time."""
    n, max_pages = table.shape
    table = table.copy()
    starts, pos, slots, owners = [0], [], [], []
    used = 0
    for r in range(n):
        c, m = max(int(lens[r]), 0), max(int(news[r]), 0)
        have = min(-(-c // page), max_pages)
        want = min(-(-(c + m) // page), max_pages)
        lacking = set()
        for p in range(have, want):
            if used < len(free):
                table[r, p] = free[used]
            else:
                lacking.add(p)
            used += 1
        for i in range(m):
            at, t = c + i, starts[-1] + i
            p = at // page
            pos.append(c + int(depths[t]) if depths is not None and t < max_tokens else at)
            ok = p < max_pages and p not in lacking and table[r, p] >= 0
            slots.append(int(table[r, p]) * page + at % page if ok else -1)
            owners.append(r)
        starts.append(starts[-1] + m)
    pad = max(0, max_tokens - len(pos))
    fill = lambda a, v: np.array((a + [v] * pad)[:max_tokens], np.int32)  # noqa: E731
    return dict(table=table, starts=np.array(starts, np.int32), used=used,
                positions=fill(pos, 0), slots=fill(slots, -1), owners=fill(owners, -1))


def rates(rot, theta, kind="none", factor=1.0, low=1.0, high=32.0, trained=0, amplitude=0.0):
    """Radians per position of each pair, and the amplitude."""
    out, amp = [], 1.0
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if kind == "linear":
            f /= factor
        elif kind == "banded":
            keep = min(max((trained * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f = f * keep + f / factor * (1 - keep)
        elif kind == "yarn":
            at = lambda t: rot * math.log(trained / (t * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
            ramp = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            f = f / factor * ramp + f * (1 - ramp)
            amp = amplitude or 0.1 * math.log(factor) + 1.0
        out.append(f)
    return np.array(out), amp


def rotate(x, positions, f, amp, layout):
    """x [T, heads, D] rotated, in 64 bits."""
    half = len(f)
    ang = np.asarray(positions, np.float64)[:, None] * f
    c, s = (amp * np.cos(ang))[:, None], (amp * np.sin(ang))[:, None]
    y = x.copy()
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    return y


def attention(q, kc, vc, table, lens, starts, page, see, positions, window, softcap, scale):
    """Rows over the keys they see only.  q [T, H, D]; caches [pages, K, page, D];
    see[r] bool [n, n].  Also the bound's ingredients: the largest sum of |q k| scale
    and the largest |v| that a row meets."""
    T, H, D = q.shape
    K = kc.shape[1]
    out = np.zeros((T, H, D))
    big_s = big_v = 0.0
    for r in range(len(lens)):
        n = int(starts[r + 1] - starts[r])
        total = int(lens[r]) + n
        at = np.arange(total)
        pages = table[r, at // page] if total else np.zeros(0, int)
        for i in range(n):
            t = int(starts[r]) + i
            vis = np.concatenate([np.ones(int(lens[r]), bool), see[r][i]])
            if window:
                where = np.concatenate([np.arange(int(lens[r])),
                                        positions[int(starts[r]):int(starts[r]) + n]])
                vis &= positions[t] - where < window
            j = np.flatnonzero(vis)
            if not len(j):
                continue
            for h in range(H):
                k = kc[pages[j], h // (H // K), j % page]
                v = vc[pages[j], h // (H // K), j % page]
                s = k @ q[t, h] * scale
                big_s = max(big_s, float((np.abs(k) @ np.abs(q[t, h])).max()) * scale)
                big_v = max(big_v, float(np.abs(v).max()))
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                w = np.exp(s - s.max())
                out[t, h] = w @ v / w.sum()
    return out, big_s, big_v
