"""Plain 64-bit forms of the operators that take prompts in and choose from their logits."""
import numpy as np

import paged_ref as ref


def norm_rotate(x, w, shift, eps, pos, f, amp, layout):
    """x [T, heads, D] normed by head (w None: not) and rotated."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (w + float(shift))
    return ref.rotate(x, pos, f, amp, layout)


def attention(q, k, v, starts, key_starts, window, softcap, scale, out):
    """Rows of out (a copy) that belong to a request, from the keys they see only; also the
    largest sum of |q k| scale and the largest |v| of the finite ones that a row meets."""
    out = out.copy()
    H, K = q.shape[1], k.shape[1]
    big_s = big_v = 0.0
    for r in range(len(starts) - 1):
        n, keys = starts[r + 1] - starts[r], key_starts[r + 1] - key_starts[r]
        for i in range(n):
            last = i + keys - n
            first = max(0, last - window + 1) if window else 0
            t = starts[r] + i
            out[t] = 0.0
            if last < first:
                continue
            kk, vv = (x[key_starts[r] + first:key_starts[r] + last + 1] for x in (k, v))
            for h in range(H):
                a, b = kk[:, h // (H // K)], vv[:, h // (H // K)]
                s = a @ q[t, h] * scale
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                with np.errstate(invalid="ignore"):
                    w = np.exp(s - s.max())
                    out[t, h] = w @ b / w.sum()
                m = (np.abs(a) @ np.abs(q[t, h])).max() * scale
                if np.isfinite(m):
                    big_s = max(big_s, m)
                big_v = max(big_v, np.abs(b[np.isfinite(b)]).max())
    return out, big_s, big_v


def adjust(logits, dtype, penalties=None, lists=None, prompts=None, biases=None, masks=None,
           mask_rows=None):
    """Rows of f32 logits after each step's own rounding, as stored; and their argmax."""
    out = logits.astype(np.float32).copy()
    n, V = out.shape
    for r in range(n):
        x = out[r]
        if penalties is not None:
            rep, freq, pres = (np.float32(p) for p in penalties[r])
            lead = int(prompts[r]) if prompts is not None else 0
            counts = {}
            for i, t in enumerate(lists[r]):
                counts[t] = counts.get(t, 0) + (i >= lead)
            for t, c in counts.items():
                x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
                if c:
                    x[t] = np.float32(x[t] - np.float32(freq * np.float32(c))) - pres
        if biases is not None:
            for t, b in dict(biases[r]).items():
                x[t] = np.float32(x[t] + np.float32(b))
        if masks is not None:
            m = int(mask_rows[r]) if mask_rows is not None else r
            if m >= 0:
                x[~masks[m]] = -np.inf
    out = ref.rounded(out, dtype)
    best = []
    for x in out:
        y = np.where(np.isnan(x) | (x <= np.float32(-3.402823e38)), -np.inf, x)
        best.append(int(y.argmax()) if y.max() > -np.inf else 0)
    return out, np.array(best)
