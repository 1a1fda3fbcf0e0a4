"""Plain 64-bit restatement of the 8-bit key/value cache, of attention over it and of token log probabilities (numpy)."""
import numpy as np

BLOCK = 64


def rotate(x, positions, inv_freq, width, pairs=False):
    """x [tokens, heads, head_width] float32 -> float32: the turn in 64 bits, one rounding."""
    out = x.astype(np.float64)
    angle = positions.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
    c, s = np.cos(angle), np.sin(angle)
    i = np.arange(width // 2)
    a, b = (2 * i, 2 * i + 1) if pairs else (i, i + width // 2)
    u, w = out[..., a].copy(), out[..., b].copy()
    out[..., a], out[..., b] = u * c - w * s, w * c + u * s
    return out.astype(np.float32)


def cached(x):
    """x [tokens, heads, head_width] float32 from position 0 on -> the float32 values the cache stands for."""
    out = np.zeros_like(x)
    for t in range(0, x.shape[0], BLOCK):
        block = x[t:t + BLOCK]
        for h in range(x.shape[1]):
            v = block[:, h]
            if not np.all(np.isfinite(v)):
                out[t:t + BLOCK, h] = np.nan
                continue
            scale = np.float32(np.abs(v).max()) / np.float32(127)
            if scale > 0:
                codes = np.clip(np.rint(v.astype(np.float64) / np.float64(scale)), -127, 127)
                out[t:t + BLOCK, h] = codes.astype(np.float32) * scale
    return out


def attend(q, k, v, start, window=0, sinks=0, scale=None):
    """q [n, heads, w], k, v [total, kv_heads, w] -> float64 [n, heads, w], and the largest scale * sum |q K| of a row."""
    n, heads, w = q.shape
    group = heads // k.shape[1]
    scale = 1.0 / np.sqrt(w) if scale is None else scale
    p, t = np.arange(start, start + n)[:, None], np.arange(k.shape[0])[None]
    hidden = t > p
    if window:
        hidden |= (t <= p - window) & (t >= sinks)
    out, reach = np.zeros(q.shape), 0.0
    for h in range(heads):
        kh, vh, qh = k[:, h // group].astype(np.float64), v[:, h // group].astype(np.float64), q[:, h].astype(np.float64)
        s = np.where(hidden, -np.inf, scale * np.einsum("nd,td->nt", qh, np.where(hidden.all(0)[:, None], 0.0, kh)))
        reach = max(reach, float(np.nanmax(scale * (np.abs(qh) @ np.abs(np.nan_to_num(kh)).T))))
        e = np.where(hidden, 0.0, np.exp(s - s.max(1, keepdims=True)))
        out[:, h] = (e @ np.where(hidden.all(0)[:, None], 0.0, vh)) / e.sum(1, keepdims=True)
    return out, reach


def log_probs(logits):
    """float64 log softmax and entropy of rows."""
    x = logits.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        d = x - x.max(1, keepdims=True)
        lp = d - np.log(np.exp(d).sum(1, keepdims=True))
        p = np.exp(lp)
        entropy = -np.where(p > 0, p * lp, 0.0).sum(1)
    return lp, entropy
