"""Oracle of the serving operators (include/bf16x_llama.h) in numpy: the 4-bit
cache format, attention over it in fp64, and token sampling in fp64."""
from __future__ import annotations

import numpy as np

LARGEST = np.float32(61440.0)


def word_shift(e: int) -> int:
    """Bit of value e (0 .. 7) in its word of codes."""
    return 14 + 2 * e if e & 1 else 2 * e


def quantise(x):
    """x fp32 [..., D] -> (codes uint8 [..., D], scale fp16 [..., D / 32], minimum fp16 [..., D / 32])."""
    x = np.asarray(x, np.float32)
    x = np.where(np.isnan(x), np.float32(0), np.clip(x, -LARGEST, LARGEST))
    g = x.reshape(*x.shape[:-1], -1, 32)
    low = g.min(-1).astype(np.float16)
    lowf = low.astype(np.float32)
    scale = (np.maximum(g.max(-1) - lowf, np.float32(0)) * np.float32(1 / 15)).astype(np.float16)
    s = scale.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        n = np.rint((g - lowf[..., None]) / s)
    n = np.where(s > 0, np.clip(n, 0, 15), 0)
    return n.astype(np.uint8).reshape(x.shape), scale, low


def pack(codes):
    """codes uint8 [..., D] -> bytes uint8 [..., D / 2]."""
    w = codes.reshape(*codes.shape[:-1], -1, 8).astype(np.uint32)
    word = np.zeros(w.shape[:-1], np.uint32)
    for e in range(8):
        word |= w[..., e] << np.uint32(word_shift(e))
    return word.view(np.uint8)


def values(packed, scales):
    """fp64 [..., D] of packed codes uint8 [..., D / 2] and (scale, minimum) fp16 [..., D / 32, 2]."""
    word = np.ascontiguousarray(packed).view(np.uint32)
    code = np.stack([(word >> np.uint32(word_shift(e))) & 15 for e in range(8)], axis=-1).astype(np.float64)
    s = np.asarray(scales, np.float64)
    g = code.reshape(*s.shape[:-1], 32)
    return (g * s[..., :1] + s[..., 1:]).reshape(*packed.shape[:-1], -1)


def rotate(x, cos_sin, positions):
    """x fp32 [B, T, heads, D] at positions [B, T] (cut to the table): products and sums rounded one by one."""
    x = np.asarray(x, np.float32)
    t = cos_sin[np.clip(positions, 0, len(cos_sin) - 1)][:, :, None]
    c, s = t[..., 0], t[..., 1]
    a, b = np.split(x, 2, axis=-1)
    return np.concatenate([a * c - b * s, b * c + a * s], axis=-1).astype(np.float32)


def attention(q, k, v, pos, start=None, window=0, scale=None):
    """q [B, T, H, D], k, v [B, KV, L, D] -> (out, bound): out [B, T, H, D] in
    fp64, and what fp16 values and weights (2^-11 relative, 2^-25 for the
    smallest) may change in it.

    A key's score moves by at most ds = scale sum |q| (2^-11 |k| + 2^-25), a
    weight by the factor exp(2 ds) (its own score and the sum's) and by its own
    rounding, a value by 2^-11 |v| + 2^-25."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    B, T, H, D = q.shape
    KV, L = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    j = np.arange(L)
    h11, tiny = 2.0 ** -11, 2.0 ** -25
    for b in range(B):
        for t in range(T):
            p = int(pos[b]) + t
            ok = j <= p
            if window:
                ok &= j > p - window
            if start is not None:
                ok &= j >= int(start[b])
            if not ok.any():
                continue
            for h in range(H):
                kk, vv = k[b, h // (H // KV)][ok], v[b, h // (H // KV)][ok]
                x = scale * (kk @ q[b, t, h])
                e = np.exp(x - x.max())
                w = e / e.sum()
                ds = abs(scale) * ((h11 * np.abs(kk) + tiny) @ np.abs(q[b, t, h])).max()
                out[b, t, h] = w @ vv
                A = w @ np.abs(vv)
                bound[b, t, h] = (np.expm1(2 * ds) + 2 * h11 + 2.0 ** -18) * A + \
                    tiny * (np.abs(vv).sum(0) / e.sum() + 1)
    return out, bound


def sample(logits, u, temperature, top_k, top_p, min_p):
    """One row in fp64 -> (token, logprob)."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    if m == -np.inf:
        return -1, -np.inf
    if not temperature > 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(x == m, 0.0, (x - m) / np.float64(np.float32(temperature)))
    y = np.where((x == -np.inf) | np.isnan(y), -np.inf, y)
    w = np.where(y >= -31.5, np.exp(y), 0.0)                   # below 2^-45: never drawn
    order = np.argsort(-x, kind="stable")
    ws = w[order]
    n = int((ws > 0).sum())
    if 0 < top_k < len(x):
        n = min(n, int(top_k))
    if top_p < 1:
        c = np.cumsum(ws[:n])
        n = min(n, int((c < max(float(np.float32(top_p)), 0.0) * c[-1]).sum()) + 1)
    kept = np.zeros(len(x), bool)
    kept[order[:n]] = True
    kept &= w >= min(float(np.float32(min_p)), 1.0)
    c = np.cumsum(np.where(kept, w, 0.0))
    token = int(np.searchsorted(c, min(max(float(u), 0.0), 1.0) * c[-1], side="right"))
    token = min(token, int(np.flatnonzero(kept & (w > 0))[-1]))
    return token, float(np.log(w[token] / c[-1]))
