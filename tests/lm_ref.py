"""Plain numpy forms, in 64 bits, of the language-model decode operators, and the error bounds the
tests hold the kernels to."""
import numpy as np

GROUP = 64
# One m16n8k16 product adds its 16 terms to the fp32 accumulator with the smaller terms cut off at
# the last bit of the largest, at most 2^-22 of the terms' absolute sum; a group of 128 columns
# takes 8 of them, so 2^-19 of the absolute sum bounds the products of any group.  The split of an
# fp32 operand in two fp16 parts leaves 2^-21, each fp32 addition across groups 2^-24.
PRODUCT = 2.0 ** -19 + 2.0 ** -21


def q4_weight(codes, scales, zeros, K, group):
    c = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)[:, :K].astype(np.float64)
    at = np.arange(K) // group
    z = 8.0 if zeros is None else zeros[:, at].astype(np.float64)
    return (c - z) * scales[:, at].astype(np.float64)


def linear(x, w, bias=None, gate_up=False, groups=1):
    """(y, bound on |error|) of x . w^T + bias, or of silu(gate) * up."""
    x = x.astype(np.float64)
    y = x @ w.T
    tol = (PRODUCT + (groups + 8) * 2.0 ** -24) * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        y = y + bias
        tol = tol + 2.0 ** -23 * (np.abs(y) + np.abs(bias))
    tol = tol + 2.0 ** -24 * np.abs(y) + 1e-37
    if not gate_up:
        return y, tol
    h = y.shape[1] // 2
    g, u, tg, tu = y[:, :h], y[:, h:], tol[:, :h], tol[:, h:]
    with np.errstate(over="ignore"):
        silu = g / (1.0 + np.exp(-g))
    # |d silu / d g| <= 1.1; expf, the division and the product round a few times each
    return silu * u, 1.1 * tg * np.abs(u) + np.abs(silu) * tu + 1.1 * tg * tu + 2.0 ** -20 * np.abs(silu * u)


def norm_rope(x, heads, hd, weight, cos, sin, pos, interleaved, eps):
    """(y, bound): sums of hd squares by trees of depth <= 16, then seven roundings at most."""
    T = x.shape[0]
    x = x.astype(np.float64).reshape(T, heads, hd)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if weight is not None:
        y = y * weight.astype(np.float64)
    out, mag = y.copy(), np.abs(y)
    if cos is not None:
        c, s = cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None]
        i, j = (np.s_[..., 0::2], np.s_[..., 1::2]) if interleaved else (np.s_[..., : hd // 2], np.s_[..., hd // 2 :])
        a, b = y[i], y[j]
        out[i], out[j] = a * c - b * s, b * c + a * s
        mag[i] = mag[j] = np.abs(a) + np.abs(b)
    return out.reshape(T, heads * hd), (2.0 ** -20 * mag).reshape(T, heads * hd) + 1e-37


def kv_hold(x):
    """The values a cache holds for x [..., hd], from IEEE fp32 and fp16 steps: bit for bit."""
    x = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)  # a NaN makes both NaN
        big = np.float32(65504.0)
        m = np.where(lo < -big, -big, np.where(lo > big, big, lo)).astype(np.float16).astype(np.float32)
        step = (hi - lo) / np.float32(15.0)
        s = np.where(step > big, big, step).astype(np.float16).astype(np.float32)
        c = np.clip(np.rint((x - m) / np.where(s > 0, s, np.float32(1))), 0, 15).astype(np.float32)
        y = m + s * np.where(s > 0, c, np.float32(0))
    return y.reshape(*y.shape[:-2], -1)


def attention(q, k, v, pos, window, sinks, scale):
    """One sequence: q [n, H, hd] at positions pos, the values held k, v [L, KVH, hd].
    Returns (out, bound).  The score's products are bounded as in PRODUCT and shift each weight by
    that factor; the weighted sum carries the same relative error as a product of 128 columns."""
    n, H, hd = q.shape
    L, KVH = k.shape[:2]
    out, tol = np.zeros((n, H, hd)), np.zeros((n, H, hd))
    j = np.arange(L)
    for i in range(n):
        see = j <= pos[i]
        if window > 0:
            see &= (j > pos[i] - window) | (j < sinks)
        if not see.any():
            continue
        for h in range(H):
            kk, vv = k[see, h // (H // KVH)].astype(np.float64), v[see, h // (H // KVH)].astype(np.float64)
            qq = q[i, h].astype(np.float64)
            x = scale * (kk @ qq)
            # the code products and the minimum's term are separate sums: codes s and minima m are
            # each at most the group's span and largest value
            span = 2.0 * np.abs(kk).max() * np.abs(qq).sum()
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, h] = p @ vv
            d = PRODUCT * scale * span
            top = np.abs(vv).max()
            tol[i, h] = (2.0 * d + 4.0 * PRODUCT) * 2.0 * top
    return out, tol + 1e-30


def rel(a, b):
    n = np.linalg.norm(b)
    return np.linalg.norm(np.asarray(a, np.float64) - b) / n if n else float(np.abs(a).max())


def attention_exact(q, k, v, pos, window, sinks, scale):
    """One sequence in 64 bits: q [n, H, hd] at positions pos, the values held k [L, KVH, hd], v [L, KVH, dv]."""
    n, H, _ = q.shape
    L, KVH = k.shape[:2]
    j, per = np.arange(L), H // KVH
    see = j <= np.asarray(pos)[:, None]
    if window > 0:
        see &= (j > np.asarray(pos)[:, None] - window) | (j < sinks)
    out = np.zeros((n, H, v.shape[2]))
    for h in range(H):
        x = np.where(see, scale * (q[:, h].astype(np.float64) @ k[:, h // per].astype(np.float64).T), -np.inf)
        top = x.max(-1, keepdims=True)
        p = np.exp(x - np.where(top > -np.inf, top, 0.0))
        total = p.sum(-1, keepdims=True)
        out[:, h] = (p / np.where(total > 0, total, 1.0)) @ v[:, h // per].astype(np.float64)
    return out
