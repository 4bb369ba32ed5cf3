"""The token-mixer operators restated in 64 bits on the CPU (numpy), element by element from their definitions, together with
the magnitudes that bound the rounding errors of an f32 or bfloat16 evaluation."""
import numpy as np

U32, U16 = 2.0 ** -24, 2.0 ** -8   # half a step of f32 and bfloat16, relative to the value

LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)


def bf16(a):
    """Values rounded to bfloat16 (nearest even), as f32."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).bfloat16().float().numpy()


def norm_rope(x, w, eps, norm, cos, sin, pos, rot_at, halves):
    """x [T, h, hd] -> (y, mag): the result and, per value, the magnitude of the pair it was rotated in."""
    y = x.astype(np.float64)
    if norm:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    if w is not None:
        y = y * w.astype(np.float64)
    mag = np.abs(y)
    if cos is not None:
        half = cos.shape[1]
        c, s = cos.astype(np.float64)[pos][:, None], sin.astype(np.float64)[pos][:, None]
        ia = rot_at + (np.arange(half) if halves else 2 * np.arange(half))
        ib = ia + (half if halves else 1)
        a, b = y[..., ia].copy(), y[..., ib].copy()
        y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
        mag[..., ia] = mag[..., ib] = np.abs(a) + np.abs(b)
    return y, mag


def mxfp4(x):
    """The values a 4-bit cache holds for rows x [..., n] (n % 32 == 0)."""
    b = x.astype(np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    b = np.where(np.isnan(b), 0.0, b)
    top = np.abs(b).max(-1, keepdims=True)
    e = np.full(top.shape, -127)
    for k in range(-126, 126):
        e = np.where(6.0 * 2.0 ** (k - 1) < top, k, e)
    a = np.minimum(np.abs(b), 1e300) / 2.0 ** e.astype(np.float64)
    i = (a[..., None] >= np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5])).sum(-1)
    return (np.where(b < 0, -1.0, 1.0) * LEVELS[i] * 2.0 ** e.astype(np.float64)).reshape(x.shape)


def attn(q, k, v, limit, scale):
    """One row: q [nh, w], k [n, nkv, w], v [n, nkv, dv] -> (out [nh, dv], bound of |error| / 2^-24 of an f32 evaluation, sum p |v|).
    Scores: a dot product of w terms errs by at most (w + 2) half steps of sum |q k|; a weight by twice the largest score
    error (the score and the maximum) and a few half steps of the exponential; the sum over n positions by n half steps."""
    nh, w = q.shape
    rep = nh // k.shape[1]
    if limit < 0:
        z = np.zeros((nh, v.shape[2]))
        return z, z, z
    out, bound, mag = [], [], []
    for h in range(nh):
        kk, vv, qq = k[:limit + 1, h // rep].astype(np.float64), v[:limit + 1, h // rep].astype(np.float64), q[h].astype(np.float64)
        s = kk @ qq * scale
        ds = (w + 2) * (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
        p = np.exp(s - s.max())
        p /= p.sum()
        m = p @ np.abs(vv)
        out.append(p @ vv)
        bound.append((2 * ds + limit + 1 + 16) * m)
        mag.append(m)
    return np.stack(out), np.stack(bound), np.stack(mag)


def linear(q, k, v, g, state, scale):
    """One sequence: q, k [T, nkh, dk], v [T, nh, dv], g [T, nh] -> (out, state, |out|-magnitude, |state|-magnitude): the magnitudes
    are the same recurrence over absolute values."""
    T, nh, dv = v.shape
    rep = nh // q.shape[1]
    q, k = np.repeat(q.astype(np.float64), rep, 1), np.repeat(k.astype(np.float64), rep, 1)
    v, S, M = v.astype(np.float64), state.astype(np.float64).copy(), np.abs(state.astype(np.float64))
    out, mag = np.zeros((T, nh, dv)), np.zeros((T, nh, dv))
    for t in range(T):
        e = np.exp(g[t].astype(np.float64))[:, None, None]
        with np.errstate(invalid="ignore"):
            S = e * S + k[t][:, :, None] * v[t][:, None, :]
            M = e * M + np.abs(k[t])[:, :, None] * np.abs(v[t])[:, None, :]
            out[t] = scale * np.einsum("hd,hde->he", q[t], S)
            mag[t] = abs(scale) * np.einsum("hd,hde->he", np.abs(q[t]), M)
    return out, S, mag, M
