"""Plain 64-bit statements of a cache that holds keys and values in 8 bits: how a row is held, what it stands for, attention over it.

A row of D numbers x: a = max|x|; scale = a / 127 (int8) or a / 448 (e4m3); code = x / scale to the nearest, ties to even; it stands
for code * scale.  Below 2^-100 a row is zeros; with an infinity or a NaN it reads as NaN.
"""
import numpy as np

MOST = {"int8": 127.0, "float8_e4m3": 448.0}


def nearest_e4m3(y):
    """The e4m3 number nearest to y (3 bits behind the leading one, least normal 2^-6, steps of 2^-9 below), ties to even."""
    y = np.asarray(y, dtype=np.float64)
    _, e = np.frexp(y)
    step = 2.0 ** (np.maximum(e - 1, -6) - 3.0)
    return np.clip(np.round(y / step) * step, -448.0, 448.0)


def held(x, kind):
    """float64 rows [..., D] -> (codes as numbers, scales [...])."""
    x = np.asarray(x, dtype=np.float64)
    fine = np.isfinite(x).all(axis=-1)
    a = np.abs(np.where(fine[..., None], x, 0.0)).max(axis=-1)
    a = np.where(a < 2.0 ** -100, 0.0, a)
    scale = a / MOST[kind]
    y = np.where(fine[..., None] & (a > 0)[..., None], np.where(fine[..., None], x, 0.0) / np.where(a > 0, scale, 1.0)[..., None], 0.0)
    codes = np.round(y) if kind == "int8" else nearest_e4m3(y)
    return codes, np.where(fine, scale, np.nan)


def stands_for(x, kind):
    codes, scale = held(x, kind)
    return codes * scale[..., None]


def half_step(codes, scale, kind):
    """Half the distance between neighbouring codes at ``codes``, in the row's units: what the rounding may be off by."""
    if kind == "int8":
        return np.broadcast_to(0.5 * scale[..., None], codes.shape)
    _, e = np.frexp(codes)
    return 2.0 ** (np.maximum(e - 1, -6) - 4.0) * scale[..., None]


def attention(q, k, v, pos, scale, window=0):
    """q [T, H, D] at positions ``pos`` [T] over one sequence's keys and values [N, G, D] (as they stand); -> (out [T, H, D],
    largest sum_d |q_d k_d| * scale over the keys a row sees [T, H], largest |v| it sees [T, H]).  A row that sees nothing: zeros."""
    T, H, D = q.shape
    N, G = k.shape[:2]
    key = np.arange(N)
    seen = key[None, :] <= np.asarray(pos)[:, None]
    if window > 0:
        seen &= key[None, :] > np.asarray(pos)[:, None] - window
    kf, vf = np.where(np.isfinite(k), k, 0.0), np.where(np.isfinite(v), v, 0.0)
    bad = ~(np.isfinite(k).all(axis=-1) & np.isfinite(v).all(axis=-1))          # [N, G]
    out, sums, most = np.zeros((T, H, D)), np.zeros((T, H)), np.zeros((T, H))
    for h in range(H):
        g = h // (H // G)
        s = np.where(seen, (q[:, h] @ kf[:, g].T) * scale, -np.inf)
        m = s.max(axis=1, keepdims=True, initial=-np.inf)
        w = np.exp(s - np.where(np.isfinite(m), m, 0.0))
        total = w.sum(axis=1, keepdims=True)
        out[:, h] = (w @ vf[:, g]) / np.where(total > 0, total, 1.0)
        out[(seen & bad[None, :, g]).any(axis=1), h] = np.nan
        sums[:, h] = np.where(seen, (np.abs(q[:, h]) @ np.abs(kf[:, g]).T) * abs(scale), 0.0).max(axis=1)
        most[:, h] = np.where(seen, np.abs(vf[:, g]).max(axis=-1)[None, :], 0.0).max(axis=1)
    return out, sums, most
