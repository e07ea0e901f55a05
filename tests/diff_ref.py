"""Differential attention in 64 bits over a pool's pages, and how far a kernel may
be from it (test infrastructure)."""
import numpy as np

import airkv

F8 = np.zeros(256)
for _c in range(256):
    _e, _m = (_c >> 3) & 15, _c & 7
    F8[_c] = (-1 if _c & 128 else 1) * ((1 + _m / 8) * 2.0 ** (_e - 7) if _e else 0.0)
F8[0x7F] = np.nan
EPS = {airkv.F32: 2.0 ** -24, airkv.BF16: 2.0 ** -8}      # half a rounding step, relative


def pool_values(pool):
    """(K, V) of every page as float64 [num_blocks][heads][bs][d]."""
    k, v, ks, vs = pool.snapshot()
    out = []
    for x, s in ((k, ks), (v, vs)):
        if pool.dtype == airkv.BF16:
            x = (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        elif pool.dtype == airkv.FP8:
            x = F8[x]
        else:
            x = x.astype(np.float64)
        if s is not None:
            x = x * np.repeat(s.astype(np.float64), pool.scale_group, axis=-1)
        out.append(x)
    return out


def sequence(values, table, n, bs):
    """[heads][n][d] of the first n tokens; None blocks (outside the pool) as zeros."""
    nb = -(-n // bs)
    x = np.stack([values[b] if 0 <= b < len(values) else np.zeros_like(values[0]) for b in table[:nb]]) if nb else \
        np.zeros((0,) + values.shape[1:])
    return x.transpose(1, 0, 2, 3).reshape(values.shape[1], -1, values.shape[3])[:, :n]


def attend(q, k, v, lam, scale, sees, norm_weight=None, norm_eps=None, out_scale=1.0, p_step=0.0, skip=None):
    """One sequence: q [rows][2 pairs][d], k / v [heads][n][d], lam [rows][pairs],
    row r sees keys 0 .. sees[r]; skip[n]: keys left out.  Returns (out [rows][pairs]
    [2 d], bound): the bound of the difference of a kernel that holds scores,
    probabilities and sums in 32 bits and rounds probabilities by p_step (0: not),
    from
      scores:  products of d terms, each sum off by at most d 2^-24 sum|q k|, three
               more roundings (scale, maximum, exponential) of a value of at most
               that size and 16: relative error of p
      sums:    (n + 64) 2^-24 of sum p |v|, and as much of sum p
      norm:    the difference's relative error twice (the value, the mean square)
    """
    rows, heads, d = q.shape
    n = k.shape[1]
    pairs, kvp = heads // 2, k.shape[0] // 2
    g = pairs // kvp
    out = np.zeros((rows, pairs, 2 * d))
    bound = np.zeros((rows, pairs, 2 * d))
    if n == 0:
        return out, bound
    hidden = np.arange(n)[None, :] > np.asarray(sees)[:, None]
    if skip is not None:
        hidden = hidden | skip[None, :]
    eps = 2.0 ** -24
    for h in range(pairs):
        p = h // g
        vv = np.concatenate([v[2 * p], v[2 * p + 1]], -1)
        x = np.zeros((rows, 2 * d))
        off = np.zeros((rows, 2 * d))
        for m in range(2):
            s = q[:, 2 * h + m] @ k[2 * p + m].T * scale
            size = np.abs(q[:, 2 * h + m]) @ np.abs(k[2 * p + m]).T * abs(scale)
            s[hidden] = -np.inf
            with np.errstate(invalid="ignore"):
                w = np.exp(s - s.max(-1, keepdims=True))
            w = np.where(hidden, 0, w)
            total = w.sum(-1, keepdims=True)
            w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
            f = np.ones((rows, 1)) if m == 0 else -lam[:, h:h + 1]
            live = np.where(hidden, 0, size)
            rel = eps * (2 * (d + 4) * live.max(-1, keepdims=True) + 2 * (n + 64) + 64) + p_step
            x += f * (w @ vv)
            off += np.abs(f) * rel * (w @ np.abs(vv))
        factor = np.full((rows, 1), out_scale)
        if norm_eps is not None:
            rms = np.sqrt((x * x).mean(-1, keepdims=True) + norm_eps)
            drms = np.sqrt((off * off).mean(-1, keepdims=True))
            # x (1 / (rms - drms) - 1 / rms) for the norm's own error
            off = off + np.abs(x) * drms / np.maximum(rms - drms, 1e-30)
            factor = out_scale / rms * (norm_weight[None] if norm_weight is not None else 1.0)
        out[:, h] = x * factor
        bound[:, h] = np.abs(off * factor) + 8 * eps * np.abs(out[:, h])
    return out, bound


def check(got, out, bound, out_dtype, what, p_step=0.0):
    """got within the bound of out, and of its own rounding."""
    bound = bound * (1 + EPS[out_dtype]) + EPS[out_dtype] * np.abs(out) + 2.0 ** -149
    bad = ~(np.abs(got - out) <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} beyond the bound, at {np.argwhere(bad)[:3].tolist()}: "
                           f"{got[bad][:3]} against {out[bad][:3]}, allowed {bound[bad][:3]}")
    # the bound lets every rounding go the same way; at random n of them add up to
    # sqrt(n) half steps: 100 * 2^-24 at 10^4 keys, against the whole result
    if out_dtype == airkv.F32 and p_step == 0.0 and out.any():
        rel = float(np.linalg.norm(got - out) / np.linalg.norm(out))
        assert rel <= 1e-5, f"{what}: {rel:.2g} off"
    return float((np.abs(got - out) / bound).max()) if got.size else 0.0
