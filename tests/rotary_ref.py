"""Rotary positions in 64 bits and in the framework's own steps (plain numpy)."""
import numpy as np


def frequencies(rot, base=10000.0):
    return (base ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)


def angles(positions, inv_freq):
    """[tokens][pairs], in 64 bits (exact: an integer times an f32)."""
    return np.asarray(positions, np.float64)[:, None] * inv_freq.astype(np.float64)


def _parts(rot, pairs):
    return (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))


def exact(x, positions, inv_freq, pairs, magnitude=1.0):
    """Rows [tokens, heads, d] turned, all in 64 bits."""
    x = np.array(x, np.float64)
    a, b = _parts(2 * len(inv_freq), pairs)
    z = (x[..., a] + 1j * x[..., b]) * (magnitude * np.exp(1j * angles(positions, inv_freq)))[:, None]
    x[..., a], x[..., b] = z.real, z.imag
    return x


def turned(x, positions, inv_freq, pairs, magnitude=1.0):
    """The same in f32: cosine and sine rounded once, products and sums one by one."""
    x = np.array(x, np.float32)
    m = np.float64(np.float32(magnitude))
    t = angles(positions, inv_freq)
    c, s = (np.cos(t) * m).astype(np.float32)[:, None], (np.sin(t) * m).astype(np.float32)[:, None]
    a, b = _parts(2 * len(inv_freq), pairs)
    u, v = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = u * c - v * s, u * s + v * c
    return x


def to_bf16(x):
    """f32 rounded to bfloat16 (nearest even), as bits."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
