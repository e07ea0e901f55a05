"""Cross attention over pages in 64 bits, and how far the kernels may be from it (plain torch on the CPU)."""
import math

import torch

HALF_STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def values(pool, snapshot, scale_group, fp8_table):
    """K and V of a pool in 64 bits, [blocks, kv, bs, d]."""
    import airkv
    out = []
    for i in range(2):
        x, s = snapshot[i], snapshot[2 + i]
        if pool.dtype == airkv.F32:
            y = torch.from_numpy(x.copy()).double()
        elif pool.dtype == airkv.BF16:
            y = torch.from_numpy(x.astype("uint32") << 16).view(torch.float32).double()
        else:
            import numpy as np
            codes = x.view(np.int8).astype(np.float64) if pool.dtype == airkv.INT8 else fp8_table[x].astype(np.float64)
            y = torch.from_numpy((codes.reshape(*s.shape, -1) * s[..., None].astype(np.float64)).reshape(codes.shape))
        out.append(y)
    return out


def cross(q, cu, k, v, tables, lens, scale, bs, precise, rounded_pages, out_type):
    """(out, bound) for rows q [rows, heads, d] in 64 bits; out is NaN and bound infinite for rows of no sequence.

    precise: f32 precision, else probabilities rounded to bf16; rounded_pages: those of 1-byte pages, rounded to f32
    or, with their probabilities, to f16.
    The bound: a score errs by what its products and their sum do, a probability by that times two (its own score
    and the row's sum) and its rounding, an output by its probabilities', its values' and its sum's errors, and by its
    own rounding."""
    rows, heads, d = q.shape
    kv = k.shape[1]
    g = heads // kv
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    bound = torch.full(q.shape, math.inf, dtype=torch.float64)
    u = 2.0 ** -11 if rounded_pages else HALF_STEP["bf16"]
    f = 2.0 ** -24
    # products that are left out of two split values (their parts are below 2^-7 and 2^-15 of them)
    split = 2.0 ** -21 if precise else 0.0
    page = u if rounded_pages and not precise else f if rounded_pages else 0.0
    for b, n in enumerate(lens):
        r0, r1 = cu[b], cu[b + 1]
        if r0 == r1:
            continue
        if n == 0:
            out[r0:r1], bound[r0:r1] = 0.0, 0.0
            continue
        at = torch.arange(n)
        blocks = torch.as_tensor(tables[b]).long()[at // bs]
        there = (blocks >= 0) & (blocks < k.shape[0])
        blocks, off = blocks[there], (at % bs)[there]
        if not len(blocks):
            out[r0:r1], bound[r0:r1] = 0.0, 0.0
            continue
        for h in range(heads):
            x, y, z = q[r0:r1, h], k[blocks, h // g, off], v[blocks, h // g, off]
            s = x @ y.t() * scale
            top = s.abs().max()
            p = torch.softmax(s, -1)
            size = x.abs() @ y.abs().t() * scale
            ds = (size * (page + split + 6 * d * f)).amax(-1, keepdim=True) + top * 2.0 ** -22
            rel = 2 * torch.expm1(ds) + 2.0 ** -20 + (u if not precise else split) + page + 6 * len(blocks) * f
            o = p @ z
            out[r0:r1, h] = o
            bound[r0:r1, h] = (p @ z.abs()) * rel + HALF_STEP[out_type] * o.abs() + 1e-37
    return out, bound
