"""Rotary positions on the way into the paged K/V cache and inside it, and cross
attention over an encoder's cached states, as measurable cases.

Append: a step's queries, keys and values (slices of one projection's rows, or
tensors of their own).  Queries and keys are rotated by their tokens'
positions, keys and values go to their pages, rounded or quantized as the pool
stores them; over 1-byte pages the sequences are read back as dense rows.

Rotate: cached keys, in their pages, from the positions they were appended at
to the ones they have after tokens were dropped.

Cross: every row of a sequence (a decoder's tokens, or beams) attends to all of
the sequence's cached states, whose number has nothing to do with the rows'.

The angle of pair i at position p is p * inv_freq[i]; its cosine and sine are
rounded to 32 bits once, and a rotated value is a product minus (plus) a product.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BYTES = {"f32": 4, "bf16": 2, "int8": 1, "fp8": 1}
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
GROUP = 32            # elements per scale of the quantized pools
BASE = 10000.0


def _append(name, dtype, tokens, batch, past, q, kv, d, bs, rot, layout="half", io="bf16", fused=True, magnitude=1.0,
            shape=0):
    return {"name": name, "kind": "append", "dtype": dtype, "tokens": tokens, "batch": batch, "past": past, "q": q, "kv": kv,
            "d": d, "bs": bs, "rot": rot, "layout": layout, "io": io, "fused": fused, "magnitude": magnitude, "shape": shape}


def _rotate(name, dtype, batch, lo, hi, kv, d, bs, rot, keep, sinks, layout="half", shape=0):
    return {"name": name, "kind": "rotate", "dtype": dtype, "batch": batch, "lo": lo, "hi": hi, "kv": kv, "d": d, "bs": bs,
            "rot": rot, "layout": layout, "keep": keep, "sinks": sinks, "shape": shape}


def _cross(name, dtype, batch, rows_lo, rows_hi, lo, hi, kv, group, d, bs, io="bf16", shape=0):
    return {"name": name, "kind": "cross", "dtype": dtype, "batch": batch, "rows_lo": rows_lo, "rows_hi": rows_hi, "lo": lo,
            "hi": hi, "kv": kv, "group": group, "d": d, "bs": bs, "io": io, "shape": shape}


def listed():
    return [
        # the smallest call: one decode step of four short chats of a small model on
        # the f32 cache, where latency and launches count
        _append("append_f32_small", "f32", 4, 4, 500, 8, 8, 64, 16, 64, io="f32", fused=False, shape=1),
        # a decode step of 64 sequences of an 8B-sized layer, out of one projection
        _append("append_bf16_step", "bf16", 64, 64, 4096, 32, 8, 128, 16, 128, shape=2),
        # one long prompt, positions scaled for a long context (a magnitude beside 1)
        _append("append_bf16_prompt", "bf16", 8192, 1, 0, 32, 8, 128, 16, 128, magnitude=1.1386, shape=3),
        # prompt chunks of a larger model's layer into int8 pages, half of each head
        # rotated, pairs side by side, and the dense rows that a layer in full precision reads
        _append("append_int8_chunks", "int8", 4096, 8, 2000, 64, 8, 128, 16, 64, layout="pairs", shape=4),
        # one sequence of a small model shrunk to its first and its newest tokens
        _rotate("rotate_f32_window", "f32", 1, 511, 511, 8, 64, 16, 64, 0.5, 4, shape=5),
        # four long sequences that kept three quarters of their tokens
        _rotate("rotate_bf16_long", "bf16", 4, 32768, 65536, 8, 128, 32, 128, 0.75, 16, shape=6),
        # four short prompts of a small model in full precision
        _cross("cross_f32_prompts", "f32", 4, 5, 200, 37, 511, 8, 1, 64, 16, io="f32", shape=7),
        # a decode step: 64 sequences, one token each, their encoder's states
        _cross("cross_bf16_step", "bf16", 64, 1, 1, 512, 4096, 8, 4, 128, 16, shape=8),
        # a few beams of one sequence, a long recording
        _cross("cross_fp8_beams", "fp8", 1, 5, 5, 32768, 32768, 8, 1, 64, 32, shape=9),
        # prompts of a batch of small heads
        _cross("cross_bf16_d64", "bf16", 8, 200, 512, 500, 3000, 8, 4, 64, 16, shape=10),
        # ragged chunks of a larger model's layer over int8 pages
        _cross("cross_int8_70b", "int8", 6, 33, 512, 100, 6000, 8, 8, 128, 16, shape=11),
        # one long document against one long encoding: the largest product
        _cross("cross_bf16_long", "bf16", 1, 4096, 4096, 8192, 8192, 8, 4, 128, 32, shape=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "rotate", "cross", "cross", "cross"])
    dtype = rng.choice(["f32", "bf16", "bf16", "int8", "fp8"])
    d = rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 256])
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    case = {"kind": kind, "dtype": dtype, "kv": kv, "d": d, "bs": rng.choice([16, 32]), "shape": rng.randrange(1 << 30)}
    token = 2 * kv * d * BYTES[dtype]                 # cached bytes of one token
    if kind != "cross":
        case["rot"] = rng.choice([d, d, d // 2, max(8, d // 4 // 8 * 8), 8 * rng.randint(1, d // 8)])
        case["layout"] = rng.choice(["half", "half", "pairs"])
    if kind == "append":
        case["q"] = kv * rng.choice([1, 2, 4, 4, 7, 8])
        case["io"] = rng.choice(["bf16", "bf16", "f32"])
        case["fused"] = rng.choice([True, False])
        case["magnitude"] = rng.choice([1.0, 1.0, round(rng.uniform(0.8, 1.4), 4)])
        row = (case["q"] + 2 * kv) * d * BYTES[case["io"]]
        case["tokens"] = max(1, min(_log(rng, 1, 16000), int(1e8 / row)))
        case["batch"] = min(case["tokens"], _log(rng, 1, 64))
        case["past"] = min(rng.choice([0, _log(rng, 10, 8000)]), int(4e8 / token / case["batch"]))
    elif kind == "rotate":
        case["batch"] = _log(rng, 1, 100)
        case["hi"] = max(17, min(_log(rng, 17, 60000), int(5e8 / token / case["batch"])))
        case["lo"] = max(1, case["hi"] // rng.choice([1, 3, 8]))
        case["keep"] = rng.choice([0.1, 0.25, 0.5, 0.75, 0.97])
        case["sinks"] = rng.choice([0, 0, 1, 4, 16])          # 0: tokens chosen one by one, else a window behind these
    else:
        case["group"] = rng.choice([1, 1, 2, 4, 4, 7, 8])
        case["io"] = rng.choice(["bf16", "bf16", "f32"])
        case["batch"] = _log(rng, 1, 64)
        case["hi"] = max(17, min(_log(rng, 17, 40000), int(4e8 / token / case["batch"])))
        case["lo"] = max(1, case["hi"] // rng.choice([1, 2, 8]))
        case["rows_hi"] = _log(rng, 1, 2000)
        case["rows_lo"] = max(1, case["rows_hi"] // rng.choice([1, 3, 10]))
        most = (1e9 if dtype != "f32" and case["io"] == "bf16" else 2e8) * 128 / max(128, d)   # (query head, row, key)s
        while case["batch"] * kv * case["group"] * case["rows_hi"] * case["hi"] > most:
            if case["rows_hi"] > 8:
                case["rows_hi"] //= 2
                case["rows_lo"] = max(1, case["rows_lo"] // 2)
            else:
                case["batch"] = max(1, case["batch"] // 2)
                case["hi"] = max(17, case["hi"] // 2)
                case["lo"] = max(1, case["lo"] // 2)
    return case


# ---- sizes, from the case alone ---------------------------------------------

def _sizes(case):
    """(cached tokens, rows) of the case's sequences; an append's rows are its new tokens."""
    r = np.random.default_rng(case["shape"])
    if case["kind"] == "append":
        new = np.full(case["batch"], case["tokens"] // case["batch"])
        new[:case["tokens"] % case["batch"]] += 1
        return new + r.integers(case["past"] // 2, case["past"] + 1, size=case["batch"]), new
    n = r.integers(case["lo"], case["hi"] + 1, size=case["batch"])
    if case["kind"] == "cross":
        return n, r.integers(case["rows_lo"], case["rows_hi"] + 1, size=case["batch"])
    return np.array([max(1, int(x * case["keep"])) for x in n]), n


def _from(case):
    """The positions that each sequence's cached tokens were appended at, ascending."""
    r = np.random.default_rng(case["shape"] + 1)
    kept = []
    for m, n in zip(*(x.tolist() for x in _sizes(case))):
        s = min(case["sinks"], m)
        kept.append(np.concatenate([np.arange(s), np.arange(n - (m - s), n)]) if s else np.sort(r.permutation(n)[:m]))
    return kept


def work(case):
    kv, d, eb = case["kv"], case["d"], BYTES[case["dtype"]]
    head = d * eb + (4 * d // GROUP if eb == 1 else 0)               # one head's key, or value, of a cached token
    lens, rows = _sizes(case)
    if case["kind"] == "append":
        n, io = case["tokens"], BYTES[case["io"]]
        dense = int(lens.sum()) * 2 * kv * (head + 2 * d) if eb == 1 else 0
        return {"bytes": n * ((2 * case["q"] + 2 * kv) * d * io + 2 * kv * head + 12) + dense,
                "flops": 3 * n * (case["q"] + kv) * case["rot"]}
    if case["kind"] == "rotate":
        moved = sum(int((k != np.arange(len(k))).sum()) for k in _from(case))
        if eb == 1:                                                  # the scale groups that hold rotated elements
            turned = -(-case["rot"] // GROUP) * (GROUP + 4)
        else:
            turned = case["rot"] * eb
        dense = int(lens.sum()) * kv * (head + 2 * d) * 2 if eb == 1 else 0
        return {"bytes": moved * kv * 2 * turned + 4 * int(lens.sum()) + dense, "flops": 3 * moved * kv * case["rot"]}
    heads = kv * case["group"]
    return {"bytes": int(lens.sum()) * 2 * kv * head + 2 * int(rows.sum()) * heads * d * BYTES[case["io"]],
            "flops": 4 * d * heads * sum(int(n) * int(c) for n, c in zip(lens, rows))}


# ---- inputs -----------------------------------------------------------------

def _fp8_value(y):
    """The values of the pools' E4M3 codes of y: halves round away from zero, a full mantissa
    does not carry, no subnormal codes, 256 and more are 448."""
    a = y.view(torch.int32) & 0x7FFFFFFF
    e = (a >> 23) - 127
    m = torch.clamp(((a & 0x7FFFFF) + (1 << 19)) >> 20, max=7)
    v = ((e.clamp(-6, 8) + 127 << 23) + (m << 20)).view(torch.float32)
    v = torch.where(e >= 8, torch.full_like(v, 448.0), v)
    return torch.where(e < -6, torch.zeros_like(v), torch.copysign(v, y))


def _codes(x, dtype):
    """f32 rows [..., d] as 1-byte pages hold them: (codes' values, scales), a scale per GROUP elements."""
    g = x.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1, keepdim=True)
    if dtype == "int8":
        s = torch.where(top == 0, torch.ones_like(top), top / torch.full_like(top, 127.0))
        y = g * (1.0 / s)
        a = y.abs()
        v = torch.copysign(torch.where(a >= 0.5, torch.floor(a + 0.5), torch.zeros_like(a)).clamp_(max=127), y)
    else:
        s = torch.where(top < 1e-8, torch.ones_like(top), top / torch.full_like(top, 448.0))
        v = _fp8_value(g / s)
    return v.flatten(-2), s.squeeze(-1)


def _stored(x, dtype):
    """f32 rows [..., d] as a pool stores them: (elements, scales or None)."""
    if dtype in TORCH:
        return x.to(TORCH[dtype]), None
    v, s = _codes(x, dtype)
    return (v.to(torch.int8) if dtype == "int8" else v.to(torch.float8_e4m3fn).view(torch.uint8)), s


class _Span:
    """Device memory of a pool as an array (it keeps the pool alive)."""

    def __init__(self, pool, ptr, shape, typestr):
        self.pool = pool
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 3}


def _on_pool(pool, index, like):
    """The pool's array `index` (K or V pages, K or V scales) as a tensor over its memory."""
    typ = {4: "<i4", 2: "<i2", 1: "|i1"}[like.element_size()]
    t = torch.as_tensor(_Span(pool, pool.device_ptrs[index], tuple(like.shape), typ), device="cuda")
    return t.view(like.dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kv, d, bs, dt, kind = case["kv"], case["d"], case["bs"], case["dtype"], case["kind"]
    lens, rows = _sizes(case)
    blocks = -(-lens // bs)
    nb = int(blocks.sum() * 9 // 8 + 1)
    # the sequences' blocks lie in random order over a pool that is an eighth larger
    perm = torch.randperm(nb, generator=gen, device="cuda").to(torch.int32).cpu().numpy()
    tables = np.full((len(lens), int(blocks.max())), -1, np.int32)
    at = 0
    for i, b in enumerate(blocks):
        tables[i, :b] = perm[at:at + b]
        at += b

    def up(x, t):
        return torch.from_numpy(np.ascontiguousarray(x.astype(t))).cuda()

    st = {"kind": kind, "dtype": dt, "bs": bs, "d": d, "kv": kv, "tables": up(tables, np.int32), "lens": up(lens, np.int32)}
    pages = [_stored(torch.randn(nb, kv, bs, d, generator=gen, device="cuda"), dt) for _ in range(2)]
    st["pages"] = [pages[0][0], pages[1][0], pages[0][1], pages[1][1]]          # K, V, K scales, V scales
    if kind != "cross":
        st["pairs"] = case["layout"] == "pairs"
        st["inv_freq"] = up(BASE ** (-np.arange(0, case["rot"], 2) / case["rot"]), np.float32)
    if kind == "append":
        n, heads = case["tokens"], case["q"] + 2 * kv
        positions = np.concatenate([np.arange(m - c, m) for m, c in zip(lens, rows)])
        seq = np.repeat(np.arange(len(lens)), rows)
        st["positions"] = up(positions, np.int32)
        st["slots"] = up(tables[seq, positions // bs].astype(np.int64) * bs + positions % bs, np.int64)
        x = torch.randn(n, heads, d, generator=gen, device="cuda").to(TORCH[case["io"]])
        parts = x.split([case["q"], kv, kv], dim=1)
        st["q"], st["k"], st["v"] = parts if case["fused"] else [t.contiguous() for t in parts]
        st["magnitude"] = case["magnitude"]
        st["q_out"] = torch.empty(n, case["q"], d, dtype=x.dtype, device="cuda")
    elif kind == "rotate":
        st["from"] = up(np.concatenate(_from(case)), np.int32)
        st["cu"] = up(np.concatenate([[0], np.cumsum(lens)]), np.int32)
    else:
        st["group"], st["rows"] = case["group"], up(rows, np.int64)
        st["cu"] = up(np.concatenate([[0], np.cumsum(rows)]), np.int32)
        st["most"] = int(rows.max())
        st["q"] = torch.randn(int(rows.sum()), kv * case["group"], d, generator=gen, device="cuda").to(TORCH[case["io"]])
        st["out"] = torch.empty_like(st["q"])
    if kind != "cross" and BYTES[dt] == 1:
        st["offsets"] = up(np.concatenate([[0], np.cumsum(lens)])[:-1] * kv * d, np.int64)
        st["dense"] = [torch.empty(int(lens.sum()), kv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        st["seq"] = up(np.repeat(np.arange(len(lens)), lens), np.int64)
        st["at"] = up(np.concatenate([np.arange(m) for m in lens]), np.int64)
    if own:
        sys.path[:0] = [p for p in [os.path.abspath("air.rs_amd")] if p not in sys.path]
        import airkv
        kinds = {"f32": airkv.F32, "bf16": airkv.BF16, "int8": airkv.INT8, "fp8": airkv.FP8}
        pool = st["pool"] = airkv.KvPool(nb, bs, kv, d, kinds[dt], GROUP)
        st["token_major"] = airkv.LAYOUT_TOKEN_MAJOR
        for i, x in enumerate(st["pages"]):
            if x is not None:
                st["pages"][i] = _on_pool(pool, i, x).copy_(x)
        if kind == "cross":
            st["ws"] = pool.new_cross_workspace(kv * case["group"], len(lens), st["most"])
    return st


# ---- one pass ---------------------------------------------------------------

def _rows(pages, scales, dtype, blocks, wide=torch.float32):
    """Cached values of blocks [...], as [..., kv, bs, d]."""
    x = pages[blocks]
    x = x.view(torch.float8_e4m3fn).to(wide) if dtype == "fp8" else x.to(wide)
    if scales is not None:
        x = (x.unflatten(-1, (-1, GROUP)) * scales[blocks].to(wide).unsqueeze(-1)).flatten(-2)
    return x


def _turned(x, positions, inv_freq, pairs, magnitude):
    """f32 rows [n, heads, d], the first 2 * len(inv_freq) elements of each rotated by its position."""
    angle = positions.double()[:, None, None] * inv_freq.double()
    c, s = (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
    rot = 2 * inv_freq.shape[0]
    if pairs:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _dense(st):
    """The sequences' cached rows, one after the other, as a layer in full precision reads them."""
    blocks, off = st["tables"].long()[st["seq"], st["at"] // st["bs"]], st["at"] % st["bs"]
    for i in range(2):
        x = st["pages"][i][blocks, :, off]
        x = x.view(torch.float8_e4m3fn).float() if st["dtype"] == "fp8" else x.float()
        x = x.unflatten(-1, (-1, GROUP)) * st["pages"][2 + i][blocks, :, off].unsqueeze(-1)
        st["dense"][i].copy_(x.flatten(-2))
    return {"k": st["dense"][0], "v": st["dense"][1]}


def _cached(st):
    return {"k": st["pages"][0], "v": st["pages"][1]}


def _put(st, i, blocks, off, x):
    """f32 rows [n, kv, d] into the K (i = 0) or V (i = 1) pages."""
    e, s = _stored(x, st["dtype"])
    st["pages"][i][blocks, :, off] = e
    if s is not None:
        st["pages"][2 + i][blocks, :, off] = s


def _plain_append(st):
    how = st["positions"], st["inv_freq"], st["pairs"], st["magnitude"]
    st["q_out"].copy_(_turned(st["q"].float(), *how))
    blocks, off = st["slots"] // st["bs"], st["slots"] % st["bs"]
    _put(st, 0, blocks, off, _turned(st["k"].float(), *how))
    _put(st, 1, blocks, off, st["v"].float())


def _plain_rotate(st):
    cu = st["cu"].long()
    n = st["from"].shape[0]
    seq = torch.bucketize(torch.arange(n, device="cuda"), cu[1:], right=True)
    at = torch.arange(n, device="cuda") - cu[seq]
    by = at - st["from"]
    moved = by != 0
    blocks, off = st["tables"].long()[seq, at // st["bs"]], at % st["bs"]
    x = st["pages"][0][blocks, :, off]
    if BYTES[st["dtype"]] == 1:
        # groups without a rotated element keep their codes and scales; so do tokens that stay
        held, s = x, st["pages"][2][blocks, :, off]
        x = x.view(torch.float8_e4m3fn).float() if st["dtype"] == "fp8" else x.float()
        x = (x.unflatten(-1, (-1, GROUP)) * s.unsqueeze(-1)).flatten(-2)
        e, t = _stored(_turned(x, by, st["inv_freq"], st["pairs"], 1.0), st["dtype"])
        groups = -(-2 * st["inv_freq"].shape[0] // GROUP)
        new = moved[:, None, None] & (torch.arange(s.shape[-1], device="cuda") < groups)
        st["pages"][0][blocks, :, off] = torch.where(new.repeat_interleave(GROUP, -1), e, held)
        st["pages"][2][blocks, :, off] = torch.where(new, t, s)
    else:
        e = _turned(x.float(), by, st["inv_freq"], st["pairs"], 1.0).to(x.dtype)
        st["pages"][0][blocks, :, off] = torch.where(moved[:, None, None], e, x)


def _plain_cross(st):
    """Every sequence padded to the longest: scores, softmax, values."""
    tables, lens, d, kv, g = st["tables"].long().clamp(min=0), st["lens"].long(), st["d"], st["kv"], st["group"]
    batch = tables.shape[0]
    kp, vp, ks, vs = st["pages"]
    k = _rows(kp, ks, st["dtype"], tables).permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, d)
    v = _rows(vp, vs, st["dtype"], tables).permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, d)
    hidden = torch.arange(k.shape[2], device="cuda") >= lens[:, None]
    v = v.masked_fill_(hidden[:, None, :, None], 0.0)
    r = torch.arange(st["most"], device="cuda")
    real = r < st["rows"][:, None]                                             # [batch][rows]
    at = (st["cu"][:-1].long()[:, None] + r).clamp(max=st["q"].shape[0] - 1)
    q = st["q"].float()[at].reshape(batch, -1, kv, g, d).permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, d)
    s = torch.matmul(q * (1 / math.sqrt(d)), k.transpose(2, 3))
    s.masked_fill_(hidden[:, None, None, :], -math.inf)
    s = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    x = torch.matmul(s, v) / s.sum(-1, keepdim=True)
    x = x.reshape(batch, kv, -1, g, d).permute(0, 2, 1, 3, 4).reshape(batch, -1, kv * g, d)
    st["out"][at[real]] = x[real].to(st["out"].dtype)


def run(st):
    pool = st.get("pool")
    if st["kind"] == "cross":
        if own:
            pool.paged_cross(st["q"], st["cu"], st["tables"], st["lens"], st["out"], max_q_len=st["most"], workspace=st["ws"])
        else:
            _plain_cross(st)
        return {"out": st["out"]}
    if st["kind"] == "append":
        if own:
            pool.append_rotary(st["q"], st["k"], st["v"], st["slots"], st["positions"], st["inv_freq"], q_out=st["q_out"],
                               interleaved=st["pairs"], magnitude=st["magnitude"])
        else:
            _plain_append(st)
        out = {"q": st["q_out"]}
    else:
        if own:
            pool.rotate(st["tables"], st["from"], st["cu"], st["inv_freq"], interleaved=st["pairs"])
        else:
            _plain_rotate(st)
        out = {}
    if "dense" not in st:
        return {**out, **_cached(st)}
    if own:
        pool.gather(st["tables"], st["lens"], st["offsets"], *st["dense"], layout=st["token_major"], validate=False)
        return {**out, "k": st["dense"][0], "v": st["dense"][1]}
    return {**out, **_dense(st)}


# ---- the same in 64 bits ------------------------------------------------------

def _exact_turn(x, positions, inv_freq, pairs, magnitude):
    """Rows [n, heads, d] as complex numbers times magnitude * exp(i angle)."""
    x = x.double().clone()
    rot = 2 * inv_freq.shape[0]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    angle = positions.double()[:, None, None] * inv_freq.double()
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(angle, magnitude), angle)
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_stored(x, dtype):
    """64-bit rows as the values that a pool's elements stand for (not rounded where those are floats)."""
    if dtype in TORCH:
        return x
    v, s = _codes(x.float(), dtype)
    return (v.double().unflatten(-1, (-1, GROUP)) * s.double().unsqueeze(-1)).flatten(-2)


def _exact_values(case, st, i):
    """All K (i = 0) or V (i = 1) pages in 64 bits."""
    return _rows(st["pages"][i], st["pages"][2 + i], case["dtype"], torch.arange(st["pages"][i].shape[0], device="cuda"),
                 torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    lens, rows = _sizes(case)
    bs, d = case["bs"], case["d"]
    tables = st["tables"].cpu().numpy()
    if case["kind"] == "cross":
        if float(lens.max()) * float(rows.sum()) * case["kv"] * case["group"] * d > 5e12:
            return None
        out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        first = 0
        for i, (n, c) in enumerate(zip(lens.tolist(), rows.tolist())):
            blocks = torch.from_numpy(tables[i, :-(-n // bs)]).long().cuda()
            k, v = (_rows(st["pages"][j], st["pages"][2 + j], case["dtype"], blocks, torch.float64).transpose(0, 1)
                    .reshape(case["kv"], -1, d)[:, :n] for j in range(2))
            for h in range(case["kv"] * case["group"]):
                s = torch.mm(st["q"][first:first + c, h].double(), k[h // case["group"]].t().contiguous()) / math.sqrt(d)
                out[first:first + c, h] = torch.mm(torch.softmax(s, -1), v[h // case["group"]])
            first += c
        return {"out": out}
    k, v = _exact_values(case, st, 0), _exact_values(case, st, 1)
    out = {}
    if case["kind"] == "append":
        how = st["positions"], st["inv_freq"], st["pairs"], case["magnitude"]
        out["q"] = _exact_turn(st["q"], *how)
        blocks, off = st["slots"] // bs, st["slots"] % bs
        k[blocks, :, off] = _exact_stored(_exact_turn(st["k"], *how), case["dtype"])
        v[blocks, :, off] = _exact_stored(st["v"].double(), case["dtype"])
    else:
        for i, was in enumerate(_from(case)):
            at = np.arange(len(was))[was != np.arange(len(was))]
            if not len(at):
                continue
            blocks, off = torch.from_numpy(tables[i, at // bs]).long().cuda(), torch.from_numpy(at % bs).cuda()
            x, by = k[blocks, :, off], torch.from_numpy(at - was[at]).cuda()
            y = _exact_stored(_exact_turn(x, by, st["inv_freq"], st["pairs"], 1.0), case["dtype"])
            if BYTES[case["dtype"]] == 1:
                whole = -(-case["rot"] // GROUP) * GROUP                 # (groups behind keep their values)
                y = torch.cat([y[..., :whole], x[..., whole:]], -1)
            k[blocks, :, off] = y
    if "dense" not in st:
        return {**out, "k": k, "v": v}
    blocks, off = torch.from_numpy(tables).long().cuda()[st["seq"], st["at"] // bs], st["at"] % bs
    return {**out, "k": k[blocks, :, off], "v": v[blocks, :, off]}
