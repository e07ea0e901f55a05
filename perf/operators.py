"""Differential attention over the paged K/V cache and the compaction of cached
sequences, as measurable cases.

Differential attention: K/V heads come in pairs (2p, 2p + 1).  A query pair h
scores both key heads of its K/V pair and attends to the pair's two value
heads side by side (2 * head_dim columns) with the difference of its two
softmax maps, P_0 - lambda * P_1; the result may be normalised over its
columns (root mean square) and scaled.  Decode takes one token per sequence,
prefill the newest tokens of each sequence, causally.

Compaction: each sequence keeps some of its cached tokens, in order, and they
move to its first positions inside its own pages.

Page contents are normal rows as the pool's append stores them (rounded, or
quantized with a scale per 32 elements).
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
EPS, OUT_SCALE = 1e-5, 0.2


def _decode(name, dtype, batch, lo, hi, kv, group, d, bs, io="bf16", norm=True, lam="head", shape=0):
    return {"name": name, "kind": "decode", "dtype": dtype, "batch": batch, "lo": lo, "hi": hi, "kv": kv,
            "group": group, "d": d, "bs": bs, "io": io, "norm": norm, "lam": lam, "shape": shape}


def _prefill(name, dtype, batch, chunk_lo, chunk_hi, prefix_lo, prefix_hi, kv, group, d, bs, io="bf16",
             norm=True, lam="head", shape=0):
    return {"name": name, "kind": "prefill", "dtype": dtype, "batch": batch, "chunk_lo": chunk_lo,
            "chunk_hi": chunk_hi, "prefix_lo": prefix_lo, "prefix_hi": prefix_hi, "kv": kv, "group": group,
            "d": d, "bs": bs, "io": io, "norm": norm, "lam": lam, "shape": shape}


def _compact(name, dtype, batch, lo, hi, kv, d, bs, keep, sinks, shape=0):
    return {"name": name, "kind": "compact", "dtype": dtype, "batch": batch, "lo": lo, "hi": hi, "kv": kv, "d": d,
            "bs": bs, "keep": keep, "sinks": sinks, "shape": shape}


def listed():
    return [
        # the smallest call: four short chats of a small model (8 heads of 64)
        # on the f32 cache, where latency and launches count
        _decode("decode_f32_small", "f32", 4, 37, 527, 8, 1, 64, 16, io="f32", shape=1),
        # one chat of an 8B-sized model: a single sequence, a ragged context
        _decode("decode_bf16_single", "bf16", 1, 1337, 1337, 8, 4, 128, 16, lam="token", shape=2),
        # the serving batch: 64 sequences of 512 to 4096 tokens
        _decode("decode_bf16_batch", "bf16", 64, 512, 4096, 8, 4, 128, 16, shape=3),
        # a larger model's layer (64 query heads) on the int8 cache
        _decode("decode_int8_70b", "int8", 32, 8192, 8192, 8, 8, 128, 16, shape=4),
        # long contexts on the fp8 cache, eight sequences of 32K to 128K
        _decode("decode_fp8_long", "fp8", 8, 32768, 131072, 8, 8, 128, 32, shape=5),
        # first prompts of the small model on the f32 cache (no prefix)
        _prefill("prefill_f32_prompts", "f32", 4, 37, 511, 0, 0, 8, 1, 64, 16, io="f32", norm=False, shape=6),
        # the prompt chunks of a continuous-batching step: eight chunks of 512
        # at most over ragged prefixes
        _prefill("prefill_bf16_chunks", "bf16", 8, 200, 512, 0, 6000, 8, 4, 128, 32, shape=7),
        # one long prompt, the largest product
        _prefill("prefill_bf16_long", "bf16", 1, 8192, 8192, 0, 0, 8, 4, 128, 16, shape=8),
        # ragged chunks of a larger model's layer over int8 pages
        _prefill("prefill_int8_70b", "int8", 6, 33, 512, 100, 6000, 8, 8, 128, 16, lam="token", shape=9),
        # one sequence shrunk to its first four and its newest tokens
        _compact("compact_f32_window", "f32", 1, 511, 511, 8, 64, 16, 0.5, 4, shape=10),
        # a batch that keeps half of its tokens, those an eviction policy chose
        _compact("compact_bf16_batch", "bf16", 64, 512, 4096, 8, 128, 16, 0.5, 0, shape=11),
        # a few long sequences on a wide window
        _compact("compact_bf16_long", "bf16", 4, 32768, 65536, 8, 128, 32, 0.75, 16, shape=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode"] * 2 + ["prefill"] * 2 + ["compact"])
    dtype = rng.choice(["f32", "bf16", "bf16", "int8", "fp8"]) if kind != "compact" else rng.choice(["f32", "bf16"])
    d = rng.choice([32, 64, 64, 96, 128, 128, 128])
    kv = rng.choice([2, 4, 6, 8, 8, 16])
    bs = rng.choice([16, 32])
    case = {"kind": kind, "dtype": dtype, "kv": kv, "d": d, "bs": bs, "shape": rng.randrange(1 << 30)}
    token = 2 * kv * d * BYTES[dtype]                 # cached bytes of one token
    if kind != "compact":
        case["group"] = rng.choice([1, 2, 3, 4, 4, 7, 8, 12])
        case["io"] = rng.choice(["bf16", "bf16", "f32"])
        case["norm"] = rng.choice([True, True, False])
        case["lam"] = rng.choice(["head", "token"])
    if kind == "decode":
        case["batch"] = _log(rng, 1, 160)
        case["hi"] = max(17, min(_log(rng, 17, 60000), int(6e8 / token / case["batch"])))
        case["lo"] = max(1, case["hi"] // rng.choice([1, 2, 8, 50]))
    elif kind == "prefill":
        case["batch"] = rng.randint(1, 8)
        case["chunk_hi"] = _log(rng, 1, 2000)
        case["chunk_lo"] = max(1, case["chunk_hi"] // rng.choice([1, 3, 10]))
        case["prefix_hi"] = rng.choice([0, _log(rng, 16, 8000)])
        case["prefix_lo"] = case["prefix_hi"] // 4
        rows = case["batch"] * (kv // 2) * case["group"] * case["chunk_hi"]
        most = 1.2e9 if dtype != "f32" and case["io"] == "bf16" else 3e8      # (query pair, key) products
        while rows * (case["prefix_hi"] + case["chunk_hi"] / 2) > most:
            case["prefix_hi"] //= 2
            case["prefix_lo"] //= 2
            if not case["prefix_hi"]:
                case["chunk_hi"] = max(1, case["chunk_hi"] // 2)
                case["chunk_lo"] = min(case["chunk_lo"], case["chunk_hi"])
                rows = case["batch"] * (kv // 2) * case["group"] * case["chunk_hi"]
    else:
        case["batch"] = _log(rng, 1, 100)
        case["hi"] = max(17, min(_log(rng, 17, 60000), int(6e8 / token / case["batch"])))
        case["lo"] = max(1, case["hi"] // rng.choice([1, 3, 8]))
        case["keep"] = rng.choice([0.1, 0.25, 0.5, 0.75, 0.97])
        case["sinks"] = rng.choice([0, 0, 1, 4, 16])          # 0: tokens chosen one by one, else a window behind these
    return case


# ---- sizes, from the case alone ---------------------------------------------

def _sizes(case):
    """(lengths, query lengths) of the case's sequences."""
    r = np.random.default_rng(case["shape"])
    if case["kind"] == "prefill":
        c = r.integers(case["chunk_lo"], case["chunk_hi"] + 1, size=case["batch"])
        return c + r.integers(case["prefix_lo"], case["prefix_hi"] + 1, size=case["batch"]), c
    n = r.integers(case["lo"], case["hi"] + 1, size=case["batch"])
    return n, np.ones_like(n)


def _kept(case):
    """The positions each sequence keeps, ascending."""
    r = np.random.default_rng(case["shape"] + 1)
    kept = []
    for n in _sizes(case)[0].tolist():
        m = max(1, int(n * case["keep"]))
        if case["sinks"]:
            s = min(case["sinks"], m)
            kept.append(np.concatenate([np.arange(s), np.arange(n - (m - s), n)]))
        else:
            kept.append(np.sort(r.permutation(n)[:m]))
    return kept


def work(case):
    kv, d, eb = case["kv"], case["d"], BYTES[case["dtype"]]
    row = 2 * kv * (d * eb + (4 * d // GROUP if eb == 1 else 0))     # K and V of one cached token
    if case["kind"] == "compact":
        kept = _kept(case)
        moved = sum(int((k != np.arange(len(k))).sum()) for k in kept)
        return {"bytes": moved * 2 * row + 4 * sum(len(k) for k in kept), "flops": 0}
    lens, qlens = _sizes(case)
    pairs = kv // 2 * case["group"]
    rows = int(qlens.sum())
    lam = 4 * pairs * (rows if case["lam"] == "token" else 1)
    keys = sum(int(c) * int(n - c) + int(c) * (int(c) + 1) // 2 for n, c in zip(lens, qlens))
    # a (query pair, key): two scores of d, and the difference's product with 2 d values
    return {"bytes": int(lens.sum() * row) + 2 * rows * pairs * 2 * d * BYTES[case["io"]] + lam,
            "flops": 8 * d * pairs * keys}


# ---- inputs -----------------------------------------------------------------

def _stored(x, dtype):
    """f32 rows [..., d] as a pool stores them: (elements, scales or None)."""
    if dtype == "f32":
        return x, None
    if dtype == "bf16":
        return x.to(torch.bfloat16), None
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    top = g.abs().amax(-1, keepdim=True).clamp_(min=1e-6)
    s = top / (127 if dtype == "int8" else 448)
    if dtype == "int8":
        c = (g / s).round_().clamp_(-127, 127).to(torch.int8)
    else:
        y = g / s
        y = torch.where(y.abs() < 2.0 ** -6, torch.zeros_like(y), y)         # the format has no subnormal codes
        c = y.to(torch.float8_e4m3fn).view(torch.uint8)
    return c.reshape(x.shape), s.squeeze(-1)


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
    kv, d, bs, dt = case["kv"], case["d"], case["bs"], case["dtype"]
    lens, qlens = _sizes(case)
    blocks = -(-lens // bs)
    nb = int(blocks.sum() * 9 // 8 + 1)
    # the sequences' blocks lie in random order over a pool that is an eighth larger
    perm = torch.randperm(nb, generator=gen, device="cuda").to(torch.int32).cpu().numpy()
    tables = np.full((len(lens), int(blocks.max())), -1, np.int32)
    at = 0
    for i, b in enumerate(blocks):
        tables[i, :b] = perm[at:at + b]
        at += b
    st = {"kind": case["kind"], "dtype": dt, "bs": bs, "d": d, "kv": kv, "tables": torch.from_numpy(tables).cuda(),
          "lens": torch.from_numpy(lens.astype(np.int32)).cuda(), "max_len": int(lens.max())}
    pages = [_stored(torch.randn(nb, kv, bs, d, generator=gen, device="cuda"), dt) for _ in range(2)]
    st["pages"] = [pages[0][0], pages[1][0], pages[0][1], pages[1][1]]          # K, V, K scales, V scales
    if case["kind"] == "compact":
        kept = _kept(case)
        cu = np.concatenate([[0], np.cumsum([len(k) for k in kept])]).astype(np.int32)
        st["keep"] = torch.from_numpy(np.concatenate(kept).astype(np.int32)).cuda()
        st["cu"] = torch.from_numpy(cu).cuda()
    else:
        pairs, rows = kv // 2 * case["group"], int(qlens.sum())
        st["q"] = torch.randn(rows, 2 * pairs, d, generator=gen, device="cuda").to(TORCH[case["io"]])
        st["lam"] = 0.2 + 0.6 * torch.rand((rows, pairs) if case["lam"] == "token" else (pairs,), generator=gen,
                                           device="cuda")
        st["norm_weight"] = 1 + 0.1 * torch.randn(2 * d, generator=gen, device="cuda") if case["norm"] else None
        st["norm_eps"] = EPS if case["norm"] else None
        st["out"] = torch.empty(rows, pairs, 2 * d, dtype=TORCH[case["io"]], device="cuda")
        cu = np.concatenate([[0], np.cumsum(qlens)]).astype(np.int32)
        st.update(cu=torch.from_numpy(cu).cuda(), qlens=torch.from_numpy(qlens).cuda(), chunk=int(qlens.max()))
    if own:
        sys.path[:0] = [p for p in [os.path.abspath("air.rs_amd")] if p not in sys.path]
        import airkv
        kinds = {"f32": airkv.F32, "bf16": airkv.BF16, "int8": airkv.INT8, "fp8": airkv.FP8}
        pool = st["pool"] = airkv.KvPool(nb, bs, kv, d, kinds[dt], GROUP)
        for i, x in enumerate(st["pages"]):
            if x is not None:
                st["pages"][i] = _on_pool(pool, i, x).copy_(x)
        if case["kind"] == "decode":
            st["ws"] = pool.new_diff_workspace(2 * pairs, len(lens), tables.shape[1])
        elif case["kind"] == "prefill":
            st["ws"] = pool.new_diff_prefill_workspace(2 * pairs, len(lens), st["chunk"])
    return st


# ---- one pass ---------------------------------------------------------------

def _rows(pages, scales, dtype, blocks, wide=torch.float32):
    """Cached values of blocks [...], as [..., kv, bs, d]."""
    x = pages[blocks]
    x = x.view(torch.float8_e4m3fn).to(wide) if dtype == "fp8" else x.to(wide)
    if scales is not None:
        x = (x.unflatten(-1, (-1, GROUP)) * scales[blocks].to(wide).unsqueeze(-1)).flatten(-2)
    return x


def _plain_attention(st):
    """Every sequence padded to the longest: scores, two softmax maps, their difference, values, norm."""
    tables, lens, d, kv = st["tables"].long(), st["lens"].long(), st["d"], st["kv"]
    batch, width = tables.shape
    kp, vp, ks, vs = st["pages"]
    blocks = tables.clamp(min=0)
    k = _rows(kp, ks, st["dtype"], blocks).permute(0, 2, 1, 3, 4).reshape(batch, kv // 2, 2, -1, d)
    v = _rows(vp, vs, st["dtype"], blocks).permute(0, 2, 1, 3, 4).reshape(batch, kv // 2, 2, -1, d)
    keys = k.shape[3]
    n = st["qlens"]
    r = torch.arange(st["chunk"], device="cuda")
    real = r < n[:, None]                                                      # [batch][chunk]
    at = (st["cu"][:-1].long()[:, None] + r).clamp(max=st["q"].shape[0] - 1)
    pairs = st["q"].shape[1] // 2
    g = pairs // (kv // 2)
    q = st["q"].float()[at].reshape(batch, -1, kv // 2, g, 2, d).permute(0, 2, 4, 1, 3, 5)
    q = q.reshape(batch, kv // 2, 2, -1, d) * (1 / math.sqrt(d))               # [batch][K/V pair][map][chunk * g][d]
    s = torch.matmul(q, k.transpose(3, 4)).reshape(batch, kv // 2, 2, -1, g, keys)
    last = lens[:, None] - n[:, None] + r                                      # the newest key a row sees
    seen = torch.arange(keys, device="cuda") <= last[:, :, None]
    s.masked_fill_(~seen[:, None, None, :, None], -math.inf)
    s = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    lam = st["lam"]
    lam = lam[at] if lam.dim() == 2 else lam.expand(batch, len(r), pairs)
    lam = lam.reshape(batch, -1, kv // 2, g).permute(0, 2, 1, 3).unsqueeze(-1)
    total = s.sum(-1, keepdim=True)
    p = s[:, :, 0].div_(total[:, :, 0]).sub_(s[:, :, 1].mul_(lam / total[:, :, 1]))
    v = v.permute(0, 1, 3, 2, 4).reshape(batch, kv // 2, keys, 2 * d)
    x = torch.matmul(p.reshape(batch, kv // 2, -1, keys), v)
    if st["norm_eps"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + st["norm_eps"]) * st["norm_weight"]
    x = (x * OUT_SCALE).reshape(batch, kv // 2, -1, g, 2 * d).permute(0, 2, 1, 3, 4).reshape(batch, -1, pairs, 2 * d)
    st["out"][at[real]] = x[real].to(st["out"].dtype)
    return st["out"]


def _plain_compact(st):
    keep, cu, bs = st["keep"].long(), st["cu"].long(), st["bs"]
    seq = torch.bucketize(torch.arange(keep.shape[0], device="cuda"), cu[1:], right=True)
    to = torch.arange(keep.shape[0], device="cuda") - cu[seq]
    tables = st["tables"].long()
    src, dst = tables[seq, keep // bs], tables[seq, to // bs]
    for x in st["pages"]:
        if x is not None:
            x[dst, :, to % bs] = x[src, :, keep % bs]
    return {"k": st["pages"][0], "v": st["pages"][1]}


def run(st):
    if not own:
        return _plain_compact(st) if st["kind"] == "compact" else {"out": _plain_attention(st)}
    pool = st["pool"]
    if st["kind"] == "compact":
        pool.compact(st["tables"], st["lens"], st["keep"], st["cu"])
        return {"k": st["pages"][0], "v": st["pages"][1]}
    more = {"norm_weight": st["norm_weight"], "norm_eps": st["norm_eps"], "out_scale": OUT_SCALE, "workspace": st["ws"]}
    if st["kind"] == "decode":
        pool.paged_diff_decode(st["q"], st["lam"], st["tables"], st["lens"], st["out"], **more)
    else:
        pool.paged_diff_prefill(st["q"], st["lam"], st["cu"], st["tables"], st["lens"], st["out"],
                                max_q_len=st["chunk"], **more)
    return {"out": st["out"]}


# ---- the same in 64 bits, sequence by sequence --------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    kp, vp, ks, vs = st["pages"]
    if case["kind"] == "compact":
        # moved values are the values that were there
        out = {"k": kp.double(), "v": vp.double()}
        for i, keep in enumerate(_kept(case)):
            keep, to = torch.from_numpy(keep).cuda(), torch.arange(len(keep), device="cuda")
            row = st["tables"][i].long()
            for name, x in (("k", kp), ("v", vp)):
                out[name][row[to // case["bs"]], :, to % case["bs"]] = x[row[keep // case["bs"]], :, keep % case["bs"]].double()
        return out
    lens, qlens = _sizes(case)
    d, g, bs = case["d"], case["group"], case["bs"]
    scale = 1.0 / math.sqrt(d)
    out = torch.empty(st["out"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, c) in enumerate(zip(lens.tolist(), qlens.tolist())):
        blocks = st["tables"][i, :-(-n // bs)].long()
        k = _rows(kp, ks, case["dtype"], blocks, torch.float64).transpose(0, 1).reshape(case["kv"], -1, d)[:, :n]
        v = _rows(vp, vs, case["dtype"], blocks, torch.float64).transpose(0, 1).reshape(case["kv"], -1, d)[:, :n]
        hidden = torch.ones(c, n, dtype=torch.bool, device="cuda").triu_(n - c + 1)
        lam = st["lam"].double()
        lam = lam[first:first + c] if lam.dim() == 2 else lam.expand(c, -1)
        for h in range(st["lam"].shape[-1]):
            p = h // g
            maps = []
            for m in range(2):
                s = torch.mm(st["q"][first:first + c, 2 * h + m].double(), k[2 * p + m].t().contiguous()) * scale
                maps.append(torch.softmax(s.masked_fill_(hidden, -math.inf), -1))
            w = maps[0] - lam[:, h, None] * maps[1]
            x = torch.cat([torch.mm(w, v[2 * p]), torch.mm(w, v[2 * p + 1])], -1)
            if case["norm"]:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * st["norm_weight"].double()
            out[first:first + c, h] = OUT_SCALE * x
        first += c
    return {"out": out}
