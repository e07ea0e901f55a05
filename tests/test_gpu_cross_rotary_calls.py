"""Rotary appends, rotations and cross attention as a program calls them: every head size of every
kind of call, captured graphs, streams, launchers, large pools, and a decoder layer from its prompt
to a compacted context.  (Against twin eager calls bit for bit, and against 64 bits.)"""
import math

import numpy as np
import pytest

import airkv
import rotary_ref
from gpu_helpers import torch_mod
from test_gpu_cross import Case

pytestmark = pytest.mark.gpu


def _dev(x):
    return torch_mod().from_numpy(np.ascontiguousarray(x)).cuda()


def _bits(t):
    return t.contiguous().view(torch_mod().uint8)


def _same(x, y, what=""):
    assert torch_mod().equal(_bits(x), _bits(y)), what


def _same_pools(x, y, what=""):
    for a, b in zip(x.snapshot(), y.snapshot()):
        if a is not None:
            assert np.array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(b).view(np.uint8)), what


# ---- sizes


@pytest.mark.parametrize("rows", ["few", "many"])
@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16, airkv.INT8, airkv.FP8])
def test_every_head_dim(dtype, d, io, rows):
    group = 2 if rows == "few" else 3
    Case(dtype, d, 2, group, 16, [1, 131, 0, 700, 64], [1, 2, 1, 0, 7] if rows == "few" else [90, 2, 1, 0, 70], io, seed=d).check()


@pytest.mark.parametrize("hint", [None, 0, 1, 16, 100000])
def test_the_most_rows_are_a_hint(hint):
    """Whatever it says, every row is answered."""
    Case(airkv.BF16, 64, 2, 4, 32, [200, 90, 400], [3, 150, 60], seed=5).check(max_q_len=hint)
    Case(airkv.F32, 96, 1, 2, 16, [200, 90, 400], [1, 150, 60], "f32", seed=6).check(max_q_len=hint)


def test_sequences_that_share_blocks():
    """Beams over one encoder's states: the same blocks, and the same block twice in a table."""
    c = Case(airkv.BF16, 128, 2, 4, 16, [160, 160, 160, 48], [1, 4, 1, 1], seed=7)
    c.tables[1] = c.tables[2] = c.tables[0]
    c.tables[3, :3] = c.tables[0, 4]
    c.check(max_q_len=4)


@pytest.mark.parametrize("dtype,io,rows", [(airkv.BF16, "bf16", 1), (airkv.FP8, "bf16", 5), (airkv.F32, "f32", 1), (airkv.INT8, "bf16", 300)])
def test_the_same_call_gives_the_same_bits(dtype, io, rows):
    c = Case(dtype, 64, 4, 2, 16, [5000, 777, 31], [rows] * 3, io, seed=8)
    first = c.call(max_q_len=rows).clone()
    for _ in range(3):
        c.out.fill_(3.0)
        _same(c.call(max_q_len=rows), first)


def test_out_over_the_queries():
    """Rows are read before they are written: the output may be the queries' memory."""
    for rows, n in ((1, 3000), (200, 900)):
        c = Case(airkv.BF16, 64, 2, 4, 16, [n, 90, 33], [rows, rows, rows], seed=9)
        want = c.call(max_q_len=rows).clone()
        q = c.q.clone()
        c.pool.paged_cross(q, _dev(c.cu), _dev(c.tables), _dev(c.lens), q, max_q_len=rows, scale=c.scale)
        _same(q, want)


def _spread(n_blocks, bs, count, r):
    """Block ids of a large pool, most from its end."""
    return np.concatenate([r.choice(np.arange(n_blocks - 4 * count, n_blocks), count - 2, replace=False), [0, 7]]).astype(np.int32)[r.permutation(count)]


@pytest.mark.parametrize("dtype,bs,n_blocks", [(airkv.BF16, 16, 140_000), (airkv.INT8, 16, 270_000), (airkv.F32, 32, 40_000)])
def test_pools_beyond_4_gib(dtype, bs, n_blocks):
    """Offsets past 32 bits: what a small pool with the same rows gives, bit for bit."""
    torch = torch_mod()
    r = np.random.default_rng(31)
    lens = np.array([1, 300, 77], np.int32)
    nb = -(-lens // bs)
    count = int(nb.sum())
    ids = [_spread(n_blocks, bs, count, r), np.arange(count, dtype=np.int32)]
    pools = [airkv.KvPool(n_blocks, bs, 8, 128, dtype), airkv.KvPool(count, bs, 8, 128, dtype)]
    assert pools[0].num_blocks * pools[0].slab_bytes > 1 << 32
    total = int(lens.sum())
    x = torch.randn(total, 32 + 8 + 8, 128, device="cuda").bfloat16()
    positions = _dev(np.concatenate([np.arange(n) for n in lens]).astype(np.int32))
    f = _dev(airkv.rotary.frequencies(128)[0])
    cu = _dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    got = []
    for pool, at in zip(pools, ids):
        tables = np.full((3, int(nb.max())), -1, np.int32)
        begin = np.concatenate([[0], np.cumsum(nb)])
        for b in range(3):
            tables[b, :nb[b]] = at[begin[b]:begin[b + 1]]
        slots = np.concatenate([tables[b, np.arange(n) // bs].astype(np.int64) * bs + np.arange(n) % bs for b, n in enumerate(lens)])
        q, k, v = x.split([32, 8, 8], dim=1)
        out = [pool.append_rotary(q, k, v, _dev(slots), positions, f)]
        pool.rotate(_dev(tables), positions, cu, f, to_pos=positions + 1000)
        for rows in (1, 40):
            q = out[0][:3 * rows].contiguous()
            o = torch.empty_like(q)
            out.append(pool.paged_cross(q, _dev(np.arange(4, dtype=np.int32) * rows), _dev(tables), _dev(lens), o, max_q_len=rows))
        assert pool.error_count() == 0
        got.append(out)
    for a, b in zip(*got):
        _same(a, b)
    pools[0].close()


# ---- streams, launchers, graphs


def _layer(dtype, seed, io="bf16", bs=16):
    """What one layer's step needs: a self pool, a cross pool, and tensors that a step reads."""
    torch = torch_mod()
    torch.manual_seed(seed)
    kv, group, d, batch = 2, 4, 64, 3
    it = torch.bfloat16 if io == "bf16" else torch.float32
    lens = torch.tensor([40, 7, 90], dtype=torch.int32, device="cuda")
    own = airkv.KvPool(24, bs, kv, d, dtype)
    far = airkv.KvPool(64, bs, kv, d, dtype)
    n = 24 * bs
    own.append(torch.randn(n, kv, d, device="cuda"), torch.randn(n, kv, d, device="cuda"), torch.arange(n, device="cuda"))
    n = 64 * bs
    far.append(torch.randn(n, kv, d, device="cuda"), torch.randn(n, kv, d, device="cuda"), torch.arange(n, device="cuda"))
    tables = torch.arange(24, dtype=torch.int32, device="cuda").view(3, 8).contiguous()
    far_tables = torch.arange(63, dtype=torch.int32, device="cuda").view(3, 21).contiguous()
    st = dict(own=own, far=far, lens=lens, tables=tables, far_tables=far_tables, batch=batch, n_q=kv * group,
              far_lens=torch.tensor([300, 1, 333], dtype=torch.int32, device="cuda"),
              x=torch.randn(batch, kv * group + 2 * kv, d, device="cuda").to(it), kv=kv,
              f=_dev(rotary_ref.frequencies(d)), cu=torch.arange(batch + 1, dtype=torch.int32, device="cuda"),
              froms=torch.arange(60, dtype=torch.int32, device="cuda") + 3,
              cu_froms=torch.tensor([0, 20, 25, 60], dtype=torch.int32, device="cuda"))
    st["slots"] = (tables[torch.arange(3, device="cuda"), (lens // bs).long()].long() * bs + lens % bs).contiguous()
    st["q_out"] = torch.zeros(batch, st["n_q"], d, dtype=it, device="cuda")
    st["out"] = torch.zeros_like(st["q_out"])
    st["ws"] = far.new_cross_workspace(st["n_q"], batch, 1)
    return st


def _step(st, stream=None):
    q, k, v = st["x"].split([st["n_q"], st["kv"], st["kv"]], dim=1)
    st["own"].append_rotary(q, k, v, st["slots"], st["lens"], st["f"], q_out=st["q_out"], stream=stream)
    st["own"].rotate(st["tables"], st["froms"], st["cu_froms"], st["f"], stream=stream)
    st["far"].paged_cross(st["q_out"], st["cu"], st["far_tables"], st["far_lens"], st["out"], max_q_len=1, workspace=st["ws"], stream=stream)


@pytest.mark.parametrize("dtype,io", [(airkv.BF16, "bf16"), (airkv.INT8, "bf16"), (airkv.F32, "f32"), (airkv.FP8, "f32")])
def test_graphs(dtype, io):
    """A captured step replays as the eager one runs, with eager work and other inputs between."""
    torch = torch_mod()
    one, two = _layer(dtype, 1, io), _layer(dtype, 1, io)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(one)                                         # (warm, and the twin with it)
    torch.cuda.current_stream().wait_stream(side)
    _step(two)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(one)
    _same_pools(one["own"], two["own"], "the capture ran nothing")
    for turn in range(4):
        x = torch.randn_like(one["x"])
        for st in (one, two):
            st["x"].copy_(x)
            st["far_lens"].copy_(torch.tensor([300 - 90 * turn, turn, 16 * turn + 1], dtype=torch.int32))
            st["out"].fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        _step(two)                                         # eager, on the default stream
        (torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")).sum().item()
        _same(one["q_out"], two["q_out"], f"queries, replay {turn}")
        _same(one["out"], two["out"], f"outputs, replay {turn}")
        _same_pools(one["own"], two["own"], f"pages, replay {turn}")
    assert one["own"].error_count() == one["far"].error_count() == 0


def test_two_graphs_with_workspaces_of_their_own():
    torch = torch_mod()
    a, b, twin = _layer(airkv.BF16, 2), _layer(airkv.BF16, 3), _layer(airkv.BF16, 2)
    graphs = []
    for st in (a, b):
        _step(st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _step(st)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    _step(twin)
    torch.cuda.synchronize()
    for turn in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        _step(twin)
        _same(a["out"], twin["out"], f"replay {turn}")


def test_two_streams_at_once():
    """Calls on two streams, each with a workspace that the call or the caller made there."""
    torch = torch_mod()
    cases = [Case(airkv.BF16, 128, 2, 4, 16, [4000, 900, 35], [1, 1, 1], seed=11), Case(airkv.FP8, 64, 4, 2, 32, [3000, 10], [5, 2], seed=12)]
    want = [c.call(max_q_len=5).clone() for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    args = [(c.q, _dev(c.cu), _dev(c.tables), _dev(c.lens), c.out) for c in cases]
    torch.cuda.synchronize()
    for turn in range(8):
        for c, s, x in zip(cases, streams, args):
            c.pool.paged_cross(*x, max_q_len=5, scale=c.scale, stream=s)
        for s in streams:
            s.synchronize()
        for c, w in zip(cases, want):
            _same(c.out, w, f"turn {turn}")
            c.out.fill_(1.0)
        torch.cuda.synchronize()


def test_a_step_on_another_stream():
    torch = torch_mod()
    one, two = _layer(airkv.INT8, 4), _layer(airkv.INT8, 4)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        _step(one, s)
        s.synchronize()
        _step(two)
        torch.cuda.synchronize()
        _same(one["out"], two["out"])
        _same_pools(one["own"], two["own"])


def test_launchers():
    """A bound call launches as the call itself, reading its tensors anew."""
    torch = torch_mod()
    one, two = _layer(airkv.BF16, 5), _layer(airkv.BF16, 5)
    q, k, v = one["x"].split([8, 2, 2], dim=1)
    append = one["own"].bind_append_rotary(q, k, v, one["slots"], one["lens"], one["f"], one["q_out"])
    cross = one["far"].bind_cross(one["q_out"], one["cu"], one["far_tables"], one["far_lens"], one["out"], max_q_len=1, workspace=one["ws"])
    for turn in range(3):
        x = torch.randn_like(one["x"])
        one["x"].copy_(x)
        two["x"].copy_(x)
        append()
        cross()
        q, k, v = two["x"].split([8, 2, 2], dim=1)
        two["own"].append_rotary(q, k, v, two["slots"], two["lens"], two["f"], q_out=two["q_out"])
        two["far"].paged_cross(two["q_out"], two["cu"], two["far_tables"], two["far_lens"], two["out"], max_q_len=1)
        _same(one["out"], two["out"])
        _same_pools(one["own"], two["own"])
    with pytest.raises(ValueError):
        one["own"].bind_append_rotary(one["q_out"], k[:3].contiguous(), v[:3].contiguous(), one["slots"], one["lens"], one["f"], one["q_out"])


def test_queries_in_place_and_padded_rows():
    """q_out may be q; rows behind the last token, here with slot -1, leave the pages as they were."""
    torch = torch_mod()
    one, two = _layer(airkv.BF16, 6), _layer(airkv.BF16, 6)
    q = [st["x"][:, :8].contiguous() for st in (one, two)]
    k, v = one["x"][:, 8:10], one["x"][:, 10:]
    slots = one["slots"].clone()
    slots[1] = -1
    got = one["own"].append_rotary(q[0], k, v, slots, one["lens"], one["f"], q_out=q[0])
    want = two["own"].append_rotary(q[1], k, v, slots, two["lens"], two["f"])
    assert got is q[0]
    _same(got, want)
    _same_pools(one["own"], two["own"])
    before = two["own"].snapshot()
    two["own"].append_rotary(None, k[1:2], v[1:2], slots[1:2], two["lens"][1:2], two["f"])
    for a, b in zip(before, two["own"].snapshot()):
        assert a is None or np.array_equal(a, b)
    assert one["own"].error_count() == two["own"].error_count() == 0


# ---- a decoder layer


def _pair_sizes(x):
    """For each element, the length of the pair it turns with."""
    half = x.shape[-1] // 2
    m = (x[..., :half] ** 2 + x[..., half:] ** 2).sqrt()
    return torch_mod().cat([m, m], -1)


def _attend(q, k, v, scale, q_off, k_off, p_off, out_step):
    """softmax(scale q k^T) v and a bound: queries and keys off by q_off and k_off [like them], a probability by
    p_off of its size; 2^-18 more for each sum in f32 (no product here has more than 64 terms, no row more than 400)."""
    torch = torch_mod()
    ds = ((q.abs() + q_off) @ (k.abs() + k_off).t() - q.abs() @ k.abs().t()) + q.abs() @ k.abs().t() * 2.0 ** -18
    p = torch.softmax(q @ k.t() * scale, -1)
    o = p @ v
    return o, (p @ v.abs()) * (2 * torch.expm1(scale * ds.amax(-1, keepdim=True)) + p_off + 2.0 ** -18) + out_step * o.abs() + 1e-30


@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.F32])
def test_decoder_layer(dtype):
    """A prompt, a token, a compacted context whose keys are turned to their new places, and another
    token; beside them cross attention to an encoder's states.  Every output against 64 bits from
    the layer's inputs."""
    torch = torch_mod()
    bf16 = dtype == airkv.BF16
    it = torch.bfloat16 if bf16 else torch.float32
    kv, group, d, bs = 2, 4, 64, 16
    nq, scale = kv * group, 1.0 / math.sqrt(d)
    r = np.random.default_rng(41)
    lens = np.array([70, 33], np.int32)
    f = rotary_ref.frequencies(d)
    own, far = airkv.KvPool(16, bs, kv, d, dtype), airkv.KvPool(40, bs, kv, d, dtype)
    tables = r.permutation(16).astype(np.int32).reshape(2, 8)
    # one rounding of a value, and what turning adds to it: c, s, two products and a sum in f32, on
    # |x c| + |y s| <= sqrt(2) |(x, y)|, so that the error is taken of the pair's size
    step = 2.0 ** -8 if bf16 else 2.0 ** -24
    turn = 6 * 2.0 ** -24
    p_off = 2.0 ** -8 if bf16 else 0.0
    out_step = 2.0 ** -8 if bf16 else 2.0 ** -24

    def fused(n):
        x = torch.from_numpy(r.standard_normal((n, nq + 2 * kv, d)).astype(np.float32)).cuda().to(it)
        return x, x.double().cpu()

    def slots(b, at):
        return tables[b, at // bs].astype(np.int64) * bs + at % bs

    def turned(x, positions):
        return torch.from_numpy(rotary_ref.exact(x.numpy(), positions, f, False))

    def compare(got, q, pos, keys, k_pos, values, roundings, what):
        """got [nq, d] for one row: q [nq, d], turned for pos, over keys [n, kv, d], turned for k_pos."""
        qt, kt = turned(q[None], [pos])[0], turned(keys, k_pos)
        for h in range(nq):
            g = h // group
            o, bound = _attend(qt[h][None], kt[:, g], values[:, g], scale, _pair_sizes(qt[h][None]) * (step + turn),
                               _pair_sizes(kt[:, g]) * roundings * (step + turn), p_off, out_step)
            off = (got[h].double().cpu() - o[0]).abs()
            assert (off <= bound[0]).all(), f"{what}, head {h}: {float((off / bound[0]).max())} of the bound"

    # the prompt
    total = int(lens.sum())
    x, x64 = fused(total)
    cu = np.array([0, 70, 103], np.int32)
    at = np.concatenate([np.arange(n) for n in lens])
    sl = np.concatenate([slots(b, np.arange(n)) for b, n in enumerate(lens)])
    q, k, v = x.split([nq, kv, kv], dim=1)
    turned_q = own.append_rotary(q, k, v, _dev(sl), _dev(at.astype(np.int32)), _dev(f))
    out = torch.empty_like(turned_q)
    own.paged_prefill(turned_q, _dev(cu), _dev(tables), _dev(lens), out, max_q_len=70, scale=scale)
    keys = [x64[cu[b]:cu[b + 1], nq:nq + kv] for b in range(2)]
    values = [x64[cu[b]:cu[b + 1], nq + kv:] for b in range(2)]
    places = [np.arange(n) for n in lens]
    for b in range(2):
        for i in (0, 1, 17, int(lens[b]) - 1):
            compare(out[cu[b] + i], x64[cu[b] + i, :nq], i, keys[b][:i + 1], np.arange(i + 1), values[b][:i + 1], 1, f"prompt {b}, {i}")

    def token(roundings, what):
        nonlocal lens
        x, x64 = fused(2)
        q, k, v = x.split([nq, kv, kv], dim=1)
        sl = np.array([slots(b, lens[b:b + 1])[0] for b in range(2)])
        tq = own.append_rotary(q, k, v, _dev(sl), _dev(lens), _dev(f))
        out = torch.empty_like(tq)
        own.paged_decode(tq, _dev(tables), _dev(lens + 1), out, scale=scale)
        for b in range(2):
            keys[b] = torch.cat([keys[b], x64[b:b + 1, nq:nq + kv]])
            values[b] = torch.cat([values[b], x64[b:b + 1, nq + kv:]])
            places[b] = np.append(places[b], lens[b])
            compare(out[b], x64[b, :nq], int(lens[b]), keys[b], places[b], values[b], roundings, f"{what} {b}")
        lens = lens + 1
        return tq, x64

    token(1, "token")
    # every other token of the first sequence, all but the first ten of the second
    keep = [np.arange(0, lens[0], 2), np.arange(10, lens[1])]
    flat = np.concatenate(keep).astype(np.int32)
    cu_keep = np.concatenate([[0], np.cumsum([len(z) for z in keep])]).astype(np.int32)
    own.compact(_dev(tables), _dev(lens), _dev(flat), _dev(cu_keep))
    own.rotate(_dev(tables), _dev(flat), _dev(cu_keep), _dev(f))
    for b in range(2):
        keys[b], values[b], places[b] = keys[b][keep[b]], values[b][keep[b]], np.arange(len(keep[b]))
    lens = np.array([len(z) for z in keep], np.int32)
    tq, x64 = token(2, "after the compaction")

    # the encoder's states, and a prompt's and a token's rows over them
    n = np.array([400, 57], np.int32)
    far_tables = np.full((2, 25), -1, np.int32)
    order = r.permutation(40).astype(np.int32)
    far_tables[0], far_tables[1, :4] = order[:25], order[25:29]
    states, states64 = fused(int(n.sum()))
    sl = np.concatenate([far_tables[b, np.arange(m) // bs].astype(np.int64) * bs + np.arange(m) % bs for b, m in enumerate(n)])
    far.append(states[:, nq:nq + kv].float().contiguous(), states[:, nq + kv:].float().contiguous(), _dev(sl))
    for rows in ([1, 1], [70, 33]):
        c = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        q, q64 = fused(int(c[-1]))
        q, q64 = q[:, :nq].contiguous(), q64[:, :nq]
        out = torch.empty_like(q)
        far.paged_cross(q, _dev(c), _dev(far_tables), _dev(n), out, max_q_len=max(rows), scale=scale)
        for b in range(2):
            k64, v64 = (states64[(0, 400)[b]:(400, 457)[b], z:z + kv] for z in (nq, nq + kv))
            for h in range(nq):
                o, bound = _attend(q64[c[b]:c[b + 1], h], k64[:, h // group], v64[:, h // group], scale, 0.0, 0.0, p_off, out_step)
                off = (out[c[b]:c[b + 1], h].double().cpu() - o).abs()
                assert (off <= bound).all(), f"cross {rows}, {b}, head {h}: {float((off / bound).max())} of the bound"
    assert own.error_count() == far.error_count() == 0
