"""Differential attention and compaction as they are used together, and the calls
around them: refusals, tables and lengths that do not fit, graphs, streams, a shared
workspace, a pool past 4 GiB."""
import numpy as np
import pytest

import airkv
from diff_ref import attend, check, pool_values, sequence
from gpu_helpers import log, torch_mod
from test_gpu_diff_attention import Cache, _p_step

pytestmark = pytest.mark.gpu


def _dev(x):
    return torch_mod().from_numpy(np.ascontiguousarray(x)).cuda()


def _decode_ref(c, q64, lam64, w64, out_scale, lens, tables, norm_eps=1e-5, skip=None):
    kv, vv = pool_values(c.pool)
    scale = float(np.float32(1.0) / np.sqrt(np.float32(c.d)))
    n, pairs = lam64.shape
    want, bound = np.zeros((n, pairs, 2 * c.d)), np.zeros((n, pairs, 2 * c.d))
    for i, m in enumerate(lens):
        k, v = (sequence(x, tables[i], int(m), c.bs) for x in (kv, vv))
        want[i:i + 1], bound[i:i + 1] = attend(q64[i:i + 1], k, v, lam64[i:i + 1], scale, [m - 1], norm_weight=w64,
                                               norm_eps=norm_eps, out_scale=out_scale, skip=None if skip is None else skip[i])
    return want, bound


def _good(c, group=2):
    torch = torch_mod()
    n = len(c.lens)
    q, lam, w, *_ = c.rows(n, group, True, False, True)
    tables, lens = c.device()
    out = torch.full((n, c.kv // 2 * group, 2 * c.d), 3.0, device="cuda")
    return q, lam, w, tables, lens, out


def test_refused_arguments():
    """Every refusal leaves the output alone."""
    torch = torch_mod()
    c = Cache(airkv.BF16, 64, 4, 16, [20, 40], seed=1)
    q, lam, w, tables, lens, out = _good(c)
    cu = _dev(np.array([0, 1, 2], np.int32))
    p = c.pool
    more = dict(norm_weight=w, norm_eps=1e-5)

    def decode(**a):
        x = dict(q=q, lam=lam, block_tables=tables, seq_lens=lens, out=out, **more)
        x.update(a)
        p.paged_diff_decode(**x)

    def prefill(**a):
        x = dict(q=q, lam=lam, cu_q=cu, block_tables=tables, seq_lens=lens, out=out, max_q_len=1, **more)
        x.update(a)
        p.paged_diff_prefill(**x)

    both = [dict(q=q[:, :, :32].contiguous()), dict(q=q.double()), dict(q=q.half()), dict(q=q.transpose(1, 2)), dict(q=q[:, :6]),
            dict(lam=lam[:-1]), dict(lam=lam.double()), dict(lam=lam[None].expand(2, -1)), dict(lam=lam[None, :3].contiguous()),
            dict(out=out[:, :3]), dict(out=out.transpose(0, 1)), dict(out=out.half()), dict(seq_lens=lens.long()), dict(seq_lens=lens[:1]),
            dict(block_tables=tables[:, ::2]), dict(block_tables=tables.long()), dict(norm_weight=w[:64].contiguous()),
            dict(norm_weight=w, norm_eps=None), dict(norm_eps=0.0), dict(norm_eps=-1.0), dict(norm_eps=float("nan")),
            dict(out_scale=float("nan")), dict(scale=float("nan")), dict(workspace=torch.empty(32, dtype=torch.uint8, device="cuda")),
            dict(q=q.cpu())]
    for call, bad in [(f, b) for f in (decode, prefill) for b in both] + \
            [(decode, dict(max_splits=0)), (decode, dict(max_splits=257)), (decode, dict(block_tables=tables[:1])),
             (prefill, dict(scale=0.0)), (prefill, dict(scale=-1.0)), (prefill, dict(cu_q=cu[:2])), (prefill, dict(cu_q=cu.long())),
             (prefill, dict(max_q_len=-1))]:
        with pytest.raises((TypeError, ValueError, airkv.AirKvError)):
            call(**bad)
    assert (out == 3.0).all() and p.error_count() == 0
    decode()
    prefill()
    assert torch.isfinite(out).all()
    # addresses that are not 16-byte aligned
    flat = torch.zeros(q.numel() + 1, device="cuda")
    with pytest.raises(airkv.AirKvError, match="aligned"):
        decode(q=flat[1:].view(q.shape))
    # pools that have no pairs, or rows too wide
    odd, wide = airkv.KvPool(4, 16, 3, 64, airkv.BF16), airkv.KvPool(4, 16, 2, 256, airkv.BF16)
    for pool, n_q, match in ((odd, 6, "odd"), (wide, 4, "head_dim"), (p, 6, "multiple"), (p, 0, "multiple")):
        with pytest.raises(airkv.AirKvError, match=match):
            pool.diff_decode_workspace_size(n_q, 1, 1)
        with pytest.raises(airkv.AirKvError, match=match):
            pool.diff_prefill_workspace_size(n_q, 1, 1)


def test_empty_calls():
    torch = torch_mod()
    c = Cache(airkv.INT8, 32, 2, 16, [5], seed=2)
    q, lam, _, tables, lens, out = _good(c)
    c.pool.paged_diff_decode(q[:0], lam, tables[:0], lens[:0], out[:0])
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.pool.paged_diff_prefill(q[:0], lam, zero, tables[:0], lens[:0], out[:0], max_q_len=0)
    c.pool.paged_diff_prefill(q[:0], lam, torch.zeros(2, dtype=torch.int32, device="cuda"), tables, lens, out[:0], max_q_len=0)
    assert (out == 3.0).all() and c.pool.error_count() == 0


@pytest.mark.parametrize("dtype,bs", [(airkv.F32, 16), (airkv.BF16, 32), (airkv.INT8, 16), (airkv.FP8, 32)])
@pytest.mark.parametrize("splits", [1, 256])
def test_decode_tables_and_lengths_outside(dtype, bs, splits):
    """Blocks outside the pool are left out of the sum and counted, lengths are
    clamped to the table and counted; a sequence that has no other block gives zeros
    where it is empty."""
    torch = torch_mod()
    c = Cache(dtype, 64, 2, bs, [300, 90, 16, 400, 0, 33], seed=5)
    q, lam, w, q64, lam64, w64 = c.rows(6, 3, True, True, True)
    tables, lens = c.tables.copy(), c.lens.copy()
    skip = [np.zeros(max(int(n), 1), bool)[:int(n)] for n in lens]
    for i, j, x in ((0, 1, -1), (0, 300 // bs, c.pool.num_blocks), (3, 0, 1 << 30)):
        tables[i, j] = x
        skip[i][j * bs:(j + 1) * bs] = True
    lens[4] = -3
    out = torch.full((6, 3, 128), float("nan"), device="cuda")
    c.pool.paged_diff_decode(q, _dev(lam.cpu().numpy()), _dev(tables), _dev(lens), out, norm_weight=w, norm_eps=1e-5, max_splits=splits)
    want, bound = _decode_ref(c, q64, lam64, w64, 1.0, c.lens, np.where(tables < c.pool.num_blocks, tables, -1), skip=skip)
    log(f"tables outside: {check(out.cpu().numpy(), want, bound, airkv.F32, 'outside'):.3f} of the bound")
    tiles = bs // 16
    last = min(bs, 300 - 300 // bs * bs)
    assert c.pool.error_count(reset=True) == 1 + tiles + -(-last // 16) + tiles
    # longer than the table: as long as the table
    lens = np.array([1 << 30, 80, 16, 80, 0, 33], np.int32)
    cols = 300 // bs
    c.pool.paged_diff_decode(q, _dev(lam.cpu().numpy()), _dev(c.tables[:, :cols]), _dev(lens), out,
                             norm_weight=w, norm_eps=1e-5, max_splits=splits)
    want, bound = _decode_ref(c, q64, lam64, w64, 1.0, [cols * bs, 80, 16, 80, 0, 33], c.tables)
    check(out.cpu().numpy(), want, bound, airkv.F32, "clamped")
    assert c.pool.error_count(reset=True) == 1
    # no block of a sequence in the pool: zeros
    tables = c.tables.copy()
    tables[[0, 2]] = -1
    c.pool.paged_diff_decode(q, _dev(lam.cpu().numpy()), _dev(tables), _dev(c.lens), out, norm_weight=w, norm_eps=1e-5, max_splits=splits)
    assert (out[0] == 0).all() and (out[2] == 0).all() and torch.isfinite(out).all()
    assert c.pool.error_count(reset=True) == -(-300 // 16) + 1


@pytest.mark.parametrize("dtype,f32", [(airkv.F32, True), (airkv.BF16, False), (airkv.INT8, False), (airkv.FP8, True)])
def test_prefill_sequences_refused(dtype, f32):
    """Sequences whose rows or lengths do not fit are zero-filled and counted, the
    others are computed as ever (against 64 bits: where a block of rows is cut, and so
    the order of its sums, goes by what the whole launch holds); rows outside every
    sequence are not touched; blocks outside the pool are zero keys and values."""
    torch = torch_mod()
    c = Cache(dtype, 64, 2, 16, [90, 70, 40, 50, 33], seed=6)
    q, lam, w, q64, lam64, w64 = c.rows(80, 2, f32, False, True)
    p_step = 0.0 if f32 else _p_step(c)
    scale = float(np.float32(1.0) / np.sqrt(np.float32(c.d)))
    kv, vv = pool_values(c.pool)

    def right(got, i, a, b, tables=c.tables):
        k, v = (sequence(x, tables[i], int(c.lens[i]), 16) for x in (kv, vv))
        want, bound = attend(q64[a:b], k, v, lam64[a:b], scale, c.lens[i] - (b - a) + np.arange(b - a), norm_weight=w64, norm_eps=1e-5,
                             p_step=p_step)
        check(got[a:b], want, bound, airkv.F32 if f32 else airkv.BF16, f"sequence {i}", p_step)

    cu = np.array([3, 20, 40, 45, 60, 70], np.int32)            # rows 0..2 and 70..79 belong to nobody
    odt = torch.float32 if f32 else torch.bfloat16

    def run(lens, cu, tables=c.tables):
        out = torch.full((80, 2, 128), 9.0, device="cuda", dtype=odt)
        c.pool.paged_diff_prefill(q, lam, _dev(cu), _dev(tables), _dev(lens), out, max_q_len=20, norm_weight=w, norm_eps=1e-5)
        return out.float().cpu().numpy()

    clean = run(c.lens, cu)
    assert c.pool.error_count() == 0 and np.isfinite(clean).all()
    assert (clean[:3] == 9).all() and (clean[70:] == 9).all() and (clean[3:70] != 9).any(axis=(1, 2)).all()
    lens = c.lens.copy()
    lens[0] = 16                                                # fewer cached than new ones
    lens[2] = 16 * c.tables.shape[1] + 1                        # past its table
    lens[3] = -4
    got = run(lens, cu)
    assert c.pool.error_count(reset=True) == 3
    for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        if i in (0, 2, 3):
            assert (got[a:b] == 0).all(), i
        else:
            right(got, i, a, b)
    assert (got[:3] == 9).all() and (got[70:] == 9).all()
    for bad in ([3, 20, 40, 45, 60, 81], [-1, 20, 40, 45, 60, 70], [3, 20, 19, 45, 60, 70]):
        got = run(c.lens, np.array(bad, np.int32))
        assert c.pool.error_count(reset=True) == 1 and (got[71:] == 9).all()
        right(got, 3, 45, 60)
    tables = c.tables.copy()
    tables[1, 2] = -7
    got = run(c.lens, cu, tables)
    assert c.pool.error_count(reset=True) >= 1
    for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        right(got, i, a, b, tables)
    assert not np.array_equal(got[20:40], clean[20:40])


def test_a_row_does_not_depend_on_its_neighbours():
    """max_splits 1 and a call of one sequence give a sequence the same bits, and a
    prefill block's rows do not see what the rows beside them hold."""
    torch = torch_mod()
    c = Cache(airkv.BF16, 64, 2, 16, [200, 200, 200], seed=8)
    q, lam, w, tables, lens, out = _good(c)
    c.pool.paged_diff_decode(q, lam, tables, lens, out, max_splits=1)
    for i in range(3):
        alone = torch.empty_like(out[:1])
        c.pool.paged_diff_decode(q[i:i + 1], lam, tables[i:i + 1], lens[i:i + 1], alone, max_splits=1)
        assert torch.equal(alone[0], out[i])
    for f32 in (True, False):
        q, lam, _, *_ = c.rows(120, 2, f32, False, False)
        cu = _dev(np.array([0, 40, 80, 120], np.int32))
        first = torch.empty(120, 2, 128, device="cuda", dtype=q.dtype)
        c.pool.paged_diff_prefill(q, lam, cu, tables, lens, first, max_q_len=40)
        q2 = q.clone()
        q2[1::2] *= 40
        second = torch.empty_like(first)
        c.pool.paged_diff_prefill(q2, lam, cu, tables, lens, second, max_q_len=40)
        assert torch.equal(first[::2], second[::2]) and not torch.equal(first[1::2], second[1::2])


@pytest.mark.parametrize("dtype,f32", [(airkv.F32, True), (airkv.BF16, False), (airkv.INT8, False)])
def test_graph_replays(dtype, f32):
    """A step -- append, differential prefill, differential decode -- and a compaction
    in two graphs that share a workspace, replayed with new values and eager work
    between: the same bits as eager calls on a twin pool."""
    torch = torch_mod()
    lens0 = [130, 40, 65, 300]
    grow = 8
    caches = [Cache(dtype, 64, 4, 16, lens0, seed=11, grow=grow) for _ in range(2)]
    g, e = caches
    odt = torch.float32 if f32 else torch.bfloat16
    n = len(lens0)
    r = np.random.default_rng(4)
    full = (g.lens + grow).astype(np.int32)
    tables, lens = _dev(g.tables), _dev(full)
    cu = _dev((np.arange(n + 1) * grow).astype(np.int32))
    pos = full[:, None] - grow + np.arange(grow)[None, :]
    slots = _dev((np.take_along_axis(g.tables, pos // 16, 1).astype(np.int64) * 16 + pos % 16).reshape(-1))
    keeps = [np.concatenate([np.arange(4), np.arange(12, m)]) for m in full]
    kcu = _dev(np.concatenate([[0], np.cumsum([len(k) for k in keeps])]).astype(np.int32))
    keep = _dev(np.concatenate(keeps).astype(np.int32))
    short = _dev(np.array([len(k) for k in keeps], np.int32))
    k_new, v_new = (torch.empty(n * grow, 4, 64, device="cuda") for _ in range(2))
    qp, qd = torch.empty(n * grow, 12, 64, device="cuda", dtype=odt), torch.empty(n, 12, 64, device="cuda", dtype=odt)
    lam = _dev(r.uniform(0.1, 0.9, (n * grow, 6)).astype(np.float32))
    w = _dev(r.uniform(0.5, 1.5, 128).astype(np.float32))
    outs = [[torch.empty(n * grow, 6, 128, device="cuda", dtype=odt), torch.empty(n, 6, 128, device="cuda", dtype=odt),
             torch.empty(n, 6, 128, device="cuda", dtype=odt)] for _ in range(2)]
    size = max(g.pool.diff_decode_workspace_size(12, n, tables.shape[1]), g.pool.diff_prefill_workspace_size(12, n, grow))
    ws = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]

    def step(c, out, ws):
        c.pool.append(k_new, v_new, slots)
        c.pool.paged_diff_prefill(qp, lam, cu, tables, lens, out[0], max_q_len=grow, norm_weight=w, norm_eps=1e-5, workspace=ws)
        c.pool.paged_diff_decode(qd, lam[:n], tables, lens, out[1], norm_weight=w, norm_eps=1e-5, workspace=ws)

    def shrink(c, out, ws):
        c.pool.compact(tables, lens, keep, kcu)
        c.pool.paged_diff_decode(qd, lam[:n], tables, short, out[2], workspace=ws)

    def fill():
        for x in (k_new, v_new, qp, qd):
            x.copy_(_dev(r.standard_normal(tuple(x.shape)).astype(np.float32)))

    fill()
    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for f in (step, shrink):
            f(g, outs[0], ws[0])                        # once eagerly, before the capture
            f(e, outs[1], ws[1])
        torch.cuda.synchronize()
        for f in (step, shrink):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                f(g, outs[0], ws[0])
            graphs.append(graph)
    torch.cuda.synchronize()
    for i in range(4):
        fill()
        torch.cuda.synchronize()
        for j in ((0, 1) if i % 2 else (0, 0, 1)):
            graphs[j].replay()
            (step, shrink)[j](e, outs[1], ws[1])
            (k_new.sum() + outs[1][0].float().sum()).item()              # eager work and a wait between
            torch.cuda.synchronize()
            for a, b in zip(*outs):
                assert torch.equal(a, b), (i, j)
        for a, b in zip(g.pool.snapshot(), e.pool.snapshot()):
            assert a is None or np.array_equal(a.view(np.uint8), b.view(np.uint8))
    assert g.pool.error_count() == 0 and e.pool.error_count() == 0


def test_streams():
    """Calls on a stream of their own, given as an argument and as the current one, two at a time."""
    torch = torch_mod()
    c = Cache(airkv.BF16, 128, 4, 16, [700, 30, 2000], seed=12)
    q, lam, w, tables, lens, out = _good(c, 4)
    c.pool.paged_diff_decode(q, lam, tables, lens, out)
    cu = _dev(np.array([0, 1, 2, 3], np.int32))
    pre = torch.empty_like(out)
    c.pool.paged_diff_prefill(q, lam, cu, tables, lens, pre, max_q_len=1)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    o1, o2, o3 = (torch.full_like(out, 5.0) for _ in range(3))
    ws = [c.pool.new_diff_workspace(q.shape[1], 3, tables.shape[1]) for _ in range(2)]
    pws = c.pool.new_diff_prefill_workspace(q.shape[1], 3, 1)
    torch.cuda.synchronize()
    for _ in range(5):
        c.pool.paged_diff_decode(q, lam, tables, lens, o1, workspace=ws[0], stream=a)
        with torch.cuda.stream(b):
            c.pool.paged_diff_decode(q, lam, tables, lens, o2, workspace=ws[1])
            launch = c.pool.bind_diff_prefill(q, lam, cu, tables, lens, o3, max_q_len=1, workspace=pws)
            launch()
    torch.cuda.synchronize()
    assert torch.equal(o1, out) and torch.equal(o2, out) and torch.equal(o3, pre)


@pytest.mark.parametrize("dtype,f32", [(airkv.F32, True), (airkv.BF16, False), (airkv.INT8, False), (airkv.FP8, True)])
def test_prompt_steps_and_compaction(dtype, f32):
    """A prompt in two chunks, steps of one token, a compaction to the first tokens and
    the newest, and further steps -- the pages' blocks from a manager, every output
    against 64 bits over what the pool holds by then."""
    torch = torch_mod()
    kv, d, bs, group = 4, 64, 16, 3
    r = np.random.default_rng(20)
    mgr = airkv.SequenceManager(64, bs)
    pool = airkv.KvPool(64, bs, kv, d, dtype)
    c = Cache.__new__(Cache)
    c.pool, c.d, c.bs, c.kv, c.r = pool, d, bs, kv, r
    s = airkv.PagedSessionCache(mgr, [pool])
    odt = airkv.F32 if f32 else airkv.BF16
    scale = float(np.float32(1.0) / np.sqrt(np.float32(d)))
    # see the tolerance of the 16-bit products in the tests of the prefill kernels
    step16 = 0.0 if f32 or dtype == airkv.F32 else 2.0 ** -11 * (2 if dtype == airkv.BF16 else 3 + 2 * (0.64 * d ** 0.5 + 8)) + 2.0 ** -16

    def table():
        return np.asarray(mgr.table(s.seq_id).physical_blocks, np.int32)[None]

    def rows(n):
        return c.rows(n, group, f32, True, True)

    def expect(q64, lam64, w64, n, new, p_step):
        kv64, vv64 = pool_values(pool)
        k, v = (sequence(x, table()[0], n, bs) for x in (kv64, vv64))
        return attend(q64, k, v, lam64, scale, n - new + np.arange(new), norm_weight=w64, norm_eps=1e-5, out_scale=0.5, p_step=p_step)

    def grow(n):
        k, v = (_dev(r.standard_normal((n, kv, d)).astype(np.float32)) for _ in range(2))
        s.append(0, k, v)
        return s.seq_len(0)

    def prompt(new):
        n = grow(new)
        q, lam, w, q64, lam64, w64 = rows(new)
        out = torch.empty(new, group * kv // 2, 2 * d, device="cuda", dtype=q.dtype)
        pool.paged_diff_prefill(q, lam, _dev(np.array([0, new], np.int32)), _dev(table()), _dev(np.array([n], np.int32)), out,
                                max_q_len=new, norm_weight=w, norm_eps=1e-5, out_scale=0.5)
        want, bound = expect(q64, lam64, w64, n, new, step16)
        return check(out.float().cpu().numpy(), want, bound, odt, "prompt", step16)

    def step():
        n = grow(1)
        q, lam, w, q64, lam64, w64 = rows(1)
        out = torch.empty(1, group * kv // 2, 2 * d, device="cuda", dtype=q.dtype)
        pool.paged_diff_decode(q, lam, _dev(table()), _dev(np.array([n], np.int32)), out, norm_weight=w, norm_eps=1e-5, out_scale=0.5)
        want, bound = expect(q64, lam64, w64, n, 1, 0.0)
        return check(out.float().cpu().numpy(), want, bound, odt, "step")

    used = [prompt(200), prompt(77)] + [step() for _ in range(4)]
    before = [x.clone() for x in s.load(0)]
    keep = np.concatenate([np.arange(4), np.arange(281 - 100, 281)])
    s.compact(keep)
    for x, y in zip(s.load(0), before):
        assert torch.equal(x, y[_dev(keep)])
    assert len(table()[0]) == -(-104 // bs)
    used += [step() for _ in range(10)] + [prompt(30), step()]
    assert pool.error_count() == 0
    log(f"prompt, steps, compaction dtype={dtype}: {max(used):.3f} of the bound")


@pytest.mark.parametrize("dtype,n_blocks", [(airkv.BF16, 140_000), (airkv.INT8, 270_000)])
def test_pool_past_4_gib(dtype, n_blocks):
    """Blocks whose bytes lie past 2^32 give the bits that a small pool's do."""
    torch = torch_mod()
    kv, d, bs = 8, 128, 16
    r = np.random.default_rng(30)
    lens = np.array([1, 100, 513, 1200], np.int32)
    nb = -(-lens // bs)
    total = int(nb.sum())
    big, small = airkv.KvPool(n_blocks, bs, kv, d, dtype), airkv.KvPool(total, bs, kv, d, dtype)
    assert n_blocks * big.slab_bytes > 1 << 32
    ids = [np.sort(r.choice(np.arange(n_blocks - 4 * total, n_blocks), total, replace=False))[::-1].astype(np.int32),
           np.arange(total, dtype=np.int32)]
    k, v = (_dev(r.standard_normal((int(lens.sum()), kv, d)).astype(np.float32)) for _ in range(2))
    pairs = kv // 2 * 2
    q = _dev(r.standard_normal((40, 2 * pairs, d)).astype(np.float32)).to(torch.bfloat16)
    lam = _dev(r.uniform(0.1, 0.9, pairs).astype(np.float32))
    cu = _dev(np.array([0, 1, 11, 25, 40], np.int32))
    keeps = [np.arange(0, m, 2) for m in lens]
    keep, kcu = _dev(np.concatenate(keeps).astype(np.int32)), _dev(np.concatenate([[0], np.cumsum([len(x) for x in keeps])]).astype(np.int32))
    got = []
    for pool, block in zip((big, small), ids):
        tables, at = np.full((4, int(nb.max())), -1, np.int32), 0
        slots = []
        for i, n in enumerate(nb):
            tables[i, :n] = block[at:at + n]
            at += n
            t = np.arange(lens[i])
            slots.append(tables[i, t // bs].astype(np.int64) * bs + t % bs)
        pool.append(k, v, _dev(np.concatenate(slots)))
        t, n = _dev(tables), _dev(lens)
        outs = [torch.empty(4, pairs, 2 * d, device="cuda", dtype=torch.bfloat16), torch.empty(40, pairs, 2 * d, device="cuda", dtype=torch.bfloat16),
                torch.empty(40, pairs, 2 * d, device="cuda")]
        pool.paged_diff_decode(q[:4], lam, t, n, outs[0])
        pool.paged_diff_prefill(q, lam, cu, t, n, outs[1], max_q_len=15)
        pool.paged_diff_prefill(q, lam, cu, t, n, outs[2], max_q_len=15)
        pool.compact(t, n, keep, kcu)
        after = torch.empty(4, pairs, 2 * d, device="cuda")
        pool.paged_diff_decode(q[:4], lam, t, _dev(np.array([len(x) for x in keeps], np.int32)), after)
        assert pool.error_count() == 0
        got.append(outs + [after])
    for a, b in zip(*got):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_many_pieces():
    """One sequence over hundreds of slices (the merge's 16 waves) on 1-byte pages."""
    torch = torch_mod()
    for dtype, kv, d in ((airkv.FP8, 2, 128), (airkv.F32, 2, 32)):
        c = Cache(dtype, d, kv, 16, [40_000, 5], seed=13)
        for f32 in (True, False):
            q, lam, w, q64, lam64, w64 = c.rows(2, 2, f32, False, True)
            tables, lens = c.device()
            out = torch.empty(2, 2, 2 * d, device="cuda", dtype=q.dtype)
            want, bound = _decode_ref(c, q64, lam64, w64, 1.0, c.lens, c.tables)
            for splits in (256, 20, 1):
                c.pool.paged_diff_decode(q, lam, tables, lens, out, norm_weight=w, norm_eps=1e-5, max_splits=splits)
                used = check(out.float().cpu().numpy(), want, bound, airkv.F32 if f32 else airkv.BF16, f"splits {splits}")
                log(f"many pieces dtype={dtype} f32={f32} splits={splits}: {used:.3f} of the bound")


@pytest.mark.parametrize("dtype,d,scale_group", [(airkv.F32, 128, 32), (airkv.BF16, 96, 32), (airkv.INT8, 128, 128), (airkv.FP8, 64, 64),
                                                 (airkv.INT8, 96, 8), (airkv.FP8, 128, 32), (airkv.INT8, 32, 16)])
@pytest.mark.parametrize("q_f32,out_f32", [(True, False), (False, True)])
def test_mixed_types_and_scale_groups(dtype, d, scale_group, q_f32, out_f32):
    """f32 queries with bf16 outputs and the other way round, scale groups from 8 to the whole row."""
    torch = torch_mod()
    c = Cache(dtype, d, 4, 16, [1, 77, 1040, 16, 300], seed=d + scale_group, scale_group=scale_group)
    q, lam, w, q64, lam64, w64 = c.rows(5, 9, q_f32, True, True)
    tables, lens = c.device()
    odt = airkv.F32 if out_f32 else airkv.BF16
    out = torch.full((5, 18, 2 * d), float("nan"), device="cuda", dtype=torch.float32 if out_f32 else torch.bfloat16)
    want, bound = _decode_ref(c, q64, lam64, w64, 1.0, c.lens, c.tables)
    for splits in (256, 1):
        c.pool.paged_diff_decode(q, lam, tables, lens, out, norm_weight=w, norm_eps=1e-5, max_splits=splits)
        used = check(out.float().cpu().numpy(), want, bound, odt, f"splits {splits}")
    cu = _dev(np.arange(6, dtype=np.int32))                     # the same rows as prompts' last tokens
    c.pool.paged_diff_prefill(q, lam, cu, tables, lens, out.fill_(float("nan")), max_q_len=1, norm_weight=w, norm_eps=1e-5)
    more = check(out.float().cpu().numpy(), want, bound, odt, "prefill")
    log(f"mixed types dtype={dtype} d={d} scale_group={scale_group}: decode {used:.3f}, prefill {more:.3f} of the bound")
    assert c.pool.error_count() == 0


def test_a_block_in_several_tables():
    """Sequences that share a prefix's blocks, one of them twice in one table."""
    torch = torch_mod()
    c = Cache(airkv.BF16, 64, 2, 16, [64, 40, 50], seed=21)
    tables = c.tables.copy()
    tables[1, :2] = tables[0, :2]
    tables[2, 3] = tables[2, 0]
    q, lam, w, q64, lam64, w64 = c.rows(3, 2, True, False, True)
    out = torch.empty(3, 2, 128, device="cuda")
    want, bound = _decode_ref(c, q64, lam64, w64, 1.0, c.lens, tables)
    c.pool.paged_diff_decode(q, lam, _dev(tables), _dev(c.lens), out, norm_weight=w, norm_eps=1e-5)
    check(out.cpu().numpy(), want, bound, airkv.F32, "decode")
    c.pool.paged_diff_prefill(q, lam, _dev(np.arange(4, dtype=np.int32)), _dev(tables), _dev(c.lens), out.fill_(3.0), max_q_len=1,
                              norm_weight=w, norm_eps=1e-5)
    check(out.cpu().numpy(), want, bound, airkv.F32, "prefill")
