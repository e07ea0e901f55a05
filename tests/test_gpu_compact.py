"""Compaction of cached sequences in their own pages (air_kv_compact,
air_kv_session_compact): every byte of the pool against moving the rows on the host."""
import numpy as np
import pytest

import airkv
from gpu_helpers import log, torch_mod

pytestmark = pytest.mark.gpu


def _pool(dtype, d, kv, bs, lens, seed, scale_group=32, spare=2):
    """A pool of random bytes, and sequences in blocks of random order."""
    r = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    nb = -(-lens // bs)
    pool = airkv.KvPool(int(nb.sum()) + spare, bs, kv, d, dtype, scale_group)
    pool.write_blocks(np.arange(pool.num_blocks, dtype=np.int32), r.integers(0, 256, (pool.num_blocks, pool.block_bytes), np.uint8))
    perm = r.permutation(pool.num_blocks).astype(np.int32)
    tables = np.full((len(lens), max(1, int(nb.max(initial=0)))), -1, np.int32)
    at = 0
    for i, n in enumerate(nb):
        tables[i, :n] = perm[at:at + n]
        at += n
    return pool, tables, lens, r


def _bytes(pool):
    return [None if x is None else np.ascontiguousarray(x).view(np.uint8).copy() for x in pool.snapshot()]


def _moved(arrays, tables, keeps, bs):
    """The arrays with each sequence's kept tokens moved (sources as they were)."""
    out = [None if x is None else x.copy() for x in arrays]
    for row, keep in zip(tables, keeps):
        keep = np.asarray(keep, np.int64)
        to = np.arange(len(keep))
        for x, y in zip(arrays, out):
            if x is not None:
                y[row[to // bs], :, to % bs] = x[row[keep // bs], :, keep % bs]
    return out


def _run(pool, tables, lens, keeps):
    torch = torch_mod()
    cu = np.concatenate([[0], np.cumsum([len(k) for k in keeps])]).astype(np.int32)
    keep = np.concatenate([np.asarray(k, np.int32) for k in keeps] + [np.zeros(0, np.int32)]).astype(np.int32)
    pool.compact(*(torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (tables, lens, keep, cu)))
    torch.cuda.synchronize()


def _same(pool, want, what):
    for x, y, name in zip(_bytes(pool), want, ("K", "V", "K scales", "V scales")):
        if x is not None:
            assert np.array_equal(x, y), f"{what}: {name} differs at {np.argwhere(x != y)[:3].tolist()}"


def _keeps(r, lens, kind):
    out = []
    for n in lens.tolist():
        if kind == "half":
            k = np.sort(r.permutation(n)[:n // 2])
        elif kind == "window":
            k = np.concatenate([np.arange(min(4, n)), np.arange(min(n, max(4, n - n // 3)), n)])
        elif kind == "all":
            k = np.arange(n)
        elif kind == "drop_one":
            k = np.arange(1, n)
        elif kind == "last":
            k = np.arange(max(0, n - 1), n)
        else:
            k = np.arange(0)
        out.append(k)
    return out


@pytest.mark.parametrize("kind", ["half", "window", "all", "drop_one", "last", "none"])
@pytest.mark.parametrize("dtype,d,kv,bs,scale_group", [
    (airkv.F32, 64, 8, 16, 32), (airkv.BF16, 128, 8, 16, 32), (airkv.BF16, 96, 3, 32, 32), (airkv.INT8, 128, 4, 16, 32),
    (airkv.FP8, 32, 2, 32, 8), (airkv.INT8, 160, 1, 16, 16), (airkv.F32, 256, 2, 32, 32), (airkv.FP8, 224, 5, 16, 32)])
def test_compact(dtype, d, kv, bs, scale_group, kind):
    pool, tables, lens, r = _pool(dtype, d, kv, bs, [1, 16, 0, 517, 2300, 33, 1025, 100], seed=d + kv, scale_group=scale_group)
    keeps = _keeps(r, lens, kind)
    want = _moved(_bytes(pool), tables, keeps, bs)
    _run(pool, tables, lens, keeps)
    _same(pool, want, kind)
    assert pool.error_count() == 0


@pytest.mark.parametrize("batch,n,kv", [(1, 9000, 2), (1, 3, 1), (70, 300, 16), (600, 90, 4)])
def test_compact_batches(batch, n, kv):
    """Few long chains, and many short ones."""
    r = np.random.default_rng(batch)
    pool, tables, lens, r = _pool(airkv.BF16, 128, kv, 16, r.integers(1, n + 1, batch), seed=batch)
    keeps = _keeps(r, lens, "half")
    want = _moved(_bytes(pool), tables, keeps, 16)
    _run(pool, tables, lens, keeps)
    _same(pool, want, "half")
    # a second time, on what is left
    lens = np.array([len(k) for k in keeps], np.int32)
    keeps = _keeps(r, lens, "window")
    want = _moved(want, tables, keeps, 16)
    _run(pool, tables, lens, keeps)
    _same(pool, want, "window")
    assert pool.error_count() == 0


def test_compact_refused_positions():
    """What is not an ascending position of the sequence is skipped and counted:
    the row it would have filled stays; so are blocks and ranges outside."""
    torch = torch_mod()
    pool, tables, lens, r = _pool(airkv.BF16, 64, 2, 16, [100, 100, 40, 50], seed=3)
    before = _bytes(pool)
    keep = [np.array([2, 2, 5, 4, 99, 100, -1, 98]),        # twice the same, a step back, past the end, negative; 98 is fine
            np.array([0, 1, 5, 9]), np.array([39]), np.arange(1, 50)]
    lens[2] = 16 * tables.shape[1] + 7                      # longer than its table: clamped
    tables[1, 0] = pool.num_blocks                          # outside the pool: its tokens are neither read nor written
    tables[2, 2] = -1
    want = _moved(before, tables[[0, 3]], [[2, 1, 5, 3, 99, 5, 6, 98], np.arange(1, 50)], 16)
    _run(pool, tables, lens, keep)
    _same(pool, want, "refused positions")
    assert pool.error_count(reset=True) == 4 + 2 + 2        # positions 0 and 1 of sequence 1 stay where they are
    # ranges outside the list: the sequence is left alone
    dev = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in
           (tables[:1], lens[:1], np.arange(5, 9, dtype=np.int32), np.array([0, 7], np.int32))]
    pool.compact(*dev)
    _same(pool, want, "a range past the list")
    assert pool.error_count(reset=True) == 1


def test_compact_wrapper_refusals():
    torch = torch_mod()
    pool, tables, lens, _ = _pool(airkv.BF16, 64, 2, 16, [100, 40], seed=3)
    t, n = torch.from_numpy(tables).cuda(), torch.from_numpy(lens).cuda()
    keep, cu = torch.arange(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for bad in ((t.long(), n, keep, cu), (t, n[:1], keep, cu), (t, n, keep.long(), cu), (t, n, keep, cu[:2]), (t[:, ::2], n, keep, cu)):
        with pytest.raises((TypeError, ValueError)):
            pool.compact(*bad)
    pool.compact(t, n, keep[:0], torch.zeros(3, dtype=torch.int32, device="cuda"))
    pool.compact(t[:0], n[:0], keep, cu[:1])


@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16, airkv.INT8])
def test_session_compact(dtype):
    """Two layers; the fork keeps its tokens, shared blocks are copied, blocks are released."""
    torch = torch_mod()
    r = np.random.default_rng(5)
    mgr = airkv.SequenceManager(40, 16)
    pools = [airkv.KvPool(40, 16, 2, 64, dtype) for _ in range(2)]
    s = airkv.PagedSessionCache(mgr, pools)
    rows = [torch.from_numpy(r.standard_normal((150, 2, 64)).astype(np.float32)).cuda() for _ in range(4)]
    for layer in range(2):
        s.append(layer, rows[2 * layer], rows[2 * layer + 1])
    child = s.fork()
    whole = [[x.clone() for x in s.load(layer)] for layer in range(2)]
    keep = np.concatenate([np.arange(4), np.sort(r.permutation(np.arange(4, 150))[:60])])
    s.compact(keep)
    at = torch.from_numpy(keep).cuda()
    for layer in range(2):
        assert s.seq_len(layer) == 64 and child.seq_len(layer) == 150
        for got, kept, x in zip(s.load(layer), child.load(layer), whole[layer]):
            assert torch.equal(got, x[at]) and torch.equal(kept, x)
    # four blocks written of ten shared ones were copied, six released by this sequence stay the fork's
    assert mgr.allocator.num_used_blocks() == 10 + 4
    # the cache goes on growing, and a prefix that does not move is a truncation
    s.append(0, rows[0][:20], rows[1][:20])
    s.append(1, rows[2][:20], rows[3][:20])
    s.compact(np.arange(70))
    assert s.seq_len(0) == 70 and torch.equal(s.load(0)[0][:64], whole[0][0][at])
    for bad in ([3, 2], [0, 0], [70], [-1, 4]):
        with pytest.raises(airkv.AirKvError):
            s.compact(bad)
    assert s.seq_len(1) == 70
    s.truncate_to(50)
    s.append(0, rows[0][:1], rows[1][:1])
    with pytest.raises(airkv.AirKvError, match="layers"):
        s.compact([1])
    child.close()
    s.clear()
    s.compact([])
    assert s.seq_len(0) == 0 and mgr.allocator.num_used_blocks() == 0


def test_session_compact_without_free_blocks():
    """Shared blocks that cannot be copied: refused, nothing changed."""
    torch = torch_mod()
    mgr = airkv.SequenceManager(4, 16)
    s = airkv.PagedSessionCache(mgr, [airkv.KvPool(4, 16, 2, 64, airkv.F32)])
    x = torch.randn(64, 2, 64, device="cuda")
    s.append(0, x, x)
    child = s.fork()
    with pytest.raises(MemoryError):
        s.compact(np.arange(1, 64))
    assert s.seq_len(0) == 64 and torch.equal(s.load(0)[0], x) and torch.equal(child.load(0)[0], x)
    child.close()
    s.compact(np.arange(1, 64))
    assert torch.equal(s.load(0)[0], x[1:])
