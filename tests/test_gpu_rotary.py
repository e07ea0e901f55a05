"""Rotary positions: append_rotary against turning on the host and appending, rotate against
turning what the pages held."""
import numpy as np
import pytest

import airkv
import oracle
import rotary_ref as ref
from gpu_helpers import torch_mod

pytestmark = pytest.mark.gpu

F32_HALF_STEP = 2.0 ** -24
KINDS = {airkv.F32: oracle.F32, airkv.BF16: oracle.BF16, airkv.INT8: oracle.INT8, airkv.FP8: oracle.FP8}
POOLS = [(airkv.F32, 64, 8, 16, 32), (airkv.BF16, 128, 8, 16, 32), (airkv.BF16, 96, 3, 32, 32), (airkv.INT8, 128, 4, 16, 32),
         (airkv.FP8, 32, 2, 32, 8), (airkv.INT8, 160, 1, 16, 16), (airkv.F32, 256, 2, 32, 32), (airkv.FP8, 224, 5, 16, 32),
         (airkv.INT8, 64, 2, 16, 64), (airkv.BF16, 32, 1, 16, 32)]
FAR = [0, 1, 7, 4095, 131071, 10 ** 6 + 3, 2 ** 31 - 1, -1, -5000, -2 ** 31]


def _same_pages(pool, want, what=""):
    for x, y, name in zip(pool.snapshot(), want, ("K", "V", "K scales", "V scales")):
        if y is not None:
            x, y = (np.ascontiguousarray(z).view(np.uint8) for z in (x, y))
            assert np.array_equal(x, y), f"{what}: {name} differs at {np.argwhere(x != y)[:3].tolist()}"


def _host(pool):
    return oracle.HostPool(pool.num_blocks, pool.block_size, pool.n_kv_heads, pool.head_dim, KINDS[pool.dtype],
                           pool.scale_group or 32)


def _pages(host):
    return host.k, host.v, getattr(host, "k_scales", None), getattr(host, "v_scales", None)


def _dev(x):
    return torch_mod().from_numpy(np.ascontiguousarray(x)).cuda()


def _up(x, bf16):
    t = _dev(np.asarray(x, np.float32))
    return t.to(torch_mod().bfloat16) if bf16 else t


def _down(t):
    return t.float().cpu().numpy()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype,d,kv,bs,group", POOLS)
@pytest.mark.parametrize("rot", ["all", "half", "odd", "least"])
def test_append(dtype, d, kv, bs, group, pairs, rot, io):
    rot = {"all": d, "half": d // 2 // 8 * 8, "odd": max(8, (d // 8 - 1) * 8 // 16 * 16 - 8), "least": 8}[rot]
    torch = torch_mod()
    r = np.random.default_rng(rot + d)
    n, nq = 37, 3 * kv
    pool = airkv.KvPool(9, bs, kv, d, dtype, group)
    x = r.standard_normal((n, nq + 2 * kv, d)).astype(np.float32)
    x[3, nq, :] = 0.0                                      # a key and a value of zeros
    x[4, -1, :] = 0.0
    fused = _up(x, io == "bf16")
    x = _down(fused)
    q, k, v = fused.split([nq, kv, kv], dim=1)
    positions = np.resize(np.array(FAR), n).astype(np.int32)
    slots = r.permutation(9 * bs)[:n].astype(np.int64)
    slots[5] = -1
    f = ref.frequencies(rot)
    got = pool.append_rotary(q, k, v, _dev(slots), _dev(positions), _dev(f), interleaved=pairs, magnitude=1.125)
    assert got.dtype is fused.dtype and pool.error_count() == 0
    # the pages: bit for bit those of the turned rows, appended
    host = _host(pool)
    turned = ref.turned(x[:, :nq + kv], positions, f, pairs, 1.125)
    host.append(np.ascontiguousarray(turned[:, nq:]), np.ascontiguousarray(x[:, nq + kv:]), slots)
    _same_pages(pool, _pages(host))
    # the queries: to 64 bits.  c and s, two products and a sum: each term of two roundings,
    # |x c| + |y s| <= 1.125 * sqrt(2) * |(x, y)|, and the output's own
    want = ref.exact(x[:, :nq], positions, f, pairs, np.float32(1.125))
    a, b = ref._parts(rot, pairs)
    size = np.zeros_like(want)
    size[..., a] = size[..., b] = np.hypot(x[:, :nq][..., a], x[:, :nq][..., b])
    bound = 3 * F32_HALF_STEP * 1.125 * 2 ** 0.5 * size + (2.0 ** -8 if io == "bf16" else F32_HALF_STEP) * np.abs(want)
    assert (np.abs(_down(got) - want) <= bound * (1 + 1e-6)).all()
    want = ref.to_bf16(turned[:, :nq]) if io == "bf16" else turned[:, :nq].view(np.uint32)
    bits = got.view(torch.int16 if io == "bf16" else torch.int32).cpu().numpy().view(want.dtype)
    assert np.array_equal(bits, want)


@pytest.mark.parametrize("n,parts", [(1, 1), (1, 5), (700, 4)])
def test_append_outputs(n, parts):
    """Other output types, queries turned in place, no queries, one token and many."""
    torch = torch_mod()
    r = np.random.default_rng(n)
    kv, d, nq = 2, 96, 2 * parts
    f = ref.frequencies(48)
    x = r.standard_normal((n, nq + 2 * kv, d)).astype(np.float32)
    positions = r.integers(0, 100000, n).astype(np.int32)
    want = ref.turned(x[:, :nq], positions, f, False)
    host = None
    for bf16_in in (False, True):
        t = [z.contiguous() for z in _up(x, bf16_in).split([nq, kv, kv], dim=1)]
        base = _down(torch.cat(t, 1)) if bf16_in else x
        want = ref.turned(base[:, :nq], positions, f, False)
        for out in (torch.float32, torch.bfloat16, "in place", None):
            pool = airkv.KvPool(-(-n // 16), 16, kv, d, airkv.F32)
            q = None if out is None else t[0].clone()
            q_out = None if out is None else q if out == "in place" else torch.empty(n, nq, d, dtype=out, device="cuda")
            got = pool.append_rotary(q, t[1], t[2], torch.arange(n, device="cuda"), _dev(positions), _dev(f), q_out)
            host = _host(pool)
            host.append(ref.turned(base[:, nq:nq + kv], positions, f, False), np.ascontiguousarray(base[:, nq + kv:]), np.arange(n))
            _same_pages(pool, _pages(host), str(out))
            if out is None:
                assert got is None
                continue
            assert got is q_out
            if got.dtype is torch.float32:
                assert np.array_equal(got.cpu().numpy(), want)
            else:
                assert np.array_equal(got.view(torch.int16).cpu().numpy().view(np.uint16), ref.to_bf16(want))


def test_append_bad_slots_and_values():
    """Slots outside, and values that are not finite: each stays where it is."""
    torch = torch_mod()
    r = np.random.default_rng(5)
    pool = airkv.KvPool(2, 16, 2, 64, airkv.F32)
    n, f = 6, ref.frequencies(32)
    x = r.standard_normal((n, 6, 64)).astype(np.float32)
    x[0, 0, 3], x[1, 2, 40], x[2, 4, 5], x[2, 2, 20] = np.inf, np.nan, -np.inf, np.inf
    slots = np.array([0, 31, 7, -1, 32, 1 << 40], np.int64)
    positions = np.arange(n, dtype=np.int32)
    q, k, v = (z.contiguous() for z in _dev(x).split([2, 2, 2], dim=1))
    got = pool.append_rotary(q, k, v, _dev(slots), _dev(positions), _dev(f)).cpu().numpy()
    assert pool.error_count() == 2
    with np.errstate(invalid="ignore"):
        want = ref.turned(x[:, :4], positions, f, False)
    host = _host(pool)
    host.append(np.ascontiguousarray(want[:3, 2:]), np.ascontiguousarray(x[:3, 4:]), slots[:3])
    np.testing.assert_array_equal(got, want[:, :2])
    pk, pv = pool.snapshot()[:2]
    np.testing.assert_array_equal(pk, host.k)
    np.testing.assert_array_equal(pv, host.v)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.F32, airkv.INT8, airkv.FP8])
def test_values_are_appends(dtype):
    """Values (and what of keys does not turn) are stored as append stores them, whatever they are:
    NaN of any payload, infinities, subnormals, halfway cases."""
    torch = torch_mod()
    r = np.random.default_rng(1)
    n, d = 64, 64
    bits = r.integers(0, 1 << 32, (n, 2, d), np.uint64).astype(np.uint32)
    bits[0::4] |= 0x7F800000
    bits[1::4] &= 0x807FFFFF
    bits[2::4, :, ::2] = (bits[2::4, :, ::2] & 0xFFFF0000) | 0x8000
    x = _dev(bits.view(np.float32))
    two = [airkv.KvPool(n // 16, 16, 2, d, dtype) for _ in range(2)]
    slots = torch.arange(n, device="cuda")
    f = _dev(ref.frequencies(8))
    two[0].append(x, x, slots)
    two[1].append_rotary(None, x, x, slots, torch.zeros(n, dtype=torch.int32, device="cuda"), f)
    a, b = two[0].snapshot(), two[1].snapshot()
    assert np.array_equal(a[1].view(np.uint8), b[1].view(np.uint8))
    if a[3] is not None:
        assert np.array_equal(a[3].view(np.uint32), b[3].view(np.uint32))
    assert np.array_equal(a[0][..., 32:].view(np.uint8), b[0][..., 32:].view(np.uint8))


# ---- rotate -----------------------------------------------------------------

def _filled(dtype, d, kv, bs, group, lens, seed, spare=2):
    """A pool of appended normal rows in blocks of random order, and the host's copy."""
    r = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    nb = -(-lens // bs)
    pool = airkv.KvPool(int(nb.sum()) + spare, bs, kv, d, dtype, group)
    host = _host(pool)
    rows = r.standard_normal((2, pool.num_blocks * bs, kv, d)).astype(np.float32)
    slots = np.arange(pool.num_blocks * bs)
    host.append(rows[0], rows[1], slots)
    pool.append(_dev(rows[0]), _dev(rows[1]), _dev(slots.astype(np.int64)))
    perm = r.permutation(pool.num_blocks).astype(np.int32)
    tables = np.full((len(lens), max(1, int(nb.max(initial=0)))), -1, np.int32)
    at = 0
    for i, n in enumerate(nb):
        tables[i, :n] = perm[at:at + n]
        at += n
    return pool, host, tables, lens, r


def _values(pool, host):
    """K pages as f32 [blocks, kv, bs, d]."""
    k = host.k
    if pool.dtype == airkv.F32:
        return k.copy()
    if pool.dtype == airkv.BF16:
        return (k.astype(np.uint32) << 16).view(np.float32)
    x = k.view(np.int8).astype(np.float32) if pool.dtype == airkv.INT8 else oracle.fp8_decode_table()[k]
    s = host.k_scales
    return (x.reshape(*s.shape, -1) * s[..., None]).reshape(x.shape)


def _rotated(pool, host, tables, lens, froms, tos, f, pairs):
    """The host's K pages after the rotation of every sequence."""
    x = _values(pool, host)
    bs, g = pool.block_size, pool.scale_group
    for row, n, was, to in zip(tables, lens.tolist(), froms, tos):
        at = np.arange(n)[np.asarray(to)[:n] != np.asarray(was)[:n]]
        if not len(at):
            continue
        blocks, off = row[at // bs], at % bs
        by = np.asarray(to, np.int64)[at] - np.asarray(was, np.int64)[at]
        y = ref.turned(x[blocks, :, off], by, f, pairs)
        one = _host(pool)
        slots = blocks.astype(np.int64) * bs + off
        one.append(y, np.zeros_like(y), slots)
        whole = pool.head_dim
        if airkv.INT8 <= pool.dtype:
            whole = -(-2 * len(f) // g) * g
            host.k_scales[blocks, :, off, :whole // g] = one.k_scales[blocks, :, off, :whole // g]
        host.k[blocks, :, off, :whole] = one.k[blocks, :, off, :whole]


def _call(pool, tables, froms, f, pairs, tos=None):
    cu = np.concatenate([[0], np.cumsum([len(x) for x in froms])]).astype(np.int32)
    flat = [np.concatenate([np.asarray(x, np.int32) for x in z] + [np.zeros(0, np.int32)]) for z in (froms, tos or froms)]
    pool.rotate(_dev(tables), _dev(flat[0]), _dev(cu), _dev(f), to_pos=None if tos is None else _dev(flat[1]), interleaved=pairs)


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rot", ["all", "odd", "least"])
@pytest.mark.parametrize("dtype,d,kv,bs,group", POOLS)
def test_rotate(dtype, d, kv, bs, group, rot, pairs):
    rot = {"all": d, "odd": max(8, (d // 8 - 1) * 8 // 16 * 16 - 8), "least": 8}[rot]
    pool, host, tables, lens, r = _filled(dtype, d, kv, bs, group, [1, 16, 0, 517, 33, 100], seed=d + rot)
    f = ref.frequencies(rot)
    froms = [np.sort(r.permutation(3 * n + 1)[:n]) for n in lens]
    froms[3][:40] = np.arange(40)                           # two runs and a half that stay
    _rotated(pool, host, tables, lens, froms, [np.arange(n) for n in lens], f, pairs)
    _call(pool, tables, froms, f, pairs)
    _same_pages(pool, _pages(host))
    # and to places of the caller's choice, back and beyond
    tos = [x + int(r.integers(-5, 90000)) for x in froms]
    _rotated(pool, host, tables, lens, froms, tos, f, pairs)
    _call(pool, tables, froms, f, pairs, tos)
    _same_pages(pool, _pages(host), "to")
    assert pool.error_count() == 0


@pytest.mark.parametrize("batch,n", [(1, 20000), (300, 40), (1, 1)])
def test_rotate_batches(batch, n):
    r = np.random.default_rng(batch)
    pool, host, tables, lens, r = _filled(airkv.BF16, 64, 2, 16, 32, r.integers(1, n + 1, batch), seed=n)
    f = ref.frequencies(64)
    froms = [np.arange(m) + 3 for m in lens]
    _rotated(pool, host, tables, lens, froms, [np.arange(m) for m in lens], f, False)
    _call(pool, tables, froms, f, False)
    _same_pages(pool, _pages(host))


def test_rotate_outside():
    """Ranges, tables and blocks outside: left alone, counted."""
    pool, host, tables, lens, r = _filled(airkv.F32, 32, 2, 16, 32, [40, 40, 40, 20], seed=9)
    f = ref.frequencies(32)
    tables[1, 1] = pool.num_blocks                          # 16 tokens
    tables[2, 0] = -1                                       # 16 tokens
    froms = [np.arange(60) + 1, np.arange(40) + 1, np.arange(40) + 1]    # 60: twelve more than the table's 48
    cu = np.array([0, 60, 100, 140, 141], np.int32)         # the last one ends outside
    tos = [np.arange(48), np.r_[np.arange(16), np.arange(16) + 17, np.arange(8) + 32], np.r_[np.arange(16) + 1, np.arange(24) + 16]]
    tables[0, 2] = tables[0, 2] if tables[0, 2] >= 0 else 0
    flat = np.concatenate(froms).astype(np.int32)
    _rotated(pool, host, tables, np.array([48, 40, 40]), [x[:48] for x in froms], tos, f, False)
    pool.rotate(_dev(tables), _dev(flat), _dev(cu), _dev(f))
    _same_pages(pool, _pages(host))
    assert pool.error_count() == 12 + 16 + 16 + 1


# ---- refusals ----------------------------------------------------------------

def _refused(fn, kind=airkv.AirKvError):
    with pytest.raises(kind):
        fn()


def test_refusals():
    """Nothing is launched on arguments that the kernels do not take."""
    torch = torch_mod()
    n, kv, d, nq = 3, 2, 64, 4
    pool = airkv.KvPool(2, 16, kv, d, airkv.F32)
    x = torch.randn(n, nq + 2 * kv, d, device="cuda")
    q, k, v = (z.contiguous() for z in x.split([nq, kv, kv], dim=1))
    slots, pos = torch.arange(n, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    f = _dev(ref.frequencies(64))

    def call(**over):
        a = dict(q=q, k=k, v=v, slot_mapping=slots, positions=pos, inv_freq=f, q_out=None)
        a.update(over)
        return lambda: pool.append_rotary(**a)
    for bad in (dict(inv_freq=_dev(ref.frequencies(64)[:6 // 2])), dict(inv_freq=_dev(ref.frequencies(128))),
                dict(inv_freq=f[:0]), dict(magnitude=float("nan")), dict(magnitude=float("inf")),
                dict(q_out=x.view(-1)[:n * nq * d].view(n, nq, d), k=x[:, nq:nq + kv]),              # overlaps k
                dict(q=x[:, :nq], q_out=x.view(-1)[:n * nq * d].view(n, nq, d)),                     # in place, not dense
                dict(q_out=q.view(-1).view(torch.bfloat16)[:n * nq * d].view(n, nq, d)),             # in place, another type
                dict(k=torch.randn(n * kv * d + 2, device="cuda")[2:].view(n, kv, d))):              # not 16-byte aligned
        _refused(call(**bad))
    for bad in (dict(v=v.bfloat16()), dict(q=q.half()), dict(k=k.cpu()), dict(positions=pos.long()), dict(slot_mapping=pos)):
        _refused(call(**bad), TypeError)
    for bad in (dict(k=k[:2]), dict(q=q[:, :, :32]), dict(v=v.transpose(0, 1).contiguous().transpose(0, 1)), dict(q=None, q_out=q),
                dict(positions=pos[:2]), dict(q_out=torch.empty(n, nq, d + 32, device="cuda")), dict(stream=torch.cuda.Stream())):
        _refused(call(**bad), ValueError)
    lib = airkv.load()
    args = [pool.handle, 0, q.data_ptr(), nq * d, nq, k.data_ptr(), kv * d, v.data_ptr(), kv * d, 0, slots.data_ptr(), pos.data_ptr(), n,
            f.data_ptr(), 64, 0, 1.0, torch.empty_like(q).data_ptr(), 0]
    for i, value in ((3, nq * d - 4), (3, nq * d + 1), (4, -1), (4, 70000), (5, None), (6, kv * d - 64), (9, 2), (10, None), (11, None), (12, -1),
                     (13, None), (14, 12), (14, 72), (14, 0), (15, 2), (17, None), (18, 3), (2, None)):
        bad = list(args)
        bad[i] = value
        assert lib.air_kv_append_rotary(*bad) == airkv.AIR_KV_E_INVALID_ARG, (i, value)
    tables, cu = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    args = [pool.handle, 0, tables.data_ptr(), 1, 2, pos.data_ptr(), None, cu.data_ptr(), 3, f.data_ptr(), 64, 0]
    for i, value in ((2, None), (3, -1), (3, 1 << 21), (4, 0), (5, None), (7, None), (8, -1), (9, None), (10, 4), (10, 128), (11, -1)):
        bad = list(args)
        bad[i] = value
        assert lib.air_kv_rotate(*bad) == airkv.AIR_KV_E_INVALID_ARG, (i, value)
    _refused(lambda: pool.rotate(tables, pos, cu[:1], f), ValueError)
    _refused(lambda: pool.rotate(tables, pos.long(), cu, f), TypeError)
    _refused(lambda: pool.rotate(tables, pos, cu, f, to_pos=pos[:2]), ValueError)
    # nothing to do is no error
    assert pool.append_rotary(q[:0], k[:0], v[:0], slots[:0], pos[:0], f).shape == (0, nq, d)
    pool.rotate(tables[:0], pos[:0], cu[:1], f)
    pool.rotate(tables, pos[:0], cu, f)
    torch.cuda.synchronize()
    assert pool.error_count() == 0 and not pool.snapshot()[0].any()
