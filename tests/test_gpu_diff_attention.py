"""Differential attention over the paged cache (air_paged_diff_decode,
air_paged_diff_prefill) against 64 bits, on pools whose other rows hold values that
are not finite."""
import numpy as np
import pytest

import airkv
from diff_ref import attend, check, pool_values, sequence
from gpu_helpers import log, torch_mod

pytestmark = pytest.mark.gpu

NAMES = {airkv.F32: "f32", airkv.BF16: "bf16", airkv.INT8: "int8", airkv.FP8: "fp8"}


def _poison(pool):
    """Every row of the pool: not finite."""
    n = pool.num_blocks
    raw = np.zeros((n, pool.block_bytes), np.uint8)
    pages = raw[:, :2 * pool.slab_bytes]
    if pool.dtype == airkv.F32:
        pages[:] = np.full(pages.shape[1] // 4, np.nan, np.float32).view(np.uint8)
    elif pool.dtype == airkv.BF16:
        pages[:] = np.full(pages.shape[1] // 2, 0x7F80, np.uint16).view(np.uint8)
    else:
        pages[:] = 0x7F
        raw[:, 2 * pool.slab_bytes:].view(np.float32)[:] = np.inf
    pool.write_blocks(np.arange(n, dtype=np.int32), raw)


class Cache:
    """A pool with sequences of `lens` tokens in blocks of random order."""

    def __init__(self, dtype, d, kv, bs, lens, seed, scale_group=32, spare=3, grow=0):
        torch = torch_mod()
        r = np.random.default_rng(seed)
        self.lens = np.asarray(lens, np.int32)
        nb = -(-(self.lens + grow) // bs)
        total = int(nb.sum()) + spare
        self.pool = airkv.KvPool(total, bs, kv, d, dtype, scale_group)
        _poison(self.pool)
        perm = r.permutation(total).astype(np.int32)
        self.tables = np.full((len(lens), max(1, int(nb.max()) + 1)), -1, np.int32)
        slots, at = [], 0
        for i, n in enumerate(nb):
            self.tables[i, :n] = perm[at:at + n]
            at += n
            pos = np.arange(self.lens[i])
            slots.append(self.tables[i, pos // bs].astype(np.int64) * bs + pos % bs)
        slots = np.concatenate(slots)
        self.k, self.v = (r.standard_normal((len(slots), kv, d)).astype(np.float32) for _ in range(2))
        if len(slots):
            self.pool.append(*(torch.from_numpy(x).cuda() for x in (self.k, self.v, slots)))
        self.r, self.bs, self.d, self.kv = r, bs, d, kv

    def rows(self, n, group, q_f32, lam_rows, norm):
        """(q, lam, norm_weight) on the device and as float64."""
        torch = torch_mod()
        pairs = self.kv // 2 * group
        q = torch.from_numpy(self.r.standard_normal((n, 2 * pairs, self.d)).astype(np.float32)).cuda()
        q = q if q_f32 else q.to(torch.bfloat16)
        lam = self.r.uniform(-0.5, 1.0, (n, pairs) if lam_rows else (pairs,)).astype(np.float32)
        w = self.r.uniform(0.5, 1.5, 2 * self.d).astype(np.float32) if norm else None
        wide = np.broadcast_to(lam.astype(np.float64), (n, pairs))
        return (q, torch.from_numpy(lam).cuda(), None if w is None else torch.from_numpy(w).cuda(),
                q.float().cpu().numpy().astype(np.float64), wide, None if w is None else w.astype(np.float64))

    def device(self):
        torch = torch_mod()
        return torch.from_numpy(self.tables).cuda(), torch.from_numpy(self.lens).cuda()


def _decode(c, group, q_f32, out_f32, norm, lam_rows, splits=(64,), out_scale=0.75):
    torch = torch_mod()
    n = len(c.lens)
    q, lam, w, q64, lam64, w64 = c.rows(n, group, q_f32, lam_rows, norm)
    more = {"norm_weight": w64, "norm_eps": 1e-5 if norm else None, "out_scale": out_scale}
    kv, vv = pool_values(c.pool)
    want, bound = np.zeros((n, lam64.shape[1], 2 * c.d)), np.zeros((n, lam64.shape[1], 2 * c.d))
    scale = float(np.float32(1.0) / np.sqrt(np.float32(c.d)))
    for i, m in enumerate(c.lens):
        k, v = (sequence(x, c.tables[i], int(m), c.bs) for x in (kv, vv))
        want[i:i + 1], bound[i:i + 1] = attend(q64[i:i + 1], k, v, lam64[i:i + 1], scale, [m - 1], **more)
    tables, lens = c.device()
    used = 0.0
    for s in splits:
        out = torch.full((n, lam64.shape[1], 2 * c.d), float("nan"), device="cuda",
                         dtype=torch.float32 if out_f32 else torch.bfloat16)
        c.pool.paged_diff_decode(q, lam, tables, lens, out, norm_weight=w, norm_eps=more["norm_eps"], out_scale=out_scale,
                                 max_splits=s)
        used = max(used, check(out.float().cpu().numpy(), want, bound, airkv.F32 if out_f32 else airkv.BF16, f"splits {s}"))
    assert c.pool.error_count() == 0
    return used


LENS = [0, 1, 15, 16, 17, 31, 33, 64, 1040, 255, 0, 700]


@pytest.mark.parametrize("d,kv,group,bs,scale_group", [(64, 8, 1, 16, 32), (128, 4, 4, 16, 32), (128, 2, 8, 32, 32), (32, 2, 3, 16, 8),
                                                       (96, 6, 2, 32, 32), (96, 2, 11, 16, 16), (128, 2, 17, 16, 64), (64, 16, 7, 32, 8)])
@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16, airkv.INT8, airkv.FP8])
def test_diff_decode(dtype, d, kv, group, bs, scale_group):
    for i, (q_f32, out_f32, norm, lam_rows) in enumerate([(True, True, True, False), (False, True, False, True),
                                                          (False, False, True, True)]):
        c = Cache(dtype, d, kv, bs, LENS, seed=d + group + i, scale_group=scale_group)
        used = _decode(c, group, q_f32, out_f32, norm, lam_rows, splits=(64, 1, 7, 256))
        log(f"diff decode {NAMES[dtype]} d={d} group={group} q_f32={q_f32} out_f32={out_f32}: {used:.3f} of the bound")


@pytest.mark.parametrize("batch,lens", [(1, [1]), (1, [5000]), (3, [1, 9000, 40]), (257, None), (300, None), (4100, None)])
def test_diff_decode_batches(batch, lens):
    lens = [(11 * i) % 47 for i in range(batch)] if lens is None else lens
    c = Cache(airkv.BF16, 64, 2, 16, lens, seed=batch)
    log(f"diff decode batch {batch}: {_decode(c, 2, False, True, True, True, splits=(64, 3)):.3f} of the bound")


def _prefill(c, qlens, group, q_f32, out_f32, norm, lam_rows, out_scale=0.75, ws=None, p_step=0.0, floor=0.0):
    torch = torch_mod()
    cu = np.concatenate([[0], np.cumsum(qlens)]).astype(np.int32)
    total = int(cu[-1])
    q, lam, w, q64, lam64, w64 = c.rows(total, group, q_f32, lam_rows, norm)
    more = {"norm_weight": w64, "norm_eps": 1e-5 if norm else None, "out_scale": out_scale}
    kv, vv = pool_values(c.pool)
    want, bound = np.zeros((total, lam64.shape[1], 2 * c.d)), np.zeros((total, lam64.shape[1], 2 * c.d))
    scale = float(np.float32(1.0) / np.sqrt(np.float32(c.d)))
    for i, (m, ql) in enumerate(zip(c.lens, qlens)):
        k, v = (sequence(x, c.tables[i], int(m), c.bs) for x in (kv, vv))
        s = slice(cu[i], cu[i + 1])
        want[s], bound[s] = attend(q64[s], k, v, lam64[s], scale, m - ql + np.arange(ql), p_step=p_step, **more)
        bound[s] += floor * out_scale * (1 + np.abs(lam64[s]).max(initial=0)) * np.abs(v).max(initial=0)
    tables, lens = c.device()
    out = torch.full((total, lam64.shape[1], 2 * c.d), float("nan"), device="cuda",
                     dtype=torch.float32 if out_f32 else torch.bfloat16)
    c.pool.paged_diff_prefill(q, lam, torch.from_numpy(cu).cuda(), tables, lens, out, norm_weight=w, norm_eps=more["norm_eps"],
                              out_scale=out_scale, workspace=ws)
    used = check(out.float().cpu().numpy(), want, bound, airkv.F32 if out_f32 else airkv.BF16, "prefill", p_step)
    assert c.pool.error_count() == 0
    return used


# (cached, of them new) of each sequence
CHUNKS = [(1, 1), (40, 33), (0, 0), (300, 17), (128, 128), (65, 64), (700, 1), (33, 32), (90, 0), (257, 250)]


def _p_step(c):
    """What the 16-bit products add to a probability's relative error: the probability
    and the value (of 1-byte pages) are rounded to 11 bits, and so are the keys of
    1-byte pages, whose scores err by 2^-11 sum |q k| scale (taken at 8 standard
    deviations of normal rows: sum |q k| / sqrt(d) <= 2/pi sqrt(d) + 8), which moves a
    probability by twice that (its own score, and the sum's).  Below f16's normal
    numbers, 2^-14, a probability errs by 2^-25 of the largest.  Where a block of rows is
    cut, each piece's means, at most its sum of p |v| in size, are rounded to 11 bits too:
    another 2^-11 of the whole."""
    if c.pool.dtype == airkv.F32:
        return 0.0
    tiny = 2.0 ** -25 * c.lens.max(initial=1)
    if c.pool.dtype == airkv.BF16:
        return 2.0 ** -11 * 2 + tiny
    return 2.0 ** -11 * (3 + 2 * (0.64 * c.d ** 0.5 + 8)) + tiny


@pytest.mark.parametrize("d,kv,group,bs,scale_group", [(64, 8, 1, 16, 32), (128, 4, 4, 16, 32), (128, 2, 8, 32, 32), (32, 2, 3, 16, 8),
                                                       (96, 6, 2, 32, 32), (96, 2, 11, 16, 16), (128, 2, 70, 16, 64), (64, 2, 7, 32, 8)])
@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16, airkv.INT8, airkv.FP8])
def test_diff_prefill(dtype, d, kv, group, bs, scale_group):
    for i, (q_f32, out_f32, norm, lam_rows) in enumerate([(True, True, True, False), (False, True, False, True),
                                                          (True, False, True, False), (False, False, True, True)]):
        c = Cache(dtype, d, kv, bs, [n for n, _ in CHUNKS], seed=d + group + i, scale_group=scale_group)
        used = _prefill(c, [m for _, m in CHUNKS], group, q_f32, out_f32, norm, lam_rows,
                        p_step=0.0 if q_f32 or out_f32 else _p_step(c))
        log(f"diff prefill {NAMES[dtype]} d={d} group={group} q_f32={q_f32} out_f32={out_f32}: {used:.3f} of the bound")


@pytest.mark.parametrize("chunks", [[(1, 1)], [(3000, 3000)], [(9000, 5)], [(2500, 700), (1, 1)], [(3, 3)] * 40, [(20, 2)] * 1030])
def test_diff_prefill_shapes(chunks):
    for dtype, d, group, f32 in ((airkv.BF16, 64, 2, True), (airkv.F32, 32, 1, True), (airkv.BF16, 128, 3, False),
                                 (airkv.INT8, 64, 1, False)):
        c = Cache(dtype, d, 2, 16, [n for n, _ in chunks], seed=len(chunks) + d)
        used = _prefill(c, [m for _, m in chunks], group, f32, f32, True, True, p_step=0.0 if f32 else _p_step(c))
        log(f"diff prefill {len(chunks)} x {chunks[0]} {NAMES[dtype]}: {used:.3f} of the bound")


def _refill(c, k_mul, v_mul):
    """The cache's rows again, times a factor per token."""
    torch = torch_mod()
    slots = np.concatenate([c.tables[i, np.arange(n) // c.bs].astype(np.int64) * c.bs + np.arange(n) % c.bs
                            for i, n in enumerate(c.lens)])
    f = [np.concatenate([m(np.arange(n)) * np.ones(n) for n in c.lens]).astype(np.float32)[:, None, None] for m in (k_mul, v_mul)]
    c.pool.append(*(torch.from_numpy((x * y).astype(np.float32)).cuda() for x, y in zip((c.k, c.v), f)), torch.from_numpy(slots).cuda())


@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16, airkv.INT8, airkv.FP8])
@pytest.mark.parametrize("case", ["tiny", "huge", "growing", "falling", "far_apart", "keys_tiny", "keys_growing"])
def test_diff_value_ranges(dtype, case):
    """Values and keys far from 1, and ones whose size changes along the sequence, in
    decode and prefill at f32 and at 16-bit products.  (Outputs are not normalised, so
    each row's error is held to its own values' size.)"""
    one = lambda t: 1.0
    k_mul, v_mul = {
        "tiny": (one, lambda t: 1e-30), "huge": (one, lambda t: 1e30), "growing": (one, lambda t: 2.0 ** (t / 12 - 20)),
        "falling": (one, lambda t: 2.0 ** (20 - t / 12)), "far_apart": (one, lambda t: np.where(t % 70 < 35, 1e12, 1e-3)),
        "keys_tiny": (lambda t: 1e-6, one), "keys_growing": (lambda t: 2.0 ** (t / 40 - 12), one)}[case]
    for f32 in (True, False):
        c = Cache(dtype, 64, 2, 16, [500, 130, 33], seed=3)
        _refill(c, k_mul, v_mul)
        # a value far below the block's largest keeps f16's absolute resolution: 2^-25 of it
        wide = dtype != airkv.F32 and not f32
        used = _prefill(c, [400, 5, 33], 2, f32, f32, False, True, p_step=_p_step(c) if wide else 0.0, floor=2.0 ** -24 if wide else 0.0)
        more = _decode(c, 2, f32, f32, False, True, splits=(64, 1))
        log(f"diff {case} {NAMES[dtype]} f32={f32}: prefill {used:.3f}, decode {more:.3f} of the bound")


@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16, airkv.INT8, airkv.FP8])
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_diff_prefill_hidden_values_that_are_not_finite(dtype, f32, bad):
    """Keys and values that are not finite at tokens a row does not see do not reach
    it; rows that see them are not finite in those columns."""
    torch = torch_mod()
    n, first, at = 200, 100, [130, 131, 171, 199]
    c = Cache(dtype, 64, 4, 16, [n, n], seed=9)
    row = c.tables[0]
    clean = None
    q, lam, _, _, _, _ = c.rows(2 * (n - first), 3, f32, False, False)
    cu = torch.tensor([0, n - first, 2 * (n - first)], dtype=torch.int32, device="cuda")
    tables, lens = c.device()
    out = torch.empty(q.shape[0], 6, 128, device="cuda", dtype=torch.float32 if f32 else torch.bfloat16)
    for step in range(2):
        c.pool.paged_diff_prefill(q, lam, cu, tables, lens, out.fill_(7.0))
        got = out.float().cpu().numpy()
        if clean is None:
            clean = got
            assert np.isfinite(clean).all()
            # one column of head 1 and the whole of head 3's group of 32, of four tokens of sequence 0
            x = torch.from_numpy(c.v[:n][at].copy()).cuda()
            x[:, 1, 5] = bad
            x[:, 3, 32:64] = bad
            k = torch.from_numpy(c.k[:n][at].copy()).cuda()
            k[2, 0, 7] = bad                                # token 171
            slots = torch.from_numpy(np.array([int(row[t // 16]) * 16 + t % 16 for t in at], np.int64)).cuda()
            c.pool.append(k, x, slots)
    r = n - first
    assert np.array_equal(got[r:], clean[r:])               # the other sequence
    assert np.array_equal(got[:at[0] - first], clean[:at[0] - first])
    after = got[at[0] - first:r]
    if dtype in (airkv.INT8, airkv.FP8):
        return                                              # what a pool stores for such a group is its own rule
    assert not np.isfinite(after[:, :3, 64 + 5]).any() and not np.isfinite(after[:, 3:, 64 + 32:]).any()
    same = after[:at[2] - at[0]]                            # rows that see no bad key: other columns as they were
    ref = clean[at[0] - first:at[2] - first]
    assert np.array_equal(same[:, :3, :64], ref[:, :3, :64]) and np.array_equal(same[:, 3:, :64], ref[:, 3:, :64])
