"""Cross attention over pages against the formula in 64 bits."""
import math

import numpy as np
import pytest

import airkv
import cross_ref
import oracle
from gpu_helpers import torch_mod

pytestmark = pytest.mark.gpu


def _dev(x):
    return torch_mod().from_numpy(np.ascontiguousarray(x)).cuda()


class Case:
    """A pool of appended rows in blocks of random order, and queries."""

    def __init__(self, dtype, d, kv, group, bs, lens, rows, io="bf16", out=None, scale_group=32, seed=0, size=1.0):
        torch = torch_mod()
        r = np.random.default_rng(seed)
        self.lens, self.rows = np.asarray(lens, np.int32), np.asarray(rows, np.int32)
        nb = -(-self.lens // bs)
        self.pool = airkv.KvPool(int(nb.sum()) + 3, bs, kv, d, dtype, scale_group)
        x = r.standard_normal((2, self.pool.num_blocks * bs, kv, d)).astype(np.float32) * size
        # (slices: a pool's tests are small, its append has its own)
        self.pool.append(_dev(x[0]), _dev(x[1]), torch.arange(self.pool.num_blocks * bs, device="cuda"))
        perm = r.permutation(self.pool.num_blocks).astype(np.int32)
        self.tables = np.full((len(lens), max(1, int(nb.max(initial=0)))), -1, np.int32)
        at = 0
        for i, n in enumerate(nb):
            self.tables[i, :n] = perm[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        self.io, self.out_io = io, out or io
        types = {"bf16": torch.bfloat16, "f32": torch.float32}
        q = r.standard_normal((int(self.rows.sum()), kv * group, d)).astype(np.float32)
        self.q = _dev(q).to(types[io])
        self.out = torch.full(self.q.shape, 7.0, dtype=types[self.out_io], device="cuda")
        self.bs, self.scale = bs, 1.0 / math.sqrt(d)
        self.precise = dtype == airkv.F32 or io == "f32" or self.out_io == "f32"
        self.byte = dtype in (airkv.INT8, airkv.FP8)

    def call(self, **more):
        more.setdefault("scale", self.scale)
        return self.pool.paged_cross(self.q, _dev(self.cu), _dev(self.tables), _dev(self.lens), self.out, **more)

    def want(self, scale=None):
        table = oracle.fp8_decode_table() if self.pool.dtype == airkv.FP8 else None
        k, v = cross_ref.values(self.pool, self.pool.snapshot(), self.pool.scale_group, table)
        return cross_ref.cross(self.q.double().cpu(), self.cu.tolist(), k, v, self.tables, self.lens.tolist(),
                               np.float32(self.scale if scale is None else scale).astype(np.float64).item(), self.bs, self.precise, self.byte,
                               self.out_io)

    def check(self, what="", errors=0, **more):
        out = self.call(**more).double().cpu()
        want, bound = self.want(more.get("scale"))
        off = (out - want).abs()
        worst = (off / bound.clamp(min=1e-300)).max()
        assert (off <= bound).all(), f"{what}: {float(worst)} of the bound at {np.argwhere((~(off <= bound)).numpy())[:3].tolist()}"
        assert self.pool.error_count() == errors
        return float(worst)


POOLS = [(airkv.BF16, 128, 32), (airkv.F32, 64, 32), (airkv.INT8, 128, 32), (airkv.FP8, 64, 32), (airkv.BF16, 64, 32), (airkv.F32, 128, 32),
         (airkv.INT8, 96, 8), (airkv.BF16, 32, 32), (airkv.F32, 96, 32), (airkv.FP8, 256, 256), (airkv.BF16, 256, 32), (airkv.F32, 256, 32),
         (airkv.INT8, 160, 16), (airkv.BF16, 192, 32), (airkv.F32, 224, 32), (airkv.FP8, 32, 8), (airkv.BF16, 160, 32), (airkv.F32, 192, 32),
         (airkv.INT8, 224, 32), (airkv.BF16, 96, 32), (airkv.F32, 32, 32), (airkv.F32, 160, 32), (airkv.BF16, 224, 32), (airkv.FP8, 192, 64)]
# rows and states: single tokens, beams, ragged prompts, more rows than states, sequences without either
RAGGED = ([1, 37, 0, 300, 16, 515, 33], [1, 40, 5, 3, 0, 70, 260])


@pytest.mark.parametrize("io,out", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("dtype,d,scale_group", POOLS)
def test_ragged(dtype, d, scale_group, io, out):
    c = Case(dtype, d, 2, 3, 16, *RAGGED, io=io, out=out, scale_group=scale_group, seed=d)
    for hint in (None, 260, 1):                        # the hint changes who takes which keys, not the result
        c.out.fill_(7.0)
        c.check(f"hint {hint}", max_q_len=hint)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dtype,d,scale_group", POOLS)
def test_single_tokens(dtype, d, scale_group, io):
    """One row a sequence: decode."""
    r = np.random.default_rng(d)
    c = Case(dtype, d, 3, 2, 32, r.integers(1, 700, 9), np.ones(9), io=io, scale_group=scale_group, seed=d + 1)
    c.check(max_q_len=1)


@pytest.mark.parametrize("kv,group", [(1, 1), (1, 40), (8, 1), (5, 7), (16, 4)])
@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.F32])
def test_heads(dtype, kv, group):
    c = Case(dtype, 64, kv, group, 16, [70, 129, 640], [9, 1, 33], io="f32" if dtype == airkv.F32 else "bf16", seed=kv)
    c.check(max_q_len=33)
    c.check(max_q_len=1)


@pytest.mark.parametrize("dtype,d,io", [(airkv.BF16, 128, "bf16"), (airkv.F32, 64, "f32"), (airkv.INT8, 64, "bf16")])
@pytest.mark.parametrize("n,rows", [(9000, 1), (9000, 33), (4096, 257)])
def test_long(dtype, d, io, n, rows):
    """Blocks that many slices hold."""
    c = Case(dtype, d, 2, 1, 16, [n], [rows], io=io, seed=rows)
    c.check(max_q_len=rows)
    c.check(max_q_len=0)


def test_batches():
    """More sequences than one launch takes, most of them without rows."""
    r = np.random.default_rng(1)
    lens, rows = r.integers(0, 40, 1500), r.integers(0, 3, 1500) * (r.random(1500) < 0.3)
    Case(airkv.BF16, 32, 1, 2, 16, lens, rows, seed=2).check(max_q_len=2)


def test_outside():
    """Refused sequences are counted and zeroed, blocks outside the pool left out, rows of no sequence left."""
    torch = torch_mod()
    c = Case(airkv.BF16, 64, 2, 2, 16, [100, 100, 70, 48, 20], [5, 6, 7, 3, 2], seed=4)
    c.q = torch.cat([c.q, torch.randn(4, 4, 64, device="cuda").bfloat16()])
    c.out = torch.full(c.q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    c.tables[0, 2] = -1
    c.tables[0, 6] = c.pool.num_blocks                 # (4 tokens of it are the sequence's)
    c.tables[3, :3] = -5                               # all of a sequence
    lens = c.lens.copy()
    lens[1], lens[2] = 16 * c.tables.shape[1] + 1, -1
    c.lens, true = lens, c.lens
    out = c.call(max_q_len=7).double().cpu()
    c.lens = np.where(lens == true, true, 0).astype(np.int32)
    want, bound = c.want()
    n = int(c.cu[-1])
    assert ((out - want).abs() <= bound)[:n].all() and (out[n:] == 7.0).all()
    assert (out[5:18] == 0).all() and (out[18:21] == 0).all()
    assert c.pool.error_count(reset=True) == 2 + 2 + 3
    # rows that do not lie in q
    c.lens, c.cu = true, np.array([0, 5, 11, 18, 40, 30], np.int32)
    c.out.fill_(7.0)
    out = c.call(max_q_len=7).double().cpu()
    assert (out[18:] == 7.0).all() and (out[:18] != 7.0).all()


@pytest.mark.parametrize("dtype,io", [(airkv.BF16, "bf16"), (airkv.F32, "f32"), (airkv.BF16, "f32")])
def test_behind_the_end(dtype, io):
    """What lies in a sequence's last block behind its end is not read."""
    c = Case(dtype, 64, 2, 2, 16, [1, 17, 250], [3, 40, 1], io=io, seed=6)
    want, bound = c.want()
    torch = torch_mod()
    bad = torch.full((16, 2, 64), math.nan, device="cuda")
    for i, n in enumerate(c.lens):
        blk, off = int(c.tables[i, (n - 1) // 16]), (n - 1) % 16 + 1
        if off < 16:
            slots = torch.arange(blk * 16 + off, blk * 16 + 16, device="cuda")
            c.pool.append(bad[off:].contiguous(), bad[off:].contiguous(), slots)
    for hint in (1, 40):
        assert ((c.call(max_q_len=hint).double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,io", [(airkv.BF16, "bf16"), (airkv.F32, "f32")])
@pytest.mark.parametrize("scale", [1e-30, 40.0, 3e4, 1e12])
def test_scales(dtype, io, scale):
    """From no preference at all to one key: scores past 2^20 keep their order."""
    c = Case(dtype, 64, 2, 2, 16, [40, 300], [20, 3], io=io, seed=7)
    if scale < 100:
        c.check(scale=scale, max_q_len=20)
        c.check(scale=scale, max_q_len=1)
        return
    out = {h: c.call(scale=scale, max_q_len=h).double().cpu() for h in (1, 20)}
    want, _ = c.want(scale)
    k, v = cross_ref.values(c.pool, c.pool.snapshot(), 0, None)
    for o in out.values():
        # a row's largest score is apart from the next by far more than its error: the key's values
        assert torch_mod().isfinite(o).all()
        near = (o - want).abs() <= 2.0 ** -6 * want.abs() + 1e-30
        assert near.double().mean() > 0.98


@pytest.mark.parametrize("dtype,io", [(airkv.BF16, "bf16"), (airkv.F32, "f32"), (airkv.INT8, "bf16")])
def test_large_values(dtype, io):
    """Values near the largest float: sums of many of them stay finite."""
    torch = torch_mod()
    c = Case(dtype, 64, 1, 1, 16, [700], [33], io=io, out="f32", seed=8)
    big = torch.full((c.pool.num_blocks * 16, 1, 64), 3.0e38, device="cuda")
    small = torch.randn(c.pool.num_blocks * 16, 1, 64, device="cuda")
    c.pool.append(small, big, torch.arange(c.pool.num_blocks * 16, device="cuda"))
    for hint in (1, 33):
        for c.out in (c.out, torch.empty_like(c.out, dtype=torch.bfloat16)):
            out = c.call(max_q_len=hint).float()
            assert torch.isfinite(out).all() and ((out / 3.0e38 - 1).abs() < 2.0 ** -7).all()


@pytest.mark.parametrize("dtype", [airkv.INT8, airkv.FP8])
@pytest.mark.parametrize("k_size,v_size", [(1.0, 1.0), (1e20, 1e30), (1e-20, 1e-30), (3e4, 3e-5), (1.0, 3e36), (1e-30, 1e-36)])
def test_codes_of_many_sizes(dtype, k_size, v_size):
    """16-bit products over 1-byte pages: tokens whose keys and values differ by powers of two, in
    units far from 1, rows of queries too; a token of zeros."""
    torch = torch_mod()
    c = Case(dtype, 64, 2, 2, 16, [700, 33, 9], [33, 3, 1], seed=11)
    n = c.pool.num_blocks * 16
    gen = torch.Generator(device="cuda").manual_seed(3)

    def rows(size, lo, hi):
        x = torch.randn(n, 2, 64, generator=gen, device="cuda")
        return x * torch.exp2(torch.randint(lo, hi + 1, (n, 1, 1), generator=gen, device="cuda").float()) * size
    k, v = rows(k_size, -9, 1), rows(v_size, -8, 4)
    k[5] = 0.0
    v[6] = 0.0
    c.pool.append(k, v, torch.arange(n, device="cuda"))
    c.q = (c.q.float() * torch.exp2(torch.arange(len(c.q), device="cuda").float() % 13 - 9)[:, None, None]).bfloat16()
    scale = c.scale / k_size
    for hint in (1, 33):
        c.out.fill_(7.0)
        c.check(f"hint {hint}", scale=scale, max_q_len=hint)


def test_not_finite():
    """A value that is not finite reaches its column only."""
    torch = torch_mod()
    c = Case(airkv.F32, 32, 1, 1, 16, [64, 64], [4, 4], io="f32", seed=9)
    k = torch.randn(1, 1, 32, device="cuda")
    v = torch.randn(1, 1, 32, device="cuda")
    v[0, 0, 5] = math.inf
    slot = torch.tensor([int(c.tables[0, 1]) * 16 + 3], device="cuda")
    c.pool.append(k, v, slot)
    out = c.call(max_q_len=4).cpu()
    bad = ~torch.isfinite(out)
    assert bad[:4, :, 5].all() and bad.sum() == 4


def test_refusals():
    torch = torch_mod()
    c = Case(airkv.BF16, 64, 2, 2, 16, [40], [3])
    tables, lens, cu = _dev(c.tables), _dev(c.lens), _dev(c.cu)

    def call(**over):
        a = dict(q=c.q, cu_q=cu, block_tables=tables, seq_lens=lens, out=c.out)
        a.update(over)
        return lambda: c.pool.paged_cross(**a)
    for bad, kind in ((dict(scale=0.0), airkv.AirKvError), (dict(scale=math.nan), airkv.AirKvError), (dict(scale=math.inf), airkv.AirKvError),
                      (dict(max_q_len=-1), airkv.AirKvError), (dict(workspace=torch.empty(64, device="cuda")), airkv.AirKvError),
                      (dict(q=c.q.view(3, 2, 128)), ValueError), (dict(q=c.q.half()), TypeError), (dict(out=c.out[:2]), ValueError),
                      (dict(cu_q=cu[:1]), ValueError), (dict(seq_lens=lens.long()), TypeError), (dict(q=c.q[:, :3].contiguous(), out=c.out[:, :3].contiguous()), airkv.AirKvError),
                      (dict(q=c.q.transpose(0, 1)), ValueError)):
        with pytest.raises(kind):
            call(**bad)()
    ws = c.pool.new_cross_workspace(4, 1, 3)
    args = [c.pool.handle, 0, c.q.data_ptr(), 1, 4, cu.data_ptr(), 3, 3, tables.data_ptr(), lens.data_ptr(), 1, 3, 0.125, ws.data_ptr(), ws.nbytes,
            c.out.data_ptr(), 1]
    lib = airkv.load()
    assert lib.air_paged_cross(*args) == airkv.AIR_KV_OK
    for i, value in ((2, None), (2, c.q.data_ptr() + 2), (3, 2), (4, 0), (4, 3), (5, None), (6, -1), (7, -1), (8, None), (9, None), (10, -1), (11, -1),
                     (11, 1 << 28), (12, -1.0), (13, None), (13, ws.data_ptr() + 8), (14, 64), (15, None), (15, c.out.data_ptr() + 4), (16, 5), (6, 2 ** 31 - 1)):
        bad = list(args)
        bad[i] = value
        assert lib.air_paged_cross(*bad) == airkv.AIR_KV_E_INVALID_ARG, (i, value)
    # nothing to do is no error
    c.pool.paged_cross(c.q[:0], cu, tables, lens, c.out[:0])
    c.pool.paged_cross(c.q[:0], cu[:1], tables[:0], lens[:0], c.out[:0])
    torch.cuda.synchronize()
