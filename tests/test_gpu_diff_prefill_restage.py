"""Differential prefill with 16-bit products: tiles that have to be staged again under
another power of two, wherever they lie in a workgroup's run of tiles."""
import numpy as np
import pytest

import airkv
from diff_ref import attend, check, pool_values, sequence
from gpu_helpers import log, torch_mod
from test_gpu_diff_attention import Cache, _p_step

pytestmark = pytest.mark.gpu

KV, D, BS, TILE = 256, 32, 16, 32                      # 128 pairs: two workgroups a pair, long runs of tiles
PAIRS = [0, 63, 127]                                   # compared with 64 bits (the others: with the f32-precision kernel)


def _run(c, new, q, lam, f32):
    torch = torch_mod()
    cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    tables, lens = c.device()
    x = q.float() if f32 else q
    out = torch.empty(new, KV // 2, 2 * D, device="cuda", dtype=x.dtype)
    c.pool.paged_diff_prefill(x, lam, cu, tables, lens, out, max_q_len=new, out_scale=0.75)
    return out.float().cpu().numpy()


def _outlier(c, token, k_mul, v_mul):
    """Token's rows of sequence 0 again, times k_mul and v_mul."""
    torch = torch_mod()
    slot = torch.tensor([int(c.tables[0, token // BS]) * BS + token % BS], dtype=torch.int64, device="cuda")
    c.pool.append(torch.from_numpy(c.k[token:token + 1] * np.float32(k_mul)).cuda(),
                  torch.from_numpy(c.v[token:token + 1] * np.float32(v_mul)).cuda(), slot)


def _expect(c, n, new, q, lam, p_step):
    """The rows of PAIRS in 64 bits: (out, bound)."""
    heads = np.array([h for p in PAIRS for h in (2 * p, 2 * p + 1)])
    k, v = (sequence(x[:, heads], c.tables[0], n, BS) for x in pool_values(c.pool))
    q64 = q.float().cpu().numpy().astype(np.float64)[:, heads]
    lam64 = np.broadcast_to(lam.cpu().numpy().astype(np.float64)[PAIRS], (new, len(PAIRS)))
    scale = float(np.float32(1.0) / np.sqrt(np.float32(D)))
    want, bound = attend(q64, k, v, lam64, scale, n - new + np.arange(new), out_scale=0.75, p_step=p_step)
    # a value far below the block's largest keeps f16's absolute resolution
    return want, bound + 2.0 ** -24 * 0.75 * (1 + np.abs(lam64).max()) * np.abs(v).max()


@pytest.mark.parametrize("dtype,what", [(airkv.BF16, "values"), (airkv.INT8, "values"), (airkv.FP8, "values"), (airkv.INT8, "keys"),
                                        (airkv.FP8, "keys")])
@pytest.mark.parametrize("tile", [62, 63, 64, 65, 127])
def test_a_tile_staged_again_keeps_its_tokens(dtype, what, tile):
    """One token whose values (or, on 1-byte pages, keys) leave the power of two that the
    tiles before it are under, in tiles around the ends of the table's windows of 64."""
    n, new = 9000, 4                                   # 282 tiles and 7 units: 145 to a workgroup
    c = Cache(dtype, D, KV, BS, [n], seed=40 + tile)
    q, lam, _, _, _, _ = c.rows(new, 1, False, False, False)
    keys = what == "keys"
    # 2^15 is where values of bf16 pages leave their first power of two, 8 times the first tile's where scales do
    _outlier(c, tile * TILE + 9, 20.0 if keys else 1.0, 1.0 if keys else 1e6)
    p_step = _p_step(c)
    if keys:                                           # its scores' own size: 20 times that of normal rows
        p_step += 2.0 ** -11 * 2 * 20 * (0.64 * D ** 0.5 + 8)
    want, bound = _expect(c, n, new, q, lam, p_step)
    got = _run(c, new, q, lam, False)
    used = check(got[:, PAIRS], want, bound, airkv.BF16, f"tile {tile}", p_step)
    if not keys:                                       # the token is most of the result: its loss would be seen
        assert np.linalg.norm(want) > 5 * np.linalg.norm(bound + 2.0 ** -8 * np.abs(want))
    f32 = _run(c, new, q, lam, True)
    rel = np.linalg.norm(got - f32) / np.linalg.norm(f32)
    assert rel <= p_step + 2.0 ** -8, rel
    assert c.pool.error_count() == 0
    log(f"staged again dtype={dtype} {what} tile={tile}: {used:.3f} of the bound, {rel:.2g} from f32 precision")


@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.INT8])
@pytest.mark.parametrize("tile,out", [(63, 64), (63, 63), (64, 64), (64, 65), (62, 64), (127, 128)])
def test_an_entry_outside_the_pool_is_counted_once(dtype, tile, out):
    """An entry outside the pool beside a tile that is staged again."""
    n, new = 9000, 4
    c = Cache(dtype, D, KV, BS, [n], seed=7)
    q, lam, _, _, _, _ = c.rows(new, 1, False, False, False)
    _outlier(c, tile * TILE + 9, 1.0, 1e6)
    c.tables[0, (out * TILE + 16) // BS] = -1          # not the outlier's block
    got = _run(c, new, q, lam, False)
    assert np.isfinite(got).all()
    assert c.pool.error_count(reset=True) == 1
