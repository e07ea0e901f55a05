"""The norm of cross attention's error against 64 bits: every kind of product, few rows and many."""
import pytest

import airkv
import cross_precision
from gpu_helpers import torch_mod
from test_gpu_cross import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", ["few", "many"])
@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.INT8, airkv.FP8])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 256])
def test_16_bit_products(d, dtype, rows):
    c = Case(dtype, d, 2, 4, 16, [2000, 333], [3, 2] if rows == "few" else [150, 90], seed=d)
    out = c.call(max_q_len=int(c.rows.max())).cpu()
    want, _ = c.want()
    got, least = cross_precision.off(out, want), cross_precision.floor(want, torch_mod().bfloat16)
    print(f"{got:.3g}, its rounding {least:.3g}")
    assert got <= cross_precision.WITHIN * least


@pytest.mark.parametrize("rows", ["few", "many"])
@pytest.mark.parametrize("dtype,io", [(airkv.F32, "f32"), (airkv.BF16, "f32"), (airkv.INT8, "f32"), (airkv.FP8, "f32"), (airkv.BF16, "bf16")])
@pytest.mark.parametrize("d", [32, 64, 128, 224])
def test_f32_precision(d, dtype, io, rows):
    c = Case(dtype, d, 2, 2, 16, [2000, 333], [3, 2] if rows == "few" else [150, 90], io, "f32", seed=d)
    got = cross_precision.off(c.call(max_q_len=int(c.rows.max())).cpu(), c.want()[0])
    print(f"2^{torch_mod().tensor(got).log2():.2f}")
    assert got <= cross_precision.F32


SIZES = {"tiny": lambda t: 1e-30, "small": lambda t: 1e-6, "large": lambda t: 1e5, "huge": lambda t: 1e30,
         # beyond f16 behind a first token's size, once and from there on; behind zeros; far below it
         "one": lambda t: 3e5 if t == 150 else 1.0, "grows": lambda t: 10.0 ** (t // 40), "zeros": lambda t: 0.0 if t < 100 else 1e8,
         "falls": lambda t: 10.0 ** -(t // 60)}


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("d,rows", [(64, 200), (128, 300), (96, 2), (160, 90)])
def test_values_of_many_sizes(d, rows, size):
    """bf16 pages: values are f16 in some products."""
    torch = torch_mod()
    c = Case(airkv.BF16, d, 2, 2, 16, [300, 61, 200], [rows, 3, rows // 2 + 1], seed=d + 1)
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i, n in enumerate(c.lens.tolist()):
        k, v = (torch.randn(n, 2, d, generator=gen, device="cuda") for _ in range(2))
        at = torch.arange(n)
        slots = torch.from_numpy(c.tables[i].astype("int64"))[at // 16] * 16 + at % 16
        c.pool.append(k, v * torch.tensor([SIZES[size](t) for t in range(n)], dtype=torch.float32, device="cuda")[:, None, None], slots.cuda())
    # blocks outside the pool are counted once, however often a block of rows is computed
    c.tables[0, 2], c.tables[2, 0] = -1, c.pool.num_blocks
    c.check(size, errors=2, max_q_len=rows)
    out, (want, _) = c.out.cpu(), c.want()
    for i in range(3):                                 # (no sequence's errors hide behind another's)
        at = slice(int(c.cu[i]), int(c.cu[i + 1]))
        got, least = cross_precision.off(out[at], want[at]), cross_precision.floor(want[at], torch.bfloat16)
        print(f"{got:.3g}, its rounding {least:.3g}")
        assert got <= cross_precision.WITHIN * least
