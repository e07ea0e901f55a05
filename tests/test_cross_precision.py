"""What cross_precision's limits let pass: the formula as the kernels compute it, and not with fewer bits."""
import math

import pytest
import torch

import cross_precision


def _parts(x, n):
    """x (f32) as n bf16 parts, cut off."""
    out = []
    for _ in range(n):
        p = (x.view(torch.int32) & -65536).view(torch.float32)
        out.append(p)
        x = x - p
    return out


def _product(a, b, parts):
    """a @ b of f32 values in `parts` bf16 parts each, their products with i + j < parts."""
    x, y = _parts(a, parts), _parts(b, parts)
    return sum(x[i] @ y[j] for i in range(parts) for j in range(parts) if i + j < parts)


def _rounded(x, bits):
    """x (64 bits) to `bits` significant ones."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 2.0 ** bits) / 2.0 ** bits, e)


def _inputs(n, d, rows=64):
    g = torch.Generator().manual_seed(n + d)
    return [torch.randn(r, d, generator=g) for r in (rows, n, n)]


def _exact(q, k, v):
    return torch.softmax(q.double() @ k.double().t() / math.sqrt(q.shape[1]), -1) @ v.double()


@pytest.mark.parametrize("n,d", [(333, 32), (2000, 64), (2000, 128), (333, 224), (9000, 256)])
def test_f32_limit(n, d):
    q, k, v = _inputs(n, d)
    want = _exact(q, k, v)

    def at(score, p=None, value=None):
        s = _product(q, k.t().contiguous(), score) * (1.0 / math.sqrt(d))
        p_ = torch.exp(s - s.amax(-1, keepdim=True))
        w = p_.bfloat16().float() if p == "bf16" else p_
        return cross_precision.off(_product(w, v, value or 3) / p_.sum(-1, keepdim=True), want)
    assert at(3) <= cross_precision.F32 / 2
    assert min(at(2), at(3, value=2), at(3, "bf16")) > 2 * cross_precision.F32


@pytest.mark.parametrize("n,d", [(333, 32), (2000, 64), (2000, 128), (333, 224), (9000, 256)])
def test_16_bit_limit(n, d):
    q, k, v = _inputs(n, d)
    q, v = q.bfloat16(), v.bfloat16()

    def at(bits, pages):
        kk, vv = (k.double(), v.double()) if pages else (k.bfloat16().double(), v.double())
        want = torch.softmax(q.double() @ kk.t() / math.sqrt(d), -1) @ vv
        kr, vr = (_rounded(kk, 11), _rounded(vv, 11)) if pages else (kk, vv)
        s = q.double() @ kr.t() / math.sqrt(d)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        w = _rounded(p, bits)
        out = ((w @ vr) / w.sum(-1, keepdim=True)).bfloat16()
        return cross_precision.off(out, want) / cross_precision.floor(want, torch.bfloat16)
    assert at(11, False) <= 1.05 and at(16, False) <= 1.05 and at(11, True) <= 1.05
    assert at(8, False) > 1.2 and at(8, True) > 1.2
