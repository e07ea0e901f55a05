"""Rotary positions as far as int32 goes, against angles that are exact.

The kernels hold the angle p * inv_freq in 64 bits.  Below 2^29 the product of a position and an f32 has at most 53
bits and is exact; beyond, it is rounded once, by at most half a step: |angle| * 2^-53 (2^-22 at 2^31, as much
as the f32 roundings that follow).  rotary_ref's angles round the same way, so that what is compared with them is not
seen to be off; these are Python's fractions, reduced by sixty digits of pi."""
from fractions import Fraction

import numpy as np
import pytest

import airkv
import rotary_ref as ref
from gpu_helpers import torch_mod

pytestmark = pytest.mark.gpu

PI = Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)
FAR = [1, 4095, 10 ** 6 + 3, 2 ** 29 - 1, 2 ** 29 + 1, 2 ** 30 + 12345, 2 ** 31 - 1, -2 ** 31, -(2 ** 30) - 777]


def _reduced(positions, f):
    """The angles modulo 2 pi, in 64 bits (rounded once more, by 2^-52 at most)."""
    return np.array([[float(Fraction(int(p)) * Fraction(float(x)) % (2 * PI)) for x in f] for p in positions])


def _turned(x, angle):
    half = angle.shape[-1]
    z = (x[..., :half].astype(np.float64) + 1j * x[..., half:]) * np.exp(1j * angle)[:, None]
    return np.concatenate([z.real, z.imag], -1)


def _size(x):
    half = x.shape[-1] // 2
    return np.tile(np.hypot(x[..., :half], x[..., half:]), 2)


def _bound(x, want, by, f):
    """c and s, two products, their sum and the output round by 2^-24 each; the angle as said above."""
    angle = np.abs(np.asarray(by, np.float64))[:, None] * f
    angle = np.where(np.abs(np.asarray(by, np.float64))[:, None] < 2 ** 29, 0.0, angle) * 2.0 ** -53 + 2.0 ** -50
    return _size(x) * (3 * 2.0 ** -24 * 2 ** 0.5 + np.tile(angle, 2)[:, None]) + 2.0 ** -24 * np.abs(want)


def test_append():
    torch = torch_mod()
    f = ref.frequencies(64)
    x = np.random.default_rng(1).standard_normal((len(FAR), 2, 64)).astype(np.float32)
    pool = airkv.KvPool(1, 16, 2, 64, airkv.F32)
    q = torch.from_numpy(x).cuda()
    n = len(FAR)
    got = pool.append_rotary(q, q, q, torch.arange(n, device="cuda"), torch.tensor(FAR, dtype=torch.int32, device="cuda"), torch.from_numpy(f).cuda())
    want = _turned(x, _reduced(FAR, f))
    near = bool((np.abs(got.cpu().numpy() - want) <= _bound(x, want, FAR, f)).all())
    assert near
    assert np.array_equal(pool.snapshot()[0][0, :, :n], got.cpu().numpy().transpose(1, 0, 2))


def test_rotate():
    """By as much as 2^32 - 1."""
    torch = torch_mod()
    f = ref.frequencies(64)
    n = len(FAR)
    x = np.random.default_rng(2).standard_normal((n, 1, 64)).astype(np.float32)
    was = [-2 ** 31 if p > 0 else 2 ** 31 - 1 for p in FAR]
    by = [p - w for p, w in zip(FAR, was)]
    assert max(by) == 2 ** 32 - 1 and min(by) == -(2 ** 32) + 1
    pool = airkv.KvPool(1, 16, 1, 64, airkv.F32)
    k = torch.from_numpy(x).cuda()
    pool.append(k, k, torch.arange(n, device="cuda"))
    ints = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0]], was, [0, n], FAR)]
    pool.rotate(ints[0], ints[1], ints[2], torch.from_numpy(f).cuda(), to_pos=ints[3])
    want = _turned(x, _reduced(by, f))
    near = bool((np.abs(pool.snapshot()[0][0, 0, :n, None] - want) <= _bound(x, want, by, f)).all())
    assert near
