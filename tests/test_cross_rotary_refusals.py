"""Cross attention and rotary positions without a GPU: calls that are refused before anything else is
looked at, and what KvPool's methods do in front of a launch."""
import contextlib
import ctypes
import types

import pytest
import torch

import airkv
from airkv import _lib
from airkv import pool as pool_module

HERE = 4096                                             # an address


def test_a_missing_pool_is_refused():
    lib, n = _lib.load(), ctypes.c_size_t()
    for got in (lib.air_paged_cross_workspace_size(None, 8, 1, 1, ctypes.byref(n)),
                lib.air_paged_cross(None, None, None, airkv.F32, 8, None, 1, 1, None, None, 1, 1, 0.125, None, 0, None, airkv.F32),
                lib.air_kv_append_rotary(None, None, None, 0, 0, None, 64, None, 64, airkv.F32, None, None, 1, None, 64, airkv.ROTARY_HALF,
                                         1.0, None, airkv.F32),
                lib.air_kv_rotate(None, None, None, 1, 1, None, None, None, 1, None, 64, airkv.ROTARY_PAIRS)):
        assert got == airkv.AIR_KV_E_INVALID_ARG


@pytest.fixture
def call(monkeypatch):
    """A pool whose launches are recorded, with the stream of every allocation."""
    now, log = [None], types.SimpleNamespace(allocated=[], launched=[])

    @contextlib.contextmanager
    def on(stream):
        before, now[0] = now[0], stream.cuda_stream
        yield
        now[0] = before

    real = torch.empty

    def empty(*shape, dtype=None, device=None):
        log.allocated.append(now[0])
        return real(*shape, dtype=dtype)

    class Lib:
        def __getattr__(self, name):
            def fn(*args):
                log.launched.append((name, args))
                return 0
            return fn

    lib = Lib()
    monkeypatch.setattr(pool_module._lib, "load", lambda: lib)
    monkeypatch.setattr(pool_module, "_dev", lambda t, dtype, what, shape=None: HERE)
    monkeypatch.setattr(pool_module, "_dev_rows", lambda t, dtype, what, shape: (HERE, t.stride(0)))
    monkeypatch.setattr(pool_module, "_stream_ptr", lambda s: 0 if s is None else s.cuda_stream)
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda p: types.SimpleNamespace(cuda_stream=p))
    p = airkv.KvPool.__new__(airkv.KvPool)
    p.handle, p.n_kv_heads, p.head_dim, p.block_size, p._scale, p.dtype = None, 2, 32, 16, 0.1, airkv.BF16
    monkeypatch.setattr(p, "cross_workspace_size", lambda *a: 64, raising=False)
    log.pool = p
    log.q, log.out = torch.zeros(3, 4, 32), torch.zeros(3, 4, 32)
    log.kv = torch.zeros(3, 4, 32).split([2, 2], dim=1)
    log.tables, log.lens, log.cu = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.arange(4, dtype=torch.int32)
    log.slots, log.f = torch.zeros(3, dtype=torch.int64), torch.ones(16)
    return log


class _Stream:
    cuda_stream = 77


def test_a_calls_own_workspace_is_its_streams(call):
    for name in ("paged_cross", "bind_cross"):
        for stream, at in ((_Stream(), 77), (None, None)):
            getattr(call.pool, name)(call.q, call.cu, call.tables, call.lens, call.out, stream=stream)
            assert call.allocated.pop() == at and call.launched[-1][1][1] == (at or 0)


def test_cross_attention_reads_nothing_back(call, monkeypatch):
    """Without max_q_len too: no wait for the device, so the call can be captured."""
    def waits(*a, **k):
        raise AssertionError("read back")
    for f in ("item", "cpu", "tolist", "__int__", "__bool__"):
        monkeypatch.setattr(torch.Tensor, f, waits)
    call.pool.paged_cross(call.q, call.cu, call.tables, call.lens, call.out)
    call.pool.append_rotary(call.q, *call.kv, call.slots, call.lens, call.f)
    call.pool.rotate(call.tables, call.lens, call.cu, call.f)
    assert [x[0] for x in call.launched] == ["air_paged_cross", "air_kv_append_rotary", "air_kv_rotate"]


def test_a_call_on_another_stream_brings_its_output(call):
    """What torch allocates here is the current stream's."""
    with pytest.raises(ValueError, match="q_out"):
        call.pool.append_rotary(call.q, *call.kv, call.slots, call.lens, call.f, stream=_Stream())
    assert not call.launched
    call.pool.append_rotary(call.q, *call.kv, call.slots, call.lens, call.f, q_out=call.out, stream=_Stream())
    call.pool.append_rotary(None, *call.kv, call.slots, call.lens, call.f, stream=_Stream())
    assert len(call.launched) == 2 and all(x[1][1] == 77 for x in call.launched) and not call.allocated


def test_strides_reach_the_call(call):
    """Slices of one projection go as they are."""
    call.pool.append_rotary(call.q, *call.kv, call.slots, call.lens, call.f, q_out=call.out)
    args = call.launched[-1][1]
    assert (args[3], args[6], args[8]) == (4 * 32, 4 * 32, 4 * 32) and args[14] == 32


def test_a_bound_append_has_a_q_out_of_its_own(call):
    """In place, a second launch would turn what the first one turned."""
    for out in (None, call.q):
        with pytest.raises(ValueError, match="q_out"):
            call.pool.bind_append_rotary(call.q, *call.kv, call.slots, call.lens, call.f, out)
    assert not call.launched
