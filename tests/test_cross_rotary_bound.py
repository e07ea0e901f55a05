"""Bound launchers of cross attention and rotary appends: what they refuse, without a GPU."""
import pytest
import torch

from test_cross_rotary_refusals import call  # noqa: F401 (a fixture)


def test_bound_cross_attention_has_an_out_of_its_own(call):  # noqa: F811
    """In place, a second launch would attend with what the first one gave as its queries."""
    with pytest.raises(ValueError, match="out"):
        call.pool.bind_cross(call.q, call.cu, call.tables, call.lens, call.q)
    assert not call.launched
    # once is fine
    call.pool.paged_cross(call.q, call.cu, call.tables, call.lens, call.q)
    assert len(call.launched) == 1


def test_bound_cross_attention_without_rows(call):  # noqa: F811
    """Tensors without elements have one address, 0, and are not each other's."""
    q, out = torch.zeros(0, 4, 32), torch.zeros(0, 4, 32)
    assert q.data_ptr() == out.data_ptr()
    call.pool.bind_cross(q, call.cu, call.tables, call.lens, out)()
    assert len(call.launched) == 2


def test_a_bound_append_without_rows(call):  # noqa: F811
    """A step of no tokens binds like any other."""
    q, out = torch.zeros(0, 4, 32), torch.zeros(0, 4, 32)
    kv = torch.zeros(0, 4, 32).split([2, 2], dim=1)
    call.pool.bind_append_rotary(q, *kv, call.slots[:0], call.lens[:0], call.f, out)()
    assert len(call.launched) == 2


def test_a_calls_own_workspace_is_on_its_queries_device(call, monkeypatch):  # noqa: F811
    """The kernel runs on the pool's device, whichever is current."""
    devices, real = [], torch.empty

    def empty(*shape, dtype=None, device=None):
        devices.append(device)
        return real(*shape, dtype=dtype)
    monkeypatch.setattr(torch, "empty", empty)
    call.pool.paged_cross(call.q, call.cu, call.tables, call.lens, call.out)
    assert devices == [call.q.device]
