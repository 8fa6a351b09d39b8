"""Checks that the Python layer of the cache operators makes before anything reaches the device: tensors whose shapes do not
fit are refused, on addresses that are never followed, so no GPU is needed."""
import ctypes

import pytest

A = 1 << 20   # stands for any device address


def tensor(*shape, itemsize=4):
    """A DeviceTensor that owns nothing."""
    from blackforge_amd import DeviceTensor
    t = DeviceTensor.__new__(DeviceTensor)
    t.shape, t.itemsize, t._bytes, t.ptr = shape, itemsize, 0, ctypes.c_void_p(A)
    return t


@pytest.fixture
def calls(monkeypatch):
    """The entry points that ops calls, recorded instead of called."""
    from blackforge_amd import ops
    made = []
    monkeypatch.setattr(ops, "_call", lambda name, *args: made.append((name, args)))
    return made


def accepted(batch, nodes):
    from blackforge_amd import ops
    return ops.AcceptedPath(tensor(batch, nodes), tensor(batch), tensor(batch))


def test_commit_refuses_groups_that_do_not_divide_the_rows(calls):
    """Rows of 64 columns and weights of five groups: no heads divide like that, and the rows would be copied at a pitch of 60."""
    from blackforge_amd import ops
    caches, new = [tensor(2, 30, 64)], [tensor(2, 4, 64)]
    with pytest.raises(ValueError, match="groups"):
        ops.kvCommit(caches, caches, new, new, accepted(2, 4), tensor(2), [tensor(2, 5, 30)])
    with pytest.raises(ValueError, match="groups"):
        ops.kvCommit(caches, caches, new, new, accepted(2, 4), tensor(2), [tensor(2, 0, 30)])
    assert calls == []
    ops.kvCommit(caches, caches, new, new, accepted(2, 4), tensor(2), [tensor(2, 4, 30)])
    assert [name for name, _ in calls] == ["bf_hip_kv_commit"]
