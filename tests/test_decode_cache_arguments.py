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


@pytest.mark.parametrize("counts", [tensor(2), tensor(4), tensor(3, 1), tensor(3, itemsize=8), tensor(3, itemsize=2)], ids=lambda t: f"{t.shape}x{t.itemsize}")
def test_counts_that_do_not_fit_are_refused(calls, counts):
    """The kernels read one 32-bit count a sequence: a shorter array would be read past its end."""
    from blackforge_amd import ops
    q, m = tensor(3, 5, 64), tensor(3, 2, 5)
    with pytest.raises(ValueError, match="count"):
        ops.attentionKeyWeights(q, q, m, m, 2, 0.125, 0, 2, tensor(3, 2, 9), counts)
    with pytest.raises(ValueError, match="count"):
        ops.treeAccept(tensor(3, 5, 99), tensor(3, 5), tensor(3, 5), counts)
    with pytest.raises(ValueError, match="count"):
        ops.attentionTree(q, q, q, tensor(3, 9, 64), tensor(3, 9, 64), tensor(3), 2, 0.125, counts)
    with pytest.raises(ValueError, match="count"):
        ops.attentionTreeWeights(q, q, q, tensor(3, 9, 64), tensor(3, 9, 64), tensor(3), 2, 0.125, tensor(3, 2, 9), counts)
    assert calls == []


def test_integers_of_another_width_are_refused(calls):
    """Lengths, parents and paths are 32-bit integers on the device: 64-bit ones would be read as pairs, 16-bit ones past their end."""
    from blackforge_amd import ops
    q, cache, weights = tensor(3, 5, 64), tensor(3, 9, 64), tensor(3, 2, 9)
    for itemsize in (2, 8):
        odd = tensor(3, itemsize=itemsize)
        with pytest.raises(ValueError, match="length"):
            ops.attentionTree(q, q, q, cache, cache, odd, 2, 0.125)
        with pytest.raises(ValueError, match="length"):
            ops.attentionTreeWeights(q, q, q, cache, cache, odd, 2, 0.125, weights)
        with pytest.raises(ValueError, match="length"):
            ops.kvEvict(cache, cache, weights, odd, 2, 4, 1)
        with pytest.raises(ValueError, match="length"):
            ops.kvCommit([cache], [cache], [q], [q], accepted(3, 5), odd)
        with pytest.raises(ValueError, match="parents"):
            ops.treeAccept(tensor(3, 5, 99), tensor(3, 5), tensor(3, 5, itemsize=itemsize))
        for path in (ops.AcceptedPath(tensor(3, 5, itemsize=itemsize), tensor(3), tensor(3)), ops.AcceptedPath(tensor(3, 5), odd, tensor(3))):
            with pytest.raises(ValueError, match="path"):
                ops.kvCommit([cache], [cache], [q], [q], path, tensor(3))
    with pytest.raises(ValueError, match="visible"):
        ops.attentionTree(q, q, q, cache, cache, tensor(3), 2, 0.125, None, tensor(3, 5))
    assert calls == []


def test_masks_come_back_as_integers_only(monkeypatch):
    """A tensor of 64-bit masks has no floats to give: copied into a float buffer it would run past that buffer's end."""
    import numpy as np
    from blackforge_amd import capi
    copied = []
    monkeypatch.setattr(capi, "call", lambda name, *args: copied.append(args[2]))
    masks, ints, halves = tensor(3, 5, itemsize=8), tensor(3, 5), tensor(3, 5, itemsize=2)
    for t in (masks, ints, halves):
        t._bytes = 15 * t.itemsize
    try:
        with pytest.raises(ValueError, match="toHostInts"):
            masks.toHost()
        with pytest.raises(ValueError, match="toHost"):
            halves.toHostInts()
        assert copied == []
        for read in (masks.toHostInts, ints.toHostInts, ints.toHost, halves.toHost):
            assert read().nbytes == copied.pop()
        assert (masks.toHostInts().dtype, ints.toHostInts().dtype) == (np.uint64, np.int32)
    finally:
        for t in (masks, ints, halves):
            t._bytes = 0
