"""Checks that the Python layer of the cache operators makes before anything reaches the device: tensors whose shapes do not
fit are refused, on addresses that are never followed, so no GPU is needed."""
import ctypes

import pytest

from test_decode_cache_refusals import EVICT, KEYS, TREE, WEIGHTS

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


def evict_layers(n=3):
    return [tensor(2, 30, 64) for _ in range(n)], [tensor(2, 30, 64) for _ in range(n)], [tensor(2, 4, 30) for _ in range(n)]


def test_eviction_cuts_the_lengths_with_the_last_layer(calls):
    """The layers share their lengths: cut with the first, they would tell the others that nothing is left to evict."""
    from blackforge_amd import ops
    k, v, w = evict_layers()
    lengths = tensor(2)
    lengths.ptr = ctypes.c_void_p(2 * A)
    ops.kvEvict(k, v, w, lengths, 8, 12, 3)
    assert [name for name, _ in calls] == ["bf_hip_kv_evict"] * 3
    assert [args[7] for _, args in calls] == [None, None, lengths.ptr]
    calls.clear()
    ops.kvEvict(k[0], v[0], w[0], lengths, 8, 12, 3)     # one layer needs no list
    assert [args[7] for _, args in calls] == [lengths.ptr]


@pytest.mark.parametrize("change", ["values", "capacity", "weights", "groups", "no groups", "sequences", "rank"])
def test_eviction_refuses_before_it_cuts_any_layer(calls, change):
    """The third layer does not fit: the first two stay whole, since the lengths would not be cut with them."""
    from blackforge_amd import ops
    k, v, w = evict_layers()
    if change == "values":
        v[2] = tensor(2, 29, 64)
    if change == "capacity":
        k[2], v[2], w[2] = tensor(2, 11, 64), tensor(2, 11, 64), tensor(2, 4, 11)
    if change == "weights":
        w[2] = tensor(2, 4, 29)
    if change == "groups":
        w[2] = tensor(2, 3, 30)
    if change == "no groups":
        w[2] = tensor(2, 0, 30)
    if change == "sequences":
        k[2], v[2], w[2] = tensor(3, 30, 64), tensor(3, 30, 64), tensor(3, 4, 30)
    if change == "rank":
        k[2] = v[2] = tensor(60, 64)
    with pytest.raises(ValueError, match="kvEvict"):
        ops.kvEvict(k, v, w, tensor(2), 8, 12, 3)
    assert calls == []


def test_eviction_refuses_budgets_and_lists_that_do_not_fit(calls):
    from blackforge_amd import ops
    k, v, w = evict_layers()
    for budget, recent in ((31, 3), (12, 13), (-1, -1), (12, -1)):
        with pytest.raises(ValueError, match="kvEvict"):
            ops.kvEvict(k, v, w, tensor(2), 8, budget, recent)
    for lists in ((k, v[:2], w), (k, v, w[:1]), ([], [], []), ([k[0], k[1], k[0]], v, w)):
        with pytest.raises(ValueError, match="kvEvict"):
            ops.kvEvict(*lists, tensor(2), 8, 12, 3)
    with pytest.raises(ValueError, match="kvEvict"):
        ops.kvEvict(k, v, w, tensor(2), 7, 12, 3)
    assert calls == []


@pytest.mark.parametrize("entry,base,change", [
    ("bf_hip_attention_tree", TREE, dict(batch=60000, heads=512, kvHeads=512, nodes=1)),                                     # row tiles
    ("bf_hip_attention_tree_weights", WEIGHTS, dict(batch=4000, heads=64, kvHeads=64, groups=64, nodes=16, capacity=1 << 13)),   # blocks of keys
    ("bf_hip_attention_tree_weights", WEIGHTS, dict(batch=16, heads=4096, kvHeads=1, groups=1, nodes=64, capacity=1 << 17)),  # products made again
    ("bf_hip_attention_key_weights", KEYS, dict(batch=60000, heads=512, kvHeads=512)),
    ("bf_hip_kv_evict", EVICT, dict(batch=60000, kvHeads=512, groups=512)),                                                  # selections
    ("bf_hip_kv_evict", EVICT, dict(kvHeads=1, groups=1, headDim=(1 << 24) - 1, capacity=8192, outCapacity=8192, budget=8192)),    # columns
])
def test_launches_too_large_are_refused_before_the_first(entry, base, change):
    """Each of several launches of a call has less than 2^32 work-items; the check comes before any of them."""
    from blackforge_amd import capi
    with pytest.raises(ValueError, match="too large"):
        capi.call(entry, *{**base, **change}.values())
