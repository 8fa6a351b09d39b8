"""Refusals of the cache operators (attention_tree and its companions): every one of them is decided on the host before
anything is enqueued, so they are checked without a GPU, with addresses that are never followed."""
import ctypes

import numpy as np
import pytest

A = 1 << 20   # stands for any device address


def pointers(*values):
    return (ctypes.c_void_p * len(values))(*values)


TREE = dict(q=A, kNew=A, vNew=A, kCache=A, vCache=A, lengths=A, counts=A, visible=A, out=A, m=A, l=A, batch=1, heads=4, kvHeads=2, nodes=3, capacity=64,
            headDim=64, scale=0.125, stream=None)
WEIGHTS = dict(q=A, kNew=A, vNew=A, kCache=A, vCache=A, lengths=A, counts=A, visible=A, out=A, m=A, l=A, weightsIn=A, weightsOut=A, batch=1, heads=4,
               kvHeads=2, groups=2, nodes=3, capacity=64, headDim=64, scale=0.125, stream=None)
KEYS = dict(q=A, k=A, m=A, l=A, counts=A, weightsIn=A, weightsOut=A, batch=1, heads=4, kvHeads=2, groups=2, newLen=16, totalLen=16, kvRows=16, headDim=64,
            scale=0.125, oldLen=0, weightRows=16, stream=None)
EVICT = dict(k=A, v=2 * A, weights=3 * A, lengths=A, kOut=4 * A, vOut=5 * A, weightsOut=6 * A, lengthsOut=A, kept=None, batch=1, kvHeads=4, groups=4,
             headDim=64, capacity=128, outCapacity=64, budget=64, recent=8, stream=None)
ACCEPT = dict(logits=A, tokens=A, parents=A, counts=A, path=A, pathCounts=A, next=A, batch=1, nodes=3, vocab=100, stream=None)
COMMIT = dict(k=pointers(A), v=pointers(A), kNew=pointers(A), vNew=pointers(A), weights=None, layers=1, path=A, pathCounts=A, lengths=A, lengthsOut=A,
              batch=1, kvHeads=4, groups=4, nodes=3, capacity=64, headDim=64, stream=None)

CASES = [
    ("bf_hip_attention_tree", TREE, dict(nodes=65), "64 nodes"),
    ("bf_hip_attention_tree", TREE, dict(kvHeads=3), "kvHeads"),
    ("bf_hip_attention_tree", TREE, dict(heads=0), "kvHeads"),
    ("bf_hip_attention_tree", TREE, dict(headDim=257), "headDim"),
    ("bf_hip_attention_tree", TREE, dict(lengths=None), "NULL"),
    ("bf_hip_attention_tree", TREE, dict(kCache=None), "NULL"),
    ("bf_hip_attention_tree", TREE, dict(out=None), "NULL"),
    ("bf_hip_attention_tree", TREE, dict(capacity=1 << 30), "too large"),
    ("bf_hip_attention_tree", TREE, dict(batch=1 << 16), "too large"),
    ("bf_hip_attention_tree", TREE, dict(heads=8194, kvHeads=2), "too large"),
    ("bf_hip_attention_tree", TREE, dict(heads=4096, kvHeads=4096, nodes=64, batch=60000), "too large"),
    ("bf_hip_attention_tree_weights", WEIGHTS, dict(groups=3), "groups"),
    ("bf_hip_attention_tree_weights", WEIGHTS, dict(groups=0), "groups"),
    ("bf_hip_attention_tree_weights", WEIGHTS, dict(weightsOut=None), "NULL"),
    ("bf_hip_attention_tree_weights", WEIGHTS, dict(nodes=65), "64 nodes"),
    ("bf_hip_attention_key_weights", KEYS, dict(weightRows=15), "weightRows"),
    ("bf_hip_attention_key_weights", KEYS, dict(kvRows=15), "kvRows"),
    ("bf_hip_attention_key_weights", KEYS, dict(l=None), "NULL"),
    ("bf_hip_attention_key_weights", KEYS, dict(weightsOut=None), "NULL"),
    ("bf_hip_attention_key_weights", KEYS, dict(headDim=300), "headDim"),
    ("bf_hip_attention_key_weights", KEYS, dict(newLen=1 << 30), "too large"),
    ("bf_hip_kv_evict", EVICT, dict(recent=65), "recent"),
    ("bf_hip_kv_evict", EVICT, dict(budget=65), "capacity"),
    ("bf_hip_kv_evict", EVICT, dict(groups=3), "groups"),
    ("bf_hip_kv_evict", EVICT, dict(kOut=A), "together"),
    ("bf_hip_kv_evict", EVICT, dict(weightsOut=3 * A), "together"),
    ("bf_hip_kv_evict", EVICT, dict(kOut=A, vOut=2 * A, weightsOut=3 * A), "capacity"),
    ("bf_hip_kv_evict", EVICT, dict(lengths=None), "NULL"),
    ("bf_hip_kv_evict", EVICT, dict(vOut=None), "NULL"),
    ("bf_hip_tree_accept", ACCEPT, dict(nodes=65), "64 nodes"),
    ("bf_hip_tree_accept", ACCEPT, dict(vocab=0), "empty"),
    ("bf_hip_tree_accept", ACCEPT, dict(vocab=(1 << 24) + 1), "2\\^24"),
    ("bf_hip_tree_accept", ACCEPT, dict(next=None), "NULL"),
    ("bf_hip_kv_commit", COMMIT, dict(nodes=65), "64 nodes"),
    ("bf_hip_kv_commit", COMMIT, dict(k=pointers(None)), "layer 0"),
    ("bf_hip_kv_commit", COMMIT, dict(weights=pointers(None)), "layer 0"),
    ("bf_hip_kv_commit", COMMIT, dict(weights=pointers(A), groups=3), "groups"),
    ("bf_hip_kv_commit", COMMIT, dict(path=None), "NULL"),
    ("bf_hip_kv_commit", COMMIT, dict(kNew=None), "NULL"),
]


@pytest.mark.parametrize("entry,base,change,message", CASES, ids=[f"{c[0][7:]}-{'-'.join(c[2])}-{i}" for i, c in enumerate(CASES)])
def test_refused_before_anything_is_enqueued(entry, base, change, message):
    from blackforge_amd import capi
    with pytest.raises(ValueError, match=message):
        capi.call(entry, *{**base, **change}.values())


def test_nothing_to_do_is_no_error():
    from blackforge_amd import capi
    for entry, base, change in [("bf_hip_attention_tree", TREE, dict(batch=0)), ("bf_hip_attention_tree", TREE, dict(nodes=0)),
                                ("bf_hip_attention_tree", TREE, dict(headDim=0)), ("bf_hip_attention_key_weights", KEYS, dict(batch=0)),
                                ("bf_hip_kv_evict", EVICT, dict(batch=0)), ("bf_hip_kv_evict", EVICT, dict(headDim=0)),
                                ("bf_hip_tree_accept", ACCEPT, dict(nodes=0)), ("bf_hip_kv_commit", COMMIT, dict(batch=0))]:
        capi.call(entry, *{**base, **change}.values())


def test_visibility_of_a_tree():
    from blackforge_amd import ops
    #      0
    #     / \
    #    1   2
    #    |   |\
    #    3   4 5      and a second root, 6
    masks = ops.treeVisibility(np.array([[-1, 0, 0, 1, 2, 2, -1]]))
    assert masks.tolist() == [[0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100101, 0b1000000]]
    chain = ops.treeVisibility(np.arange(64) - 1)
    assert [int(x) for x in chain] == [(1 << (i + 1)) - 1 for i in range(64)]
    with pytest.raises(ValueError, match="before its parent"):
        ops.treeVisibility([-1, 2, 0])
    with pytest.raises(ValueError, match="64 nodes"):
        ops.treeVisibility(np.arange(65) - 1)
