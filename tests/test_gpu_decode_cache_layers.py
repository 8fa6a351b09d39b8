"""GPU tests of the cache operators over several layers that share their sequences' lengths, and at sizes with nothing in them."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from test_gpu_decode_cache import check_tree, check_weights, ints, kept_rows, make, reference, run_tree, tree_masks

pytestmark = pytest.mark.gpu
f32 = np.float32


def test_eviction_of_layers_that_share_their_lengths(hip, rng):
    """Every layer keeps its own heaviest rows; the lengths are cut once, after the last."""
    D, batch, kv, groups, hd, cap, budget, recent = hip.DeviceTensor, 2, 4, 2, 32, 90, 40, 6
    lengths = [90, 33]
    k, v = ([rng.standard_normal((batch, cap, kv * hd)).astype(f32) for _ in range(3)] for _ in range(2))
    w = [np.abs(rng.standard_normal((batch, groups, cap))).astype(f32) for _ in range(3)]
    dk, dv, dw = ([D.fromHost(x) for x in t] for t in (k, v, w))
    dl = ints(hip, lengths)
    hip.ops.kvEvict(dk, dv, dw, dl, kv, budget, recent)
    assert dl.toHostInts().tolist() == [40, 33]
    slab = kv * hd // groups
    for x in range(3):
        ek, ev, ew = k[x].copy(), v[x].copy(), w[x].copy()
        for b in range(batch):
            for g in range(groups):
                rows, at = kept_rows(w[x][b, g], lengths[b], budget, recent), slice(g * slab, (g + 1) * slab)
                ek[b, :len(rows), at], ev[b, :len(rows), at], ew[b, g, :len(rows)] = k[x][b, rows, at], v[x][b, rows, at], w[x][b, g, rows]
        for got, want, what in ((dk, ek, "keys"), (dv, ev, "values"), (dw, ew, "weights")):
            assert got[x].toHost().tobytes() == want.tobytes(), f"{what} of layer {x}"


def test_the_cpp_layer_cuts_all_layers_or_none(hip):
    """tests/cpp/decode_cache_layers_test.cpp: a layer that does not fit is refused before any other is cut."""
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "blackforge_amd", "host", "bin", "decode_cache_layers_test")
    assert os.path.exists(exe), "blackforge_amd/host has not been built"
    proc = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stdout + proc.stderr


@pytest.mark.parametrize("budget", [0, 5])
def test_eviction_from_caches_without_rows_still_cuts_the_lengths(hip, budget):
    """No capacity, so no sequence has rows, whatever its length says: lengthsOut is 0, the result's tensors stay as they were."""
    D, batch, kv, hd = hip.DeviceTensor, 3, 2, 32
    before = [np.full(s, 7, f32) for s in ((batch, 8, kv * hd), (batch, 8, kv * hd), (batch, kv, 8))]
    out = [D.fromHost(x) for x in before]
    lengths, left, kept = ints(hip, [4, 0, -2]), ints(hip, [9, 9, 9]), ints(hip, np.full((batch, kv, max(budget, 1)), 9))
    hip.capi.call("bf_hip_kv_evict", None, None, None, lengths.ptr, *(t.ptr for t in out), left.ptr, kept.ptr, batch, kv, kv, hd, 0, 8, budget, 0, None)
    assert left.toHostInts().tolist() == [0, 0, 0] and lengths.toHostInts().tolist() == [4, 0, -2]
    assert (kept.toHostInts() == 9).all()
    for t, x in zip(out, before):
        assert t.toHost().tobytes() == x.tobytes()
    hip.capi.call("bf_hip_kv_evict", None, None, None, lengths.ptr, *(t.ptr for t in out), lengths.ptr, None, batch, kv, kv, hd, 0, 8, budget, 0, None)
    assert lengths.toHostInts().tolist() == [0, 0, 0]


def test_a_draft_without_nodes_accepts_none(hip):
    """The counts are 0, whatever their memory held before, and an append of nothing leaves the lengths alone."""
    D, batch = hip.DeviceTensor, 3
    dirty = ints(hip, [9] * batch)
    del dirty      # its block is the pool's next of this size
    taken = hip.ops.treeAccept(D((batch, 0, 50)), D((batch, 0)), D((batch, 0)))
    assert taken.counts.toHostInts().tolist() == [0] * batch and taken.next.toHost().tolist() == [0] * batch
    cache, lengths = D.zeros((batch, 4, 8)), ints(hip, [1, 4, 0])
    hip.ops.kvCommit([cache], [cache], [D((batch, 0, 8))], [D((batch, 0, 8))], taken, lengths)
    assert lengths.toHostInts().tolist() == [1, 4, 0]


@pytest.mark.parametrize("nodes,hd", [(0, 64), (3, 0), (0, 0)])
def test_a_step_without_new_tokens_carries_the_weights(hip, rng, nodes, hd):
    """No node or no column: no row receives any weight, so those in use have what they had, and the others stay as they were."""
    D, batch, heads, groups, cap = hip.DeviceTensor, 3, 4, 2, 700
    lengths = [700, 0, 257]
    before = rng.random((batch, groups, cap)).astype(f32)
    q, cache, w_in, dl = D((batch, nodes, heads * hd)), D((batch, cap, heads * hd)), D.fromHost(before), ints(hip, lengths)
    for weights_in in (w_in, None):
        out = D.fromHost(np.full(before.shape, 7, f32))
        hip.capi.call("bf_hip_attention_tree_weights", q.ptr, q.ptr, q.ptr, cache.ptr, cache.ptr, dl.ptr, None, None, q.ptr, None, None,
                      weights_in.ptr if weights_in else None, out.ptr, batch, heads, heads, groups, nodes, cap, hd, 0.125, None)
        used = np.arange(cap) < np.array(lengths)[:, None, None]
        np.testing.assert_array_equal(out.toHost(), np.where(used, before if weights_in else np.zeros_like(before), f32(7)))
    hip.capi.call("bf_hip_attention_tree_weights", q.ptr, q.ptr, q.ptr, cache.ptr, cache.ptr, dl.ptr, None, None, q.ptr, None, None,
                  w_in.ptr, w_in.ptr, batch, heads, heads, groups, nodes, cap, hd, 0.125, None)
    np.testing.assert_array_equal(w_in.toHost(), before)


@pytest.mark.parametrize("stats", [True, False])
@pytest.mark.parametrize("nodes", [1, 3, 4, 17])
def test_weights_over_caches_whose_products_pass_a_gibibyte(hip, rng, nodes, stats):
    """Many heads to a key head over a cache with room for 5 million rows: products kept (up to three nodes) and made again, on
    statistics of the caller's or of the call's own; the workspace is what the header says."""
    heads, hd, cap = 64, 4, 5_000_000
    scale, lengths, counts = 0.5, [300], [nodes]
    q, kn, vn, k, v = make(rng, 1, heads, 1, hd, nodes, 301, lengths, counts)
    visible = tree_masks(rng, 1, nodes)
    want = reference(q, kn, vn, k, v, lengths, counts, visible, heads, 1, 1, scale)
    k, v = (np.concatenate([x, np.full((1, cap - 301, hd), np.nan, f32)], 1) for x in (k, v))
    weights = rng.random((1, 1, cap)).astype(f32)
    hip.capi.call("bf_hip_pool_trim")

    def from_driver():
        stats = hip.capi.PoolStats()
        hip.capi.call("bf_hip_pool_stats", ctypes.byref(stats))
        return stats.bytes_from_driver
    before = from_driver()
    got = run_tree(hip, q, kn, vn, k, v, lengths, counts, visible, heads, 1, scale, weights, 1, stats=stats)
    taken = from_driver() - before
    if stats:
        check_tree(got, want, counts, 5.5, "past a gibibyte")
    else:
        assert (got[1] == 7).all() and (got[2] == 7).all()
        check_tree((got[0], want[1], want[2]), want, counts, 5.5, "past a gibibyte without statistics")
    check_weights(got[3], weights, want[3], lengths, counts, heads * nodes, want[4], "past a gibibyte")
    del got
    workspace = 4 * heads * cap * (nodes if nodes <= 3 else 1)
    # operands and weights twice, 1/4 more at most for the pool's size classes, and 64 MiB for what grows with neither
    assert taken <= 1.25 * (workspace + 4 * cap * (2 * hd + 2)) + (64 << 20), f"{taken / 2**20:.0f} MiB taken"
    hip.capi.call("bf_hip_pool_trim")
