"""GPU tests of the cache operators (attention_tree, its weights, eviction, verification of a draft) against float64 numpy.

Bounds, with e = 2^-24 (half a step of fp32): a score is a dot product of headDim terms, its error at most
ds = (headDim + 4) e scale max(|q| . |k|), including the rounding of its scaling; its exponential's argument adds
4 e max|score| and the exponential itself a few e.  A probability is then off by at most 3 ds + 8 e max|score| + (N + 16) e
relative to itself (N visible keys in the sum), and a weighted mean of values by twice that times max|v|, N e max|v| included.
"""
import ctypes
import os
import subprocess

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32, E = np.float32, 2.0 ** -24


def ints(hip, x):
    return hip.DeviceTensor.fromHostInts(x)


def masks(hip, x):
    return hip.DeviceTensor.fromHostInts(x, np.uint64)


def reference(q, kn, vn, k, v, lengths, counts, visible, heads, kv, groups, scale):
    """out, m, l and the weight received, in float64; rows past counts zero.  And the bound of a probability's relative error."""
    q, kn, vn, k, v = (np.asarray(x, np.float64) for x in (q, kn, vn, k, v))
    batch, nodes, dim = q.shape
    hd, cap = dim // heads, k.shape[1]
    out, m, l = np.zeros(q.shape), np.zeros((batch, heads, nodes)), np.zeros((batch, heads, nodes))
    received = np.zeros((batch, groups, cap + nodes))
    rel = 0.0
    for b in range(batch):
        L, n = lengths[b], counts[b]
        sees = np.ones((n, L + n), bool)
        for i in range(n):
            sees[i, L:] = [int(visible[b, i]) >> j & 1 for j in range(n)]
        for h in range(heads):
            g = h * kv // heads
            at = slice(g * hd, (g + 1) * hd)
            K = np.concatenate([k[b, :L, at], kn[b, :n, at]])
            V = np.concatenate([v[b, :L, at], vn[b, :n, at]])
            Q = q[b, :n, h * hd:(h + 1) * hd]
            with np.errstate(invalid="ignore"):
                s = np.where(sees, Q @ K.T * scale, -np.inf)
                abs_s = np.where(sees, np.abs(Q) @ np.abs(K).T * abs(scale), 0.0)
            if s.size == 0:
                m[b, h, :n] = -np.inf
                continue
            top = s.max(1)
            e = np.where(sees, np.exp(s - np.where(top == -np.inf, 0.0, top)[:, None]), 0.0)
            total = e.sum(1)
            p = e / np.where(total == 0, 1.0, total)[:, None]
            m[b, h, :n], l[b, h, :n] = top, total
            for i in range(n):
                out[b, i, h * hd:(h + 1) * hd] = p[i, sees[i]] @ V[sees[i]]
            received[b, h * groups // heads, :L + n] += p.sum(0)
            big = float(np.nanmax(abs_s[np.isfinite(abs_s)], initial=0.0))
            rel = max(rel, 3 * (hd + 4) * E * big + 8 * E * big + (L + n + 16) * E)
    return out, m, l, received, rel


def tree_masks(rng, batch, nodes):
    out = np.zeros((batch, nodes), np.uint64)
    for b in range(batch):
        for i in range(nodes):
            parent = int(rng.integers(max(0, i - 4), i)) if i else -1
            out[b, i] = (out[b, parent] if parent >= 0 else np.uint64(0)) | np.uint64(1) << np.uint64(i)
    return out


def make(rng, batch, heads, kv, hd, nodes, cap, lengths, counts, poison=True):
    def r(*s, scale=1.0):
        return (rng.standard_normal(s) * scale).astype(f32)
    q, kn, vn = r(batch, nodes, heads * hd, scale=2), r(batch, nodes, kv * hd), r(batch, nodes, kv * hd)
    k, v = r(batch, cap, kv * hd), r(batch, cap, kv * hd)
    if poison:   # what is not in use holds NaN: past the lengths and past the counts
        for b in range(batch):
            k[b, lengths[b]:] = v[b, lengths[b]:] = np.nan
            kn[b, counts[b]:] = vn[b, counts[b]:] = q[b, counts[b]:] = np.nan
    return q, kn, vn, k, v


def run_tree(hip, q, kn, vn, k, v, lengths, counts, visible, heads, kv, scale, weights=None, groups=1, stats=True, offset=0):
    """Results on rows that held 7 before, so that rows left alone show; `offset` floats shift every operand off its alignment."""
    D = hip.DeviceTensor
    batch, nodes, dim = q.shape

    def up(x):
        if not offset:
            return D.fromHost(x), 0
        return D.fromHost(np.concatenate([np.full(offset, np.nan, f32), x.ravel()])), 4 * offset
    held = [up(x) for x in (q, kn, vn, k, v)]
    p = [ctypes.c_void_p(t.ptr.value + o) if t.ptr.value else None for t, o in held]
    out, m, l = (D.fromHost(np.full(s, 7, f32)) for s in (q.shape, (batch, heads, nodes), (batch, heads, nodes)))
    ln, cn, vs = ints(hip, lengths), ints(hip, counts) if counts is not None else None, masks(hip, visible) if visible is not None else None
    args = [*p, ln.ptr, cn.ptr if cn else None, vs.ptr if vs else None, out.ptr, m.ptr if stats else None, l.ptr if stats else None]
    tail = [nodes, k.shape[1], dim // heads, scale, None]
    if weights is None:
        hip.capi.call("bf_hip_attention_tree", *args, batch, heads, kv, *tail)
        return out.toHost(), m.toHost(), l.toHost()
    w_in, w_out = D.fromHost(weights), D.fromHost(np.full(weights.shape, 7, f32))
    hip.capi.call("bf_hip_attention_tree_weights", *args, w_in.ptr, w_out.ptr, batch, heads, kv, groups, *tail)
    return out.toHost(), m.toHost(), l.toHost(), w_out.toHost()


def check_tree(got, want, counts, vmax, what):
    out, m, l = (np.asarray(x, np.float64) for x in got[:3])
    eo, em, el, _, rel = want
    for b, n in enumerate(counts):
        assert (out[b, n:] == 7).all() and (m[b, :, n:] == 7).all() and (l[b, :, n:] == 7).all(), f"{what}: rows past the count were written"
        assert np.isfinite(out[b, :n]).all(), f"{what}: non-finite output, sequence {b}"
        worst = np.abs(out[b, :n] - eo[b, :n]).max(initial=0.0)
        assert worst <= 2 * rel * vmax, f"{what}: output off by {worst:.3e}, bound {2 * rel * vmax:.3e} (sequence {b})"
        empty = np.isneginf(em[b, :, :n])
        assert (np.isneginf(m[b, :, :n]) == empty).all() and (l[b, :, :n][empty] == 0).all(), f"{what}: rows that see nothing"
        dm = np.abs(m[b, :, :n][~empty] - em[b, :, :n][~empty]).max(initial=0.0)
        dl = np.abs(l[b, :, :n][~empty] / el[b, :, :n][~empty] - 1).max(initial=0.0)
        assert dm <= rel and dl <= 2 * rel, f"{what}: statistics off by {dm:.3e}, {dl:.3e}, bound {rel:.3e}"


TREES = [
    # batch, heads, kvHeads, headDim, nodes, capacity, lengths, counts
    (1, 12, 12, 64, 1, 1024, [700], [1]),
    (1, 1, 1, 64, 1, 1, [1], [1]),
    (1, 2, 2, 64, 1, 8, [0], [1]),
    (3, 2, 2, 64, 7, 64, [0, 15, 64], [7, 3, 0]),
    (4, 3, 3, 64, 16, 300, [16, 17, 255, 300], [16, 15, 1, 9]),
    (2, 4, 4, 32, 17, 130, [129, 130], [17, 16]),
    (2, 4, 2, 128, 33, 520, [513, 31], [33, 20]),
    (1, 4, 4, 64, 64, 2000, [1999], [64]),
    (2, 8, 1, 64, 20, 700, [699, 1], [20, 11]),
    (1, 6, 2, 128, 64, 300, [287], [61]),
    (2, 3, 3, 20, 5, 90, [90, 33], [5, 5]),
    (2, 2, 2, 33, 9, 120, [119, 64], [9, 2]),
    (1, 5, 5, 1, 3, 40, [40], [3]),
    (1, 2, 1, 100, 31, 260, [259], [31]),
    (1, 2, 2, 192, 12, 200, [161], [12]),
    (2, 2, 2, 256, 40, 150, [150, 3], [40, 7]),
    (1, 4, 2, 252, 64, 90, [77], [64]),
    (2, 2, 2, 80, 40, 500, [499, 64], [40, 33]),
    (1, 4, 2, 96, 9, 700, [700], [9]),
    (2, 2, 1, 81, 7, 300, [299, 17], [7, 7]),
    (1, 2, 2, 160, 20, 330, [330], [20]),
    (1, 12, 12, 40, 2, 1000, [1000], [2]),
    (1, 2, 2, 64, 8, 20000, [19999], [8]),
    (5, 16, 16, 128, 3, 3000, [2999, 0, 1024, 5, 2048], [3, 3, 1, 2, 3]),
    (12, 2, 2, 64, 20, 3000, [3000] * 12, [0] * 11 + [20]),                       # sequences without nodes, with long caches
    (9, 3, 3, 64, 40, 2100, [2100, 64, 0, 2099, 700, 1, 1337, 63, 65], [40, 33, 40, 1, 17, 40, 0, 40, 16]),
    (66, 4, 2, 128, 12, 400, [(61 * i) % 401 for i in range(66)], [(5 * i) % 13 for i in range(66)]),
    (70, 2, 2, 64, 2, 50, [(7 * i) % 51 for i in range(70)], [i % 3 for i in range(70)]),
    # enough rows, or rows and room, for the forms that hold two and four tiles of rows
    (1, 33, 1, 64, 63, 16400, [8137], [63]),
    (1, 33, 1, 64, 63, 16400, [130], [40]),
    (2, 40, 2, 32, 50, 18000, [300, 9000], [50, 41]),
    (2, 34, 2, 60, 63, 8400, [77, 4900], [9, 63]),
    (1, 33, 1, 33, 63, 16400, [1021], [63]),
    (1, 33, 1, 64, 63, 300, [299], [63]),
    (1, 33, 1, 20, 63, 300, [237], [61]),
    (1, 33, 1, 96, 63, 300, [300], [62]),
    (1, 33, 1, 80, 63, 700, [650], [63]),
    (1, 33, 1, 81, 63, 100, [37], [63]),
    (2, 66, 2, 128, 33, 700, [700, 0], [33, 30]),
    (1, 33, 1, 100, 63, 300, [170], [63]),
    (2, 33, 1, 192, 63, 500, [500, 1], [63, 17]),
    (1, 33, 1, 160, 63, 300, [300], [63]),
    (1, 33, 1, 189, 63, 200, [100], [63]),
    (1, 33, 1, 256, 63, 200, [200], [63]),
]


@pytest.mark.parametrize("case", TREES, ids=[f"b{c[0]}h{c[1]}of{c[2]}hd{c[3]}n{c[4]}cap{c[5]}" for c in TREES])
def test_attention_of_a_tree_over_a_cache(hip, rng, case):
    batch, heads, kv, hd, nodes, cap, lengths, counts = case
    visible = tree_masks(rng, batch, nodes)
    q, kn, vn, k, v = make(rng, batch, heads, kv, hd, nodes, cap, lengths, counts)
    scale = 1.0 / np.sqrt(hd)
    want = reference(q, kn, vn, k, v, lengths, counts, visible, heads, kv, 1, scale)
    got = run_tree(hip, q, kn, vn, k, v, lengths, counts, visible, heads, kv, scale)
    check_tree(got, want, counts, 5.5, "tree")
    for groups in sorted({1, kv}):
        weights = np.abs(rng.standard_normal((batch, groups, cap))).astype(f32)
        want = reference(q, kn, vn, k, v, lengths, counts, visible, heads, kv, groups, scale)
        got = run_tree(hip, q, kn, vn, k, v, lengths, counts, visible, heads, kv, scale, weights, groups)
        check_tree(got, want, counts, 5.5, "tree with weights")
        check_weights(got[3], weights, want[3], lengths, counts, heads * nodes, want[4], f"groups {groups}")


def check_weights(got, before, received, lengths, counts, terms, rel, what):
    got = np.asarray(got, np.float64)
    cap = got.shape[2]
    for b, (L, n) in enumerate(zip(lengths, counts)):
        end = min(L + n, cap)
        assert (got[b, :, end:] == 7).all(), f"{what}: weights past the rows in use were written"
        add = received[b, :, :end]
        want = add + np.where(np.arange(end) < L, before[b, :, :end], 0)
        # every term off by `rel` of itself, `terms` additions, and the last one rounding the total
        bound = (rel + terms * E) * add + 2 * E * np.abs(want) + 1e-37
        off = np.abs(got[b, :, :end] - want) - bound
        assert (off <= 0).all(), f"{what}: weight off by {np.abs(got[b, :, :end] - want).max():.3e}, over its bound by {off.max():.3e} (sequence {b})"


def test_masks_that_leave_nothing_and_chains(hip, rng):
    """No mask bits at all (with and without cached rows), bits past the count, no mask (a chain), no counts, no statistics."""
    batch, heads, hd, nodes, cap = 4, 2, 64, 6, 40
    lengths, counts = [0, 0, 17, 40], [6, 4, 6, 5]
    q, kn, vn, k, v = make(rng, batch, heads, heads, hd, nodes, cap, lengths, counts)
    visible = tree_masks(rng, batch, nodes)
    visible[0, 2] = visible[0, 5] = visible[2, 3] = 0
    visible[1] |= np.uint64(0xFFFFFFFFFFFFFFF0)   # bits of nodes past the count
    scale = 0.125
    want = reference(q, kn, vn, k, v, lengths, counts, visible, heads, heads, heads, scale)
    weights = np.ones((batch, heads, cap), f32)
    got = run_tree(hip, q, kn, vn, k, v, lengths, counts, visible, heads, heads, scale, weights, heads)
    check_tree(got, want, counts, 5.5, "sparse masks")
    check_weights(got[3], weights, want[3], lengths, counts, nodes, want[4], "sparse masks")
    assert np.isneginf(got[1][0, :, [2, 5]]).all() and (got[0][0, [2, 5]] == 0).all()

    chain = np.tile(np.array([(2 << i) - 1 for i in range(nodes)], np.uint64), (batch, 1))
    full = [nodes] * batch
    q, kn, vn, k, v = make(rng, batch, heads, heads, hd, nodes, cap, lengths, full)
    want = reference(q, kn, vn, k, v, lengths, full, chain, heads, heads, 1, scale)
    check_tree(run_tree(hip, q, kn, vn, k, v, lengths, None, None, heads, heads, scale), want, full, 5.5, "chain")
    no_stats = run_tree(hip, q, kn, vn, k, v, lengths, None, None, heads, heads, scale, stats=False)
    assert (no_stats[1] == 7).all()
    check_tree((no_stats[0], np.where(True, want[1], 0), want[2]), want, full, 5.5, "chain without statistics")


def test_infinities_and_nan_in_rows_a_node_does_not_see(hip, rng):
    """Siblings' values and keys of NaN and infinity touch their own descendants only; scores of -infinity weigh nothing."""
    batch, heads, hd, nodes, cap = 1, 3, 64, 20, 200
    lengths, counts = [133], [20]
    visible = np.array([[1] + [1 | 1 << i for i in range(1, nodes)]], np.uint64)    # a root and its children
    q, kn, vn, k, v = make(rng, batch, heads, heads, hd, nodes, cap, lengths, counts)
    want = reference(q, kn, vn, k, v, lengths, counts, visible, heads, heads, heads, 0.125)
    bad_k, bad_v = kn.copy(), vn.copy()
    bad_v[0, 5], bad_v[0, 6], bad_k[0, 7] = np.nan, np.inf, np.nan
    weights = np.zeros((1, heads, cap), f32)
    got = run_tree(hip, q, bad_k, bad_v, k, v, lengths, counts, visible, heads, heads, 0.125, weights, heads)
    clean = [i for i in range(nodes) if i not in (5, 6, 7)]
    worst = np.abs(got[0][0, clean] - want[0][0, clean]).max()
    assert worst <= 2 * want[4] * 5.5, worst
    assert np.isnan(got[0][0, 5]).all() and np.isnan(got[0][0, 7]).all()
    assert not np.isfinite(got[0][0, 6]).any()
    # a key of -infinity against positive queries: score -infinity, weight 0, as if it were not there
    q2, k2 = np.abs(q), k.copy()
    k2[0, 50:70] = -np.inf
    keep = np.r_[0:50, 70:133]
    want = reference(q2, kn, vn, k[:, keep], v[:, keep], [113], counts, visible, heads, heads, heads, 0.125)
    got = run_tree(hip, q2, kn, vn, k2, v, lengths, counts, visible, heads, heads, 0.125, weights, heads)
    check_tree(got, want, counts, 5.5, "keys of -infinity")
    assert (got[3][0, :, 50:70] == 0).all()
    # nothing but scores of -infinity: as a row that sees nothing
    k2[:, :] = -np.inf
    got = run_tree(hip, q2, np.full_like(kn, -np.inf), vn, k2, v, lengths, counts, visible, heads, heads, 0.125)
    assert (got[0] == 0).all() and np.isneginf(got[1]).all() and (got[2] == 0).all()


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_operands_off_their_alignment(hip, rng, offset):
    batch, heads, kv, hd, nodes, cap, lengths, counts = 2, 4, 2, 64, 10, 150, [149, 60], [10, 4]
    visible = tree_masks(rng, batch, nodes)
    q, kn, vn, k, v = make(rng, batch, heads, kv, hd, nodes, cap, lengths, counts)
    want = reference(q, kn, vn, k, v, lengths, counts, visible, heads, kv, 1, 0.125)
    check_tree(run_tree(hip, q, kn, vn, k, v, lengths, counts, visible, heads, kv, 0.125, offset=offset), want, counts, 5.5, f"offset {offset}")


def test_counters_outside_their_range_are_held_inside(hip, rng):
    batch, heads, hd, nodes, cap = 3, 2, 64, 4, 50
    q, kn, vn, k, v = make(rng, batch, heads, heads, hd, nodes, cap, [0, 50, 50], [4, 4, 0])
    visible = tree_masks(rng, batch, nodes)
    want = reference(q, kn, vn, k, v, [0, 50, 50], [4, 4, 0], visible, heads, heads, 1, 0.125)
    got = run_tree(hip, q, kn, vn, k, v, [-3, 51, 1 << 30], [9, 64, -1], visible, heads, heads, 0.125)
    check_tree(got, want, [4, 4, 0], 5.5, "counters outside")


def test_no_cache_at_all(hip, rng):
    heads, hd, nodes = 2, 64, 9
    visible = tree_masks(rng, 1, nodes)
    q, kn, vn, k, v = make(rng, 1, heads, heads, hd, nodes, 0, [0], [nodes])
    want = reference(q, kn, vn, k, v, [0], [nodes], visible, heads, heads, 1, 0.125)
    check_tree(run_tree(hip, q, kn, vn, k, v, [5], [nodes], visible, heads, heads, 0.125), want, [nodes], 5.5, "no cache")


def test_large_and_growing_scores(hip, rng):
    """Scores in the hundreds whose maximum keeps growing along the cache: the running maximum moves at every tile."""
    heads, hd, nodes, cap = 2, 64, 5, 600
    q, kn, vn, k, v = make(rng, 1, heads, heads, hd, nodes, cap, [600], [nodes])
    k *= np.linspace(0, 30, cap, dtype=f32)[None, :, None]
    visible = tree_masks(rng, 1, nodes)
    want = reference(q, kn, vn, k, v, [600], [nodes], visible, heads, heads, heads, 0.125)
    weights = np.zeros((1, heads, cap), f32)
    got = run_tree(hip, q, kn, vn, k, v, [600], [nodes], visible, heads, heads, 0.125, weights, heads)
    check_tree(got, want, [nodes], 5.5, "growing scores")
    check_weights(got[3], weights, want[3], [600], [nodes], nodes, want[4], "growing scores")


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_any_scale(hip, rng, scale):
    heads, hd, cap = 2, 64, 300
    for nodes in (5, 40):
        q, kn, vn, k, v = make(rng, 1, heads, heads, hd, nodes, cap, [260], [nodes])
        visible = tree_masks(rng, 1, nodes)
        want = reference(q, kn, vn, k, v, [260], [nodes], visible, heads, heads, heads, scale)
        weights = np.ones((1, heads, cap), f32)
        got = run_tree(hip, q, kn, vn, k, v, [260], [nodes], visible, heads, heads, scale, weights, heads)
        check_tree(got, want, [nodes], 5.5, f"scale {scale}")
        check_weights(got[3], weights, want[3], [260], [nodes], nodes, want[4], f"scale {scale}")


def test_weights_of_rows_too_many_to_keep_their_products(hip, rng):
    """4096 rows to the key head over room for 66000: their dot products would be more than 1 GiB."""
    heads, hd, nodes, cap = 64, 4, 64, 66000
    q, kn, vn, k, v = make(rng, 1, heads, 1, hd, nodes, cap, [300], [nodes])
    visible = tree_masks(rng, 1, nodes)
    want = reference(q, kn, vn, k, v, [300], [nodes], visible, heads, 1, 1, 0.5)
    weights = np.ones((1, 1, cap), f32)
    got = run_tree(hip, q, kn, vn, k, v, [300], [nodes], visible, heads, 1, 0.5, weights, 1)
    check_tree(got, want, [nodes], 5.5, "rows too many to keep")
    check_weights(got[3], weights, want[3], [300], [nodes], heads * nodes, want[4], "rows too many to keep")


@pytest.mark.parametrize("heads,cap", [(1, 200), (33, 200), (33, 16600)])
def test_many_rows_to_a_key_head_with_values_that_are_not_finite(hip, rng, heads, cap):
    """Sixty-four nodes, one to four tiles of rows at a time: what a sibling holds touches its own descendants only."""
    hd, nodes = 64, 64
    visible = np.array([[1] + [1 | 1 << i for i in range(1, nodes)]], np.uint64)
    q, kn, vn, k, v = make(rng, 1, heads, 1, hd, nodes, cap, [133], [nodes])
    want = reference(q, kn, vn, k, v, [133], [nodes], visible, heads, 1, 1, 0.125)
    bad_k, bad_v = kn.copy(), vn.copy()
    bad_v[0, 5], bad_v[0, 37, 3], bad_k[0, 50] = np.nan, np.inf, np.nan
    got = run_tree(hip, q, bad_k, bad_v, k, v, [133], [nodes], visible, heads, 1, 0.125)
    clean = [i for i in range(nodes) if i not in (5, 37, 50)]
    worst = np.abs(got[0][0, clean] - want[0][0, clean]).max()
    assert worst <= 2 * want[4] * 5.5, worst
    assert np.isnan(got[0][0, 5]).all() and np.isnan(got[0][0, 50]).all()
    infinite = got[0][0, 37].reshape(heads, hd)
    assert not np.isfinite(infinite[:, 3]).any() and np.isfinite(np.delete(infinite, 3, 1)).all()


def test_results_do_not_change_from_run_to_run(hip, rng):
    batch, heads, hd, nodes, cap = 2, 8, 64, 24, 5000
    lengths, counts = [5000, 3111], [24, 20]
    q, kn, vn, k, v = make(rng, batch, heads, heads, hd, nodes, cap, lengths, counts)
    visible = tree_masks(rng, batch, nodes)
    weights = np.ones((batch, 1, cap), f32)
    first = run_tree(hip, q, kn, vn, k, v, lengths, counts, visible, heads, heads, 0.125, weights, 1)
    for _ in range(3):
        again = run_tree(hip, q, kn, vn, k, v, lengths, counts, visible, heads, heads, 0.125, weights, 1)
        for a, c in zip(first, again):
            assert a.tobytes() == c.tobytes()


# ---- the account of a pass that has run --------------------------------------------------------
KEYS = [
    # batch, heads, kvHeads, groups, headDim, newLen, totalLen, kvRows, oldLen, counts
    (1, 1, 1, 1, 64, 1, 1, 1, 0, None),
    (2, 3, 3, 3, 64, 100, 100, 100, 0, None),
    (2, 4, 4, 1, 64, 257, 257, 300, 0, [257, 130]),
    (1, 4, 2, 2, 128, 200, 200, 200, 0, None),
    (1, 8, 2, 1, 64, 65, 165, 170, 100, None),
    (3, 2, 2, 2, 32, 33, 33, 33, 0, [0, 1, 33]),
    (1, 2, 2, 2, 20, 70, 70, 70, 0, None),
    (1, 2, 2, 1, 33, 70, 70, 70, 0, None),
    (1, 2, 1, 1, 192, 40, 90, 90, 50, None),
    (1, 2, 2, 2, 256, 130, 130, 140, 0, None),
    (1, 2, 2, 2, 64, 50, 80, 80, 80, None),        # every key visible to every query
    (1, 2, 2, 2, 64, 3, 2000, 2000, 1997, None),
    (1, 3, 3, 3, 64, 1500, 1500, 1500, 0, None),
    (1, 2, 2, 2, 80, 120, 120, 120, 0, None),
    (1, 2, 1, 1, 160, 50, 130, 130, 80, None),
    (2, 2, 2, 2, 64, 60, 100, 100, 10, None),      # keys 70.. that no query sees
]


@pytest.mark.parametrize("case", KEYS, ids=[f"b{c[0]}h{c[1]}of{c[2]}g{c[3]}hd{c[4]}n{c[5]}t{c[6]}+{c[8]}" for c in KEYS])
def test_weight_of_keys_from_the_statistics(hip, rng, case):
    batch, heads, kv, groups, hd, n, total, rows, old, counts = case
    q, k = ((rng.standard_normal((batch, r, w * hd)) * s).astype(f32) for r, w, s in ((n, heads, 2.0), (rows, kv, 1.0)))
    k[:, total:] = np.nan
    scale = 1 / np.sqrt(hd)
    sees = np.arange(total)[None] <= old + np.arange(n)[:, None]
    want, m, l, rel = np.zeros((batch, groups, total)), np.zeros((batch, heads, n), f32), np.zeros((batch, heads, n), f32), 0.0
    live = [n] * batch if counts is None else counts
    for b in range(batch):
        for h in range(heads):
            Q, K = q[b, :, h * hd:(h + 1) * hd].astype(np.float64), k[b, :total, h * kv // heads * hd:(h * kv // heads + 1) * hd].astype(np.float64)
            s = np.where(sees, Q @ K.T * scale, -np.inf)
            m[b, h] = s.max(1)
            l[b, h] = np.exp(s - s.max(1)[:, None]).sum(1)
            p = np.exp(s - m[b, h].astype(np.float64)[:, None]) / l[b, h].astype(np.float64)[:, None]
            want[b, h * groups // heads] += p[:live[b]].sum(0)
            big = (np.abs(Q) @ np.abs(K).T).max() * scale
            rel = max(rel, (hd + 4) * E * big + 8 * E * big + 16 * E)
        q[b, live[b]:] = m[b, :, live[b]:] = np.nan      # rows past the count are not read
    dq, dk, dm, dl = (hip.DeviceTensor.fromHost(x) for x in (q, k, m, l))
    cn = ints(hip, counts) if counts is not None else None
    for before in (None, np.abs(rng.standard_normal((batch, groups, rows + 3))).astype(f32)):
        out = hip.DeviceTensor.fromHost(np.full((batch, groups, rows + 3), 7, f32) if before is None else before)
        hip.capi.call("bf_hip_attention_key_weights", dq.ptr, dk.ptr, dm.ptr, dl.ptr, cn.ptr if cn else None, None if before is None else out.ptr, out.ptr,
                      batch, heads, kv, groups, n, total, rows, hd, scale, old, rows + 3, None)
        got = out.toHost().astype(np.float64)
        start = np.zeros_like(want) if before is None else before[:, :, :total]
        bound = (rel + heads // groups * n * E) * want + 2 * E * np.abs(want + start) + 1e-37
        off = np.abs(got[:, :, :total] - (want + start))
        assert (off <= bound).all(), f"off by {off.max():.3e}, over its bound by {(off - bound).max():.3e}"
        rest = np.full_like(got[:, :, total:], 7) if before is None else before[:, :, total:]
        assert (got[:, :, total:] == rest).all(), "weights past totalLen were written"


@pytest.mark.parametrize("n", [20, 100])
def test_statistics_that_are_nan_reach_the_keys_their_query_sees(hip, rng, n):
    heads, hd, row = 2, 64, n - 7
    q, k = (hip.DeviceTensor.fromHost(rng.standard_normal((1, n, heads * hd)).astype(f32)) for _ in range(2))
    m = hip.DeviceTensor.fromHost(np.full((1, heads, n), 9, f32))
    sums = np.ones((1, heads, n), f32)
    sums[0, 1, row] = np.nan
    l, out = hip.DeviceTensor.fromHost(sums), hip.DeviceTensor.zeros((1, heads, n))
    hip.capi.call("bf_hip_attention_key_weights", q.ptr, k.ptr, m.ptr, l.ptr, None, None, out.ptr, 1, heads, heads, heads, n, n, n, hd, 0.125, 0, n, None)
    got = out.toHost()
    assert np.isfinite(got[0, 0]).all()
    assert np.isnan(got[0, 1, :row + 1]).all() and np.isfinite(got[0, 1, row + 1:]).all()


# ---- eviction ----------------------------------------------------------------------------------
def kept_rows(weights, length, budget, recent):
    if length <= budget:
        return list(range(length))
    n = length - recent
    w = np.where(np.isnan(weights[:n]), -np.inf, weights[:n])
    order = sorted(range(n), key=lambda i: (-w[i], i))
    return sorted(order[:budget - recent]) + list(range(n, length))


EVICT = [
    # batch, kvHeads, groups, headDim, capacity, outCapacity, budget, recent, lengths
    (1, 12, 12, 64, 1024, 512, 512, 64, [1024]),
    (2, 4, 1, 64, 300, 128, 100, 10, [300, 99]),
    (3, 2, 2, 32, 200, 200, 150, 150, [200, 150, 151]),
    (2, 3, 3, 20, 130, 64, 64, 0, [130, 65]),
    (2, 2, 1, 33, 90, 40, 33, 5, [90, 34]),
    (1, 2, 2, 64, 64, 1, 1, 0, [64]),
    (1, 2, 2, 64, 64, 1, 1, 1, [64]),
    (2, 2, 2, 64, 64, 8, 0, 0, [64, 0]),
    (1, 4, 2, 128, 9000, 4000, 3999, 77, [8999]),
    (4, 2, 2, 100, 2500, 1300, 1300, 1, [2500, 0, 1301, 1299]),
    (1, 1, 1, 1, 70000, 65000, 65000, 3, [70000]),
]


def evict_weights(rng, shape, kind):
    w = np.abs(rng.standard_normal(shape)).astype(f32)
    if kind == "ties":
        w = np.round(w * 2).astype(f32)
        w[w == 0] = np.where(rng.random((w == 0).sum()) < 0.5, 0.0, -0.0)
    if kind == "odd values":
        w *= np.where(rng.random(shape) < 0.3, -1, 1)
        for x in (np.nan, np.inf, -np.inf, 1e-42, 3e38):
            w[rng.random(shape) < 0.08] = x
    if kind == "equal":
        w[:] = 0.25
    return w


@pytest.mark.parametrize("kind", ["plain", "ties", "odd values", "equal"])
@pytest.mark.parametrize("case", EVICT, ids=[f"b{c[0]}kv{c[1]}g{c[2]}hd{c[3]}cap{c[4]}to{c[6]}+{c[7]}" for c in EVICT])
def test_eviction_keeps_the_recent_and_the_heaviest_rows(hip, rng, case, kind):
    batch, kv, groups, hd, cap, out_cap, budget, recent, lengths = case
    D, call = hip.DeviceTensor, hip.capi.call
    k, v = (rng.standard_normal((batch, cap, kv * hd)).astype(f32) for _ in range(2))
    w = evict_weights(rng, (batch, groups, cap), kind)
    slab = kv * hd // groups
    dk, dv, dw, dl = D.fromHost(k), D.fromHost(v), D.fromHost(w), ints(hip, lengths)

    def expect(into_k, into_v, into_w):
        ek, ev, ew, kept = into_k.copy(), into_v.copy(), into_w.copy(), np.full((batch, groups, budget), -5, np.int32)
        for b in range(batch):
            for g in range(groups):
                rows = kept_rows(w[b, g], lengths[b], budget, recent)
                at = slice(g * slab, (g + 1) * slab)
                ek[b, :len(rows), at], ev[b, :len(rows), at], ew[b, g, :len(rows)] = k[b, rows, at], v[b, rows, at], w[b, g, rows]
                kept[b, g, :len(rows)] = rows
        return ek, ev, ew, kept

    sizes = (batch, out_cap, kv * hd), (batch, out_cap, kv * hd), (batch, groups, out_cap)
    before = [np.full(s, 7, f32) for s in sizes]
    ok, ov, ow, ol, kept = *(D.fromHost(x) for x in before), ints(hip, [-1] * batch), ints(hip, np.full((batch, groups, budget), -5))
    call("bf_hip_kv_evict", dk.ptr, dv.ptr, dw.ptr, dl.ptr, ok.ptr, ov.ptr, ow.ptr, ol.ptr, kept.ptr, batch, kv, groups, hd, cap, out_cap, budget, recent,
         None)
    ek, ev, ew, ekept = expect(*before)
    if budget:
        np.testing.assert_array_equal(kept.toHostInts(), ekept)
    for got, want, what in ((ok, ek, "keys"), (ov, ev, "values"), (ow, ew, "weights")):
        assert got.toHost().tobytes() == want.tobytes(), what
    left = [min(x, budget) for x in lengths]
    assert ol.toHostInts().tolist() == left and dl.toHostInts().tolist() == list(lengths)
    assert dk.toHost().tobytes() == k.tobytes() and dw.toHost().tobytes() == w.tobytes(), "the inputs of a call out of place"

    ek, ev, ew, _ = expect(k, v, w)      # in place: rows past those that remain keep what they held
    call("bf_hip_kv_evict", dk.ptr, dv.ptr, dw.ptr, dl.ptr, dk.ptr, dv.ptr, dw.ptr, dl.ptr, None, batch, kv, groups, hd, cap, cap, budget, recent, None)
    for got, want, what in ((dk, ek, "keys"), (dv, ev, "values"), (dw, ew, "weights")):
        assert got.toHost().tobytes() == want.tobytes(), f"{what} in place"
    assert dl.toHostInts().tolist() == left


def test_eviction_off_alignment_and_lengths_outside(hip, rng):
    D, cap, dim = hip.DeviceTensor, 100, 64
    k, v = (rng.standard_normal((1, cap, dim)).astype(f32) for _ in range(2))
    w = np.abs(rng.standard_normal((1, 1, cap))).astype(f32)
    pad = [np.concatenate([np.zeros(1, f32), x.ravel()]) for x in (k, v)]
    dk, dv, dw, dl = D.fromHost(pad[0]), D.fromHost(pad[1]), D.fromHost(w), ints(hip, [cap + 50])
    pk, pv = (ctypes.c_void_p(t.ptr.value + 4) for t in (dk, dv))
    hip.capi.call("bf_hip_kv_evict", pk, pv, dw.ptr, dl.ptr, pk, pv, dw.ptr, dl.ptr, None, 1, 1, 1, dim, cap, cap, 30, 4, None)
    rows = kept_rows(w[0, 0], cap, 30, 4)
    assert (dk.toHost()[1:].reshape(cap, dim)[:30] == k[0, rows]).all() and (dv.toHost()[1:].reshape(cap, dim)[:30] == v[0, rows]).all()
    assert dl.toHostInts().tolist() == [30]
    neg = ints(hip, [-4])
    hip.capi.call("bf_hip_kv_evict", pk, pv, dw.ptr, neg.ptr, pk, pv, dw.ptr, neg.ptr, None, 1, 1, 1, dim, cap, cap, 30, 4, None)
    assert neg.toHostInts().tolist() == [0]


# ---- verification ------------------------------------------------------------------------------
def accept(logits, tokens, parents, count):
    def choice(row):
        best = 0
        for c in range(len(row)):
            if row[c] > row[best]:
                best = c
        return best
    if count == 0:
        return [], None
    path = [0]
    while True:
        want = choice(logits[path[-1]])
        nxt = next((j for j in range(path[-1] + 1, count) if parents[j] == path[-1] and round(float(tokens[j])) == want), None)
        if nxt is None:
            return path, want
        path.append(nxt)


@pytest.mark.parametrize("batch,nodes,vocab", [(1, 1, 1), (3, 7, 10), (5, 64, 33), (2, 26, 5000), (4, 13, 1025), (2, 5, 50257)])
def test_path_of_a_draft(hip, rng, batch, nodes, vocab):
    D = hip.DeviceTensor
    logits = np.round(rng.standard_normal((batch, nodes, vocab)) * 3).astype(f32)      # many ties
    tokens = rng.integers(0, vocab, (batch, nodes))
    parents = np.array([[-1] + [int(rng.integers(max(0, j - 5), j)) for j in range(1, nodes)] for _ in range(batch)], np.int32)
    for b in range(batch):
        for j in range(1, nodes):
            if rng.random() < 0.7:
                logits[b, parents[b, j], tokens[b, j]] = 50
                if rng.random() < 0.3 and j + 1 < nodes:
                    tokens[b, j + 1], parents[b, j + 1] = tokens[b, j], parents[b, j]    # a sibling with the same token
        logits[b, rng.integers(0, nodes), rng.integers(0, vocab)] = np.nan
        logits[b, rng.integers(0, nodes), 0] = np.nan if b % 2 else -np.inf
    logits[0, nodes // 2] = np.nan
    counts = [nodes] + [int(rng.integers(0, nodes + 1)) for _ in range(batch - 1)]
    dl, dt, dp = D.fromHost(logits), D.fromHost(tokens.astype(f32)), ints(hip, parents)
    for cn in (None, counts):
        path, found, nxt = ints(hip, np.full((batch, nodes), 9)), ints(hip, [9] * batch), D.fromHost(np.full(batch, 9, f32))
        dc = ints(hip, cn) if cn else None
        hip.capi.call("bf_hip_tree_accept", dl.ptr, dt.ptr, dp.ptr, dc.ptr if dc else None, path.ptr, found.ptr, nxt.ptr, batch, nodes, vocab, None)
        for b in range(batch):
            want, then = accept(logits[b], tokens[b], parents[b], cn[b] if cn else nodes)
            assert found.toHostInts()[b] == len(want) and path.toHostInts()[b].tolist() == want + [-1] * (nodes - len(want)), f"sequence {b}"
            assert nxt.toHost()[b] == (9 if then is None else then)


@pytest.mark.parametrize("layers,dim,groups,cap,with_weights,alias", [(1, 64, 2, 30, False, True), (3, 33, 3, 30, True, False),
                                                                     (50, 96, 2, 64, True, True), (100, 8, 2, 20, False, False),
                                                                     (0, 64, 2, 30, False, True)])
def test_accepted_rows_are_appended_to_every_layer(hip, rng, layers, dim, groups, cap, with_weights, alias):
    D, batch, nodes = hip.DeviceTensor, 6, 9
    path = np.full((batch, nodes), -1, np.int32)
    path[:5, :4] = [0, 2, 3, 8]
    path[3, 1] = nodes                    # no node: sequence 3 is left alone
    counts = [4, 0, 4, 4, 10, 1]          # sequence 4: more than there are nodes
    path[5, 0] = 6
    lengths = [5, 7, cap - 3, 5, 5, cap - 1]     # sequence 2: no room
    good = {0: [0, 2, 3, 8], 1: [], 5: [6]}

    def r(*s):
        return rng.standard_normal(s).astype(f32)
    k, v, kn, vn = ([r(batch, rows, dim) for _ in range(layers)] for rows in (cap, cap, nodes, nodes))
    w = [r(batch, groups, cap) for _ in range(layers)] if with_weights else []
    dev = [[D.fromHost(x) for x in t] for t in (k, v, kn, vn)]
    dw = [D.fromHost(x) for x in w]
    ptrs = [(ctypes.c_void_p * max(layers, 1))(*[x.ptr for x in t]) for t in dev]
    wp = (ctypes.c_void_p * layers)(*[x.ptr for x in dw]) if w else None
    dl, dp, dc = ints(hip, lengths), ints(hip, path), ints(hip, counts)
    out = dl if alias else ints(hip, [-9] * batch)
    hip.capi.call("bf_hip_kv_commit", *ptrs, wp, layers, dp.ptr, dc.ptr, dl.ptr, out.ptr, batch, groups, groups, nodes, cap, dim // groups, None)
    for x in range(layers):
        for b, rows in good.items():
            at = lengths[b]
            k[x][b, at:at + len(rows)], v[x][b, at:at + len(rows)] = kn[x][b, rows], vn[x][b, rows]
            if w:      # a weight that would lie past the capacity was never kept
                moved = [w[x][b, :, at + i].copy() if at + i < cap else 0 for i in rows]
                for n, value in enumerate(moved):
                    w[x][b, :, at + n] = value
        assert dev[0][x].toHost().tobytes() == k[x].tobytes() and dev[1][x].toHost().tobytes() == v[x].tobytes(), f"layer {x}"
        if w:
            assert dw[x].toHost().tobytes() == w[x].tobytes(), f"weights of layer {x}"
    assert out.toHostInts().tolist() == [n + (len(good[b]) if b in good else 0) for b, n in enumerate(lengths)]


# ---- together ----------------------------------------------------------------------------------
def test_a_drafted_generation_with_a_bounded_cache(hip, rng):
    """A prompt, its weights, eviction to a budget, then rounds of draft, verification and append, on the device throughout, against
    the same in float64 numpy (one attention layer over embedded tokens, its output the logits' features)."""
    ops, D = hip.ops, hip.DeviceTensor
    heads, hd, vocab, prompt, budget, recent, cap, nodes = 2, 32, 50, 60, 40, 8, 160, 7
    dim = heads * hd
    table, wq, wk, wv, wo = ((rng.standard_normal(s) * x).astype(f32) for s, x in (((vocab, dim), 1.0), ((dim, dim), 0.2), ((dim, dim), 0.2),
                                                                                ((dim, dim), 0.2), ((dim, vocab), 1.0)))
    ids = rng.integers(0, vocab, prompt)
    scale = 1 / np.sqrt(hd)
    x = table[ids][None]
    q, k, v = (D.fromHost((x @ w).astype(f32)) for w in (wq, wk, wv))
    full = ops.fusedAttentionForward(q, k, v, heads, scale, 0)
    weights = D.zeros((1, heads, cap))
    ops.attentionKeyWeights(q, k, full.m, full.l, heads, scale, 0, heads, weights)
    kc, vc = D.zeros((1, cap, dim)), D.zeros((1, cap, dim))
    hip.capi.call("bf_hip_kv_append", kc.ptr, vc.ptr, k.ptr, v.ptr, 1, prompt, dim, cap, 0, None)
    lengths = ints(hip, [prompt])
    ops.kvEvict(kc, vc, weights, lengths, heads, budget, recent)

    # the oracle's state after the prompt
    def heads_of(t):
        return t.astype(np.float64).reshape(-1, heads, hd).transpose(1, 0, 2)
    Q, K, V = (heads_of(t.toHost()[0]) for t in (q, k, v))
    s = np.where(np.tril(np.ones((prompt, prompt), bool)), Q @ K.transpose(0, 2, 1) * scale, -np.inf)
    P = np.exp(s - s.max(-1, keepdims=True))
    P /= P.sum(-1, keepdims=True)
    acc = P.sum(1)
    state = []
    for h in range(heads):
        rows = kept_rows(acc[h].astype(f32), prompt, budget, recent)
        state.append([K[h][rows], V[h][rows], acc[h][rows]])
    assert lengths.toHostInts().tolist() == [budget]
    wk_ = weights.toHost()[0, :, :budget]
    assert np.abs(wk_ - np.array([st[2] for st in state])).max() <= 1e-4     # 60 terms of at most 1, each off by some e times scores of a few tens

    token, committed = int(ids[-1]), budget
    for _ in range(6):
        parents = np.array([[-1, 0, 0, 1, 1, 2, 3]], np.int32)
        draft = rng.integers(0, vocab, nodes)
        draft[0] = token
        masks_host = hip.ops.treeVisibility(parents)

        def projected(tok):
            return [(table[tok] @ w).astype(f32) for w in (wq, wk, wv)]

        def step(rows):
            qn, kn, vn = (heads_of(t) for t in rows)
            sees = np.array([[int(masks_host[0, i]) >> j & 1 for j in range(nodes)] for i in range(nodes)], bool)
            o, got = np.zeros((nodes, heads, hd)), []
            for h in range(heads):
                sc = np.concatenate([qn[h] @ state[h][0].T, np.where(sees, qn[h] @ kn[h].T, -np.inf)], 1) * scale
                p = np.exp(sc - sc.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                o[:, h] = p @ np.concatenate([state[h][1], vn[h]])
                got.append(p.sum(0))
            return o.reshape(nodes, dim) @ wo.astype(np.float64), kn, vn, got
        for j in range(1, nodes):   # the greedy continuation is drafted in places, so that paths of several lengths are accepted
            if rng.random() < 0.75:
                draft[j] = int(np.argmax(step(projected(draft))[0][parents[0, j]]))
        rows = projected(draft)
        logits64, kn, vn, got = step(rows)
        margin = np.sort(logits64, 1)
        assert (margin[:, -1] - margin[:, -2]).min() > 1e-3      # no choice hangs on a rounding: fp32 logits of this size are good to 1e-5

        dq, dkn, dvn = (D.fromHost(t[None]) for t in rows)
        res = ops.attentionTreeWeights(dq, dkn, dvn, kc, vc, lengths, heads, scale, weights, visible=masks(hip, masks_host))
        logits = ops.matmul(res.output.reshaped((nodes, dim)), D.fromHost(wo)).reshaped((1, nodes, vocab))
        taken = ops.treeAccept(logits, D.fromHost(draft[None].astype(f32)), ints(hip, parents))
        ops.kvCommit([kc], [vc], [dkn], [dvn], taken, lengths, [weights])

        path, then = accept(logits64, draft, parents[0], nodes)
        assert taken.path.toHostInts()[0].tolist() == path + [-1] * (nodes - len(path)) and int(taken.next.toHost()[0]) == then
        for h in range(heads):
            n = len(state[h][0])
            state[h] = [np.concatenate([state[h][0], kn[h][path]]), np.concatenate([state[h][1], vn[h][path]]),
                        np.concatenate([state[h][2] + got[h][:n], got[h][n:][path]])]
        committed += len(path)
        assert lengths.toHostInts().tolist() == [committed]
        host = weights.toHost()[0, :, :committed]
        assert np.abs(host - np.array([st[2] for st in state])).max() <= 2e-4
        np.testing.assert_array_equal(kc.toHost()[0, :committed].reshape(committed, heads, hd).transpose(1, 0, 2), np.array([st[0] for st in state]).astype(f32))
        token = then


@pytest.mark.parametrize("nodes", [5, 40])
def test_captured_and_replayed(hip, rng, nodes):
    """A round of weights, verification, append and eviction recorded once and replayed, beside an eager run of the same."""
    D, call = hip.DeviceTensor, hip.capi.call
    batch, heads, hd, cap, vocab, budget = 2, 4, 64, 300, 200, 200
    dim = heads * hd

    def state():
        rng = np.random.default_rng(3)
        t = dict(q=D.fromHost(rng.standard_normal((batch, nodes, dim)).astype(f32)), kn=D.fromHost(rng.standard_normal((batch, nodes, dim)).astype(f32)),
                 vn=D.fromHost(rng.standard_normal((batch, nodes, dim)).astype(f32)), k=D.fromHost(rng.standard_normal((batch, cap, dim)).astype(f32)),
                 v=D.fromHost(rng.standard_normal((batch, cap, dim)).astype(f32)), w=D.fromHost(rng.random((batch, heads, cap)).astype(f32)),
                 out=D.zeros((batch, nodes, dim)), lengths=ints(hip, [190, 120]), logits=D.fromHost(rng.standard_normal((batch, nodes, vocab)).astype(f32)),
                 parents=ints(hip, [list(range(-1, nodes - 1))] * batch), path=ints(hip, np.zeros((batch, nodes))), found=ints(hip, [0] * batch), next=D.zeros((batch,)))
        logits, tokens = t["logits"].toHost(), rng.integers(0, vocab, (batch, nodes))
        for j in (1, 2):
            logits[:, j - 1][np.arange(batch), tokens[:, j]] = 30
        t["logits"], t["tokens"] = D.fromHost(logits), D.fromHost(tokens.astype(f32))
        return t

    def one(t, stream):
        call("bf_hip_attention_tree_weights", t["q"].ptr, t["kn"].ptr, t["vn"].ptr, t["k"].ptr, t["v"].ptr, t["lengths"].ptr, None, None, t["out"].ptr, None,
             None, t["w"].ptr, t["w"].ptr, batch, heads, heads, heads, nodes, cap, hd, 0.125, stream)
        call("bf_hip_tree_accept", t["logits"].ptr, t["tokens"].ptr, t["parents"].ptr, None, t["path"].ptr, t["found"].ptr, t["next"].ptr, batch, nodes, vocab,
             stream)
        arrays = [(ctypes.c_void_p * 1)(t[n].ptr) for n in ("k", "v", "kn", "vn", "w")]
        call("bf_hip_kv_commit", *arrays, 1, t["path"].ptr, t["found"].ptr, t["lengths"].ptr, t["lengths"].ptr, batch, heads, heads, nodes, cap, hd, stream)
        call("bf_hip_kv_evict", t["k"].ptr, t["v"].ptr, t["w"].ptr, t["lengths"].ptr, t["k"].ptr, t["v"].ptr, t["w"].ptr, t["lengths"].ptr, None, batch, heads,
             heads, hd, cap, cap, budget, 16, stream)

    stream = hip.Stream()
    eager, replayed = state(), state()
    hip.capi.call("bf_hip_synchronize")
    graph = ctypes.c_void_p()
    call("bf_hip_capture_begin", stream.handle)
    one(replayed, stream.handle)
    call("bf_hip_capture_end", ctypes.byref(graph))
    for step in range(5):
        one(eager, None)
        call("bf_hip_graph_launch", graph, stream.handle)
        call("bf_hip_synchronize")
        for name in ("out", "k", "v", "w", "next"):
            assert eager[name].toHost().tobytes() == replayed[name].toHost().tobytes(), f"step {step}: {name}"
        for name in ("lengths", "path", "found"):
            assert (eager[name].toHostInts() == replayed[name].toHostInts()).all(), f"step {step}: {name}"
    assert eager["lengths"].toHostInts().tolist() == [200, 135]
    call("bf_hip_graph_destroy", graph)


def test_rounds_on_alternating_streams(hip, rng):
    """Weights (workspace from the pool), verification, append and eviction, each on the other stream than the last."""
    call = hip.capi.call
    batch, heads, hd, cap, nodes, vocab, budget = 2, 4, 64, 3000, 40, 900, 2000
    dim = heads * hd
    host = dict(q=rng.standard_normal((batch, nodes, dim)), kn=rng.standard_normal((batch, nodes, dim)), vn=rng.standard_normal((batch, nodes, dim)),
                k=rng.standard_normal((batch, cap, dim)), v=rng.standard_normal((batch, cap, dim)), w=rng.random((batch, heads, cap)),
                logits=rng.standard_normal((batch, nodes, vocab)), tokens=np.zeros((batch, nodes)), out=np.zeros((batch, nodes, dim)), next=np.zeros(batch))
    host["logits"][:, :6, 0] = 30      # the model's choice is token 0 six times over

    def run(streams):
        t = {n: hip.DeviceTensor.fromHost(x.astype(f32)) for n, x in host.items()}
        t.update(lengths=ints(hip, [2900, 1990]), path=ints(hip, np.zeros((batch, nodes))), found=ints(hip, [0] * batch),
                 parents=ints(hip, [list(range(-1, nodes - 1))] * batch))
        arrays = [(ctypes.c_void_p * 1)(t[n].ptr) for n in ("k", "v", "kn", "vn", "w")]
        for step in range(4):
            s = [streams[(step + i) % len(streams)].handle for i in range(4)]
            call("bf_hip_attention_tree_weights", t["q"].ptr, t["kn"].ptr, t["vn"].ptr, t["k"].ptr, t["v"].ptr, t["lengths"].ptr, None, None, t["out"].ptr,
                 None, None, t["w"].ptr, t["w"].ptr, batch, heads, heads, heads, nodes, cap, hd, 0.125, s[0])
            call("bf_hip_tree_accept", t["logits"].ptr, t["tokens"].ptr, t["parents"].ptr, None, t["path"].ptr, t["found"].ptr, t["next"].ptr, batch, nodes,
                 vocab, s[1])
            call("bf_hip_kv_commit", *arrays, 1, t["path"].ptr, t["found"].ptr, t["lengths"].ptr, t["lengths"].ptr, batch, heads, heads, nodes, cap, hd, s[2])
            call("bf_hip_kv_evict", t["k"].ptr, t["v"].ptr, t["w"].ptr, t["lengths"].ptr, t["k"].ptr, t["v"].ptr, t["w"].ptr, t["lengths"].ptr, None, batch,
                 heads, heads, hd, cap, cap, budget, 16, s[3])
        call("bf_hip_synchronize")
        return {n: t[n].toHost().tobytes() for n in ("out", "k", "v", "w", "next")}, t["lengths"].toHostInts().tolist()

    want = run([hip.Stream()])
    assert want[1] == [2000, 2000]
    two = [hip.Stream(), hip.Stream()]
    for _ in range(3):
        assert run(two) == want


def test_caches_past_two_to_the_32_elements(hip, rng):
    """The last sequence of caches of 4.6e9 elements each: offsets past 32 bits in reading, moving and appending."""
    D, call = hip.DeviceTensor, hip.capi.call
    batch, heads, hd, cap, nodes, used = 35, 16, 128, 65536, 3, 700
    dim = heads * hd
    lengths = [0] * (batch - 1) + [used]
    q, kn, vn = ((rng.standard_normal((batch, nodes, dim))).astype(f32) for _ in range(3))
    last = [(rng.standard_normal((1, used, dim))).astype(f32) for _ in range(2)]
    k, v = D.zeros((batch, cap, dim)), D.zeros((batch, cap, dim))
    for t, rows in zip((k, v), last):
        call("bf_hip_memcpy_h2d", ctypes.c_void_p(t.ptr.value + 4 * (batch - 1) * cap * dim), rows.ctypes.data_as(ctypes.c_void_p), rows.nbytes)
    w = D.fromHost(rng.random((batch, 1, cap)).astype(f32))
    host_w = w.toHost()
    out, dl = D.zeros((batch, nodes, dim)), ints(hip, lengths)
    dq, dkn, dvn = D.fromHost(q), D.fromHost(kn), D.fromHost(vn)
    call("bf_hip_attention_tree", dq.ptr, dkn.ptr, dvn.ptr, k.ptr, v.ptr, dl.ptr, None, None, out.ptr, None, None, batch, heads, heads, nodes, cap, hd, 0.0883883,
         None)
    chain = np.array([[1, 3, 7]], np.uint64)
    want = reference(q[-1:], kn[-1:], vn[-1:], last[0], last[1], [used], [nodes], chain, heads, heads, 1, 0.0883883)
    worst = np.abs(out.toHost()[-1] - want[0][0]).max()
    assert worst <= 2 * want[4] * 5.5, worst
    path, found = ints(hip, np.tile([0, 1, 2], (batch, 1))), ints(hip, [0] * (batch - 1) + [3])
    arrays = [(ctypes.c_void_p * 1)(t.ptr) for t in (k, v, dkn, dvn)]
    call("bf_hip_kv_commit", *arrays, None, 1, path.ptr, found.ptr, dl.ptr, dl.ptr, batch, heads, 1, nodes, cap, hd, None)
    call("bf_hip_kv_evict", k.ptr, v.ptr, w.ptr, dl.ptr, k.ptr, v.ptr, w.ptr, dl.ptr, None, batch, heads, 1, hd, cap, cap, 300, 10, None)
    rows = kept_rows(host_w[-1, 0], used + nodes, 300, 10)
    for t, old, new in ((k, last[0], kn), (v, last[1], vn)):
        got = np.empty((300, dim), f32)
        call("bf_hip_memcpy_d2h", got.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(t.ptr.value + 4 * (batch - 1) * cap * dim), got.nbytes)
        np.testing.assert_array_equal(got, np.concatenate([old[0], new[-1]])[rows])
    assert dl.toHostInts().tolist() == [0] * (batch - 1) + [300]
    del k, v
    call("bf_hip_pool_trim")


def test_the_cpp_layer(hip):
    """tests/cpp/decode_cache_test.cpp: the same operators through namespace blackforge::backend::hip."""
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "blackforge_amd", "host", "bin", "decode_cache_test")
    assert os.path.exists(exe), "blackforge_amd/host has not been built"
    proc = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stdout + proc.stderr
