"""GPU tests of the cache operators over several layers that share their sequences' lengths, and at sizes with nothing in them."""
import os
import subprocess

import numpy as np
import pytest

from test_gpu_decode_cache import ints, kept_rows

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
