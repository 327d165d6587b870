"""Tangent caches of points where the maps take their other branches (beyond the rim, all alike, at the
origin), for rows that are read four values a load and for rows that are not: the oracle's bits."""
import numpy as np
import pytest

import oracle as O

rv = pytest.importorskip("ruvector_amd")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [3, 4, 13, 20, 64])
@pytest.mark.parametrize("kind", ["ball", "rim", "opposite", "alike", "origin"])
def test_centroid(d, kind):
    g = np.random.default_rng(d)
    x = g.normal(size=(700, d)).astype(np.float32)
    x /= np.linalg.norm(x, axis=1, keepdims=True)
    if kind == "ball":
        x *= (0.9 * g.random((700, 1))).astype(np.float32)
    elif kind == "opposite":
        x = np.where(np.arange(700)[:, None] % 2, x[:1], -x[:1]).astype(np.float32)
    elif kind == "alike":
        x[:] = x[0] * np.float32(0.4)
    elif kind == "origin":
        x *= np.float32(1e-6)
        x[::3] = 0
    h, o = rv.HyperbolicHnsw(rv.HyperbolicHnswConfig(seed=3)), O.Hyp(d, seed=3)
    h.insert_batch(x)
    o.insert(x)
    h.build_tangent_cache()
    o.build_tangent_cache()
    assert np.array_equal(h.tangent_centroid(), o.centroid())
    if d % 4 == 0:
        ids, dist, _ = h.search_with_pruning_batch(x[:40] * np.float32(0.9), 5)
        rids, rd = o.search_with_pruning(x[:40] * np.float32(0.9), 5)
        assert np.array_equal(dist, rd)
        if kind in ("ball", "rim"):
            assert np.array_equal(ids, rids)
