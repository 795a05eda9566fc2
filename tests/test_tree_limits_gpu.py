"""Tree attention under the largest norm weights that its header allows."""
import numpy as np
import pytest

import shv
import test_tree_gpu as G

pytestmark = pytest.mark.gpu
A = shv.api


@pytest.mark.parametrize("leads", [False, True])
@pytest.mark.parametrize("layout,norm,rows,pos,n_splits", [
    ((16, 2, 256, 0), 1500, 1, [3000, 700], 16), ((16, 2, 256, 0), 2000, 5, [2500], 3), ((16, 2, 256, 0), 2000, 64, [900], 7), ((12, 2, 128, 0), 2000, 9, [2500, 300], 16),
    ((8, 8, 64, 0), 2000, 33, [2500], 8), ((16, 2, 256, 0), 4000, 12, [900, 77], 5)])
def test_scores_of_the_largest_norm_weights(ctx, monkeypatch, layout, norm, rows, pos, n_splits, leads):
    """Scores past 2^24 powers of two, whose last places are several powers of two each: a row's output is a mean of the values it sees whatever its weights are, so between their
    smallest and their largest; where one cell leads by more than all roundings it is that cell's value.  Weights enter to 22 bits and sums of at most a hundred tiles are float32:
    2^-21 + 100 2^-24 < 1e-5 of the largest value."""
    monkeypatch.setitem(G.LAYOUTS, "own", layout)
    t = G.AttnTree(norm + rows + pos[0], "own", rows, pos)
    u = np.sign(t.rng.standard_normal(t.d)).astype(np.float32)
    t.q_norm[:] = t.k_norm[:] = norm
    t.qkv[:, :, :2 * t.nh * t.d].reshape(len(pos), rows, t.nh, 2, t.d)[:, :, :, 0] = u
    t.qkv[:, :, 2 * t.nh * t.d:2 * t.nh * t.d + t.nkv * t.d] = np.tile(np.where(np.arange(t.d) < 8, 1e-3, 1) * u, t.nkv)
    few = (0.03 * t.rng.standard_normal(t.kc.shape)).astype(np.float16)  # a few powers of two by the first dims
    t.kc[:] = np.where(np.arange(t.d) < 8, few, (norm * u).astype(np.float16))
    lead = [int(t.rng.integers(0, p)) for p in pos]
    if leads:
        for s, c in enumerate(lead):
            t.kc[t.slot[s], c] = (norm * u).astype(np.float16)
    t.upload(ctx)
    ctx.enqueue(A.OP_ATTN_TREE, t.args(ctx, n_splits))
    out, _, vx = t.results()
    for s in range(len(pos)):
        cells = t.vc[t.slot[s], :pos[s]].astype(np.float64)
        for i in range(rows):
            path, at = [], i
            while at >= 0:
                path.append(at)
                at = int(t.parent[s, at])
            v = np.concatenate([cells, vx[s, path].astype(np.float64)])
            got, tol = out[s, i].reshape(t.nkv, -1, t.d), 1e-5 * np.abs(v).max()
            low, high = (v[lead[s]], v[lead[s]]) if leads else (v.min(0), v.max(0))
            assert np.isfinite(got).all(), (s, i)
            assert (got >= low[:, None] - tol).all() and (got <= high[:, None] + tol).all(), (s, i)
