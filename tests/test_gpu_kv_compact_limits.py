"""Compaction of cached values at the end of f32's range, on the GPU against tests/kv_branch_ref.py."""
import numpy as np
import pytest

from tests.kv_branch_ref import BranchPair

pytestmark = pytest.mark.gpu

MOST = np.finfo(np.float32).max


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("style", ["pairs", "halves"])
def test_compact_of_the_largest_values(ctx, dim, style):
    """The scale of a block that holds f32's largest number, times 127, rounds past it: read back that is infinite,
    but the code and the scale stand for a number, which a compaction codes again as such."""
    assert 127.0 * float(np.float32(np.float64(MOST) / 127)) > float(MOST)
    p = BranchPair(ctx, 4, 2, dim, seqs=1, n_pages=20, page=32, style=style, seed=dim)
    q, k, v = p.rows(32 * 4)
    for x in (k, v):
        x[:64] *= MOST / (4 * np.abs(x[:64]).max())
        x[7, 0, 3], x[20, 0, 5], x[40, 1, 7] = MOST, -MOST, -MOST
    p.append([0], [32 * 4], (q, k, v))
    p.compact([0], [np.r_[1:128]])
    assert np.isfinite(p.ref.v[0].scales).all() and (np.abs(p.ref.v[0].codes) == 127).any()
    p.check_values()
    p.compact([0], [np.r_[:3, 5:127]])
    p.check_values()
    p.free()
