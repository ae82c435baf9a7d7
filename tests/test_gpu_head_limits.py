"""Log probabilities straight from a head and the rows' gradient where scales, weights and
probabilities come to their formats' ends, on the GPU against tests/head_ref.py."""
import numpy as np
import pytest

from tests.head_ref import Head
from tests.test_gpu_head import check, rows_of, targets_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["q4_0", "q4_1", "q8_0", "q6_k", "f16"])
@pytest.mark.parametrize("M", [2, 6, 40])
@pytest.mark.parametrize("top", [0, 3])
def test_smallest_scales(ctx, kind, M, top):
    """Heads whose largest block scale (F16: unit) is 2^-24, the smallest half, or 2^(top - 24), and some blocks
    are zeros."""
    rng = np.random.default_rng(M + top)
    lo, hi = {"q4_0": (-8, 7), "q4_1": (0, 15), "q8_0": (-127, 127), "q6_k": (-31, 31), "f16": (-100, 100)}[kind]
    w = rng.integers(lo, hi + 1, (700, 8, 32)).astype(np.float64)
    w[..., 0], w[..., 1] = lo, hi
    w[rng.random((700, 8)) < 0.2] = 0
    if kind == "q6_k":
        w *= 127  # (sixteen values' own scales are up to 127)
    head = Head(ctx, kind, w.reshape(700, 256) * 2.0 ** (top - 24))
    assert head.values.any()
    size = 2 / np.linalg.norm(head.values, axis=1).max()
    x = rows_of(M, 256, size=size)
    got, dx = check(head, x, targets_of(M, 700), np.ones(M))
    assert dx.any()
    head.free()


@pytest.mark.parametrize("M", [2, 100])
@pytest.mark.parametrize("scale", [1e-30, 1e-33])
def test_tiny_weights_as_pairs(ctx, M, scale):
    """F32 heads that become pairs of halves, all of whose weights are below 2^-97."""
    rng = np.random.default_rng(8)
    w = scale * rng.standard_normal((13000, 1024)) * np.logspace(-2, 0, 13000)[rng.permutation(13000)][:, None]
    head = Head(ctx, "f32", w)
    check(head, rows_of(M, 1024, size=0.05 / scale), targets_of(M, 13000), np.ones(M))
    head.free()
