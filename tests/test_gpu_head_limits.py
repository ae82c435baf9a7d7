"""Log probabilities straight from a head and the rows' gradient where scales, weights and
probabilities come to their formats' ends, on the GPU against tests/head_ref.py."""
import numpy as np
import pytest

from tests.head_ref import U, TYPES, Head, forward, gradient
from tests.kv_ref import within
from tests.test_gpu_head import Call, check, rows_of, targets_of

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


@pytest.mark.parametrize("M", [1, 2, 3])
@pytest.mark.parametrize("V,K", [(700, 512), (1000, 1024), (333, 2048), (200, 2560)])
def test_columns_far_larger_than_the_rest(ctx, M, V, K):
    """Rows before a head have outliers: 256 columns are 10^5 times the others, which keep their bits.  Their weights
    are zeros, so the answer is that of the rows without them."""
    rng = np.random.default_rng(V)
    w = 0.05 * rng.standard_normal((V, K))
    w[:, 256:512] = 0
    head = Head(ctx, "q6_k", w)
    assert not head.values[:, 256:512].any()
    x, target = rows_of(M, K, seed=K), rng.integers(0, V, M)
    clean = x.copy()
    x[:, 256:512] *= 1e5
    clean[:, 256:512] = 0
    c = Call(head, x, target)
    c.forward()
    c.backward()
    got, dx = c.answers(), c.gradient()
    want, tol, _ = forward(head.values, clean, target)
    for n in got:
        within(got[n], want[n], tol[n])
    within(dx, *gradient(head.values, clean, target, np.ones(M)))
    c.free()
    head.free()


def likely_gradient(W, x, target):
    """(rows' gradient where targets are likelier than not, a bound for each value, one for each row's norm).

    1 - p of the target is the sum of the others' p, so its error is theirs, p_v each_v, and the sum's (96 roundings of
    it), however small it is.  The rest as in tests/head_ref.py: pairs of halves, 2^-40 of 1 at least, whose roundings
    of different entries are independent (the norm: four deviations of their sum, 2^-40 / sqrt 3 each at most)."""
    x = np.asarray(x, np.float64)
    _, _, more = forward(W, x, target)
    z, off, lse = more["z"], more["off"], more["lse"]
    d = z - lse[:, None]
    each = off + (more["tol_lse"] + 4 * U * np.abs(lse))[:, None] + (np.abs(d) + 8) * 2 * U
    p = np.exp(d)
    p[np.arange(len(x)), target] = 0
    rest, aw = p.sum(1, keepdims=True), np.abs(W)
    want = rest * W[target] - p @ W
    off = (p * each).sum(1, keepdims=True) + 96 * U * rest
    tol = off * aw[target] + (p * (each + 3 * 2.0 ** -22 + (len(W) / 16 + 128) * U)) @ aw \
        + rest * 2.0 ** -26 * aw.max() + 4 * U * np.abs(want)
    length = np.linalg.norm(tol, axis=1) + 4 * 2.0 ** -40 / 3 ** 0.5 * np.linalg.norm(W)
    return want, tol + 2.0 ** -40 * aw.sum(0), length


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,V,K", [(48, 3000, 512), (2, 3000, 512), (4, 9000, 512), (48, 13000, 1024)])
def test_all_but_certain_targets(ctx, kind, M, V, K):
    """A row's gradient keeps its bits where the target's 1 - p comes to 10^-7: neither the target's term nor the
    others' is lost.  (The logits' own errors, up to 10^-3 in these bounds, are what is left.)"""
    rng = np.random.default_rng(M)
    head = Head(ctx, kind, 0.05 * rng.standard_normal((V, K)))
    target = rng.integers(0, V, M)
    W = head.values[target]
    lean = np.linspace(8, 27, M) if M > 4 else np.linspace(19, 23, M)
    x = (rows_of(M, K, size=1.0) + lean[:, None] * W / (W ** 2).sum(1, keepdims=True)).astype(np.float32)
    c = Call(head, x, target)
    c.forward()
    c.backward()
    got, dx = c.answers(), c.gradient().astype(np.float64)
    c.free()
    want, tol, length = likely_gradient(head.values, x, target)
    exact = forward(head.values, x, target)[0]["logp"]
    likely = exact > np.log(0.5)
    within(dx[likely], want[likely], tol[likely])
    rows = (exact > -1e-4) & (exact < -1e-7)
    assert rows.sum() >= min(M, 4) / 2
    size = np.linalg.norm(want, axis=1)
    assert (length < 0.02 * size)[rows].all()  # (so a row without its target's term, or of zeros, fails)
    assert (np.linalg.norm(dx - want, axis=1) <= length)[rows].all()
    head.free()
