"""Log probabilities straight from a head and the rows' gradient at the ends of the pieces that a vocabulary is taken
in, and of rows with outliers, on the GPU against tests/head_ref.py."""
import numpy as np
import pytest

from tests.head_ref import TYPES, Head, forward, gradient
from tests.kv_ref import within
from tests.test_gpu_head import Call, check, rows_of
from tests.test_gpu_head_limits import likely_gradient

pytestmark = pytest.mark.gpu

# 64 MB of factors a piece, rows padded to 64: 1,500 rows are 1,536, so pieces of 10,880 entries
EDGES = [0, 10879, 10880, 10881, 21759, 21760, 30010]


@pytest.mark.parametrize("kind", list(TYPES))
def test_targets_at_the_ends_of_pieces(ctx, kind):
    """Ordinary targets and all but certain ones, whose sums of other entries come from every piece."""
    M, V, K = 1500, 30011, 256 if kind == "q6_k" else 32
    head = Head(ctx, kind, 0.2 * np.random.default_rng(1).standard_normal((V, K)))
    x, target = rows_of(M, K), np.random.default_rng(2).integers(0, V, M)
    n = len(EDGES)
    target[:3 * n] = EDGES * 3
    W = head.values[target[n:3 * n]]
    lean = np.repeat([12.0, 25.0], n)[:, None]  # likely, and likelier
    x[n:3 * n] = 0.2 * x[n:3 * n] + lean * W / (W ** 2).sum(1, keepdims=True)
    grad = np.ones(M)
    c = Call(head, x, target, grad)
    c.forward()
    c.backward()
    got, dx = c.answers(), c.gradient()
    c.free()
    few = slice(0, 3 * n + 20)
    want, tol, _ = forward(head.values, x[few], target[few])
    for name in got:
        within(got[name][few], want[name], tol[name])
    within(dx[few], *gradient(head.values, x[few], target[few], grad[few]))
    likely = np.flatnonzero(want["logp"] > np.log(0.5))
    assert len(likely) >= n
    want, tol, _ = likely_gradient(head.values, x[likely], target[likely])
    within(dx[likely], want, tol)
    head.free()


@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "f32"])
def test_one_row_of_several_pieces(ctx, kind):
    """Logits that are written, 262,144 a piece: kernels of their own for the gradient's first factor."""
    V, K = 600011, 32
    head = Head(ctx, kind, 0.2 * np.random.default_rng(1).standard_normal((V, K)))
    for t in (0, 262143, 262144, 524287, 524288, V - 1):
        check(head, rows_of(1, K, seed=t), np.array([t]), np.ones(1))
        W = head.values[t]
        x = (0.2 * rows_of(1, K, seed=t) + 24 * W / (W ** 2).sum()).astype(np.float32)
        _, dx = check(head, x, np.array([t]), np.ones(1))
        if forward(head.values, x, [t])[0]["logp"][0] > np.log(0.5):
            want, tol, _ = likely_gradient(head.values, x, np.array([t]))
            within(dx, want, tol)
    head.free()


@pytest.mark.parametrize("kind,M,V,K", [(kind, M, 700, 512) for kind in TYPES for M in (1, 2, 5, 40, 130)] +
                         [("f32", 2, 20011, 512), ("f32", 40, 20011, 512), ("q6_k", 100, 20011, 512),
                          ("q8_0", 2, 25000, 512), ("f16", 1, 13000, 512), ("q4_0", 20, 13000, 512)])
def test_columns_far_larger_than_the_rest(ctx, kind, M, V, K):
    """256 columns are 10^4 times the others, which keep their bits: the weights there are zeros, so the answer is that
    of the rows without them, to its own bounds (a pair of halves is good to 2^-39 of a row's largest, 10^-7)."""
    rng = np.random.default_rng(V)
    w = 0.05 * rng.standard_normal((V, K))
    w[:, 256:512] = 0
    head = Head(ctx, kind, w)
    assert not head.values[:, 256:512].any()
    x, target = rows_of(M, K, seed=K), rng.integers(0, V, M)
    clean = x.copy()
    x[:, 256:512] *= 1e4
    clean[:, 256:512] = 0
    c = Call(head, x, target)
    c.forward()
    c.backward()
    got, dx = c.answers(), c.gradient()
    c.free()
    want, tol, _ = forward(head.values, clean, target)
    for n in got:
        within(got[n], want[n], tol[n])
    within(dx, *gradient(head.values, clean, target, np.ones(M)))
    head.free()
