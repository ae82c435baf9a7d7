"""Log probabilities straight from a head's weights and the rows' gradient, on the GPU
against tests/head_ref.py."""
import ctypes

import numpy as np
import pytest

import purebee_amd as pb
from purebee_amd import native
from tests.head_ref import TYPES, Head, forward, gradient
from tests.kv_ref import Rows, within
from tests.test_gpu_kv_branch import Graph

pytestmark = pytest.mark.gpu


def head_of(ctx, kind, V, K, seed=0, std=0.05):
    return Head(ctx, kind, std * np.random.default_rng(seed).standard_normal((V, K)))


def rows_of(M, K, seed=1, size=1.5):
    return (size * np.random.default_rng(seed).standard_normal((M, K))).astype(np.float32)


class Call:
    """The two calls on M rows, with everything around outputs and workspace watched."""

    def __init__(self, head, x, target, grad=None):
        ctx = self.ctx = head.ctx
        self.head, self.M = head, len(x)
        M, K = x.shape
        self.x = Rows(ctx, M, K, x)
        self.target = ctx.alloc(4 * M + 4).upload(np.ascontiguousarray(target, np.int32))
        self.out = {n: Rows(ctx, 1, M) for n in ("logp", "entropy", "lse")}
        self.dx = Rows(ctx, M, K)
        self.grad = Rows(ctx, 1, M, np.ones(M) if grad is None else grad)
        self.bytes = [ctx.linear_logprobs_workspace(head.w, M, grad=g) for g in (False, True)]
        self.work = [ctx.alloc(n + 64).upload(np.full(n + 64, 0x7b, np.uint8)) for n in self.bytes]

    def forward(self, logp=True, entropy=True, lse=True):
        self.ctx.linear_logprobs_dev(self.head.w, self.x.ptr, self.M, self.target.ptr if logp else None,
                                     self.out["logp"].ptr if logp else None,
                                     self.out["entropy"].ptr if entropy else None,
                                     self.out["lse"].ptr if lse else None, self.work[0].ptr, self.bytes[0])

    def backward(self):
        self.ctx.linear_logprobs_grad_dev(self.head.w, self.x.ptr, self.M, self.target.ptr, self.out["lse"].ptr,
                                          self.grad.ptr, self.dx.ptr, self.work[1].ptr, self.bytes[1])

    def answers(self):
        self.ctx.sync()
        for n, w in zip(self.bytes, self.work):
            assert (w.download(np.uint8, n + 64)[n:] == 0x7b).all(), "written past the workspace"
        self.x.get()
        return {n: r.get()[0] for n, r in self.out.items()}

    def gradient(self):
        self.ctx.sync()
        return self.dx.get()

    def free(self):
        for r in (self.x, self.target, self.dx, self.grad, *self.out.values(), *self.work):
            r.free()


def check(head, x, target, grad):
    c = Call(head, x, target, grad)
    c.forward()
    c.backward()
    got, dx = c.answers(), c.gradient()
    want, tol, _ = forward(head.values, x, target)
    for n in got:
        assert np.array_equal(np.isnan(got[n]), np.isnan(want[n])), n
        within(got[n], want[n], tol[n])
    want, tol = gradient(head.values, x, target, grad)
    within(dx, want, tol)
    assert not np.isnan(dx).any()
    c.free()
    return got, dx


def targets_of(M, V, seed=2):
    rng = np.random.default_rng(seed)
    t = rng.integers(0, V, M)
    if M > 4:
        t[rng.integers(0, M, 2)] = [-1, V]  # rows without a target
    return t


SHAPES = [(1, 1, 32), (2, 5, 64), (3, 64, 96), (1, 1000, 288), (3, 513, 2048), (4, 63, 32), (5, 65, 160),
          (16, 1000, 576), (17, 129, 32), (31, 4097, 64), (32, 300, 1056), (33, 128, 32), (40, 1003, 288),
          (64, 2000, 576), (65, 127, 64), (100, 8193, 96), (129, 640, 2048), (300, 1111, 160)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,V,K", SHAPES)
def test_scores_and_gradient(ctx, kind, M, V, K):
    if kind == "q6_k":
        K = (K + 255) // 256 * 256
    print(f"[case] head {kind} {M} x {V} x {K}", flush=True)
    head = head_of(ctx, kind, V, K, seed=V + K)
    grad = np.random.default_rng(3).standard_normal(M)
    check(head, rows_of(M, K, seed=M), targets_of(M, V), grad)
    head.free()


# few rows of large vocabularies, where the GEMM's epilogue takes the logits
WIDE = [(1, 13001, 32), (2, 24705, 64), (3, 7999, 32), (17, 8001, 288), (32, 16005, 64), (5, 25000, 1056), (31, 7777, 512)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,V,K", WIDE)
def test_few_rows_of_large_vocabularies(ctx, kind, M, V, K):
    test_scores_and_gradient(ctx, kind, M, V, K)


@pytest.mark.parametrize("M", [1, 2, 3])
@pytest.mark.parametrize("V,K", [(1, 256), (3, 512), (4097, 768), (999, 1024), (514, 1280), (131, 2048), (70, 2304),
                                 (13, 4096), (37, 16384), (13000, 256)])
def test_few_rows_of_q6_k(ctx, M, V, K):
    """Superblocks that fill an eighth of a wave to eight passes of it."""
    test_scores_and_gradient(ctx, "q6_k", M, V, K)


# heads that become pairs of halves on the way
@pytest.mark.parametrize("kind,M,V,K", [("f32", 2, 20011, 512), ("f32", 40, 20011, 512), ("f32", 33, 19999, 544),
                                        ("f32", 130, 5000, 2048), ("f32", 700, 999, 1024), ("q6_k", 100, 20011, 512),
                                        ("q6_k", 33, 16001, 768), ("q6_k", 330, 9001, 2304), ("f32", 2, 70001, 512),
                                        ("q6_k", 96, 70001, 512)])
def test_heads_as_pairs(ctx, kind, M, V, K):
    test_scores_and_gradient(ctx, kind, M, V, K)


@pytest.mark.parametrize("kind", ["f32", "q6_k"])
def test_rows_of_very_different_size_as_pairs(ctx, kind):
    """Every vocabulary entry keeps its bits, however small its weights; rows of zeros; huge and tiny heads."""
    rng = np.random.default_rng(6)
    w = rng.standard_normal((13000, 1024)).astype(np.float32)
    w *= np.logspace(-4, 0, 13000)[rng.permutation(13000)][:, None].astype(np.float32)
    w[::97] = 0
    for scale in (0.05, 3e-5 if kind == "q6_k" else 1e-20, 50.0 if kind == "q6_k" else 1e15) + \
            ((1e-28,) if kind == "f32" else ()):
        head = Head(ctx, kind, scale * w)
        check(head, rows_of(100, 1024, size=0.05 / scale), targets_of(100, 13000), np.ones(100))
        head.free()


@pytest.mark.parametrize("kind", ["q8_0", "f16", "f32", "q6_k"])
def test_many_pieces(ctx, kind):
    """A vocabulary of several pieces and a ragged last one."""
    M, V, K = 1500, 30011, 256 if kind == "q6_k" else 32
    head = head_of(ctx, kind, V, K, std=0.2)
    target = targets_of(M, V)
    target[:4] = [0, V - 1, 11135, 11136]
    check(head, rows_of(M, K), target, np.full(M, -1.0 / M))
    head.free()


@pytest.mark.parametrize("kind", list(TYPES))
def test_likely_targets(ctx, kind):
    """Rows that lean on their target's weights, from unlikely to all but certain."""
    M, V, K = 48, 3000, 512
    head = head_of(ctx, kind, V, K)
    target = np.random.default_rng(5).integers(0, V, M)
    W = head.values[target]
    x = rows_of(M, K, size=1.0) + np.linspace(0, 30, M)[:, None] * W / (W ** 2).sum(1, keepdims=True)
    got, _ = check(head, x.astype(np.float32), target, np.ones(M))
    assert got["logp"].max() > -1e-4 and got["logp"].min() < -5
    head.free()


@pytest.mark.parametrize("M", [1, 3, 8, 40, 200])
@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "f32"])
def test_rows_that_differ_by_orders(ctx, kind, M):
    """Huge and tiny rows and zeros beside ordinary ones; logits far apart."""
    head = head_of(ctx, kind, 700, 256)
    x = rows_of(M, 256) * np.logspace(-6, 2.5, M)[:, None].astype(np.float32)
    x[M // 2] = 0
    check(head, x, targets_of(M, 700), np.ones(M))
    head.free()


@pytest.mark.parametrize("kind", list(TYPES))
def test_heads_of_other_sizes(ctx, kind):
    """Heads whose weights are far from 1, whose rows differ, and one of zeros."""
    rng = np.random.default_rng(7)
    w = rng.standard_normal((900, 256))
    for scale, size in ((1e-5, 1e4), (300.0, 1e-3)):
        if kind in ("q4_0", "q4_1", "q8_0") and scale < 1e-4:
            scale, size = 1e-4, 1e3  # (scales of blocks are fp16: what they are below that the file decides)
        head = Head(ctx, kind, scale * w)
        check(head, rows_of(40, 256, size=size), targets_of(40, 900), np.ones(40))
        check(head, rows_of(3, 256, size=size), targets_of(3, 900), np.ones(3))
        head.free()
    head = Head(ctx, kind, w * np.logspace(-3, 0, 900)[:, None] * 0.1)
    check(head, rows_of(40, 256), targets_of(40, 900), np.ones(40))
    head.free()
    head = Head(ctx, kind, 0 * w)
    got, dx = check(head, rows_of(40, 256), targets_of(40, 900), np.ones(40))
    assert not dx.any() and np.allclose(got["lse"], np.log(900), rtol=1e-6)
    head.free()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M", [2, 6, 70])
def test_rows_without_a_distribution(ctx, kind, M):
    """NaN and infinite activations answer NaN in their own row and nowhere else."""
    head = head_of(ctx, kind, 500, 256)
    x, target, grad = rows_of(M, 256), np.arange(M), np.ones(M)
    clean = Call(head, x, target, grad)
    clean.forward()
    clean.backward()
    a, da = clean.answers(), clean.gradient()
    bad = x.copy()
    bad[0, 7] = np.nan
    if M > 2:
        bad[3, 100] = np.inf
    dirty = Call(head, bad, target, grad)
    dirty.forward()
    dirty.backward()
    b, db = dirty.answers(), dirty.gradient()
    rows = [0, 3] if M > 2 else [0]
    for n in a:
        assert np.isnan(b[n][rows]).all()
        assert np.array_equal(np.delete(a[n], rows), np.delete(b[n], rows))
    assert np.isnan(db[rows]).all()
    assert np.array_equal(np.delete(da, rows, 0), np.delete(db, rows, 0))
    clean.free()
    dirty.free()
    head.free()


def test_answers_left_out(ctx):
    head = head_of(ctx, "q8_0", 500, 64)
    for M in (1, 5, 50):
        c = Call(head, rows_of(M, 64), targets_of(M, 500))
        c.forward()
        all_ = c.answers()
        for pick in ({"logp": False}, {"entropy": False}, {"lse": False}, {"logp": False, "entropy": False}):
            for n, r in c.out.items():
                r.buf.upload(r.host)
            c.forward(**pick)
            got = c.answers()
            for n in got:
                if pick.get(n, True):
                    assert np.array_equal(got[n], all_[n], equal_nan=True)
                else:
                    assert (got[n] == 12345.25).all()
        c.free()
    head.free()


def test_gradient_against_differences(ctx):
    """Along random directions: differences of the kernel's own log probabilities."""
    M, V, K = 24, 700, 288
    head = head_of(ctx, "q8_0", V, K)
    x, target = rows_of(M, K), np.random.default_rng(2).integers(0, V, M)
    c = Call(head, x, target)
    c.forward()
    c.backward()
    dx = c.gradient().astype(np.float64)
    c.free()
    u = np.random.default_rng(9).standard_normal((M, K))
    u /= np.linalg.norm(u, axis=1, keepdims=True)
    eps, logp, tol = 2.0 ** -3, [], []
    for sign in (1, -1):
        y = (x + sign * eps * u).astype(np.float32)
        c = Call(head, y, target)
        c.forward()
        logp.append(c.answers()["logp"].astype(np.float64))
        _, t, _ = forward(head.values, y, target)
        # (y is rounded: the step is off by up to 2^-24 of it, the log probability by as much times its gradient)
        tol.append(t["logp"] + 2.0 ** -24 * np.abs(y).max() * 2 * np.abs(head.values).sum(1).max())
        c.free()
    # the difference is the derivative up to eps^2 / 6 of the third one, which for log softmax is at most
    # 8 (max |W u|)^3: the third cumulant of numbers in [-a, a] is at most (2 a)^3
    a = np.abs(u @ head.values.T).max(1)
    within((logp[0] - logp[1]) / (2 * eps), (dx * u).sum(1),
           (tol[0] + tol[1]) / (2 * eps) + eps ** 2 / 6 * 8 * a ** 3 + 1e-4 * np.abs(dx * u).sum(1))
    head.free()


@pytest.mark.parametrize("kind", ["q4_0", "q6_k", "f32"])
@pytest.mark.parametrize("M", [1, 20, 90])
def test_captured_calls(ctx, kind, M):
    """Replays, with eager work between them, give what eager calls give, bit for bit."""
    head = head_of(ctx, kind, 1500, 256)
    c = Call(head, rows_of(M, 256), targets_of(M, 1500), np.linspace(-1, 1, M))
    c.forward()
    c.backward()
    a, da = c.answers(), c.gradient()
    other = Call(head, rows_of(M + 1, 256, seed=8), targets_of(M + 1, 1500))
    g = Graph(ctx, lambda: (c.forward(), c.backward()))
    for _ in range(3):
        c.dx.buf.upload(c.dx.host)
        for r in c.out.values():
            r.buf.upload(r.host)
        other.forward()
        other.backward()
        g.launch()
        ctx.sync()
        b, db = c.answers(), c.gradient()
        assert all(np.array_equal(a[n], b[n], equal_nan=True) for n in a) and np.array_equal(da, db)
    g.free()
    c.free()
    other.free()
    head.free()


def test_nothing_is_allocated(ctx):
    """The calls live in the caller's workspace: the context's own does not grow."""
    head = head_of(ctx, "q4_0", 70000, 64)
    c = Call(head, rows_of(300, 64), targets_of(300, 70000))
    before = ctx.workspace_info()
    c.forward()
    c.backward()
    ctx.sync()
    assert ctx.workspace_info() == before
    c.free()
    head.free()


def test_refusals(ctx):
    head = head_of(ctx, "q8_0", 100, 64)
    c = Call(head, rows_of(5, 64), targets_of(5, 100))
    w, x, t, lse, dx, g = head.w, c.x.ptr, c.target.ptr, c.out["lse"].ptr, c.dx.ptr, c.grad.ptr
    logp, ws, n0, n1 = c.out["logp"].ptr, [b.ptr for b in c.work], c.bytes[0], c.bytes[1]

    def refused(code, match, f, *args):
        with pytest.raises(pb.PbxError, match=match) as e:
            f(*args)
        assert e.value.code == code

    f, b = ctx.linear_logprobs_dev, ctx.linear_logprobs_grad_dev
    refused(-1, "rows", f, w, x, -1, t, logp, None, lse, ws[0], n0)
    refused(-5, "rows", f, w, x, 65536, t, logp, None, lse, ws[0], n0)
    refused(-1, "16-byte", f, w, None, 5, t, logp, None, lse, ws[0], n0)
    refused(-1, "16-byte", f, w, x + 4, 5, t, logp, None, lse, ws[0], n0)
    refused(-1, "together", f, w, x, 5, None, logp, None, lse, ws[0], n0)
    refused(-1, "together", f, w, x, 5, t, None, None, lse, ws[0], n0)
    refused(-1, "workspace", f, w, x, 5, t, logp, None, lse, None, n0)
    refused(-1, "workspace", f, w, x, 5, t, logp, None, lse, ws[0], n0 - 1)
    refused(-1, "workspace", f, w, x, 5, t, logp, None, lse, ws[0] + 16, n0)
    refused(-1, "16-byte", b, w, x, 5, t, lse, g, None, ws[1], n1)
    refused(-1, "16-byte", b, w, x, 5, t, lse, g, dx + 4, ws[1], n1)
    for args in ((None, lse, g), (t, None, g), (t, lse, None)):
        refused(-1, "NULL", b, w, x, 5, *args, dx, ws[1], n1)
    refused(-1, "workspace", b, w, x, 5, t, lse, g, dx, ws[1], n1 - 1)
    refused(-1, "dX itself", b, w, x, 5, t, lse, g, x, ws[1], n1)
    q, s = pb.quantize_q8_ref(np.ones((32, 64), np.float32))
    ref = ctx.upload_q8ref(32, 64, q, s)
    refused(-5, "Q8_REF", f, ref, x, 1, t, logp, None, lse, ws[0], n0)
    refused(-5, "Q8_REF", ctx.linear_logprobs_workspace, ref, 1)
    ref.free()
    dead = native.Weight(ctx, None, 8, 1, 32)
    refused(-1, "live weight", f, dead, x, 1, t, logp, None, lse, ws[0], n0)
    refused(-1, "live weight", ctx.linear_logprobs_workspace, dead, 1)
    assert ctx.L.pbx_linear_logprobs_workspace(ctx._p, w.ptr, 5, 0, None) == -1
    size = ctypes.c_size_t(7)
    assert ctx.L.pbx_linear_logprobs_workspace(ctx._p, w.ptr, 0, 1, ctypes.byref(size)) == 0 and size.value == 0
    f(w, None, 0, None, None, None, None, None, 0)  # no rows: nothing is looked at
    b(w, None, 0, None, None, None, None, None, 0)
    assert (c.answers()["lse"] == 12345.25).all() and (c.gradient() == 12345.25).all()
    c.free()
    head.free()
