"""Log probabilities, entropy and top tokens of rows of logits against 64-bit
numpy."""
import ctypes

import numpy as np
import pytest

import purebee_amd as pb

pytestmark = pytest.mark.gpu


def reference(x, targets, top):
    """(logp, entropy, ids, top logp, bounds of a kernel's error in the first
    two) in 64 bits.

    The bounds, for f32 with sums of at most 260 + 64 terms after another (2^-24
    each): e^d is off by 2^-22 + 2^-23 |d| relative, sums by 324 * 2^-24 more,
    logarithm and differences by an ulp of what they give."""
    x = np.asarray(x, np.float64)
    m, v = x.shape
    logp, ent = np.full(m, np.nan), np.full(m, np.nan)
    ids, tops = np.full((m, top), -1), np.full((m, top), np.nan)
    t1, t2 = np.ones(m), np.ones(m)
    for r in range(m):
        row = x[r]
        if np.isnan(row).any() or (row == np.inf).any() or (row == -np.inf).all():
            continue
        peak = row.max()
        d = row - peak
        p = np.exp(d)
        s = p.sum()
        lp = d - np.log(s)
        p /= s
        dd = np.where(p > 0, d, 0)
        if targets is not None and 0 <= targets[r] < v:
            logp[r] = lp[targets[r]]
        ent[r] = np.log(s) - (p * dd).sum()
        order = np.lexsort((np.arange(v), -row))[:top]
        ids[r], tops[r] = order, lp[order]
        chain = 324 * 2.0 ** -24
        rel = chain + 2.0 ** -22 + (p * np.abs(dd)).sum() * 2.0 ** -23
        big = 0 if not np.isfinite(logp[r]) else np.abs(logp[r]) + abs(x[r, targets[r]])
        t1[r] = rel + 2.0 ** -22 * (np.log(s) + abs(peak) * 2 + big + 1)
        rel2 = chain * 2 + 2.0 ** -20
        t2[r] = rel + 2.0 ** -22 * (np.log(s) + 1) + rel2 * -(p * dd).sum() + 2.0 ** -22 * (p * dd * dd).sum()
    return logp, ent, ids, tops, t1, t2


def run(ctx, x, targets, top, stride=None, skew=0):
    """The kernels' answers; logits `stride` floats apart from an address `skew`
    floats past a 16-byte border."""
    m, v = x.shape
    stride = stride or v
    host = np.full(skew + m * stride, np.nan, np.float32)  # NaN around the rows must not matter
    for r in range(m):
        host[skew + r * stride:][:v] = x[r]
    dx = ctx.alloc(host.nbytes).upload(host)
    dt = None if targets is None else ctx.alloc(4 * m).upload(np.asarray(targets, np.int32))
    size = ctx.logprobs_workspace(m, v, top)
    work = ctx.alloc(max(16, size)).upload(np.full(max(16, size), 0xff, np.uint8))
    guard = np.full(m * max(top, 1) + 16, 77.0, np.float32)
    dl, de, di, dp = (ctx.alloc(guard.nbytes).upload(guard) for _ in range(4))
    ctx.logprobs_dev(dx.ptr + 4 * skew, m, v, dt.ptr if dt else None, top, dl.ptr if dt else None, de.ptr, di.ptr,
                     dp.ptr, work.ptr, size, stride)
    ctx.sync()
    out = []
    for b, n, dtype in ((dl, m if dt else 0, np.float32), (de, m, np.float32), (di, m * top, np.int32),
                        (dp, m * top, np.float32)):
        got = b.download(np.float32, guard.size)
        assert (got[n:] == 77.0).all()  # nothing past the rows
        out.append(got[:n].view(dtype).copy())
        b.free()
    for b in (dx, dt, work):
        if b:
            b.free()
    return out[0], out[1], out[2].reshape(m, top), out[3].reshape(m, top)


def check(ctx, x, targets, top, **kw):
    logp, ent, ids, tops = run(ctx, x, targets, top, **kw)
    rl, re, ri, rt, t1, t2 = reference(x, targets, top)
    if targets is not None:
        near(logp, rl, t1)
    near(ent, re, t2)
    assert np.array_equal(ids, ri)
    near(tops, rt, t1[:, None] + np.zeros(rt.shape), 2.0 ** -22)


def near(got, want, tol, rel=0.0):
    """NaN and -inf where they are wanted, every other value to its bound."""
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got == -np.inf, want == -np.inf)
    ok = np.isfinite(want)
    over = np.abs(got[ok] - want[ok]) - tol[ok] - rel * np.abs(want[ok])
    assert not over.size or over.max() <= 0, f"{int((over > 0).sum())} of {over.size} values off by up to {over.max():.3g} more than allowed"


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 63, 64, 65, 257, 1000, 2049, 4097, 32003, 128256, 300001])
@pytest.mark.parametrize("rows", [1, 2, 37])
def test_shapes(ctx, rows, vocab):
    """Any vocabulary, odd ones among them (rows then start anywhere in a 16-byte group), one part or many."""
    if rows > 2 and vocab > 200000:
        rows = 5
    print(f"[case] logprobs {rows} x {vocab}", flush=True)
    rng = np.random.default_rng(vocab + rows)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    t = rng.integers(0, vocab, rows)
    for top in sorted({0, 1, min(5, vocab), min(32, vocab)}):
        check(ctx, x, t, top)


def test_many_rows(ctx):
    """One workgroup a row."""
    rng = np.random.default_rng(1)
    check(ctx, (rng.standard_normal((700, 5003)) * 2).astype(np.float32), rng.integers(0, 5003, 700), 20)


@pytest.mark.parametrize("skew", [0, 1, 2, 3])
@pytest.mark.parametrize("stride", [1003, 1004, 1100])
def test_strides_and_addresses(ctx, skew, stride):
    rng = np.random.default_rng(skew)
    check(ctx, rng.standard_normal((9, 1003)).astype(np.float32), rng.integers(0, 1003, 9), 7, stride=stride, skew=skew)


def test_equal_logits_go_to_the_lower_index(ctx):
    rng = np.random.default_rng(2)
    for v in (40, 5000, 128256):
        for kinds in (1, 2, 30):
            x = rng.integers(0, kinds, (3, v)).astype(np.float32)
            x[1] *= -1  # -0.0 equals 0.0
            check(ctx, x, [0, v // 2, v - 1], 32)
    check(ctx, np.zeros((600, 9000), np.float32), np.arange(600), 32)


@pytest.mark.parametrize("vocab", [8181, 8184, 8192, 8200, 131061, 131064, 131072, 131080])
def test_equal_logits_at_a_workgroups_share(ctx, vocab):
    """Rows of equal logits around the most that a workgroup takes: every element of the chosen threads is a candidate."""
    for rows in (600, 2):
        if rows * vocab > 1 << 25:
            rows = 257  # one workgroup a row as far as it can take one
        x = np.zeros((rows, vocab), np.float32)
        logp, ent, ids, tops = run(ctx, x, np.arange(rows), 32)
        assert np.array_equal(ids, np.tile(np.arange(32), (rows, 1)))
        # log of a sum of ones: f32 sums of up to 2^17 are exact, the logarithm and the entropy are an ulp off
        for got, want in ((logp, -np.log(vocab)), (tops, -np.log(vocab)), (ent, np.log(vocab))):
            assert np.abs(got - want).max() <= 2.0 ** -22 * np.log(vocab)


def test_sorted_rows(ctx):
    """Rising and falling rows: every thread's best lies at its end, or at its start."""
    x = np.linspace(-20, 20, 128256, dtype=np.float32)
    check(ctx, np.stack([x, x[::-1]]), [5, 9], 32)


def test_masked_logits(ctx):
    """-inf and the type's lowest value as masks: all but a few tokens, all but one, and everything."""
    rng = np.random.default_rng(3)
    low = np.finfo(np.float32).min
    for mask in (-np.inf, low):
        for v in (50, 3001, 128256):
            x = (rng.standard_normal((5, v)) * 2).astype(np.float32)
            keep = rng.choice(v, 7, replace=False)
            for r, n in ((0, 7), (1, 1), (2, 0)):
                row = np.full(v, mask, np.float32)
                row[keep[:n]] = x[r, keep[:n]]
                x[r] = row
            x[3, ::2] = mask
            check(ctx, x, [keep[0], keep[1], keep[2], 0, 1], 10)


def test_rows_without_a_distribution(ctx):
    """NaN and +inf spoil their own row."""
    rng = np.random.default_rng(4)
    for v in (33, 70000):
        x = rng.standard_normal((6, v)).astype(np.float32)
        x[1, 20], x[3, v - 1], x[4, 0] = np.nan, np.inf, np.nan
        x[4, 1] = np.inf
        logp, ent, ids, tops = run(ctx, x, [1] * 6, 4)
        spoilt = np.array([0, 1, 0, 1, 1, 0], bool)
        assert np.array_equal(np.isnan(logp), spoilt) and np.array_equal(np.isnan(ent), spoilt)
        assert (ids[spoilt] == -1).all() and np.isnan(tops[spoilt]).all()
        check(ctx, x, [1] * 6, 4)


def test_targets_outside_the_vocabulary_and_answers_left_out(ctx):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, 999)).astype(np.float32)
    check(ctx, x, [-1, 999, 2**31 - 1, 3], 3)
    check(ctx, x, None, 3)
    dx, o = ctx.alloc(x.nbytes).upload(x), ctx.alloc(4096)
    size = ctx.logprobs_workspace(4, 999, 0)
    w = ctx.alloc(max(16, size))
    ctx.logprobs_dev(dx.ptr, 4, 999, None, 0, None, o.ptr, None, None, w.ptr, size)
    ctx.logprobs_dev(dx.ptr, 0, 999, None, 0, None, o.ptr, None, None)
    ctx.sync()
    assert np.abs(o.download(np.float32, 4) - reference(x, None, 0)[1]).max() < 1e-4
    for b in (dx, o, w):
        b.free()


def test_extreme_values(ctx):
    """Rows far from zero, spread wide, and with one token that is certain."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((5, 2000)).astype(np.float32)
    x[0] += 1000
    x[1] *= 1e30
    x[2, 7] = 300
    x[3] = x[3] * 1e-30
    x[4] = -3e38
    check(ctx, x, [3, 4, 7, 6, 1999], 6)


def test_refusals(ctx):
    b = ctx.alloc(1 << 20)
    for rows, vocab, top in ((-1, 10, 0), (1, 0, 0), (1, 10, -1), (1, 10, 11), (1, 100, 33), (1, 1 << 29, 0),
                             (1 << 25, 10, 0)):
        with pytest.raises(pb.PbxError):
            ctx.logprobs_workspace(rows, vocab, top)
        with pytest.raises(pb.PbxError):
            ctx.logprobs_dev(b.ptr, rows, vocab, b.ptr, top, b.ptr, b.ptr, b.ptr, b.ptr, b.ptr, 1 << 20)
    size = ctx.logprobs_workspace(2, 100000, 4)
    assert size > 0
    for kw in (dict(dLogits=None), dict(dLogits=b.ptr + 2), dict(dTargets=None), dict(dLogp=None), dict(dWork=None),
               dict(work_bytes=size - 1), dict(dWork=b.ptr + 8), dict(stride=99999)):
        a = dict(dLogits=b.ptr, rows=2, vocab=100000, dTargets=b.ptr, top=4, dLogp=b.ptr, dEntropy=b.ptr,
                 dTopIds=b.ptr, dTopLogp=b.ptr, dWork=b.ptr, work_bytes=size)
        a.update(kw)
        with pytest.raises(pb.PbxError):
            ctx.logprobs_dev(**a)
    b.free()


def test_captured_calls_replay(ctx):
    """Both launches of a split row captured: every replay equals the eager call, with other calls of the same
    workspace and synchronisations between."""
    hip = ctypes.CDLL("libamdhip64.so")
    vp = ctypes.c_void_p
    hip.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    hip.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, ctypes.c_char_p, ctypes.c_size_t]
    hip.hipGraphLaunch.argtypes = [vp, vp]
    hip.hipGraphExecDestroy.argtypes = [vp]
    hip.hipGraphDestroy.argtypes = [vp]
    rng = np.random.default_rng(7)
    x = (3 * rng.standard_normal((2, 3, 50257))).astype(np.float32)
    dx = [ctx.alloc(x[i].nbytes).upload(x[i]) for i in range(2)]
    dt = ctx.alloc(12).upload(np.array([1, 50256, 9], np.int32))
    size = ctx.logprobs_workspace(3, 50257, 7)
    assert size > 0
    work, blank = ctx.alloc(size), np.full(48, 77, np.float32)
    outs = [ctx.alloc(blank.nbytes) for _ in range(4)]

    def call(i):
        ctx.logprobs_dev(dx[i].ptr, 3, 50257, dt.ptr, 7, *(o.ptr for o in outs), work.ptr, size)

    def answers():
        ctx.sync()
        return [o.download(np.uint32, 48) for o in outs]

    def clear():
        for o in outs:
            o.upload(blank)

    clear()
    call(0)
    eager = answers()
    clear()
    call(1)
    other = answers()
    stream, graph, gexec = vp(ctx.stream()), vp(), vp()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    call(0)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(gexec), graph, None, None, 0) == 0
    for rep in range(3):
        clear()
        assert hip.hipGraphLaunch(gexec, stream) == 0
        for got, want in zip(answers(), eager):
            assert np.array_equal(got, want), rep
        clear()
        call(1)
        for got, want in zip(answers(), other):
            assert np.array_equal(got, want), rep
    hip.hipGraphExecDestroy(gexec)
    hip.hipGraphDestroy(graph)
    for b in (*dx, dt, work, *outs):
        b.free()


def test_rows_around_where_they_are_split(ctx):
    """Vocabularies in one workgroup and in several, many rows over several workgroups each (joined in the same
    launch, or past 512 rows in a second one)."""
    rng = np.random.default_rng(8)
    for rows, vocab, top in ((3, 35999, 9), (3, 36000, 32), (3, 36001, 32), (200, 36003, 3), (2, 131075, 32)):
        print(f"[case] logprobs {rows} x {vocab}", flush=True)
        x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
        check(ctx, x, rng.integers(0, vocab, rows), top)
    x = np.tile((3 * rng.standard_normal((3, 131073))).astype(np.float32), (171, 1))  # 513 rows, two parts each
    assert ctx.logprobs_workspace(513, 131073, 2) > 0
    t = np.tile([5, 131072, 70000], 171)
    logp, ent, ids, tops = run(ctx, x, t, 2)
    rl, re, ri, rt, t1, t2 = reference(x[:3], t[:3], 2)
    for r in range(0, 513, 3):
        near(logp[r:r + 3], rl, t1)
        near(ent[r:r + 3], re, t2)
        assert np.array_equal(ids[r:r + 3], ri)
        near(tops[r:r + 3], rt, t1[:, None] + np.zeros(rt.shape), 2.0 ** -22)
