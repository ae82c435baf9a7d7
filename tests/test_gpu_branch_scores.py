"""Branches, compaction and scores from a head's weights run together, as a search over continuations and a trainer use
them: every step against 64 bits."""
import numpy as np
import pytest

import purebee_amd as pb
from tests.kv_branch_ref import BranchPair
from tests.kv_ref import Rows, within
from tests.test_gpu_head import Call, check, head_of
from tests.head_ref import forward
from tests.test_gpu_model_kv import CONFIGS, TOL, Server
from tests.conftest import rel_l2
from tests.test_gpu_logprobs import near, reference

pytestmark = pytest.mark.gpu


def attention(p, seqs, starts, counts, q):
    """Attention in 64 bits and its bound, with what tests/kv_ref.py's leaves out: a block's probabilities are fp16 pairs
    times 2^6 against the block's largest rounded up to a power of two (at most twice it), and pairs of
    values below 2^6 end at fp16's least step, 2^-24, so each is off by half a step, 2^-25 / 2^6 of that power, at most
    2^-30 of the block's largest.  That is seen where the row's strong key has the value 0 and all else is small."""
    want, tol = p.ref.attention(seqs, starts, counts, q)
    group, r = p.heads // p.kv_heads, 0
    for s, a, n in zip(seqs, starts, counts):
        k, v = (x[s].values().astype(np.float64) for x in (p.ref.k, p.ref.v))
        for t in range(n):
            for h in range(p.heads):
                x = k[:a + t + 1, h // group] @ q[r + t, h].astype(np.float64) / np.sqrt(p.dim)
                w = np.exp(x - x.max())
                w /= w.sum()
                for at in range(0, len(w), 32):
                    tol[r + t, h] += 2.0 ** -30 * w[at:at + 32].max() * np.abs(v[at:at + 32, h // group][:len(w) - at]).sum(0)
        r += n
    return want, tol


@pytest.mark.parametrize("heads,kv_heads,dim,kind", [(4, 2, 64, "q8_0"), (8, 1, 32, "f16"), (4, 4, 96, "f32"),
                                                    (2, 1, 256, "q6_k")])
def test_a_search_over_branches(ctx, heads, kv_heads, dim, kind):
    """Attention's rows go to the head where they are; the likelier half of the branches is forked over the others, all
    of them forget their middle, and the last rows have their gradient."""
    rng = np.random.default_rng(7)
    p = BranchPair(ctx, heads, kv_heads, dim, seqs=4, page=64, n_pages=24, seed=3)
    K = heads * dim
    head = head_of(ctx, kind, 777, K, std=1.0)
    p.append([0], [90])
    p.fork([1, 2, 3], [0, 0, 0])
    total = np.zeros(4)
    for step, n in enumerate((1, 3, 1)):
        seqs, counts = [2, 0, 3, 1], [n] * 4
        starts = [p.ref.length(s) for s in seqs]
        q, k, v = p.rows(4 * n, 3.0)
        rows = 4 * n
        target = rng.integers(0, head.N, rows).astype(np.int32)
        b = p.cache.batch(seqs, counts)
        w = kv_heads * dim
        dq, dk, dv = Rows(ctx, rows, K, q), Rows(ctx, rows, w, k), Rows(ctx, rows, w, v)
        turned = Rows(ctx, rows, K)
        c = Call(head, np.zeros((rows, K), np.float32), target)
        # append, attention and scores on one stream, with nothing between them
        b.append_dev(0, dq.ptr, dk.ptr, dv.ptr, turned.ptr)
        b.attention_dev(0, turned.ptr, c.x.ptr)
        c.forward()
        ctx.sync()
        tq = turned.get().reshape(q.shape)
        want = p.ref.append(seqs, counts, q, k, v)
        within(tq, want, 2.0 ** -24 * np.abs(want) + 1e-14 * np.abs(q).max())  # one rounding of 64-bit sums
        x = c.x.get()
        want, tol = attention(p, seqs, starts, counts, tq)
        within(x.reshape(want.shape), want, tol)
        logp, tol, _ = forward(head.values, x, target)
        got = c.out["logp"].get()[0]
        within(got, logp["logp"], tol["logp"])
        for i, s in enumerate(seqs):
            total[s] += got[i * n:(i + 1) * n].sum()
        for r in (c, dq, dk, dv, turned, b):
            r.free()
        best = list(np.argsort(-total)[:2])
        rest = [s for s in range(4) if s not in best]
        p.fork(rest, best)
        total[rest] = total[best]
        p.check_values()
    lengths = [p.ref.length(s) for s in range(4)]
    p.compact([3, 1, 0, 2], [np.r_[:4, n - 40:n] for n in (lengths[s] for s in (3, 1, 0, 2))])
    p.check_values()
    starts = [p.ref.length(s) for s in range(4)]
    b, q = p.append([0, 1, 2, 3], [2, 1, 40, 1])
    dq, do = Rows(ctx, 44, K, q), Rows(ctx, 44, K)
    b.attention_dev(0, dq.ptr, do.ptr)
    ctx.sync()
    x = do.get()
    want, tol = attention(p, [0, 1, 2, 3], starts, [2, 1, 40, 1], q)
    within(x.reshape(want.shape), want, tol)
    for r in (dq, do, b):
        r.free()
    # of each branch the rows but its last are trained on
    target = rng.integers(0, head.N, 44)
    target[[1, 2, 42, 43]] = -1
    check(head, x, target, -rng.random(44).astype(np.float32))
    for s in range(4):
        p.truncate(s, 0)
    assert p.cache.info()["free_pages"] == 24
    head.free()
    p.free()


@pytest.mark.parametrize("name", ["f32", "q8_0"])
def test_a_models_branches(ctx, name):
    """Model.forward_kv over a prompt's branches and over sequences that were compacted."""
    cfg = CONFIGS[name]
    rng = np.random.default_rng(61)
    s = Server(ctx, cfg, seqs=4, n_pages=16)
    b = pb.KvBatch(s.cache)

    def step(seqs, counts, targets=None):
        starts = [s.cache.length(i) for i in seqs]
        tokens = rng.integers(0, cfg["vocab_size"], sum(counts)).astype(np.int32)
        got = s.model.forward_kv(b.set(seqs, counts), tokens, all_rows=True, targets=targets)
        want = s.expect(seqs, starts, counts, tokens)
        assert all(rel_l2(g, w) <= TOL for g, w in zip(got[0], want))
        assert np.array_equal(got[1], got[0].argmax(-1))
        if targets is not None:
            logp, ent, _, _, t1, t2 = reference(got[0], np.asarray(targets), 0)
            near(got[2]["logp"], logp, t1)
            near(got[2]["entropy"], ent, t2)

    def fork(dsts, srcs, lengths=None):
        s.cache.fork(dsts, srcs, lengths)
        n = s.appends.copy()
        for d, i in zip(dsts, srcs):
            for (seq, blk), count in n.items():
                if seq == i:
                    s.appends[d, blk] = count

    step([0], [45])
    fork([1, 2], [0, 0], [45, 33])
    step([2, 0, 1], [1, 1, 1], [3, 4, 5])
    fork([3, 0], [1, 2])               # 0 becomes a branch of 2
    step([0, 1, 2, 3], [3, 1, 4, 20])
    for i in (1, 3):                   # what the middle said is forgotten
        n = s.cache.length(i)
        s.cache.compact([i], [np.r_[:8, 20:n]])
        for blk in range(4):
            s.appends[i, blk] = s.appends.get((i, blk), 0) + 1
    step([3, 1, 0], [1, 1, 1], [0, 299, 7])
    s.free()
