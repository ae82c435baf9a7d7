"""Branches of sequences in the paged 8-bit KV cache and compaction, on the GPU
against tests/kv_branch_ref.py."""
import ctypes

import numpy as np
import pytest

import purebee_amd as pb
from tests.kv_branch_ref import BranchPair
from tests.kv_ref import Rows
from tests.test_gpu_kv import HEADS

pytestmark = pytest.mark.gpu


def free_pages(p):
    return p.cache.info()["free_pages"]


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("layers", [1, 3])
def test_branches_grow_apart(ctx, heads, kv_heads, dim, layers):
    """Branches at a page's end, inside a block and inside a page go on with rows of their own."""
    print(f"[case] fork {heads}/{kv_heads}/{dim} layers {layers}", flush=True)
    p = BranchPair(ctx, heads, kv_heads, dim, seqs=5, layers=layers, page=64, seed=dim)
    layer = layers - 1
    p.append([0], [150], layer=layer)
    used = free_pages(p)
    p.fork([1, 2, 3], [0, 0, 0], [150, 128, 37])
    assert free_pages(p) == used
    p.check_values(layer=layer)
    p.append([1, 2, 3], [1, 1, 40], p.rows(42, 3.0), layer=layer)
    p.check_values(layer=layer, pad=4)
    p.fork([4, 1], [1, 4])  # 4 was empty: they change places
    p.append([4, 0], [5, 70], layer=layer)
    p.check_values(layer=layer)
    b, q = p.append([0, 2, 3, 4], [1, 2, 1, 3], layer=layer)
    starts = [p.ref.length(s) - n for s, n in zip([0, 2, 3, 4], [1, 2, 1, 3])]
    p.attend(b, [0, 2, 3, 4], starts, [1, 2, 1, 3], q, layer=layer)
    for s in range(5):
        p.truncate(s, 0)
    assert free_pages(p) == 64
    p.free()


@pytest.mark.parametrize("lengths", [[1], [31], [32], [33], [64], [65], [100]])
@pytest.mark.parametrize("rows", [1, 33])
def test_branches_at_lengths(ctx, lengths, rows):
    """Every branch, and then the source, gets rows; the last one to hold a page keeps it."""
    n = lengths[0]
    p = BranchPair(ctx, 4, 2, 64, seqs=4, page=64, n_pages=40, seed=n)
    p.append([0], [n])
    p.fork([1, 2, 3], [0] * 3)
    p.append([3], [rows], p.rows(rows, 0.1))  # raises no scale
    p.check_values()
    p.append([1, 2, 0], [rows] * 3, p.rows(3 * rows, 5.0))  # raises them: earlier codes are rounded again
    p.check_values()
    p.free()


def test_beams(ctx):
    """Eight steps of four beams that take each other's places."""
    p = BranchPair(ctx, 9, 3, 64, seqs=4, page=32, n_pages=40, seed=3)
    p.append([0], [61])
    p.fork([1, 2, 3], [0] * 3)
    rng = np.random.default_rng(5)
    for _ in range(8):
        b, q = p.append(range(4), [1] * 4)
        p.attend(b, range(4), [p.ref.length(s) - 1 for s in range(4)], [1] * 4, q)
        b.free()
        p.fork(range(4), rng.integers(0, 4, 4))
    p.check_values()
    p.free()


def test_fork_that_shortens(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=2, page=32, n_pages=8, seed=4)
    p.append([0], [100])
    b = p.cache.batch([0], [60], [0])
    p.fork([0], [0], [70])  # drops nothing that the batch reads
    got = Rows(ctx, 60, 128)
    b.read_dev(0, got.ptr, None)
    p.fork([0], [0], [59])
    with pytest.raises(pb.PbxError, match="dropped or moved"):
        b.read_dev(0, got.ptr, None)
    p.fork([1, 0], [0, 1])
    assert p.cache.length(0) == 0 and p.cache.length(1) == 59
    p.check_values()
    p.fork([], [])
    got.free()
    p.free()


def test_refused_forks_change_nothing(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=3, page=32, n_pages=8, seed=4)
    p.append([0], [40])
    for args in (([1], [3]), ([3], [0]), ([-1], [0]), ([1], [-1]), ([1, 1], [0, 0]), ([1], [0], [41]), ([1], [0], [-1])):
        with pytest.raises(pb.PbxError, match="EINVAL"):
            p.cache.fork(*args)
    with pytest.raises(ValueError):
        p.cache.fork([1], [0, 0])
    with pytest.raises(ValueError):
        p.cache.fork([1], [0], [1, 2])
    with pytest.raises(OverflowError):
        p.cache.fork([2**32], [0])
    assert ctx.L.pbx_kv_fork(p.cache._ptr, 1, None, None, None) == -1
    assert ctx.L.pbx_kv_fork(p.cache._ptr, -1, None, None, None) == -1
    assert free_pages(p) == 6 and p.cache.length(1) == 0
    p.check_values()
    p.free()


def test_a_pool_without_a_page_for_the_copy(ctx):
    """The batch is refused and the branch stays shared; with a page it goes on."""
    p = BranchPair(ctx, 4, 2, 64, seqs=3, page=64, n_pages=3, seed=4)
    p.append([0], [90])
    p.append([2], [1])
    p.fork([1], [0])
    with pytest.raises(pb.PbxError, match="ENOMEM"):
        p.cache.batch([1], [1])
    assert p.cache.length(1) == 90
    p.check_values()
    p.truncate(2, 0)
    p.append([1], [1])
    p.append([0], [2])  # holds its page alone by now
    assert free_pages(p) == 0
    p.check_values()
    p.free()


def test_batches_that_know_pages_left_behind(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=3, page=64, n_pages=20, seed=4)
    p.append([0], [90])
    p.fork([1], [0])
    reads = p.cache.batch([1], [90], [0])
    early = p.cache.batch([1], [60], [0])  # only the page that stays
    p.append([1], [3])
    got = Rows(ctx, 90, 128)
    with pytest.raises(pb.PbxError, match="dropped or moved"):
        reads.read_dev(0, got.ptr, None)
    early.read_dev(0, got.ptr, None)
    reads.set([1], [90], [0]).read_dev(0, got.ptr, None)
    ctx.sync()
    p.check_values()
    got.free()
    p.free()


def test_rows_in_shared_pages_are_not_written(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=3, page=64, n_pages=20, seed=4)
    p.append([0], [90])
    q, k, v = p.rows(2)
    dk, dv = Rows(ctx, 2, 128, k), Rows(ctx, 2, 128, v)
    grown = p.cache.batch([0], [2])
    p.cache.fork([1], [0], [90])  # takes the page with the rows that the batch has not appended yet
    with pytest.raises(pb.PbxError, match="shares pages"):
        grown.append_dev(0, None, dk.ptr, dv.ptr, None)
    p.cache.truncate(0, 90)
    p.ref.fork([1], [0])
    p.append([0], [2], (q, k, v))
    p.check_values()
    # rows that were there: the batch may read and attend, not append
    again = p.cache.batch([1], [30], [60])
    dkk = Rows(ctx, 30, 128)
    again.read_dev(0, dkk.ptr, None)
    p.fork([2], [1])
    with pytest.raises(pb.PbxError, match="truncate it to 60"):
        again.append_dev(0, None, dkk.ptr, dkk.ptr, None)
    p.truncate(1, 60)
    p.append([1], [30])
    p.check_values()
    for x in (dk, dv, dkk):
        x.free()
    p.free()


def hip():
    h = ctypes.CDLL("libamdhip64.so")
    h.hipStreamBeginCapture.argtypes = [ctypes.c_void_p, ctypes.c_int]
    h.hipStreamEndCapture.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]
    h.hipGraphInstantiate.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p, ctypes.c_void_p,
                                      ctypes.c_void_p, ctypes.c_size_t]
    h.hipGraphLaunch.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    h.hipGraphDestroy.argtypes = [ctypes.c_void_p]
    h.hipGraphExecDestroy.argtypes = [ctypes.c_void_p]
    return h


class Graph:
    """What `calls` enqueues on the context's stream, to be launched again and again."""

    def __init__(self, ctx, calls):
        self.h, self.stream = hip(), ctx.stream()
        graph, self.run = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.h.hipStreamBeginCapture(self.stream, 2) == 0  # relaxed
        try:
            calls()
        finally:
            rc = self.h.hipStreamEndCapture(self.stream, ctypes.byref(graph))
        assert rc == 0
        assert self.h.hipGraphInstantiate(ctypes.byref(self.run), graph, None, None, 0) == 0
        assert self.h.hipGraphDestroy(graph) == 0

    def launch(self):
        assert self.h.hipGraphLaunch(self.run, self.stream) == 0

    def free(self):
        assert self.h.hipGraphExecDestroy(self.run) == 0


def test_captured_batches(ctx):
    """Pages that a graph appends to are not shared; pages that a graph reads are not left."""
    p = BranchPair(ctx, 4, 2, 64, seqs=4, page=64, n_pages=20, seed=6)
    p.append([0, 3], [90, 70])
    q, k, v = p.rows(1)
    dk, dv = Rows(ctx, 1, 128, k), Rows(ctx, 1, 128, v)
    b = p.cache.batch([0], [1])

    def append():
        b.append_dev(0, None, dk.ptr, dv.ptr, None)
        for call in (lambda: p.cache.fork([1], [3]), lambda: p.cache.compact([3], [[0]])):
            with pytest.raises(pb.PbxError, match="captured"):
                call()

    g = Graph(ctx, append)
    g.launch()
    p.ref.append([0], [1], q, k, v)
    with pytest.raises(pb.PbxError, match="captured graph appends"):
        p.cache.fork([1], [0])
    p.fork([1], [0], [64])  # the page before it
    p.append([1], [4])
    p.check_values()
    for _ in range(3):  # the same rows at the same positions again
        g.launch()
        p.check_values()
    # a graph that reads a branch's shared pages: the branch cannot move out of them
    p.fork([2], [3])
    got = Rows(ctx, 70, 128)
    reads = p.cache.batch([2], [70], [0])
    g2 = Graph(ctx, lambda: reads.read_dev(0, got.ptr, None))
    with pytest.raises(pb.PbxError, match="captured graph runs"):
        p.cache.batch([2], [1])
    assert p.cache.length(2) == 70
    p.append([3], [5])  # the other one can
    want = p.ref.values([2], [0], [70])[0].reshape(70, 128)
    for _ in range(3):
        g2.launch()
        ctx.sync()
        assert np.array_equal(got.get(), want)
        p.check_values([0, 1, 3])
    g.free()
    g2.free()
    b.free()
    reads.free()
    p.append([2], [1])
    p.check_values()
    for x in (dk, dv, got):
        x.free()
    p.free()


# ---- compaction ------------------------------------------------------------------

def kept_of(kind, n, rng):
    if kind == "window":
        return np.r_[:min(4, n), max(4, n - n // 3):n]
    if kind == "cut":
        a = n // 4
        return np.r_[:a, min(n, a + 50):n]
    if kind == "scattered":
        return np.flatnonzero(rng.random(n) < 0.4)
    if kind == "first":
        return np.arange(n // 2)
    if kind == "all":
        return np.arange(n)
    return np.array([n - 1])  # "one"


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("style,part", [("pairs", 1), ("halves", 2), ("none", 1)])
def test_compact(ctx, heads, kv_heads, dim, style, part):
    print(f"[case] compact {heads}/{kv_heads}/{dim} {style} 1/{part}", flush=True)
    p = BranchPair(ctx, heads, kv_heads, dim, seqs=3, n_pages=40, layers=2, style=style,
                   rope_dim=dim // part // 4 * 4, theta=500000.0, scale=2.0 if part == 2 else 1.0,
                   factors=np.linspace(1, 8, dim // part // 4 * 2) if part == 2 else None,
                   page=64 if dim % 64 else 32, seed=dim)
    p.append([0, 1, 2], [200, 65, 333], layer=1)
    p.append([0, 1, 2][:1], [13], p.rows(13, 4.0), layer=1)
    p.compact([2, 0], [kept_of("cut", 333, p.rng), kept_of("scattered", 213, p.rng)])
    p.check_values(layer=1, pad=4)
    b, q = p.append([0, 1, 2], [1, 3, 40], layer=1)
    starts = [p.ref.length(s) - n for s, n in zip([0, 1, 2], [1, 3, 40])]
    p.attend(b, [0, 1, 2], starts, [1, 3, 40], q, layer=1)
    p.compact([0, 1, 2], [kept_of("window", p.ref.length(s), p.rng) for s in range(3)])
    p.check_values(layer=1)
    got = Rows(ctx, 1, kv_heads * dim)
    b = p.cache.batch([0], [1], [0])
    b.read_dev(0, got.ptr, None)
    ctx.sync()
    assert not got.get().any()  # layer 0 was never written
    got.free()
    p.free()


@pytest.mark.parametrize("kind", ["window", "cut", "scattered", "first", "all", "one"])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 129, 1000])
def test_compact_lengths(ctx, kind, n):
    p = BranchPair(ctx, 4, 2, 64, seqs=2, n_pages=80, page=64, seed=n)
    p.append([0, 1], [n, 5])
    kept = kept_of(kind, n, p.rng)
    p.compact([0], [kept])
    assert p.cache.length(0) == len(kept) and free_pages(p) == 80 - 1 - -(-len(kept) // 64)
    p.check_values()
    p.append([0], [2])
    p.check_values()
    p.free()


def test_compact_to_nothing_and_nobody(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=3, n_pages=8, page=32, seed=1)
    p.append([0, 1], [40, 3])
    p.compact([], [])
    p.compact([0, 2], [[], []])
    assert p.cache.length(0) == 0 and free_pages(p) == 7
    p.append([0], [33])
    p.check_values()
    p.free()


def test_compact_leaves_branches_alone(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=3, n_pages=40, page=32, seed=2)
    p.append([0], [300])
    p.fork([1, 2], [0, 0])
    p.compact([1], [kept_of("window", 300, p.rng)])
    p.compact([2], [np.r_[:100, 200:300]])
    assert free_pages(p) == 40 - 10 - 4 - 4  # of sequence 2 the first three pages are still shared
    p.check_values()
    p.append([0, 1, 2], [3, 3, 3])
    p.check_values()
    p.free()


@pytest.mark.parametrize("spare", [1, 2, 5])
def test_compact_with_few_free_pages(ctx, spare):
    """The pool is all but full: pages go round, in several launches."""
    p = BranchPair(ctx, 4, 2, 64, seqs=3, n_pages=32 + spare, page=32, layers=2, seed=spare)
    p.append([0, 1], [700, 310], layer=1)
    assert free_pages(p) == spare
    p.compact([0, 1], [np.r_[1:700], np.r_[5:50, 60:310]])
    p.check_values(layer=1)
    p.compact([1, 0], [np.r_[0:200], kept_of("scattered", 699, p.rng)])
    p.check_values(layer=1)
    p.free()


def test_compact_in_a_full_pool_is_refused(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=2, n_pages=4, page=32, seed=2)
    p.append([0], [128])
    with pytest.raises(pb.PbxError, match="ENOMEM"):
        p.cache.compact([0], [np.r_[1:128]])
    p.check_values()
    p.compact([0], [np.r_[:96]])  # only drops: takes none
    p.compact([0], [np.r_[1:96]])
    p.check_values()
    p.free()


def test_refused_compactions_change_nothing(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=3, page=32, n_pages=8, seed=4)
    p.append([0, 1], [40, 40])
    for seqs, kept in (([3], [[0]]), ([-1], [[0]]), ([0, 0], [[0], [1]]), ([0], [[40]]), ([0], [[-1]]), ([0], [[1, 1]]),
                       ([0], [[2, 1]]), ([0], [list(range(41))]), ([1, 0], [[3], [0, 40]]), ([2], [[0]])):
        with pytest.raises(pb.PbxError, match="EINVAL"):
            p.cache.compact(seqs, kept)
    with pytest.raises(ValueError):
        p.cache.compact([0], [])
    with pytest.raises(OverflowError):
        p.cache.compact([0], [[2**31]])
    one = (ctypes.c_int32 * 1)(1)
    zero = (ctypes.c_int32 * 1)(0)
    assert ctx.L.pbx_kv_compact(p.cache._ptr, 1, zero, one, None) == -1
    assert ctx.L.pbx_kv_compact(p.cache._ptr, -1, None, None, None) == -1
    assert free_pages(p) == 4
    p.check_values()
    p.free()


def test_compact_makes_batches_stale(ctx):
    p = BranchPair(ctx, 4, 2, 64, seqs=3, page=32, n_pages=12, seed=4)
    p.append([0], [100])
    first, all_ = p.cache.batch([0], [32], [0]), p.cache.batch([0], [100], [0])
    p.compact([0], [np.r_[:40, 50:100]])
    got = Rows(ctx, 100, 128)
    first.read_dev(0, got.ptr, None)
    with pytest.raises(pb.PbxError, match="dropped or moved"):
        all_.read_dev(0, got.ptr, None)
    ctx.sync()
    got.free()
    p.free()


def test_compact_of_extreme_blocks(ctx):
    """NaN and infinite rows, zeros, subnormal and huge values."""
    p = BranchPair(ctx, 4, 2, 64, seqs=1, n_pages=40, page=32, seed=8)
    q, k, v = p.rows(32 * 7)
    k[:32] = 0
    v[32:64] *= 1e-39
    k[64:96] *= 2.5e38 / np.abs(k[64:96]).max()
    v[64:96] *= 2.5e38 / np.abs(v[64:96]).max()
    v[100, 1, 3] = np.nan
    k[130, 0, 5] = np.inf
    k[160:192] *= 1e-30
    p.append([0], [32 * 7], (q, k, v))
    p.compact([0], [np.r_[3:90, 97, 98, 120:224]])
    p.check_values()
    p.compact([0], [np.r_[1:p.ref.length(0)]])
    p.check_values()
    p.free()


def test_long_moves(ctx):
    """Angles of a distance of 100,000 positions, and many turns one after the other."""
    p = BranchPair(ctx, 4, 1, 128, seqs=1, n_pages=110, page=1024, max_seq=1 << 17, style="halves", theta=1e6, seed=9)
    # (angles are products in 64 bits, so at 100,000 they are off by up to 100,000 * 2^-52 = 2e-11 here and there:
    # one value in 4e8 may be coded otherwise, and 104 rows of 128 are looked at; queries are checked in the tests above)
    p.fill(0, 100000)
    p.compact([0], [np.r_[:4, 99900:100000]])
    p.check_values()
    for _ in range(5):
        p.append([0], [1])
        p.compact([0], [np.r_[:4, 5:p.ref.length(0)]])
    p.check_values()
    p.free()


def test_more_blocks_than_a_launch_takes(ctx):
    """A launch takes 2^22 blocks over all layers and heads: here 10 sequences of 210 blocks of 4,096 layers, compacted
    and branched; the last layer's values are looked at, and the first one's, which nobody wrote."""
    layers, n = 4096, 6700
    p = BranchPair(ctx, 1, 1, 32, seqs=20, n_pages=20 * 7 + 80, page=1024, max_seq=8192, layers=layers, seed=4)
    for s in range(10):
        q, k, v = p.rows(n)
        b = p.cache.batch([s], [n])
        dk, dv = Rows(ctx, n, 32, k), Rows(ctx, n, 32, v)
        b.append_dev(layers - 1, None, dk.ptr, dv.ptr, None)
        ctx.sync()
        p.ref.append([s], [n], q, k, v)
        for x in (dk, dv, b):
            x.free()
    p.compact(list(range(10)), [np.r_[1:n]] * 10)
    p.check_values(range(10), layer=layers - 1)
    p.fork(list(range(10, 20)), list(range(10)))
    p.append(list(range(10, 20)), [1] * 10, layer=layers - 1)
    p.check_values(layer=layers - 1)
    got = Rows(ctx, 1, 32)
    b = p.cache.batch([3], [1], [5000])
    b.read_dev(0, got.ptr, None)
    ctx.sync()
    assert not got.get().any()
    got.free()
    b.free()
    p.free()
