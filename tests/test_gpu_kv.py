"""The paged 8-bit KV cache on the GPU against tests/kv_ref.py: append with the
position rotation, attention over the cache, reading back, and refusals."""
import ctypes

import numpy as np
import pytest

import purebee_amd as pb
from tests.kv_ref import BLOCK, RefCache, Rows, rotate, within

pytestmark = pytest.mark.gpu


class Pair:
    """A cache on the GPU and the reference beside it."""

    def __init__(self, ctx, heads, kv_heads, dim, seqs=4, n_pages=64, page=32, max_seq=4096, layers=1, style="pairs",
                 rope_dim=0, theta=10000.0, scale=1.0, factors=None, seed=0):
        self.ctx, self.heads, self.kv_heads, self.dim = ctx, heads, kv_heads, dim
        self.rng = np.random.default_rng(seed)
        self.cache = pb.KvCache(ctx, layers, heads, kv_heads, dim, n_pages, seqs, max_seq, page_tokens=page,
                                rope=style, rope_dim=rope_dim, rope_theta=theta, rope_scale=scale,
                                rope_factors=factors)
        self.ref = RefCache(seqs, heads, kv_heads, dim, style, rope_dim, theta, scale, factors)

    def rows(self, n, size=1.0):
        r = self.rng
        return (size * r.standard_normal((n, self.heads, self.dim)).astype(np.float32),
                size * r.standard_normal((n, self.kv_heads, self.dim)).astype(np.float32),
                size * r.standard_normal((n, self.kv_heads, self.dim)).astype(np.float32))

    def append(self, seqs, counts, data=None, layer=0, pad=0):
        """Appends and checks the rotated queries; returns the batch and them."""
        n = sum(counts)
        q, k, v = data or self.rows(n)
        b = self.cache.batch(seqs, counts)
        assert b.rows == n
        qw, kw = self.heads * self.dim, self.kv_heads * self.dim
        dq, do = Rows(self.ctx, n, qw, q, qw + pad), Rows(self.ctx, n, qw, None, qw + 2 * pad)
        dk, dv = Rows(self.ctx, n, kw, k, kw + 3 * pad), Rows(self.ctx, n, kw, v, kw + pad)
        b.append_dev(layer, dq.ptr, dk.ptr, dv.ptr, do.ptr, dq.stride, dk.stride, dv.stride, do.stride)
        self.ctx.sync()
        got = do.get().reshape(q.shape)
        want = self.ref.append(seqs, counts, q, k, v)
        # one rounding to f32 of 64-bit sums
        within(got, want, 2.0 ** -24 * np.abs(want) + 1e-14 * np.abs(q).max())
        for x in (dq, dk, dv):
            x.get()
        for x in (dq, dk, dv, do):
            x.free()
        return b, got

    def check_values(self, seqs=None, layer=0, pad=0):
        """Every position of the sequences, read back, equals the reference's."""
        seqs = range(len(self.ref.k)) if seqs is None else seqs
        counts = [self.ref.length(s) for s in seqs]
        for s, n in zip(seqs, counts):
            assert self.cache.length(s) == n
        b = self.cache.batch(seqs, counts, [0] * len(counts))
        n, w = sum(counts), self.kv_heads * self.dim
        dk, dv = Rows(self.ctx, n, w, None, w + pad), Rows(self.ctx, n, w, None, w + 2 * pad)
        b.read_dev(layer, dk.ptr, dv.ptr, dk.stride, dv.stride)
        self.ctx.sync()
        want = self.ref.values(seqs, [0] * len(counts), counts)
        for got, ref in zip((dk.get(), dv.get()), want):
            assert bool(np.array_equal(got.reshape(ref.shape), ref, equal_nan=True))
        for x in (dk, dv, b):
            x.free()

    def attend(self, batch, seqs, starts, counts, q, layer=0, pad=0, scale=None):
        """Attention of rows q of the batch, checked against the reference."""
        n, w = sum(counts), self.heads * self.dim
        dq, do = Rows(self.ctx, n, w, q, w + pad), Rows(self.ctx, n, w, None, w + 2 * pad)
        batch.attention_dev(layer, dq.ptr, do.ptr, scale or 0.0, dq.stride, do.stride)
        self.ctx.sync()
        got = do.get().reshape(n, self.heads, self.dim)
        want, tol = self.ref.attention(seqs, starts, counts, q, scale)
        assert bool((np.isnan(got) == np.isnan(want)).all()) and not np.isinf(got).any()
        within(got, want, tol)
        for x in (dq, do):
            x.free()
        return got

    def free(self):
        self.cache.free()


HEADS = [(32, 8, 64), (9, 3, 64), (6, 6, 48), (4, 1, 32), (2, 1, 36), (20, 1, 64), (3, 3, 80), (4, 2, 96),
         (8, 2, 100), (16, 4, 128), (2, 1, 160), (2, 2, 192), (8, 1, 256)]


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("style,part", [("pairs", 1), ("halves", 1), ("pairs", 2), ("halves", 2), ("none", 1)])
def test_append_in_steps(ctx, heads, kv_heads, dim, style, part):
    """Blocks filled by one row, by a few, across borders, in whole; other layers and sequences are left alone."""
    print(f"[case] append {heads}/{kv_heads}/{dim} {style} 1/{part}", flush=True)
    p = Pair(ctx, heads, kv_heads, dim, seqs=3, layers=2, style=style, rope_dim=dim // part // 4 * 4, theta=500000.0,
             scale=2.0 if part == 2 else 1.0, factors=np.linspace(1, 8, dim // part // 4 * 2) if part == 2 else None,
             page=64 if dim % 64 else 32, seed=dim)
    for seqs, counts in (([0], [1]), ([0, 2], [30, 31]), ([2, 0], [1, 1]), ([1, 0, 2], [33, 1, 70]), ([0], [64])):
        p.append(seqs, counts, layer=1, pad=4 * len(seqs))
    p.check_values(layer=1, pad=4)
    got = Rows(ctx, 1, kv_heads * dim)
    b = p.cache.batch([0], [1], [0])
    b.read_dev(0, got.ptr, None)
    ctx.sync()
    assert not got.get().any()  # layer 0 was never written
    got.free()
    p.free()


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_attention_of_chunks_and_tokens(ctx, heads, kv_heads, dim):
    """A prompt, single tokens, a few rows and a long chunk, packed, at ragged lengths."""
    print(f"[case] attention {heads}/{kv_heads}/{dim}", flush=True)
    p = Pair(ctx, heads, kv_heads, dim, seqs=4, seed=heads + dim)
    for seqs, counts in (([0, 1], [31, 1]), ([0, 1, 3], [1, 1, 5]), ([2, 0, 1], [40, 3, 2]), ([3, 1], [17, 90])):
        starts = [p.ref.length(s) for s in seqs]
        b, q = p.append(seqs, counts)
        p.attend(b, seqs, starts, counts, q, pad=8)
    p.free()


@pytest.mark.parametrize("lengths", [[1], [2], [31], [32], [33], [255], [256], [257], [1000], [3000, 5, 700, 64]])
def test_attention_of_tokens_at_lengths(ctx, lengths):
    """One row a sequence over contexts that are not split, just split and split many ways."""
    print(f"[case] token attention at {lengths}", flush=True)
    p = Pair(ctx, 8, 2, 64, n_pages=130, page=32, seed=len(lengths) + lengths[0])
    seqs = list(range(len(lengths)))
    if max(lengths) > 1:
        p.append([s for s in seqs if lengths[s] > 1], [n - 1 for n in lengths if n > 1])
    b, q = p.append(seqs, [1] * len(seqs))
    p.attend(b, seqs, [n - 1 for n in lengths], [1] * len(seqs), 3 * q)
    p.attend(b, seqs, [n - 1 for n in lengths], [1] * len(seqs), q, scale=0.7)
    p.attend(b, seqs, [n - 1 for n in lengths], [1] * len(seqs), q, scale=-0.2)
    p.free()


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 8, 16, 17, 33, 64, 129])
@pytest.mark.parametrize("past", [0, 1, 30, 100, 511])
def test_attention_rows_by_past(ctx, rows, past):
    """Row counts around the kernels' tiles, on pasts around block borders."""
    print(f"[case] {rows} rows after {past}", flush=True)
    p = Pair(ctx, 8, 2, 64, page=128, n_pages=16, seed=rows * 1000 + past)
    if past:
        p.append([1], [past])
    b, q = p.append([1], [rows])
    p.attend(b, [1], [past], [rows], q)
    p.free()


def test_attention_of_earlier_rows(ctx):
    """A batch over positions in the middle of its sequences sees what lay before them, not what came after; append refuses it."""
    p = Pair(ctx, 4, 2, 64, seed=3)
    p.append([0, 1], [150, 90])
    seqs, starts, counts = [1, 0], [20, 64], [30, 7]
    b = p.cache.batch(seqs, counts, starts)
    q = p.rows(37)[0]
    p.attend(b, seqs, starts, counts, q)
    k = Rows(ctx, 37, 128)
    with pytest.raises(pb.PbxError, match="not the last"):
        b.append_dev(0, None, k.ptr, k.ptr, None)
    k.free()
    p.free()


def test_scales_grow_and_do_not_fall(ctx):
    """Rows of rising and falling size in one block: codes are rounded again when the scale grows, and stay otherwise."""
    p = Pair(ctx, 2, 2, 64, seed=5)
    for size in (1.0, 0.5, 3.0, 3.0, 1e-3, 40.0, 41.0, 1e20, 1.0):
        p.append([0], [3], p.rows(3, size))
        p.check_values([0])
    p.free()


def test_zero_and_tiny_and_huge_rows(ctx):
    """Blocks of zeros, of values below the least scale, and near f32's ends."""
    p = Pair(ctx, 2, 1, 32, style="none", seed=6)
    for size in (0.0, 1e-40, 1e-37, 1e-30, 1e38):
        b, q = p.append([0], [32], p.rows(32, size / 4))
    p.check_values([0])
    p.free()


@pytest.mark.parametrize("size,scale", [(0.0, 1.0), (1e-30, 1e29), (1e-42, 1e38), (1e10, 1e-11), (1e37, 1e-38)])
def test_queries_of_any_size(ctx, size, scale):
    """Queries near f32's ends, the scale bringing the scores to ordinary size."""
    p = Pair(ctx, 2, 1, 32, style="none", seed=18)
    p.append([0], [70])
    p.attend(p.cache.batch([0], [2], [68]), [0], [68], [2], p.rows(2, size)[0], scale=np.float32(scale))
    p.free()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_bad_value_stays_in_its_block(ctx, bad):
    """A NaN or infinity makes its block (of its head, keys or values) read as NaN, the rows that see it NaN, and nothing else."""
    p = Pair(ctx, 2, 2, 64, style="none", seed=7)
    data = p.rows(100)
    data[1][40, 0, 3] = bad   # a key of block 1, head 0
    data[2][70, 1, 9] = bad   # a value of block 2, head 1
    b, q = p.append([0], [100], data)
    p.check_values([0])
    got = p.attend(b, [0], [0], [100], q)
    # head 0: rows before block 1 see nothing of it
    assert np.isfinite(got[:32, 0]).all() and np.isnan(got[40:, 0]).all()
    assert np.isfinite(got[:64, 1]).all() and np.isnan(got[70:, 1]).all()
    p.free()


@pytest.mark.parametrize("rows", [6, 12, 60])
def test_a_bad_block_does_not_reach_rows_before_it(ctx, rows):
    """Rows that share a tile with rows that see a NaN block, and do not see it themselves, stay as they are."""
    p = Pair(ctx, 4, 2, 64, style="none", seed=19)
    p.append([0], [28])
    data = p.rows(rows)
    data[1][4:, 0], data[2][5:, 1] = np.nan, np.inf  # block 1: keys of head 0, values of head 1
    b, q = p.append([0], [rows], data)
    got = p.attend(b, [0], [28], [rows], q)
    assert np.isfinite(got[:4]).all() and np.isnan(got[5:]).all()
    p.free()


def test_a_bad_query_is_its_own_row(ctx):
    p = Pair(ctx, 4, 2, 64, style="none", seed=8)
    b, q = p.append([0], [40])
    q = q.copy()
    q[3, 1, 5], q[7, 2, 0] = np.nan, np.inf
    got = p.attend(b, [0], [0], [40], q)
    assert np.isnan(got[3, 1]).all() and np.isnan(got[7, 2]).all() and np.isnan(got).sum() == 2 * 64
    p.free()


def test_masked_positions_do_not_matter(ctx):
    """What a page held before, and rows of the same block that lie behind a query, leave no trace."""
    p = Pair(ctx, 4, 2, 64, seqs=2, n_pages=4, style="none", seed=9)
    data = p.rows(128)
    for x in data[1:]:
        x[:] = np.nan
    p.append([0], [128], data)          # all four pages hold NaN
    p.cache.truncate(0)
    p.ref.truncate(0, 0)
    b, q = p.append([1], [50])
    got = p.attend(b, [1], [0], [50], q)
    assert np.isfinite(got).all()
    p.check_values([1])
    # a row in the same block, behind: NaN there makes the block NaN, so cut back first
    p.cache.truncate(1, 33)
    p.ref.truncate(1, 33)
    b, q = p.append([1], [1])
    assert np.isfinite(p.attend(b, [1], [33], [1], q)).all()
    p.free()


def test_truncate_and_append_again(ctx):
    """A speculative round: rows rejected, others appended in their place, with pages given back and taken again."""
    p = Pair(ctx, 4, 2, 64, seqs=2, n_pages=6, seed=10)
    p.append([0, 1], [60, 20])
    free = p.cache.info()["free_pages"]
    assert free == 6 - 2 - 1
    p.append([0], [5])
    assert p.cache.info()["free_pages"] == free - 1
    p.cache.truncate(0, 62)
    p.ref.truncate(0, 62)
    assert p.cache.info()["free_pages"] == free
    b, q = p.append([1, 0], [13, 4])
    p.attend(b, [1, 0], [20, 62], [13, 4], q)
    p.check_values()
    p.free()


def test_pages_of_sequences_that_grew_in_turn(ctx):
    """Page tables whose ids are mixed among sequences, pages longer than a block."""
    p = Pair(ctx, 4, 2, 64, seqs=3, n_pages=24, page=64, seed=11)
    for _ in range(7):
        for s in (2, 0, 1):
            p.append([s], [50])
    p.check_values()
    b, q = p.append([0, 1, 2], [1, 2, 3])
    p.attend(b, [0, 1, 2], [350] * 3, [1, 2, 3], q)
    p.free()


def test_empty_sequences_and_batches(ctx):
    """Sequences without rows in a batch, batches without rows or sequences."""
    p = Pair(ctx, 4, 2, 64, seed=12)
    p.append([0, 1, 2], [0, 40, 0])
    b, q = p.append([2, 3, 1, 0], [0, 7, 0, 1])
    p.attend(b, [2, 3, 1, 0], [0, 0, 40, 0], [0, 7, 0, 1], q)
    p.check_values()
    none = p.cache.batch([], [])
    zero = p.cache.batch([0, 1], [0, 0])
    for e in (none, zero):
        assert e.rows == 0
        e.append_dev(0, None, None, None, None)
        e.attention_dev(0, None, None)
        e.read_dev(0, None, None)
    ctx.sync()
    p.free()


def test_keys_and_values_alone_and_queries_in_place(ctx):
    """append without queries, and with the queries rotated where they lie, inside rows of q | k | v."""
    p = Pair(ctx, 4, 2, 64, seed=13)
    q, k, v = p.rows(37)
    w = (4 + 2 + 2) * 64
    rows = Rows(ctx, 37, w, np.concatenate([x.reshape(37, -1) for x in (q, k, v)], 1))
    b = p.cache.batch([0], [37])
    b.append_dev(0, rows.ptr, rows.ptr + 1024, rows.ptr + 1536, rows.ptr, w, w, w, w)
    ctx.sync()
    want = p.ref.append([0], [37], q, k, v)
    got = rows.get()
    assert np.abs(got[:, :256].reshape(want.shape) - want).max() <= 2.0 ** -24 * 8
    assert np.array_equal(got[:, 256:], np.concatenate([k.reshape(37, -1), v.reshape(37, -1)], 1))
    p.check_values([0])
    b2 = p.cache.batch([1], [37])
    b2.append_dev(0, None, rows.ptr + 1024, rows.ptr + 1536, None, 0, w, w, 0)
    p.ref.append([1], [37], q, k, v)
    p.check_values()
    rows.free()
    p.free()


def test_far_positions_and_long_pools(ctx):
    """Angles of far positions, and pages past 4 GiB of the pool."""
    # 1200 pages of 32 blocks x 8 heads x 16 KiB: 4.7 GiB of codes
    p = Pair(ctx, 8, 8, 256, seqs=3, n_pages=1200, page=1024, max_seq=1 << 20, theta=500000.0, seed=14)
    assert p.cache.info()["device_bytes"] > 4 << 30
    p.cache.batch([0], [1 << 20]).free()        # takes 1024 pages, written never
    p.cache.batch([2], [160 * 1024]).free()     # the next 160
    b, q = p.append([1], [40])                  # page 1184 and on: past 4 GiB
    p.attend(b, [1], [0], [40], q)
    p.check_values([1])
    # the last rows of sequence 0: positions next to 2^20
    p.cache.truncate(0, (1 << 20) - 2)
    q, k, v = p.rows(2)
    b = p.cache.batch([0], [2])
    dq, dk, dv = (Rows(ctx, 2, 2048, x) for x in (q, k, v))
    b.append_dev(0, dq.ptr, dk.ptr, dv.ptr, dq.ptr)
    ctx.sync()
    want = rotate(q, [(1 << 20) - 2, (1 << 20) - 1], "pairs", 256, 500000.0)
    # angles up to 2^20 in 64 bits are good to 2^-32
    assert np.abs(dq.get().reshape(want.shape) - want).max() <= (2.0 ** -24 + 2.0 ** -31) * 2 * np.abs(q).max()
    for x in (dq, dk, dv):
        x.free()
    p.free()


def _hip():
    hip = ctypes.CDLL("libamdhip64.so")
    vp = ctypes.c_void_p
    hip.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    hip.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, ctypes.c_char_p, ctypes.c_size_t]
    hip.hipGraphLaunch.argtypes = [vp, vp]
    hip.hipGraphExecDestroy.argtypes = [vp]
    hip.hipGraphDestroy.argtypes = [vp]
    return hip


def test_captured_calls_replay(ctx):
    """append, attention over a split context and read back captured into one graph: every replay equals the eager calls, with other eager
    work between; a captured batch keeps its rows."""
    hip = _hip()
    p = Pair(ctx, 8, 2, 64, n_pages=80, seed=15)
    p.append([0, 1], [1500, 40])
    q, k, v = p.rows(3)
    b = p.cache.batch([0, 1], [1, 2])
    dq, dk, dv = Rows(ctx, 3, 512, q), Rows(ctx, 3, 128, k), Rows(ctx, 3, 128, v)
    dr, do, rk, rv = Rows(ctx, 3, 512), Rows(ctx, 3, 512), Rows(ctx, 3, 128), Rows(ctx, 3, 128)

    def calls():
        b.append_dev(0, dq.ptr, dk.ptr, dv.ptr, dr.ptr)
        b.attention_dev(0, dr.ptr, do.ptr)
        b.read_dev(0, rk.ptr, rv.ptr)

    calls()
    ctx.sync()
    eager = [x.get() for x in (dr, do, rk, rv)]
    stream = ctypes.c_void_p(ctx.stream())
    graph, gexec = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    calls()
    with pytest.raises(pb.PbxError, match="captured"):
        b.set([0], [1])
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(gexec), graph, None, None, 0) == 0
    other = Pair(ctx, 8, 2, 64, seed=16)
    for rep in range(3):
        for x in (dr, do, rk, rv):
            x.buf.upload(x.host)
        assert hip.hipGraphLaunch(gexec, stream) == 0
        ctx.sync()
        for got, want in zip((dr, do, rk, rv), eager):
            assert np.array_equal(got.get(), want), rep
        ob, oq = other.append([0], [300])
        other.attend(ob, [0], [300 * rep], [300], oq)
    with pytest.raises(pb.PbxError, match="captured"):
        b.set([0], [1])
    hip.hipGraphExecDestroy(gexec)
    hip.hipGraphDestroy(graph)
    for x in (dq, dk, dv, dr, do, rk, rv):
        x.free()
    other.free()
    p.free()


def test_a_batch_is_set_again_and_again(ctx):
    """One batch for every step of a decode, without waiting between the steps."""
    p = Pair(ctx, 4, 2, 64, seqs=2, seed=17)
    b = p.cache.batch([0, 1], [40, 7])
    steps = [([0, 1], [40, 7])] + [([1, 0], [1, 1])] * 40
    bufs = []
    for i, (seqs, counts) in enumerate(steps):
        if i:
            b.set(seqs, counts)
        q, k, v = p.rows(sum(counts))
        n = len(q)
        d = [Rows(ctx, n, 256, q), Rows(ctx, n, 128, k), Rows(ctx, n, 128, v), Rows(ctx, n, 256)]
        starts = [p.ref.length(s) for s in seqs]
        b.append_dev(0, d[0].ptr, d[1].ptr, d[2].ptr, d[0].ptr)
        b.attention_dev(0, d[0].ptr, d[3].ptr)
        bufs.append((d, p.ref.attention(seqs, starts, counts, np.float32(p.ref.append(seqs, counts, q, k, v)))))
    ctx.sync()
    for d, (want, tol) in bufs:
        within(d[3].get().reshape(want.shape), want, tol)
        for x in d:
            x.free()
    p.check_values()
    p.free()


def test_refusals(ctx):
    def make(**kw):
        a = dict(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=64, n_pages=4, max_seqs=2, max_seq=100)
        a.update(kw)
        return pb.KvCache(ctx, **a)

    for kw in (dict(n_layers=0), dict(n_kv_heads=3), dict(head_dim=30), dict(head_dim=28), dict(head_dim=260),
               dict(page_tokens=16), dict(page_tokens=48), dict(page_tokens=2048), dict(n_pages=0), dict(max_seqs=0),
               dict(max_seq=0), dict(max_seq=(1 << 20) + 1), dict(rope_dim=6), dict(rope_dim=68), dict(rope_dim=-4),
               dict(rope_theta=0.0), dict(rope_theta=float("nan")), dict(rope_scale=0.0),
               dict(rope_factors=[1.0] * 31 + [0.0]), dict(n_pages=1 << 26, n_kv_heads=4)):
        with pytest.raises(pb.PbxError):
            make(**kw)
    with pytest.raises(ValueError):
        make(rope_factors=[1.0])
    c = make()
    unset = pb.KvBatch(c)
    with pytest.raises(pb.PbxError, match="not set"):
        unset.attention_dev(0, 16, 16)
    for seqs, counts, starts in (([2], [1], None), ([-1], [1], None), ([0, 0], [1, 1], None), ([0], [-1], None),
                                 ([0], [101], None), ([0], [1], [1]), ([0], [1], [-1])):
        with pytest.raises(pb.PbxError):
            unset.set(seqs, counts, starts)
    with pytest.raises(pb.PbxError) as e:   # 2 x 100 positions in 4 pages of 64
        c.batch([0, 1], [100, 100]) and make(n_pages=3).batch([0, 1], [100, 100])
    assert e.value.code == -3
    b = c.batch([0], [0])
    assert c.length(0) == 100
    with pytest.raises(pb.PbxError):
        c.truncate(0, 101)
    with pytest.raises(pb.PbxError):
        c.truncate(2, 0)
    with pytest.raises(pb.PbxError):
        c.length(2)
    b.set([0], [10], [90])
    x = Rows(ctx, 10, 256)
    for call in (lambda: b.append_dev(1, x.ptr, x.ptr, x.ptr, x.ptr), lambda: b.append_dev(-1, x.ptr, x.ptr, x.ptr, x.ptr),
                 lambda: b.append_dev(0, x.ptr, None, x.ptr, x.ptr), lambda: b.append_dev(0, x.ptr, x.ptr, x.ptr, None),
                 lambda: b.append_dev(0, None, x.ptr, x.ptr, x.ptr), lambda: b.append_dev(0, x.ptr + 4, x.ptr, x.ptr, x.ptr),
                 lambda: b.append_dev(0, x.ptr, x.ptr, x.ptr, x.ptr, q_stride=260),
                 lambda: b.append_dev(0, x.ptr, x.ptr, x.ptr, x.ptr, k_stride=124),
                 lambda: b.append_dev(0, x.ptr, x.ptr, x.ptr, x.ptr, v_stride=130),
                 lambda: b.attention_dev(0, None, x.ptr), lambda: b.attention_dev(0, x.ptr, None),
                 lambda: b.attention_dev(0, x.ptr, x.ptr, q_stride=252), lambda: b.attention_dev(0, x.ptr, x.ptr, float("nan")),
                 lambda: b.read_dev(0, x.ptr + 8, None), lambda: b.read_dev(2, x.ptr, None)):
        with pytest.raises(pb.PbxError):
            call()
    c.truncate(0, 95)
    for call in (lambda: b.append_dev(0, None, x.ptr, x.ptr, None), lambda: b.attention_dev(0, x.ptr, x.ptr),
                 lambda: b.read_dev(0, x.ptr, None)):
        with pytest.raises(pb.PbxError, match="dropped"):
            call()
    b.set([0], [5], [90])       # positions that are still there
    b.read_dev(0, x.ptr, None)
    more = c.batch([0], [1])    # the sequence grew: b's rows are not its last any more
    with pytest.raises(pb.PbxError, match="grew"):
        b.append_dev(0, None, x.ptr, x.ptr, None)
    ctx.sync()
    c.free()
    for h in (b, more):         # batches end with their cache
        with pytest.raises(pb.PbxError):
            h.read_dev(0, x.ptr, None)
    x.free()
    assert BLOCK == pb.native.KV_BLOCK


def test_a_pool_whose_size_overflows_is_refused(ctx):
    """2^25 layers x 2^26 pages x 2 heads x 16 KiB are 2^66 bytes: nothing, in 64 bits."""
    with pytest.raises(pb.PbxError) as e:
        pb.KvCache(ctx, 1 << 25, 2, 2, 256, 1 << 26, 1, 100, page_tokens=32)
    assert e.value.code == -3


def test_nothing_is_made_or_freed_inside_a_capture(ctx):
    """Both would wait for the stream and spoil the capture, which goes on."""
    hip = _hip()
    p = Pair(ctx, 4, 2, 64, seed=18)
    b, q = p.append([0], [50])
    dq, do = Rows(ctx, 50, 256, q), Rows(ctx, 50, 256)
    b.attention_dev(0, dq.ptr, do.ptr)
    ctx.sync()
    eager = do.get()
    stream, graph, gexec = ctypes.c_void_p(ctx.stream()), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    b.attention_dev(0, dq.ptr, do.ptr)
    for call in (b.free, p.cache.free, lambda: Pair(ctx, 4, 2, 64), lambda: p.cache.batch([0], [1])):
        with pytest.raises(pb.PbxError, match="captured"):
            call()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(gexec), graph, None, None, 0) == 0
    for _ in range(3):
        do.buf.upload(do.host)
        assert hip.hipGraphLaunch(gexec, stream) == 0
        ctx.sync()
        assert np.array_equal(do.get(), eager)
    hip.hipGraphExecDestroy(gexec)
    hip.hipGraphDestroy(graph)
    for x in (dq, do):
        x.free()
    p.free()
    assert p.cache._kv is None


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 32), (9, 3, 64), (8, 2, 96), (4, 2, 128), (4, 1, 192), (8, 1, 256)])
def test_rows_of_long_contexts(ctx, heads, kv_heads, dim):
    """Tiles of every width whose blocks are split over workgroups and joined, in place as well; the last tile is ragged."""
    print(f"[case] rows of long contexts {heads}/{kv_heads}/{dim}", flush=True)
    p = Pair(ctx, heads, kv_heads, dim, seqs=3, n_pages=150, seed=dim)
    p.append([0, 1, 2], [2600, 1, 700])
    b, q = p.append([0, 1, 2], [45, 2, 9])
    got = p.attend(b, [0, 1, 2], [2600, 1, 700], [45, 2, 9], q, pad=4)
    d = Rows(ctx, 56, heads * dim, q, heads * dim + 8)
    for _ in range(2):
        d.buf.upload(d.host)
        b.attention_dev(0, d.ptr, d.ptr, 0.0, d.stride, d.stride)
        ctx.sync()
        assert np.array_equal(d.get().reshape(got.shape), got)
    with pytest.raises(pb.PbxError, match="one stride"):
        b.attention_dev(0, d.ptr, d.ptr, 0.0, d.stride, d.stride + 4)
    d.free()
    p.free()


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (71, 1), (6, 6)])
def test_many_sequences(ctx, heads, kv_heads):
    """Hundreds of short sequences in a batch, one row or two each, and groups of many heads."""
    print(f"[case] 600 sequences {heads}/{kv_heads}", flush=True)
    n = 600
    p = Pair(ctx, heads, kv_heads, 32, seqs=n, n_pages=2 * n, seed=heads)
    lengths = [i % 37 for i in range(n)]
    seqs = [7 * i % n for i in range(n)]  # 7 and 600 have no common divisor
    p.append(seqs, [lengths[s] for s in seqs])
    counts = [1 + i % 2 for i in range(n)]
    b, q = p.append(seqs, counts)
    p.attend(b, seqs, [lengths[s] for s in seqs], counts, q)
    p.check_values()
    p.free()


def test_tokens_and_prompts_in_one_batch(ctx):
    """Single tokens over enough context for a launch of their own, beside prompts of wide tiles."""
    p = Pair(ctx, 32, 8, 32, seqs=42, n_pages=42 * 34, seed=19)
    past = [1050] * 40 + [0, 30]
    p.append(list(range(42)), past)
    seqs, counts = [41] + list(range(40)) + [40], [150] + [1] * 40 + [700]
    b, q = p.append(seqs, counts)
    p.attend(b, seqs, [past[s] for s in seqs], counts, q)
    p.free()


def test_the_same_rows_appended_again(ctx):
    """An append made twice (a replay, a retry) leaves what one leaves, in blocks that others began as well."""
    p = Pair(ctx, 4, 2, 64, seed=20)
    p.append([0, 1], [40, 31])
    q, k, v = p.rows(37, 3.0)
    b, got = p.append([1, 0], [30, 7], (q, k, v))
    dq, dk, dv = Rows(ctx, 37, 256, q), Rows(ctx, 37, 128, k), Rows(ctx, 37, 128, v)
    for _ in range(2):
        dq.buf.upload(dq.host)
        b.append_dev(0, dq.ptr, dk.ptr, dv.ptr, dq.ptr)
        ctx.sync()
        assert np.array_equal(dq.get().reshape(got.shape), got)
        p.check_values()
    for x in (dq, dk, dv):
        x.free()
    p.free()


def test_two_batches_in_two_graphs(ctx):
    """Split contexts of two batches, captured apart, replayed in turn and with eager calls between: nothing is shared."""
    hip = _hip()
    p = Pair(ctx, 8, 2, 64, seqs=3, n_pages=200, seed=21)
    p.append([0, 1, 2], [2000, 1500, 900])
    stream = ctypes.c_void_p(ctx.stream())
    made = []
    for seqs, counts in (([0], [1]), ([1, 2], [2, 20])):
        b, q = p.append(seqs, counts)
        n = sum(counts)
        dq, do = Rows(ctx, n, 512, q), Rows(ctx, n, 512)
        b.attention_dev(0, dq.ptr, do.ptr)
        ctx.sync()
        graph, gexec = ctypes.c_void_p(), ctypes.c_void_p()
        want = do.get()
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        b.attention_dev(0, dq.ptr, do.ptr)
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(gexec), graph, None, None, 0) == 0
        made.append((b, dq, do, want, graph, gexec))
    for rep in range(3):
        for b, dq, do, want, graph, gexec in made:
            do.buf.upload(do.host)
            assert hip.hipGraphLaunch(gexec, stream) == 0
        ctx.sync()
        for b, dq, do, want, graph, gexec in made:
            assert np.array_equal(do.get(), want), rep
        b, dq, do, want = made[rep % 2][:4]
        do.buf.upload(do.host)
        b.attention_dev(0, dq.ptr, do.ptr)
        ctx.sync()
        assert np.array_equal(do.get(), want), rep
    for b, dq, do, want, graph, gexec in made:
        hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
        dq.free()
        do.free()
    p.free()


def test_a_context_closes_over_its_caches():
    """Caches and batches end with their context, and say so afterwards."""
    c = pb.Context(0)
    cache = pb.KvCache(c, 1, 4, 2, 64, 4, 2, 100)
    b = cache.batch([0], [3])
    c.close()
    for call in (lambda: b.attention_dev(0, 16, 16), lambda: cache.length(0), lambda: cache.batch([1], [1])):
        with pytest.raises(pb.PbxError):
            call()
    b.free()
    cache.free()
