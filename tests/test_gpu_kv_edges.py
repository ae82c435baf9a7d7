"""The paged KV cache at the ends of its numbers, against tests/kv_ref.py, and around captures."""
import ctypes
import json
import os

import numpy as np
import pytest

import purebee_amd as pb
from purebee_amd import synth
from tests.kv_ref import Rows, within
from tests.test_gpu_js import JS, run_node
from tests.test_gpu_kv import Pair, _hip
from tests.test_gpu_model_kv import CONFIGS, Server

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("style", ["pairs", "halves"])
@pytest.mark.parametrize("held", [0, 5])
def test_keys_that_leave_f32_when_turned(ctx, style, held):
    """Pairs of finite keys that turn to values past f32's largest (and do not all have the block's largest code), beside
    ordinary ones in the same four dims: codes are those of the 64-bit values, earlier rows' codes too."""
    print(f"[case] keys past f32, {style}, {held} held", flush=True)
    p = Pair(ctx, 2, 2, 64, seqs=1, style=style, seed=31 + held)
    if held:
        p.append([0], [held], p.rows(held, 1e36))
    n = 40
    q, k, v = p.rows(n)
    sign = np.where(p.rng.random(k.shape) < 0.5, np.float32(-1), np.float32(1))
    big = (sign * p.rng.uniform(2.4e38, 3.4e38, k.shape)).astype(np.float32)
    small = (1e37 * p.rng.standard_normal(k.shape)).astype(np.float32)
    pair = np.arange(64) // 2 if style == "pairs" else np.arange(64) % 32
    k = np.where(pair % 2 == 0, big, small)   # every unit of four dims holds a large pair and an ordinary one
    p.append([0], [n], (q, k, v))
    codes = p.ref.k[0].codes
    assert np.isfinite(p.ref.k[0].scales).all() and (np.abs(codes[held:]).max(-1) > 100).any()
    turned = np.abs(codes * np.repeat(p.ref.k[0].scales.astype(np.float64), 32, 0)[:held + n, :, None])
    past = np.abs(codes[turned > float(np.finfo(np.float32).max)])
    assert past.min() < 110 and past.max() == 127   # past f32's largest, not only at the largest code
    p.check_values([0])
    p.free()


def one_key_and_a_tail(ctx, heads, kv_heads, dim, past, rows, at, strength, others=0):
    """`rows` query rows after `past` positions whose keys and values are alike but for one, at `at`, whose score is
    `strength` (natural) above the others' and whose value is 0: the answer is the others' alone.  `others` sequences hold
    the same and are in the batch.

    The bound is RefCache.attention's for roundings relative to each probability, and one for what a probability far below
    its block's largest loses: a pair of fp16 resolves 2^-25, a block's largest is held above 2^5, so 2^-30 of it each
    (2^-36 and less of the sums that other blocks bring), counted for the sum as well."""
    n, seqs = past + rows, 1 + others
    p = Pair(ctx, heads, kv_heads, dim, seqs=seqs, n_pages=seqs * -(-n // 64), page=64, max_seq=8192, style="none",
             seed=int(strength) * 100 + n)
    k = np.zeros((n, kv_heads, dim), np.float32)
    k[..., 1] = 0.25
    k[at, :, 0] = 2 * strength
    v = (1 + 0.1 * p.rng.standard_normal(k.shape)).astype(np.float32)
    v[at] = 0
    q = np.zeros((n, heads, dim), np.float32)
    q[..., 0] = np.sqrt(dim) / 2 * (1 + 0.02 * p.rng.random((n, heads)))
    q[..., 1] = p.rng.standard_normal((n, heads))
    part = lambda a, e: tuple(x[a:e] for x in (q, k, v))  # noqa: E731
    p.append([0], [past], part(0, past))
    _, qr = p.append([0], [rows], part(past, n))
    dk, dv = Rows(ctx, n, kv_heads * dim, k), Rows(ctx, n, kv_heads * dim, v)
    for s in range(1, seqs):
        for a, m in ((0, past), (past, rows)):
            p.cache.batch([s], [m]).append_dev(0, None, dk.ptr + 4 * a * dk.width, dv.ptr + 4 * a * dv.width, None)
    b = p.cache.batch(range(seqs), [rows] * seqs, [past] * seqs)
    want, tol = p.ref.attention([0], [past], [rows], qr)
    kk, vv = p.ref.k[0].values().astype(np.float64), p.ref.v[0].values().astype(np.float64)
    for t in range(rows):
        e = past + t + 1
        for h in range(heads):
            g = h // (heads // kv_heads)
            x = kk[:e, g] @ qr[t, h].astype(np.float64) / np.sqrt(dim)
            pr = np.exp(x - x.max())
            pr /= pr.sum()
            top = np.repeat(np.maximum.reduceat(pr, np.arange(0, e, 32)), 32)[:e] * 2.0 ** -30
            tol[t, h] += top @ np.abs(vv[:e, g]) + top.sum() * np.abs(want[t, h])
    w = heads * dim
    dq, do = Rows(ctx, seqs * rows, w, np.tile(qr, (seqs, 1, 1))), Rows(ctx, seqs * rows, w)
    b.attention_dev(0, dq.ptr, do.ptr)
    ctx.sync()
    for got in do.get().reshape(seqs, *want.shape):
        within(got, want, tol)
    for x in (dq, do, dk, dv):
        x.free()
    p.free()


@pytest.mark.parametrize("strength", [6, 9, 13, 18, 23, 40])
@pytest.mark.parametrize("past,at", [(300, 0), (300, 37), (300, 298), (6000, 0), (6000, 3000), (6000, 5998)])
@pytest.mark.parametrize("rows", [1, 24])
def test_one_key_before_a_long_tail(ctx, strength, past, at, rows):
    """Keys far below a row's largest add up: none is lost to the one that outweighs them, in whole and in split contexts."""
    print(f"[case] one key {strength} above {past}, at {at}, {rows} rows", flush=True)
    one_key_and_a_tail(ctx, 8, 2, 64, past, rows, at, strength)


@pytest.mark.parametrize("dim", [32, 96, 128, 192, 256])
@pytest.mark.parametrize("past", [200, 3000])
@pytest.mark.parametrize("rows", [1, 9])
def test_one_key_before_a_tail_by_head_size(ctx, dim, past, rows):
    print(f"[case] one key, heads of {dim}, {past}, {rows} rows", flush=True)
    one_key_and_a_tail(ctx, 4, 2, dim, past, rows, 70, 16)


@pytest.mark.parametrize("strength", [13, 16, 18, 20, 21, 23])
@pytest.mark.parametrize("heads,kv_heads,dim,past,rows", [(16, 8, 64, 4000, 1), (8, 8, 64, 2500, 40), (8, 8, 128, 4000, 1),
                                                          (8, 8, 256, 4000, 1)])
def test_one_key_before_tails_that_are_not_split(ctx, strength, heads, kv_heads, dim, past, rows):
    """As many sequences as fill the GPU: a wave goes through a quarter or half of a context by itself."""
    print(f"[case] one key {strength} above {past}, heads of {dim}, {rows} rows, 64 sequences", flush=True)
    one_key_and_a_tail(ctx, heads, kv_heads, dim, past, rows, 0, strength, others=63)


def test_calls_that_a_capture_does_not_hold_leave_the_batch_free(ctx):
    """Refused calls, and those of a batch without rows, put nothing into a graph: the batch can be set again after them."""
    hip = _hip()
    p = Pair(ctx, 4, 2, 64, seed=41)
    b, q = p.append([0], [50])
    none = p.cache.batch([0], [0])
    x = Rows(ctx, 50, 256, q)
    stream, graph = ctypes.c_void_p(ctx.stream()), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    for call in (lambda: b.attention_dev(0, None, x.ptr), lambda: b.attention_dev(0, x.ptr, x.ptr, float("nan")),
                 lambda: b.attention_dev(1, x.ptr, x.ptr), lambda: b.append_dev(0, x.ptr, None, x.ptr, x.ptr),
                 lambda: b.append_dev(0, x.ptr, x.ptr, x.ptr, x.ptr, q_stride=252), lambda: b.read_dev(0, x.ptr + 4, None)):
        with pytest.raises(pb.PbxError):
            call()
    b.read_dev(0, None, None)           # nothing is asked for
    none.append_dev(0, None, None, None, None)
    none.attention_dev(0, None, None)
    none.read_dev(0, x.ptr, x.ptr)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    hip.hipGraphDestroy(graph)
    none.set([0], [0])
    b.set([0], [50], [0])
    p.attend(b, [0], [0], [50], q)
    # a call that a graph does hold keeps the batch's rows, thrown away or not; another batch takes its place
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    b.attention_dev(0, x.ptr, x.ptr)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    hip.hipGraphDestroy(graph)
    with pytest.raises(pb.PbxError, match="captured"):
        b.set([0], [50], [0])
    b.free()
    b = p.cache.batch([0], [50], [0])
    p.attend(b, [0], [0], [50], q)
    x.free()
    p.free()


def test_forwards_wait_and_are_refused_in_a_capture(ctx):
    """forward_kv and logprobs wait for their answers: inside a capture they are refused before they begin, the capture goes
    on, and the batch stays free."""
    hip = _hip()
    s = Server(ctx, CONFIGS["f32"])
    tokens = np.arange(1, 41, dtype=np.int32)
    b = s.cache.batch([0], [40])
    want = s.model.forward_kv(b, tokens)[0]
    lp = s.model.logprobs(tokens, 0, tokens)
    k = Rows(ctx, 40, 64)
    stream, graph, gexec = ctypes.c_void_p(ctx.stream()), ctypes.c_void_p(), ctypes.c_void_p()
    other = s.cache.batch([0], [40], [0])
    other.read_dev(0, k.ptr, None)
    ctx.sync()
    held = k.get()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    other.read_dev(0, k.ptr, None)
    for call in (lambda: s.model.forward_kv(b, tokens), lambda: s.model.logprobs(tokens, 0, tokens)):
        with pytest.raises(pb.PbxError, match="captured"):
            call()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(gexec), graph, None, None, 0) == 0
    for _ in range(3):
        k.buf.upload(k.host)
        assert hip.hipGraphLaunch(gexec, stream) == 0
        ctx.sync()
        assert np.array_equal(k.get(), held)
        assert np.array_equal(s.model.forward_kv(b.set([0], [40], [0]), tokens)[0], want)
        assert np.array_equal(s.model.logprobs(tokens, 0, tokens)["logp"], lp["logp"])
    hip.hipGraphExecDestroy(gexec)
    hip.hipGraphDestroy(graph)
    k.free()
    s.free()


def test_a_cache_whose_theta_was_left_out(ctx):
    """A model of another theta than the default refuses it (its tokens would be wrong without an error); a rotation that
    was given is taken as meant."""
    s = Server(ctx, dict(CONFIGS["f32"], rope_theta=500000.0))
    tokens = [1, 2, 3]
    want = s.model.forward_kv(s.cache.batch([0], [3]), tokens)[0]
    shape = (ctx, 2, 4, 2, 32, 8, 2, 64)
    left_out = pb.KvCache(*shape)
    with pytest.raises(ValueError, match="500000"):
        s.model.forward_kv(left_out.batch([0], [3]), tokens)
    for kw, same in ((dict(rope_theta=500000.0), True), (dict(rope_theta=10000.0), False), (dict(rope="none"), False),
                     (dict(rope_theta=500000.0, rope_scale=2.0), False), (dict(rope="halves", rope_theta=500000.0), False)):
        c = pb.KvCache(*shape, **kw)
        assert np.array_equal(s.model.forward_kv(c.batch([0], [3]), tokens)[0], want) == same, kw
        c.free()
    left_out.free()
    s.free()
    s = Server(ctx, CONFIGS["f32"])     # the default is this model's
    want = s.model.forward_kv(s.cache.batch([0], [3]), tokens)[0]
    left_out = pb.KvCache(*shape)
    assert np.array_equal(s.model.forward_kv(left_out.batch([0], [3]), tokens)[0], want)
    left_out.free()
    s.free()


def test_ids_that_int32_does_not_hold(ctx):
    """64-bit ids a multiple of 2^32 away from tokens are not those tokens: no distribution's probability, or refused."""
    s = Server(ctx, CONFIGS["f32"])
    tokens, far = np.arange(5), np.arange(5, dtype=np.int64) + 2 ** 32
    for targets in (far, -far, np.uint64(far), list(far)):
        assert np.isnan(s.model.logprobs(tokens, 0, targets)["logp"]).all()
        lp = s.model.forward_kv(s.cache.batch([0], [5], [0]), tokens, all_rows=True, targets=targets)[2]
        assert np.isnan(lp["logp"]).all()
    for bad in (far, -far):
        with pytest.raises(pb.PbxError, match="out of range"):
            s.model.logprobs(bad, 0)
        with pytest.raises(pb.PbxError, match="out of range"):
            s.model.forward_kv(s.cache.batch([0], [5], [0]), bad)
    want = s.model.logprobs(np.int32(tokens), 0, np.int32(tokens))["logp"]
    for call in (lambda: s.model.logprobs(tokens, 2 ** 32), lambda: s.cache.truncate(2 ** 32), lambda: s.cache.length(2 ** 32),
                 lambda: s.cache.truncate(0, 2 ** 32)):
        with pytest.raises(OverflowError):
            call()
    assert s.cache.length(0) == 5
    for kind in (np.int64, np.uint8, list):
        assert np.array_equal(s.model.logprobs(kind(tokens), 0, kind(tokens))["logp"], want)
    s.free()


def test_ids_and_positions_that_int32_does_not_hold_from_node(ctx, tmp_path):
    cfg = CONFIGS["f32"]
    names, files = dict(synth.GGUF_NAMES), []

    def keep(spec, data):
        tid, layer, N, K, t = spec
        fn = f"t{len(files)}.bin"
        np.ascontiguousarray(data).tofile(tmp_path / fn)
        files.append([names[tid] if layer < 0 else f"blk.{layer}.{names[tid]}", fn])

    synth.build(ctx, cfg, 77, keep).free()
    out = run_node(tmp_path, f"""
const {{ HipLlamaRuntime }} = require({os.path.join(JS, 'llama-hip.js')!r});
const c = meta.cfg, far = 2 ** 32;
const rt = new HipLlamaRuntime({{ dim: c.dim, hiddenDim: c.hidden_dim, nLayers: c.n_layers, nHeads: c.n_heads,
  nKvHeads: c.n_kv_heads, vocabSize: c.vocab_size, seqLen: c.max_seq, ropeTheta: c.rope_theta,
  weightType: 'f32', embedType: 'f32' }});
for (const [nm, fn] of meta.files) rt.loadTensor(nm, rd(fn, Float32Array));
const a = rt.logprobs([1, 2, 3], 0, {{ targets: [2, far + 3, 4] }});
let refused = 0;
for (const [t, at] of [[[1, far + 2, 3], 0], [[1, 2, 3], far], [[1, 2, 3], -far]]) {{
  try {{ rt.logprobs(t, at); }} catch (e) {{ refused++; }}
}}
console.log(JSON.stringify({{ logp: [...a.logp].map(Number.isNaN), refused }}));
rt.free();
""", {"cfg": cfg, "files": files})
    assert json.loads(out.strip().splitlines()[-1]) == {"logp": [False, True, False], "refused": 3}


def test_a_batch_that_was_never_set(ctx):
    """It is refused by the library, and one whose arguments do not match is not left behind."""
    s = Server(ctx, CONFIGS["f32"])
    with pytest.raises(pb.PbxError):
        s.model.forward_kv(pb.KvBatch(s.cache), [])
    made = []
    free = pb.KvBatch.free
    pb.KvBatch.free = lambda b: (made.append(b), free(b))
    try:
        for args in (([0], [1, 2]), ([0], [2 ** 40])):
            with pytest.raises((ValueError, OverflowError)):
                s.cache.batch(*args)
    finally:
        pb.KvBatch.free = free
    assert len(made) == 2 and not any(b._b for b in made)
    s.free()


@pytest.mark.parametrize("size", [1e3, 1e6, 3e7, 9.5e7])
@pytest.mark.parametrize("past,rows", [(70, 2), (1500, 1), (40, 40)])
def test_scores_of_any_size(ctx, size, past, rows):
    """Scores up to 10^8, of either sign, with the largest far ahead of the next: the answer is its value."""
    print(f"[case] scores of {size} after {past}, {rows} rows", flush=True)
    n = past + rows
    for sign in (1, -1):
        p = Pair(ctx, 4, 2, 64, seqs=1, n_pages=60, style="none", seed=61 + past)
        q, k, v = p.rows(n)
        # one dim counts: whole codes 1 to 127 (of either sign) times a power of two, the best key alone at its end
        code = p.rng.integers(30, 100, (n, 2)) if sign > 0 else -p.rng.integers(30, 100, (n, 2))
        best = past // 2
        code[best] = 127 if sign > 0 else -10
        k[:], q[:] = 0, 0
        k[..., 0], k[..., 1] = code / 128, 127 / 128      # (every block's scale is 1 / 128)
        q[..., 0] = size
        part = lambda a, e: tuple(x[a:e] for x in (q, k, v))  # noqa: E731
        p.append([0], [past], part(0, past))
        b, qr = p.append([0], [rows], part(past, n))
        dq, do = Rows(ctx, rows, 256, qr), Rows(ctx, rows, 256)
        b.attention_dev(0, dq.ptr, do.ptr, 128 / 127)
        ctx.sync()
        want = np.broadcast_to(np.repeat(p.ref.v[0].values()[best], 2, axis=0), (rows, 4, 64))
        # the others lie 20 codes and more below, size / 127 each: nothing of them is left; a rounding of 1 / sum and one more
        tol = 2.0 ** -22 * np.abs(want) + 2 * n * np.abs(v).max() * np.exp(-20 * size / 127)
        within(do.get().reshape(want.shape), want, tol)
        for x in (dq, do):
            x.free()
        p.free()
