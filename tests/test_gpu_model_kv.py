"""The resident model over a paged 8-bit cache of many sequences
(Model.forward_kv) and its log probabilities (Model.logprobs): append,
attention and log probabilities run together as a server runs them."""
import json

import numpy as np
import pytest

import oracle
import purebee_amd as pb
from purebee_amd import native, synth
from tests.conftest import rel_l2
from tests.kv_ref import BLOCK, rotate
from tests.test_gpu_logprobs import near, reference

pytestmark = pytest.mark.gpu

SMALL = dict(dim=128, hidden_dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=300, max_seq=256,
             weight_type=pb.TYPE_F32, embed_type=pb.TYPE_F32, rope_theta=10000.0, weight_std=0.08)
CONFIGS = {
    "f32": SMALL,
    "q8_0": dict(SMALL, weight_type=pb.TYPE_Q8_0, embed_type=pb.TYPE_Q8_0, n_heads=2, n_kv_heads=1, dim=128),
    # the shapes of the rows kernels (1 to 8 rows of a Q4_0 model of this width)
    "q4_0": dict(SMALL, dim=2048, hidden_dim=8192, n_layers=1, n_heads=32, n_kv_heads=8, vocab_size=512,
                 weight_type=pb.TYPE_Q4_0, embed_type=pb.TYPE_Q4_0, rope_theta=500000.0, weight_std=0.02),
}


class Server:
    """A model, a cache, and the same model in 64 bits over the values that the
    GPU's cache holds."""

    def __init__(self, ctx, cfg, seqs=3, n_pages=24, page=32, **kv):
        self.ctx, self.cfg = ctx, cfg
        self.w = {}
        self.model = synth.build(ctx, cfg, 4242, self._keep)
        self.hd = cfg["dim"] // cfg["n_heads"]
        self.cache = pb.KvCache(ctx, cfg["n_layers"], cfg["n_heads"], cfg["n_kv_heads"], self.hd, n_pages, seqs, 512,
                                page_tokens=page, rope_theta=cfg["rope_theta"], **kv)
        self.appends = {}  # (sequence, block): batches that appended to it

    def _keep(self, spec, data):
        tid, layer, N, K, t = spec
        f = np.asarray(data, np.float32) if t == pb.TYPE_F32 else oracle.dequant(t, data, N * K)
        self.w[tid, layer] = f.astype(np.float64).reshape(N, K)

    def free(self):
        self.cache.free()
        self.model.free()

    def held(self, layer, seq):
        """Keys and values of a sequence in the GPU's cache."""
        n, G = self.cache.length(seq), self.cfg["n_kv_heads"]
        b = self.cache.batch([seq], [n], [0])
        k, v = (self.ctx.alloc(4 * n * G * self.hd) for _ in range(2))
        b.read_dev(layer, k.ptr, v.ptr)
        self.ctx.sync()
        out = [x.download(np.float32, n * G * self.hd).reshape(n, G, self.hd).astype(np.float64) for x in (k, v)]
        for x in (k, v, b):
            x.free()
        return out

    def expect(self, seqs, starts, counts, tokens):
        """Logits of every row in 64 bits; the cache's new rows lie within their codes' roundings of the keys and values."""
        c, H, G, hd, n = self.cfg, self.cfg["n_heads"], self.cfg["n_kv_heads"], self.hd, sum(counts)
        for s, a, m in zip(seqs, starts, counts):
            for blk in range(a // BLOCK, (a + m + BLOCK - 1) // BLOCK if m else 0):
                if a <= blk * BLOCK:
                    self.appends[s, blk] = 0
                self.appends[s, blk] += 1

        def norm(x, w):
            return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w

        x = self.w[native.T_TOKEN_EMBD, -1][tokens]
        pos = np.concatenate([a + np.arange(m) for a, m in zip(starts, counts)])
        for l in range(c["n_layers"]):
            W = lambda t: self.w[t, l]  # noqa: B023,E731
            y = norm(x, W(native.T_ATTN_NORM)[0])
            q = rotate((y @ W(native.T_ATTN_Q).T).reshape(n, H, hd), pos, "pairs", hd, c["rope_theta"])
            k = rotate((y @ W(native.T_ATTN_K).T).reshape(n, G, hd), pos, "pairs", hd, c["rope_theta"])
            v = (y @ W(native.T_ATTN_V).T).reshape(n, G, hd)
            o = np.empty((n, H, hd))
            r = 0
            for s, a, m in zip(seqs, starts, counts):
                kk, vv = self.held(l, s)
                for got, new in ((kk, k[r:r + m]), (vv, v[r:r + m])):
                    for t in range(m):
                        blk = (a + t) // BLOCK
                        # half a step of the block's scale, and one more for every batch that may have raised it
                        step = np.abs(got[blk * BLOCK:(blk + 1) * BLOCK]).max((0, 2)) / 127
                        off = np.abs(got[a + t] - new[t]).max(-1)
                        assert (off <= 0.5 * (1 + self.appends[s, blk]) * step * 1.01 + 1e-5 * np.abs(new).max()).all()
                for t in range(m):
                    e = a + t + 1
                    for h in range(H):
                        p = kk[:e, h * G // H] @ q[r + t, h] / np.sqrt(hd)
                        p = np.exp(p - p.max())
                        o[r + t, h] = p @ vv[:e, h * G // H] / p.sum()
                r += m
            x = x + o.reshape(n, -1) @ W(native.T_ATTN_OUTPUT).T
            y = norm(x, W(native.T_FFN_NORM)[0])
            g = y @ W(native.T_FFN_GATE).T
            x = x + (g / (1 + np.exp(-g)) * (y @ W(native.T_FFN_UP).T)) @ W(native.T_FFN_DOWN).T
        return norm(x, self.w[native.T_OUTPUT_NORM, -1][0]) @ self.w[native.T_TOKEN_EMBD, -1].T


# Roundings of a few layers in 22 bits and more, relative to a row's logits: a
# linear's 32-bit sums and fp16-pair activations are up to 1e-6 off, and a layer
# has five of them in a chain.
TOL = 3e-5


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_batches_of_sequences(ctx, name):
    """Prompts, chunks and single tokens of several sequences, packed: every kernel path that the row count chooses."""
    s = Server(ctx, CONFIGS[name])
    rng = np.random.default_rng(7)
    for seqs, counts in (([0], [40]), ([1, 0], [3, 1]), ([2, 1, 0], [5, 1, 1]), ([0, 2], [1, 1]), ([1], [1]),
                         ([2, 0, 1], [20, 1, 4]), ([1, 2], [33, 2])):
        print(f"[case] forward_kv {name} {seqs} {counts}", flush=True)
        starts = [s.cache.length(i) for i in seqs]
        tokens = rng.integers(0, s.cfg["vocab_size"], sum(counts)).astype(np.int32)
        b = s.cache.batch(seqs, counts)
        logits, nxt = s.model.forward_kv(b, tokens, all_rows=True)
        want = s.expect(seqs, starts, counts, tokens)
        assert logits.shape == want.shape
        for got, ref in zip(logits, want):
            assert rel_l2(got, ref) <= TOL
        assert np.array_equal(nxt, logits.argmax(-1))
        b.free()
    s.free()


def test_last_rows_and_answers(ctx):
    """The last rows alone are the batch's last rows; log probabilities are those of the logits."""
    s = Server(ctx, CONFIGS["q8_0"], page=64)
    rng = np.random.default_rng(8)
    seqs, counts = [2, 0, 1], [35, 0, 6]
    tokens = rng.integers(0, 300, 41).astype(np.int32)
    b = s.cache.batch(seqs, counts)
    every, _ = s.model.forward_kv(b, tokens, all_rows=True)
    logits, nxt, lp = s.model.forward_kv(b, tokens, targets=[5, 7], top=4)   # the same rows once more
    assert logits.shape == (2, 300)
    for got, row in zip(logits, (34, 40)):
        assert rel_l2(got, every[row]) <= TOL
    assert np.array_equal(nxt, logits.argmax(-1))
    rl, re, ri, rt, t1, t2 = reference(logits, [5, 7], 4)
    near(lp["logp"], rl, t1)
    near(lp["entropy"], re, t2)
    assert np.array_equal(lp["top_ids"], ri)
    near(lp["top_logp"], rt, t1[:, None] + np.zeros(rt.shape), 2.0 ** -22)
    assert s.model.forward_kv(b, tokens, want_logits=False)[0] is None
    none = s.cache.batch([0, 1], [0, 0])
    logits, nxt = s.model.forward_kv(none, [])
    assert logits.shape == (0, 300) and len(nxt) == 0
    s.free()


def test_a_server_loop(ctx):
    """Greedy tokens of three sequences that start at different times, one rolled back and one replaced, equal those of the same
    sequences served alone."""
    cfg = CONFIGS["f32"]
    prompts = [[3, 7, 9, 250], [100, 101, 102, 103, 104, 105, 106], [42]]

    def alone(prompt, steps):
        s = Server(ctx, cfg, seqs=1)
        toks, margins = list(prompt), []
        logits, nxt = s.model.forward_kv(s.cache.batch([0], [len(prompt)]), prompt)
        for _ in range(steps):
            top = np.sort(logits[0])
            margins.append((top[-1] - top[-2]) / np.linalg.norm(logits[0]))
            toks.append(int(nxt[0]))
            logits, nxt = s.model.forward_kv(s.cache.batch([0], [1]), [toks[-1]])
        s.free()
        # codes of f32 keys and values next to a border may differ between row counts: only clear choices are compared
        clear = next((i for i, m in enumerate(margins) if m < 1e-2), steps)
        return toks[:len(prompt) + clear]

    want = [alone(p, 12) for p in prompts]
    s = Server(ctx, cfg)
    b = pb.KvBatch(s.cache)
    got = {0: list(prompts[0]), 1: list(prompts[1])}
    _, nxt = s.model.forward_kv(b.set([0, 1], [4, 7]), prompts[0] + prompts[1])
    got[0].append(int(nxt[0])), got[1].append(int(nxt[1]))
    got[2] = list(prompts[2])
    order = [2, 0, 1]
    for t in range(11):
        feed = [got[i][-1] for i in order]
        _, nxt = s.model.forward_kv(b.set(order, [1] * 3), feed)
        for i, n in zip(order, nxt):
            got[i].append(int(n))
        if t == 4:  # a rejected draft: three positions of sequence 1 are cut and taken again
            s.cache.truncate(1, s.cache.length(1) - 3)
            got[1] = got[1][:-3]
            for _ in range(3):
                _, nxt = s.model.forward_kv(b.set([1], [1]), [got[1][-1]])
                got[1].append(int(nxt[0]))
    for i in range(3):
        n = min(len(want[i]), len(got[i]))
        assert got[i][:n] == want[i][:n], i
    assert max(len(w) - len(p) for w, p in zip(want, prompts)) > 0
    s.free()


def test_logprobs_of_the_models_own_cache(ctx):
    """Model.logprobs: those of forward_batch's logits, the cache left as forward_batch leaves it."""
    for name in ("f32", "q4_0"):
        m = synth.build(ctx, CONFIGS[name], 99)
        rng = np.random.default_rng(9)
        tokens = rng.integers(0, m.vocab, 45).astype(np.int32)
        for a, e in ((0, 40), (40, 41), (41, 45)):
            logits, nxt = m.forward_batch(tokens[a:e], a)
            m.rollback(a)
            targets = np.append(tokens[a + 1:e], -1)
            lp = m.logprobs(tokens[a:e], a, targets, top=3)
            rl, re, ri, rt, t1, t2 = reference(logits, targets, 3)
            near(lp["logp"], rl, t1)
            near(lp["entropy"], re, t2)
            assert np.array_equal(lp["top_ids"], ri) and np.array_equal(lp["top_ids"][:, 0], nxt)
            near(lp["top_logp"], rt, t1[:, None] + np.zeros(rt.shape), 2.0 ** -22)
        assert "logp" not in m.logprobs(tokens[:3], 0)
        m.free()


def test_the_models_own_cache_is_left_alone(ctx):
    s = Server(ctx, CONFIGS["f32"])
    tokens = np.arange(1, 31, dtype=np.int32)
    s.model.forward(tokens, 0)
    before, _ = s.model.forward([5], 30)
    s.model.rollback(30)
    s.model.forward_kv(s.cache.batch([0], [30]), tokens[::-1].copy())
    after, _ = s.model.forward([5], 30)
    assert np.array_equal(before, after)
    s.free()


def test_refusals(ctx):
    s = Server(ctx, CONFIGS["f32"])
    b = s.cache.batch([0], [3])
    m = s.model
    with pytest.raises(ValueError):
        m.forward_kv(b, [1, 2])
    for bad in ([1, 2, 300], [-1, 2, 3]):
        with pytest.raises(pb.PbxError, match="out of range"):
            m.forward_kv(b, bad)
    with pytest.raises(pb.PbxError, match="top"):
        m.forward_kv(b, [1, 2, 3], top=33)
    with pytest.raises(pb.PbxError, match="top"):
        m.logprobs([1, 2, 3], 0, top=33)
    with pytest.raises(pb.PbxError, match="max_seq"):
        m.logprobs([1], 256)
    with pytest.raises(ValueError):
        m.logprobs([1, 2], 0, targets=[1])
    other = pb.KvCache(ctx, 2, 4, 4, 32, 4, 1, 64)
    with pytest.raises(pb.PbxError, match="shape"):
        m.forward_kv(other.batch([0], [1]), [1])
    L, n = m.ctx.L, np.zeros(4, np.int32)
    out = np.zeros(4, np.float32)
    assert L.pbx_model_forward_kv(m._m, pb.KvBatch(s.cache)._ptr, n.ctypes.data, 0, None, None, None, 0, None, None,
                                  None, None) == -1   # not set
    assert L.pbx_model_forward_kv(m._m, b._ptr, None, 0, None, None, None, 0, None, None, None, None) == -1
    assert L.pbx_model_forward_kv(m._m, b._ptr, n.ctypes.data, 0, None, None, n.ctypes.data, 0, None, None, None,
                                  None) == -1         # targets without logp
    assert L.pbx_model_logprobs(m._m, n.ctypes.data, 4, 0, None, 0, out.ctypes.data, None, None, None) == -1
    with pb.Context(0) as fresh:
        far = pb.KvCache(fresh, 2, 4, 2, 32, 4, 1, 64)
        with pytest.raises(pb.PbxError, match="contexts"):
            m.forward_kv(far.batch([0], [1]), [1])
        far.free()
    s.cache.truncate(0, 1)
    with pytest.raises(pb.PbxError, match="dropped"):
        m.forward_kv(b, [1, 2, 3])
    other.free()
    s.free()


def test_logprobs_from_node(ctx, tmp_path):
    """HipLlamaRuntime.logprobs answers as Model.logprobs does."""
    import os
    from tests.test_gpu_js import JS, run_node
    cfg = CONFIGS["q8_0"]
    names = dict(synth.GGUF_NAMES)
    files = []

    def keep(spec, data):
        tid, layer, N, K, t = spec
        nm = names[tid] if layer < 0 else f"blk.{layer}.{names[tid]}"
        fn = f"t{len(files)}.bin"
        np.ascontiguousarray(data).tofile(tmp_path / fn)
        files.append([nm, fn, "f32" if data.dtype == np.float32 else "u8"])

    m = synth.build(ctx, cfg, 77, keep)
    tokens = [int(t) for t in synth.random_tokens(78, 9, cfg["vocab_size"])]
    want = m.logprobs(tokens[:-1], 0, tokens[1:], top=3)
    m.free()
    out = run_node(tmp_path, f"""
const {{ HipLlamaRuntime }} = require({os.path.join(JS, 'llama-hip.js')!r});
const c = meta.cfg;
const rt = new HipLlamaRuntime({{ dim: c.dim, hiddenDim: c.hidden_dim, nLayers: c.n_layers, nHeads: c.n_heads,
  nKvHeads: c.n_kv_heads, vocabSize: c.vocab_size, seqLen: c.max_seq, ropeTheta: c.rope_theta,
  weightType: 'q8_0', embedType: 'q8_0' }});
for (const [nm, fn, ty] of meta.files) rt.loadTensor(nm, rd(fn, ty === 'f32' ? Float32Array : Uint8Array));
const t = meta.tokens;
const a = rt.logprobs(t.slice(0, -1), 0, {{ targets: t.slice(1), top: 3 }});
rt.rollbackCache(0);
const b = rt.logprobs(t.slice(0, -1), 0);
let refused = 0;
for (const o of [{{ targets: [1] }}, {{ top: 33 }}, {{ top: -1 }}]) {{
  try {{ rt.logprobs(t, 0, o); }} catch (e) {{ refused++; }}
}}
console.log(JSON.stringify({{ logp: [...a.logp], entropy: [...a.entropy], ids: [...a.topIds], top: [...a.topLogp],
  none: b.logp, entropy2: [...b.entropy], empty: b.topIds.length, refused }}));
rt.free();
""", {"cfg": cfg, "files": files, "tokens": tokens})
    got = json.loads(out.strip().splitlines()[-1])
    assert np.array_equal(np.float32(got["logp"]), want["logp"])
    assert np.array_equal(np.float32(got["entropy"]), want["entropy"])
    assert np.array_equal(got["ids"], want["top_ids"].ravel())
    assert np.array_equal(np.float32(got["top"]), want["top_logp"].ravel())
    assert got["none"] is None and got["entropy2"] == got["entropy"] and got["empty"] == 0 and got["refused"] == 3
