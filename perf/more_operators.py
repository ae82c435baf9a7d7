"""Performance cases of the operators for many answers to one prompt: branches of cached sequences,
caches that forget, and scores of rows straight from the head's weights.

fork     branches of sequences of the paged 8-bit cache (KvCache.fork) get their own next rows
         (KvBatch.set and append_dev), and everything that they then hold is read back;
compact  branches keep some of their positions, moved together (KvCache.compact), and are read back;
scores   log probabilities of given tokens, entropy and log of the summed exponentials of rows of hidden
         values against a quantised head, without its logits (Context.linear_logprobs_dev);
grad     the rows' gradient of those log probabilities (Context.linear_logprobs_grad_dev).

With `own` false run() computes the same in elementary torch operations.  The cache holds, for every block of
32 positions and every KV head, int8 codes and one f32 scale s: s = max |x| / 127 over the block's rows as
they were appended, code = x / s rounded half to even; when rows appended later raise s, the block's earlier
codes are rounded again.  A compacted block is coded anew from the values that the old codes stand for, keys
turned on by the distance that they moved; blocks whose rows all stay where they are keep their codes.
Borders between codes, and the angles of far positions, are taken in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 32  # positions that share a scale
THETA = 500000.0


def listed():
    return [
        # Beam search of a small model: four beams go on from a short text.
        _fork("fork_beams", 9, 3, 64, prompts=1, length=(150, 150), branches=4, rows=(1, 1)),
        # Sixteen samples of one prompt get their first token.
        _fork("fork_samples", 32, 8, 64, prompts=1, length=(1500, 1500), branches=16, rows=(1, 1)),
        # Chats that share their system prompts, each with its first turn; the other rotation layout.
        _fork("fork_chats", 32, 8, 128, prompts=4, length=(100, 2000), branches=6, rows=(1, 60), rope="halves",
              rope_dim=64),
        # A turn is cut out of a short chat.
        _compact("compact_turn", 32, 8, 64, seqs=1, length=(300, 300), keep="cut", share=0.8),
        # A long chat keeps its first tokens and its last 1,024 positions or so.
        _compact("compact_window", 32, 8, 64, seqs=1, length=(5000, 5000), keep="window", share=0.2),
        # Half of the positions of many sequences is dropped, here and there.
        _compact("compact_evict", 32, 8, 128, seqs=8, length=(500, 6000), keep="scattered", share=0.5,
                 rope="halves"),
        # The score of one token under the head of a 1B model's GGUF file.
        _linear("scores_token", "scores", 1, 128256, 2048, "q6_k"),
        # A few rows of a small model with an odd vocabulary.
        _linear("scores_odd", "scores", 37, 32003, 576, "q8_0"),
        # A document's rows.
        _linear("scores_prompt", "scores", 1000, 128256, 2048, "q8_0"),
        # A draft's rows, small and with an odd vocabulary, and a training batch of a 1B model's head.
        _linear("grad_draft", "grad", 5, 49152, 576, "q4_0"),
        _linear("grad_odd", "grad", 37, 32003, 2048, "f16"),
        _linear("grad_prompt", "grad", 512, 128256, 2048, "q8_0"),
    ]


def _named(name, c):
    return dict(c, name=name) if name else c


def _fork(name, heads, kv_heads, dim, prompts, length, branches, rows, rope="pairs", rope_dim=0, page=64, layers=2):
    """Prompts of length[0]..length[1] positions with `branches` branches each, which get rows[0]..rows[1]
    rows of their own."""
    return _named(name, {"kind": "fork", "heads": heads, "kv_heads": kv_heads, "dim": dim, "seqs": prompts,
                         "length_lo": length[0], "length_hi": length[1], "branches": branches, "rows_lo": rows[0],
                         "rows_hi": rows[1], "rope": rope, "rope_dim": rope_dim or dim, "page": page,
                         "layers": layers})


def _compact(name, heads, kv_heads, dim, seqs, length, keep, share, rope="pairs", rope_dim=0, page=64, layers=2):
    """Sequences of length[0]..length[1] positions keep about `share` of them: "window" the first four and the
    last ones, "cut" all but a range, "scattered" any."""
    return _named(name, {"kind": "compact", "heads": heads, "kv_heads": kv_heads, "dim": dim, "seqs": seqs,
                         "length_lo": length[0], "length_hi": length[1], "keep": keep, "share": share, "rope": rope,
                         "rope_dim": rope_dim or dim, "page": page, "layers": layers})


def _linear(name, kind, rows, vocab, dim, weight):
    return _named(name, {"kind": kind, "rows": rows, "vocab": vocab, "dim": dim, "type": weight})


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["fork", "compact", "scores", "grad"])
    if kind in ("scores", "grad"):
        weight = rng.choice(["q4_0", "q4_1", "q8_0", "q6_k", "f16", "f32"])
        dim = 256 * _log_int(rng, 1, 16) if weight == "q6_k" else 32 * _log_int(rng, 2, 128)
        vocab = _log_int(rng, 300, min(128256, 128256 * 2048 // dim))
        top = 1000 if kind == "scores" else 512
        return _linear(None, kind, _log_int(rng, 1, top), vocab, dim, weight)
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (9, 3, 64), (6, 6, 48), (32, 8, 128), (12, 4, 96), (8, 1, 256),
                                       (20, 5, 80)])
    rope_dim = dim if rng.random() < 0.7 else dim // 2
    more = {"rope": rng.choice(["pairs", "halves"]), "rope_dim": rope_dim, "page": rng.choice([32, 64, 128, 256]),
            "layers": rng.randint(1, 3)}
    values = 50000000 // (kv_heads * dim * more["layers"])  # positions read back
    seqs = _log_int(rng, 1, 8)
    if kind == "fork":
        branches = _log_int(rng, 1, 16)
        hi = _log_int(rng, 20, max(20, min(4000, values // (seqs * branches))))
        rows = _log_int(rng, 1, 64)
        return _fork(None, heads, kv_heads, dim, seqs, (rng.randint(1, hi), hi), branches, (rng.randint(1, rows), rows),
                     **more)
    hi = _log_int(rng, 20, min(8000, 2 * values // seqs))
    return _compact(None, heads, kv_heads, dim, seqs, (rng.randint(1, hi), hi),
                    rng.choice(["window", "cut", "scattered"]), round(rng.uniform(0.05, 0.98), 2), **more)


def _lengths(case):
    """Positions of every source sequence, and the new rows of every branch: given by the case alone."""
    rng = random.Random("%(seqs)d %(length_lo)d %(length_hi)d" % case)
    lengths = [rng.randint(case["length_lo"], case["length_hi"]) for _ in range(case["seqs"])]
    lengths[0] = case["length_hi"]
    rows = [rng.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"] * case["branches"])] \
        if case["kind"] == "fork" else []
    return lengths, rows


def _kept(case):
    """The positions that every sequence keeps, rising."""
    rng = np.random.default_rng([case["seqs"], case["length_lo"], case["length_hi"], int(1000 * case["share"])])
    kept = []
    for n in _lengths(case)[0]:
        k = max(1, round(n * case["share"]))
        if case["keep"] == "window":
            first = min(4, k - 1)
            at = np.r_[:first, n - (k - first):n]
        elif case["keep"] == "cut":
            begin = int(rng.integers(0, k + 1))
            at = np.r_[:begin, begin + n - k:n]
        else:
            at = np.sort(rng.permutation(n)[:k])
        kept.append(at.astype(np.int32))
    return kept


# ---- inputs ------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _rows(g, n, heads, dim, spread):
    """Rows of projections: channels of different size, as trained models have."""
    size = torch.exp(spread * torch.randn(heads, dim, device="cuda", generator=g))
    return torch.randn(n, heads, dim, device="cuda", generator=g) * size


def _cache_inputs(case, seed):
    """Per layer: keys and values of the sources, packed, then of the branches' new rows."""
    g = _generator(seed)
    lengths, rows = _lengths(case)
    G, D = case["kv_heads"], case["dim"]
    return [(_rows(g, sum(lengths), G, D, 0.3), _rows(g, sum(lengths), G, D, 0.2),
             _rows(g, sum(rows), G, D, 0.35), _rows(g, sum(rows), G, D, 0.25)) for _ in range(case["layers"])]


# name: (type in the library, bits of a code)
TYPES = {"f32": (0, 0), "f16": (1, 0), "q4_0": (2, 4), "q4_1": (3, 4), "q8_0": (8, 8), "q6_k": (14, 6)}


def _bytes(x):
    return x.contiguous().view(torch.uint8)


def _weight(case, g):
    """(a head's rows as a file holds them, one row of bytes each; their values in f32)."""
    N, K, kind = case["vocab"], case["dim"], case["type"]
    std = 0.03
    if kind in ("f32", "f16"):
        w = std * torch.randn(N, K, device="cuda", generator=g)
        w = w if kind == "f32" else w.half()
        return _bytes(w), w.float()
    bits = TYPES[kind][1]
    mid = 2 ** (bits - 1)
    if kind == "q6_k":
        B = K // 256
        q = (torch.randn(N, B, 256, device="cuda", generator=g) * 8).round_().clamp_(-32, 31)
        d = (torch.rand(N, B, 1, device="cuda", generator=g) + 0.5).mul_(std / 8 / 64).half()
        sc = (64 + 12 * torch.randn(N, B, 16, device="cuda", generator=g)).round_().clamp_(-128, 127)
        w = q * (d.float() * sc).repeat_interleave(16, dim=-1)
        c = (q + 32).to(torch.uint8).view(N, B, 2, 4, 32)  # [half][quarter][l]
        ql = torch.cat([c[..., 0, :] & 15 | (c[..., 2, :] & 15) << 4, c[..., 1, :] & 15 | (c[..., 3, :] & 15) << 4], -1)
        qh = c[..., 0, :] >> 4 | (c[..., 1, :] >> 4) << 2 | (c[..., 2, :] >> 4) << 4 | (c[..., 3, :] >> 4) << 6
        raw = torch.cat([ql.flatten(-2), qh.flatten(-2), _bytes(sc.to(torch.int8)), _bytes(d)], -1)
        return raw.view(N, -1), w.view(N, K)
    B = K // 32
    q = (torch.randn(N, B, 32, device="cuda", generator=g) * (mid * 0.3)).round_().clamp_(-mid, mid - 1)
    d = (torch.rand(N, B, 1, device="cuda", generator=g) + 0.5).mul_(std / (mid * 0.3)).half()
    if kind == "q8_0":
        return torch.cat([_bytes(d), _bytes(q.to(torch.int8))], -1).view(N, -1), (q * d.float()).view(N, K)
    c = (q + mid).to(torch.uint8)
    c = c[..., :16] | c[..., 16:] << 4
    if kind == "q4_0":
        return torch.cat([_bytes(d), c], -1).view(N, -1), (q * d.float()).view(N, K)
    m = (d.float() * (-mid + torch.randn(N, B, 1, device="cuda", generator=g))).half()
    return torch.cat([_bytes(d), _bytes(m), c], -1).view(N, -1), ((q + mid) * d.float() + m.float()).view(N, K)


def _linear_inputs(case, seed):
    """(head, its values, rows, targets, gradients of the log probabilities): rows that lean on their target's
    weights by different amounts, so that it is anything from likely to unlikely."""
    g = _generator(seed)
    M = case["rows"]
    raw, w = _weight(case, g)
    target = torch.randint(0, case["vocab"], (M,), device="cuda", generator=g)
    row = w[target]
    x = 1.5 * torch.randn(M, case["dim"], device="cuda", generator=g)
    lean = (math.log(case["vocab"]) + 2) * 0.9  # where all have it, most of the probability is the targets'
    x += lean * torch.rand(M, 1, device="cuda", generator=g) * row / row.square().sum(1, keepdim=True).clamp_min(1e-3)
    grad = -torch.rand(M, device="cuda", generator=g) / M
    if case["kind"] == "grad":  # some rows of a batch are padding, without a target
        target = torch.where(torch.rand(M, device="cuda", generator=g) < (0.1 if M >= 8 else 0.0), -1, target)
    return raw, w, x, target.to(torch.int32), grad


class _State:
    """What a program holds on to; gives its device memory back when dropped."""

    cache = weight = None

    def __del__(self):
        if self.cache is not None:
            self.cache.free()
        if self.weight is not None:
            self.weight.free()


_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        import purebee_amd as pb
        _ctx = pb.Context(0)
    return _ctx


def _packed(starts, counts):
    """(sequence, position) of every row of a packed batch."""
    counts = torch.tensor(counts)
    seq = torch.repeat_interleave(torch.arange(len(counts)), counts)
    first = torch.tensor(starts) - (torch.cumsum(counts, 0) - counts)
    return seq.cuda(), (torch.arange(len(seq)) + first[seq]).cuda()


def _prepare_cache(case, seed):
    s = _State()
    s.case = case
    lengths, rows = _lengths(case)
    layers = _cache_inputs(case, seed)
    if case["kind"] == "fork":
        s.parents = [p for p in range(case["seqs"]) for _ in range(case["branches"])]
        s.rows = rows
        s.held = [lengths[p] + r for p, r in zip(s.parents, rows)]
    else:
        s.parents = list(range(case["seqs"]))
        s.kept = _kept(case)
        s.held = [len(k) for k in s.kept]
    n = len(s.parents)
    s.new = [(k, v) for _, _, k, v in layers]
    s.k_out = torch.empty(case["layers"], sum(s.held), case["kv_heads"], case["dim"], device="cuda")
    s.v_out = torch.empty_like(s.k_out)
    if own:
        import purebee_amd as pb
        s.branches = list(range(case["seqs"], case["seqs"] + n))
        page = case["page"]
        most = max(lengths) + max(rows + [0])
        s.cache = pb.KvCache(_context(), n_layers=case["layers"], n_heads=case["heads"], n_kv_heads=case["kv_heads"],
                             head_dim=case["dim"], page_tokens=page,
                             n_pages=sum(-(-a // page) for a in lengths) + sum(-(-h // page) + 1 for h in s.held),
                             max_seqs=case["seqs"] + n, max_seq=most, rope=case["rope"], rope_dim=case["rope_dim"],
                             rope_theta=THETA)
        torch.cuda.synchronize()  # the context works on a stream of its own
        fill = s.cache.batch(range(case["seqs"]), lengths)
        for layer, (k, v, _, _) in enumerate(layers):
            fill.append_dev(layer, None, k.data_ptr(), v.data_ptr(), None)
        _context().sync()
        fill.free()
        s.grown, s.whole = pb.KvBatch(s.cache), pb.KvBatch(s.cache)
    else:
        i = torch.arange(case["rope_dim"] // 2, dtype=torch.float64)
        s.freq = torch.pow(torch.tensor(THETA, dtype=torch.float64), -2 * i / case["rope_dim"]).cuda()
        s.lengths = torch.tensor(lengths, device="cuda")
        s.codes = [_plain_cache(case, lengths, k, v, s.freq) for k, v, _, _ in layers]
        if case["kind"] == "compact":
            s.seq, s.at = _packed([0] * n, s.held)
            s.old = torch.from_numpy(np.concatenate(s.kept)).long().cuda()
        else:
            s.seq, s.at = _packed([lengths[p] for p in s.parents], rows)
            s.all_seq, s.all_at = _packed([0] * n, s.held)
        s.parent = torch.tensor(s.parents, device="cuda")
    torch.cuda.synchronize()
    return s


def _prepare_linear(case, seed):
    s = _State()
    s.case = case
    raw, w, s.x, s.target, s.grad = _linear_inputs(case, seed)
    M = case["rows"]
    if case["kind"] == "grad":
        lse = torch.empty(M, device="cuda")
        for at in range(0, M, 64):
            lse[at:at + 64] = torch.logsumexp(_products64(s.x[at:at + 64], w), 1).float()
        s.lse = lse
        s.dx = torch.empty_like(s.x)
    else:
        s.logp, s.entropy, s.lse = (torch.empty(M, device="cuda") for _ in range(3))
    if own:
        ctx = _context()
        s.weight = ctx.upload(TYPES[case["type"]][0], case["vocab"], case["dim"], raw.cpu().numpy().ravel())
        s.work = torch.empty(max(1, ctx.linear_logprobs_workspace(s.weight, M, grad=case["kind"] == "grad")),
                             device="cuda", dtype=torch.uint8)
    else:
        s.w = w
    torch.cuda.synchronize()
    return s


def prepare(case, seed):
    return _prepare_linear(case, seed) if case["kind"] in ("scores", "grad") else _prepare_cache(case, seed)


# ---- the plain form ------------------------------------------------------------

def _rotate(x, by, freq, case):
    """x: [rows, heads, dim] in 64 bits, turned by `by` positions each."""
    ang = (by.double()[:, None] * freq)[:, None]
    c, s = ang.cos(), ang.sin()
    r = case["rope_dim"]
    if case["rope"] == "pairs":
        u, v = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([u * c - v * s, u * s + v * c], -1).flatten(-2)
    else:
        u, v = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([u * c - v * s, u * s + v * c], -1)
    return torch.cat([y, x[..., r:]], -1)


def _scale_of(x):
    """f32 scales of blocks: [.., blocks, heads] of x: [.., blocks, BLOCK, heads, dim]."""
    s = (x.abs().amax((-3, -1)) / 127).float()
    return torch.where(s < 2.0 ** -120, torch.zeros_like(s), s)


def _codes(x, s):
    s = s.double()[..., None, :, None]
    return torch.where(s > 0, (x / s).round(), torch.zeros_like(x))


def _blocks(x):
    return x.unflatten(-3, (-1, BLOCK))


def _padded(x, seq, at, n, length):
    out = torch.zeros(n, length, *x.shape[1:], device="cuda", dtype=x.dtype)
    out[seq, at] = x
    return out


def _plain_cache(case, lengths, k, v, freq):
    """(codes [seqs, positions, heads, dim], scales [seqs, blocks, heads]) of keys, then of values."""
    seq, pos = _packed([0] * len(lengths), lengths)
    length = -(-max(lengths) // BLOCK) * BLOCK
    made = []
    for x, turn in ((k, True), (v, False)):
        codes = torch.zeros(case["seqs"], length, case["kv_heads"], case["dim"], device="cuda", dtype=torch.int8)
        scale = torch.zeros(case["seqs"], length // BLOCK, case["kv_heads"], device="cuda")
        for h in range(case["kv_heads"]):  # one head at a time bounds the 64-bit copies
            y = x[:, h:h + 1].double()
            y = _blocks(_padded(_rotate(y, pos, freq, case) if turn else y, seq, pos, case["seqs"], length))
            scale[..., h:h + 1] = _scale_of(y)
            codes[:, :, h:h + 1] = _codes(y, scale[..., h:h + 1]).flatten(1, 2).to(torch.int8)
        made.append((codes, scale))
    return made


def _plain_fork(s):
    """Every branch's copy of its parent's codes; its new rows into the blocks at its end."""
    c = s.case
    n = len(s.parents)
    length = -(-max(s.held) // BLOCK) * BLOCK
    out = {"k": [], "v": []}
    start = s.lengths[s.parent]
    first = start // BLOCK  # block of a branch's first new row
    window = -(-(c["rows_hi"] + BLOCK - 1) // BLOCK)  # blocks that new rows may touch
    each = torch.arange(n, device="cuda")
    for layer in range(c["layers"]):
        for name, (codes, scale), new, turn in (("k", s.codes[layer][0], s.new[layer][0], True),
                                                ("v", s.codes[layer][1], s.new[layer][1], False)):
            mine = torch.zeros(n, length + window * BLOCK, *codes.shape[2:], device="cuda", dtype=torch.int8)
            mine[:, :codes.shape[1]] = codes[s.parent]
            scl = torch.zeros(n, mine.shape[1] // BLOCK, codes.shape[2], device="cuda")
            scl[:, :scale.shape[1]] = scale[s.parent]
            y = new.double()
            y = _rotate(y, s.at, s.freq, c) if turn else y
            y = _blocks(_padded(y, s.seq, s.at - first[s.seq] * BLOCK, n, window * BLOCK))
            asked = _scale_of(y)
            held = (start - first * BLOCK)[:, None] > torch.arange(BLOCK, device="cuda")  # older rows of that block
            old = torch.where(held.any(1)[:, None], scl[each, first], torch.zeros_like(scl[:, 0]))
            asked[:, 0] = torch.maximum(asked[:, 0], old)
            got = _codes(y, asked)
            past = mine.unflatten(1, (-1, BLOCK))[each, first].double()  # [n, BLOCK, heads, dim]
            past = _codes((past * old.double()[:, None, :, None])[:, None], asked[:, :1])[:, 0]
            got[:, 0] = torch.where(held[:, :, None, None], past, got[:, 0])
            at = first[:, None] + torch.arange(window, device="cuda")
            mine.unflatten(1, (-1, BLOCK))[each[:, None], at] = got.to(torch.int8)
            scl[each[:, None], at] = asked
            picked = mine[s.all_seq, s.all_at].float()
            out[name].append(picked * scl[s.all_seq, s.all_at // BLOCK][..., None])
    return {name: torch.stack(x) for name, x in out.items()}


def _plain_compact(s):
    c = s.case
    n = len(s.parents)
    length = -(-max(s.held) // BLOCK) * BLOCK
    out = {"k": [], "v": []}
    moved = _padded((s.old != s.at)[:, None], s.seq, s.at, n, length)[..., 0].unflatten(1, (-1, BLOCK)).any(2)
    for layer in range(c["layers"]):
        for name, (codes, scale), turn in (("k", s.codes[layer][0], True), ("v", s.codes[layer][1], False)):
            was = scale[s.seq, s.old // BLOCK]
            x = codes[s.seq, s.old].double() * was.double()[..., None]
            y = _blocks(_padded(_rotate(x, s.at - s.old, s.freq, c) if turn else x, s.seq, s.at, n, length))
            scl = _scale_of(y)
            fresh = (_codes(y, scl).float() * scl[..., None, :, None]).flatten(1, 2)[s.seq, s.at]
            kept = codes[s.seq, s.old].float() * was[..., None]
            out[name].append(torch.where(moved[s.seq, s.at // BLOCK][:, None, None], fresh, kept))
    return {name: torch.stack(x) for name, x in out.items()}


PIECE = 16384  # vocabulary entries at a time


def _plain_scores(s):
    M, V = s.case["rows"], s.case["vocab"]
    top = torch.full((M, 1), -math.inf, device="cuda")
    total, spread = torch.zeros(M, 1, device="cuda"), torch.zeros(M, 1, device="cuda")
    hit = torch.zeros(M, 1, device="cuda")
    target = s.target.long()[:, None]
    for at in range(0, V, PIECE):
        z = torch.matmul(s.x, s.w[at:at + PIECE].T)
        here = (target >= at) & (target < at + z.shape[1])
        hit = torch.where(here, z.gather(1, (target - at).clamp(0, z.shape[1] - 1)), hit)
        more = torch.maximum(top, z.amax(1, keepdim=True))
        shrink = (top - more).exp()
        spread = torch.where(total > 0, shrink * (spread + total * (top - more)), torch.zeros_like(spread))
        z -= more
        e = z.exp()
        total = total * shrink + e.sum(1, keepdim=True)
        spread += (e * z).sum(1, keepdim=True)
        top = more
    lse = top + total.log()
    return {"logp": (hit - lse)[:, 0], "entropy": (total.log() - spread / total)[:, 0], "lse": lse[:, 0]}


def _plain_grad(s):
    V = s.case["vocab"]
    target = s.target.long()
    dx = torch.zeros_like(s.x)
    for at in range(0, V, PIECE):
        w = s.w[at:at + PIECE]
        p = torch.matmul(s.x, w.T)
        p -= s.lse[:, None]
        p.exp_()
        dx -= torch.matmul(p, w)
    dx += s.w[target.clamp(min=0)]
    return torch.where(target[:, None] < 0, torch.zeros_like(dx), dx * s.grad[:, None])


def run(s):
    kind = s.case["kind"]
    if not own:
        return {"fork": _plain_fork, "compact": _plain_compact, "scores": _plain_scores, "grad": _plain_grad}[kind](s)
    M = s.case.get("rows")
    if kind == "scores":
        _context().linear_logprobs_dev(s.weight, s.x.data_ptr(), M, s.target.data_ptr(), s.logp.data_ptr(),
                                       s.entropy.data_ptr(), s.lse.data_ptr(), s.work.data_ptr(), s.work.numel())
        return {"logp": s.logp, "entropy": s.entropy, "lse": s.lse}
    if kind == "grad":
        _context().linear_logprobs_grad_dev(s.weight, s.x.data_ptr(), M, s.target.data_ptr(), s.lse.data_ptr(),
                                            s.grad.data_ptr(), s.dx.data_ptr(), s.work.data_ptr(), s.work.numel())
        return s.dx
    s.cache.fork(s.branches, s.parents)
    if kind == "fork":
        s.grown.set(s.branches, s.rows)
        for layer, (k, v) in enumerate(s.new):
            s.grown.append_dev(layer, None, k.data_ptr(), v.data_ptr(), None)
    else:
        s.cache.compact(s.branches, s.kept)
    s.whole.set(s.branches, s.held, [0] * len(s.held))
    for layer in range(s.case["layers"]):
        s.whole.read_dev(layer, s.k_out[layer].data_ptr(), s.v_out[layer].data_ptr())
    return {"k": s.k_out, "v": s.v_out}


def _row_bytes(case):
    """Of a head's row in its type."""
    K = case["dim"]
    return {"f32": 4 * K, "f16": 2 * K, "q4_0": K // 32 * 18, "q4_1": K // 32 * 20, "q8_0": K // 32 * 34,
            "q6_k": K // 256 * 210}[case["type"]]


def work(case):
    if case["kind"] in ("scores", "grad"):
        M, V, K = case["rows"], case["vocab"], case["dim"]
        head = V * _row_bytes(case) + 4 * M * K
        if case["kind"] == "scores":
            return {"bytes": head + 16 * M, "flops": 2 * M * V * K + 5 * M * V}
        return {"bytes": head + 12 * M + 4 * M * K, "flops": 4 * M * V * K + 3 * M * V}
    lengths, rows = _lengths(case)
    L, G, D = case["layers"], case["kv_heads"], case["dim"]
    if case["kind"] == "fork":
        start = [lengths[p] for p in range(case["seqs"]) for _ in range(case["branches"])]
        held = sum(start) + sum(rows)
        own_rows = sum(a % BLOCK + r for a, r in zip(start, rows))  # of blocks that a branch does not share
        read = sum(lengths) + own_rows
        # new rows in, the blocks that they touch in and out, everything held read once and its values out
        return {"bytes": 2 * L * G * D * (4 * sum(rows) + 2 * own_rows + read + 4 * held), "flops": 3 * L * G * D * held}
    held = sum(len(k) for k in _kept(case))
    # kept rows in, coded rows out and in again, their values out
    return {"bytes": 2 * L * G * D * (3 + 4) * held, "flops": 10 * L * G * D * held}


# ---- in 64 bits ----------------------------------------------------------------

def _turn(x, by, case):
    """Rows turned by `by` positions, as complex numbers times e^(i angle)."""
    r = case["rope_dim"]
    half = r // 2
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    ang = torch.outer(by.double(), torch.exp(i * (-2 * math.log(THETA) / r)))
    y = x.double().clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if case["rope"] == "pairs" else (slice(0, half), slice(half, r))
    z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.ones_like(ang), ang)[:, None]
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _held(x, pieces):
    """Values of rows x (64 bits) that were appended to an empty sequence in `pieces` (their ends)."""
    n = len(x)
    blocks = -(-n // BLOCK)
    pad = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, blocks * BLOCK - n)).view(blocks, BLOCK, *x.shape[1:])
    at = torch.arange(blocks * BLOCK, device="cuda").view(blocks, BLOCK)[:, :, None, None]
    scale = torch.zeros(blocks, 1, x.shape[1], 1, device="cuda", dtype=torch.float64)
    code = torch.zeros_like(pad)
    begin = 0
    for end in pieces:
        new = (at >= begin) & (at < end)
        peak = torch.where(new, pad, 0.0).abs().amax((1, 3), keepdim=True)
        grown = torch.maximum(scale, (peak / 127).float().double())
        code = torch.where(new, torch.round(pad / grown), torch.round(code * scale / grown).nan_to_num(0.0))
        scale, begin = grown, end
    return torch.where(at < n, code * scale, 0.0).reshape(-1, *x.shape[1:])[:n]


def _exact_cache(case, seed):
    lengths, rows = _lengths(case)
    kept = _kept(case) if case["kind"] == "compact" else None
    got = {"k": [], "v": []}
    for pk, pv, k, v in _cache_inputs(case, seed):
        layer = {"k": [], "v": []}
        past = at = 0
        for p, n in enumerate(lengths):
            pos = torch.arange(n, device="cuda")
            for name, old, new in (("k", pk[past:past + n], k), ("v", pv[past:past + n], v)):
                turned = _turn(old, pos, case) if name == "k" else old.double()
                if kept is None:
                    row = at
                    for r in rows[p * case["branches"]:(p + 1) * case["branches"]]:
                        more = new[row:row + r]
                        more = _turn(more, torch.arange(n, n + r, device="cuda"), case) if name == "k" else more.double()
                        layer[name].append(_held(torch.cat([turned, more]), [n, n + r]).float())
                        row += r
                else:
                    at_old = torch.from_numpy(kept[p]).long().cuda()
                    x = _held(turned, [n])[at_old]
                    j = torch.arange(len(at_old), device="cuda")
                    y = _held(_turn(x, j - at_old, case) if name == "k" else x, [len(j)])
                    stay = int((at_old == j).sum())  # positions rise: those before the first that moves
                    whole = torch.arange(len(j), device="cuda") < (len(j) if stay == len(j) else stay // BLOCK * BLOCK)
                    layer[name].append(torch.where(whole[:, None, None], x, y).float())
            if kept is None:
                at += sum(rows[p * case["branches"]:(p + 1) * case["branches"]])
            past += n
        for name in got:
            got[name].append(torch.cat(layer[name]))
    return {name: torch.stack(x).double() for name, x in got.items()}


def _products64(x, w):
    """x . w in 64 bits, a part of the vocabulary at a time."""
    return torch.cat([x.double() @ part.double().T for part in w.split(32768)], 1)


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return _exact_cache(case, seed)
    _, w, x, target, grad = _linear_inputs(case, seed)
    out = {"logp": [], "entropy": [], "lse": []}
    dx = []
    for rows, t, g in zip(x.split(128), target.long().split(128), grad.double().split(128)):
        z = _products64(rows, w)
        lp = torch.log_softmax(z, 1)
        p = lp.exp()
        if case["kind"] == "scores":
            out["logp"].append(lp.gather(1, t[:, None])[:, 0])
            out["entropy"].append(-(p * lp).sum(1))
            out["lse"].append((z - lp).amax(1))
            continue
        p.neg_()
        p[torch.arange(len(t), device="cuda"), t.clamp(min=0)] += 1
        p *= torch.where(t < 0, 0.0, g)[:, None]
        dx.append(sum(p[:, at:at + 32768] @ w[at:at + 32768].double() for at in range(0, case["vocab"], 32768)))
    return torch.cat(dx) if dx else {name: torch.cat(v) for name, v in out.items()}
