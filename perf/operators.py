"""Performance cases of the operators that serve many sequences from one resident model.

append     rotate a batch's queries and keys by their positions and append keys and values to the
           paged 8-bit cache (KvBatch.append_dev), then read the blocks it touched back as the
           values they stand for (KvBatch.read_dev);
attention  causal grouped-query attention of a batch's rows over that cache (KvBatch.attention_dev);
logprobs   log probabilities of given tokens, the entropy and the most likely tokens of rows of
           logits (Context.logprobs_dev).

With `own` false run() computes the same in elementary torch operations.  The cache holds, for every
block of 32 positions and every KV head, int8 codes and one f32 scale s: s = max |x| / 127 over the
block's rows as they were appended, code = x / s rounded half to even; when rows appended later raise
s, the block's earlier codes are rounded again, code * s_old / s_new.  Borders between codes, and the
angles of far positions, are taken in 64 bits.
"""
import math
import random

import torch

own = False

BLOCK = 32  # positions that share a scale


def listed():
    return [
        # One user's next token at the start of a chat: the smallest append.
        _kv("append", "append_token", 32, 8, 64, seqs=1, start=(127, 127), rows=(1, 1)),
        # A decode step of a full server, every sequence at its own length.
        _kv("append", "append_tokens_64", 32, 8, 64, seqs=64, start=(16, 4000), rows=(1, 1)),
        # New prompts packed into one batch; the other rotation layout, half of each head rotated.
        _kv("append", "append_prompts", 32, 8, 128, seqs=6, start=(0, 0), rows=(200, 1500),
            rope="halves", rope_dim=64),
        # The attention of one user's next token: short, and at the end of a very long document.
        _kv("attention", "attend_token", 32, 8, 64, seqs=1, start=(128, 128), rows=(1, 1)),
        _kv("attention", "attend_token_long", 32, 8, 64, seqs=1, start=(131000, 131000), rows=(1, 1)),
        # A decode step of a full server.
        _kv("attention", "attend_tokens_64", 32, 8, 64, seqs=64, start=(64, 8000), rows=(1, 1)),
        # Speculative verifies of a small model's sequences: four drafts and the bonus position.
        _kv("attention", "attend_verify", 9, 3, 64, seqs=16, start=(30, 480), rows=(5, 5)),
        # A whole prompt, and later turns of conversations (ragged chunks on top of a past).
        _kv("attention", "attend_prompt", 32, 8, 64, seqs=1, start=(0, 0), rows=(2000, 2000)),
        _kv("attention", "attend_turns", 32, 8, 128, seqs=5, start=(100, 2000), rows=(20, 500), rope="halves"),
        # The probabilities of one step's token, of a whole prompt's, and of a
        # few rows of a small, odd-sized vocabulary.
        {"name": "logprobs_step", "kind": "logprobs", "rows": 1, "vocab": 128256, "top": 8},
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 512, "vocab": 128256, "top": 20},
        {"name": "logprobs_odd", "kind": "logprobs", "rows": 37, "vocab": 32003, "top": 5},
    ]


def _kv(kind, name, heads, kv_heads, dim, seqs, start, rows, rope="pairs", rope_dim=0, page=64):
    """seqs sequences that hold a past of start[0]..start[1] positions and get
    rows[0]..rows[1] new rows."""
    c = {"name": name, "kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "seqs": seqs,
         "start_lo": start[0], "start_hi": start[1], "rows_lo": rows[0], "rows_hi": rows[1],
         "rope": rope, "rope_dim": rope_dim or dim, "page": page}
    if name is None:
        del c["name"]
    return c


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "logprobs", "logprobs"])
    if kind == "logprobs":
        return {"kind": kind, "rows": _log_int(rng, 1, 500), "vocab": _log_int(rng, 300, 128256),
                "top": rng.choice([0, rng.randint(1, 20)])}
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 64), (9, 3, 64), (6, 6, 48), (32, 8, 128), (12, 4, 96),
                                       (8, 1, 256), (20, 5, 80)])
    seqs = _log_int(rng, 1, 64)
    shape = rng.choice(["token", "token", "few", "chunk", "prompt"])
    top = min(131000, 130000000 // (seqs * kv_heads * dim))  # caches up to those of the listed cases
    if shape == "prompt":
        start, seqs = (0, 0), min(seqs, 8)
    else:
        lo = _log_int(rng, 1, top)
        start = (lo, min(top, lo * rng.randint(1, 20)))
    if shape == "token":
        rows = (1, 1)
    elif shape == "few":
        rows = (1, rng.randint(2, 9))
    else:
        hi = _log_int(rng, 16, 1500 // seqs + 16)
        rows = (_log_int(rng, 8, hi), hi)
        start = (min(start[0], 4000 // seqs), min(start[1], 6000 // seqs))
    rope_dim = dim if rng.random() < 0.7 else dim // 2
    return _kv(kind, None, heads, kv_heads, dim, seqs, start, rows, rope=rng.choice(["pairs", "halves"]),
               rope_dim=rope_dim, page=rng.choice([32, 64, 128, 256]))


THETA = 500000.0


def _lengths(case):
    """(past positions, new rows) of every sequence: ragged, given by the case alone."""
    rng = random.Random("%(seqs)d %(start_lo)d %(start_hi)d %(rows_lo)d %(rows_hi)d" % case)
    starts = [rng.randint(case["start_lo"], case["start_hi"]) for _ in range(case["seqs"])]
    rows = [rng.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    starts[0], rows[0] = case["start_hi"], case["rows_hi"]
    return starts, rows


# ---- inputs ------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _frequencies(case):
    i = torch.arange(case["rope_dim"] // 2, dtype=torch.float64)
    return torch.pow(torch.tensor(THETA, dtype=torch.float64), -2 * i / case["rope_dim"]).cuda()


def _packed(starts, counts):
    """(sequence, position) of every row of a packed batch."""
    seq = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    first = torch.tensor(starts) - (torch.cumsum(torch.tensor(counts), 0) - torch.tensor(counts))
    return seq.cuda(), (torch.arange(len(seq)) + first[seq]).cuda()


def _rows(g, n, heads, dim, spread):
    """Rows of projections: channels of different size, as trained models have."""
    size = torch.exp(spread * torch.randn(heads, dim, device="cuda", generator=g))
    return torch.randn(n, heads, dim, device="cuda", generator=g) * size


class _State:
    """What a program holds on to; gives its device memory back when dropped."""

    cache = None

    def __del__(self):
        if self.cache is not None:
            self.cache.free()


_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        import purebee_amd as pb
        _ctx = pb.Context(0)
    return _ctx


def _inputs(case, seed):
    """Data of a pass, on the GPU."""
    g = _generator(seed)
    if case["kind"] == "logprobs":
        x = 3 * torch.randn(case["rows"], case["vocab"], device="cuda", generator=g)
        target = torch.randint(0, case["vocab"], (case["rows"],), device="cuda", generator=g, dtype=torch.int32)
        return x, target
    starts, counts = _lengths(case)
    past = starts if case["kind"] == "append" else [a + n for a, n in zip(starts, counts)]
    G, D, n = case["kv_heads"], case["dim"], sum(counts)
    pk, pv = _rows(g, sum(past), G, D, 0.3), _rows(g, sum(past), G, D, 0.2)
    q = _rows(g, n, case["heads"], D, 0.2)
    if case["kind"] == "attention":
        return pk, pv, q
    return pk, pv, q, _rows(g, n, G, D, 0.3), _rows(g, n, G, D, 0.2)


def _fill(case, starts, lengths, pk, pv):
    """A cache that holds lengths[i] positions of sequence i."""
    import purebee_amd as pb
    cache = pb.KvCache(_context(), n_layers=1, n_heads=case["heads"], n_kv_heads=case["kv_heads"],
                       head_dim=case["dim"], page_tokens=case["page"],
                       n_pages=sum(-(-(a + case["rows_hi"]) // case["page"]) for a in starts),
                       max_seqs=case["seqs"], max_seq=max(starts) + case["rows_hi"],
                       rope=case["rope"], rope_dim=case["rope_dim"], rope_theta=THETA)
    torch.cuda.synchronize()  # the context works on a stream of its own
    if sum(lengths):
        fill = cache.batch(range(case["seqs"]), lengths)
        fill.append_dev(0, None, pk.data_ptr(), pv.data_ptr(), None)
        _context().sync()
        fill.free()
    return cache


def prepare(case, seed):
    s = _State()
    s.case = case
    if case["kind"] == "logprobs":
        s.x, s.target = _inputs(case, seed)
        M, k = case["rows"], case["top"]
        s.logp, s.entropy = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        s.ids = torch.empty(M, k, device="cuda", dtype=torch.int32)
        s.top = torch.empty(M, k, device="cuda")
        if own:
            s.ctx = _context()
            s.work = torch.empty(max(1, s.ctx.logprobs_workspace(M, case["vocab"], k)), device="cuda",
                                 dtype=torch.uint8)
        torch.cuda.synchronize()
        return s
    starts, counts = _lengths(case)
    first = [a // BLOCK * BLOCK for a in starts]  # of the blocks that the new rows touch
    touched = [a + n - f for a, n, f in zip(starts, counts, first)]
    if case["kind"] == "append":
        pk, pv, s.q, s.k, s.v = _inputs(case, seed)
        s.q_out = torch.empty_like(s.q)
        s.k_out = torch.empty(sum(touched), case["kv_heads"], case["dim"], device="cuda")
        s.v_out = torch.empty_like(s.k_out)
        past = starts
    else:
        pk, pv, s.q = _inputs(case, seed)
        s.out = torch.empty_like(s.q)
        past = [a + n for a, n in zip(starts, counts)]
    if own:
        s.cache = _fill(case, starts, past, pk, pv)
        if case["kind"] == "append":
            s.batch = s.cache.batch(range(case["seqs"]), counts)
            s.touched = s.cache.batch(range(case["seqs"]), touched, first)
        else:
            s.batch = s.cache.batch(range(case["seqs"]), counts, starts)
        _context().sync()
    else:
        s.seq, s.pos = _packed(starts, counts)
        s.freq = _frequencies(case)
        s.start = torch.tensor(starts, device="cuda")
        s.first = torch.tensor(first, device="cuda")
        s.touched_seq, s.touched_pos = _packed(first, touched)
        s.row = s.pos - s.start[s.seq]
        s.k_codes, s.k_scale, s.v_codes, s.v_scale = _plain_cache(case, past, pk, pv, s.freq)
    torch.cuda.synchronize()
    return s


# ---- the plain form ------------------------------------------------------------

def _rotate(x, pos, freq, case):
    """x: [rows, heads, dim] in 64 bits, rotated by its rows' positions."""
    ang = (pos.double()[:, None] * freq)[:, None]
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


def _plain_cache(case, lengths, pk, pv, freq):
    """Codes [seqs, positions, heads, dim] and scales [seqs, blocks, heads] of a past."""
    seq, pos = _packed([0] * len(lengths), lengths)
    length = max(1, -(-max(lengths) // BLOCK)) * BLOCK
    made = []
    for x, turn in ((pk, True), (pv, False)):
        codes = torch.zeros(case["seqs"], length, case["kv_heads"], case["dim"], device="cuda", dtype=torch.int8)
        scale = torch.zeros(case["seqs"], length // BLOCK, case["kv_heads"], device="cuda")
        for h in range(case["kv_heads"]):  # one head at a time bounds the 64-bit copies
            y = x[:, h:h + 1].double()
            y = _blocks(_padded(_rotate(y, pos, freq, case) if turn else y, seq, pos, case["seqs"], length))
            scale[..., h:h + 1] = _scale_of(y)
            codes[:, :, h:h + 1] = _codes(y, scale[..., h:h + 1]).flatten(1, 2).to(torch.int8)
        made += [codes, scale]
    return made


def _plain_append(s):
    c = s.case
    n = c["seqs"]
    window = -(-int(c["rows_hi"] + BLOCK - 1) // BLOCK) * BLOCK  # positions from s.first on
    at = s.pos - s.first[s.seq]
    held = (s.start - s.first)[:, None] > torch.arange(BLOCK, device="cuda")  # older rows of a first block
    out = [_rotate(s.q.double(), s.pos, s.freq, c).float()]
    for new, codes, scale, turn in ((s.k, s.k_codes, s.k_scale, True), (s.v, s.v_codes, s.v_scale, False)):
        y = new.double()
        y = _blocks(_padded(_rotate(y, s.pos, s.freq, c) if turn else y, s.seq, at, n, window))
        scl = _scale_of(y)
        block = (s.first // BLOCK).clamp(max=scale.shape[1] - 1)
        each = torch.arange(n, device="cuda")
        old = torch.where(held.any(1)[:, None], scale[each, block], torch.zeros_like(scl[:, 0]))
        scl[:, 0] = torch.maximum(scl[:, 0], old)
        got = _codes(y, scl)
        past = codes.unflatten(1, (-1, BLOCK))[each, block].double()  # [n, BLOCK, heads, dim]
        past = _codes((past * old.double()[:, None, :, None])[:, None], scl[:, :1])[:, 0]
        got[:, 0] = torch.where(held[:, :, None, None], past, got[:, 0])
        value = (got.float() * scl[:, :, None, :, None]).flatten(1, 2)
        out.append(value[s.touched_seq, s.touched_pos - s.first[s.touched_seq]])
    return {"q": out[0], "k": out[1], "v": out[2]}


def _plain_attention(s):
    c = s.case
    n, H, G, D, R = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["rows_hi"]
    length = s.k_codes.shape[1]
    k, v = ((codes.unflatten(1, (-1, BLOCK)).float() * scale[:, :, None, :, None]).flatten(1, 2)
            for codes, scale in ((s.k_codes, s.k_scale), (s.v_codes, s.v_scale)))
    q = _padded(s.q, s.seq, s.row, n, R).view(n, R, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(n, G, H // G * R, D)
    p = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * (1 / math.sqrt(D))
    hidden = (torch.arange(length, device="cuda")
              > (s.start[:, None] + torch.arange(R, device="cuda"))[:, :, None])  # [n, R, length]
    p = p.view(n, G, H // G, R, length)
    p.masked_fill_(hidden[:, None, None], -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, G, H // G * R, length), v.permute(0, 2, 1, 3).contiguous())
    o = o.view(n, G, H // G, R, D).permute(0, 3, 1, 2, 4).reshape(n, R, H, D)
    return o[s.seq, s.row]


def _plain_logprobs(s):
    m = s.x.amax(-1, keepdim=True)
    d = s.x - m
    e = d.exp()
    total = e.sum(-1)
    lse = m[:, 0] + total.log()
    entropy = total.log() - (e * d).sum(-1) / total
    logp = s.x.gather(1, s.target.long()[:, None])[:, 0] - lse
    # unique keys: the value's bits in order, then the lowest index
    bits = (s.x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -2147483648 - bits, bits)
    key = bits * 2 ** 32 + (2 ** 32 - 1 - torch.arange(s.case["vocab"], device="cuda"))
    ids = key.topk(s.case["top"], dim=-1).indices
    return {"logp": logp, "entropy": entropy, "ids": ids.to(torch.int32), "top": s.x.gather(1, ids) - lse[:, None]}


def run(s):
    kind = s.case["kind"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}[kind](s)
    if kind == "append":
        s.batch.append_dev(0, s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.q_out.data_ptr())
        s.touched.read_dev(0, s.k_out.data_ptr(), s.v_out.data_ptr())
        return {"q": s.q_out, "k": s.k_out, "v": s.v_out}
    if kind == "attention":
        s.batch.attention_dev(0, s.q.data_ptr(), s.out.data_ptr())
        return s.out
    s.ctx.logprobs_dev(s.x.data_ptr(), s.case["rows"], s.case["vocab"], s.target.data_ptr(), s.case["top"],
                       s.logp.data_ptr(), s.entropy.data_ptr(), s.ids.data_ptr(), s.top.data_ptr(),
                       s.work.data_ptr(), s.work.numel())
    return {"logp": s.logp, "entropy": s.entropy, "ids": s.ids, "top": s.top}


def work(case):
    if case["kind"] == "logprobs":
        M, V, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4 * M * V + 4 * M + 8 * M + 8 * M * k, "flops": 6 * M * V}
    starts, counts = _lengths(case)
    H, G, D, n = case["heads"], case["kv_heads"], case["dim"], sum(counts)
    if case["kind"] == "append":
        touched = sum(a % BLOCK + r for a, r in zip(starts, counts))
        # q in and out, k and v in, their codes written, the touched blocks' codes read and their values written
        return {"bytes": 8 * n * H * D + 2 * G * D * (4 * n + n + 5 * touched), "flops": 6 * n * (H + G) * D}
    held = sum(a + r for a, r in zip(starts, counts))
    blocks = sum(-(-(a + r) // BLOCK) for a, r in zip(starts, counts))
    pairs = sum(r * a + r * (r + 1) // 2 for a, r in zip(starts, counts))  # (row, visible position)
    return {"bytes": 2 * G * (held * D + 4 * blocks) + 8 * n * H * D, "flops": 4 * H * D * pairs}


# ---- in 64 bits ----------------------------------------------------------------

def _turn(x, at, case):
    """Rows at positions at..at + n, as complex numbers times e^(i angle)."""
    r = case["rope_dim"]
    half = r // 2
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    ang = torch.outer(torch.arange(at, at + len(x), device="cuda", dtype=torch.float64),
                      torch.exp(i * (-2 * math.log(THETA) / r)))
    y = x.double().clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if case["rope"] == "pairs" else (slice(0, half), slice(half, r))
    z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.ones_like(ang), ang)[:, None]
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _held(x, pieces):
    """Values of a sequence's cache rows x (64 bits) that were appended in `pieces` (their ends), whole blocks
    of it at a time: what the codes and scales stand for."""
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


def exact(case, seed):
    if case["kind"] == "logprobs":
        x, target = _inputs(case, seed)
        got = {"logp": [], "entropy": [], "top": []}
        for row, t in zip(x, target):
            lp = torch.log_softmax(row.double(), 0)
            got["logp"].append(lp[t])
            got["entropy"].append(-(lp.exp() * lp).sum())
            got["top"].append(lp.topk(case["top"]).values)
        return {"logp": torch.stack(got["logp"]), "entropy": torch.stack(got["entropy"]), "ids": None,
                "top": torch.stack(got["top"])}
    starts, counts = _lengths(case)
    G, group, D = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        pk, pv, q, k, v = _inputs(case, seed)
        got, past, row = {"q": [], "k": [], "v": []}, 0, 0
        for a, n in zip(starts, counts):
            f, tail = a // BLOCK * BLOCK, a % BLOCK
            got["q"].append(_turn(q[row:row + n], a, case))
            old = _turn(pk[past + f:past + a], f, case), pv[past + f:past + a].double()
            new = _turn(k[row:row + n], a, case), v[row:row + n].double()
            for name, x, y in (("k", old[0], new[0]), ("v", old[1], new[1])):
                got[name].append(_held(torch.cat([x, y]), [tail, tail + n]))
            past, row = past + a, row + n
        return {name: torch.cat(x) for name, x in got.items()}
    pk, pv, q = _inputs(case, seed)
    out, past, row = [], 0, 0
    for a, n in zip(starts, counts):
        e = a + n
        heads = []
        for g in range(G):
            k = _held(_turn(pk[past:past + e, g:g + 1], 0, case), [e])[:, 0]
            v = _held(pv[past:past + e, g:g + 1].double(), [e])[:, 0]
            for h in range(g * group, (g + 1) * group):
                p = q[row:row + n, h].double() @ k.T / math.sqrt(D)
                p = p.masked_fill(torch.ones(n, e, device="cuda", dtype=torch.bool).triu(a + 1), -math.inf)
                heads.append(p.softmax(-1) @ v)
        out.append(torch.stack(heads, 1))
        past, row = past + e, row + n
    return torch.cat(out)
