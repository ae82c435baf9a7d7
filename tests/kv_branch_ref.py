"""Forks and compactions of the paged 8-bit KV cache in plain 64-bit numpy (the
definitions in include/pbx.h), over tests/kv_ref.py."""
import numpy as np

from tests.kv_ref import BLOCK, RefCache, Rows, Store, rotate
from tests.test_gpu_kv import Pair


def copied(store, n):
    out = Store(store.codes.shape[1], store.codes.shape[2])
    out.codes, out.scales = store.codes.copy(), store.scales.copy()
    out.truncate(n)
    return out


def packed(store, kept, turn):
    """The store with the rows `kept`, those that move coded anew; turn(x, by): rows turned by positions."""
    kept = np.asarray(kept, np.int64)
    n, new = len(kept), np.arange(len(kept))
    out = Store(store.codes.shape[1], store.codes.shape[2])
    stay = int((kept == new).sum())
    whole = n if stay == n else stay // BLOCK * BLOCK  # rows of blocks that stay as they are
    out.codes, out.scales = store.codes[:whole].copy(), store.scales[:-(-whole // BLOCK)].copy()
    with np.errstate(all="ignore"):
        x = store.codes[kept] * store.scales[kept // BLOCK].astype(np.float64)[..., None]
        y = turn(x, new - kept)
        for at in range(whole, n, BLOCK):
            out.append(y[at:at + BLOCK])
    return out


class BranchRef(RefCache):
    def fork(self, dsts, srcs, lengths=None):
        lengths = [self.length(s) for s in srcs] if lengths is None else lengths
        for side in (self.k, self.v):
            made = [copied(side[s], n) for s, n in zip(srcs, lengths)]
            for d, x in zip(dsts, made):
                side[d] = x

    def compact(self, seqs, kept):
        for s, at in zip(seqs, kept):
            self.k[s] = packed(self.k[s], at, lambda x, by: rotate(x, by, *self.rope))
            self.v[s] = packed(self.v[s], at, lambda x, by: x)


class BranchPair(Pair):
    """A cache on the GPU and the reference beside it, forked and compacted together."""

    def __init__(self, ctx, heads, kv_heads, dim, seqs=4, style="pairs", rope_dim=0, theta=10000.0, scale=1.0,
                 factors=None, **more):
        super().__init__(ctx, heads, kv_heads, dim, seqs=seqs, style=style, rope_dim=rope_dim, theta=theta,
                         scale=scale, factors=factors, **more)
        self.ref = BranchRef(seqs, heads, kv_heads, dim, style, rope_dim, theta, scale, factors)

    def fork(self, dsts, srcs, lengths=None):
        self.cache.fork(dsts, srcs, lengths)
        self.ref.fork(dsts, srcs, lengths)

    def compact(self, seqs, kept):
        self.cache.compact(seqs, kept)
        self.ref.compact(seqs, kept)

    def fill(self, s, n):
        """n rows of keys and values (no queries) to sequence s."""
        q, k, v = self.rows(n)
        b = self.cache.batch([s], [n])
        w = self.kv_heads * self.dim
        dk, dv = Rows(self.ctx, n, w, k), Rows(self.ctx, n, w, v)
        b.append_dev(0, None, dk.ptr, dv.ptr, None)
        self.ctx.sync()
        self.ref.append([s], [n], q, k, v)
        for x in (dk, dv, b):
            x.free()

    def truncate(self, s, n):
        self.cache.truncate(s, n)
        self.ref.truncate(s, n)
