"""The paged 8-bit KV cache in plain 64-bit numpy: what append, attention and
read back have to give (the definition in include/pbx.h), and device rows."""
import numpy as np

BLOCK = 32


def rotate(x, pos, style, rope_dim, theta, scale=1.0, factors=None):
    """x [rows, heads, dim] turned by its rows' positions, in 64 bits."""
    x = np.asarray(x, np.float64).copy()
    if style == "none":
        return x
    half = rope_dim // 2
    ang = np.outer(np.asarray(pos, np.float64) / scale, theta ** (-2.0 * np.arange(half) / rope_dim))
    if factors is not None:
        ang = ang / np.asarray(factors, np.float32).astype(np.float64)  # f32, as the cache takes them
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = (slice(0, rope_dim, 2), slice(1, rope_dim, 2)) if style == "pairs" else \
        (slice(0, half), slice(half, rope_dim))
    u, v = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = u * c - v * s, u * s + v * c
    return x


def within(got, want, tol):
    """Every finite value of want is met to its tolerance."""
    ok = np.isfinite(want)
    over = np.abs(got[ok] - want[ok]) - np.broadcast_to(tol, want.shape)[ok]
    worst = float(over.max()) if over.size else 0.0
    assert worst <= 0, f"{int((over > 0).sum())} of {over.size} values off by up to {worst:.3g} more than allowed"


class Store:
    """Codes and scales of one sequence's keys or values, head by head."""

    def __init__(self, heads, dim):
        self.codes = np.zeros((0, heads, dim))
        self.scales = np.zeros((0, heads), np.float32)

    def truncate(self, n):
        self.codes = self.codes[:n]
        self.scales = self.scales[:-(-n // BLOCK)]

    def append(self, x):
        """x [rows, heads, dim] in 64 bits, after the positions held."""
        n = len(self.codes)
        codes = np.concatenate([self.codes, np.zeros_like(x)])
        blocks = -(-len(codes) // BLOCK)
        scales = np.concatenate([self.scales, np.zeros((blocks - len(self.scales), x.shape[1]), np.float32)])
        with np.errstate(all="ignore"):
            for b in range(n // BLOCK, blocks):
                lo, hi = max(n, b * BLOCK), min(len(codes), (b + 1) * BLOCK)
                new = x[lo - n:hi - n]
                old = codes[b * BLOCK:lo]
                for h in range(x.shape[1]):
                    asked = np.float32(np.abs(new[:, h]).max() / 127) if hi > lo else np.float32(0)
                    asked = np.float32(0) if asked < np.float32(2.0 ** -120) else asked
                    had = scales[b, h] if len(old) else np.float32(0)
                    s = np.maximum(had, asked)  # NaN where either is
                    quotient = (lambda y: np.rint(y / np.float64(s))) if 0 < s < np.inf else np.zeros_like
                    codes[lo:hi, h] = quotient(new[:, h])
                    if len(old) and not s == had:
                        codes[b * BLOCK:lo, h] = quotient(old[:, h] * np.float64(had))
                    scales[b, h] = s
        self.codes, self.scales = codes, scales

    def values(self):
        """f32, as the cache's codes and scales stand for."""
        s = np.repeat(self.scales, BLOCK, axis=0)[:len(self.codes), :, None]
        with np.errstate(all="ignore"):
            return (self.codes.astype(np.float32) * s).astype(np.float32)


class RefCache:
    def __init__(self, seqs, heads, kv_heads, dim, style="pairs", rope_dim=0, theta=10000.0, scale=1.0,
                 factors=None):
        self.rope = (style, rope_dim or dim, theta, scale, factors)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.k = [Store(kv_heads, dim) for _ in range(seqs)]
        self.v = [Store(kv_heads, dim) for _ in range(seqs)]

    def length(self, s):
        return len(self.k[s].codes)

    def truncate(self, s, n):
        self.k[s].truncate(n)
        self.v[s].truncate(n)

    def append(self, seqs, counts, q, k, v):
        """Rotated queries in 64 bits."""
        out, r = [], 0
        for s, n in zip(seqs, counts):
            pos = self.length(s) + np.arange(n)
            out.append(rotate(q[r:r + n], pos, *self.rope))
            self.k[s].append(rotate(k[r:r + n], pos, *self.rope))
            self.v[s].append(np.asarray(v[r:r + n], np.float64))
            r += n
        return np.concatenate(out) if out else np.zeros((0, self.heads, self.dim))

    def values(self, seqs, starts, counts):
        pick = lambda x: np.concatenate([x[s].values()[a:a + n] for s, a, n in zip(seqs, starts, counts)])  # noqa: E731
        return pick(self.k), pick(self.v)

    def attention(self, seqs, starts, counts, q, scale=None):
        """(rows in 64 bits, a bound on a kernel's error in each of their values).

        The bound, for a kernel that takes queries and probabilities as pairs of
        fp16 (an error of 2^-22 relative each, 2^-25 of the row's largest query at
        least) and everything else in f32 (2^-24 a rounding): a score s = sum q k
        over dim products, each with 2^-22 + 2^-25 peak / |q| and the sum's
        (dim + 4) roundings of 2^-24 relative to sum |q k|, then two factors'
        roundings and that of the difference from the maximum, 2^-24 |s| each and
        2^-23 of exp2, is off by at most `off`; a probability by e^off - 1
        relative, and so is their sum; sums over the keys run over at most
        keys / 32 + 40 f32 roundings; the two are counted twice for the quotient.
        """
        q = np.asarray(q, np.float64)
        out, tol, r = np.zeros_like(q), np.zeros_like(q), 0
        group = self.heads // self.kv_heads
        f = 1 / np.sqrt(self.dim) if scale is None else scale
        with np.errstate(all="ignore"):
            for s, a, n in zip(seqs, starts, counts):
                k, v = self.k[s].values().astype(np.float64), self.v[s].values().astype(np.float64)
                for t in range(n):
                    e = a + t + 1
                    for h in range(self.heads):
                        kk, vv, qq = k[:e, h // group], v[:e, h // group], q[r + t, h]
                        x = kk @ qq * f
                        p = np.exp(x - x.max())
                        p /= p.sum()
                        out[r + t, h] = p @ vv
                        mass = np.abs(kk) @ np.abs(qq)
                        floor = np.abs(kk).sum(1) * np.abs(qq).max() * 2.0 ** -25
                        off = abs(f) * (mass * (2.0 ** -22 + (self.dim + 4) * 2.0 ** -24) + floor) \
                            + 2.0 ** -22 * (np.abs(x) + np.abs(x.max()) + 4)
                        each = np.expm1(off) + 2.0 ** -22
                        chain = (e / 32 + 40) * 2.0 ** -24
                        tol[r + t, h] = (p * (each + chain)) @ np.abs(vv) + (p @ (each + chain)) * np.abs(out[r + t, h])
                r += n
        return out, tol + 2.0 ** -23 * np.abs(out) + 1e-37


class Rows:
    """f32 rows on the device inside a larger buffer: `stride` floats apart, with
    `lead` and `tail` floats of a pattern around them that nothing may touch."""

    def __init__(self, ctx, n, width, data=None, stride=None, lead=64, tail=64):
        self.n, self.width, self.stride, self.lead = n, width, stride or width, lead
        total = lead + max(0, n - 1) * self.stride + (width if n else 0) + tail
        self.host = np.full(total, 12345.25, np.float32)
        if data is not None:
            self._view(self.host)[:] = np.asarray(data, np.float32).reshape(n, width)
        self.buf = ctx.alloc(total * 4).upload(self.host)
        self.ptr = self.buf.ptr + 4 * lead

    def _view(self, a):
        return np.lib.stride_tricks.as_strided(a[self.lead:], (self.n, self.width), (4 * self.stride, 4))

    def get(self):
        """The rows; whatever lies around them has to be as it was."""
        got = self.buf.download(np.float32, len(self.host))
        rows = self._view(got).copy()
        around = got.copy()
        self._view(around)[:] = self._view(self.host)
        assert np.array_equal(around.view(np.uint32), self.host.view(np.uint32)), "something outside the rows was written"
        return rows

    def free(self):
        self.buf.free()
