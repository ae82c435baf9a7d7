"""Log probabilities of rows against a head's weights, and the rows' gradient, in plain
64-bit numpy, each with a bound on what a kernel that works as include/pbx.h says may be off.

Logits: activations enter with 22 bits, as fp16 pairs (2^-22 of each) or as fixed point
(2^-22 of the row's largest); products are summed in f32, 32 wide and then over the K / 32
blocks, a rounding of 2^-24 each, and a few more to put partial sums together.
"""
import numpy as np

import purebee_amd as pb
from purebee_amd import native

QUANT = {native.TYPE_Q4_0: pb.quantize_q4_0, native.TYPE_Q4_1: pb.quantize_q4_1, native.TYPE_Q8_0: pb.quantize_q8_0,
         native.TYPE_Q6_K: pb.quantize_q6_k, native.TYPE_F16: pb.to_f16_bytes,
         native.TYPE_F32: lambda w: np.ascontiguousarray(w, np.float32)}
TYPES = {"q4_0": native.TYPE_Q4_0, "q4_1": native.TYPE_Q4_1, "q8_0": native.TYPE_Q8_0, "q6_k": native.TYPE_Q6_K,
         "f16": native.TYPE_F16, "f32": native.TYPE_F32}
U = 2.0 ** -24


class Head:
    """A resident head and its values in 64 bits."""

    def __init__(self, ctx, kind, w):
        self.ctx, self.N, self.K = ctx, *w.shape
        t = TYPES[kind]
        self.w = ctx.upload(t, self.N, self.K, QUANT[t](np.ascontiguousarray(w, np.float32)))
        self.values = ctx.dequant(self.w).astype(np.float64)

    def free(self):
        self.w.free()


def forward(W, x, target):
    """({logp, entropy, lse}, a bound for each) of rows x against the values W."""
    x = np.asarray(x, np.float64)
    K = x.shape[1]
    with np.errstate(all="ignore"):
        z = x @ W.T
        mass = np.abs(x) @ np.abs(W).T
        peak = np.abs(x).max(1, keepdims=True) * np.abs(W).sum(1)
        off = 2.0 ** -22 * (mass + peak) + (K / 32 + 64) * U * mass  # of a logit
        m = z.max(1, keepdims=True)
        d = z - m
        e = np.exp(d)
        s = e.sum(1, keepdims=True)
        p = e / s
        lse = (m + np.log(s))[:, 0]
        lp = d - np.log(s)
        entropy = -(p * np.where(p > 0, lp, 0)).sum(1)
        # an exponential: its argument's roundings (the difference and the product with log2 e) and its own
        each = off + (np.abs(d) + 4) * 4 * U
        joined = 96 * U  # roundings of a sum of exponentials, each relative to it
        tol_lse = (p * each).sum(1) + joined + 4 * U * (np.abs(lse) + np.abs(m[:, 0]))
        tol_h = (p * np.abs(np.where(p > 0, lp, 0) + entropy[:, None]) * each).sum(1) \
            + joined * (1 + (p * np.abs(d)).sum(1)) + 8 * U * (np.abs(entropy) + np.log(s)[:, 0])
        t = np.asarray(target, np.int64)
        ok = (t >= 0) & (t < len(W))
        at = np.where(ok, t, 0)
        r = np.arange(len(x))
        logp = np.where(ok, lp[r, at], np.nan)
        tol_logp = off[r, at] + tol_lse + 4 * U * (np.abs(z[r, at]) + np.abs(logp))
    return ({"logp": logp, "entropy": entropy, "lse": lse}, {"logp": tol_logp, "entropy": tol_h, "lse": tol_lse},
            {"z": z, "off": off, "tol_lse": tol_lse, "lse": lse})


def gradient(W, x, target, grad, largest=None):
    """(rows' gradient, a bound for each value).  Probabilities: e^(l - lse) with the logit's and lse's errors, the
    difference's rounding and the exponential's; then probabilities and weights as pairs (2^-22 each, and their low
    halves' product is left out: 2^-22; weights 2^-26 of the largest at least), summed in f32 over the vocabulary."""
    x, grad = np.asarray(x, np.float64), np.asarray(grad, np.float64)
    _, _, more = forward(W, x, np.zeros(len(x), int))
    z, off, lse = more["z"], more["off"], more["lse"]
    with np.errstate(all="ignore"):
        d = z - lse[:, None]
        p = np.exp(d)
        t = np.asarray(target, np.int64)
        ok = (t >= 0) & (t < len(W))
        G = -p
        r = np.arange(len(x))
        G[r, np.where(ok, t, 0)] += 1
        each = off + (more["tol_lse"] + 4 * U * np.abs(lse))[:, None] + (np.abs(d) + 8) * 2 * U
        chain = (len(W) / 16 + 128) * U
        largest = np.abs(W).max() if largest is None else largest
        floor = 2.0 ** -26 * largest
        dx = G @ W
        aw = np.abs(W)
        tol = (p * each) @ aw + (np.abs(G) * (3 * 2.0 ** -22 + chain)) @ aw + np.abs(G).sum(1, keepdims=True) * floor \
            + 2.0 ** -40 * aw.sum(0)
        dx, tol = dx * grad[:, None], tol * np.abs(grad)[:, None] + 4 * U * np.abs(dx * grad[:, None])
    return np.where(ok[:, None], dx, 0.0), np.where(ok[:, None], tol, 0.0)
