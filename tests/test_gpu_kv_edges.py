"""The paged KV cache at the ends of its numbers, against tests/kv_ref.py."""
import numpy as np
import pytest

from tests.test_gpu_kv import Pair

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
