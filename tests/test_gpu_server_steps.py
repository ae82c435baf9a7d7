"""A server's steps over one model and one cache, each step's logits against 64 bits: sequences that begin at different
times, a draft that is rejected, a sequence that ends and whose id and pages another one takes."""
import numpy as np
import pytest

import purebee_amd as pb
from tests.conftest import rel_l2
from tests.test_gpu_model_kv import CONFIGS, TOL, Server

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["f32", "q8_0"])
def test_steps_of_a_server(ctx, name):
    """The tokens are given, not the model's own, so that every row of every step can be compared, whatever the margins are."""
    cfg = CONFIGS[name]
    rng = np.random.default_rng(51)
    s = Server(ctx, cfg, seqs=4, n_pages=7)          # pages of 32: the four cannot all grow, so pages change hands
    b = pb.KvBatch(s.cache)
    said = {}                                        # the tokens that a sequence holds

    def step(seqs, counts, all_rows=False):
        starts = [s.cache.length(i) for i in seqs]
        tokens = rng.integers(0, cfg["vocab_size"], sum(counts)).astype(np.int32)
        logits, nxt = s.model.forward_kv(b.set(seqs, counts), tokens, all_rows=all_rows)
        want = s.expect(seqs, starts, counts, tokens)
        last = np.cumsum(counts) - 1
        rows = range(len(want)) if all_rows else [e for e, n in zip(last, counts) if n]
        assert len(logits) == len(rows)
        for got, r in zip(logits, rows):
            assert rel_l2(got, want[r]) <= TOL, (seqs, counts, r)
        assert np.array_equal(nxt, logits.argmax(-1))
        for i, a, n, e in zip(seqs, starts, counts, last):
            assert s.cache.length(i) == a + n == len(said.setdefault(i, [])) + n
            said[i] += list(tokens[e + 1 - n:e + 1])

    def cut(seq, n):
        s.cache.truncate(seq, n)
        said[seq] = said[seq][:n]

    step([0, 1], [20, 37])
    for _ in range(3):
        step([1, 0], [1, 1])
    step([2, 0, 1], [9, 1, 1])                       # a third begins beside single tokens
    for n in (2, 3):
        step([1], [5], all_rows=True)                # drafts and their verify: some of the rows go
        cut(1, len(said[1]) - n)
        step([0, 1, 2], [1, 1, 1])
    step([1], [25], all_rows=True)                   # a draft over a block's and a page's end, gone up to the block before
    assert len(said[1]) > 64
    cut(1, 60)
    step([2, 1], [1, 5])
    free = s.cache.info()["free_pages"]
    cut(1, 0)                                        # it ends: three pages back
    assert s.cache.info()["free_pages"] == free + 3
    step([3, 0, 2], [70, 1, 1])                      # another takes them: pages that held other keys and values
    step([1, 3], [64, 1])                            # and another the id: every page is taken now
    assert s.cache.info()["free_pages"] == 0
    before = {i: s.cache.length(i) for i in range(4)}
    with pytest.raises(pb.PbxError) as e:
        b.set([0, 2, 1], [1, 1, 1])                  # no page for sequence 1's next block
    assert e.value.code == -3 and before == {i: s.cache.length(i) for i in range(4)}
    for _ in range(2):
        step([0, 3, 2], [1, 1, 1])
    cut(3, 31)
    for order in ([1, 0, 2, 3], [3, 2, 1, 0]):
        step(order, [1, 1, 1, 1], all_rows=True)
    s.free()
