"""The calls for drafted tokens and scoring as callers make them: arrays of other
integer types, one token at a time."""
import numpy as np
import pytest

import tree_reference as ref
from cheetah_amd import configs, synth

pytestmark = pytest.mark.gpu

SHAPES = [configs.TINY_QWEN2, configs.TINY_LLAMA]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


@pytest.mark.parametrize("call", ["tree", "chunk"])
@pytest.mark.parametrize("dtype", [np.int64, np.uint8, np.int16])
def test_page_tables_of_other_types(hip, dtype, call):
    """numpy's default integers (read as they lie, pairs of words) and narrow ones."""
    rng = np.random.default_rng(3)
    k, v = ref.make_cache(rng, 200, 2, 64, "bf16")
    kp, vp, table = ref.paged(k, v, "bf16", rng)
    q = rng.standard_normal((8, 8 * 64)).astype(np.float32)
    parents = ref.parents_of("random", 8, rng)

    def run(t):
        if call == "tree":
            return hip.tree_attention(q, kp, vp, t, 8, parents, 192)
        return hip.attention(q, kp, vp, t, 8, 8, 192)

    assert np.array_equal(run(table.astype(dtype)).view(np.uint32), run(table).view(np.uint32))


@pytest.mark.parametrize("quant", [None, "q8"])
@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: s.name)
def test_a_token_scored_alone_is_forwards_decode_step(hip, shape, kv, quant):
    """Tokens scored one at a time, and a last one behind a chunk: the K/V rows of
    forward bit for bit, and the scores of forward's own logits (f32 sums of up
    to 16 terms a thread, 2^-22 + 17 * 2^-24 of them, and a rounding of results
    below 32)."""
    w = synth.make_weights(shape)
    g, plain = (hip.HipForward(shape, w, quant=quant, kv_capacity=256, max_chunk_rows=64, kv=kv) for _ in "gp")
    text = synth.make_tokens(shape.vocab_size, 45, seed=61)
    for m in (g, plain):
        m.forward(text[:40], 0)
    for i in range(40, 44):
        lp, ent, ids, tops = g.forward_logprobs(text[i:i + 1], i, targets=text[i + 1:i + 2], top=5)
        x = plain.forward(text[i:i + 1], i).astype(np.float64)
        lse = x.max() + np.log(np.exp(x - x.max()).sum())
        order = np.argsort(-x, kind="stable")[:5]
        assert np.array_equal(ids[0], order)
        bar = 2.0**-22 + 17 * 2.0**-24 + 2.0**-20
        assert abs(lp[0] - (x[text[i + 1]] - lse)) < bar
        assert (np.abs(tops[0] - (x[order] - lse)) < bar).all()
        p = np.exp(x - lse)
        assert abs(ent[0] + (p * (x - lse)).sum()) < 2 * bar * (1 + ent[0])
    assert g.kv_len() == 44
    for layer in range(shape.num_layers):
        for a, b in zip(g.kv_rows(layer, 0, 44), plain.kv_rows(layer, 0, 44)):
            assert np.array_equal(np.asarray(a, np.float32).view(np.uint32), np.asarray(b, np.float32).view(np.uint32))
    assert np.array_equal(g.forward(text[44:], 44).view(np.uint32), plain.forward(text[44:], 44).view(np.uint32))


@pytest.mark.parametrize("top", [0, 1])
def test_more_rows_than_a_launch_has_threads_for(hip, top):
    """2^24 rows of 256 threads are 2^32."""
    rows = 2**24 + 5
    x = np.random.default_rng(5).standard_normal((rows, 2)).astype(np.float32)
    tokens = (np.arange(rows) % 2).astype(np.uint32)
    lp, ent, ids, tops = hip.logprobs(x, tokens, top)
    d = x[:, 1].astype(np.float64) - x[:, 0]
    # log p of the second of two, and of the first.
    second, first = -np.logaddexp(0, -d), -np.logaddexp(0, d)
    want = np.where(tokens == 1, second, first)
    bar = 2.0**-21 + 2.0**-24 * np.abs(want)  # an exponential, two roundings; the result's own
    assert (np.abs(lp - want) <= bar).all()
    assert (np.abs(ent + np.exp(first) * first + np.exp(second) * second) <= 2.0**-20).all()
    if top:
        assert np.array_equal(ids[:, 0], (d > 0).astype(np.uint32))
        assert (np.abs(tops[:, 0] - np.maximum(first, second)) <= 2.0**-21).all()


def test_a_call_that_finds_no_pages_leaves_the_tree(hip):
    """Refused calls run nothing: the tree that waits is still there to commit, as
    if they had not been made."""
    shape = configs.TINY_LLAMA
    w = synth.make_weights(shape)
    g = hip.HipForward(shape, w, kv_capacity=256, max_chunk_rows=64)
    other = g.clone()
    text = synth.make_tokens(shape.vocab_size, 128, seed=36)
    other.forward(text, 0)  # half of the pages
    g.forward(text[:120], 0)
    parents = [-1, 0, 0, 1, 1, 3, 2, 6]
    drafts = synth.make_tokens(shape.vocab_size, 8, seed=37)
    g.forward_tree(drafts, parents, 120)
    for call in (lambda: g.forward(text[:20], 120), lambda: g.forward_greedy(text[:20], 120),
                 lambda: g.decode_greedy(1, 120, 20), lambda: g.time_decode(1, 120, 20),
                 lambda: g.forward_tree([1] * 20, [-1] * 20, 120), lambda: g.verify_tree([1] * 20, [-1] + [0] * 19, 120),
                 lambda: g.forward_logprobs(text[:20], 120)):
        with pytest.raises(hip.HipError, match="pool exhausted"):
            call()
    g.commit_tree([0, 2, 6])
    assert g.kv_len() == 123
    plain = hip.HipForward(shape, w, kv_capacity=256, max_chunk_rows=64)
    plain.forward(text[:120], 0)
    plain.forward_tree(drafts, parents, 120)
    plain.commit_tree([0, 2, 6])
    assert np.array_equal(g.forward([5], 123).view(np.uint32), plain.forward([5], 123).view(np.uint32))
