"""Trees of drafted tokens through a model over thousands of cached positions,
where the tree attention is split over the keys and joined, and over values that it
computes again key by key.

A node's logits against the same tokens run alone behind the same cached rows (a
clone restored from a snapshot), as a chunk: the same products but the attention's,
whose two kernels' f32 results differ by rounding, and the K/V rows of the nodes
behind their first layer, which a BF16 cache rounds a whole step (2^-7) when they
are near a boundary. 3,000 positions average a few such elements out: 1e-3, the
chunked forward's bar; one token alone is a decode step, f32 inputs for 16 bits,
within it too."""
import numpy as np
import pytest

from cheetah_amd import configs, synth

pytestmark = pytest.mark.gpu

BAR = 1e-3
FIVE = [-1, 0, 0, 2, 1]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def rel_err(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return float(np.max(np.abs(got - want)) / np.max(np.abs(want)))


def random_parents(n, seed):
    p = np.maximum(np.arange(n) - np.random.default_rng(seed).integers(1, 9, n), 0)
    p[0] = -1
    return p.tolist()


def path(parents, node):
    out = []
    while node >= 0:
        out.append(node)
        node = parents[node]
    return out[::-1]


@pytest.mark.parametrize("prefix", [3000, 900])
@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [configs.TINY_QWEN2, configs.TINY_LLAMA], ids=lambda s: s.name)
def test_trees_over_a_long_cache(hip, shape, kv, prefix):
    """5, 64, 200, then 5 nodes again on one instance: the partials' buffer grows
    and is used again by fewer (24 and 47 splits of 3,000 positions, joined by four
    waves a row; 8 and 15 of 900, by one). A branch is kept between them."""
    g = hip.HipForward(shape, synth.make_weights(shape), kv_capacity=4096, max_chunk_rows=256, kv=kv)
    alone = g.clone()
    g.forward(synth.make_tokens(shape.vocab_size, prefix, seed=71), 0, chunk_rows=256)
    first = None
    for turn, parents in enumerate([FIVE, random_parents(64, 1), random_parents(200, 2), FIVE]):
        n, at = len(parents), g.kv_len()
        drafts = synth.make_tokens(shape.vocab_size, n, seed=72 + turn)
        snap = g.kv_snapshot()
        nxt, logits = g.forward_tree(drafts, parents, at, want_logits=True)
        assert np.array_equal(g.forward_tree(drafts, parents, at), nxt)
        for i in sorted({0, 1, n // 2, n - 2, n - 1}):
            alone.restore_kv_prefix(snap, at)
            assert rel_err(logits[i], alone.forward(drafts[path(parents, i)], at)) < BAR, (turn, i)
        if turn == 0:
            first = (drafts, snap, logits)
        branch = path(parents, n - 1)
        g.commit_tree(branch)
        assert g.kv_len() == at + len(branch)
        alone.restore_kv_prefix(snap, at)
        alone.forward(drafts[branch], at)
        assert rel_err(g.forward([9], at + len(branch)), alone.forward([9], at + len(branch))) < BAR
    # The first tree again, in buffers that larger ones have used: the same bits.
    drafts, snap, logits = first
    g.restore_kv_prefix(snap, prefix)
    again = g.forward_tree(drafts, FIVE, prefix, want_logits=True)[1]
    assert np.array_equal(again.view(np.uint32), logits.view(np.uint32))


@pytest.mark.parametrize("size", [2.0**123, 2.0**126])
@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_rows_computed_again_give_their_halves(hip, kv, size):
    """Some dims of every V row hold `size` (the projection's bias) and are read by
    no later weight: sums overflow on the matrix cores, averages do not, and the
    output projection's input halves are those of rows computed key by key. The
    logits are those of the same model without that bias, whose other dims were summed
    in another order: input halves near a boundary round otherwise, by 2^-17 of
    them, in six products (1e-4 is twice that), and so do K/V elements of a BF16
    cache (2^-7 of the only position that a root sees)."""
    shape = configs.TINY_QWEN2
    hd = shape.head_dim
    w = dict(synth.make_weights(shape))
    dims = np.arange(0, shape.kv_dim, 7)
    columns = np.concatenate([h * hd + dims[dims // hd == h // (shape.q_heads // shape.kv_heads)] % hd
                              for h in range(shape.q_heads)])
    for layer in range(shape.num_layers):
        p = f"model.layers.{layer}.self_attn."
        o = np.array(w[p + "o_proj.weight"])
        o.reshape(shape.hidden_size, shape.q_dim)[:, columns] = 0
        w[p + "o_proj.weight"] = o
    loud = dict(w)
    for layer in range(shape.num_layers):
        name = f"model.layers.{layer}.self_attn.v_proj.bias"
        bias = np.array(loud[name])
        bias.reshape(-1)[dims] = synth.f32_to_bf16(np.full(dims.size, size, np.float32)).reshape(-1)
        loud[name] = bias
    parents = random_parents(40, 5)
    drafts = synth.make_tokens(shape.vocab_size, 40, seed=80)
    got, want = (hip.HipForward(shape, x, kv_capacity=256, max_chunk_rows=64, kv=kv)
                 .forward_tree(drafts, parents, 0, want_logits=True)[1] for x in (loud, w))
    assert np.isfinite(got).all()
    assert rel_err(got, want) < (1e-4 if kv == "f32" else 2.0**-7)
