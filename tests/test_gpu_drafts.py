"""A model's calls for drafted tokens (forward_tree, commit_tree, verify_tree)
and for scoring (forward_logprobs) against the CPU oracle and against its other
forwards.

Logits are held to the oracle with the device's K/V precision. f32 cache: 1e-3,
the bar of the chunked forward (the same products, inputs of 16 bits in two BF16
halves). BF16 cache: a K/V element that lies within the kernels' error of a
rounding boundary rounds the other way, and is then a whole step, up to 2^-7 of
it, from the oracle's. A long context averages that out; a node that attends to
one position (an empty cache) does not, its attention is that V row: 2^-7. (Of 13
tokens at position 0 the decode forward reaches 1.0e-3 that way and the tree
1.4e-3; with an f32 cache 4e-7 and 8e-6.) A log
probability is x - log(sum exp x): both terms move by at most the logits' error,
so it is held to twice that error and 1e-5 for its own f32 result (a half step of
values below 32 is 2^-20). An entropy, sum p (log Z - x), moves by at most
sum |dp| (log V) + sum p |dx| <= e (2 log V + 2) for errors e of the logits.
"""
import threading

import numpy as np
import pytest

from cheetah_amd import configs, synth

pytestmark = pytest.mark.gpu

TINY = [configs.TINY_QWEN2, configs.TINY_LLAMA]
BARS = {"bf16": 2.0 ** -7, "f32": 1e-3}
# (prefix, parents): the cached text's length and a tree: two roots, forks, a
# chain, a node far from its parent.
FORK = [-1, -1, 0, 0, 1, 2, 2, 3, 5, 8, 9, 4, 6]
TREES = [(45, FORK), (60, FORK), (0, FORK), (64, [-1]), (63, [-1, 0]), (1, [-1] * 9), (129, list(range(-1, 24)))]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def rel_err(got, ref):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    return float(np.max(np.abs(got - ref)) / max(np.max(np.abs(ref)), 1e-30))


def bits(a):
    return np.asarray(a, np.float32).view(np.uint32)


_WEIGHTS = {}


def weights(shape):
    if shape.name not in _WEIGHTS:
        _WEIGHTS[shape.name] = synth.make_weights(shape)
    return _WEIGHTS[shape.name]


def model(hip, shape, quant=None, kv="bf16", capacity=512, chunk=64):
    return hip.HipForward(shape, weights(shape), quant=quant, kv_capacity=capacity, max_chunk_rows=chunk, kv=kv)


def path(parents, node):
    out = []
    while node >= 0:
        out.append(node)
        node = parents[node]
    return out[::-1]


def greedy(logits):
    return int(len(logits) - 1 - np.argmax(logits[::-1]))


@pytest.mark.parametrize("prefix,parents", TREES, ids=lambda t: str(len(t)) if isinstance(t, list) else str(t))
@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("shape", TINY, ids=lambda s: s.name)
def test_tree_matches_each_branch_alone(hip, oracle, shape, kv, prefix, parents):
    g, r = model(hip, shape, kv=kv), oracle.RefModel(shape, weights(shape), kv_bf16=(kv == "bf16"))
    text = synth.make_tokens(shape.vocab_size, max(prefix, 1), seed=21)[:prefix]
    drafts = synth.make_tokens(shape.vocab_size, len(parents), seed=22)
    if prefix:
        g.forward(text, 0)
        r.forward(text, 0)
    snap = r.kv_snapshot()
    nxt, logits = g.forward_tree(drafts, parents, prefix, want_logits=True)
    assert g.kv_len() == prefix
    assert np.array_equal(g.forward_tree(drafts, parents, prefix), nxt)
    for i in range(len(parents)):
        r.clear_cache()
        if prefix:
            r.restore_kv_prefix(snap, prefix)
        want = r.forward(drafts[path(parents, i)], prefix)
        assert rel_err(logits[i], want) < BARS[kv], i
        assert int(nxt[i]) == greedy(logits[i]), i


@pytest.mark.parametrize("quant", ["q8", "q4"])
@pytest.mark.parametrize("shape", TINY, ids=lambda s: s.name)
def test_tree_of_quantized_weights(hip, oracle, shape, quant):
    g, r = model(hip, shape, quant=quant), oracle.RefModel(shape, weights(shape), quant=quant, kv_bf16=True)
    text = synth.make_tokens(shape.vocab_size, 30, seed=23)
    drafts = synth.make_tokens(shape.vocab_size, len(FORK), seed=24)
    g.forward(text, 0)
    r.forward(text, 0)
    snap = r.kv_snapshot()
    _, logits = g.forward_tree(drafts, FORK, 30, want_logits=True)
    for i in range(len(FORK)):
        r.clear_cache()
        r.restore_kv_prefix(snap, 30)
        assert rel_err(logits[i], r.forward(drafts[path(FORK, i)], 30)) < BARS["bf16"], i


@pytest.mark.parametrize("node", [0, 1, 10, 11, 12])
@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("shape", TINY, ids=lambda s: s.name)
def test_a_committed_branch_is_the_branch_run_alone(hip, oracle, shape, kv, node):
    """The first layer's K/V rows bit for bit (they depend on token and position
    only), the other layers' within the bar, and the next tokens' logits. A branch
    of one token run alone is a decode step, whose products take f32 inputs and
    not 16 bits of them: its row is held to the other layers' bar."""
    g, alone = model(hip, shape, kv=kv), model(hip, shape, kv=kv)
    r = oracle.RefModel(shape, weights(shape), kv_bf16=(kv == "bf16"))
    text = synth.make_tokens(shape.vocab_size, 58, seed=25)
    drafts = synth.make_tokens(shape.vocab_size, len(FORK), seed=26)
    branch = path(FORK, node)
    end = 58 + len(branch)
    g.forward(text, 0)
    g.forward_tree(drafts, FORK, 58)
    g.commit_tree(branch)
    assert g.kv_len() == end
    for m in (alone, r):
        m.forward(text, 0)
        m.forward(drafts[branch], 58)
    exact = end if len(branch) > 1 else 58
    for a, b in zip(g.kv_rows(0, 0, exact), alone.kv_rows(0, 0, exact)):
        assert np.array_equal(bits(a), bits(b))
    step = 2.0 ** -7 if kv == "bf16" else 0.0  # a K/V element may round the other way: a whole step
    for layer in (0, 1):
        for a, b in zip(g.kv_rows(layer, 0, end), alone.kv_rows(layer, 0, end)):
            assert np.array_equal(bits(a[:58]), bits(b[:58]))
            assert rel_err(a, b) < BARS["f32"] + step
    for pos, t in ((end, 5), (end + 1, 7)):
        assert rel_err(g.forward([t], pos), r.forward([t], pos)) < BARS[kv]
    more = synth.make_tokens(shape.vocab_size, 20, seed=27)
    assert rel_err(g.forward(more, end + 2), r.forward(more, end + 2)) < BARS[kv]


@pytest.mark.parametrize("quant,kv", [(None, "bf16"), (None, "f32"), ("q8", "bf16"), ("q4", "bf16")])
@pytest.mark.parametrize("shape", TINY, ids=lambda s: s.name)
def test_verified_drafts_give_the_greedy_tokens(hip, oracle, shape, quant, kv):
    """A drafter that is right for a few tokens, then wrong, with decoys beside
    it. Every token is the oracle's argmax behind the ones before it, within the
    bar. The first shape's best two logits are 0.157 of the largest apart or more
    at every step (CPU oracle), ten times what the bar allows two of them to
    move, so there the tokens are decode_greedy's, and exactly the right drafts
    are accepted."""
    want_of, g = model(hip, shape, quant, kv), model(hip, shape, quant, kv)
    text = synth.make_tokens(shape.vocab_size, 50, seed=28)
    total = 48
    first = want_of.forward_greedy(text, 0)
    want = [first] + want_of.decode_greedy(first, 50, total + 16).tolist()
    got = [g.forward_greedy(text, 0)]
    rng = np.random.default_rng(29)
    runs, clear = [], shape is configs.TINY_QWEN2
    while len(got) <= total:
        at = len(got) - 1
        right, wrong = int(rng.integers(0, 6)), int(rng.integers(0, 3))
        tokens, parents, cur = [got[-1]], [-1], 0
        for k in range(right):
            for _ in range(int(rng.integers(0, 3))):  # decoys of the same parent
                tokens.append((want[at + 1 + k] + 1 + int(rng.integers(0, 50))) % shape.vocab_size)
                parents.append(cur)
            tokens.append(want[at + 1 + k])
            parents.append(cur)
            cur = len(tokens) - 1
        for k in range(wrong):
            tokens.append((want[at + 1 + right + k] + 1) % shape.vocab_size)
            parents.append(cur)
            cur = len(tokens) - 1
        accepted, nxt = g.verify_tree(tokens, parents, 50 + at)
        runs.append(len(accepted))
        assert accepted[0] == 0 and (len(accepted) == right + 1 or not clear)
        assert [parents[i] for i in accepted[1:]] == accepted[:-1].tolist()
        assert nxt not in [t for t, p in zip(tokens, parents) if p == accepted[-1]]
        got += [tokens[i] for i in accepted[1:]] + [nxt]
        assert g.kv_len() == 50 + len(got) - 1
    assert got == want[:len(got)] or not clear
    assert max(runs) > 3 and min(runs) == 1
    r = oracle.RefModel(shape, weights(shape), quant=quant, kv_bf16=(kv == "bf16"))
    logits = r.forward(text, 0)
    for i, t in enumerate(got):
        assert logits[t] >= logits.max() - 2 * BARS[kv] * np.abs(logits).max(), i
        logits = r.forward([t], 50 + i)


def test_the_first_of_two_equal_children_is_taken(hip):
    shape = configs.TINY_LLAMA
    g = model(hip, shape)
    text = synth.make_tokens(shape.vocab_size, 12, seed=30)
    first = g.forward_greedy(text, 0)
    a = int(g.forward_tree([first], [-1], 12)[0])
    b = int(g.forward_tree([first, a], [-1, 0], 12)[1])
    # Nodes 1 and 2 are both right; 3 hangs on the second, 4 on the first.
    tokens, parents = [first, a, a, b, b], [-1, 0, 0, 2, 1]
    accepted, _ = g.verify_tree(tokens, parents, 12)
    assert accepted.tolist() == [0, 1, 4]
    assert g.kv_len() == 15


@pytest.mark.parametrize("shape", TINY, ids=lambda s: s.name)
def test_a_dropped_tree_leaves_no_trace(hip, shape):
    g, plain = model(hip, shape), model(hip, shape)
    text = synth.make_tokens(shape.vocab_size, 61, seed=31)
    drafts = synth.make_tokens(shape.vocab_size, len(FORK), seed=32)
    g.forward(text, 0)
    want = plain.forward(text, 0)
    want = [plain.forward([3], 61), plain.forward(drafts, 62)]
    g.forward_tree(drafts, FORK, 61)
    g.commit_tree([])
    g.forward_tree(drafts[::-1].copy(), FORK, 61)
    assert np.array_equal(bits(g.forward([3], 61)), bits(want[0]))
    with pytest.raises(hip.HipError, match="no tree"):
        g.commit_tree([0])
    g.forward_tree(drafts, FORK, 62)
    assert np.array_equal(bits(g.forward(drafts, 62)), bits(want[1]))
    for drop in (lambda: g.decode_greedy(1, g.kv_len(), 2), lambda: g.forward_logprobs([1], g.kv_len()),
                 lambda: g.restore_kv_prefix(g.kv_snapshot(), 70), g.clear_cache):
        g.forward_tree(drafts, FORK, g.kv_len())
        drop()
        with pytest.raises(hip.HipError, match="no tree"):
            g.commit_tree([0])


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_a_snapshot_taken_while_a_tree_waits(hip, kv):
    """The commit moves rows in the instance's own copy of the shared page."""
    shape = configs.TINY_QWEN2
    g = model(hip, shape, kv=kv)
    text = synth.make_tokens(shape.vocab_size, 60, seed=33)
    drafts = synth.make_tokens(shape.vocab_size, len(FORK), seed=34)
    g.forward(text, 0)
    g.forward_tree(drafts, FORK, 60)
    snap = g.kv_snapshot()
    other = g.clone()
    other.restore_kv_prefix(snap, 60)
    before = [other.kv_rows(l, 0, 60) for l in range(shape.num_layers)]
    logits = other.forward(drafts[:3], 60)
    branch = path(FORK, 12)
    g.commit_tree(branch)
    alone = model(hip, shape, kv=kv)
    alone.forward(text, 0)
    alone.forward(drafts[branch], 60)
    end = 60 + len(branch)
    for a, b in zip(g.kv_rows(0, 0, end), alone.kv_rows(0, 0, end)):
        assert np.array_equal(bits(a), bits(b))
    third = g.clone()
    third.restore_kv_prefix(snap, 60)
    for l in range(shape.num_layers):
        for a, b in zip(third.kv_rows(l, 0, 60), before[l]):
            assert np.array_equal(bits(a), bits(b))
    assert np.array_equal(bits(third.forward(drafts[:3], 60)), bits(logits))


def test_refusals_leave_the_model_as_it_was(hip):
    shape = configs.TINY_QWEN2
    g = model(hip, shape, capacity=128, chunk=32)
    text = synth.make_tokens(shape.vocab_size, 100, seed=35)
    g.forward(text, 0)
    for tokens, parents, offset, says in [([1, 2], [-1, 1], 100, "comes before it"), ([1], [-2], 100, "comes before it"),
                                          ([1], [-1], 99, "does not match"), ([1], [-1], 101, "does not match"),
                                          ([1, 1000], [-1, 0], 100, "vocabulary"), ([], [], 100, "empty"),
                                          ([1] * 29, [-1] * 29, 100, "capacity"),
                                          ([1] * 33, [-1] * 33, 100, "chunk rows"),
                                          ([1] * 257, [-1] * 257, 100, "at most 256 nodes")]:
        with pytest.raises(hip.HipError, match=says):
            g.forward_tree(tokens, parents, offset)
    with pytest.raises(hip.HipError, match="no tree"):
        g.commit_tree([0])
    with pytest.raises(hip.HipError, match="no tree"):
        g.commit_tree([])
    parents = [-1, -1, 0, 2, 1]
    g.forward_tree([1, 2, 3, 4, 5], parents, 100)
    for nodes in ([2], [0, 1], [0, 3], [0, 2, 3, 4], [5], [1, 4, 4], [0, 2, 3, 3, 3, 3], [0xffffffff]):
        with pytest.raises(hip.HipError, match="branch"):
            g.commit_tree(nodes)
    with pytest.raises(hip.HipError, match="one root"):
        g.verify_tree([1, 2], [-1, -1], 100)
    for kw, says in [(dict(top=65), "at most 64"), (dict(targets=None, offset=99), "does not match")]:
        with pytest.raises(hip.HipError, match=says):
            g.forward_logprobs([1, 2], kw.pop("offset", 100), **kw)
    with pytest.raises(hip.HipError, match="capacity"):
        g.forward_logprobs([1] * 29, 100)
    g.commit_tree([0, 2, 3])  # none of them dropped it
    assert g.kv_len() == 103
    plain = model(hip, shape, capacity=128, chunk=32)
    plain.forward(text, 0)
    plain.forward([1, 3, 4], 100)
    assert rel_err(g.forward([9], 103), plain.forward([9], 103)) < BARS["bf16"]
    # Up to the last position.
    g.forward_tree([1] * 24, list(range(-1, 23)), 104)
    g.commit_tree(list(range(24)))
    with pytest.raises(hip.HipError, match="capacity"):
        g.forward_tree([1], [-1], 128)


def test_arrays_of_other_lengths_are_refused(hip):
    g = model(hip, configs.TINY_QWEN2)
    g.forward([1, 2, 3], 0)
    for call in (lambda: g.forward_tree([1, 2], [-1], 3), lambda: g.verify_tree([1], [-1, 0], 3),
                 lambda: g.forward_logprobs([1, 2], 3, targets=[1])):
        with pytest.raises(ValueError, match="one (parent|target) a token"):
            call()
    assert g.kv_len() == 3


def test_the_pool_runs_out_under_a_tree(hip):
    """A clone holds the pages that a tree would need: refused, nothing lost."""
    shape = configs.TINY_LLAMA
    g = model(hip, shape, capacity=256, chunk=64)
    other = g.clone()
    text = synth.make_tokens(shape.vocab_size, 128, seed=36)
    other.forward(text, 0)
    g.forward(text[:120], 0)
    with pytest.raises(hip.HipError, match="pool exhausted"):
        g.forward_tree([1] * 20, [-1] * 20, 120)
    want = g.forward_tree([1] * 8, [-1] * 8, 120, want_logits=True)[1]
    assert np.array_equal(bits(want), bits(np.repeat(want[:1], 8, 0)))
    g.commit_tree([5])
    assert g.kv_len() == 121


def test_evicted_weights_give_the_same_bits(hip):
    shape = configs.TINY_LLAMA
    text = synth.make_tokens(shape.vocab_size, 40, seed=37)
    drafts = synth.make_tokens(shape.vocab_size, len(FORK), seed=38)
    for quant in (None, "q8"):
        g = model(hip, shape, quant=quant)
        runs = []
        for _ in range(2):
            g.forward(text, 0)
            nxt, logits = g.forward_tree(drafts, FORK, 40, want_logits=True)
            accepted = g.verify_tree(drafts, [-1, 0] + [0] * 11, 40)
            scores = g.forward_logprobs(drafts, g.kv_len(), targets=drafts, top=3)
            runs.append([nxt, bits(logits), accepted[0], accepted[1]] + [np.asarray(s).view(np.uint32) for s in scores])
            g.clear_cache()
            for unit in ("model.layers.0.mlp.down_proj.weight", "model.layers.1.self_attn.q_proj.weight",
                         "model.layers.1.mlp.down_proj.weight"):
                assert g.evict_unit(unit)
        for a, b in zip(*runs):
            assert np.array_equal(a, b)


def test_instances_in_threads(hip):
    """Clones that verify and score at once, each on its own stream."""
    shape = configs.TINY_QWEN2
    base = model(hip, shape, capacity=2048)
    texts = [synth.make_tokens(shape.vocab_size, 40 + 9 * i, seed=40 + i) for i in range(4)]

    def run(text, out):
        g = base.clone()
        t = g.forward_greedy(text, 0)
        for k in range(6):
            drafts = [t] + synth.make_tokens(shape.vocab_size, 11, seed=60 + k).tolist()
            acc, t = g.verify_tree(drafts, [-1] + [0] * 11, g.kv_len())
            out.append((acc.tolist(), t))
        out.append([np.asarray(s).tobytes() for s in g.forward_logprobs(text, g.kv_len(), targets=text, top=5)])

    alone = [[] for _ in texts]
    for text, out in zip(texts, alone):
        run(text, out)
    together = [[] for _ in texts]
    threads = [threading.Thread(target=run, args=a) for a in zip(texts, together)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert together == alone


def log_softmax(x):
    x = np.asarray(x, np.float64)
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


@pytest.mark.parametrize("n,chunk,top", [(37, 16, 5), (1, 0, 3), (40, 40, 64), (9, 2, 0)])
@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("shape", TINY, ids=lambda s: s.name)
def test_scores_match_the_oracle(hip, oracle, shape, kv, n, chunk, top):
    g, r = model(hip, shape, kv=kv), oracle.RefModel(shape, weights(shape), kv_bf16=(kv == "bf16"))
    text = synth.make_tokens(shape.vocab_size, 20 + n + 1, seed=50)
    g.forward(text[:20], 0)
    r.forward(text[:20], 0)
    lp, ent, ids, tops = g.forward_logprobs(text[20:20 + n], 20, targets=text[21:], top=top, chunk_rows=chunk)
    assert g.kv_len() == 20 + n
    for i in range(n):
        x = r.forward(text[20 + i:21 + i], 20 + i)
        want = log_softmax(x)
        e = BARS[kv] * float(np.abs(x).max())
        assert abs(lp[i] - want[text[21 + i]]) < 2 * e + 1e-5, i
        assert abs(ent[i] + (np.exp(want) * want).sum()) < e * (2 * np.log(x.size) + 2) + 1e-5, i
        order = np.sort(want)[::-1]
        assert len(set(ids[i].tolist())) == top
        assert np.all(np.abs(tops[i] - order[:top]) < 2 * e + 1e-5), i
        assert np.all(np.abs(tops[i] - want[ids[i]]) < 2 * e + 1e-5), i
    assert rel_err(g.forward([4], 20 + n), r.forward([4], 20 + n)) < BARS[kv]


def test_scoring_keeps_the_cache_of_forward(hip):
    """The same chunks give the same K/V bits, and the last row's scores are its
    logits'; rows in groups (a chunk of 520) and outputs left out."""
    shape = configs.TINY_QWEN2
    g, plain = model(hip, shape, capacity=1024, chunk=600), model(hip, shape, capacity=1024, chunk=600)
    text = synth.make_tokens(shape.vocab_size, 520, seed=51)
    targets = np.append(text[1:], 0).astype(np.uint32)
    targets[7] = shape.vocab_size  # no such token
    lp, ent, ids, tops = g.forward_logprobs(text, 0, targets=targets, top=4, chunk_rows=600)
    logits = plain.forward(text, 0, chunk_rows=600)
    for l in range(shape.num_layers):
        for a, b in zip(g.kv_rows(l, 0, 520), plain.kv_rows(l, 0, 520)):
            assert np.array_equal(bits(a), bits(b))
    assert np.isnan(lp[7]) and np.isnan(lp).sum() == 1
    e = BARS["f32"] * float(np.abs(logits).max())  # the same K/V bits
    assert abs(lp[519] - log_softmax(logits)[0]) < 2 * e + 1e-5
    assert np.all(np.abs(tops[519] - log_softmax(logits)[ids[519]]) < 2 * e + 1e-5)
    g.clear_cache()
    again = g.forward_logprobs(text, 0, top=4, chunk_rows=600)
    assert again[0] is None
    for a, b in zip((ent, ids, tops), again[1:]):
        assert a.tobytes() == b.tobytes()
    g.clear_cache()
    none = g.forward_logprobs(text, 0, chunk_rows=600)
    assert none[1].tobytes() == ent.tobytes() and none[2].size == 0
