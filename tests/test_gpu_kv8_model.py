"""A model over an 8-bit K/V cache (kv="e4m3"): prefill, decode, windows,
snapshots and clones, scoring, host-tier weights; what it refuses."""
import threading

import numpy as np
import pytest

import kv8_reference as ref
from cheetah_amd import configs, synth

pytestmark = pytest.mark.gpu

TINY = [configs.TINY_QWEN2, configs.TINY_LLAMA]
GROUP7 = configs.TINY_QWEN2.replace(name="tiny-7", q_heads=7, kv_heads=1, hidden_size=192)

# The logits are held to 64-bit ones that attend to the very values the cache holds
# (read back), so the codes' own rounding is no part of the difference: projections
# take inputs of 2^-17 / sqrt(3) (5e-6, ten of them in two layers: 1.5e-5 at random),
# rotation angles are f32 (2^-24 of up to 600, 4e-5). A wrong code moves its value by
# 2^-4. 5e-4 of the largest logit.
TOL = 5e-4

_W = {}


def weights(shape):
    if shape.name not in _W:
        units = synth.make_weights(shape)
        _W[shape.name] = units, {k: synth.bf16_to_f32(v).astype(np.float64).reshape(v.shape) for k, v in units.items()}
    return _W[shape.name]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def model(hip, shape, quant=None, capacity=1024, chunk=64):
    return hip.HipForward(shape, weights(shape)[0], quant=quant, kv_capacity=capacity, max_chunk_rows=chunk, kv="e4m3")


def rel_err(got, want):
    return float(np.max(np.abs(np.asarray(got, np.float64) - want)) / np.max(np.abs(want)))


def held(g, layer, n):
    return tuple(x.astype(np.float64) for x in g.kv_rows(layer, 0, n))


def check(g, shape, tokens, logits):
    """The last row's logits against 64 bits over the cache's own values, and
    those against the rows that were to be quantised: half a step of a code
    (2^-4 of a value), or of the smallest (2^-10 of a scale, which is below 2^-7.8 of
    the block's largest), at each growth of the block's scale once more, and
    1e-3 of the block's largest for the rows' own difference."""
    n = len(tokens)
    want, rows = ref.decoder64(shape, weights(shape)[1], tokens, lambda layer: held(g, layer, n), shape.sliding_window)
    assert rel_err(logits, want[-1]) < TOL
    for layer, pair in enumerate(rows):
        for got, x in zip(held(g, layer, n), pair):
            for b in range(0, n, 32):
                y, z = got[b:b + 32], x[b:b + 32]
                most = np.abs(z).max((0, 2), keepdims=True)
                assert (np.abs(y - z) <= 2.0 ** -4 * np.abs(z) + (2.0 ** -16.8 + 1e-3) * most).all(), (layer, b)


@pytest.mark.parametrize("shape", TINY + [GROUP7], ids=lambda s: s.name)
@pytest.mark.parametrize("n,chunk", [(2, 64), (31, 64), (64, 64), (100, 64), (130, 37), (257, 20)])
def test_prefill(hip, shape, n, chunk):
    g = model(hip, shape)
    tokens = synth.make_tokens(shape.vocab_size, n)
    check(g, shape, tokens, g.forward(tokens, 0, chunk_rows=chunk))
    assert g.kv_len() == n


@pytest.mark.parametrize("fused", ["1", "0"])
@pytest.mark.parametrize("graph", ["1", "0"])
@pytest.mark.parametrize("shape", TINY + [GROUP7], ids=lambda s: s.name)
def test_decode_steps(hip, shape, graph, fused, monkeypatch):
    """Prefill, then steps over block, page and split boundaries; captured steps
    are replayed with other work between them."""
    monkeypatch.setenv("CHEETAH_HIP_GRAPH", graph)
    monkeypatch.setenv("CHEETAH_HIP_FUSED", fused)
    g, other = model(hip, shape), model(hip, shape)
    tokens = list(synth.make_tokens(shape.vocab_size, 250))
    g.forward(tokens, 0)
    for step in range(20):
        tokens.append((7 * step + 3) % shape.vocab_size)
        logits = g.forward(tokens[-1:], len(tokens) - 1)
        if step % 6 == 0:
            other.clear_cache()
            other.forward(tokens[:50], 0)
        if step % 5 == 4:
            check(g, shape, tokens, logits)


def test_decode_from_an_empty_cache(hip):
    shape = configs.TINY_LLAMA
    g, tokens = model(hip, shape), []
    for step in range(40):
        tokens.append((11 * step + 5) % shape.vocab_size)
        logits = g.forward(tokens[-1:], step)
    check(g, shape, tokens, logits)


@pytest.mark.parametrize("quant", [None, "q8", "q4"])
def test_greedy_loop_is_the_steps(hip, quant):
    shape = configs.TINY_QWEN2
    a, b = model(hip, shape, quant), model(hip, shape, quant)
    prompt = synth.make_tokens(shape.vocab_size, 90)
    first = a.forward_greedy(prompt, 0)
    assert b.forward_greedy(prompt, 0) == first
    loop, steps, token = a.decode_greedy(first, 90, 60), [], first
    for i in range(60):
        token = b.forward_greedy([token], 90 + i)
        steps.append(token)
    assert loop.tolist() == steps
    np.testing.assert_array_equal(a.kv_rows(1, 0, 150), b.kv_rows(1, 0, 150))


@pytest.mark.parametrize("window", [1, 33, 100, 500])
def test_sliding_window(hip, window):
    """A model with a window: every row of prefill and decode sees the last
    `window` positions; over the other caches such a model is refused."""
    shape = configs.TINY_LLAMA.replace(sliding_window=window)
    g = model(hip, shape)
    tokens = list(synth.make_tokens(shape.vocab_size, 210))
    check(g, shape, tokens, g.forward(tokens, 0, chunk_rows=50))
    for step in range(5):
        tokens.append(step + 9)
        logits = g.forward(tokens[-1:], len(tokens) - 1)
    check(g, shape, tokens, logits)
    for kv in ("bf16", "f32"):
        with pytest.raises(hip.HipError, match="sliding-window"):
            hip.HipForward(shape, weights(shape)[0], kv=kv)


@pytest.mark.parametrize("hd", [64, 128])
def test_a_step_that_raises_a_scale(hip, hd):
    """Decode steps whose K and V outgrow their block: its earlier rows are rounded
    again (normal codes, from 2^-6 of the new scale on, keep their values; others
    move by at most half a step, 2^-10), other blocks are as they were."""
    shape = configs.TINY_QWEN2 if hd == 64 else configs.TINY_LLAMA
    assert shape.head_dim == hd
    units = dict(weights(shape)[0])
    loud = 77
    x = synth.bf16_to_f32(units["model.embed_tokens.weight"]).reshape(shape.vocab_size, -1)[loud]
    for name in ("k", "v"):
        key = f"model.layers.0.self_attn.{name}_proj.weight"
        w = synth.bf16_to_f32(units[key]).reshape(-1, x.size)
        w = w + np.where(np.arange(len(w)) % 5 == 0, 4.0, 0.0)[:, None] * (x / np.linalg.norm(x))[None]
        units[key] = synth.f32_to_bf16(w.astype(np.float32)).reshape(units[key].shape)
    g = hip.HipForward(shape, units, kv_capacity=1024, max_chunk_rows=64, kv="e4m3")
    tokens = [t for t in synth.make_tokens(shape.vocab_size, 200) if t != loud][:70]
    g.forward(tokens, 0)
    raised = moved = 0
    for step in range(60):
        n = 70 + step
        before = g.kv_rows(0, 0, n)
        g.forward([loud if step % 13 == 5 else 3 * step + 200], n)
        for old, new in zip(before, g.kv_rows(0, 0, n + 1)):
            b = n // 32 * 32
            np.testing.assert_array_equal(old[:b], new[:b])
            _, e = np.frexp(np.abs(new[b:]).max((0, 2)) / 448)  # 2^e: at least the block's scale, at most twice
            unit = 2.0 ** e[None, :, None]
            move = np.abs(old[b:].astype(np.float64) - new[b:n])
            assert (move <= unit * 2.0 ** -10).all()
            assert (move[np.abs(old[b:]) >= unit * 2.0 ** -6] == 0).all()
            moved += int((move > 0).any())
            raised += int(n > b and (np.abs(new[n]).max(1) > 2 * np.abs(old[b:]).max((0, 2), initial=0)).any())
            last = np.abs(new[n]).max(1)
            assert (last > 0).all() and np.isfinite(new).all()
    # Two blocks have a first loud row, for K and for V; values far enough below it to
    # move (2^-13.8) are a hundredth of all.
    assert raised >= 4 and moved >= 1


ODD = configs.TINY_QWEN2.replace(name="tiny-odd", q_heads=5, kv_heads=1, head_dim=128)


@pytest.mark.parametrize("graph", ["1", "0"])
@pytest.mark.parametrize("shape", [configs.TINY_QWEN2, GROUP7, ODD], ids=lambda s: s.name)
def test_cached_rows_are_the_rotated_ones_quantised(hip, shape, graph, monkeypatch):
    """With k_proj and v_proj zero a row is the bias, K's rotated: the rows that a
    model with an f32 cache holds. The 8-bit cache holds exactly these, quantised in
    the same pieces, through prefill and decode. (The first pair of K, 4 long, turns
    past 3.5 = 448 * 2^-7 at position 33 and not at 32: the block's scale rises.)"""
    monkeypatch.setenv("CHEETAH_HIP_GRAPH", graph)
    units = dict(weights(shape)[0])
    for layer in range(shape.num_layers):
        p = f"model.layers.{layer}.self_attn."
        for name in ("k_proj", "v_proj"):
            units[p + name + ".weight"] = np.zeros_like(units[p + name + ".weight"])
        bias = synth.bf16_to_f32(units[p + "k_proj.bias"]).reshape(shape.kv_heads, -1).copy()
        bias[:, 0], bias[:, shape.head_dim // 2] = 4, 0
        units[p + "k_proj.bias"] = synth.f32_to_bf16(bias.astype(np.float32)).reshape(units[p + "k_proj.bias"].shape)
    tokens = synth.make_tokens(shape.vocab_size, 100)
    models = [hip.HipForward(shape, units, kv_capacity=256, max_chunk_rows=64, kv=kv) for kv in ("f32", "e4m3")]
    for g in models:
        g.forward(tokens[:20], 0)
        for pos in range(20, 100):
            g.forward(tokens[pos:pos + 1], pos)
    for layer in range(shape.num_layers):
        rows = models[0].kv_rows(layer, 0, 100)
        cpu = ref.Cache(100, shape.kv_heads, shape.head_dim)
        cpu.append(*(x[:20] for x in rows), 0)
        for pos in range(20, 100):
            risen = cpu.exps[0, pos // 32, 0]
            cpu.append(*(x[pos:pos + 1] for x in rows), pos)
            assert pos != 33 or cpu.exps[0, 1, 0] == risen + 1
        for got, want in zip(models[1].kv_rows(layer, 0, 100), cpu.values(0, 100)):
            np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("window", [2**31 - 1, 2**31, 2**32 - 1])
def test_a_window_past_every_position_is_none(hip, window):
    shape = configs.TINY_LLAMA
    g, plain = model(hip, shape.replace(sliding_window=window)), model(hip, shape)
    tokens = synth.make_tokens(shape.vocab_size, 150)
    np.testing.assert_array_equal(g.forward(tokens, 0), plain.forward(tokens, 0))
    np.testing.assert_array_equal(g.forward([5], 150), plain.forward([5], 150))


@pytest.mark.parametrize("at", [33, 64, 90])
def test_snapshots_and_clones(hip, at):
    """A snapshot inside a block keeps its values and scales while the instance
    goes on (larger rows would raise them); a clone that restores it, or a
    shorter prefix of it, goes on as a cache of its own."""
    shape = configs.TINY_QWEN2
    g = model(hip, shape)
    tokens = synth.make_tokens(shape.vocab_size, 200)
    g.forward(tokens[:at], 0)
    before = [g.kv_rows(layer, 0, at) for layer in range(2)]
    snap = g.kv_snapshot()
    after = g.forward(tokens[at:], at)
    other = g.clone()
    other.restore_kv_prefix(snap, at)
    for layer in range(2):
        np.testing.assert_array_equal(other.kv_rows(layer, 0, at), before[layer])
    np.testing.assert_array_equal(other.forward(tokens[at:], at), after)
    for layer in range(2):
        np.testing.assert_array_equal(other.kv_rows(layer, 0, 200), g.kv_rows(layer, 0, 200))
    other.restore_kv_prefix(snap, at - 11)
    logits = other.forward(tokens[at - 11:150], at - 11)
    check(other, shape, tokens[:150], logits)
    third = g.clone()
    third.restore_kv_prefix(snap, at)
    for layer in range(2):
        np.testing.assert_array_equal(third.kv_rows(layer, 0, at), before[layer])


def test_a_reused_page_starts_afresh(hip):
    """Pages that held large rows serve a new text: the blocks' scales are the
    new rows' (the old ones would cost it its small values)."""
    shape = configs.TINY_QWEN2
    units = dict(weights(shape)[0])
    g, fresh = (hip.HipForward(shape, units, kv_capacity=128, max_chunk_rows=64, kv="e4m3") for _ in "gf")
    tokens = synth.make_tokens(shape.vocab_size, 128)
    g.forward(tokens, 0)
    g.clear_cache()
    np.testing.assert_array_equal(g.forward(tokens[64:128], 0), fresh.forward(tokens[64:128], 0))


def test_scoring_follows_the_logits(hip):
    shape = configs.TINY_QWEN2
    g, plain = model(hip, shape), model(hip, shape)
    tokens = synth.make_tokens(shape.vocab_size, 120)
    lp, ent, ids, tops = g.forward_logprobs(tokens[:-1], 0, targets=tokens[1:], top=3)
    logits = plain.forward(tokens[:-1], 0).astype(np.float64)
    p = logits - logits.max()
    p -= np.log(np.exp(p).sum())
    assert abs(lp[-1] - p[tokens[-1]]) < 1e-4 and ids[-1, 0] == logits.argmax()
    np.testing.assert_array_equal(g.kv_rows(1, 0, 119), plain.kv_rows(1, 0, 119))


def test_host_tier_weights_give_the_same_bits(hip):
    shape = configs.TINY_QWEN2
    g, plain = model(hip, shape), model(hip, shape)
    tokens = synth.make_tokens(shape.vocab_size, 70)
    assert g.evict_unit("model.layers.1.mlp.up_proj.weight")
    assert g.evict_unit("model.layers.0.self_attn.q_proj.weight")
    np.testing.assert_array_equal(g.forward(tokens, 0), plain.forward(tokens, 0))
    np.testing.assert_array_equal(g.forward([5], 70), plain.forward([5], 70))


@pytest.mark.parametrize("window", [0, 60])
def test_clones_in_threads(hip, window):
    """Clones share pages (a prefix ends inside a block) and nothing else: each in a
    thread of its own gives what it gives alone."""
    shape = configs.TINY_LLAMA.replace(sliding_window=window)
    base = model(hip, shape, capacity=4096)
    prefix = synth.make_tokens(shape.vocab_size, 77)
    base.forward(prefix, 0)
    snap = base.kv_snapshot()
    texts = [synth.make_tokens(shape.vocab_size, n, seed=n) for n in (2, 30, 101, 400)]

    def run(text, out):
        g = base.clone()
        g.restore_kv_prefix(snap, len(prefix))
        token = g.forward_greedy(text, len(prefix))
        out.append(g.decode_greedy(token, len(prefix) + len(text), 50).tolist())
        out.append([x.tobytes() for layer in range(2) for x in g.kv_rows(layer, 0, g.kv_len())])

    alone = [[] for _ in texts]
    for args in zip(texts, alone):
        run(*args)
    assert len({x[0][0] for x in alone}) > 1
    # Several times: clones are made while others capture their first steps.
    for _ in range(8):
        together = [[] for _ in texts]
        threads = [threading.Thread(target=run, args=args) for args in zip(texts, together)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert together == alone


def test_drafted_tokens_are_refused(hip):
    g = model(hip, configs.TINY_QWEN2)
    g.forward([1, 2, 3], 0)
    with pytest.raises(hip.HipError, match="drafted tokens"):
        g.forward_tree([4, 5], [-1, 0], 3)
    with pytest.raises(hip.HipError, match="drafted tokens"):
        g.verify_tree([4, 5], [-1, 0], 3)
    assert g.kv_len() == 3
    g.forward([4], 3)


def test_the_last_position_of_the_capacity(hip):
    """kv_download at the end of the capacity, and the refusal past it."""
    g = model(hip, configs.TINY_QWEN2, capacity=130)
    tokens = synth.make_tokens(1000, 130)
    g.forward(tokens, 0)
    k, v = g.kv_rows(0, 65, 65)
    assert np.isfinite(k).all() and np.isfinite(v).all()
    with pytest.raises(hip.HipError, match="capacity"):
        g.forward([1], 130)


def test_unknown_cache_formats_are_refused(hip):
    import ctypes
    cfg = hip.make_config(configs.TINY_QWEN2)
    assert not hip.lib().cheetah_hip_model_create(ctypes.byref(cfg), 0, 3, 0, 0)
    assert b"kv_format" in hip.lib().cheetah_hip_last_error()
    with pytest.raises(ValueError, match="kv must be one of"):
        hip.HipForward(configs.TINY_QWEN2, kv="e5m2")
