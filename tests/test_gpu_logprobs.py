"""Log probabilities, entropies and alternatives against 64 bits.

A logit's difference to the maximum is rounded once (2^-24 of it, weighed by
e^-d: at most 2^-25 in all), its exponential to 2^-22, a thread's sum over at
most 32 terms to 32 * 2^-24 before it goes on in 64 bits: 2.2e-6 of the sums,
that much in their logarithm, and the results are rounded to f32 once."""
import ctypes

import numpy as np
import pytest

import tree_reference as ref
from cheetah_amd import synth

pytestmark = pytest.mark.gpu

SUMS = 2.0**-22 + 33 * 2.0**-24


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def check(got, x, tokens, top):
    lp, entropy, ids, tops = got
    wlp, went, wids, wtops = ref.logprobs64(x, tokens, top)
    assert np.array_equal(ids, wids)
    for g, w in ((lp, wlp), (tops, wtops)):
        fine = np.isfinite(w)
        assert np.array_equal(g[~fine], w[~fine])  # -inf
        assert (np.abs(g[fine] - w[fine]) <= SUMS + 2.0**-24 * np.abs(w[fine])).all()
    # Positive terms only, each within its own error and its factor d's: relative.
    assert (np.abs(entropy - went) <= (2 * SUMS + 2.0**-22) * went).all()


def logits(rng, rows, vocab, stride, fmt, scale=3.0):
    x = (rng.standard_normal((rows, stride)) * scale).astype(np.float32)
    x[np.arange(rows), rng.integers(0, vocab, rows)] += rng.random(rows).astype(np.float32) * 20
    x[:, vocab:] = np.nan
    if fmt == "f32":
        return x, x
    b = synth.f32_to_bf16(x)
    return b, synth.bf16_to_f32(b).reshape(x.shape)


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,pad,top", [
    (1, 1, 0, 1), (1, 1, 3, 0), (3, 2, 0, 2), (2, 5, 1, 5), (4, 64, 0, 64), (3, 65, 2, 64), (5, 100, 0, 64), (1, 255, 1, 20),
    (2, 256, 0, 20), (2, 257, 5, 1), (7, 1000, 0, 5), (3, 4095, 0, 20), (3, 4097, 0, 64), (1, 8192, 0, 20),
    (2, 8193, 7, 20), (1, 32000, 0, 5), (37, 32001, 31, 64), (1, 151936, 0, 20), (3, 151937, 1, 64), (1, 200003, 0, 64),
    (300, 5001, 0, 20), (700, 9001, 0, 5), (520, 32003, 0, 1), (600, 20000, 0, 64), (1500, 300, 0, 20)])
def test_logprobs_match_64_bits(hip, rows, vocab, pad, top, fmt):
    """One logit to 200,003, odd sizes and rows off 16 bytes, few rows (split)
    and many; NaN in the padding between rows."""
    rng = np.random.default_rng(rows * 7 + vocab)
    x, values = logits(rng, rows, vocab, vocab + pad, fmt)
    tokens = rng.integers(0, vocab, rows).astype(np.uint32)
    check(hip.logprobs(x, tokens, top, vocab), values[:, :vocab], tokens, top)


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 40, 600])
@pytest.mark.parametrize("kind", ["equal", "zeros", "two", "rising", "falling", "late", "masked", "few", "empty", "lowest",
                                  "blocks"])
def test_logprobs_ties_orders_and_masks(hip, kind, rows, fmt):
    """Equal logits (lowest ids first), -0 and 0, sorted rows, the best ones at
    the end, masks that leave few tokens or none, masks of the type's lowest
    value, runs of equal logits as long as what a block reads at once."""
    rng = np.random.default_rng(rows)
    vocab, top = (20011 if rows < 600 else 9011), 64
    x = np.zeros((rows, vocab), np.float32)
    low = np.float32(synth.bf16_to_f32(np.array([0xFF7F], np.uint16))[0])
    if kind == "equal":
        x[:] = 2.5
    elif kind == "zeros":
        x[:, rng.random(vocab) < 0.5] = -0.0
    elif kind == "two":
        x[rng.random(x.shape) < 0.01] = 1.0
    elif kind in ("rising", "falling"):
        x[:] = np.arange(vocab) // 16 * 0.125 * (1 if kind == "rising" else -1)
    elif kind == "late":
        x[:, -200:] = 3
        x[:, -1] = 4
    elif kind == "blocks":
        x[:] = (np.arange(vocab) // 2048 % 3).astype(np.float32)
    else:
        x = (rng.standard_normal(x.shape) * 3).astype(np.float32)
        share = {"masked": 0.5, "few": 0.9995, "empty": 1.0, "lowest": 0.9}[kind]
        x[rng.random(x.shape) < share] = low if kind == "lowest" else -np.inf
    if fmt == "bf16":
        x = synth.f32_to_bf16(x)
        values = synth.bf16_to_f32(x).reshape(x.shape)
    else:
        values = x
    tokens = rng.integers(0, vocab, rows).astype(np.uint32)
    check(hip.logprobs(x, tokens, top), values, tokens, top)


@pytest.mark.parametrize("rows", [1, 530])
def test_one_token_nearly_certain(hip, rows):
    """Its log probability is a small number with all of its digits: the sum
    over the others, relative."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((rows, 5000)).astype(np.float32)
    x[:, 1234] = 25 + rng.random(rows)
    tokens = np.full(rows, 1234, np.uint32)
    lp, entropy, _, _ = hip.logprobs(x, tokens, 1)
    wlp, went, _, _ = ref.logprobs64(x, tokens, 1)
    assert (wlp > -1e-6).all()
    # d is 20 to 29 here: its rounding (2^-24 of it) goes into each term whole.
    tol = 2 * SUMS + 30 * 2.0**-24 + 2.0**-24
    assert (np.abs(lp - wlp) <= tol * np.abs(wlp)).all()
    assert (np.abs(entropy - went) <= tol * went).all()


@pytest.mark.parametrize("rows", [2, 520])
@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_nan_or_infinite_logit_stays_in_its_row(hip, bad, fmt, rows):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((rows, 9000)).astype(np.float32)
    x[1, 7777] = bad
    x = x if fmt == "f32" else synth.f32_to_bf16(x)
    values = x if fmt == "f32" else synth.bf16_to_f32(x).reshape(x.shape)
    tokens = rng.integers(0, 9000, rows).astype(np.uint32)
    lp, entropy, ids, tops = hip.logprobs(x, tokens, 20)
    assert np.isnan(lp[1]) and np.isnan(entropy[1]) and np.isnan(tops[1]).all()
    order = np.where(np.isnan(values[1]), -np.inf, values[1])
    assert np.array_equal(ids[1], np.argsort(-order, kind="stable")[:20])
    rest = np.arange(rows) != 1
    check((lp[rest], entropy[rest], ids[rest], tops[rest]), values[rest], tokens[rest], 20)


def test_nan_everywhere_still_orders_by_id(hip):
    for rows in (1, 600):
        lp, entropy, ids, tops = hip.logprobs(np.full((rows, 300), np.nan, np.float32), np.zeros(rows, np.uint32), 64)
        assert np.isnan(lp).all() and np.isnan(entropy).all() and np.isnan(tops).all()
        assert np.array_equal(ids, np.tile(np.arange(64, dtype=np.uint32), (rows, 1)))


def test_an_id_past_the_vocabulary_gives_nan(hip):
    x = np.zeros((4, 1000), np.float32)
    lp, entropy, _, _ = hip.logprobs(x, np.array([0, 1000, 2**32 - 1, 999], np.uint32), 0)
    assert np.isnan(lp[[1, 2]]).all()
    assert np.allclose(lp[[0, 3]], -np.log(1000)) and np.allclose(entropy, np.log(1000))


@pytest.mark.parametrize("rows", [1, 520])
def test_outputs_left_out_change_nothing(hip, rows):
    """Each output alone gives the bits it has beside the others; the buffers
    of the others stay as they were."""
    rng = np.random.default_rng(8)
    x, _ = logits(rng, rows, 7001, 7001, "f32")
    tokens = rng.integers(0, 7001, rows).astype(np.uint32)
    want = hip.logprobs(x, tokens, 20)
    xd, td = hip.DeviceBuffer.from_array(x), hip.DeviceBuffer.from_array(tokens)
    for which in range(3):
        bufs = [hip.DeviceBuffer.from_array(np.full(rows * (1 if i < 2 else 20), 77, np.uint32)) for i in range(4)]
        p = [b.ptr for b in bufs]
        args = [(p[0], None, None, None), (None, p[1], None, None), (None, None, p[2], p[3])][which]
        hip.check(hip.lib().cheetah_hip_logprobs(xd.ptr, 1, rows, 7001, 7001, td.ptr if which == 0 else None,
                                                 20 if which == 2 else 0, *args))
        got = [b.download(np.uint32) for b in bufs]
        for i in range(4):
            written = i == which or (which == 2 and i == 3)
            assert np.array_equal(got[i], want[i].view(np.uint32).reshape(-1) if written else np.full(got[i].size, 77))


def test_rows_past_4_gib(hip):
    """A stride that puts the second row past 2^32 bytes (and elements)."""
    stride, vocab = (1 << 30) + 12345, 3000
    rng = np.random.default_rng(10)
    rows = [(rng.standard_normal(vocab) * 3).astype(np.float32) for _ in range(2)]
    big = hip.DeviceBuffer((stride + vocab) * 4)
    for r, at in zip(rows, (0, stride * 4)):
        hip.check(hip.lib().cheetah_hip_upload(big.ptr + at, r.ctypes.data, r.nbytes))
    tokens = np.array([5, 2999], np.uint32)
    td, lp, ent = hip.DeviceBuffer.from_array(tokens), hip.DeviceBuffer(8), hip.DeviceBuffer(8)
    ids, tops = hip.DeviceBuffer(2 * 5 * 4), hip.DeviceBuffer(2 * 5 * 4)
    hip.check(hip.lib().cheetah_hip_logprobs(big.ptr, 1, 2, vocab, stride, td.ptr, 5, lp.ptr, ent.ptr, ids.ptr, tops.ptr))
    check((lp.download(np.float32), ent.download(np.float32), ids.download(np.uint32).reshape(2, 5),
           tops.download(np.float32).reshape(2, 5)), np.stack(rows), tokens, 5)


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
def test_rows_between_one_segment_and_many(hip, fmt):
    """Row counts where a row's segments go from many to two to one, in turn on
    one thread's workspace, which grows and is used again by fewer rows."""
    rng = np.random.default_rng(14)
    x, values = logits(rng, 600, 20011, 20011, fmt)
    tokens = rng.integers(0, 20011, 600).astype(np.uint32)
    for rows in (2, 256, 1, 128, 600, 257, 200, 3, 255, 64, 2):
        check(hip.logprobs(x[:rows], tokens[:rows], 7), values[:rows], tokens[:rows], 7)


def test_threads_call_at_once(hip):
    """Each thread's segments are counted in a workspace of its own."""
    import threading

    rng = np.random.default_rng(15)
    cases = []
    for i in range(4):
        x, values = logits(rng, 3 + 40 * i, 30011, 30011, "f32")
        cases.append((x, values, rng.integers(0, 30011, len(x)).astype(np.uint32)))
    got = [[] for _ in cases]

    def run(i):
        for _ in range(5):
            got[i].append(hip.logprobs(cases[i][0], cases[i][2], 9))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for results, (_, values, tokens) in zip(got, cases):
        for r in results:
            check(r, values, tokens, 9)


def test_the_same_bits_again(hip):
    rng = np.random.default_rng(12)
    x, _ = logits(rng, 5, 100003, 100003, "f32")
    tokens = rng.integers(0, 100003, 5).astype(np.uint32)
    a, b = (hip.logprobs(x, tokens, 64) for _ in range(2))
    for p, q in zip(a, b):
        assert np.array_equal(p.view(np.uint32), q.view(np.uint32))
