"""Log probabilities and entropies at bars of the kernel's own roundings.

A term e^d, d = x - M <= 0: d is rounded to 2^-24 of itself, as are log2(e) and
their product, which moves the term by 3 * 2^-24 |d| e^d <= 3 * 2^-24 * 0.37; its
exponential is off by at most 2^-23. As if all erred one way: 1.9e-7 of the sum. A
thread adds up to 16 terms of a chunk in f32, 15 * 2^-24 at most, but 256 threads'
sums and more are joined in 64 bits and their roundings are independent: 2^-24 *
sqrt(15) / 16 = 1.4e-8, three deviations 4.3e-8. Together below 2^-22. Each rise of
a thread's maximum scales its sums by one more exponential, another 2^-23 (and 2^-24
|d|) of what was there before. Results are rounded to f32 once."""
import numpy as np
import pytest

from cheetah_amd import synth

pytestmark = pytest.mark.gpu

SUM, RISE = 2.0**-22, 2.0**-22  # of the sums; of them for each rise at most


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def check(hip, x, values, rises):
    rows, vocab = values.shape
    tokens = np.random.default_rng(3).integers(0, vocab, rows).astype(np.uint32)
    lp, entropy, ids, tops = hip.logprobs(x, tokens, 4)
    v = values.astype(np.float64)
    d = v - v.max(1, keepdims=True)
    e = np.exp(d)
    total = e.sum(1)
    exact = d - np.log(total)[:, None]
    bar = SUM + rises * RISE
    want = exact[np.arange(rows), tokens]
    assert (np.abs(lp - want) <= bar + 2.0**-24 * np.abs(want)).all()
    order = np.argsort(-values, axis=1, kind="stable")[:, :4]
    assert np.array_equal(ids, order)
    want = np.take_along_axis(exact, order, 1)
    assert (np.abs(tops - want) <= bar + 2.0**-24 * np.abs(want)).all()
    # H = log Z + sum e^d (-d) / Z, positive terms: either sum within the bar, the
    # second also by its factor d's rounding, 2^-24.
    want = np.log(total) - (e * d).sum(1) / total
    assert (np.abs(entropy - want) <= 2 * bar * (1 + want) + 2.0**-23 * want).all()


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (5, 32003), (64, 128256), (300, 32000), (600, 50001)])
def test_ordinary_logits(hip, rows, vocab, fmt):
    """A thread's maximum rises log(chunks) times, by logits of little weight by
    then: at most two of the rises count whole."""
    x = (np.random.default_rng(vocab).standard_normal((rows, vocab)) * 3).astype(np.float32)
    if fmt == "bf16":
        x = synth.f32_to_bf16(x)
        check(hip, x, synth.bf16_to_f32(x).reshape(x.shape), 2)
    else:
        check(hip, x, x, 2)


@pytest.mark.parametrize("rows", [1, 40, 300, 600])
@pytest.mark.parametrize("step", [1e-6, 1e-4])
def test_logits_that_rise_in_every_chunk(hip, step, rows):
    """Every chunk of 4,096 raises every thread's maximum a little (0.004, 0.4):
    16 rises of a segment's sums, one when it is joined with others."""
    vocab = 65536
    x = (np.arange(vocab) * np.float32(step)).astype(np.float32) * np.ones((rows, 1), np.float32)
    check(hip, x, x, 17)
