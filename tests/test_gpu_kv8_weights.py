"""Attention over an 8-bit cache where weights differ by many powers of two: one key
far above a long tail (an attention sink), large values behind small weights. Each
row and head is measured by its own largest output."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import TOL, make

pytestmark = pytest.mark.gpu

# (q heads, KV heads, head dim, rows, offset, window, sinks): a token over short and
# long contexts and a window, blocks of 16 rows, chunks whose keys are split and not.
CALLS = [(4, 1, 128, 1, 3000, 0, 0), (14, 2, 64, 1, 575, 0, 0), (28, 4, 128, 1, 31999, 0, 0),
         (32, 8, 128, 1, 5999, 2048, 4), (32, 8, 128, 13, 1999, 0, 0), (5, 1, 64, 3, 1200, 0, 0),
         (14, 2, 64, 333, 0, 0, 0), (32, 8, 128, 512, 4096, 0, 0), (28, 4, 128, 1000, 1088, 1024, 16),
         (28, 4, 128, 300, 16000, 0, 0), (8, 8, 64, 700, 3000, 0, 0)]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def filled(hip, rng, call, k, v):
    _, kvh, hd, rows, offset, *_ = call
    n = offset + rows
    dev, cpu = make(hip, rng, n, kvh, hd), ref.Cache(n, kvh, hd)
    dev.append(k.reshape(n, -1), v.reshape(n, -1), 0)
    cpu.append(k, v, 0)
    return dev, cpu.values(0, n)


def check(call, dev, held, q, what=""):
    """Some rows of the call against 64 bits over what the cache holds."""
    q_heads, _, hd, rows, offset, window, sinks = call
    got = dev.attention(q.reshape(rows, -1), q_heads, offset, window, sinks).reshape(rows, q_heads, hd)
    for i in sorted({0, rows // 7, rows // 2, 2 * rows // 3, rows - 2, rows - 1} & set(range(rows))):
        want = ref.attention64(q[i].reshape(1, -1), *held, q_heads, offset + i, window, sinks).reshape(q_heads, hd)
        off, most = np.abs(got[i] - want).max(1), np.abs(want).max(1)
        assert (off <= TOL * most).all(), (what, i, off, most)


@pytest.mark.parametrize("value", [0.0, 0.02])
@pytest.mark.parametrize("call", CALLS)
def test_one_key_far_above_a_long_tail(hip, call, value):
    """The first position scores `gap` powers of two above the others, whose scores
    are equal or nearly so, and its value is small or zero: the output is the tail's.
    TOL holds: 22 bits of the query put up to 26 * 2^-22 = 6.2e-6 between the key and
    the tail, exponents of up to 26 in f32 2^-20 = 1e-6, a tail's weight of at least
    2^-18 in the wave of the key rounds by 2^-36, 4e-6 of it: 1.2e-5."""
    q_heads, kvh, hd, rows, offset, *_ = call
    rng = np.random.default_rng(rows + hd)
    n = offset + rows
    k, v = (rng.standard_normal((n, kvh, hd)).astype(np.float32) for _ in "kv")
    k[..., 0] = 0
    k[0] = 0
    k[0, :, 0] = 16
    v[0] *= np.float32(value)
    dev, held = filled(hip, rng, call, k, v)
    for gap in (8, 13, 18, 26):
        for spread in (0, 0.3):
            q = (spread * rng.standard_normal((rows, q_heads, hd))).astype(np.float32)
            q[..., 0] = gap * np.log(2) * np.sqrt(hd) / 16
            check(call, dev, held, q, (gap, spread))


@pytest.mark.parametrize("call", [c for c in CALLS if not c[5] and c[4]])
def test_keys_that_dominate_some_heads_in_mid_context(hip, call):
    """Keys of one value each at two thirds and at nine tenths of the context, far above
    the rest for some rows and heads of a tile and far below it for others: sums move to
    the later maxima and the tails on either side keep their weights (as above)."""
    q_heads, kvh, hd, rows, offset, *_ = call
    rng = np.random.default_rng(rows + hd)
    n = offset + rows
    k, v = (rng.standard_normal((n, kvh, hd)).astype(np.float32) for _ in "kv")
    k[..., :2] = 0
    for c, at in enumerate((offset * 2 // 3, offset * 9 // 10)):
        k[at] = 0
        k[at, :, c] = 16
        v[at] = 0
    dev, held = filled(hip, rng, call, k, v)
    q = (0.3 * rng.standard_normal((rows, q_heads, hd))).astype(np.float32)
    gap = rng.integers(-26, 25, (rows, q_heads))
    q[..., 0] = gap * np.log(2) * np.sqrt(hd) / 16
    q[..., 1] = (gap + 2) * np.log(2) * np.sqrt(hd) / 16
    check(call, dev, held, q)


@pytest.mark.parametrize("call", CALLS)
def test_large_values_behind_small_weights(hip, call):
    """Every fourth block scores 25 powers of two below the others and holds values
    2^18 times theirs: some 2^-8 of the outputs is theirs (weights of 2^-17 that round
    by 2^-36: 2^-19 of that)."""
    q_heads, kvh, hd, rows, offset, *_ = call
    rng = np.random.default_rng(rows + hd)
    n = offset + rows
    k, v = (rng.standard_normal((n, kvh, hd)).astype(np.float32) for _ in "kv")
    far = np.arange(n) // 32 % 4 == 1
    k[..., 0] = 0
    k[far, :, 0] = -16
    v[far] *= 2.0 ** 18
    q = (0.3 * rng.standard_normal((rows, q_heads, hd))).astype(np.float32)
    q[..., 0] = 25 * np.log(2) * np.sqrt(hd) / 16
    check(call, *filled(hip, rng, call, k, v), q)


# 256 KV heads of the same rows: a few rows are a block a CU, whose waves see every 8th,
# 4th, 2nd or each block of positions. Blocks of 8 rows, of 16, of one, two and four
# waves of 32.
HEADS = 256


def alike(hip, rng, k, v, rows, hd, far):
    """Attention of the last `rows` of the positions, rows of queries whose channel 0
    puts `far` powers of two between k's of 16 and -16, and its 64 bits."""
    n = len(k)
    dev, cpu = make(hip, rng, n, HEADS, hd), ref.Cache(n, 1, hd)
    dev.append(np.tile(k, HEADS), np.tile(v, HEADS), 0)
    cpu.append(k, v, 0)
    q = (0.3 * rng.standard_normal((rows, HEADS, hd))).astype(np.float32)
    q[..., 0] = far * np.log(2) * np.sqrt(hd) / 32
    got = dev.attention(q.reshape(rows, -1), HEADS, n - rows).reshape(q.shape)
    ck, cv = (x[:, 0] for x in cpu.values(0, n))
    want = np.empty(q.shape)
    for i, x in enumerate(q.astype(np.float64)):
        s = x @ ck[:n - rows + i + 1].T / np.sqrt(hd)
        w = np.exp(s - s.max(1, keepdims=True))
        want[i] = w @ cv[:n - rows + i + 1] / w.sum(1, keepdims=True)
    return got, want


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 16, 32, 64, 128])
@pytest.mark.parametrize("sizes", [(-90, 0, 90), (-60, -20, 60), (-9, 0, 9), (90, 0, -90), (0, -200, 0), (-200, 0, 0)])
def test_values_that_grow_and_shrink_in_steps(hip, rows, hd, sizes):
    """The first eight blocks hold values of one size and all of the weight, the next
    eight and the rest others (2^-200: zeros), whose weights are 2^-300: none of it shows,
    in whatever steps a wave's sums change their unit. Scores are +-150 powers of two, so
    each of the hd sums that make one rounds by up to 2^-17 (half of the last bit of 128 to
    256), 2^-17 sqrt(hd / 3) at random, times ln 2 in the weight: 2.0e-5 (hd 64) and 3.4e-5
    of a weight, as much of an output, at most three deviations of it 1e-4 = 5 TOL."""
    rng = np.random.default_rng(rows + hd)
    n = 1120 + rows
    k, v = (rng.standard_normal((n, hd)).astype(np.float32) for _ in "kv")
    block = np.arange(n) // 32
    k[:, 0] = np.where(block < 8, 16, -16)
    v = (v.astype(np.float64) * 2.0 ** np.array(sizes)[np.minimum(block // 8, 2)][:, None]).astype(np.float32)
    got, want = alike(hip, rng, k, v, rows, hd, 300)
    if sizes[0] == -200:  # the weight is all on values of 0
        assert (got == 0).all()
        return
    assert (np.abs(got - want).max(2) <= 5 * TOL * np.abs(want).max(2)).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 16, 32, 64, 128])
def test_large_queries_over_tiny_keys_computed_again(hip, rows, hd):
    """Values near the largest, so that every row is computed again (their sums pass the
    type's range), and queries of 2^122 over keys near the least: products of codes and
    queries pass it too, those of values do not. Channels 0 and 1 cancel exactly."""
    rng = np.random.default_rng(rows + hd)
    n = 300 + rows
    k = (rng.standard_normal((n, hd)) * 2.0 ** -117).astype(np.float32)
    k[:, :2] = 64 * 2.0 ** -117
    v = (3e38 * rng.uniform(0.5, 1.0, (n, hd))).astype(np.float32)
    dev, cpu = make(hip, rng, n, HEADS, hd), ref.Cache(n, 1, hd)
    dev.append(np.tile(k, HEADS), np.tile(v, HEADS), 0)
    cpu.append(k, v, 0)
    q = (2.0 ** 117 * rng.standard_normal((rows, HEADS, hd))).astype(np.float32)
    q[..., 0], q[..., 1] = 2.0 ** 122, -2.0 ** 122
    got = dev.attention(q.reshape(rows, -1), HEADS, n - rows).reshape(q.shape)
    ck, cv = (x[:, 0] for x in cpu.values(0, n))
    for i, x in enumerate(q.astype(np.float64)):
        s = x @ ck[:n - rows + i + 1].T / np.sqrt(hd)
        w = np.exp(s - s.max(1, keepdims=True))
        want = w @ cv[:n - rows + i + 1] / w.sum(1, keepdims=True)
        assert (np.abs(got[i] - want).max(1) <= TOL * np.abs(want).max(1)).all()
