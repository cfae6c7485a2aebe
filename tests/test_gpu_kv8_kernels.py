"""Attention over an 8-bit cache: every kernel that a call may be served by, over
values that could spoil it. 256 KV heads hold the same rows (each has queries of its
own), so that a few rows are a block a CU: blocks of 8 rows, of 16, of one, two and
four waves of 32."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import TOL, make

pytestmark = pytest.mark.gpu

HEADS, OFFSET = 256, 170
ROWS = [1, 6, 9, 16, 27, 32, 50, 64, 100, 128]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def rows_of(rng, n, hd):
    k, v = ref.some_rows(rng, n, 1, hd)
    return k[:, 0], v[:, 0]


def caches(hip, rng, k, v):
    """The device's cache and the values that it holds (NaN as 0)."""
    n, hd = k.shape
    dev, cpu = make(hip, rng, n, HEADS, hd), ref.Cache(n, 1, hd)
    dev.append(np.tile(k, HEADS), np.tile(v, HEADS), 0)
    cpu.append(np.nan_to_num(k, posinf=0, neginf=0), np.nan_to_num(v, posinf=0, neginf=0), 0)
    return dev, *(x[:, 0] for x in cpu.values(0, n))


def attention64(q, k, v, window=0, sinks=0):
    """q [rows, HEADS, hd] -> the same, a row at a time."""
    out = np.empty(q.shape)
    p = np.arange(len(k))
    for i, x in enumerate(np.asarray(q, np.float64)):
        pos = OFFSET + i
        seen = (p <= pos) & ((p > pos - window) | (p < sinks) if window else True)
        s = x @ k[seen].T / np.sqrt(k.shape[1])
        w = np.exp(s - s.max(1, keepdims=True))
        out[i] = w @ v[seen] / w.sum(1, keepdims=True)
    return out


def attend(dev, q, window=0, sinks=0):
    return dev.attention(q.reshape(len(q), -1), HEADS, OFFSET, window, sinks).reshape(q.shape)


def near(got, want):
    """Each row against its own largest output."""
    return (np.abs(got - want).max((1, 2)) <= TOL * np.abs(want).max((1, 2))).all()


def queries(rng, rows, hd):
    return rng.standard_normal((rows, HEADS, hd)).astype(np.float32)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", ROWS)
def test_plain_and_windowed(hip, rows, hd):
    rng = np.random.default_rng(rows + hd)
    k, v = rows_of(rng, OFFSET + rows, hd)
    dev, k, v = caches(hip, rng, k, v)
    q = queries(rng, rows, hd)
    for window, sinks in [(0, 0), (1, 0), (45, 3), (100, 40)]:
        assert near(attend(dev, q, window, sinks), attention64(q, k, v, window, sinks)), (window, sinks)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", ROWS)
def test_nan_rows(hip, rows, hd):
    """Behind the last position, between sinks and window: they do not show. Inside
    the chunk: in the rows that see it alone."""
    rng = np.random.default_rng(rows + hd)
    k, v = rows_of(rng, OFFSET + rows + 70, hd)
    window, sinks = 90, 5
    bad = [*range(sinks, OFFSET + 1 - window), *range(OFFSET + rows, OFFSET + rows + 70)]
    k[bad] = v[bad] = np.nan
    at = OFFSET + rows // 2
    q = queries(rng, rows, hd)
    dev, ck, cv = caches(hip, rng, k, v)
    want = attention64(q, ck, cv, window, sinks)
    assert near(attend(dev, q, window, sinks), want)
    if rows > 1:
        k[at] = v[at] = np.nan
        dev, ck, cv = caches(hip, rng, k, v)
        got, want = attend(dev, q, window, sinks), attention64(q, ck, cv, window, sinks)
        sees = OFFSET + np.arange(rows) >= at
        assert np.isnan(got[sees]).all() and near(got[~sees], want[~sees])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", ROWS)
def test_a_nan_value_and_a_nan_query(hip, rows, hd):
    """In its element, and in its row and head."""
    rng = np.random.default_rng(rows + hd)
    k, v = rows_of(rng, OFFSET + rows, hd)
    v[33, hd - 3] = np.nan
    q = queries(rng, rows, hd)
    q[rows // 2, 17, 5], q[rows - 1, 200, hd - 1] = np.nan, -np.inf
    dev, k, v = caches(hip, rng, k, v)
    bad = np.zeros(q.shape, bool)
    bad[:, :, hd - 3] = bad[rows // 2, 17] = bad[rows - 1, 200] = True
    got, want = attend(dev, q), attention64(np.nan_to_num(q, neginf=0), k, v)
    assert np.isnan(got[bad]).all()
    assert near(np.where(bad, 0, got), np.where(bad, 0, want))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("what", ["spread 3", "spread 12", "spread 30", "spread 110", "zeros first", "zeros between",
                                  "zeros", "largest", "least"])
def test_scales(hip, rows, hd, what):
    """V's blocks of very different sizes, of zeros, near the largest number (of one
    sign: finite sums of weights times V would pass it) and at the least scale."""
    rng = np.random.default_rng(rows + hd + len(what))
    n = OFFSET + rows
    k, v = rows_of(rng, n, hd)
    block = np.arange(n) // 32
    if what.startswith("spread"):
        far = int(what.split()[1])
        e = rng.integers(-far, far + 1, block[-1] + 1)[block]
        v = (v.astype(np.float64) * 2.0 ** e[:, None]).astype(np.float32)
    elif what == "largest" or what == "least":
        v = (3e38 if what == "largest" else 2.0 ** -110) * rng.uniform(0.5, 1.0, v.shape)
        v = v.astype(np.float32)
    else:
        v[{"zeros first": block < 3, "zeros between": block % 2 == 1, "zeros": block >= 0}[what]] = 0
    q = queries(rng, rows, hd)
    dev, k, v = caches(hip, rng, k, v)
    got, want = attend(dev, q), attention64(q, k, v)
    assert np.isfinite(got).all() and near(got, want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-3, 30.0])
def test_queries_of_any_size(hip, rows, hd, size):
    """Rows that average all values, and rows of nearly one value each (their scores
    are 30 times as large, and so is a rounding of them)."""
    rng = np.random.default_rng(rows + hd)
    k, v = rows_of(rng, OFFSET + rows, hd)
    dev, k, v = caches(hip, rng, k, v)
    q = (size * queries(rng, rows, hd)).astype(np.float32)
    got, want = attend(dev, q), attention64(q, k, v)
    assert (np.abs(got - want).max((1, 2)) <= (30 if size > 1 else 1) * TOL * np.abs(want).max((1, 2))).all()
