"""Attention over an 8-bit cache where values could spoil it: NaN codes in rows
that a query does not see and in rows that it does, values near the type's
largest and smallest, scales far apart, large and tiny queries."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import TOL, filled, make, rel_err

pytestmark = pytest.mark.gpu

# One split, several, two rows (8 with their heads), and many rows (shared tiles).
SHAPES = [(1, 40), (1, 700), (1, 5000), (2, 45), (2, 600), (9, 300), (70, 1500), (300, 200)]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def poison(dev, positions):
    """NaN codes in K and V at the positions."""
    codes, hd = [b.download(np.uint8).reshape(dev.codes_shape) for b in dev._codes], dev.head_dim
    for p in positions:
        page, sub, i = dev.table[p // dev.page_size], p % dev.page_size // 32, p % 32
        k = codes[0][page, :, sub].reshape(dev.kv_heads, hd // 32, 32, 32)
        k[:, :, i] = 0x7F
        v = codes[1][page, :, sub].reshape(dev.kv_heads, hd, 32)
        v[:, :, i] = 0xFF
    for b, c in zip(dev._codes, codes):
        b.upload(c)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,offset", SHAPES)
def test_rows_that_nobody_sees_may_hold_nan(hip, rows, offset, hd):
    """Behind the last position, before a window and between sinks and window."""
    rng, dev, cpu = filled(hip, rows + offset + hd, offset + rows + 100, 2, hd)
    q = rng.standard_normal((rows, 8 * hd)).astype(np.float32)
    window, sinks = max(1, offset // 3), 5
    lo = offset + 1 - window
    poison(dev, [*range(sinks, lo), *range(offset + rows, offset + rows + 100)])
    want = ref.attention64(q, *cpu.values(0, offset + rows), 8, offset, window, sinks)
    assert rel_err(dev.attention(q, 8, offset, window, sinks), want) < TOL


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,offset", [s for s in SHAPES if s[0] > 1])
def test_a_nan_row_shows_in_the_rows_that_see_it_alone(hip, rows, offset, hd):
    """A NaN position inside the chunk: earlier rows are as without it, the rows
    whose window holds it are NaN, later ones are as without it again."""
    rng, dev, cpu = filled(hip, rows + offset + hd, offset + rows, 2, hd)
    q = rng.standard_normal((rows, 8 * hd)).astype(np.float32)
    window, at = rows // 3 + 1, offset + rows // 3
    want = ref.attention64(q, *cpu.values(0, offset + rows), 8, offset, window, 3)
    poison(dev, [at])
    got = dev.attention(q, 8, offset, window, 3)
    pos = offset + np.arange(rows)
    sees = (pos >= at) & (pos - window < at)
    assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all()
    assert rel_err(got[~sees], want[~sees]) < TOL


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,offset", SHAPES)
def test_a_nan_value_shows_in_its_element(hip, rows, offset, hd):
    """One NaN in V in the prefix: that element of every row, and no other."""
    rng = np.random.default_rng(rows + offset)
    k, v = ref.some_rows(rng, offset + rows, 2, hd)
    v[offset // 2, 1, 37] = np.nan
    dev, cpu = make(hip, rng, offset + rows, 2, hd), ref.Cache(offset + rows, 2, hd)
    dev.append(k, v, 0)
    cpu.append(k, np.nan_to_num(v), 0)
    q = rng.standard_normal((rows, 8 * hd)).astype(np.float32)
    got = dev.attention(q, 8, offset).reshape(rows, 8, hd)
    want = ref.attention64(q, *cpu.values(0, offset + rows), 8, offset).reshape(rows, 8, hd)
    hit = np.zeros((8, hd), bool)
    hit[4:, 37] = True
    assert np.isnan(got[:, hit]).all()
    assert rel_err(got[:, ~hit], want[:, ~hit]) < TOL


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,offset", SHAPES)
@pytest.mark.parametrize("size", [3e38, 2.0 ** 90, 2.0 ** -100])
def test_values_of_any_size_average(hip, rows, offset, hd, size):
    """Finite V of one sign near the largest: finite averages (the weights' sum
    times V would pass the largest number); and tiny ones."""
    rng = np.random.default_rng(rows + offset)
    k, v = ref.some_rows(rng, offset + rows, 2, hd)
    v = (size * rng.uniform(0.5, 1.0, v.shape)).astype(np.float32)
    dev, cpu = make(hip, rng, offset + rows, 2, hd), ref.Cache(offset + rows, 2, hd)
    dev.append(k, v, 0)
    cpu.append(k, v, 0)
    q = rng.standard_normal((rows, 8 * hd)).astype(np.float32)
    want = ref.attention64(q, *cpu.values(0, offset + rows), 8, offset)
    got = dev.attention(q, 8, offset)
    assert np.isfinite(got).all() and rel_err(got, want) < TOL


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,offset", SHAPES)
@pytest.mark.parametrize("spread", [3, 12, 30, 110])
def test_scales_far_apart(hip, rows, offset, hd, spread):
    """Blocks whose V differ by powers of two up to 2^spread either way, in any
    order; each row's own outputs are its measure, dominated by the largest."""
    rng = np.random.default_rng(rows + offset + spread)
    total = offset + rows
    k, v = ref.some_rows(rng, total, 2, hd)
    e = rng.integers(-spread, spread + 1, -(-total // 32)).repeat(32)[:total]
    v = (v.astype(np.float64) * 2.0 ** e[:, None, None]).astype(np.float32)
    dev, cpu = make(hip, rng, total, 2, hd), ref.Cache(total, 2, hd)
    dev.append(k, v, 0)
    cpu.append(k, v, 0)
    q = rng.standard_normal((rows, 8 * hd)).astype(np.float32)
    want = ref.attention64(q, *cpu.values(0, total), 8, offset)
    got = dev.attention(q, 8, offset)
    off = np.abs(got - want).max(1) / np.abs(want).max(1)
    assert off.max() < TOL


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,offset", SHAPES)
@pytest.mark.parametrize("zero", ["first", "last", "every other", "all"])
def test_blocks_of_zeros(hip, rows, offset, hd, zero):
    """A block of zeros has the least scale, far from the others'."""
    rng = np.random.default_rng(rows + offset)
    total = offset + rows
    k, v = ref.some_rows(rng, total, 2, hd)
    block = np.arange(total) // 32
    at = {"first": block < 9, "last": block >= block[-1] - 1, "every other": block % 2 == 1, "all": block >= 0}[zero]
    v[at] = 0
    dev, cpu = make(hip, rng, total, 2, hd), ref.Cache(total, 2, hd)
    dev.append(k, v, 0)
    cpu.append(k, v, 0)
    q = rng.standard_normal((rows, 8 * hd)).astype(np.float32)
    want = ref.attention64(q, *cpu.values(0, total), 8, offset)
    assert np.abs(dev.attention(q, 8, offset) - want).max() <= TOL * np.abs(want).max()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,offset", [(1, 40000), (200, 20000)])
def test_the_least_scale_under_many_positions(hip, rows, offset, hd):
    """Weights' sums of 2^15 and values of the least scale: quotients keep their
    bits (2^-110 or so, while a unit over the sum is no normal number)."""
    rng = np.random.default_rng(rows + offset)
    k, v = ref.some_rows(rng, offset + rows, 1, hd)
    v = (2.0 ** -110 * rng.uniform(0.5, 1.0, v.shape)).astype(np.float32)
    dev, cpu = make(hip, rng, offset + rows, 1, hd), ref.Cache(offset + rows, 1, hd)
    dev.append(k, v, 0)
    cpu.append(k, v, 0)
    q = (2.0 ** -8 * rng.standard_normal((rows, 4 * hd))).astype(np.float32)
    want = ref.attention64(q, *cpu.values(0, offset + rows), 4, offset)
    assert rel_err(dev.attention(q, 4, offset), want) < TOL


@pytest.mark.parametrize("rows,offset", [(1, 700), (70, 100)])
@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-20, 1e-3, 30.0])
def test_queries_of_any_size(hip, rows, offset, size):
    """Rows of zeros and tiny ones average all values; rows of large ones are
    nearly one value each."""
    rng, dev, cpu = filled(hip, rows + offset, offset + rows, 2, 128)
    q = (size * rng.standard_normal((rows, 8 * 128))).astype(np.float32)
    want = ref.attention64(q, *cpu.values(0, offset + rows), 8, offset)
    assert rel_err(dev.attention(q, 8, offset), want) < TOL


def test_keys_of_any_size(hip):
    """Scores past f32's range are infinities: the row whose products overflow
    is the formula's, the others are as they are."""
    rng = np.random.default_rng(9)
    k, v = ref.some_rows(rng, 200, 1, 64)
    dev, cpu = make(hip, rng, 200, 1, 64), ref.Cache(200, 1, 64)
    k = (k * 2.0 ** 60).astype(np.float32)
    dev.append(k, v, 0)
    cpu.append(k, v, 0)
    q = (rng.standard_normal((3, 4 * 64)) * 2.0 ** -60).astype(np.float32)
    q[1] = 0
    want = ref.attention64(q, *cpu.values(0, 200), 4, 197)
    assert rel_err(dev.attention(q, 4, 197), want) < TOL
    q[2] = 3e38
    got = dev.attention(q, 4, 197)
    assert rel_err(got[:2], want[:2]) < TOL and not np.isfinite(got[2]).any()


def test_a_query_with_nan_or_infinity_is_nan_alone(hip):
    rng, dev, cpu = filled(hip, 21, 320, 2, 128)
    q = rng.standard_normal((20, 8 * 128)).astype(np.float32)
    want = ref.attention64(q, *cpu.values(0, 320), 8, 300).reshape(20, 8, 128)
    q.reshape(20, 8, 128)[3, 2, 5] = np.nan
    q.reshape(20, 8, 128)[7, 6, 100] = np.inf
    got = dev.attention(q, 8, 300).reshape(20, 8, 128)
    bad = np.zeros((20, 8), bool)
    bad[3, 2] = bad[7, 6] = True
    assert np.isnan(got[bad]).all() and rel_err(got[~bad], want[~bad]) < TOL


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,offset", SHAPES)
def test_a_nan_whose_weight_rounds_to_zero_shows(hip, rows, offset, hd):
    """The key of one position scores hundreds below the others for every row: its
    weight is 0, in its own split too, and its NaN value shows all the same."""
    rng = np.random.default_rng(rows + offset + hd)
    k, v = ref.some_rows(rng, offset + rows, 1, hd)
    at = offset // 3
    k[:, :, 0] = 8
    k[at] = 0
    k[at, :, 0] = -300
    v[at, 0, 5] = np.nan
    q = rng.standard_normal((rows, 4 * hd)).astype(np.float32)
    q.reshape(rows, 4, hd)[:, :, 0] = 30
    dev, cpu = make(hip, rng, offset + rows, 1, hd), ref.Cache(offset + rows, 1, hd)
    dev.append(k, v, 0)
    cpu.append(k, np.nan_to_num(v), 0)
    got = dev.attention(q, 4, offset).reshape(rows, 4, hd)
    want = ref.attention64(q, *cpu.values(0, offset + rows), 4, offset).reshape(rows, 4, hd)
    assert np.isnan(got[:, :, 5]).all()
    clean = np.arange(hd) != 5
    assert rel_err(got[:, :, clean], want[:, :, clean]) < 2 * TOL  # scores of 30 * 8 / 8 more, of 2^-21 each
