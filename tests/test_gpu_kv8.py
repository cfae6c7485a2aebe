"""The 8-bit K/V cache on the device: codes, scales and attention against their
64-bit restatement."""
import ctypes

import numpy as np
import pytest

import kv8_reference as ref
from cheetah_amd import synth

pytestmark = pytest.mark.gpu

# Codes are exact operands; queries and probabilities carry at least 21 bits
# (2^-22 each after rounding), products are exact in f32, sums are f32: of 6,000
# keys' weights at most 6,000 roundings of 2^-25 at random, 5e-6 of the largest
# output at two deviations, exponentials add 2^-22: 2e-5.
TOL = 2e-5


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def rel_err(got, want):
    return float(np.max(np.abs(got.astype(np.float64) - want)) / np.max(np.abs(want)))


def make(hip, rng, positions, kvh, hd, page=64):
    """A device cache with shuffled pages, some of the pool's never listed."""
    pages = -(-positions // page) + 2
    return hip.Kv8Cache(positions, kvh, hd, page, rng.permutation(pages)[:pages - 2], pages)


def filled(hip, seed, positions, kvh, hd, page=64):
    rng = np.random.default_rng(seed)
    k, v = ref.some_rows(rng, positions, kvh, hd)
    dev, cpu = make(hip, rng, positions, kvh, hd, page), ref.Cache(positions, kvh, hd)
    dev.append(k, v, 0)
    cpu.append(k, v, 0)
    return rng, dev, cpu


def same(dev, cpu, begin, n):
    for got, want in zip(dev.read(begin, n), cpu.values(begin, n)):
        np.testing.assert_array_equal(got, want)


PIECES = [[1], [31], [32], [33], [64, 1], [5, 1, 1, 40], [30, 2, 32, 1], [100, 7, 150], [1] * 40, [17] * 9]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kvh,hd", [(2, 64), (8, 128), (1, 128), (3, 64)])
@pytest.mark.parametrize("pieces", PIECES)
def test_rows_come_back_as_written(hip, pieces, kvh, hd, bf16):
    """Appends of every alignment, the later ones larger and smaller: the values
    are those of the definition, bit for bit, in both types."""
    rng = np.random.default_rng(sum(pieces) * hd + kvh)
    total = sum(pieces)
    dev, cpu = make(hip, rng, total, kvh, hd), ref.Cache(total, kvh, hd)
    at = 0
    for i, n in enumerate(pieces):
        k, v = ref.some_rows(rng, n, kvh, hd)
        k, v = k * np.float32(3.0 ** (i % 5 - 1)), v * np.float32(7.0 ** (i % 4 - 2))
        if bf16:
            kb, vb = synth.f32_to_bf16(k), synth.f32_to_bf16(v)
            k, v = synth.bf16_to_f32(kb).reshape(k.shape), synth.bf16_to_f32(vb).reshape(v.shape)
            dev.append(kb, vb, at)
        else:
            dev.append(k, v, at)
        cpu.append(k, v, at)
        at += n
        same(dev, cpu, 0, at)
    for begin in {0, total // 3, total - 1}:
        same(dev, cpu, begin, total - begin)
        for got, want in zip(dev.read(begin, total - begin, bf16=True), cpu.values(begin, total - begin)):
            np.testing.assert_array_equal(synth.bf16_to_f32(got).reshape(want.shape), want)


def test_every_code_and_every_scale(hip):
    """A block of all finite codes' values under scales over the whole range
    comes back unchanged; so do the values half a step off, rounded."""
    values = ref.code_values()
    row = np.zeros(256)
    row[:254] = values[[c for c in range(256) if c & 127 != 127]]
    x = np.tile(row.reshape(4, 64), (8, 1))
    for e in (-117, -116, -60, -1, 0, 1, 59, 118, 119):
        dev, cpu = hip.Kv8Cache(64, 1, 64), ref.Cache(64, 1, 64)
        k = (x * 2.0 ** e).astype(np.float32)
        v = (x * (1 + 2.0 ** -4) * 2.0 ** (e - 1)).astype(np.float32)
        dev.append(k, v, 0)
        cpu.append(k, v, 0)
        got = dev.read(0, 32)
        np.testing.assert_array_equal(got[0].reshape(-1), k.reshape(-1))
        same(dev, cpu, 0, 32)


def test_the_largest_and_smallest_magnitudes(hip):
    """Magnitudes past the largest scale saturate, tiny ones round under the
    smallest, zeros stay zeros; infinities and NaN are NaN and leave their
    neighbours alone."""
    rng = np.random.default_rng(5)
    big = rng.choice([3.3e38, -3.4e38, 1e38, 1.0], (32, 64)).astype(np.float32)
    tiny = (rng.standard_normal((32, 64)) * 2.0 ** -125).astype(np.float32)
    odd = rng.standard_normal((32, 64)).astype(np.float32)
    odd[3, 7], odd[9, 1], odd[30, 63] = np.inf, -np.inf, np.nan
    dev, cpu = hip.Kv8Cache(128, 1, 64), ref.Cache(128, 1, 64)
    k, v = np.concatenate([big, tiny, odd, np.zeros_like(odd)]), np.concatenate([tiny, odd, big, odd])
    dev.append(k, v, 0)
    cpu.append(k, v, 0)
    same(dev, cpu, 0, 128)


def test_rows_behind_the_last_keep_their_codes(hip):
    """Appending over the middle of written blocks leaves the codes behind it
    and every other block's bytes."""
    _, dev, cpu = filled(hip, 3, 200, 2, 128)
    before = dev.codes()
    rng = np.random.default_rng(4)
    k, v = ref.some_rows(rng, 41, 2, 128)
    dev.append(k, v, 70)
    after = dev.codes()
    for t, (a, b) in enumerate(zip(before[:2], after[:2])):
        a, b = (x.reshape(*x.shape[:3], -1) for x in (a, b))
        for blk in range(7):
            page, sub = dev.table[blk // 2], blk % 2
            x, y = a[page, :, sub], b[page, :, sub]
            if t == 0:
                x, y = (w.reshape(2, 4, 32, 32).swapaxes(1, 2).reshape(2, 32, 128) for w in (x, y))
            else:
                x, y = (w.reshape(2, 128, 32).swapaxes(1, 2) for w in (x, y))
            pos = blk * 32 + np.arange(32)
            np.testing.assert_array_equal(x[:, pos >= 111], y[:, pos >= 111])
            np.testing.assert_array_equal(x[:, pos < 64], y[:, pos < 64])
    cpu.append(k, v, 70)
    same(dev, cpu, 0, 111)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("shift,stride", [(0, 384), (1, 384), (0, 381), (3, 129), (4, 256)])
def test_rows_out_of_packed_projections(hip, shift, stride, f32):
    """K and V rows inside wider rows, aligned for wide loads or not."""
    rng = np.random.default_rng(shift + stride)
    n, kvh, hd = 45, 2, 64
    x = rng.standard_normal(n * stride * 2 + 64).astype(np.float32)
    bits = x if f32 else synth.f32_to_bf16(x)
    x = x if f32 else synth.bf16_to_f32(bits)
    buf = hip.DeviceBuffer.from_array(bits)
    dev, cpu = hip.Kv8Cache(100, kvh, hd), ref.Cache(100, kvh, hd)
    size, v0 = bits.itemsize, n * stride
    hip.check(hip.lib().cheetah_hip_kv8_append(buf.ptr + shift * size, buf.ptr + (shift + v0) * size, int(f32), n, stride,
                                               0, ctypes.byref(dev.view)))
    at = np.arange(n)[:, None] * stride + np.arange(kvh * hd)
    cpu.append(x[shift + at], x[shift + v0 + at], 0)
    same(dev, cpu, 0, n)


LAYOUTS = [(14, 2, 64), (32, 8, 128), (28, 4, 128), (5, 1, 64), (3, 3, 128), (16, 2, 64), (6, 2, 128), (6, 1, 64)]


@pytest.mark.parametrize("q_heads,kvh,hd", LAYOUTS)
@pytest.mark.parametrize("rows,offset", [(1, 0), (1, 31), (1, 300), (2, 63), (3, 1), (7, 64), (16, 500), (33, 95), (70, 130)])
def test_attention_matches_64_bits(hip, q_heads, kvh, hd, rows, offset):
    rng, dev, cpu = filled(hip, rows * 1000 + offset + q_heads, offset + rows, kvh, hd)
    q = rng.standard_normal((rows, q_heads * hd)).astype(np.float32)
    got = dev.attention(q, q_heads, offset)
    assert rel_err(got, ref.attention64(q, *cpu.values(0, offset + rows), q_heads, offset)) < TOL


@pytest.mark.parametrize("q_heads,kvh,hd", [(32, 8, 128), (7, 1, 64)])
@pytest.mark.parametrize("rows,offset", [(1, 6000), (1, 2047), (5, 4099), (31, 0), (40, 1000), (130, 700), (257, 1500),
                                         (520, 64), (1, 1024), (12, 3000)])
def test_attention_sizes(hip, q_heads, kvh, hd, rows, offset):
    rng, dev, cpu = filled(hip, rows + offset, offset + rows, kvh, hd)
    q = rng.standard_normal((rows, q_heads * hd)).astype(np.float32)
    got = dev.attention(q, q_heads, offset)
    assert rel_err(got, ref.attention64(q, *cpu.values(0, offset + rows), q_heads, offset)) < TOL


@pytest.mark.parametrize("q_heads,kvh,hd", [(14, 2, 64), (8, 2, 128), (28, 4, 128)])
@pytest.mark.parametrize("rows,offset,window,sinks", [
    (1, 500, 1, 0), (1, 500, 1, 1), (1, 500, 32, 4), (1, 511, 64, 32), (1, 500, 500, 3), (1, 500, 501, 0),
    (1, 500, 10**9, 7), (1, 3000, 700, 100), (9, 500, 5, 0), (9, 500, 5, 2), (40, 0, 7, 3), (40, 0, 1, 0),
    (50, 333, 33, 31), (130, 700, 64, 5), (130, 700, 300, 650), (64, 1024, 2, 1000), (200, 100, 2000, 5),
    (300, 2000, 128, 33), (1, 0, 1, 5), (1, 4096, 4096, 4)])
def test_windows_and_sinks_match_64_bits(hip, q_heads, kvh, hd, rows, offset, window, sinks):
    """Windows from one position to all of them, sinks that end inside a block,
    inside the window or past it; pages that nobody sees are not listed."""
    rng, dev, cpu = filled(hip, rows + offset + window % 1000 + sinks, offset + rows, kvh, hd)
    q = rng.standard_normal((rows, q_heads * hd)).astype(np.float32)
    first = max(0, offset + 1 - window)
    gone = [p for p in range(dev.table.size) if p * 64 >= min(sinks, first) and (p + 1) * 64 <= first]
    table = dev.table.copy()
    table[gone] = -(2**31)
    dev._table.upload(table)
    got = dev.attention(q, q_heads, offset, window, sinks)
    want = ref.attention64(q, *cpu.values(0, offset + rows), q_heads, offset, window, sinks)
    assert rel_err(got, want) < TOL


@pytest.mark.parametrize("page", [128, 192, 512])
def test_larger_pages(hip, page):
    rng, dev, cpu = filled(hip, page, 800, 2, 128, page)
    same(dev, cpu, 0, 800)
    q = rng.standard_normal((20, 8 * 128)).astype(np.float32)
    want = ref.attention64(q, *cpu.values(0, 797), 8, 777)
    assert rel_err(dev.attention(q, 8, 777), want) < TOL


def test_pools_past_four_gigabytes(hip):
    """Pages whose codes lie past 2^32 bytes (and, of V, past 2^31 from the first):
    the values and outputs of a cache with small offsets."""
    kvh, hd, pages, n = 8, 128, 70000, 300
    table = np.array([69999, 3, 65541, 40000, 69001], np.int32)
    codes = [hip.DeviceBuffer(pages * kvh * 64 * hd) for _ in "kv"]
    scales = [hip.DeviceBuffer(pages * kvh * 2) for _ in "kv"]
    t = hip.DeviceBuffer.from_array(table)
    far = hip.Kv8Cache.__new__(hip.Kv8Cache)
    far.table, far.page_size, far.kv_heads, far.head_dim = table, 64, kvh, hd
    far.view = hip.Kv8View(*(b.ptr for b in codes + scales), t.ptr, 64, kvh, hd)
    rng = np.random.default_rng(8)
    near, cpu = make(hip, rng, n, kvh, hd), ref.Cache(n, kvh, hd)
    for at, some in ((0, 170), (170, 1), (171, 129)):
        k, v = ref.some_rows(rng, some, kvh, hd)
        for cache in (far, near, cpu):
            cache.append(k, v, at)
    same(far, cpu, 0, n)
    for rows in (1, 100):
        q = rng.standard_normal((rows, 32 * hd)).astype(np.float32)
        np.testing.assert_array_equal(far.attention(q, 32, n - rows), near.attention(q, 32, n - rows))


def test_a_wave_with_more_blocks_than_lanes(hip):
    """256 KV heads leave each one block of waves, of which one takes more than 64
    blocks of positions, so page entries and scales are looked up again on the way.
    Every head has the same rows and queries of its own. (2e-5 has room for 16,600
    keys: their weights' roundings are 1.7 times those of 6,000.)"""
    rng, n, kvh, hd = np.random.default_rng(5), 16600, 256, 64
    k, v = ref.some_rows(rng, n, 1, hd)
    k, v = (synth.f32_to_bf16(x.reshape(n, hd)) for x in (k, v))
    dev, cpu = make(hip, rng, n, kvh, hd, 128), ref.Cache(n, 1, hd)
    for at in range(0, n, 3300):
        dev.append(np.tile(k[at:at + 3300], kvh), np.tile(v[at:at + 3300], kvh), at)
        cpu.append(*(synth.bf16_to_f32(x[at:at + 3300]) for x in (k, v)), at)
    k, v = (x[:, 0] for x in cpu.values(0, n))
    for rows, window in [(1, 0), (8, 0), (9, 0), (30, 0), (40, 0), (100, 0), (3, 16450)]:
        q = rng.standard_normal((rows, kvh * hd)).astype(np.float32)
        got = dev.attention(q, kvh, n - rows, window)
        for i in {0, rows // 3, rows // 2, rows - 1}:
            pos = n - rows + i
            seen = slice(max(pos + 1 - window, 0) if window else 0, pos + 1)
            s = q[i].astype(np.float64).reshape(kvh, hd) @ k[seen].T / np.sqrt(hd)
            w = np.exp(s - s.max(1, keepdims=True))
            want = (w @ v[seen] / w.sum(1, keepdims=True)).reshape(-1)
            assert rel_err(got[i], want) < TOL, (rows, window, i)


@pytest.mark.parametrize("q_heads,kvh,hd", [(4, 4, 64), (8, 4, 128), (12, 4, 64), (16, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("offset,window,sinks", [(0, 0, 0), (29, 0, 0), (700, 0, 0), (700, 5, 2), (3000, 1000, 40)])
def test_few_rows(hip, q_heads, kvh, hd, rows, offset, window, sinks):
    """Up to 8 query rows x heads of a group, and a few more."""
    rng, dev, cpu = filled(hip, rows + offset, offset + rows, kvh, hd)
    q = rng.standard_normal((rows, q_heads * hd)).astype(np.float32)
    want = ref.attention64(q, *cpu.values(0, offset + rows), q_heads, offset, window, sinks)
    assert rel_err(dev.attention(q, q_heads, offset, window, sinks), want) < TOL


def test_the_wrapper_refuses_positions_that_the_table_does_not_list(hip):
    cache = hip.Kv8Cache(200, 1, 64, table=np.array([2, 0, -1, 1], np.int64), pages=3)
    rows = np.zeros((10, 64), np.float32)
    cache.append(rows, rows, 100)
    for call in (lambda: cache.append(rows, rows, 120), lambda: cache.read(120, 10), lambda: cache.append(rows, rows, 250),
                 lambda: cache.attention(rows, 1, 140), lambda: cache.attention(rows, 1, 2**40)):
        with pytest.raises(ValueError, match="page table"):
            call()
    with pytest.raises(ValueError, match="outside the pool"):
        hip.Kv8Cache(100, 1, 64, table=np.array([2**32, 1]), pages=3)


def test_a_page_listed_twice_is_read_twice_and_written_once(hip):
    rng = np.random.default_rng(3)
    k, v = ref.some_rows(rng, 128, 1, 64)
    dev, cpu = hip.Kv8Cache(192, 1, 64, table=np.array([1, 0, 1]), pages=2), ref.Cache(192, 1, 64)
    dev.append(k, v, 0)
    cpu.append(k, v, 0)
    cpu.append(k[:64], v[:64], 128)
    same(dev, cpu, 0, 192)
    q = rng.standard_normal((5, 4 * 64)).astype(np.float32)
    assert rel_err(dev.attention(q, 4, 187), ref.attention64(q, *cpu.values(0, 192), 4, 187)) < TOL
    with pytest.raises(ValueError, match="a page twice"):
        dev.append(np.concatenate([k, k])[:192], np.concatenate([v, v])[:192], 0)


@pytest.mark.parametrize("order", [[0, 1, 2], [2, 1, 0]])
def test_calls_of_growing_and_shrinking_size_share_their_scratch(hip, order):
    """Calls with many splits, few and none, back to back on one stream: each is
    what it is alone, twice over."""
    shapes = [(1, 6000, 4, 28), (70, 900, 8, 32), (3, 40, 1, 5)]
    made = []
    for rows, offset, kvh, qh in shapes:
        rng, dev, _ = filled(hip, rows, offset + rows, kvh, 128)
        q = rng.standard_normal((rows, qh * 128)).astype(np.float32)
        made.append((dev, q, qh, offset, dev.attention(q, qh, offset)))
    for _ in range(2):
        for i in order:
            dev, q, qh, offset, want = made[i]
            np.testing.assert_array_equal(dev.attention(q, qh, offset), want)
