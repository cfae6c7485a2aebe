"""CPU-only: what the calls over an 8-bit K/V cache refuse, each with a sentence
and before any device work (the library is not initialized here)."""
import ctypes

import numpy as np
import pytest

import kv8_reference as ref

D = 4096  # stands for a device pointer; never dereferenced
FAR = 2**31 - 1 - 1023  # positions end here


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    return h


def refused(hip, rc, text):
    assert rc == -1
    assert text in hip.lib().cheetah_hip_last_error().decode()


def view(hip, **kw):
    a = dict(k=D, v=2 * D, ks=3 * D, vs=4 * D, table=5 * D, page=64, kvh=2, hd=64)
    a.update(kw)
    return hip.Kv8View(a["k"], a["v"], a["ks"], a["vs"], a["table"], a["page"], a["kvh"], a["hd"])


VIEWS = [(dict(k=None), "null pointer"), (dict(v=None), "null pointer"), (dict(ks=None), "null pointer"),
         (dict(vs=None), "null pointer"), (dict(table=None), "null pointer"), (dict(kvh=0), "out of range"),
         (dict(kvh=70000), "out of range"), (dict(page=2**32 - 64), "out of range"), (dict(page=0), "multiple of 64"),
         (dict(page=96), "multiple of 64"), (dict(hd=0), "head_dim 64 or 128"), (dict(hd=96), "head_dim 64 or 128"),
         (dict(k=D + 8), "aligned"), (dict(v=D + 2), "aligned"), (dict(table=D + 1), "aligned"),
         (dict(v=D), "same pool"), (dict(vs=3 * D), "same pool")]


def append(hip, kv, **kw):
    a = dict(k=D, v=D, fmt=1, rows=8, stride=128, offset=100)
    a.update(kw)
    return hip.lib().cheetah_hip_kv8_append(*a.values(), kv)


def read(hip, kv, **kw):
    a = dict(begin=100, n=8, fmt=1, k=D, v=D)
    a.update(kw)
    return hip.lib().cheetah_hip_kv8_read(kv, *a.values())


def attend(hip, kv, **kw):
    a = dict(q=D, q_heads=4, rows=8, offset=100, window=0, sinks=0, out=D)
    a.update(kw)
    return hip.lib().cheetah_hip_kv8_attention(a["q"], kv, a["q_heads"], a["rows"], a["offset"], a["window"],
                                               a["sinks"], a["out"])


@pytest.mark.parametrize("call", [append, read, attend])
def test_views_refused(hip, call):
    refused(hip, call(hip, None), "null pointer")
    for change, text in VIEWS:
        refused(hip, call(hip, ctypes.byref(view(hip, **change))), text)


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null pointer"), (dict(v=None), "null pointer"), (dict(fmt=2), "row_format"),
    (dict(rows=0), "at least one row"), (dict(rows=FAR - 99), "out of range"), (dict(offset=FAR - 7), "out of range"),
    (dict(offset=2**64 - 1), "out of range"), (dict(rows=2**64 - 1), "out of range"), (dict(stride=127), "stride"),
    (dict(stride=2**63), "stride"), (dict(k=D + 2), "misaligned"), (dict(v=D + 1, fmt=0), "misaligned")])
def test_append_refuses(hip, change, text):
    refused(hip, append(hip, ctypes.byref(view(hip)), **change), text)


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null pointer"), (dict(v=None), "null pointer"), (dict(fmt=2), "row_format"),
    (dict(n=0), "at least one row"), (dict(n=FAR - 99), "out of range"), (dict(begin=2**64 - 1), "out of range"),
    (dict(k=D + 8), "aligned"), (dict(v=D + 4), "aligned")])
def test_read_refuses(hip, change, text):
    refused(hip, read(hip, ctypes.byref(view(hip)), **change), text)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null pointer"), (dict(out=None), "null pointer"), (dict(rows=0), "at least one query row"),
    (dict(q_heads=0), "multiple of kv_heads"), (dict(q_heads=3), "multiple of kv_heads"),
    (dict(q_heads=1 << 31), "multiple of kv_heads"), (dict(q_heads=18), "1..8 query heads"),
    (dict(offset=FAR - 7), "out of range"), (dict(rows=2**64 - 1), "out of range"), (dict(sinks=1), "sinks"),
    (dict(q=D + 4), "aligned"), (dict(out=D + 8), "aligned")])
def test_attention_refuses(hip, change, text):
    refused(hip, attend(hip, ctypes.byref(view(hip)), **change), text)


def test_valid_arguments_reach_the_device_check(hip):
    if hip._initialized:
        pytest.skip("library already initialized in this process")
    kv = ctypes.byref(view(hip))
    for rc in (append(hip, kv, offset=FAR - 8), read(hip, kv, begin=FAR - 8), attend(hip, kv, offset=FAR - 8),
               attend(hip, kv, window=2**64 - 1, sinks=2**64 - 1)):
        refused(hip, rc, "not initialized")


def test_the_reference_rounds_to_nearest_even():
    """The oracle's codes: every value is its own code, midpoints go to the even
    one, a hair on either side to the nearer."""
    values = ref.code_values()
    at = np.array([c for c in range(256) if c & 127 != 127])
    assert (ref.encode(values[at]) == at).all()
    steps = values[:127]
    mid = (steps[1:] + steps[:-1]) / 2
    even = np.arange(126) + np.arange(126) % 2
    assert (ref.encode(mid) == even).all() and (ref.encode(-mid) == (even | 128)).all()
    assert (ref.encode(mid * (1 + 1e-9)) == np.arange(1, 127)).all()
    assert (ref.encode(mid * (1 - 1e-9)) == np.arange(126)).all()
    assert (ref.encode([500.0, -1e30, np.inf, np.nan]) == [0x7E, 0xFE, 0x7F, 0x7F]).all()


def test_the_reference_grows_a_scale_without_moving_normal_codes():
    """Rows one by one or all at once: values that are normal codes under the last
    scale (2^-6 of it; the largest is over 224 of it, 2^7.8) are equal. Others are
    rounded once more at every growth, half a step of 2^-9 each, the earlier ones
    under at most half the scale: a step apart in all, 2^-16.8 of the largest."""
    rng = np.random.default_rng(1)
    k, v = ref.some_rows(rng, 20, 1, 64)
    whole, pieces = ref.Cache(20, 1, 64), ref.Cache(20, 1, 64)
    k[13] *= 37
    whole.append(k, v, 0)
    for i in range(20):
        pieces.append(k[i:i + 1], v[i:i + 1], i)
    a, b = whole.values(0, 20)[0], pieces.values(0, 20)[0]
    most = np.abs(a).max()
    assert (np.abs(a - b)[np.abs(a) >= most * 2.0 ** -13] == 0).all() and np.abs(a - b).max() <= most * 2.0 ** -16.8


def wrapper(hip, table):
    """A cache's Python side alone, over a table."""
    cache = hip.Kv8Cache.__new__(hip.Kv8Cache)
    cache.table, cache.page_size, cache.kv_heads, cache.head_dim = np.asarray(table, np.int32), 64, 1, 64
    cache.view = view(hip, kvh=1)
    return cache


@pytest.mark.parametrize("kw", [dict(window=-1), dict(window=64, sinks=-1), dict(window=-64, sinks=3)])
def test_the_wrapper_refuses_negative_windows_and_sinks(hip, kw):
    """Taken as whole numbers without a sign they would reach every page, those that the
    table does not list among them."""
    cache = wrapper(hip, [-1, -1, 0, 1])
    with pytest.raises(ValueError, match="window"):
        cache.attention(np.zeros((1, 64), np.float32), 1, 200, **kw)
