"""Tree attention over infinities and values near the type's largest in V rows
that nodes see: the definition's infinity, or the finite average, whatever the
cache's type, the position and the number of splits."""
import numpy as np
import pytest

import tree_reference as ref
from cheetah_amd import synth

pytestmark = pytest.mark.gpu

# Rows that overflow on the matrix cores are averaged key by key in f32: 6,000
# weights' roundings of 2^-24 (the exponential 2^-22 once) at random and as many of
# the running sums, sqrt(12,000) 2^-24 = 6.6e-6 of the largest V they average, three
# deviations. Averages of one sign are at least a quarter of that.
TOL = 2e-5

# (nodes, cached positions): one split; f32 in splits; BF16 in splits that one wave
# joins, and that four waves join.
SHAPES = [(10, 70), (7, 700), (24, 1700), (9, 5000)]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def round_to(x, kv):
    x = np.asarray(x, np.float32)
    return synth.bf16_to_f32(synth.f32_to_bf16(x)).reshape(x.shape) if kv == "bf16" else x


def case(seed, n, offset, hd, kv, kvh=2, q_heads=8):
    rng = np.random.default_rng(seed)
    k, v = ref.make_cache(rng, offset + n, kvh, hd, kv)
    q = rng.standard_normal((n, q_heads * hd)).astype(np.float32)
    return rng, q, k, v, ref.parents_of("random", n, rng)


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,offset", SHAPES)
def test_an_infinity_in_the_prefix_shows(hip, n, offset, hd, kv):
    """Infinities in dims of their own at many prefix positions, the row's
    largest key (a weight of one) among them: every row has them, and no NaN;
    the other elements are as without. One dim with both signs is NaN."""
    rng, q, k, v, parents = case(n + hd, n, offset, hd, kv)
    scores = np.einsum("nhd,pd->nhp", q.reshape(n, 8, hd)[:, :4].astype(np.float64), k[:offset, 0].astype(np.float64))
    best = np.unique(scores.argmax(-1))[:24]
    for d, p in enumerate(best):
        v[p, 0, d] = np.inf if d % 2 else -np.inf
    a, b = rng.choice(offset, 2, replace=False)
    v[a, 1, 40], v[b, 1, 40] = np.inf, -np.inf
    with np.errstate(invalid="ignore"):
        want = ref.attention64(q, k, v, 8, parents, offset)
    kp, vp, table = ref.paged(k, v, kv, rng)
    got = hip.tree_attention(q, kp, vp, table, 8, parents, offset)
    fine = np.isfinite(want)
    assert (~fine).sum() == n * 4 * (len(best) + 1)
    assert np.array_equal(got[~fine], want[~fine].astype(np.float32), equal_nan=True)
    assert (np.abs(got[fine] - want[fine]) <= TOL * np.abs(want[fine]).max()).all()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,offset", SHAPES)
def test_an_infinity_of_no_weight_still_shows(hip, n, offset, hd, kv):
    """Scores hundreds apart: the weight of the infinity's key rounds to 0 in
    f32 for most rows, and 0 times infinity is NaN, in one split or many."""
    rng, q, k, v, parents = case(n + hd + 1, n, offset, hd, kv)
    q *= 60
    d = 5
    v[offset // 3, :, d] = np.inf
    kp, vp, table = ref.paged(k, v, kv, rng)
    got = hip.tree_attention(q, kp, vp, table, 8, parents, offset).reshape(n, 8, hd)
    assert not np.isfinite(got[:, :, d]).any()
    assert np.isfinite(np.delete(got, d, 2)).all()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,offset", SHAPES + [(12, 0)])
@pytest.mark.parametrize("what", ["one", "120", "123", "126", "1e38", "most", "signs"])
def test_large_finite_values_average(hip, what, n, offset, hd, kv):
    """One prefix row of 1e37, then values of one size in every row: 2^120 to
    2^126 (weights of up to 2^8 or their sums overflow, in a block, between the
    key waves or between splits), 1e38, BF16's largest, and 2^126 of both signs.
    Every average is finite; dims without them keep their own accuracy."""
    rng, q, k, v, parents = case(n + hd + 2, n, offset, hd, kv)
    large = np.zeros(hd, bool)
    large[::3] = True
    if what == "one":
        v[offset // 2, :, large] = 1e37  # (without a prefix: the root's)
    else:
        size = {"1e38": 1e38, "most": 3.3895314e38, "signs": 2.0**126}.get(what) or 2.0**int(what)
        at = rng.uniform(0.75, 1, v.shape)
        if what == "signs":
            at *= rng.choice([-1, 1], v.shape)
        v[:, :, large] = (size * at)[:, :, large]
    v = round_to(v, kv)
    assert np.isfinite(v).all()
    want = ref.attention64(q, k, v, 8, parents, offset)
    kp, vp, table = ref.paged(k, v, kv, rng)
    got = hip.tree_attention(q, kp, vp, table, 8, parents, offset)
    assert np.isfinite(got).all()
    want, got = (t.astype(np.float64).reshape(n, 8, hd) for t in (want, got))
    for dims in (large, ~large):
        assert (np.abs(got - want)[..., dims] <= TOL * np.abs(v[..., dims]).max()).all()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,offset", SHAPES)
def test_an_infinity_among_scores_of_minus_infinity_shows(hip, n, offset, hd, kv):
    """A run of keys whose scores are all -inf, as long as a split: they weigh
    nothing, and nothing times infinity is NaN."""
    rng, q, k, v, parents = case(n + hd + 3, n, offset, hd, kv)
    q.reshape(n, 8, hd)[:, :, 0] = 1.0
    k[:min(offset - 30, 128), :, 0] = -np.inf
    clean = ref.attention64(q, k, v, 8, parents, offset)
    kp, vp, table = ref.paged(k, v, kv, rng)
    got = hip.tree_attention(q, kp, vp, table, 8, parents, offset)
    assert (np.abs(got - clean) <= TOL * np.abs(clean).max()).all()
    v[20, :, 7] = np.inf
    kp, vp, table = ref.paged(k, v, kv, rng)
    got = hip.tree_attention(q, kp, vp, table, 8, parents, offset).reshape(n, 8, hd)
    assert np.isnan(got[:, :, 7]).all()
    clean = clean.reshape(n, 8, hd)
    assert (np.abs(np.delete(got - clean, 7, 2)) <= TOL * np.abs(clean).max()).all()
