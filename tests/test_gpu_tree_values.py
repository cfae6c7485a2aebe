"""Tree attention over infinities in V rows that nodes see: the definition's
infinity, whatever the cache's type, the position and the number of splits."""
import numpy as np
import pytest

import tree_reference as ref

pytestmark = pytest.mark.gpu

# Rows with an infinity are averaged key by key in f32: 6,000 weights' roundings of
# 2^-24 (the exponential 2^-22 once) at random and as many of the running sums,
# sqrt(12,000) 2^-24 = 6.6e-6 of the largest output, three deviations.
TOL = 2e-5

# (nodes, cached positions): one split; f32 in splits; BF16 in splits that one wave
# joins, and that four waves join.
SHAPES = [(10, 70), (7, 700), (24, 1700), (9, 5000)]


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


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
