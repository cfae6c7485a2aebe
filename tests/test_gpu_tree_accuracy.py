"""Tree attention's accuracy, relative to the output's norm, at bars that a part
product missing from the kernel does not pass (tests/test_tree_parts.py)."""
import numpy as np
import pytest

import tree_parts as tp
import tree_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def error(hip, q_heads, kvh, hd, n, offset, kv, scale):
    rng = np.random.default_rng(n + hd + offset)
    k, v = ref.make_cache(rng, offset + n, kvh, hd, kv)
    q = (rng.standard_normal((n, q_heads * hd)) * scale).astype(np.float32)
    parents = ref.parents_of("random", n, rng)
    kp, vp, table = ref.paged(k, v, kv, rng)
    got = hip.tree_attention(q, kp, vp, table, q_heads, parents, offset)
    return tp.norm_err(got, ref.attention64(q, k, v, q_heads, parents, offset))


# One and two row waves a block, one split, splits joined by one wave and by four.
@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("q_heads,kvh,hd", [(8, 2, 64), (8, 2, 128), (28, 4, 128), (3, 3, 64)])
@pytest.mark.parametrize("n,offset", [(4, 30), (12, 300), (40, 700), (200, 300), (6, 2000), (9, 6000)])
def test_ordinary_scores(hip, n, offset, q_heads, kvh, hd, kv):
    assert error(hip, q_heads, kvh, hd, n, offset, kv, 1.5) < tp.ORDINARY


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,offset", [(12, 300), (40, 700), (9, 6000)])
def test_scores_in_the_hundreds(hip, n, offset, hd, kv):
    assert error(hip, 8, 2, hd, n, offset, kv, 30) < tp.LARGE
