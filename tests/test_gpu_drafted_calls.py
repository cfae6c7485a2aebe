"""The calls for drafted tokens and scoring as callers make them: arrays of other
integer types, one token at a time."""
import numpy as np
import pytest

import tree_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


@pytest.mark.parametrize("call", ["tree", "chunk"])
@pytest.mark.parametrize("dtype", [np.int64, np.uint8, np.int16])
def test_page_tables_of_other_types(hip, dtype, call):
    """numpy's default integers (read as they lie, pairs of words) and narrow ones."""
    rng = np.random.default_rng(3)
    k, v = ref.make_cache(rng, 200, 2, 64, "bf16")
    kp, vp, table = ref.paged(k, v, "bf16", rng)
    q = rng.standard_normal((8, 8 * 64)).astype(np.float32)
    parents = ref.parents_of("random", 8, rng)

    def run(t):
        if call == "tree":
            return hip.tree_attention(q, kp, vp, t, 8, parents, 192)
        return hip.attention(q, kp, vp, t, 8, 8, 192)

    assert np.array_equal(run(table.astype(dtype)).view(np.uint32), run(table).view(np.uint32))
