"""CPU-only: the accuracy bars of tree attention tell every part product that the
kernel takes from a kernel without it (tree_parts.py restates them)."""
import numpy as np
import pytest

import tree_parts as tp
import tree_reference as ref


@pytest.mark.parametrize("scale,bar", [(1.5, tp.ORDINARY), (30, tp.LARGE)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_a_missing_part_product_passes_no_bar(kv, hd, scale, bar):
    n, offset = 12, 300
    rng = np.random.default_rng(n + hd)
    k, v = ref.make_cache(rng, offset + n, 2, hd, kv)
    q = (rng.standard_normal((n, 8 * hd)) * scale).astype(np.float32)
    parents = ref.parents_of("random", n, rng)
    want = ref.attention64(q, k, v, 8, parents, offset)
    every = tp.products(kv)

    def err(scores, values):
        return tp.norm_err(tp.attention_parts(q, k, v, 8, parents, offset, kv, scores, values), want)

    assert err(every, every) < bar / 4
    for p in every:
        less = [x for x in every if x != p]
        assert err(less, every) > 2 * bar, p
        if scale == 1.5:  # (one key with nearly all of the weight is one of its parts)
            assert err(every, less) > 2 * bar, p


def test_parts_sum_to_the_value():
    x = np.random.default_rng(0).standard_normal(1000).astype(np.float32) * 1e3
    assert np.array_equal(sum(tp.cut(x)), x.astype(np.float64))
