"""Tree attention and tree commit against 64-bit restatements."""
import ctypes

import numpy as np
import pytest

import tree_reference as ref
from cheetah_amd import synth

pytestmark = pytest.mark.gpu

# Every product is as exact as an f32 one (three BF16 parts of queries and
# probabilities, and of an f32 cache), sums are f32: of 6,000 keys' weights at most
# 6,000 roundings of 2^-25 at random, 5e-6 of the largest output at two deviations;
# exponentials add 2^-22. 2e-5.
TOL = 2e-5


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    h.init(0)
    return h


def rel_err(got, want):
    return float(np.max(np.abs(got.astype(np.float64) - want)) / np.max(np.abs(want)))


def case(seed, q_heads, kvh, hd, n, offset, kv, page=64):
    rng = np.random.default_rng(seed)
    k, v = ref.make_cache(rng, offset + n, kvh, hd, kv)
    return rng, rng.standard_normal((n, q_heads * hd)).astype(np.float32), k, v, ref.paged(k, v, kv, rng, page)


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("q_heads,kvh,hd", [(14, 2, 64), (32, 8, 128), (28, 4, 128), (5, 1, 64), (3, 3, 128), (16, 2, 64),
                                            (6, 2, 128), (6, 1, 64)])
@pytest.mark.parametrize("n,offset,tree", [(1, 0, "chain"), (1, 300, "chain"), (2, 63, "star"), (3, 1, "chain"),
                                           (7, 64, "random"), (16, 500, "random"), (33, 95, "roots"), (65, 130, "random")])
def test_tree_attention_matches_64_bits(hip, q_heads, kvh, hd, n, offset, tree, kv):
    """Every head layout over trees that start inside, at the end and at the
    start of a page; rows that nothing has written hold NaN."""
    rng, q, k, v, (kp, vp, table) = case(n * 1000 + offset + q_heads, q_heads, kvh, hd, n, offset, kv)
    parents = ref.parents_of(tree, n, rng)
    got = hip.tree_attention(q, kp, vp, table, q_heads, parents, offset)
    assert np.isfinite(got).all()
    assert rel_err(got, ref.attention64(q, k, v, q_heads, parents, offset)) < TOL


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("q_heads,kvh,hd", [(32, 8, 128), (7, 1, 64)])
@pytest.mark.parametrize("n,offset,tree", [
    (8, 2113, "random"), (9, 6000, "star"), (31, 0, "random"), (32, 64, "chain"), (40, 1000, "star"), (63, 1, "roots"),
    (64, 0, "random"), (64, 2048, "roots"), (100, 700, "chain"), (128, 127, "random"), (129, 63, "roots"),
    (200, 300, "random"), (256, 0, "chain"), (256, 65, "random"), (256, 1500, "star")])
def test_tree_attention_sizes(hip, q_heads, kvh, hd, n, offset, tree, kv):
    """Trees from a few nodes to the most, of every shape, over no prefix, one
    tile and many."""
    rng, q, k, v, (kp, vp, table) = case(n + offset, q_heads, kvh, hd, n, offset, kv)
    parents = ref.parents_of(tree, n, rng)
    got = hip.tree_attention(q, kp, vp, table, q_heads, parents, offset)
    assert np.isfinite(got).all()
    assert rel_err(got, ref.attention64(q, k, v, q_heads, parents, offset)) < TOL


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("page", [128, 192, 512])
def test_tree_attention_larger_pages(hip, page, kv):
    rng, q, k, v, (kp, vp, table) = case(page, 8, 2, 128, 20, 777, kv, page)
    parents = ref.parents_of("random", 20, rng)
    got = hip.tree_attention(q, kp, vp, table, 8, parents, 777)
    assert rel_err(got, ref.attention64(q, k, v, 8, parents, 777)) < TOL


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("offset", [0, 40, 130])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_a_branch_reaches_no_other(hip, bad, offset, hd, kv):
    """NaN, infinities and the largest values in one branch's K and V: the nodes
    that do not see them give the same results as without, bit for bit."""
    n = 24
    rng, q, k, v, (kp, vp, table) = case(int(offset + hd), 8, 2, hd, n, offset, kv)
    parents = ref.parents_of("random", n, rng)
    clean = hip.tree_attention(q, kp, vp, table, 8, parents, offset)
    sick = 9
    k[offset + sick] = bad
    v[offset + sick, :, ::3] = bad
    kp2, vp2, table2 = ref.paged(k, v, kv, np.random.default_rng(3))
    got = hip.tree_attention(q, kp2, vp2, table2, 8, parents, offset)
    sees = np.array([sick in path for path in ref.seen_by(parents)])
    assert sees.any() and not sees.all()
    assert np.array_equal(got[~sees].view(np.uint32), clean[~sees].view(np.uint32))


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_a_seen_infinite_value_shows(hip, kv):
    """An infinite V element gives every row that sees it an infinity or NaN
    there, and leaves the other elements as they are."""
    n, offset = 10, 70
    rng, q, k, v, _ = case(5, 4, 1, 64, n, offset, kv)
    parents = ref.parents_of("chain", n, rng)
    want = ref.attention64(q, k, v, 4, parents, offset).reshape(n, 4, 64)
    v[offset + 4, 0, 7] = np.inf
    kp, vp, table = ref.paged(k, v, kv, rng)
    got = hip.tree_attention(q, kp, vp, table, 4, parents, offset).reshape(n, 4, 64)
    assert not np.isfinite(got[4:, :, 7]).any() and np.isfinite(got[:4]).all()
    keep = np.arange(64) != 7
    assert rel_err(got[:, :, keep], want[:, :, keep]) < TOL


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_a_parent_that_is_no_earlier_node_makes_a_root(hip, kv):
    n, offset = 8, 100
    _, q, k, v, (kp, vp, table) = case(8, 4, 2, 64, n, offset, kv)
    odd = np.array([5, 1, 0, -7, 3, 2**31 - 1, 4, -2**31], np.int32)
    plain = np.array([-1, -1, 0, -1, 3, -1, 4, -1], np.int32)
    a, b = (hip.tree_attention(q, kp, vp, table, 4, p, offset) for p in (odd, plain))
    assert np.array_equal(a, b)
    assert rel_err(a, ref.attention64(q, k, v, 4, odd, offset)) < TOL


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_attention_large_scores(hip, hd, kv):
    """Scores in the hundreds, where one key takes nearly all of the weight:
    the running maximum moves at almost every tile."""
    n, offset = 20, 700
    rng, q, k, v, (kp, vp, table) = case(hd, 8, 2, hd, n, offset, kv)
    q *= 30
    parents = ref.parents_of("random", n, rng)
    got = hip.tree_attention(q, kp, vp, table, 8, parents, offset)
    # A score of s is off by about 2^-17 |s| / sqrt(hd): its weight by that many times
    # 2^-17; |s| reaches 30 * sqrt(hd) * 4.
    assert rel_err(got, ref.attention64(q, k, v, 8, parents, offset)) < 120 * 2.0**-17


def test_a_chain_is_causal_attention(hip):
    rng, q, k, v, (kp, vp, table) = case(2, 14, 2, 64, 30, 400, "bf16")
    got = hip.tree_attention(q, kp, vp, table, 14, ref.parents_of("chain", 30, rng), 400)
    want = hip.attention(q, kp, vp, table, 14, 30, 400)
    assert rel_err(got, want.astype(np.float64)) < TOL


def test_calls_are_repeatable(hip):
    """The same bits again, also after a larger call has used the scratch."""
    rng, q, k, v, (kp, vp, table) = case(12, 32, 8, 128, 20, 3000, "bf16")
    parents = ref.parents_of("random", 20, rng)
    first = hip.tree_attention(q, kp, vp, table, 32, parents, 3000)
    rng2, q2, _, _, (kp2, vp2, table2) = case(13, 32, 8, 128, 130, 5000, "bf16")
    hip.tree_attention(q2, kp2, vp2, table2, 32, ref.parents_of("random", 130, rng2), 5000)
    assert np.array_equal(hip.tree_attention(q, kp, vp, table, 32, parents, 3000), first)


def test_two_threads_call_at_once(hip):
    import threading

    cases = []
    for i in range(4):
        rng, q, k, v, pages = case(40 + i, 28, 4, 128, 10 + 20 * i, 900, "bf16")
        cases.append((q, k, v, pages, ref.parents_of("random", 10 + 20 * i, rng)))
    got = [None] * len(cases)

    def run(i):
        q, _, _, (kp, vp, table), parents = cases[i]
        got[i] = hip.tree_attention(q, kp, vp, table, 28, parents, 900)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, (q, k, v, _, parents) in zip(got, cases):
        assert rel_err(g, ref.attention64(q, k, v, 28, parents, 900)) < TOL


@pytest.mark.parametrize("kv,page_elems", [("bf16", 8 * 64 * 128), ("f32", 8 * 64 * 128)])
def test_pools_past_4_gib(hip, kv, page_elems):
    """Pages whose byte offsets (and, in BF16, element offsets) pass 32 bits."""
    n, offset, q_heads, kvh, hd = 6, 100, 32, 8, 128
    rng = np.random.default_rng(77)
    k, v = ref.make_cache(rng, offset + n, kvh, hd, kv)
    kp, vp, table = ref.paged(k, v, kv, rng, spare=0)
    elem = kp.dtype.itemsize
    far = (1 << 32) // page_elems + 3  # first page past 2^32 elements
    q = rng.standard_normal((n, q_heads * hd)).astype(np.float32)
    parents = ref.parents_of("random", n, rng)
    pools = [hip.DeviceBuffer((far + 2) * page_elems * elem) for _ in "kv"]
    for pool, pages in zip(pools, (kp, vp)):
        assert len(pages) == 2
        hip.check(hip.lib().cheetah_hip_upload(pool.ptr + far * page_elems * elem, pages.ctypes.data, pages.nbytes))
    qd, pd, od = hip.DeviceBuffer.from_array(q), hip.DeviceBuffer.from_array(parents), hip.DeviceBuffer(q.nbytes)
    td = hip.DeviceBuffer.from_array((table + far).astype(np.int32))
    view = hip.KvView(pools[0].ptr, pools[1].ptr, td.ptr, 64, kvh, hd)
    f32 = int(kv == "f32")
    hip.check(hip.lib().cheetah_hip_tree_attention(qd.ptr, ctypes.byref(view), f32, q_heads, pd.ptr, n, offset, od.ptr))
    got = od.download(np.float32, q.size).reshape(q.shape)
    assert rel_err(got, ref.attention64(q, k, v, q_heads, parents, offset)) < TOL
    nodes = (ctypes.c_uint32 * 2)(0, 4)
    hip.check(hip.lib().cheetah_hip_tree_commit((hip.KvView * 1)(view), 1, f32, offset, nodes, 2))
    back = np.empty_like(kp)
    hip.check(hip.lib().cheetah_hip_download(back.ctypes.data, pools[0].ptr + far * page_elems * elem, back.nbytes))
    a, b = (back[table[p // 64], :, p % 64] for p in (offset + 1, offset + 4))
    assert np.array_equal(a, b) and np.array_equal(b, kp[table[1], :, (offset + 4) % 64])


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,offset", [(140, 4200), (130, 4096 - 64)])
def test_a_split_of_many_pages(hip, n, offset, hd, kv):
    """64 query heads over 8: so many row blocks that a KV head's keys are one
    split, whose page entries are looked up 64 at a time. One KV head's queries
    are compared."""
    rng, q, k, v, (kp, vp, table) = case(n + hd, 64, 8, hd, n, offset, kv)
    parents = ref.parents_of("random", n, rng)
    got = hip.tree_attention(q, kp, vp, table, 64, parents, offset)
    assert np.isfinite(got).all()
    head = slice(40 * hd, 48 * hd)
    want = ref.attention64(np.ascontiguousarray(q[:, head]), k[:, 5:6], v[:, 5:6], 8, parents, offset)
    assert rel_err(got[:, head], want) < TOL


# ---------------------------------------------------------------------------
# Commit.
# ---------------------------------------------------------------------------

def moved(pool, table, offset, nodes, page):
    out = pool.copy()
    for j, node in enumerate(nodes):
        to, at = offset + j, offset + node
        out[table[to // page], :, to % page] = pool[table[at // page], :, at % page]
    return out


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("kvh,hd,page", [(2, 64, 64), (8, 128, 64), (3, 128, 192)])
@pytest.mark.parametrize("offset,nodes", [
    (0, [0]), (5, []), (60, [0, 1, 2, 3, 4]), (63, [0, 2, 3]), (64, [1]), (100, [255]), (17, [0, 2, 3, 5, 8, 13, 21, 34, 55]),
    (1, list(range(1, 256))), (120, list(range(0, 20)) + list(range(40, 256, 3))), (62, [0, 7, 8, 9, 10, 11, 12, 13, 14, 15])])
def test_commit_moves_the_branch(hip, kvh, hd, page, offset, nodes, kv):
    """Bit for bit: whole runs that shift by one (each row the source of the
    next move), moves across pages, rows in place, one and no node; every other
    row stays as it was."""
    rng = np.random.default_rng(offset + len(nodes))
    caches = []
    for _ in range(3):  # layers with page tables of their own
        k, v = ref.make_cache(rng, offset + 256, kvh, hd, kv)
        caches.append(ref.paged(k, v, kv, rng, page, fill=1.5))
    got = hip.tree_commit(caches, offset, nodes)
    for (gk, gv), (kp, vp, table) in zip(got, caches):
        for g, pool in ((gk, kp), (gv, vp)):
            assert np.array_equal(g.view(np.uint8), moved(pool, table, offset, nodes, page).view(np.uint8))


def test_commit_of_more_views_than_a_launch_holds(hip):
    rng = np.random.default_rng(9)
    caches = []
    for _ in range(131):
        k, v = ref.make_cache(rng, 20, 1, 64, "bf16")
        caches.append(ref.paged(k, v, "bf16", rng, spare=0, fill=0))
    nodes = [0, 3, 4, 9]
    for (gk, gv), (kp, vp, table) in zip(hip.tree_commit(caches, 10, nodes), caches):
        assert np.array_equal(gk, moved(kp, table, 10, nodes, 64))
        assert np.array_equal(gv, moved(vp, table, 10, nodes, 64))


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_verify_then_commit_then_continue(hip, kv):
    """A tree judged, its branch kept, the next tree judged on the longer
    prefix: what attention over the branch's own rows gives."""
    n, offset, q_heads, kvh, hd = 12, 58, 8, 2, 64
    rng = np.random.default_rng(21)
    k, v = ref.make_cache(rng, offset + n, kvh, hd, kv)
    parents = ref.parents_of("random", n, rng)
    path = ref.seen_by(parents)[-1]
    kp, vp, table = ref.paged(k, v, kv, rng)
    (kp, vp), = hip.tree_commit([(kp, vp, table)], offset, path)
    keep = np.concatenate([np.arange(offset), offset + np.array(path)])
    left = offset + n - len(keep)  # the next tree's rows: what lies behind the branch
    m = min(left, 4)
    q = rng.standard_normal((m, q_heads * hd)).astype(np.float32)
    nk, nv = (np.concatenate([t[keep], t[len(keep):len(keep) + m]]) for t in (k, v))
    after = ref.parents_of("star", m, rng)
    got = hip.tree_attention(q, kp, vp, table, q_heads, after, len(keep))
    # Rows behind the branch are left as they were, so the restatement has them too.
    assert rel_err(got, ref.attention64(q, nk, nv, q_heads, after, len(keep))) < TOL
