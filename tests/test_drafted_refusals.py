"""CPU-only: what the calls for drafted tokens and scoring refuse, each with a
sentence and before any device work (the library is not initialized here)."""
import ctypes

import numpy as np
import pytest

D = 4096  # stands for a device pointer; never dereferenced


@pytest.fixture(scope="module")
def hip():
    from cheetah_amd import hip as h
    return h


def refused(hip, rc, text):
    assert rc == -1
    assert text in hip.lib().cheetah_hip_last_error().decode()


def view(hip, **kw):
    a = dict(k=D, v=2 * D, table=3 * D, page=64, kvh=2, hd=64)
    a.update(kw)
    return hip.KvView(a["k"], a["v"], a["table"], a["page"], a["kvh"], a["hd"])


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null pointer"), (dict(parents=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(n=0), "1 to 256 nodes"), (dict(n=257), "1 to 256 nodes"), (dict(n=1 << 40), "1 to 256 nodes"),
    (dict(fmt=2), "kv_format"), (dict(q_heads=0), "multiple of kv_heads"), (dict(q_heads=3), "multiple of kv_heads"),
    (dict(q_heads=18), "1..8 query heads"), (dict(q_heads=1 << 31), "multiple of kv_heads"),
    (dict(offset=2**31 - 5), "position out of range"), (dict(offset=2**31 - 1024), "position out of range"), (dict(offset=2**64 - 1), "position out of range"),
    (dict(q=D + 4), "aligned"), (dict(out=D + 8), "aligned"), (dict(parents=D + 2), "aligned"),
    (dict(view=dict(k=None)), "null cache"), (dict(view=dict(v=None)), "null cache"),
    (dict(view=dict(table=None)), "null cache"), (dict(view=dict(kvh=0)), "out of range"),
    (dict(view=dict(kvh=70000)), "out of range"), (dict(view=dict(page=0)), "multiple of 64"),
    (dict(view=dict(page=96)), "multiple of 64"), (dict(view=dict(page=2**32 - 64)), "out of range"),
    (dict(view=dict(hd=0)), "head_dim 64 and 128"), (dict(view=dict(hd=96)), "head_dim 64 and 128"),
    (dict(view=dict(k=D + 8)), "aligned"), (dict(view=dict(v=D + 2)), "aligned"), (dict(view=dict(table=D + 1)), "aligned"),
])
def test_tree_attention_refuses(hip, change, text):
    a = dict(q=D, fmt=0, q_heads=4, parents=D, n=8, offset=100, out=D)
    a.update({k: v for k, v in change.items() if k != "view"})
    kv = view(hip, **change.get("view", {}))
    refused(hip, hip.lib().cheetah_hip_tree_attention(a["q"], ctypes.byref(kv), a["fmt"], a["q_heads"], a["parents"],
                                                      a["n"], a["offset"], a["out"]), text)


def test_tree_attention_refuses_a_null_view(hip):
    refused(hip, hip.lib().cheetah_hip_tree_attention(D, None, 0, 4, D, 8, 0, D), "null pointer")


@pytest.mark.parametrize("nodes,text", [([0, 0], "strictly increasing"), ([1, 0], "strictly increasing"),
                                        ([0, 256], "below 256"), ([2**32 - 1], "below 256")])
def test_tree_commit_refuses_a_branch(hip, nodes, text):
    arr = (ctypes.c_uint32 * len(nodes))(*nodes)
    refused(hip, hip.lib().cheetah_hip_tree_commit((hip.KvView * 1)(view(hip)), 1, 0, 10, arr, len(nodes)), text)


def test_tree_commit_refuses_views(hip):
    call, nodes = hip.lib().cheetah_hip_tree_commit, (ctypes.c_uint32 * 2)(0, 2)
    refused(hip, call(None, 1, 0, 0, nodes, 2), "null argument")
    refused(hip, call((hip.KvView * 1)(view(hip)), 0, 0, 0, nodes, 2), "null argument")
    refused(hip, call((hip.KvView * 1)(view(hip)), 1, 0, 0, None, 2), "null argument")
    refused(hip, call((hip.KvView * 1)(view(hip)), 1, 2, 0, nodes, 2), "kv_format")
    refused(hip, call((hip.KvView * 1)(view(hip)), 1, 0, 2**31 - 100, nodes, 2), "position out of range")
    refused(hip, call((hip.KvView * 1)(view(hip, hd=32)), 1, 0, 0, nodes, 2), "head_dim")
    for other in (dict(page=128), dict(kvh=4), dict(hd=128)):
        refused(hip, call((hip.KvView * 2)(view(hip), view(hip, **other)), 2, 0, 0, nodes, 2), "one geometry")


@pytest.mark.parametrize("other", [dict(), dict(v=5 * D), dict(k=5 * D), dict(k=2 * D, v=5 * D), dict(k=5 * D, v=D)])
def test_tree_commit_refuses_a_cache_listed_twice(hip, other):
    """Two views that share a pool and its page table, or one whose K and V are
    the same pool; a pool with another page table (another sequence) may come."""
    call, nodes = hip.lib().cheetah_hip_tree_commit, (ctypes.c_uint32 * 2)(0, 2)
    refused(hip, call((hip.KvView * 3)(view(hip), view(hip, k=7 * D, v=8 * D), view(hip, **other)), 3, 0, 0, nodes, 2),
            "listed twice")
    refused(hip, call((hip.KvView * 1)(view(hip, v=D)), 1, 0, 0, nodes, 2), "listed twice")
    if not hip._initialized:  # (it would run)
        two = (hip.KvView * 2)(view(hip), view(hip, table=6 * D, **other))
        refused(hip, call(two, 2, 0, 0, nodes, 2), "not initialized")


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null pointer"), (dict(fmt=2), "logit_format"), (dict(rows=0), "out of range"),
    (dict(vocab=0), "out of range"), (dict(rows=2**31), "out of range"), (dict(vocab=2**31, stride=2**31), "out of range"),
    (dict(stride=99), "stride below vocab"), (dict(top=65), "at most 64"), (dict(vocab=3, top=4), "at most the vocabulary"),
    (dict(lp=None, ent=None, top=0, ids=None, tops=None), "without an output"), (dict(tokens=None), "needs the tokens"),
    (dict(ids=None), "alternatives, or none"), (dict(tops=None), "alternatives, or none"),
    (dict(top=0), "alternatives, or none"), (dict(x=D + 2), "misaligned"), (dict(x=D + 1, fmt=0), "misaligned"),
    (dict(tokens=D + 1), "misaligned"), (dict(lp=D + 2), "misaligned"), (dict(ent=D + 2), "misaligned"),
    (dict(ids=D + 2), "misaligned"), (dict(tops=D + 2), "misaligned"),
])
def test_logprobs_refuses(hip, change, text):
    a = dict(x=D, fmt=1, rows=4, vocab=100, stride=104, tokens=D, top=5, lp=D, ent=D, ids=D, tops=D)
    a.update(change)
    refused(hip, hip.lib().cheetah_hip_logprobs(*a.values()), text)


def test_valid_arguments_reach_the_device_check(hip):
    if hip._initialized:
        pytest.skip("library already initialized in this process")
    kv = view(hip)
    refused(hip, hip.lib().cheetah_hip_tree_attention(D, ctypes.byref(kv), 0, 4, D, 256, 0, D), "not initialized")
    refused(hip, hip.lib().cheetah_hip_tree_commit((hip.KvView * 1)(kv), 1, 1, 0, (ctypes.c_uint32 * 1)(3), 1),
            "not initialized")
    refused(hip, hip.lib().cheetah_hip_logprobs(D, 0, 1, 10, 10, D, 10, D, None, D, D), "not initialized")


def test_host_wrappers_check_their_arrays(hip):
    q, kp = np.zeros((2, 128), np.float32), np.zeros((2, 2, 64, 64), np.uint16)
    with pytest.raises(ValueError, match="page table ends"):
        hip.tree_attention(q, kp, kp, np.array([0], np.int32), 2, [-1, 0], 63)
    with pytest.raises(ValueError, match="outside the pool"):
        hip.tree_attention(q, kp, kp, np.array([0, 2], np.int32), 2, [-1, 0], 63)
    with pytest.raises(ValueError, match="both"):
        hip.tree_attention(q, kp, kp.astype(np.float32), np.array([0, 1], np.int32), 2, [-1, 0], 63)
    with pytest.raises(ValueError, match="page table ends"):
        hip.tree_commit([(kp, kp, np.array([0], np.int32))], 60, [0, 4])
    with pytest.raises(ValueError, match="one token a row"):
        hip.logprobs(np.zeros((3, 5), np.float32), [1, 2])
    with pytest.raises(ValueError, match="matrix"):
        hip.logprobs(np.zeros((3, 5), np.float64))


def test_model_calls_refuse_what_they_see_first(hip):
    """Null outputs, a second root and a null model, before any device work."""
    L = hip.lib()
    toks, par = (ctypes.c_uint32 * 3)(1, 2, 3), (ctypes.c_int32 * 3)(-1, 0, -1)
    out, count, f = (ctypes.c_uint32 * 3)(), ctypes.c_size_t(0), (ctypes.c_float * 3)()
    refused(hip, L.cheetah_hip_forward_tree(None, toks, par, 3, 0, None, None), "without an output")
    refused(hip, L.cheetah_hip_forward_tree(None, toks, par, 3, 0, out, None), "no model")
    refused(hip, L.cheetah_hip_commit_tree(None, out, 1), "no model")
    refused(hip, L.cheetah_hip_verify_tree(None, toks, par, 3, 0, None, ctypes.byref(count), out), "null output")
    refused(hip, L.cheetah_hip_verify_tree(None, toks, par, 3, 0, out, None, out), "null output")
    refused(hip, L.cheetah_hip_verify_tree(None, toks, par, 3, 0, out, ctypes.byref(count), None), "null output")
    refused(hip, L.cheetah_hip_verify_tree(None, toks, par, 3, 0, out, ctypes.byref(count), out), "one root")
    par[2] = 1
    refused(hip, L.cheetah_hip_verify_tree(None, toks, par, 3, 0, out, ctypes.byref(count), out), "no model")
    par[0] = 0
    refused(hip, L.cheetah_hip_verify_tree(None, toks, par, 3, 0, out, ctypes.byref(count), out), "one root")
    refused(hip, L.cheetah_hip_forward_logprobs(None, toks, 3, 0, 0, None, 0, None, f, None, None), "no model")
