"""The operators of speculative decoding and scoring, as measurable cases.

A caller that drafts several continuations of one sequence has the decoder
judge all of them in one forward. Three calls of the C-ABI stand for that work
beside the attention and projection calls (``perf/cases.py`` has those):

* ``cheetah_hip_tree_attention``: attention of a tree of drafted tokens over
  the paged K/V cache. Each node sees the cached prefix, its ancestors and
  itself, not its siblings.
* ``cheetah_hip_tree_commit``: the accepted branch's K/V rows move to the
  positions that follow the prefix, in every layer's cache at once.
* ``cheetah_hip_logprobs``: for rows of logits the log probability of a given
  token, the entropy and the most likely alternatives.

``own`` selects the framework's calls; otherwise ``run`` computes the same in
elementary torch operations. Head layouts and vocabularies are those of
``cheetah_amd.configs`` or generic.
"""
import ctypes
import math

import numpy as np
import torch

own = False

PAGE = 64
# (q heads, KV heads, head dim): the decoders served, then generic layouts.
HEADS = ((14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 64), (6, 2, 128), (5, 1, 64), (16, 2, 128))
VOCABS = (151936, 128256, 152064, 32000)
# (layers, KV heads, head dim) of the decoders served.
CACHES = ((24, 2, 64), (32, 8, 128), (28, 4, 128))
TREE_MOST = 64 * 32 * 128 * 16447   # n x q heads x head dim x keys
LOGITS_MOST = 512 * 151936
POOL_MOST = 32 * 2 * 12 * 8 * PAGE * 128


def _tree(name, heads, n, offset, tree, width=4, kv="bf16"):
    qh, kvh, hd = heads
    return {"name": name, "kind": "tree", "q_heads": qh, "kv_heads": kvh, "hd": hd, "n": n, "offset": offset,
            "tree": tree, "width": width, "kv": kv}


def listed():
    return [
        # A handful of drafted tokens early in a small decoder's answer: latency.
        _tree("tree_5_on_60", HEADS[0], 5, 60, "random"),
        # A common draft tree in an ordinary conversation.
        _tree("tree_16_on_2k", HEADS[1], 16, 2047, "beam", 4),
        # The exact (f32) cache, ragged sizes.
        _tree("tree_13_on_2900_f32", HEADS[1], 13, 2900, "random", kv="f32"),
        # A few drafted tokens after a long document.
        _tree("tree_26_on_32k", HEADS[2], 26, 32767, "beam", 5),
        # A wide tree on a long context.
        _tree("tree_64_on_16k", HEADS[1], 64, 16383, "random"),
        # The largest tree.
        _tree("tree_256_on_4k", HEADS[2], 256, 4097, "random"),
        # The sampled token's log probability and five alternatives.
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 151936, "pad": 0, "top": 5, "logits": "f32"},
        # A draft tree's nodes with the alternatives an API returns.
        {"name": "logprobs_64", "kind": "logprobs", "rows": 64, "vocab": 128256, "pad": 0, "top": 20, "logits": "f32"},
        # An odd vocabulary in padded rows, many alternatives.
        {"name": "logprobs_37_odd", "kind": "logprobs", "rows": 37, "vocab": 32001, "pad": 31, "top": 64,
         "logits": "bf16"},
        # A prompt's rows scored: the largest.
        {"name": "logprobs_512", "kind": "logprobs", "rows": 512, "vocab": 151936, "pad": 0, "top": 1, "logits": "f32"},
        # Three accepted tokens of a small tree, the small decoder's cache.
        {"name": "commit_3_of_8", "kind": "commit", "layers": 24, "kv_heads": 2, "hd": 64, "offset": 577, "n": 8,
         "count": 3, "kv": "bf16"},
        # A long branch of a large tree, the exact cache of a large decoder.
        {"name": "commit_40_of_256_f32", "kind": "commit", "layers": 32, "kv_heads": 8, "hd": 128, "offset": 200,
         "n": 256, "count": 40, "kv": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "tree", "logprobs", "logprobs", "commit"))
    if kind == "tree":
        qh, kvh, hd = rng.choice(HEADS)
        n = _log_int(rng, 1, 256)
        kv = rng.choice(("bf16", "bf16", "f32"))
        most = TREE_MOST // (3 if kv == "f32" else 1) // (n * qh * hd) - n
        offset = 0 if rng.random() < 0.05 else min(_log_int(rng, 1, 32768), most)
        return {"kind": kind, "q_heads": qh, "kv_heads": kvh, "hd": hd, "n": n, "offset": offset,
                "tree": rng.choice(("chain", "beam", "random")), "width": rng.randint(2, 9), "kv": kv}
    if kind == "logprobs":
        vocab = rng.choice(VOCABS) if rng.random() < 0.5 else _log_int(rng, 100, 200000)
        rows = min(_log_int(rng, 1, 512), LOGITS_MOST // vocab)
        return {"kind": kind, "rows": rows, "vocab": vocab, "pad": rng.choice((0, 0, 3, 64)),
                "top": rng.choice((0, 1, 5, 20, 64)), "logits": rng.choice(("f32", "f32", "bf16"))}
    layers, kvh, hd = rng.choice(CACHES)
    n = _log_int(rng, 3, 256)
    count = min(_log_int(rng, 1, 64), n - 1)
    kv = rng.choice(("bf16", "f32"))
    pages = POOL_MOST // (layers * 2 * kvh * PAGE * hd)
    return {"kind": kind, "layers": layers, "kv_heads": kvh, "hd": hd, "offset": min(_log_int(rng, 1, 4096),
            (pages - 2) * PAGE - n), "n": n, "count": count, "kv": kv}


# ---------------------------------------------------------------------------
# Inputs, made from the seed alone.
# ---------------------------------------------------------------------------

def _parents(case, seed):
    """Draft trees: one chain, `width` chains out of the root, or each node
    under one of the eight before it."""
    n = case["n"]
    node = np.arange(n)
    if case["tree"] == "chain":
        parents = node - 1
    elif case["tree"] == "beam":
        parents = np.maximum(node - case["width"], 0)
    else:
        back = np.random.RandomState(seed % (1 << 32)).randint(1, 9, n)
        parents = np.maximum(node - back, 0)
    parents[0] = -1
    return parents.astype(np.int32)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _kv_type(case):
    return torch.float32 if case["kv"] == "f32" else torch.bfloat16


def prepare(case, seed):
    g = _gen(seed)
    state = dict(case)
    if case["kind"] == "tree":
        qh, kvh, hd, n, ctx = case["q_heads"], case["kv_heads"], case["hd"], case["n"], case["offset"] + case["n"]
        pages = -(-ctx // PAGE)
        table = torch.randperm(pages + 3, generator=g, device="cuda")[:pages]
        k, v = (torch.randn(pages + 3, kvh, PAGE, hd, generator=g, device="cuda").to(_kv_type(case)) for _ in "kv")
        # The rows past the last node and the pool's other pages were never written.
        free = torch.ones(pages + 3, PAGE, dtype=torch.bool, device="cuda")
        at = torch.arange(ctx, device="cuda")
        free[table[at // PAGE], at % PAGE] = False
        k, v = (t.masked_fill_(free[:, None, :, None], math.nan) for t in (k, v))
        state.update(k=k, v=v, table=table.to(torch.int32),
                     q=torch.randn(n, qh * hd, generator=g, device="cuda") * 1.5,
                     parents=torch.from_numpy(_parents(case, seed)).cuda(), out=torch.empty(n, qh * hd, device="cuda"))
        return state
    if case["kind"] == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        x = torch.randn(rows, vocab + case["pad"], generator=g, device="cuda") * 2.5
        likely = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        x[torch.arange(rows, device="cuda"), likely] += torch.rand(rows, generator=g, device="cuda") * 25
        # Rows that a grammar masks to few tokens, and some that it leaves empty.
        row = torch.arange(rows, device="cuda")[:, None]
        masked = torch.rand(x.shape, generator=g, device="cuda") < 0.98
        x.masked_fill_(((row % 7 == 3) & masked) | (row % 29 == 11), -math.inf)
        x[:, vocab:] = math.nan  # padding of the rows
        other = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        half = torch.rand(rows, generator=g, device="cuda") < 0.5
        state.update(x=x if case["logits"] == "f32" else x.to(torch.bfloat16),
                     tokens=torch.where(half, likely, other).to(torch.int32),
                     out=[torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")])
        if top:
            state["out"] += [torch.empty(rows, top, dtype=torch.int32, device="cuda"),
                             torch.empty(rows, top, device="cuda")]
        return state
    layers, kvh, hd = case["layers"], case["kv_heads"], case["hd"]
    pages = -(-(case["offset"] + case["n"]) // PAGE)
    pool = torch.randn(layers, 2, pages, kvh, PAGE, hd, generator=g, device="cuda").to(_kv_type(case))
    state.update(pool=pool, table=torch.randperm(pages, generator=g, device="cuda").to(torch.int32),
                 nodes=_branch(case, seed))
    return state


def _branch(case, seed):
    """The accepted nodes: the root, then count - 1 later ones, none of them
    in its place already."""
    later = np.random.RandomState(seed % (1 << 32)).permutation(case["n"] - 2)[:case["count"] - 1] + 2
    return np.concatenate([[0], np.sort(later)]).astype(np.uint32)


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"tree": _plain_tree, "logprobs": _plain_logprobs, "commit": _plain_commit}[state["kind"]](state)


def _ancestors(parents):
    """[n, n]: whether column j is row i or an ancestor of it. Paths of twice
    the length at each squaring; 2^8 is the largest tree."""
    n = parents.numel()
    node = torch.arange(n, device=parents.device)
    reach = ((node[None, :] == parents[:, None]) | (node[None, :] == node[:, None])).float()
    for _ in range(8):
        reach = (reach @ reach > 0).float()
    return reach > 0


def _plain_tree(s):
    qh, kvh, hd, n, offset = s["q_heads"], s["kv_heads"], s["hd"], s["n"], s["offset"]
    table, ctx = s["table"].long(), offset + n

    def rows(pool):  # [kv_heads, ctx, hd]
        return pool[table].transpose(0, 1).reshape(kvh, -1, hd)[:, :ctx].float()

    q = s["q"].view(n, kvh, -1, hd).transpose(0, 1).reshape(kvh, -1, hd)  # rows (node, head of the group)
    scores = q @ rows(s["k"]).transpose(1, 2).contiguous() / math.sqrt(hd)
    seen = torch.ones(n, ctx, dtype=torch.bool, device=q.device)
    seen[:, offset:] = _ancestors(s["parents"])
    scores = scores.view(kvh, n, -1, ctx).masked_fill_(~seen[None, :, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(kvh, -1, ctx)
    return (p @ rows(s["v"])).view(kvh, n, -1, hd).transpose(0, 1).reshape(n, qh * hd)


def _plain_logprobs(s):
    vocab, top = s["vocab"], s["top"]
    x = s["x"][:, :vocab].float()
    most = x.amax(1, keepdim=True)
    z = x - torch.where(most == -math.inf, torch.zeros_like(most), most)
    e = torch.exp(z)
    total = e.sum(1, dtype=torch.float64)  # log of it near 1 in 64 bits
    log_total = torch.log(total)
    mixed = torch.where(e > 0, e * z, torch.zeros_like(e)).sum(1, dtype=torch.float64)
    empty = total == 0
    entropy = torch.where(empty, torch.zeros_like(total), log_total - mixed / total).float()

    def logprob(zt):
        zt = zt.double() - (log_total if zt.dim() == 1 else log_total[:, None])
        return torch.where(empty if zt.dim() == 1 else empty[:, None], torch.full_like(zt, -math.inf), zt).float()

    out = [logprob(z.gather(1, s["tokens"].long()[:, None])[:, 0]), entropy]
    if top:
        # Value in the high half (as an ordered integer), the lower id first.
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        key = order * (1 << 32) + (0xFFFFFFFF - torch.arange(vocab, device=x.device))
        ids = 0xFFFFFFFF - (key.topk(top, dim=1).values & 0xFFFFFFFF)
        out += [ids.to(torch.int32), logprob(z.gather(1, ids))]
    return out


def _plain_commit(s):
    """Every source row read, then every destination written."""
    src = s["offset"] + torch.from_numpy(s["nodes"].astype(np.int64)).cuda()
    dst = s["offset"] + torch.arange(len(s["nodes"]), device="cuda")
    table, pool = s["table"].long(), s["pool"]
    pool[:, :, table[dst // PAGE], :, dst % PAGE] = pool[:, :, table[src // PAGE], :, src % PAGE]
    return pool


def _plan(s):
    """The call's arguments, as a program that holds these buffers keeps them."""
    from cheetah_amd import hip

    hip.init(0)
    f32 = int(s.get("kv", s.get("logits")) == "f32")  # formats: 0 = BF16, 1 = f32
    if s["kind"] == "tree":
        view = hip.KvView(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), PAGE, s["kv_heads"], s["hd"])
        args = (s["q"].data_ptr(), ctypes.byref(view), f32, s["q_heads"], s["parents"].data_ptr(), s["n"],
                s["offset"], s["out"].data_ptr())
        return hip.check, hip.lib().cheetah_hip_tree_attention, args, s["out"], view
    if s["kind"] == "logprobs":
        o = [t.data_ptr() for t in s["out"]] + [None, None]
        args = (s["x"].data_ptr(), f32, s["rows"], s["vocab"], s["x"].stride(0), s["tokens"].data_ptr(), s["top"],
                o[0], o[1], o[2], o[3])
        return hip.check, hip.lib().cheetah_hip_logprobs, args, s["out"], None
    pool = s["pool"]
    views = (hip.KvView * s["layers"])(*(hip.KvView(pool[i, 0].data_ptr(), pool[i, 1].data_ptr(),
                                                    s["table"].data_ptr(), PAGE, s["kv_heads"], s["hd"])
                                         for i in range(s["layers"])))
    args = (views, s["layers"], f32, s["offset"], s["nodes"].ctypes.data_as(ctypes.POINTER(ctypes.c_uint32)),
            s["count"])
    return hip.check, hip.lib().cheetah_hip_tree_commit, args, pool, None


def _run_own(s):
    if "plan" not in s:
        s["plan"] = _plan(s)
    check, call, args, out, _ = s["plan"]
    check(call(*args))
    return out


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------

def work(case):
    e = 4 if "f32" in (case.get("kv"), case.get("logits")) else 2
    if case["kind"] == "tree":
        qh, kvh, hd, n, offset = case["q_heads"], case["kv_heads"], case["hd"], case["n"], case["offset"]
        depth = np.ones(n)
        for i, p in enumerate(_parents(case, 0)[1:], 1):
            depth[i] = depth[p] + 1
        return {"bytes": 2 * (offset + n) * kvh * hd * e + 2 * 4 * n * qh * hd + 4 * n,
                "flops": 4 * qh * hd * (n * offset + float(depth.sum()))}
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # Difference, exponential, two sums and a comparison for each logit.
        return {"bytes": rows * vocab * e + rows * (12 + 8 * case["top"]), "flops": 6 * rows * vocab}
    row = 2 * case["layers"] * case["kv_heads"] * case["hd"] * e
    return {"bytes": 2 * row * (case["count"] - 1) + 4 * case["count"], "flops": 0}


# ---------------------------------------------------------------------------
# The same results in 64 bits, from the definitions.
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tree":
        return _exact_tree(s)
    if case["kind"] == "logprobs":
        return _exact_logprobs(s)
    pool, table = s["pool"].double(), s["table"].tolist()
    before = pool.clone()
    for j, node in enumerate(s["nodes"].tolist()):
        to, at = s["offset"] + j, s["offset"] + node
        pool[:, :, table[to // PAGE], :, to % PAGE] = before[:, :, table[at // PAGE], :, at % PAGE]
    return pool


def _exact_tree(s):
    qh, kvh, hd, n, offset = s["q_heads"], s["kv_heads"], s["hd"], s["n"], s["offset"]
    parents = s["parents"].tolist()
    hidden = np.ones((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            hidden[i, j] = False
            j = parents[j]
    mask = torch.zeros(n, offset + n, dtype=torch.bool, device="cuda")
    mask[:, offset:] = torch.from_numpy(hidden).cuda()
    table = s["table"].long()
    k, v = (s[c].index_select(0, table) for c in "kv")
    out = torch.empty(n, qh, hd, dtype=torch.float64, device="cuda")
    for h in range(qh):
        g = h // (qh // kvh)
        kh, vh = (t[:, g].reshape(-1, hd)[:offset + n].double() for t in (k, v))
        score = s["q"].view(n, qh, hd)[:, h].double().contiguous() @ kh.t().contiguous() * hd ** -0.5
        out[:, h] = torch.softmax(score.masked_fill_(mask, -math.inf), 1) @ vh
    return out.reshape(n, qh * hd)


def _exact_logprobs(s):
    top, out = s["top"], [[], [], [], []]
    for row, token in zip(s["x"], s["tokens"].tolist()):
        x = row[:s["vocab"]].double()
        if bool((x == -math.inf).all()):
            lp, entropy = x, x.new_zeros(())
        else:
            m = x.max()
            tail = torch.exp(x - m)
            tail[x.argmax()] = 0
            lp = x - m - torch.log1p(tail.sum())  # exact where one token is nearly certain
            entropy = -(torch.exp(lp) * lp.clamp(min=-1e6)).sum()
        out[0].append(lp[token])
        out[1].append(entropy)
        if top:
            value, index = torch.sort(x, descending=True, stable=True)
            out[2].append(index[:top].to(torch.int32))
            out[3].append(lp[index[:top]])
    return [torch.stack(o) for o in out if o]
