"""64-bit restatements of tree attention and of log probabilities, and the
trees and caches their tests use."""
import numpy as np

from cheetah_amd import synth


def parents_of(kind, n, rng):
    p = np.arange(n) - 1
    if kind == "star":
        p[1:] = 0
    elif kind == "roots":  # a forest
        p = np.where(rng.random(n) < 0.4, -1, np.floor(rng.random(n) * np.arange(n)))
    elif kind == "random":
        p = np.maximum(np.arange(n) - rng.integers(1, 9, n), 0)
    p[0] = -1
    return p.astype(np.int32)


def seen_by(parents):
    """Per node its ancestors and itself; a parent outside [0, i) ends the walk."""
    out = []
    for i in range(len(parents)):
        path = [i]
        while 0 <= parents[path[-1]] < path[-1]:
            path.append(int(parents[path[-1]]))
        out.append(path[::-1])
    return out


def attention64(q, k, v, q_heads, parents, offset):
    """q [n, q_heads * hd], k / v [offset + n, kv_heads, hd]."""
    n = len(parents)
    _, kvh, hd = k.shape
    q = q.reshape(n, q_heads, hd).astype(np.float64)
    k, v = k.astype(np.float64), v.astype(np.float64)
    out = np.empty((n, q_heads, hd))
    for i, path in enumerate(seen_by(parents)):
        at = np.concatenate([np.arange(offset), offset + np.array(path)])
        for h in range(q_heads):
            g = h // (q_heads // kvh)
            s = k[at, g] @ q[i, h] / np.sqrt(hd)
            w = np.exp(s - s.max())
            out[i, h] = w @ v[at, g] / w.sum()
    return out.reshape(n, -1)


def make_cache(rng, ctx, kvh, hd, kv):
    """K and V values [ctx, kvh, hd] as the cache type holds them (f32 arrays)."""
    k, v = (rng.standard_normal((ctx, kvh, hd)).astype(np.float32) for _ in "kv")
    if kv == "bf16":
        k, v = (synth.bf16_to_f32(synth.f32_to_bf16(t)).reshape(t.shape) for t in (k, v))
    return k, v


def paged(k, v, kv, rng, page=64, spare=2, fill=np.nan):
    """Shuffled pages [page][kv_head][position][hd] of the cache type and the
    page table; positions without a row hold `fill`, as does the whole of the
    pool's spare pages."""
    ctx, kvh, hd = k.shape
    need = -(-ctx // page)
    table = rng.permutation(need + spare)[:need].astype(np.int32)
    pools = []
    for t in (k, v):
        pool = np.full((need + spare, kvh, page, hd), fill, np.float32)
        for lp in range(need):
            rows = t[lp * page:(lp + 1) * page]
            pool[table[lp], :, :len(rows)] = rows.transpose(1, 0, 2)
        pools.append(pool if kv == "f32" else synth.f32_to_bf16(pool).reshape(pool.shape))
    return pools[0], pools[1], table


def logprobs64(x, tokens, top):
    """Log probabilities of the tokens, entropies, ids and log probabilities of
    the alternatives of rows of finite or -inf logits."""
    x = np.asarray(x, np.float64)
    rows, vocab = x.shape
    lp = np.full(x.shape, -np.inf)
    entropy = np.zeros(rows)
    for r in range(rows):
        m = x[r].max()
        if m == -np.inf:
            continue
        first = int(x[r].argmax())
        e = np.exp(x[r] - m)
        e[first] = 0
        lp[r] = x[r] - m - np.log1p(e.sum())
        p = np.exp(lp[r])
        entropy[r] = -(p[p > 0] * lp[r][p > 0]).sum()
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return lp[np.arange(rows), tokens], entropy, ids, np.take_along_axis(lp, ids, 1)
