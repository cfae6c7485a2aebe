"""Tree attention's part products restated on the host: what the output loses
when one of them is missing. Everything else is in 64 bits, so that an error here
is the missing product's alone."""
import numpy as np

import tree_reference as ref


def cut(x):
    """Three BF16 parts, each the top 8 bits of what the ones before leave, in 64
    bits: their sum is the f32 value."""
    left, out = np.ascontiguousarray(x, np.float32), []
    for _ in range(3):
        part = (left.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out.append(part.astype(np.float64))
        left = left - part
    return out


def products(kv):
    """(part of the cache's value, part of the f32 operand): three with a BF16
    cache, which is one part itself, six of nine with an f32 one."""
    return [(0, 0), (0, 1), (0, 2)] if kv == "bf16" else [(0, 0), (0, 1), (1, 0), (0, 2), (1, 1), (2, 0)]


def attention_parts(q, k, v, q_heads, parents, offset, kv, score_products, value_products):
    """ref.attention64 with the listed products only."""
    n = len(parents)
    _, kvh, hd = k.shape
    scale = np.float32(1 / np.sqrt(np.float32(hd))) * np.float32(1.44269504088896340736)
    qp = cut(q.reshape(n, q_heads, hd) * scale)
    kp, vp = (cut(t) if kv == "f32" else [t.astype(np.float64)] for t in (k, v))
    out = np.empty((n, q_heads, hd))
    for i, path in enumerate(ref.seen_by(parents)):
        at = np.concatenate([np.arange(offset), offset + np.array(path)])
        for h in range(q_heads):
            g = h // (q_heads // kvh)
            s = sum(kp[a][at, g] @ qp[b][i, h] for a, b in score_products)
            w = np.exp2(s - s.max()).astype(np.float32)
            p = cut(w)
            out[i, h] = sum(p[b] @ vp[a][at, g] for a, b in value_products) / w.astype(np.float64).sum()
    return out.reshape(n, -1)


def norm_err(got, want):
    """Relative to the output's norm."""
    return float(np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want))


# Bars for errors relative to the output's norm. A score is an f32 sum of 24 matrix
# products (f32 cache: 48, all but 8 of them small ones), each rounded to 2^-24 of a
# partial sum, some 0.6 of the score's s log2 units: sqrt(24) * 2^-24 / sqrt(3) *
# 0.6 s ln 2 of its weight. Ordinary scores (s 2): 2e-7; the running sums of weights
# and outputs (200 steps of 2^-25 at random) 4e-7; exponentials (2^-23 at random)
# 7e-8: 5e-7 together, four deviations. Scores in the hundreds (s 150): 1.1e-5, in
# rows whose largest keys are close enough to share the weight.
ORDINARY, LARGE = 2e-6, 1.2e-5
