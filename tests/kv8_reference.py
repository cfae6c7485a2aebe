"""The 8-bit K/V cache restated in 64 bits: its codes, its scales, its attention."""
import numpy as np

BLOCK, LEAST, MOST = 32, -117, 119


def code_values():
    """What the 256 E4M3 codes stand for."""
    out = np.empty(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        out[c] = np.nan if c & 127 == 127 else (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
        if c & 128:
            out[c] = -out[c]
    return out


_VALUES = code_values()
_POSITIVE = _VALUES[:127]  # ascending, the last 448


def encode(y):
    """The nearest code of each value, ties to an even code; magnitudes past 448
    as that, infinities and NaN as NaN."""
    y = np.asarray(y, np.float64)
    a = np.minimum(np.where(np.isfinite(y), np.abs(y), 0), 448.0)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 1, 126)
    lo = hi - 1
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.isfinite(y), code, 0x7F).astype(np.uint8)
    return code | (np.signbit(y) & np.isfinite(y)).astype(np.uint8) << 7


def exponent(x):
    """The least e with every finite |x| <= 448 * 2^e, in the scale's range."""
    a = np.abs(np.asarray(x, np.float64))
    most = a[np.isfinite(a)].max(initial=0.0)
    if most == 0:
        return LEAST
    e = LEAST
    while e < MOST and most > 448 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """Rows as the cache holds them: appended in any pieces, read as values."""

    def __init__(self, positions, kvh, hd):
        blocks = -(-positions // BLOCK)
        self.codes = np.full((2, blocks * BLOCK, kvh, hd), 0x7F, np.uint8)
        self.exps = np.full((2, blocks, kvh), LEAST)

    def append(self, k, v, offset):
        n = len(k)
        for t, x in enumerate((k, v)):
            x = np.asarray(x, np.float64).reshape(n, *self.codes.shape[2:])
            for b in range(offset // BLOCK, (offset + n - 1) // BLOCK + 1):
                lo, hi = max(b * BLOCK, offset), min((b + 1) * BLOCK, offset + n)
                for h in range(x.shape[1]):
                    rows = x[lo - offset:hi - offset, h]
                    e = exponent(rows)
                    if lo > b * BLOCK:
                        old = self.exps[t, b, h]
                        e = max(e, old)
                        at = (t, slice(b * BLOCK, lo), h)
                        if e > old:
                            kept = _VALUES[self.codes[at]]
                            self.codes[at] = np.where(np.isnan(kept), self.codes[at], encode(kept * 2.0 ** (old - e)))
                    self.exps[t, b, h] = e
                    self.codes[t, lo:hi, h] = encode(rows * 2.0 ** -e)

    def values(self, begin, n):
        e = np.repeat(self.exps, BLOCK, axis=1)[:, begin:begin + n]
        return tuple(_VALUES[self.codes[:, begin:begin + n]] * 2.0 ** e[..., None])


def attention64(q, k, v, q_heads, offset, window=0, sinks=0):
    """k, v: [positions, kvh, hd] values; q [rows, q_heads * hd]."""
    kvh, hd = k.shape[1:]
    rows = len(q)
    q = np.asarray(q, np.float64).reshape(rows, q_heads, hd)
    out = np.empty((rows, q_heads, hd))
    for i in range(rows):
        pos = offset + i
        p = np.arange(pos + 1)
        seen = p[(p > pos - window) | (p < sinks)] if window else p
        for h in range(q_heads):
            g = h // (q_heads // kvh)
            s = k[seen, g] @ q[i, h] / np.sqrt(hd)
            with np.errstate(invalid="ignore"):
                w = np.exp(s - s.max())
                out[i, h] = (w / w.sum()) @ v[seen, g]
    return out.reshape(rows, -1)


def some_rows(rng, n, kvh, hd):
    """Keys with a few large channels, values whose positions differ in size."""
    k = rng.standard_normal((n, kvh, hd)).astype(np.float32)
    k[..., 3::29] += 5
    v = (rng.standard_normal((n, kvh, hd)) * np.exp(0.8 * rng.standard_normal((n, 1, 1)))).astype(np.float32)
    return k, v


def decoder64(shape, w, tokens, cache, window=0):
    """The decoder's logits at every position of `tokens` in 64 bits, and each
    layer's rotated K and V rows before they are quantised. cache(layer): the K and V
    values [positions, kvh, hd] that attention reads; w: widened weights."""
    n, hd = len(tokens), shape.head_dim
    half = shape.rotary_dim // 2

    def norm(x, gain):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + shape.rms_eps) * gain

    freq = np.float32(shape.rope_theta) ** (np.float32(-2) * np.arange(half, dtype=np.float32) / np.float32(2 * half))
    angle = (np.arange(n, dtype=np.float32)[:, None] * freq.astype(np.float32)).astype(np.float64)[:, None]

    def rotate(x):
        a, b = x[..., :half], x[..., half:2 * half]
        c, s = np.cos(angle), np.sin(angle)
        return np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)

    x, rows = w["model.embed_tokens.weight"][tokens], []
    for layer in range(shape.num_layers):
        p = f"model.layers.{layer}."
        h = norm(x, w[p + "input_layernorm.weight"])
        q, k, v = (h @ w[p + f"self_attn.{c}_proj.weight"].T + w.get(p + f"self_attn.{c}_proj.bias", 0) for c in "qkv")
        q = rotate(q.reshape(n, -1, hd)).reshape(n, -1)
        rows.append((rotate(k.reshape(n, -1, hd)), v.reshape(n, -1, hd)))
        x = x + attention64(q, *cache(layer), shape.q_heads, 0, window) @ w[p + "self_attn.o_proj.weight"].T
        h = norm(x, w[p + "post_attention_layernorm.weight"])
        g = h @ w[p + "mlp.gate_proj.weight"].T
        x = x + (g / (1 + np.exp(-g)) * (h @ w[p + "mlp.up_proj.weight"].T)) @ w[p + "mlp.down_proj.weight"].T
    x = norm(x, w["model.norm.weight"])
    return x @ w["model.embed_tokens.weight" if shape.tie_word_embeddings else "lm_head.weight"].T, rows
