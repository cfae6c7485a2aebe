"""The operators of an 8-bit K/V cache, as measurable cases.

A decoder that serves long contexts holds more of them when a cached value
takes one byte. Three calls of the C-ABI stand for that beside the calls over
BF16 and f32 caches (``perf/cases.py`` and ``perf/operators.py`` have those):

* ``cheetah_hip_kv8_append``: K/V rows are quantised as they are written:
  E4M3 codes with one power-of-two scale for each block of 32 positions of a
  KV head, grown when a later row of the block needs it.
* ``cheetah_hip_kv8_read``: cached rows come back as f32 or BF16.
* ``cheetah_hip_kv8_attention``: causal attention of one token or a chunk over
  such a cache, over all of it or over a sliding window and a few first
  positions that stay visible (sinks).

A block holds its codes in the order in which the matrix cores take them: K as
``[head_dim / 32][32 positions][32 dims]``, V as ``[head_dim][32 positions]``.

``own`` selects the framework's calls; otherwise ``run`` computes the same in
elementary torch operations. Head layouts are those of ``cheetah_amd.configs``
or generic.
"""
import ctypes
import math

import torch

own = False

PAGE, BLOCK = 64, 32
# (q heads, KV heads, head dim): the decoders served, then generic layouts.
HEADS = ((14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 64), (6, 2, 128), (5, 1, 64), (16, 2, 128))
SCALE_LEAST, SCALE_MOST = -117, 119     # exponents: every code times its scale is a normal f32
ATTEND_MOST = 32 * 128 * 512 * 4352     # q heads x head dim x keys that the rows see
SCORES_MOST = 32 * 1024 * 16384         # q heads x rows x keys in reach
ROWS_MOST = 4096 * 4 * 128              # values of K that a call writes
READ_MOST = 32768 * 4 * 128


def _attend(name, heads, rows, offset, window=0, sinks=0):
    qh, kvh, hd = heads
    return {"name": name, "kind": "attend", "q_heads": qh, "kv_heads": kvh, "hd": hd, "rows": rows, "offset": offset,
            "window": window, "sinks": sinks}


def listed():
    return [
        # One token of a small decoder over a short, ragged context: latency.
        _attend("attend_1_on_576", HEADS[0], 1, 576),
        # One token after a long document.
        _attend("attend_1_on_32k", HEADS[2], 1, 32767),
        # One token of an endless conversation: the last 4,096 and the first four positions.
        _attend("attend_1_window_4k", HEADS[1], 1, 19999, 4096, 4),
        # A user's short turn late in a conversation.
        _attend("attend_13_on_2k", HEADS[1], 13, 1999),
        # A short prompt through the small decoder.
        _attend("attend_333_on_0", HEADS[0], 333, 0),
        # A chunk of a long prompt under a sliding window.
        _attend("attend_1000_window_1k", HEADS[2], 1000, 7001, 1024, 16),
        # A chunk late in a long prompt: the largest.
        _attend("attend_512_on_4k", HEADS[1], 512, 4096),
        # The row of one decoded token, into a block that has rows already, and the block read back.
        {"name": "store_1", "kind": "store", "q_heads": 14, "kv_heads": 2, "hd": 64, "rows": 1, "offset": 577,
         "type": "f32", "packed": True},
        # A chunk's rows out of the packed projections, ragged at both ends, and what the cache then holds.
        {"name": "store_500", "kind": "store", "q_heads": 32, "kv_heads": 8, "hd": 128, "rows": 500, "offset": 1003,
         "type": "f32", "packed": True},
        # A long BF16 prompt taken over into an 8-bit cache.
        {"name": "store_4096_bf16", "kind": "store", "q_heads": 28, "kv_heads": 4, "hd": 128, "rows": 4096,
         "offset": 0, "type": "bf16", "packed": False},
        # A few cached rows looked at.
        {"name": "read_70", "kind": "read", "kv_heads": 8, "hd": 128, "begin": 1001, "n": 70, "type": "f32"},
        # A long prefix handed to a BF16 cache.
        {"name": "read_32k_bf16", "kind": "read", "kv_heads": 4, "hd": 128, "begin": 0, "n": 32768, "type": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "store", "read"))
    qh, kvh, hd = rng.choice(HEADS)
    if kind == "attend":
        case = {"kind": kind, "q_heads": qh, "kv_heads": kvh, "hd": hd,
                "rows": rng.choice((1, _log_int(rng, 1, 1024))),
                "offset": 0 if rng.random() < 0.05 else _log_int(rng, 1, 32768), "window": 0, "sinks": 0}
        if rng.random() < 0.5:
            case.update(window=_log_int(rng, 1, 8192), sinks=rng.choice((0, 4, _log_int(rng, 1, 200))))
        while qh * hd * int(_seen(case).sum()) > ATTEND_MOST or qh * case["rows"] * len(_reach(case)) > SCORES_MOST:
            case["offset"] //= 2
            case["rows"] = max(1, case["rows"] * 3 // 4)
        return case
    if kind == "store":
        return {"kind": kind, "q_heads": qh, "kv_heads": kvh, "hd": hd,
                "rows": min(_log_int(rng, 1, 4096), ROWS_MOST // (kvh * hd)), "offset": _log_int(rng, 1, 8192) - 1,
                "type": rng.choice(("f32", "bf16")), "packed": rng.random() < 0.5}
    return {"kind": kind, "kv_heads": kvh, "hd": hd, "begin": _log_int(rng, 1, 4096) - 1,
            "n": min(_log_int(rng, 1, 32768), READ_MOST // (kvh * hd)), "type": rng.choice(("f32", "bf16"))}


def _reach(case):
    """The positions that some row of the chunk sees, in order."""
    end, first = case["offset"] + case["rows"], 0
    if case["window"]:
        first = max(0, case["offset"] + 1 - case["window"])
    sinks = min(case["sinks"], first)
    return torch.cat([torch.arange(sinks), torch.arange(first, end)])


def _seen(case):
    """How many positions each row sees."""
    pos = case["offset"] + torch.arange(case["rows"])
    if not case["window"]:
        return pos + 1
    first = (pos + 1 - case["window"]).clamp(min=0)
    return pos + 1 - first + first.clamp(max=case["sinks"])


# ---------------------------------------------------------------------------
# The format: codes and scales of a block, in elementary operations.
# ---------------------------------------------------------------------------

def _two_to(e):
    """2 ** e of whole numbers -126 .. 127, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent_for(most):
    """The least e with most <= 448 * 2 ** e, within the scale's range."""
    fraction, e = torch.frexp(most)  # fraction in [1/2, 1)
    e = e - 9 + (fraction > 0.875).to(e.dtype)
    return torch.where(most > 0, e, torch.full_like(e, SCALE_LEAST)).clamp(SCALE_LEAST, SCALE_MOST)


def _encode(x, e):
    return (x.float() * _two_to(-e)[..., None, None]).to(torch.float8_e4m3fn)


def _decode(codes, e):
    return codes.float() * _two_to(e)[..., None, None]


def _rows_to_blocks(x, kvh, hd):
    """[32 blocks of rows, KV heads * hd] -> [blocks, KV heads, 32, hd]"""
    return x.view(-1, BLOCK, kvh, hd).transpose(1, 2)


def _blocks_to_rows(x):
    blocks, kvh, _, hd = x.shape
    return x.transpose(1, 2).reshape(blocks * BLOCK, kvh * hd)


def _lay_k(codes):
    """[blocks, KV heads, 32, hd] -> the order of a K block."""
    b, kvh, _, hd = codes.shape
    return codes.view(b, kvh, BLOCK, hd // 32, 32).transpose(2, 3).contiguous()


def _take_k(codes, hd):
    """The reverse, of [..., hd / 32, 32, 32]."""
    return codes.transpose(-3, -2).reshape(*codes.shape[:-3], BLOCK, hd)


def _at(s, blocks):
    """Pages and block numbers in them of a list of block numbers."""
    per = PAGE // BLOCK
    return s["table"].long()[blocks // per], blocks % per


def _block_codes(s, which, blocks):
    """Codes as [blocks, KV heads, 32, hd] (float8) and exponents [blocks, KV heads]."""
    page, sub = _at(s, blocks)
    codes = s[which][page, :, sub].view(torch.float8_e4m3fn)
    codes = _take_k(codes, s["hd"]) if which == "k" else codes.transpose(-1, -2)
    return codes, s[which + "_scales"][page, :, sub].to(torch.int32) - 127


# ---------------------------------------------------------------------------
# Inputs, made from the seed alone.
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _some_rows(n, kvh, hd, g):
    """K/V rows of n positions: keys have a few large channels (biases of the
    projection), some positions are large as a whole."""
    k, v = (torch.randn(n, kvh, hd, generator=g, device="cuda") for _ in "kv")
    k[:, :, 5::29] *= 3
    k[:, :, 3::61] += 6
    v *= torch.exp(0.8 * torch.randn(n, 1, 1, generator=g, device="cuda"))
    return k.view(n, kvh * hd), v.view(n, kvh * hd)


def _pools(s, written, pages, g):
    """A shuffled paged cache whose first `written` positions hold rows; the
    others were never written (NaN codes)."""
    kvh, hd, per = s["kv_heads"], s["hd"], PAGE // BLOCK
    s["table"] = torch.randperm(pages + 2, generator=g, device="cuda")[:pages].to(torch.int32)
    blocks = -(-written // BLOCK)
    at = torch.arange(blocks, device="cuda")
    rows = _some_rows(blocks * BLOCK, kvh, hd, g)
    for which, x in zip("kv", rows):
        x = _rows_to_blocks(x, kvh, hd)
        there = (at[:, None] * BLOCK + torch.arange(BLOCK, device="cuda") < written)[:, None, :, None]
        e = _exponent_for((x * there).abs().amax((-1, -2)))
        codes = _encode(x, e).view(torch.uint8)
        codes = torch.where(there, codes, torch.full_like(codes, 0x7F))
        codes = _lay_k(codes) if which == "k" else codes.transpose(-1, -2).contiguous()
        pool = torch.full((pages + 2, kvh, per, *codes.shape[2:]), 0x7F, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(pages + 2, kvh, per, dtype=torch.uint8, device="cuda")
        page, sub = _at(s, at)
        pool[page, :, sub] = codes
        scales[page, :, sub] = (e + 127).to(torch.uint8)
        s[which], s[which + "_scales"] = pool, scales


def _row_type(case):
    return torch.float32 if case["type"] == "f32" else torch.bfloat16


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    kvh, hd = case["kv_heads"], case["hd"]
    if case["kind"] == "attend":
        rows, end = case["rows"], case["offset"] + case["rows"]
        _pools(s, end, -(-end // PAGE), g)
        reach = _reach(case)
        gone = torch.ones(s["table"].numel(), dtype=torch.bool)
        gone[reach // PAGE] = False
        s["table"][gone.cuda()] = -1  # pages behind the window were given back
        width = case["q_heads"] * hd
        s.update(q=torch.randn(rows, width, generator=g, device="cuda") * 1.2, reach=reach.cuda(),
                 out=torch.empty(rows, width, device="cuda"))
        return s
    if case["kind"] == "store":
        end = case["offset"] + case["rows"]
        _pools(s, case["offset"], -(-end // PAGE), g)
        k, v = (x.to(_row_type(case)) for x in _some_rows(case["rows"], kvh, hd, g))
        if case["packed"]:  # the rows of the fused projection: q, then k, then v
            packed = torch.zeros(case["rows"], (case["q_heads"] + 2 * kvh) * hd, dtype=k.dtype, device="cuda")
            at = case["q_heads"] * hd
            packed[:, at:at + kvh * hd], packed[:, at + kvh * hd:] = k, v
            k, v = packed[:, at:at + kvh * hd], packed[:, at + kvh * hd:]
        begin = case["offset"] // BLOCK * BLOCK
        s.update(rows_k=k, rows_v=v, begin=begin, n=end - begin)
    else:
        end = case["begin"] + case["n"]
        _pools(s, end, -(-end // PAGE), g)
    s["out"] = [torch.empty(s["n"], kvh * hd, dtype=_row_type(case), device="cuda") for _ in "kv"]
    return s


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "attend":
        return _plain_attend(state)
    if state["kind"] == "store":
        _plain_append(state)
    return _plain_read(state)


def _plain_attend(s):
    kvh, hd, rows, reach = s["kv_heads"], s["hd"], s["rows"], s["reach"]
    group = s["q_heads"] // kvh
    blocks = torch.unique_consecutive(reach // BLOCK)
    at = torch.searchsorted(blocks, reach // BLOCK) * BLOCK + reach % BLOCK

    def cached(which):  # [KV heads, keys in reach, hd]
        x = _decode(*_block_codes(s, which, blocks)).transpose(0, 1).reshape(kvh, -1, hd)
        return x[:, at].contiguous()

    q = s["q"].view(rows, kvh, group, hd).transpose(0, 1).reshape(kvh, rows * group, hd)
    scores = q @ cached("k").transpose(1, 2).contiguous() / math.sqrt(hd)
    pos = s["offset"] + torch.arange(rows, device=q.device)[:, None]
    seen = reach[None, :] <= pos
    if s["window"]:
        seen &= (reach[None, :] > pos - s["window"]) | (reach[None, :] < s["sinks"])
    scores = scores.view(kvh, rows, group, -1).masked_fill_(~seen[None, :, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(kvh, rows * group, -1)
    return (p @ cached("v")).view(kvh, rows, group, hd).transpose(0, 1).reshape(rows, -1)


def _plain_append(s):
    kvh, hd, offset, rows = s["kv_heads"], s["hd"], s["offset"], s["rows"]
    first, last = offset // BLOCK, (offset + rows - 1) // BLOCK
    blocks = torch.arange(first, last + 1, device="cuda")
    at = offset - first * BLOCK
    place = blocks[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    new = ((place >= offset) & (place < offset + rows))[:, None, :, None]
    earlier = (blocks * BLOCK < offset)[:, None]
    page, sub = _at(s, blocks)
    for which in "kv":
        x = torch.zeros(blocks.numel() * BLOCK, kvh * hd, device="cuda")
        x[at:at + rows] = s["rows_" + which].float()
        x = _rows_to_blocks(x, kvh, hd)
        codes, e_old = _block_codes(s, which, blocks)
        e = _exponent_for(x.abs().amax((-1, -2)))
        e = torch.where(earlier, torch.maximum(e, e_old), e)
        # Earlier rows are rounded again to a grown scale; rows behind the last one stay as they are.
        kept = torch.where(earlier, _two_to((e_old - e).clamp(min=-126)), torch.ones(1, device="cuda"))
        kept = (codes.float() * kept[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        kept = torch.where((place < offset)[:, None, :, None], kept, codes.view(torch.uint8))
        codes = torch.where(new, _encode(x, e).view(torch.uint8), kept)
        s[which][page, :, sub] = _lay_k(codes) if which == "k" else codes.transpose(-1, -2).contiguous()
        s[which + "_scales"][page, :, sub] = (e + 127).to(torch.uint8)


def _plain_read(s):
    first = s["begin"] // BLOCK
    blocks = torch.arange(first, (s["begin"] + s["n"] - 1) // BLOCK + 1, device="cuda")
    at = s["begin"] - first * BLOCK
    return [_blocks_to_rows(_decode(*_block_codes(s, which, blocks)))[at:at + s["n"]].to(_row_type(s))
            for which in "kv"]


def _plan(s):
    """The calls' arguments, as a program that holds these buffers keeps them."""
    from cheetah_amd import hip

    hip.init(0)
    lib = hip.lib()
    view = hip.Kv8View(*(s[p].data_ptr() for p in ("k", "v", "k_scales", "v_scales", "table")), PAGE, s["kv_heads"],
                       s["hd"])
    ref = ctypes.byref(view)
    if s["kind"] == "attend":
        calls = [(lib.cheetah_hip_kv8_attention, (s["q"].data_ptr(), ref, s["q_heads"], s["rows"], s["offset"],
                                                  s["window"], s["sinks"], s["out"].data_ptr()))]
        return hip.check, calls, view
    f32 = int(s["type"] == "f32")  # formats: 0 = BF16, 1 = f32
    calls = [(lib.cheetah_hip_kv8_read, (ref, s["begin"], s["n"], f32, *(t.data_ptr() for t in s["out"])))]
    if s["kind"] == "store":
        k, v = s["rows_k"], s["rows_v"]
        calls.insert(0, (lib.cheetah_hip_kv8_append, (k.data_ptr(), v.data_ptr(), f32, s["rows"], k.stride(0),
                                                      s["offset"], ref)))
    return hip.check, calls, view


def _run_own(s):
    if "plan" not in s:
        s["plan"] = _plan(s)
    check, calls, _ = s["plan"]
    for call, args in calls:
        check(call(*args))
    return s["out"]


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------

def work(case):
    kvh, hd = case["kv_heads"], case["hd"]
    if case["kind"] == "attend":
        row = case["q_heads"] * hd
        keys = len(_reach(case))
        return {"bytes": 2 * keys * kvh * hd + 2 * 4 * case["rows"] * row, "flops": 4 * row * int(_seen(case).sum())}
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "read":
        return {"bytes": 2 * case["n"] * kvh * hd * (1 + size), "flops": 0}
    n = case["offset"] % BLOCK + case["rows"]
    # Rows in, codes out, then codes in and rows out; a comparison and a product for each value.
    return {"bytes": 2 * kvh * hd * (case["rows"] * (size + 1) + n * (1 + size)), "flops": 4 * case["rows"] * kvh * hd}


# ---------------------------------------------------------------------------
# The same results in 64 bits, from the definitions.
# ---------------------------------------------------------------------------

def _e4m3_values():
    """What each of the 256 codes stands for: sign, four bits of exponent (bias
    7, none of them infinite), three of fraction."""
    table = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        value = math.nan if code & 127 == 127 else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        table.append(-value if code & 128 else value)
    return torch.tensor(table, dtype=torch.float64, device="cuda")


def _round_e4m3(y):
    """To the nearest of those values, ties to an even fraction."""
    unit = torch.exp2((torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))) - 3).clamp(min=-9))
    return torch.round(y / unit) * unit


def _exact_values(s, which, first, end):
    """Rows [first, end) of the cache and the exponent of each one's block:
    [rows, KV heads, hd], [rows, KV heads]."""
    pos = torch.arange(first, end, device="cuda")
    page, sub, row = s["table"].long()[pos // PAGE], pos % PAGE // BLOCK, pos % BLOCK
    codes = s[which][page, :, sub, :, row] if which == "k" else s[which][page, :, sub, :, :]
    codes = codes.flatten(2) if which == "k" else codes.gather(
        3, row[:, None, None, None].expand(-1, codes.shape[1], codes.shape[2], 1))[..., 0]
    return _e4m3_values()[codes.long()], s[which + "_scales"][page, :, sub].double() - 127


def exact(case, seed):
    s = prepare(case, seed)
    kvh, hd = case["kv_heads"], case["hd"]
    if case["kind"] == "read":
        out = []
        for which in "kv":
            value, e = _exact_values(s, which, s["begin"], s["begin"] + s["n"])
            out.append((value * torch.exp2(e)[..., None]).reshape(s["n"], kvh * hd))
        return out
    if case["kind"] == "store":
        return [_exact_store(s, which) for which in "kv"]
    return _exact_attend(s)


def _exact_store(s, which):
    kvh, hd, offset = s["kv_heads"], s["hd"], s["offset"]
    begin, end, out = s["begin"], offset + s["rows"], []
    new = s["rows_" + which].double().view(s["rows"], kvh, hd)
    for b in range(begin, end, BLOCK):
        stop = min(b + BLOCK, end)
        here = new[max(b, offset) - offset:stop - offset]
        most = here.abs().amax((0, 2))
        e = torch.ceil(torch.log2(most / 448)).clamp(SCALE_LEAST, SCALE_MOST)
        rows = []
        if b < offset:
            value, old = _exact_values(s, which, b, offset)
            e = torch.maximum(e, old[0])
            rows.append(_round_e4m3(value * torch.exp2(old - e)[..., None]))
        rows.append(_round_e4m3(here / torch.exp2(e)[:, None]))
        out.append(torch.cat(rows) * torch.exp2(e)[:, None])
    return torch.cat(out).reshape(end - begin, kvh * hd)


def _exact_attend(s):
    qh, kvh, hd, rows, offset = s["q_heads"], s["kv_heads"], s["hd"], s["rows"], s["offset"]
    reach = s["reach"]
    gap = (reach[1:] != reach[:-1] + 1).nonzero().flatten().tolist()  # behind the sinks, if anywhere
    split = gap[0] + 1 if gap else 0
    runs = [(0, split)] * (split > 0) + [(int(reach[split]), int(reach[-1]) + 1)]

    def cached(which):
        parts = [_exact_values(s, which, a, b) for a, b in runs]
        return torch.cat([v * torch.exp2(e)[..., None] for v, e in parts])

    k, v = cached("k"), cached("v")
    pos = offset + torch.arange(rows, device="cuda")[:, None]
    hidden = reach[None, :] > pos
    if s["window"]:
        hidden |= (reach[None, :] <= pos - s["window"]) & (reach[None, :] >= s["sinks"])
    out = torch.empty(rows, qh, hd, dtype=torch.float64, device="cuda")
    for h in range(qh):
        g = h // (qh // kvh)
        score = s["q"].view(rows, qh, hd)[:, h].double().contiguous() @ k[:, g].t().contiguous() * hd ** -0.5
        out[:, h] = torch.softmax(score.masked_fill_(hidden, -math.inf), 1) @ v[:, g].contiguous()
    return out.reshape(rows, qh * hd)
