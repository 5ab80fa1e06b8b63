"""Workloads of the 4-bit reader operators: what is run, on which inputs, in a plain torch form
and through this package.

The operators (``coraanns_b200.lowbit``) serve a language model that reads what the search
retrieved, on the GPU that already holds the index: its weights and its attention cache are
kept in 4 bits, because the index takes most of the memory.

* append:  rotate new keys (and queries) by position, quantise keys and values to 4 bits, store
           them in a paged cache;
* attend:  softmax attention of one or many new tokens per sequence over that cache;
* step:    append, then attend, as one decoding step of one layer does;
* matvec:  products of a few activation rows with a 4-bit weight matrix.

Format (all of them): a group of G consecutive values holds 4-bit codes c and two fp16 numbers,
and stands for  scale * c + low.  Quantisation of a group x:  low = fp16(min x),
scale = fp16((max x - min x) / 15),  c = clamp(round((x - low) * (1 / scale)), 0, 15), halves to
even, and c = 0 where scale is 0; scale and low saturate at the largest fp16.

Cache page, one block of bytes per (page, key head), P tokens of head size D:
P x D/2 bytes of key codes (byte j of a row: dimension 2j in the low half, 2j + 1 in the high
half), P x D/2 of value codes, P x D/G x (scale, low) of the keys, the same of the values.

Weight rows (N x K, K padded to 128 with zeros): a segment of 128 columns is 16 words of 32 bits;
the word stored at 4t + j holds columns 32j + 8t .. 32j + 8t + 7 of the segment, column e of
those 8 in the nibble (0, 4, 2, 6, 1, 5, 3, 7)[e].
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

PACKAGE = Path(__file__).resolve().parent.parent / "cgcl-coraanns_b200"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NIBBLE_OF = (0, 4, 2, 6, 1, 5, 3, 7)
FP16_MAX = 65504.0


def _lowbit():
    if str(PACKAGE) not in sys.path:
        sys.path.insert(0, str(PACKAGE))
    from coraanns_b200 import lowbit
    return lowbit


# ---- cases --------------------------------------------------------------------------------


def listed():
    return [
        # the next token of a single conversation: latency of one launch
        dict(name="append_one", kind="append", tokens=1, q_heads=32, kv_heads=8, dim=128, group=128,
             page=64, rotary=128, interleaved=False, dtype="bf16"),
        # one token of each of 61 conversations, small heads, partial interleaved rotation
        dict(name="append_batch", kind="append", tokens=61, q_heads=16, kv_heads=4, dim=64, group=64,
             page=16, rotary=32, interleaved=True, dtype="fp16"),
        # the prompt: retrieved passages entering the cache at once
        dict(name="append_prompt", kind="append", tokens=16384, q_heads=32, kv_heads=8, dim=128,
             group=64, page=64, rotary=128, interleaved=False, dtype="bf16"),
        # a short question: latency again, little work for many SMs
        dict(name="attend_short", kind="attend", seqs=1, queries=1, low=701, high=701, lengths=1,
             q_heads=32, kv_heads=8, dim=128, group=128, page=64, window=0, dtype="bf16"),
        # one reader over a very long context of retrieved text
        dict(name="attend_long", kind="attend", seqs=1, queries=1, low=131072, high=131072, lengths=1,
             q_heads=32, kv_heads=8, dim=128, group=128, page=64, window=0, dtype="bf16"),
        # many readers of very different context lengths in one batch
        dict(name="attend_batch", kind="attend", seqs=64, queries=1, low=200, high=16384, lengths=7,
             q_heads=32, kv_heads=8, dim=128, group=64, page=32, window=0, dtype="fp16"),
        # five drafted tokens per sequence checked at once, large heads, sliding window
        dict(name="attend_verify", kind="attend", seqs=24, queries=5, low=500, high=8192, lengths=3,
             q_heads=16, kv_heads=8, dim=256, group=128, page=16, window=4096, dtype="bf16"),
        # a chunk of a long prompt against everything before it (and itself)
        dict(name="attend_chunk", kind="attend", seqs=1, queries=2048, low=16384, high=16384, lengths=1,
             q_heads=32, kv_heads=8, dim=128, group=128, page=64, window=0, dtype="bf16"),
        # one decoding step of one layer for 32 sequences: append, then attend
        dict(name="step_batch", kind="step", seqs=32, queries=1, low=1000, high=8000, lengths=5,
             q_heads=32, kv_heads=4, dim=128, group=128, page=64, window=0, rotary=128,
             interleaved=False, dtype="bf16"),
        # a projection for one token
        dict(name="matvec_one", kind="matvec", rows=1, out=4096, inner=4096, group=128, bias=False,
             dtype="bf16"),
        # the largest projection for one token
        dict(name="matvec_wide", kind="matvec", rows=1, out=32768, inner=8192, group=128, bias=False,
             dtype="fp16"),
        # a small batch, ragged in every size, with a bias
        dict(name="matvec_batch", kind="matvec", rows=13, out=10007, inner=5000, group=64, bias=True,
             dtype="bf16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("append", "attend", "attend", "step", "matvec"))
        dtype = rng.choice(("bf16", "fp16"))
        if kind == "matvec":
            case = dict(kind=kind, rows=_log(rng, 1, 64), out=_log(rng, 64, 32768),
                        inner=_log(rng, 128, 16384), group=rng.choice((32, 64, 128)),
                        bias=rng.random() < 0.3, dtype=dtype)
        else:
            dim, group = rng.choice(((64, 64), (128, 64), (128, 128), (256, 64), (256, 128)))
            kv_heads = rng.choice((1, 2, 4, 8))
            case = dict(kind=kind, q_heads=kv_heads * rng.choice((1, 2, 4, 7, 8)), kv_heads=kv_heads,
                        dim=dim, group=group, page=rng.choice((16, 32, 64, 128)), dtype=dtype)
            if kind == "append":
                case["tokens"] = _log(rng, 1, 16384)
            else:
                case["seqs"] = _log(rng, 1, 64)
                case["queries"] = 1 if rng.random() < 0.4 else _log(rng, 1, 2048)
                case["high"] = max(case["queries"], _log(rng, 1, 131072))
                case["low"] = max(case["queries"], case["high"] // rng.choice((1, 4, 50)))
                case["lengths"] = rng.randrange(1 << 16)
                case["window"] = rng.choice((0, 0, 0, 1000))
            if kind != "attend":
                case["rotary"] = rng.choice((dim, dim // 2))
                case["interleaved"] = rng.random() < 0.5
        if _cost(case) <= most and _room(case) <= 24e9:
            return case


def _lengths(case):
    rng = random.Random(case["lengths"])
    return [_log(rng, case["low"], case["high"]) for _ in range(case["seqs"])]


def _room(case):
    """Bytes of the largest array of the plain form."""
    if case["kind"] in ("append", "matvec"):
        return 0
    longest = -(-max(_lengths(case)) // case["page"]) * case["page"]
    return 4 * case["seqs"] * longest * max(case["q_heads"] * case["queries"], case["kv_heads"] * case["dim"])


# ---- inputs -------------------------------------------------------------------------------


def _quantize(x, group):
    """fp32 values (..., D) -> codes, scale, low (..., D / G, G | 1 | 1); scale and low hold fp16."""
    g = x.unflatten(-1, (-1, group))
    least = g.amin(-1, keepdim=True)
    scale = ((g.amax(-1, keepdim=True) - least) / 15.0).clamp(max=FP16_MAX).half().float()
    low = least.clamp(-FP16_MAX, FP16_MAX).half().float()
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    return ((g - low) * inverse).round().clamp(0, 15), scale, low


def _block(codes_k, meta_k, codes_v, meta_v):
    """codes (..., P, D) and meta (..., P, D / G, 2) in fp16 -> page blocks (..., bytes)."""
    parts = []
    for c in (codes_k, codes_v):
        c = c.to(torch.uint8).unflatten(-1, (-1, 2))
        parts.append((c[..., 0] | (c[..., 1] << 4)).flatten(-2))
    for m in (meta_k, meta_v):
        parts.append(m.contiguous().view(torch.uint8).flatten(-3))
    return torch.cat(parts, -1)


def _dense(blocks, case):
    """Page blocks (..., bytes) -> the fp32 keys and values (..., P, D) that they stand for."""
    P, D, G = case["page"], case["dim"], case["group"]
    n, m = P * D // 2, P * (D // G) * 4
    out = []
    for c, s in ((blocks[..., :n], blocks[..., 2 * n:2 * n + m]),
                 (blocks[..., n:2 * n], blocks[..., 2 * n + m:])):
        codes = torch.stack((c & 15, c >> 4), -1).unflatten(-2, (P, D // 2)).flatten(-2).unflatten(-1, (-1, G))
        meta = s.contiguous().view(torch.float16).float().unflatten(-1, (P, D // G, 2))
        out.append((meta[..., :1] * codes + meta[..., 1:]).flatten(-2))
    return out


def _keys(shape, gen):
    """Keys or values: normal, with an offset of its own and a few loud channels per head."""
    x = torch.randn(shape, generator=gen, device="cuda")
    gain = torch.where(torch.rand(shape[-2:], generator=gen, device="cuda") < 0.03, 4.0, 1.0)
    return x * gain + 0.5 * torch.randn(shape[-2:], generator=gen, device="cuda")


def _rope(case, positions):
    half = case["rotary"] // 2
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * (
        10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    st = {"case": case, "handles": {}}
    if case["kind"] == "matvec":
        N, K, G = case["out"], case["inner"], case["group"]
        padded = -(-K // 128) * 128
        w = torch.randn(N, K, generator=gen, device="cuda") * (0.4 + torch.rand(N, 1, generator=gen, device="cuda"))
        codes, scale, low = _quantize(torch.nn.functional.pad(w, (0, padded - K)), G)
        codes = codes.flatten(-2).to(torch.int64).view(N, -1, 4, 4, 8).transpose(2, 3)  # segment, t, j, e
        shift = 4 * torch.tensor(NIBBLE_OF, device="cuda")
        words = (codes << shift).sum(-1)
        st["codes"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).reshape(N, -1).view(torch.uint8)
        st["meta"] = torch.cat((scale, low), -1).half()
        x = torch.randn(case["rows"], K, generator=gen, device="cuda")
        st["x"] = (x * torch.where(torch.rand(K, generator=gen, device="cuda") < 0.01, 8.0, 1.0)).to(dtype)
        st["bias"] = torch.randn(N, generator=gen, device="cuda").to(dtype) if case["bias"] else None
        return st
    H, Hq, D, P, G = (case[k] for k in ("kv_heads", "q_heads", "dim", "page", "group"))
    block = P * D + P * (D // G) * 8
    if case["kind"] == "append":
        T = case["tokens"]
        pages = -(-T // P) + 3
        lens, first = [T + 2 * P], 2 * P
    else:
        lens = _lengths(case)
        T = case["seqs"] * case["queries"]
        pages = sum(-(-n // P) for n in lens) + 3
    if case["kind"] != "attend":
        qkv = torch.cat((1.5 * torch.randn(T, Hq, D, generator=gen, device="cuda"), _keys((T, H, D), gen),
                         _keys((T, H, D), gen)), 1).to(dtype)  # one projection's output: strided views
        st["q"], st["k"], st["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
        st["cos"], st["sin"] = _rope(case, max(lens) + 1)
    else:
        st["q"] = (1.5 * torch.randn(T, Hq, D, generator=gen, device="cuda")).to(dtype)
    order = torch.randperm(pages, generator=gen, device="cuda")
    if case["kind"] == "append":
        st["pool"] = torch.zeros(pages, H, block, dtype=torch.uint8, device="cuda")
        where = torch.arange(first, first + T, device="cuda")
        st["positions"] = where.to(torch.int32)
        where = where - first
        st["slots"] = order[where // P] * P + where % P
        return st
    pool = []
    for at in range(0, pages, 2048):  # in pieces, for the memory of the fp32 values
        n = min(2048, pages - at)
        kv = []
        for _ in range(2):
            codes, scale, low = _quantize(_keys((n, P, H, D), gen).transpose(1, 2), G)
            kv += [codes.flatten(-2), torch.cat((scale, low), -1).half()]
        pool.append(_block(*kv))
    st["pool"] = torch.cat(pool)
    need = torch.tensor([-(-n // P) for n in lens], device="cuda")
    column = torch.arange(int(need.max()), device="cuda")
    index = (need.cumsum(0) - need)[:, None] + column
    st["page_table"] = torch.where(column < need[:, None], order[index.clamp(max=pages - 1)], -1).to(torch.int32)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["q_start"] = torch.arange(0, T + 1, case["queries"], dtype=torch.int32, device="cuda")
    if case["kind"] == "step":
        n = case["queries"]
        positions = (st["lens"][:, None] - n + torch.arange(n, device="cuda", dtype=torch.int32)).flatten()
        table = st["page_table"].repeat_interleave(n, 0).gather(1, (positions // P)[:, None].long())[:, 0]
        st["positions"] = positions
        st["slots"] = table.long() * P + positions % P
    return st


# ---- the plain forms ------------------------------------------------------------------------


def _rotate(x, cos, sin, case):
    """fp32 (T, heads, D): pairs (i, i + R/2), or (2i, 2i + 1) interleaved, of the first R dims."""
    R = case["rotary"]
    head, rest = x[..., :R], x[..., R:]
    a, b = (head[..., 0::2], head[..., 1::2]) if case["interleaved"] else (head[..., :R // 2], head[..., R // 2:])
    c, s = cos[:, None], sin[:, None]
    u, v = a * c - b * s, b * c + a * s
    turned = torch.stack((u, v), -1).flatten(-2) if case["interleaved"] else torch.cat((u, v), -1)
    return torch.cat((turned, rest), -1)


def _append_plain(st):
    case, dtype = st["case"], st["q"].dtype
    P, D, G, H = case["page"], case["dim"], case["group"], case["kv_heads"]
    at = st["positions"].long()
    cos, sin = st["cos"][at], st["sin"][at]
    q = _rotate(st["q"].float(), cos, sin, case).to(dtype)
    page, off = st["slots"] // P, st["slots"] % P
    pool, n, m = st["pool"], P * D // 2, P * (D // G) * 4
    codes_of = lambda at, size: pool[:, :, at:at + size].unflatten(-1, (P, -1))  # noqa: E731
    values = []
    for x, c_at, m_at in ((_rotate(st["k"].float(), cos, sin, case), 0, 2 * n), (st["v"].float(), n, 2 * n + m)):
        codes, scale, low = _quantize(x, G)
        values.append((scale * codes + low).flatten(-2).to(dtype))
        c = codes.flatten(-2).to(torch.uint8).unflatten(-1, (-1, 2))
        codes_of(c_at, n)[page, :, off] = c[..., 0] | (c[..., 1] << 4)
        codes_of(m_at, m)[page, :, off] = torch.cat((scale, low), -1).half().view(torch.uint8).flatten(-2)
    return {"q": q, "k": values[0], "v": values[1]}


def _visible(lens, queries, longest, window):
    """(B, n, L): whether query i of a sequence, at position len - n + i, sees token j."""
    j = torch.arange(longest, device=lens.device)
    i = lens[:, None] - queries + torch.arange(queries, device=lens.device)
    seen = j <= i[..., None]
    return seen & (j > i[..., None] - window) if window else seen


def _attend_plain(st, q):
    case = st["case"]
    B, n, H, D = case["seqs"], case["queries"], case["kv_heads"], case["dim"]
    K, V = _dense(st["pool"][st["page_table"].clamp(min=0).long()], case)  # (B, pages, H, P, D)
    K, V = K.transpose(1, 2).flatten(2, 3), V.transpose(1, 2).flatten(2, 3)
    Q = q.float().view(B, n, H, -1, D).permute(0, 2, 3, 1, 4)  # (B, H, g, n, D)
    scores = (Q.flatten(2, 3) @ K.transpose(-1, -2)).unflatten(2, (-1, n)) * D ** -0.5
    scores = scores.masked_fill(~_visible(st["lens"], n, K.shape[2], case["window"])[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ V).unflatten(2, (-1, n))
    return out.permute(0, 3, 1, 2, 4).reshape(B * n, -1, D).to(q.dtype)


def _matvec_plain(st):
    case = st["case"]
    shift = 4 * torch.tensor(NIBBLE_OF, device="cuda")
    codes = (st["codes"].view(torch.int32)[..., None] >> shift) & 15
    codes = codes.view(case["out"], -1, 4, 4, 8).transpose(2, 3).reshape(case["out"], -1, case["group"])
    meta = st["meta"].float()
    w = (meta[..., :1] * codes + meta[..., 1:]).flatten(-2)[:, :case["inner"]]
    y = st["x"].float() @ w.T
    return (y if st["bias"] is None else y + st["bias"].float()).to(st["x"].dtype)


# ---- one pass -------------------------------------------------------------------------------


def _cache(st):
    """The framework's cache over the pool, kept with the state as a user's program keeps it."""
    if "cache" not in st["handles"]:
        case = st["case"]
        st["handles"]["cache"] = _lowbit().Cache4.from_pool(st["pool"], page_size=case["page"], head_dim=case["dim"],
                                                            group=case["group"])
    return st["handles"]["cache"]


def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        if kind == "matvec":
            return _matvec_plain(st)
        if kind == "append":
            return _append_plain(st)
        q = _append_plain(st)["q"] if kind == "step" else st["q"]
        return _attend_plain(st, q)
    if kind == "matvec":
        if "weight" not in st["handles"]:
            st["handles"]["weight"] = _lowbit().Weight4(st["codes"], st["meta"], case["inner"])
        return _lowbit().matvec(st["x"], st["handles"]["weight"], bias=st["bias"])
    cache = _cache(st)
    q = st["q"]
    if kind != "attend":
        got = cache.append(st["k"], st["v"], st["slots"], q=q, rope=(st["cos"], st["sin"]), positions=st["positions"],
                           interleaved=case["interleaved"], values=kind == "append")
        if kind == "append":
            return {"q": got.q, "k": got.k, "v": got.v}
        q = got.q
    return cache.attend(q, st["page_table"], st["lens"], q_start=st["q_start"], max_queries=case["queries"],
                        window=case["window"])


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    if case["kind"] == "matvec":
        M, N, K, G = case["rows"], case["out"], case["inner"], case["group"]
        return {"bytes": N * K / 2 + 4 * N * -(-K // G) + 2 * M * (K + N) + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    H, Hq, D, G = case["kv_heads"], case["q_heads"], case["dim"], case["group"]
    row = H * (D + 8 * (D // G))  # a cached token, keys and values
    size, flops = 0, 0
    if case["kind"] != "attend":
        T = case["tokens"] if case["kind"] == "append" else case["seqs"] * case["queries"]
        values = 4 * T * H * D if case["kind"] == "append" else 0
        size += T * (4 * H * D + 4 * Hq * D + row + 4 * case["rotary"] + 12) + values
        flops += T * (3 * (H + Hq) * case["rotary"] + 8 * H * D)
    if case["kind"] != "append":
        n, w = case["queries"], case["window"]
        for length in _lengths(case):
            first = max(0, length - n - w + 1) if w else 0  # the oldest token that any query sees
            size += (length - first) * row + 4 * -(-length // case["page"]) + 4 * n * Hq * D
            full = [min(p + 1, w) if w else p + 1 for p in range(length - n, length)]
            flops += 4 * D * Hq * sum(full)
    return {"bytes": size, "flops": flops}


# ---- the definitions in 64 bits -------------------------------------------------------------


def _exact_unpack(raw, case):
    """Page blocks of one sequence (pages, H, bytes), numpy -> keys, values (H, tokens, D) float64."""
    P, D, G = case["page"], case["dim"], case["group"]
    n, m = P * D // 2, P * D // G * 4
    got = []
    for c_at, m_at in ((0, 2 * n), (n, 2 * n + m)):
        c = raw[:, :, c_at:c_at + n].reshape(*raw.shape[:2], P, D // 2)
        codes = np.empty((*c.shape[:3], D), np.float64)
        codes[..., 0::2], codes[..., 1::2] = c & 15, c >> 4
        meta = np.ascontiguousarray(raw[:, :, m_at:m_at + m]).view(np.float16).astype(np.float64)
        meta = meta.reshape(*raw.shape[:2], P, D // G, 2).repeat(G, 3)
        got.append((codes * meta[..., 0] + meta[..., 1]).transpose(1, 0, 2, 3).reshape(raw.shape[1], -1, D))
    return got


def _exact_turn(x, positions, case):
    """Rotation of (T, heads, D) by complex multiplication, with the table's own fp32 angles."""
    R = case["rotary"]
    cos, sin = (t[positions].double().cpu().numpy() for t in case["tables"])
    turn = (cos + 1j * sin)[:, None]
    y = x.copy()
    if case["interleaved"]:
        z = (x[..., 0:R:2] + 1j * x[..., 1:R:2]) * turn
        y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
    else:
        z = (x[..., :R // 2] + 1j * x[..., R // 2:R]) * turn
        y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
    return y


def _exact_round4(x, G):
    """(values, codes, meta) of float64 (..., D)."""
    g = x.reshape(*x.shape[:-1], -1, G)
    scale = np.minimum((g.max(-1) - g.min(-1)) / 15, FP16_MAX).astype(np.float16)
    low = np.clip(g.min(-1), -FP16_MAX, FP16_MAX).astype(np.float16)
    s, b = scale.astype(np.float64)[..., None], low.astype(np.float64)[..., None]
    codes = np.clip(np.rint(np.divide(g - b, s, out=np.zeros_like(g), where=s > 0)), 0, 15)
    return (codes * s + b).reshape(x.shape)


def exact(case, seed):
    if work(case)["flops"] > 2e12:
        return None
    st = prepare(case, seed)
    host = lambda t: t.double().cpu().numpy()  # noqa: E731
    if case["kind"] == "matvec":
        words = st["codes"].cpu().numpy().view(np.uint32).reshape(case["out"], -1, 4, 4)
        w = np.empty((case["out"], words.shape[1], 4, 4, 8))
        for t in range(4):
            for j in range(4):
                for e in range(8):
                    w[:, :, j, t, e] = (words[:, :, t, j] >> np.uint32(4 * NIBBLE_OF[e])) & np.uint32(15)
        meta = host(st["meta"]).repeat(case["group"], 1)
        w = (w.reshape(case["out"], -1) * meta[..., 0] + meta[..., 1])[:, :case["inner"]]
        y = host(st["x"]) @ w.T
        return y if st["bias"] is None else y + host(st["bias"])
    if case["kind"] != "attend":
        turned = dict(case, tables=(st["cos"], st["sin"]))
        q, k = (_exact_turn(host(st[name]), st["positions"].long(), turned) for name in "qk")
        k, v = _exact_round4(k, case["group"]), _exact_round4(host(st["v"]), case["group"])
        if case["kind"] == "append":
            return {"q": q, "k": k, "v": v}
        q = torch.from_numpy(q).to(st["q"].dtype).double().numpy()  # the query is handed on in its type
    else:
        q = host(st["q"])
    n, H, D = case["queries"], case["kv_heads"], case["dim"]
    out = np.zeros(q.shape)
    for b, length in enumerate(_lengths(case)):
        pages = st["page_table"][b, :-(-length // case["page"])].long()
        K, V = (x[:, :length] for x in _exact_unpack(st["pool"][pages].cpu().numpy(), case))
        if case["kind"] == "step":
            K[:, length - n:], V[:, length - n:] = (x[b * n:b * n + n].transpose(1, 0, 2) for x in (k, v))
        rows = slice(b * n, b * n + n)
        position = torch.arange(length - n, length, device="cuda", dtype=torch.float64)[:, None]
        token = torch.arange(length, device="cuda", dtype=torch.float64)
        hidden = (token > position) | ((token <= position - case["window"]) if case["window"] else False)
        for h in range(H):
            Kh, Vh = (torch.from_numpy(np.ascontiguousarray(x[h])).cuda() for x in (K, V))
            heads = case["q_heads"] // H
            for g in range(h * heads, h * heads + heads):
                s = torch.from_numpy(np.ascontiguousarray(q[rows, g])).cuda() @ Kh.T / math.sqrt(D)
                s[hidden] = -math.inf
                out[rows, g] = (torch.softmax(s, -1) @ Vh).cpu().numpy()
    return out
