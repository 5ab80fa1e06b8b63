"""The 4-bit reader operators on the GPU against plain implementations in 64 bits.

Tolerances. Append: codes and factors are defined by fp32 operations in a fixed order, so they are
compared bit for bit with the same formulas in numpy fp32. Attention and matvec: the result is
rounded once to the output type (half a unit in the last place: 2^-8 of the value for bf16's 8
significant bits, 2^-11 for fp16's 11); before that, fp16 rounding of the second product's operand
p scale (2^-11 relative, times |code - 7.5|: at most 2^-11 of sum p |v - middle of its group|),
ex2.approx (2^-22) and fp32 sums over L terms. With the magnitudes below (|score| <= 60 in
fp32: absolute error of a score under 60 * 2^-20, which is its relative effect on p) the bound per
element is 2^-8 or 2^-11 of |out| plus 2^-10 of sum p (|v| + |v - middle|): TOL_OUT and TOL_MASS."""
from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TOL_OUT = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
TOL_MASS = 2.0 ** -10
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
NIB = (0, 4, 2, 6, 1, 5, 3, 7)


@pytest.fixture(scope="module")
def lb():
    from coraanns_b200 import lowbit
    return lowbit


# ---- plain implementations -----------------------------------------------------------------


def quantize32(x, G):
    """The format's formulas in numpy fp32, one rounding per operation."""
    g = x.astype(np.float32).reshape(*x.shape[:-1], -1, G)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        s = ((hi - lo) * np.float32(1 / 15)).astype(np.float32)
        s = np.minimum(s, np.float32(65504)).astype(np.float16)
        b = np.clip(lo, -65504, 65504).astype(np.float16)
        sf, bf = s.astype(np.float32), b.astype(np.float32)
        inv = np.where(sf > 0, np.float32(1) / np.where(sf > 0, sf, 1), np.float32(0)).astype(np.float32)
        c = np.clip(np.rint(((g - bf) * inv).astype(np.float32)), 0, 15)
    return c.reshape(x.shape), s[..., 0], b[..., 0]


def unpack(pool, page, D, G):
    """pool (pages, H, bytes) -> codes and factors of keys and values: (pages, H, page, D) and
    (pages, H, page, D / G) x (scale, low), as numpy."""
    raw = pool.cpu().numpy()
    n, m = page * D // 2, page * (D // G) * 4
    out = []
    for ca, ma in ((0, 2 * n), (n, 2 * n + m)):
        c = raw[:, :, ca:ca + n].reshape(*raw.shape[:2], page, D // 2)
        codes = np.stack((c & 15, c >> 4), -1).reshape(*raw.shape[:2], page, D)
        f = np.ascontiguousarray(raw[:, :, ma:ma + m]).view(np.float16).reshape(*raw.shape[:2], page, D // G, 2)
        out.append((codes, f[..., 0], f[..., 1]))
    return out


def values64(codes, scale, low, G):
    s, b = (np.repeat(x.astype(np.float64), G, -1) for x in (scale, low))
    return codes * s + b


def random_cache(lb, pages, H, D, page, G, seed, noise=True):
    """A cache whose every page holds data (unused tokens too: they must not matter)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cache = lb.Cache4(pages, H, D, page_size=page, group=G)
    k, v = (torch.randn(pages * page, H, D, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    slots = torch.arange(pages * page, device="cuda")
    cache.append(k, v, slots)
    return cache


def attend64(cache, q, table, lens, q_start, causal, window, scale):
    """(out, sum p (|v| + |v - middle|), lse) in 64 bits."""
    (kc, ks, kl), (vc, vs, vl) = unpack(cache.pool, cache.page_size, cache.head_dim, cache.group)
    G = cache.group
    q = q.double().cpu().numpy()
    out, mass, lse = np.zeros(q.shape), np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    per = q.shape[1] // cache.kv_heads
    P = cache.page_size
    for b, L in enumerate(lens):
        pg = table[b][:-(-L // P)]
        if L == 0:
            continue
        K = values64(kc[pg], ks[pg], kl[pg], G).transpose(1, 0, 2, 3).reshape(cache.kv_heads, -1, cache.head_dim)[:, :L]
        V = values64(vc[pg], vs[pg], vl[pg], G).transpose(1, 0, 2, 3).reshape(cache.kv_heads, -1, cache.head_dim)[:, :L]
        M = np.abs(V) + np.abs(V - values64(7.5, vs[pg], vl[pg], G).transpose(1, 0, 2, 3).reshape(cache.kv_heads, -1, cache.head_dim)[:, :L])
        n = q_start[b + 1] - q_start[b]
        for i in range(n):
            pos = L - n + i
            hi = min(L, pos + 1) if causal else L
            lo = max(0, pos - window + 1) if window else 0
            if hi <= lo:
                continue
            for h in range(q.shape[1]):
                s = K[h // per, lo:hi] @ q[q_start[b] + i, h] * scale
                m = s.max()
                p = np.exp(s - m)
                l = p.sum()
                out[q_start[b] + i, h] = p @ V[h // per, lo:hi] / l
                mass[q_start[b] + i, h] = p @ M[h // per, lo:hi] / l
                lse[q_start[b] + i, h] = m + math.log(l)
    return out, mass, lse


def page_tables(lens, page, pages, seed):
    rng = np.random.default_rng(seed)
    order = rng.permutation(pages)
    width = max(1, max(-(-n // page) for n in lens))
    table = np.full((len(lens), width), -1, np.int64)
    at = 0
    for b, n in enumerate(lens):
        need = -(-n // page)
        table[b, :need] = order[at:at + need]
        at += need
    assert at <= pages
    return table, torch.from_numpy(table.astype(np.int32)).cuda()


def check_attend(lb, cache, lens, per, counts, dtype, causal=True, window=0, seed=0, q_scale=1.0, scale=None,
                 strided=False):
    table, dtable = page_tables(lens, cache.page_size, cache.num_pages, seed + 1)
    q_start = np.concatenate(([0], np.cumsum(counts))).astype(np.int64)
    T, Hq, D = int(q_start[-1]), cache.kv_heads * per, cache.head_dim
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if strided:  # a slice of a wider projection
        q = (q_scale * torch.randn(T, Hq + 3, D, generator=gen, device="cuda")).to(DT[dtype])[:, 1:Hq + 1]
    else:
        q = (q_scale * torch.randn(T, Hq, D, generator=gen, device="cuda")).to(DT[dtype])
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = None if all(c == 1 for c in counts) and seed % 2 else torch.from_numpy(q_start.astype(np.int32)).cuda()
    out, lse = cache.attend(q, dtable, dl, q_start=qs, max_queries=max(1, max(counts)), causal=causal, window=window,
                            scale=scale, return_lse=True)
    cache.check()
    want, mass, wlse = attend64(cache, q, table, lens, q_start, causal, window, D ** -0.5 if scale is None else scale)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    err = np.abs(got - want)
    bound = TOL_OUT[dtype] * np.abs(want) + TOL_MASS * mass
    assert (err <= bound).all(), (err / np.maximum(bound, 1e-30)).max()
    gl = lse.double().cpu().numpy()
    empty = np.isneginf(wlse)
    assert np.array_equal(np.isneginf(gl), empty) and (got[empty] == 0).all()
    assert np.abs(gl[~empty] - wlse[~empty]).max(initial=0) <= 2e-4
    return out


# ---- append --------------------------------------------------------------------------------


def rotate32(x, cos, sin, R, interleaved):
    x = x.astype(np.float32)
    y = x.copy()
    c, s = cos[:, None].astype(np.float32), sin[:, None].astype(np.float32)
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y[..., :R // 2], y[..., R // 2:R] = a * c - b * s, b * c + a * s
    return y


@pytest.mark.parametrize("T,Hq,H,D,G,page,R,inter,dtype", [
    (1, 4, 1, 64, 64, 16, 64, False, "bf16"),
    (1, 0, 2, 128, 128, 64, 0, False, "fp16"),
    (5, 6, 2, 128, 64, 16, 128, True, "fp16"),
    (33, 7, 1, 256, 128, 32, 48, False, "bf16"),
    (257, 3, 3, 256, 64, 128, 256, True, "bf16"),
    (1000, 8, 4, 64, 64, 16, 32, True, "bf16"),
    (2500, 12, 8, 128, 128, 64, 96, False, "fp16"),
])
def test_append_matches_the_formulas_bit_for_bit(lb, T, Hq, H, D, G, page, R, inter, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T + D)
    pages = -(-T // page) + 4
    cache = lb.Cache4(pages, H, D, page_size=page, group=G)
    before = torch.randint(0, 256, cache.pool.shape, generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)
    cache.pool.copy_(before)
    x = torch.randn(T, Hq + 2 * H + 1, D, generator=gen, device="cuda").to(DT[dtype])  # strided heads
    q, k, v = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:Hq + 2 * H]
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:T]
    slots[torch.rand(T, generator=gen, device="cuda") < 0.1] = -1
    table = max(1, R // 2)
    angle = torch.rand(500, table, generator=gen, device="cuda") * 6.3
    rope = (angle.cos(), angle.sin()) if R else None
    pos = torch.randint(0, 500, (T,), generator=gen, device="cuda", dtype=torch.int32)
    got = cache.append(k, v, slots, q=q if Hq else None, rope=rope, positions=pos if R else None, interleaved=inter, values=True)
    cache.check()
    kn, vn, qn = (t.float().cpu().numpy() for t in (k, v, q))
    if R:
        c, s = (t[pos.long()].cpu().numpy() for t in rope)
        kn, qn = rotate32(kn, c, s, R, inter), rotate32(qn, c, s, R, inter)
    if Hq:
        assert torch.equal(got.q.cpu(), torch.from_numpy(qn).to(DT[dtype]))
    else:
        assert got.q is None
    fresh = unpack(cache.pool, page, D, G)
    old = unpack(before, page, D, G)
    sl = slots.cpu().numpy()
    keep = sl >= 0
    pg, off = sl[keep] // page, sl[keep] % page
    for x, val, (fc, fs, fl), (oc, os_, ol) in ((kn, got.k, fresh[0], old[0]), (vn, got.v, fresh[1], old[1])):
        codes, scale, low = quantize32(x, G)
        want = (np.repeat(scale.astype(np.float32), G, -1) * codes + np.repeat(low.astype(np.float32), G, -1)).astype(np.float32)
        assert torch.equal(val.cpu(), torch.from_numpy(want).to(DT[dtype]))
        for have, new, was in ((fc, codes, oc), (fs, scale, os_), (fl, low, ol)):
            expect = was.copy()
            expect[pg, :, off] = new[keep]
            assert np.array_equal(np.ascontiguousarray(have).view(np.uint8), np.ascontiguousarray(expect.astype(have.dtype)).view(np.uint8))


def test_append_extreme_groups(lb):
    """Constant groups, ranges that underflow the scale, values past fp16, infinities and NaN."""
    D, G = 64, 64
    rows = torch.zeros(7, 1, D)
    rows[0] = 0.1                      # constant: codes 0, the low alone
    rows[1] = torch.linspace(0, 1e-8, D)  # scale rounds to 0
    rows[2] = torch.linspace(-3e5, 3e5, D)  # low saturates
    rows[3, 0, 5] = float("inf")
    rows[4, 0, 7] = float("nan")
    rows[5] = -0.0
    rows[6] = torch.linspace(-1e4, 1e4, D)
    k = rows.to(torch.bfloat16).cuda()
    cache = lb.Cache4(1, 1, D, page_size=16, group=G)
    got = cache.append(k, k, torch.arange(7, device="cuda"), values=True)
    cache.check()
    kv = got.k.float().cpu().numpy()
    (codes, scale, low), _ = unpack(cache.pool, 16, D, G)
    codes, scale, low = codes[0, 0], scale[0, 0, :, 0], low[0, 0, :, 0]
    x = k.float().cpu().numpy()[:, 0]
    c32, s32, l32 = quantize32(x[[0, 1, 2, 5, 6]], G)
    for i, j in enumerate((0, 1, 2, 5, 6)):
        assert np.array_equal(codes[j], c32[i]) and scale[j] == s32[i, 0] and low[j] == l32[i, 0]
    assert scale[0] == 0 and (codes[0] == 0).all() and abs(kv[0, 0, 0] - 0.1) < 1e-3
    assert low[2] == -65504
    assert scale[3] == 65504 and np.isfinite(kv[3]).all() and codes[3, 5] == 15
    assert np.isnan(low[4]) and np.isnan(kv[4]).all()


def test_append_reports_bad_slots_and_positions(lb):
    cache = lb.Cache4(2, 1, 64, page_size=16)
    k = torch.randn(3, 1, 64, device="cuda").to(torch.bfloat16)
    cache.append(k, k, torch.tensor([0, 32, -5], device="cuda"))
    with pytest.raises(Exception, match="outside"):
        cache.check()
    cache.check()  # cleared
    rope = (torch.ones(4, 32, device="cuda"), torch.zeros(4, 32, device="cuda"))
    cache.append(k, k, torch.tensor([1, 2, 3], device="cuda"), rope=rope,
                 positions=torch.tensor([0, 4, 1], dtype=torch.int32, device="cuda"))
    with pytest.raises(Exception, match="outside"):
        cache.check()


def test_append_unaligned_rows(lb):
    """Rows whose start is not 16-byte aligned go through element loads, with the same result."""
    base = torch.randn(40 * 2 * 130 + 3, device="cuda").to(torch.float16)
    k = base[3:].view(40, 2, 130)[:, :, 1:129]
    assert k.data_ptr() % 16
    a, b = (lb.Cache4(4, 2, 128, page_size=16) for _ in range(2))
    slots = torch.arange(40, device="cuda")
    x, y = a.append(k, k, slots, values=True), b.append(k.contiguous(), k.contiguous(), slots, values=True)
    assert torch.equal(a.pool, b.pool) and torch.equal(x.k, y.k)


# ---- attention -----------------------------------------------------------------------------


@pytest.mark.parametrize("D,G", [(64, 64), (128, 64), (128, 128), (256, 64), (256, 128)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend_one_token(lb, D, G, dtype):
    cache = random_cache(lb, 140, 2, D, 16, G, seed=D + G)
    check_attend(lb, cache, [1, 2, 31, 32, 33, 700, 0, 1000], 4, [1] * 8, dtype, seed=1)


@pytest.mark.parametrize("per", [1, 3, 7, 8, 16])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_attend_shared_heads_and_pages(lb, per, page):
    cache = random_cache(lb, 800 // page + 8, 2, 128, page, 128, seed=per)
    check_attend(lb, cache, [257, 5, 130], per, [1, 1, 1], "bf16", seed=2 * per, strided=True)


@pytest.mark.parametrize("D,G", [(64, 64), (128, 128), (128, 64), (256, 128)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 37), (True, 1), (False, 0)])
def test_attend_several_tokens_ragged(lb, D, G, causal, window):
    """Ragged query counts, one with none, one longer than its cache (its first rows see nothing)."""
    cache = random_cache(lb, 60, 2, D, 16, G, seed=D)
    check_attend(lb, cache, [100, 64, 9, 3, 333, 20], 4, [5, 0, 9, 7, 70, 1], "fp16", causal=causal, window=window, seed=4)


@pytest.mark.parametrize("n,L,per,D,G", [(129, 129, 2, 128, 128), (200, 517, 4, 128, 64), (64, 1000, 8, 64, 64),
                                         (33, 900, 1, 256, 128), (300, 300, 3, 256, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend_chunks(lb, n, L, per, D, G, dtype):
    cache = random_cache(lb, -(-L // 32) + 8, 1, D, 32, G, seed=n)
    check_attend(lb, cache, [L, 40], per, [n, 17], dtype, seed=6)
    check_attend(lb, cache, [L, 40], per, [n, 17], dtype, window=50, seed=7)


def test_attend_long_split_over_blocks(lb):
    """One sequence cut over every block, twice in a row on the same workspace."""
    cache = random_cache(lb, 330, 1, 128, 64, 128, seed=3)
    a = check_attend(lb, cache, [20011], 2, [1], "fp16", seed=10)
    b = check_attend(lb, cache, [20011], 2, [1], "fp16", seed=10)
    assert torch.equal(a, b)


@pytest.mark.parametrize("D,G,H,per,n,lens", [
    (128, 128, 8, 4, [1024], [4096]), (64, 64, 4, 8, [600, 70], [2000, 7000]), (128, 64, 8, 4, [500, 100, 7], [4096, 100, 3000]),
    (256, 128, 4, 3, [300, 17, 200], [3000, 40, 900]), (128, 128, 2, 16, [1], [30000]), (128, 64, 2, 2, [1, 2, 3], [9000, 20, 700])])
def test_attend_repeats_bit_for_bit(lb, D, G, H, per, n, lens):
    """A hand-over that came too early anywhere in the pipelines would show as a changing result."""
    pages = sum(-(-x // 32) for x in lens)
    cache = random_cache(lb, pages, H, D, 32, G, seed=8)
    _, table = page_tables(lens, 32, pages, 9)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = torch.tensor(np.concatenate(([0], np.cumsum(n))), dtype=torch.int32, device="cuda")
    q = torch.randn(sum(n), H * per, D, device="cuda").to(torch.bfloat16)
    want = cache.attend(q, table, dl, q_start=qs, max_queries=max(n))
    for _ in range(60):
        assert torch.equal(cache.attend(q, table, dl, q_start=qs, max_queries=max(n)), want)
    cache.check()


def test_attend_many_sequences(lb):
    """More sequences than one launch takes (their offsets live in shared memory)."""
    rng = np.random.default_rng(0)
    lens = [int(x) for x in rng.integers(0, 40, 1300)]
    cache = random_cache(lb, 4000, 1, 64, 16, 64, seed=5)
    check_attend(lb, cache, lens, 2, [1] * len(lens), "bf16", seed=12)


def test_attend_sharp_and_large_scores(lb):
    cache = random_cache(lb, 30, 2, 128, 16, 128, seed=9)
    check_attend(lb, cache, [300, 77], 4, [1, 1], "fp16", seed=14, q_scale=6.0, scale=0.05)
    check_attend(lb, cache, [300, 77], 4, [1, 1], "fp16", seed=16, q_scale=1e-3, scale=1.0)
    check_attend(lb, cache, [300, 77], 4, [1, 1], "bf16", seed=18, q_scale=1e-20, scale=1e20)
    check_attend(lb, cache, [300, 77], 4, [1, 1], "bf16", seed=20, scale=0.0)


@pytest.mark.parametrize("n", [1, 3, 40])
def test_attend_hidden_tokens_may_be_anything(lb, n):
    """NaN and infinite factors in tokens past the end, outside the window, or after the query."""
    D, page = 128, 16
    cache = random_cache(lb, 12, 1, D, page, 128, seed=2)
    lens, window = [100, 50], 20
    table, dtable = page_tables(lens, page, 12, 3)
    half = cache.pool.view(torch.float16)
    n0 = page * D // 2 * 2 // 2  # factors begin after the codes, in halves
    clean = cache.pool.clone()
    qs = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    q = torch.randn(2 * n, 4, D, device="cuda").to(torch.float16)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = cache.attend(q, dtable, dl, q_start=qs, max_queries=n, window=window)
    seen = set()
    for b, L in enumerate(lens):
        for j in range(max(0, L - n - window + 1), L):
            seen.add((int(table[b, j // page]), j % page))
    for p in range(12):
        for o in range(page):
            if (p, o) not in seen:
                for sec in (0, page * 2):
                    half[p, 0, n0 + sec + 2 * o] = float("nan") if o % 2 else float("inf")
                    half[p, 0, n0 + sec + 2 * o + 1] = float("-inf") if o % 3 else float("nan")
    got = cache.attend(q, dtable, dl, q_start=qs, max_queries=n, window=window)
    cache.check()
    assert torch.equal(got, want) and torch.isfinite(got).all()
    cache.pool.copy_(clean)
    # the last token turns bad: only queries that see it change
    half = cache.pool.view(torch.float16)
    half[int(table[0, 99 // page]), 0, n0 + page * 2 + 2 * (99 % page) + 1] = float("nan")
    got = cache.attend(q, dtable, dl, q_start=qs, max_queries=n, window=window)
    assert torch.equal(got[:n - 1], want[:n - 1]) and torch.equal(got[n:], want[n:])
    assert torch.isnan(got[n - 1]).all()


def test_attend_nan_query_keeps_to_its_row(lb):
    cache = random_cache(lb, 12, 1, 128, 16, 128, seed=2)
    table, dtable = page_tables([90], 16, 12, 3)
    q = torch.randn(1, 4, 128, device="cuda").to(torch.bfloat16)
    dl = torch.tensor([90], dtype=torch.int32, device="cuda")
    want = cache.attend(q, dtable, dl)
    q[0, 1, 3] = float("nan")
    q[0, 2, 9] = float("inf")
    got = cache.attend(q, dtable, dl)
    assert torch.equal(got[0, [0, 3]], want[0, [0, 3]]) and not torch.isfinite(got[0, 1:3]).any()


def test_attend_reports_bad_tables_and_lengths(lb):
    cache = random_cache(lb, 4, 1, 64, 16, 64, seed=2)
    q = torch.randn(1, 1, 64, device="cuda").to(torch.bfloat16)
    for table, n in (([[0, 9]], 20), ([[0, -1]], 20), ([[0, 1]], 33), ([[0, 1]], -1)):
        cache.attend(q, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda"))
        with pytest.raises(Exception, match="outside"):
            cache.check()
    cache.check()


def test_attend_on_another_stream(lb):
    cache = random_cache(lb, 60, 2, 128, 16, 128, seed=2)
    table, dtable = page_tables([800], 16, 60, 3)
    q = torch.randn(1, 8, 128, device="cuda").to(torch.bfloat16)
    dl = torch.tensor([800], dtype=torch.int32, device="cuda")
    want = cache.attend(q, dtable, dl)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(cache.attend(q, dtable, dl))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_attend_offsets_past_32_bits(lb):
    """A pool over 4 GB, pages at its end."""
    page, D, H = 256, 128, 8
    block = page * D + 8 * page
    pages = (1 << 32) // (block * H) + 40
    cache = lb.Cache4(pages, H, D, page_size=page, group=128)
    assert cache.pool.numel() > 1 << 32
    small = random_cache(lb, 4, H, D, page, 128, seed=1)
    cache.pool[pages - 4:].copy_(small.pool)
    q = torch.randn(1, 2 * H, D, device="cuda").to(torch.bfloat16)
    dl = torch.tensor([1000], dtype=torch.int32, device="cuda")
    t = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    assert torch.equal(cache.attend(q, t + (pages - 4), dl), small.attend(q, t, dl))
    k = torch.randn(3, H, D, device="cuda").to(torch.bfloat16)
    cache.append(k, k, torch.arange(3, device="cuda") + pages * page - 3)
    small.append(k, k, torch.arange(3, device="cuda") + 4 * page - 3)
    cache.check()
    assert torch.equal(cache.pool[pages - 4:], small.pool)


# ---- matvec --------------------------------------------------------------------------------


def weight64(w):
    words = w.codes.cpu().numpy().view(np.uint32).reshape(w.rows, -1, 4, 4)
    codes = np.empty((w.rows, words.shape[1], 4, 4, 8))
    for t in range(4):
        for j in range(4):
            for e in range(8):
                codes[:, :, j, t, e] = words[:, :, t, j] >> np.uint32(4 * NIB[e]) & np.uint32(15)
    meta = np.repeat(w.meta.cpu().numpy().astype(np.float64), w.group, 1)
    return (codes.reshape(w.rows, -1) * meta[..., 0] + meta[..., 1])[:, :w.cols]


@pytest.mark.parametrize("M", [1, 2, 8, 9, 17, 33, 64, 70])
@pytest.mark.parametrize("N,K,G", [(1, 1, 32), (16, 128, 128), (100, 384, 32), (257, 1000, 64), (1024, 2052, 128), (333, 4104, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_matvec(lb, M, N, K, G, dtype):
    """Error: the fp32 sums hold the products of 128 + c (bf16) or c (fp16), at most 2^-20 of
    sum |x| (|128 scale| + |low|) before the one rounding of the result."""
    gen = torch.Generator(device="cuda").manual_seed(M * N + K)
    w = lb.Weight4.quantize(torch.randn(N, K, generator=gen, device="cuda") + 0.3, group=G)
    x = torch.randn(M, K, generator=gen, device="cuda").to(DT[dtype])
    bias = torch.randn(N, generator=gen, device="cuda").to(DT[dtype]) if M % 2 else None
    y = lb.matvec(x, w, bias=bias).double().cpu().numpy()
    w64, x64 = weight64(w), x.double().cpu().numpy()
    want = x64 @ w64.T + (0 if bias is None else bias.double().cpu().numpy())
    meta = np.repeat(w.meta.cpu().numpy().astype(np.float64), w.group, 1)[:, :K]
    mass = np.abs(x64) @ (128 * meta[..., 0] + np.abs(meta[..., 1])).T
    bound = TOL_OUT[dtype] * np.abs(want) + 2.0 ** -20 * mass + 1e-7
    assert (np.abs(y - want) <= bound).all(), (np.abs(y - want) / bound).max()


def test_matvec_quantize_matches_the_format(lb):
    x = torch.randn(50, 300, device="cuda")
    w = lb.Weight4.quantize(x, group=32)
    padded = np.pad(x.cpu().numpy(), ((0, 0), (0, 84)))
    codes, scale, low = quantize32(padded, 32)
    want = values64(codes, scale, low, 32)[:, :300]
    assert np.array_equal(weight64(w), want)


def test_matvec_strides_and_views(lb):
    w = lb.Weight4.quantize(torch.randn(64, 200, device="cuda"))
    big = torch.randn(6, 411, device="cuda").to(torch.bfloat16)
    x = big[:, 5:205]  # rows neither aligned nor contiguous
    y = lb.matvec(x, w)
    assert torch.equal(y, lb.matvec(x.contiguous(), w))
    assert torch.equal(lb.matvec(x[3], w), y[3])
    assert torch.equal(lb.matvec(x.contiguous().view(2, 3, 200), w), y.view(2, 3, 64))
    out = torch.empty_like(y)
    assert lb.matvec(x, w, out=out) is out and torch.equal(out, y)
    assert lb.matvec(x[:0], w).shape == (0, 64)


def test_matvec_rows_do_not_touch(lb):
    """NaN and infinity in one activation row leave the others as they are."""
    w = lb.Weight4.quantize(torch.randn(70, 256, device="cuda"))
    x = torch.randn(5, 256, device="cuda").to(torch.float16)
    want = lb.matvec(x, w)
    x[2, 7], x[4, 9] = float("nan"), float("inf")
    got = lb.matvec(x, w)
    assert torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])
    assert torch.isnan(got[2]).all() and not torch.isfinite(got[4]).any()


# ---- refusals ------------------------------------------------------------------------------


def test_refusals(lb):
    from coraanns_b200 import InvalidArgument
    for kw in (dict(head_dim=96), dict(head_dim=128, page_size=24), dict(head_dim=128, page_size=8),
               dict(head_dim=128, group=32), dict(head_dim=64, group=128)):
        with pytest.raises(InvalidArgument):
            lb.Cache4(2, 1, **kw)
    cache = lb.Cache4(2, 2, 128)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda")
    s = torch.arange(3, device="cuda")
    ones = torch.ones(8, 64, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    bad = [lambda: cache.append(k.float(), k.float(), s), lambda: cache.append(k, k.half(), s),
           lambda: cache.append(k[:, :1], k, s), lambda: cache.append(k, k, s.int()), lambda: cache.append(k, k, s[:2]),
           lambda: cache.append(k, k, s, rope=(ones, ones)), lambda: cache.append(k.cpu(), k, s),
           lambda: cache.append(k, k, s, rope=(ones[:, :7].contiguous(), ones[:, :7].contiguous()), positions=pos),
           lambda: cache.append(k, k, s, q=k[:2]), lambda: cache.append(k.transpose(1, 2), k, s)]
    t = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    n = torch.ones(3, dtype=torch.int32, device="cuda")
    bad += [lambda: cache.attend(k[:, :1], t, n), lambda: cache.attend(k[:2], t, n), lambda: cache.attend(k, t.long(), n),
            lambda: cache.attend(k, t, n.long()), lambda: cache.attend(k.float(), t, n),
            lambda: cache.attend(k, t, n, causal=False, window=3), lambda: cache.attend(k, t, n, out=k[:2]),
            lambda: cache.attend(k, t, n, q_start=n)]
    w = lb.Weight4.quantize(torch.zeros(4, 128, device="cuda"))
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda")
    bad += [lambda: lb.matvec(x[:, :64], w), lambda: lb.matvec(x.float(), w), lambda: lb.matvec(x, w, bias=x[0, :3]),
            lambda: lb.matvec(x, w, out=x), lambda: lb.Weight4(w.codes, w.meta, 129), lambda: lb.Weight4(w.codes, w.meta[:2], 128)]
    for f in bad:
        with pytest.raises(InvalidArgument):
            f()
    cache.check()


# ---- together ------------------------------------------------------------------------------


def test_reader_example_searches_and_reads():
    """The example's decoder agrees with plain torch on the same 4-bit values: activations are
    rounded to bf16 (2^-8) some 8 times per layer on the way to the logits, so 10 % is far above
    what two layers leave, and far below what a wrong operator gives."""
    import importlib.util
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("reader", ROOT / "cgcl-coraanns_b200" / "apps" / "reader.py")
    reader = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(reader)
    ids, off = reader.main(["--passages", "600", "--tokens", "5"])
    assert ids[0] == 17 and off < 0.1
