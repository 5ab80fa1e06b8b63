"""Edges of the 4-bit reader operators on the GPU: values past the fp16 range, long flat tails,
rows and tokens that must not touch one another, row ranges with gaps, the kernels' rarer paths.

Plain implementations and the tolerances of attention and matvec are those of test_gpu_lowbit
(2^-8 or 2^-11 of the result, 2^-10 of sum p (|v| + |v - middle|)). Where a test needs another one
it is derived there."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_lowbit import DT, TOL_MASS, TOL_OUT, attend64, check_attend, lb, page_tables, random_cache  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def slots_of(cache, lens, seed, at):
    """Slots of tokens `at` of sequence 0, under the page table that check_attend draws for `seed`."""
    table, _ = page_tables(lens, cache.page_size, cache.num_pages, seed + 1)
    at = np.asarray(at)
    return torch.from_numpy(table[0][at // cache.page_size] * cache.page_size + at % cache.page_size).cuda()


# ---- values past the fp16 range --------------------------------------------------------------


@pytest.mark.parametrize("D,G,per,n", [(64, 64, 4, 40), (128, 128, 4, 40), (128, 64, 2, 20), (256, 128, 4, 40), (256, 64, 1, 33),
                                       (128, 128, 4, 3)])
@pytest.mark.parametrize("window", [0, 60])
def test_attend_values_past_fp16(lb, D, G, per, n, window):
    """Groups of finite factors whose values pass 65504: queries that see such a token get its
    finite value, queries before it (or past the window) are as if it were not there."""
    lens, seed = [300], 30
    cache = random_cache(lb, 24, 1, D, 16, G, seed=D)
    k = torch.randn(3, 1, D, device="cuda").to(torch.bfloat16)
    v = torch.stack([torch.linspace(-20000, 70000, D), torch.linspace(3e5, -3e5, D), torch.full((D,), 1.0)])
    v[2, ::5] = -60000.0
    v[2, 1::5] = 69000.0
    cache.append(k, v[:, None].to(torch.bfloat16).cuda(), slots_of(cache, lens, seed, [200, 299 - n // 2, 299]))
    check_attend(lb, cache, lens, per, [n], "bf16", window=window, seed=seed)


def test_attend_values_past_fp16_cut_over_blocks(lb):
    """The same in one job whose stretches lie in different blocks, some with such a token, and in
    fp16 (a group over +-65504 has a rounded scale that gives 65536)."""
    lens, seed = [30000], 32
    cache = random_cache(lb, 1900, 1, 128, 16, 128, seed=3)
    k = torch.zeros(2, 1, 128, dtype=torch.float16, device="cuda")
    v = torch.linspace(-65504, 65504, 128, device="cuda").to(torch.float16)[None, None].expand(2, 1, 128)
    cache.append(k, v, slots_of(cache, lens, seed, [11000, 29999]))
    check_attend(lb, cache, lens, 4, [10], "fp16", seed=seed)


# ---- long flat tails --------------------------------------------------------------------------


@pytest.mark.parametrize("per,n,L,H", [(4, 1, 16384, 1184), (4, 20, 16384, 148), (4, 40, 32768, 148), (2, 17, 65536, 148)])
def test_attend_flat_tail_behind_a_sink(lb, per, n, L, H):
    """One early token 17.7 nats above all others, its value 0: what remains of the output is the
    sum of L tiny probabilities. As many key heads as give each block (streaming: warp) a whole
    sequence, so that all its tokens are weighed against that one.

    A probability is an fp16 operand times 2^7 relative to the maximum: below the normal range it
    is off by half of 2^-24, that is 2^-32 of the maximum's, per token and unit of value (the
    streaming kernel's operand p scale likewise, times half the range of a group). So L 2^-32
    max |v| is added to the bound."""
    D, page = 128, 64
    one = lb.Cache4(L // page, 1, D, page_size=page)
    gen = torch.Generator(device="cuda").manual_seed(L)
    direction = torch.randn(D, generator=gen, device="cuda")
    k = torch.zeros(L, 1, D, device="cuda")
    v = 1.0 + 0.25 * torch.randn(L, 1, D, generator=gen, device="cuda")
    k[5, 0] = direction * (17.7 / (direction.square().sum() * D ** -0.5))
    v[5] = 0.0
    one.append(k.to(torch.bfloat16), v.to(torch.bfloat16), torch.arange(L, device="cuda"))
    cache = lb.Cache4.from_pool(one.pool.expand(-1, H, -1).contiguous(), page, D)
    q = direction.expand(n, per * H, D).to(torch.bfloat16)
    table = torch.arange(L // page, dtype=torch.int32, device="cuda")[None]
    dl = torch.tensor([L], dtype=torch.int32, device="cuda")
    qs = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got, lse = cache.attend(q, table, dl, q_start=qs, max_queries=n, return_lse=True)
    cache.check()
    want, mass, wlse = attend64(one, q[:, :per], table.cpu().numpy(), [L], [0, n], True, 0, D ** -0.5)
    bound = TOL_OUT["bf16"] * np.abs(want) + TOL_MASS * mass + L * 2.0 ** -32 * float(v.abs().max())
    got, lse = (x.double().cpu().numpy() for x in (got.view(n, H, per, D), lse.view(n, H, per)))
    for h in range(H):
        assert (np.abs(got[:, h] - want) <= bound).all(), (h, (np.abs(got[:, h] - want) / bound).max())
        assert np.abs(lse[:, h] - wlse).max() <= 2e-4


# ---- rows and tokens that must not touch one another ------------------------------------------


@pytest.mark.parametrize("D,G", [(64, 64), (128, 64), (128, 128), (256, 128)])
@pytest.mark.parametrize("n", [1, 3, 12])
def test_attend_huge_query_keeps_to_its_row(lb, D, G, n):
    """A finite but huge query changes nothing in the rows that share its instructions."""
    cache = random_cache(lb, 12, 1, D, 16, G, seed=2)
    table, dtable = page_tables([90], 16, 12, 3)
    q = torch.randn(n, 4, D, device="cuda").to(torch.bfloat16)
    dl = torch.tensor([90], dtype=torch.int32, device="cuda")
    qs = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    want = cache.attend(q, dtable, dl, q_start=qs, max_queries=n)
    big = q.clone()
    big[0, 1] *= 2.0 ** 60
    big[n - 1, 3, 5] = 1e30
    got = cache.attend(big, dtable, dl, q_start=qs, max_queries=n)
    touched = torch.zeros(n, 4, dtype=torch.bool, device="cuda")
    touched[0, 1] = touched[n - 1, 3] = True
    assert torch.equal(got[~touched], want[~touched])


@pytest.mark.parametrize("per,n", [(4, 1), (8, 3), (2, 4)])
def test_attend_hidden_tokens_of_wide_range(lb, per, n):
    """Value factors of the largest finite size in tokens that no query sees (outside the window,
    past the end) or only the last query does: the others keep their accuracy, for values that are
    small beside them."""
    D, page, L, window, seed = 128, 16, 90, 20, 40
    lens = [L]
    cache = lb.Cache4(8, 1, D, page_size=page)
    k, v = (torch.randn(8 * page, 1, D, device="cuda") for _ in range(2))
    cache.append(k.to(torch.bfloat16), (1e-3 * v).to(torch.bfloat16), torch.arange(8 * page, device="cuda"))
    hidden = list(range(L - n - window + 1)) + list(range(L, 96)) + ([L - 1] if n > 1 and per == 8 else [])
    wide = torch.linspace(-6e4, 6e4, D, device="cuda").to(torch.bfloat16)[None, None].expand(len(hidden), 1, D)
    cache.append(wide, wide, slots_of(cache, [96], seed, hidden))
    table, dtable = page_tables([96], page, 8, seed + 1)
    q = torch.randn(n, per, D, device="cuda").to(torch.bfloat16)
    got = cache.attend(q, dtable, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                       q_start=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_queries=n, window=window)
    cache.check()
    want, mass, _ = attend64(cache, q, table, lens, [0, n], True, window, D ** -0.5)
    err = np.abs(got.double().cpu().numpy() - want)
    bound = TOL_OUT["bf16"] * np.abs(want) + TOL_MASS * mass
    assert (err <= bound).all(), (err / bound).max()


def test_attend_window_of_any_size(lb):
    """A window as large as an int holds, with more queries than cached tokens."""
    for D, G, per in ((128, 128, 2), (64, 64, 4), (256, 128, 1)):
        cache = random_cache(lb, 20, 1, D, 16, G, seed=6)
        check_attend(lb, cache, [100, 70], per, [200, 80], "bf16", window=2 ** 31 - 1, seed=50)


# ---- rows that no sequence asks for -------------------------------------------------------------


@pytest.mark.parametrize("D,G,n", [(64, 64, 2), (128, 128, 2), (256, 64, 2), (64, 64, 50), (128, 64, 50), (256, 128, 50)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend_rows_outside_every_range(lb, D, G, n, dtype):
    """Padding rows before the first range and after the last give zeros and a log-sum of -inf."""
    cache = random_cache(lb, 30, 2, D, 16, G, seed=7)
    _, table = page_tables([100, 33], 16, 30, 8)
    lens = torch.tensor([100, 33], dtype=torch.int32, device="cuda")
    q = torch.randn(3 + 2 * n + 5, 8, D, device="cuda").to(DT[dtype])
    qs = torch.tensor([3, 3 + n, 3 + 2 * n], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    got, lse = cache.attend(q, table, lens, q_start=qs, max_queries=n, out=out, return_lse=True)
    cache.check()
    inside = slice(3, 3 + 2 * n)
    want, wlse = cache.attend(q[inside], table, lens, q_start=qs - 3, max_queries=n, return_lse=True)
    assert torch.equal(got[inside], want) and torch.equal(lse[inside], wlse)
    rest = torch.ones(len(q), dtype=torch.bool, device="cuda")
    rest[inside] = False
    assert (got[rest] == 0).all() and torch.isneginf(lse[rest]).all()


def test_attend_rows_outside_every_range_of_many_sequences(lb):
    """More sequences than one launch takes: the gaps are those of the whole call."""
    lens = [5] * 700
    cache = random_cache(lb, 700, 1, 64, 16, 64, seed=5)
    _, table = page_tables(lens, 16, 700, 3)
    q = torch.randn(712, 2, 64, device="cuda").to(torch.bfloat16)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = torch.arange(701, dtype=torch.int32, device="cuda") + 4
    for most in (1, 40):  # both kernels
        got = cache.attend(q, table, dl, q_start=qs, max_queries=most, out=torch.full_like(q, 7.0))
        cache.check()
        want = cache.attend(q[4:704], table, dl, q_start=qs - 4, max_queries=most)
        assert torch.equal(got[4:704], want)
        assert (got[:4] == 0).all() and (got[704:] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend_without_sequences(lb, dtype):
    cache = random_cache(lb, 2, 1, 64, 16, 64, seed=5)
    q = torch.randn(3, 2, 64, device="cuda").to(DT[dtype])
    got, lse = cache.attend(q, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"),
                            q_start=torch.zeros(1, dtype=torch.int32, device="cuda"), out=torch.full_like(q, 7.0), return_lse=True)
    assert (got == 0).all() and torch.isneginf(lse).all()


# ---- the kernels' rarer paths -------------------------------------------------------------------


@pytest.mark.parametrize("D,G", [(64, 64), (128, 128), (128, 64), (256, 128), (256, 64)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 37), (True, 1), (False, 0)])
@pytest.mark.parametrize("per,counts", [(4, [5, 0, 8, 7, 3, 1]), (1, [32, 9, 10, 2, 31, 1]), (7, [4, 1, 2, 3, 0, 4])])
def test_attend_several_tokens_streamed(lb, D, G, causal, window, per, counts):
    """2 to 32 rows per key head: several query tokens through the streaming kernel, one sequence
    with more of them than it has cached tokens."""
    cache = random_cache(lb, 60, 2, D, 16, G, seed=D)
    check_attend(lb, cache, [100, 64, 9, 3, 333, 20], per, counts, "fp16" if per == 4 else "bf16", causal=causal, window=window,
                 seed=4)


@pytest.mark.parametrize("D,G", [(64, 64), (128, 128), (128, 64), (256, 128), (256, 64)])
@pytest.mark.parametrize("n,scale", [(4, 0.1), (40, 0.1), (4, -0.1), (40, -0.1), (40, 0.0), (150, 0.1)])
def test_attend_maxima_that_keep_growing(lb, D, G, n, scale):
    """Keys that grow from token to token (and scales of either sign): the running maximum is
    raised, and the sums rescaled, many times along a sequence. |score| stays under 60."""
    seed, L = 60, 500
    cache = random_cache(lb, 40, 1, D, 16, G, seed=D)
    gen = torch.Generator(device="cuda").manual_seed(D)
    k = torch.randn(L, 1, D, generator=gen, device="cuda") * torch.linspace(0.05, 10.0 * (64 / D) ** 0.5, L, device="cuda")[:, None, None]
    v = torch.randn(L, 1, D, generator=gen, device="cuda")
    cache.append(k.to(torch.bfloat16), v.to(torch.bfloat16), slots_of(cache, [L], seed, np.arange(L)))
    check_attend(lb, cache, [L], 3, [n], "fp16", scale=scale, seed=seed, q_scale=1.2)


@pytest.mark.parametrize("D,G", [(64, 64), (128, 64), (256, 128)])
def test_attend_value_scales_that_grow(lb, D, G):
    """Values whose size doubles every 20 tokens: the streaming kernel's bound on the value scales is
    raised, and its sums shrunk, along the sequence."""
    seed, L = 70, 320
    cache = random_cache(lb, 24, 1, D, 16, G, seed=D)
    gen = torch.Generator(device="cuda").manual_seed(D)
    v = torch.randn(L, 1, D, generator=gen, device="cuda") * 2.0 ** (torch.arange(L, device="cuda") / 20 - 8)[:, None, None]
    k = torch.randn(L, 1, D, generator=gen, device="cuda")
    cache.append(k.to(torch.bfloat16), v.to(torch.bfloat16), slots_of(cache, [L], seed, np.arange(L)))
    check_attend(lb, cache, [L], 4, [1], "bf16", seed=seed)
    check_attend(lb, cache, [L], 4, [7], "fp16", seed=seed)


# ---- captured graphs ------------------------------------------------------------------------------


def graph_inputs(lb, lens, n, per=4, H=2, D=128, seed=1):
    cache = random_cache(lb, 700, H, D, 16, 128, seed=seed)
    _, table = page_tables(lens, 16, 700, seed)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = torch.arange(len(lens) + 1, dtype=torch.int32, device="cuda") * n
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(len(lens) * n, H * per, D, generator=gen, device="cuda").to(torch.bfloat16)
    return cache, lambda out=None: cache.attend(q, table, dl, q_start=qs, max_queries=n, out=out)


@pytest.mark.parametrize("warm", [True, False])
def test_captured_steps_survive_larger_calls(lb, warm):
    """Decoding steps of two caches captured on a stream, then larger eager calls there and memory
    that others take: the replays give the eager results."""
    a, step_a = graph_inputs(lb, [3000, 40, 5000], 1, seed=1)
    b, step_b = graph_inputs(lb, [2000, 700], 1, seed=2)
    _, chunk = graph_inputs(lb, [1500], 64, seed=3)
    want, more = [step_a(), step_b()], chunk()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    if warm:
        with torch.cuda.stream(s):
            step_a(), step_b()
        s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = [step_a(), step_b()]
    with torch.cuda.stream(s):
        first = chunk()
        junk = [torch.full((size,), 0xff, dtype=torch.uint8, device="cuda") for size in (1 << 20, 6 << 20, 7 << 20, 20 << 20)]
        for _ in range(3):
            graph.replay()
            second = chunk()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert torch.equal(first, more) and torch.equal(second, more)
    assert all((j == 0xff).all() for j in junk)
    a.check(), b.check()


def test_graphs_of_one_stream_replayed_in_any_order(lb):
    """Two graphs captured on a stream that never ran a call eagerly, of both kernels; the second is
    replayed first, then both at once on two streams."""
    a, step = graph_inputs(lb, [9000], 1, seed=4)
    b, chunk = graph_inputs(lb, [2500], 100, seed=5)
    want, more = step(), chunk()
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, outs = [], []
    for f in (step, chunk, step):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(f())
        graphs.append(g)
    for g in reversed(graphs):
        g.replay()
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[0].replay()
            graphs[1].replay()
        with torch.cuda.stream(t):
            graphs[2].replay()
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], more) and torch.equal(outs[2], want)
        assert torch.equal(eager, want)
    a.check(), b.check()


# ---- errors found on the device -------------------------------------------------------------------


def test_check_loses_no_error(lb):
    """Calls on one stream set the status word while check() reads and clears it on another: each
    error is reported."""
    import threading
    cache = lb.Cache4(2, 1, 64, page_size=16)
    k = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    bad = torch.tensor([32], device="cuda")
    torch.cuda.synchronize()
    raised, lost = threading.Event(), []

    def caller():
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(400):
                raised.clear()
                cache.append(k, k, bad)
                torch.cuda.current_stream().synchronize()
                if not raised.wait(2):
                    lost.append(i)
                    return

    thread = threading.Thread(target=caller)
    thread.start()
    while thread.is_alive():
        try:
            cache.check()
        except Exception:
            raised.set()
    thread.join()
    assert not lost


# ---- products: the variant for matrices of many rows ------------------------------------------------


def wide_rows():
    return 2 * 32 * torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("M", [1, 5, 8])
@pytest.mark.parametrize("over,K,G", [(-1, 200, 64), (0, 128, 128), (1, 7, 32), (31, 260, 64), (535, 384, 32), (535, 1003, 128)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_matvec_of_many_rows(lb, M, over, K, G, dtype):
    """Row counts on both sides of where a warp takes two row tiles, with ragged last blocks, and few
    columns (warps without a segment). Bound as in test_matvec."""
    from test_gpu_lowbit import weight64
    N = wide_rows() + over
    gen = torch.Generator(device="cuda").manual_seed(M + N + K)
    w = lb.Weight4.quantize(torch.randn(N, K, generator=gen, device="cuda") + 0.3, group=G)
    x = torch.randn(M, K, generator=gen, device="cuda").to(DT[dtype])
    bias = torch.randn(N, generator=gen, device="cuda").to(DT[dtype]) if M != 5 else None
    y = lb.matvec(x, w, bias=bias).double().cpu().numpy()
    x64 = x.double().cpu().numpy()
    want = x64 @ weight64(w).T + (0 if bias is None else bias.double().cpu().numpy())
    meta = np.repeat(w.meta.cpu().numpy().astype(np.float64), w.group, 1)[:, :K]
    mass = np.abs(x64) @ (128 * meta[..., 0] + np.abs(meta[..., 1])).T
    bound = TOL_OUT[dtype] * np.abs(want) + 2.0 ** -20 * mass + 1e-7
    assert (np.abs(y - want) <= bound).all(), (np.abs(y - want) / bound).max()


# ---- outputs over inputs ------------------------------------------------------------------------


def test_matvec_refuses_an_output_over_its_input(lb):
    from coraanns_b200 import InvalidArgument
    w = lb.Weight4.quantize(torch.randn(256, 256, device="cuda"))
    buf = torch.randn(9, 256, device="cuda").to(torch.bfloat16)
    for x, out in ((buf, buf), (buf[:4], buf[3:7]), (buf[3:7], buf[:4]), (buf[4], buf[4]), (buf[::2], buf[4:])):
        with pytest.raises(InvalidArgument):
            lb.matvec(x, w, out=out)
    x = buf[:4].clone()
    assert torch.equal(lb.matvec(buf[:4], w, out=buf[4:8]), lb.matvec(x, w)) and torch.equal(buf[:4], x)
    assert torch.equal(lb.matvec(buf[4:8].clone(), w, out=buf[:4]), lb.matvec(buf[4:8], w))


@pytest.mark.parametrize("n,lens,H,per", [(1, [30000], 2, 4), (5, [700, 300], 2, 4), (200, [3000, 900], 2, 4), (64, [500] * 20, 4, 1)])
def test_attend_in_place(lb, n, lens, H, per):
    """Over its own queries, jobs whole and cut over blocks."""
    pages = sum(-(-x // 32) for x in lens)
    cache = random_cache(lb, pages, H, 128, 32, 128, seed=8)
    _, table = page_tables(lens, 32, pages, 9)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = torch.arange(len(lens) + 1, dtype=torch.int32, device="cuda") * n
    q = torch.randn(n * len(lens), H * per, 128, device="cuda").to(torch.bfloat16)
    want = cache.attend(q, table, dl, q_start=qs, max_queries=n)
    for _ in range(20):
        x = q.clone()
        assert cache.attend(x, table, dl, q_start=qs, max_queries=n, out=x) is x and torch.equal(x, want)


# ---- sizes of one and none ------------------------------------------------------------------------


def test_strides_of_sizes_of_one_do_not_matter(lb):
    cache = random_cache(lb, 4, 1, 64, 16, 64, seed=2)
    q = torch.randn(3, 2, 64, device="cuda").to(torch.bfloat16)
    lens = torch.tensor([3, 16, 9], dtype=torch.int32, device="cuda")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda").t()  # (3, 1), strides (1, 3)
    assert table.stride(1) != 1
    assert torch.equal(cache.attend(q, table, lens), cache.attend(q, table.contiguous().view(3, 1), lens))
    w = lb.Weight4.quantize(torch.randn(70, 1, device="cuda"))
    x = torch.randn(1, 5, device="cuda").to(torch.float16).t()  # (5, 1), strides (1, 5)
    assert x.stride(1) != 1
    assert torch.equal(lb.matvec(x, w), lb.matvec(x.clone(memory_format=torch.contiguous_format).reshape(5).view(5, 1), w))


def test_weights_without_rows_or_columns(lb):
    from coraanns_b200 import InvalidArgument
    w = lb.Weight4.quantize(torch.zeros(0, 200, device="cuda"))
    assert w.rows == 0 and lb.matvec(torch.zeros(3, 200, device="cuda", dtype=torch.float16), w).shape == (3, 0)
    with pytest.raises(InvalidArgument):
        lb.Weight4.quantize(torch.zeros(5, 0, device="cuda"))
    with pytest.raises(InvalidArgument):
        lb.Weight4.quantize(torch.zeros(5, 4, device="cuda"), group=48)
