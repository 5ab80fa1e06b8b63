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
