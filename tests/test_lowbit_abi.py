"""CPU tests of the 4-bit reader operators' C boundary: sizes, and refusals that come before any
device work (there may be no GPU here)."""
from __future__ import annotations

import ctypes as C
import struct

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from coraanns_b200 import lowbit
    return lowbit._library()


def message(lib):
    return lib.cora_last_error().decode()


def cache_arg(**kw):
    from coraanns_b200 import lowbit
    f = dict(pool=1 << 20, num_pages=4, kv_heads=2, head_dim=128, page_size=64, group=128, status=1 << 12)
    f.update(kw)
    return lowbit._CacheArg(**f)


def test_block_bytes_counts_codes_and_factors(lib):
    assert lib.cora_kv4_block_bytes(64, 128, 128) == 64 * (128 + 8)
    assert lib.cora_kv4_block_bytes(16, 256, 64) == 16 * (256 + 32)
    assert lib.cora_kv4_block_bytes(16, 128, 0) == 0 and lib.cora_kv4_block_bytes(16, 100, 64) == 0


def test_packed_arguments_have_the_structs_sizes():
    """The Python packers write the C structs byte for byte (x86-64 layout of include/cora_b200.h)."""
    from coraanns_b200 import lowbit

    class Append(C.Structure):
        _fields_ = ([(f"p{i}", C.c_void_p) for i in range(6)] + [(f"s{i}", C.c_int64) for i in range(6)]
                    + [(f"q{i}", C.c_void_p) for i in range(4)] + [("t", C.c_uint64), ("r", C.c_uint64)]
                    + [(f"u{i}", C.c_uint32) for i in range(4)])

    class Attend(C.Structure):
        _fields_ = ([(f"p{i}", C.c_void_p) for i in range(3)] + [("a", C.c_int64), ("b", C.c_int64)]
                    + [(f"q{i}", C.c_void_p) for i in range(3)] + [("c", C.c_int64), ("d", C.c_uint64), ("e", C.c_uint64),
                                                                    ("w", C.c_void_p), ("f", C.c_float)]
                    + [(f"u{i}", C.c_uint32) for i in range(7)])

    class Matvec(C.Structure):
        _fields_ = [("x", C.c_void_p), ("b", C.c_void_p), ("y", C.c_void_p), ("s", C.c_int64), ("t", C.c_int64),
                    ("r", C.c_uint64), ("d", C.c_uint32)]

    assert len(lowbit._APPEND(*[0] * 22)) == C.sizeof(Append) == struct.calcsize("6Q6q4Q2Q4I")
    assert len(lowbit._ATTEND(*[0] * 12, 0.5, *[0] * 7)) == C.sizeof(Attend)
    assert len(lowbit._MATVEC(*[0] * 7)) == C.sizeof(Matvec)


@pytest.mark.parametrize("kw,word", [
    (dict(head_dim=96), "head_dim"), (dict(group=32), "group"), (dict(head_dim=64, group=128), "group"),
    (dict(page_size=48), "page_size"), (dict(page_size=8), "page_size"), (dict(page_size=2048), "page_size"),
    (dict(kv_heads=0), "kv_heads"), (dict(pool=None), "pool"), (dict(pool=(1 << 20) + 4), "pool"),
    (dict(status=None), "status"), (dict(num_pages=1 << 33), "num_pages")])
def test_bad_caches_are_refused(lib, kw, word):
    from coraanns_b200 import CORA_EINVAL, lowbit
    c = cache_arg(**kw)
    for f, args in ((lib.cora_kv4_append, lowbit._APPEND(*[0] * 22)), (lib.cora_kv4_attend, lowbit._ATTEND(*[0] * 12, 0.5, *[0] * 7))):
        assert f(C.addressof(c), args, None) == CORA_EINVAL and word in message(lib)


def test_null_structs_are_refused(lib):
    from coraanns_b200 import CORA_EINVAL
    c = cache_arg()
    assert lib.cora_kv4_append(None, None, None) == CORA_EINVAL
    assert lib.cora_kv4_append(C.addressof(c), None, None) == CORA_EINVAL
    assert lib.cora_kv4_attend(C.addressof(c), None, None) == CORA_EINVAL
    assert lib.cora_w4_matvec(None, None, None) == CORA_EINVAL
    assert lib.cora_kv4_status(None, None) == CORA_EINVAL
    assert lib.cora_kv4_attend_workspace(None, 8, 1) == 0


def append_args(**kw):
    from coraanns_b200 import lowbit
    f = dict(k=1 << 16, v=1 << 16, q=0, k_out=0, v_out=0, q_out=0, kt=256, kh=128, vt=256, vh=128, qt=0, qh=0, slots=1 << 16,
             positions=0, cos=0, sin=0, tokens=3, rows=0, q_heads=0, rotary=0, interleaved=0, dtype=0)
    f.update(kw)
    return lowbit._APPEND(*f.values())


@pytest.mark.parametrize("kw", [dict(k=0), dict(slots=0), dict(q=1 << 16), dict(q=1 << 16, q_out=1 << 16), dict(rotary=24, rows=1),
                                dict(rotary=256), dict(rotary=64), dict(dtype=7), dict(k_out=(1 << 16) + 2)])
def test_bad_appends_are_refused(lib, kw):
    from coraanns_b200 import CORA_EINVAL
    c = cache_arg()
    assert lib.cora_kv4_append(C.addressof(c), append_args(**kw), None) == CORA_EINVAL and message(lib)


def test_empty_calls_do_nothing(lib):
    from coraanns_b200 import lowbit
    c = cache_arg()
    assert lib.cora_kv4_append(C.addressof(c), append_args(tokens=0), None) == 0
    assert lib.cora_kv4_attend(C.addressof(c), lowbit._ATTEND(*[0] * 12, 0.5, *[0] * 7), None) == 0


def attend_args(**kw):
    from coraanns_b200 import lowbit
    f = dict(q=1 << 16, out=1 << 16, lse=0, qt=512, qh=128, table=1 << 16, lens=1 << 16, q_start=0, stride=4, tokens=2, size=0,
             work=1 << 16, scale=0.1, seqs=2, width=4, q_heads=4, max_queries=1, window=0, causal=1, dtype=0)
    f.update(kw)
    return lowbit._ATTEND(*f.values())


@pytest.mark.parametrize("kw", [dict(q=0), dict(out=0), dict(out=(1 << 16) + 2), dict(table=0), dict(lens=0), dict(q_heads=3),
                                dict(q_heads=0), dict(tokens=1), dict(window=5, causal=0), dict(width=1 << 30),
                                dict(tokens=1 << 40)])
def test_bad_attentions_are_refused(lib, kw):
    from coraanns_b200 import CORA_EINVAL
    c = cache_arg()
    assert lib.cora_kv4_attend(C.addressof(c), attend_args(**kw), None) == CORA_EINVAL and message(lib)


@pytest.mark.parametrize("wkw,kw", [(dict(group=16), {}), (dict(cols=0), {}), (dict(codes=0), {}), (dict(meta=(1 << 16) + 4), {}),
                                    ({}, dict(x=0)), ({}, dict(y=0)), ({}, dict(dtype=3))])
def test_bad_products_are_refused(lib, wkw, kw):
    from coraanns_b200 import CORA_EINVAL, lowbit
    w = dict(codes=1 << 16, meta=1 << 16, rows=4, cols=128, group=128)
    w.update(wkw)
    a = dict(x=1 << 16, bias=0, y=1 << 16, xs=128, ys=4, rows=2, dtype=0)
    a.update(kw)
    w = lowbit._WeightArg(**w)
    assert lib.cora_w4_matvec(C.addressof(w), lowbit._MATVEC(*a.values()), None) == CORA_EINVAL and message(lib)
