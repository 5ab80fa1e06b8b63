"""CPU tests of the 4-bit reader operators: what the source has to keep to, host-side logic."""
from __future__ import annotations

import contextlib
import ctypes as C
import re
import struct
import threading
import time

import pytest

from conftest import ROOT

CORA_ERUNTIME = 3
torch = pytest.importorskip("torch")

CSRC = ROOT / "cgcl-coraanns_b200" / "csrc"


def code_of(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_roles_of_the_tile_kernel_meet_with_a_limit():
    """A role that gives up after a wait that ran out goes straight to the end of the block; whoever
    waits for it must do so with a limit. So between the block's first and last barrier (which every
    thread reaches) there is no barrier without one: no block or named barrier, no endless loop."""
    code = code_of("kernels_lowbit_chunk.cuh")
    kernel = code[code.index("kv4_chunk_kernel(const AttendParams p) {"):]
    parts = kernel.split("__syncthreads();")
    assert len(parts) == 3
    roles = parts[1]
    for forbidden in ("named_barrier_sync", "bar.sync", "barrier.sync", "barrier.cluster", "mbar_try_wait", "while (true)", "for (;;)"):
        assert forbidden not in roles, forbidden
    assert "mbar_wait_short" in roles


@pytest.mark.parametrize("width,page,tokens", [((1 << 31) // 64 - 1, 64, 2), ((1 << 31) // 1024 - 8, 1024, 2),
                                               ((1 << 31) // 16 - 33, 16, 100), (1 << 20, 1024, (1 << 30))])
def test_tables_whose_positions_pass_an_int_are_refused(width, page, tokens):
    """The kernels hold positions, and pages up to 32 ahead, as ints."""
    from test_lowbit_abi import attend_args, cache_arg
    from coraanns_b200 import CORA_EINVAL, lowbit
    lib = lowbit._library()
    c = cache_arg(page_size=page)
    assert lib.cora_kv4_attend(C.addressof(c), attend_args(width=width, tokens=tokens), None) == CORA_EINVAL
    assert b"table_width" in lib.cora_last_error()


# ---- attention's workspaces, on host memory with the C calls replaced -----------------------------


class FakeCalls:
    """The C entries that attention's host side uses. An attention call looks at its workspace (the
    first byte has to be zero unless the call is captured) and leaves it used."""

    def __init__(self):
        self.stream, self.capturing, self.sizes, self.calls, self.timed_out = 1, False, 0, [], False

    def cora_kv4_block_bytes(self, page, dim, group):
        return page * dim + 8 * page * (dim // group)

    def cora_kv4_attend_workspace(self, cache, heads, queries):
        self.sizes += 1
        rows = queries * heads // 2  # (two key heads below)
        return 1 << 12 if rows <= 32 else 1 << 14 if rows <= 128 else 1 << 16

    def cora_kv4_attend(self, cache, args, stream):
        v = struct.unpack("3Q2q3Qq3Qf7I", args)  # cora_kv4_attend_args
        size, work = v[10], v[11]
        first = C.c_ubyte.from_address(work)
        self.calls.append((work, size, first.value))
        first.value = 0xff if self.capturing else 0  # a captured call runs later: nothing has readied its memory
        return 0

    def cora_kv4_status(self, cache, stream):
        return CORA_ERUNTIME if self.timed_out else 0


@pytest.fixture
def fake(monkeypatch):
    from coraanns_b200 import lowbit
    f = FakeCalls()
    monkeypatch.setattr(lowbit, "_library", lambda: f)
    monkeypatch.setattr(lowbit, "_stream", lambda index: f.stream)
    monkeypatch.setattr(lowbit, "_current_device", lambda: -1)
    monkeypatch.setattr(lowbit, "_capturing", lambda: f.capturing, raising=False)
    monkeypatch.setattr(lowbit, "_index", lambda t, *_: t.data_ptr())
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())

    def cache():
        c = lowbit.Cache4(2, 2, 64, page_size=16, device="cpu")
        c._dev = -1
        return c

    def attend(c, queries=1):
        one = torch.ones(1, dtype=torch.int32)
        c.attend(torch.zeros(1, 2, 64, dtype=torch.bfloat16), one[None], one, max_queries=queries)
        return f.calls[-1]

    f.cache, f.attend = cache, attend
    return f


def test_captured_attention_has_a_workspace_of_its_own(fake):
    """A captured call neither takes an eager call's workspace (its replays would share it, and find
    it freed once a larger call replaced it) nor leaves its own to others (that was never zeroed)."""
    c = fake.cache()
    fake.capturing = True
    fake.attend(c)
    fake.capturing = False
    eager = fake.attend(c)
    assert eager[2] == 0
    fake.capturing = True
    assert fake.attend(c)[0] != eager[0]
    fake.capturing = False
    assert fake.attend(c) == eager
    big = fake.attend(c, 40)
    assert big[1] > eager[1] and big[2] == 0
    assert fake.attend(c) == big  # the larger one serves both


def test_caches_share_a_streams_workspace(fake):
    a, b = fake.cache(), fake.cache()
    first = fake.attend(a)
    assert fake.attend(b) == first
    fake.stream = 2
    assert fake.attend(b)[0] != first[0]
    fake.stream = 1
    grown = fake.attend(b, 500)
    assert fake.attend(a) == grown


def test_workspace_sizes_are_not_kept_for_every_length(fake):
    c = fake.cache()
    for n in range(1, 500):
        fake.attend(c, n)
    assert fake.sizes <= 33
    sizes = {fake.attend(fake.cache(), n)[1] for n in (1, 32)}
    assert len(sizes) == 1


def test_workspace_after_a_wait_that_ran_out(fake):
    """A call that gave up may leave arrival counters standing: no later call starts from them."""
    from coraanns_b200 import CoraRuntimeError
    a, b = fake.cache(), fake.cache()
    work = fake.attend(a)[0]
    C.c_ubyte.from_address(work).value = 5
    fake.timed_out = True
    with pytest.raises(CoraRuntimeError):
        a.check()
    assert fake.attend(b)[2] == 0 and fake.attend(a)[2] == 0


def test_threads_share_the_first_workspace_of_a_stream(fake, monkeypatch):
    """Two threads' first calls on one stream end up with one workspace, not one that the other frees."""
    zeros = torch.zeros

    def slow(*shape, **kw):
        t = zeros(*shape, **kw)
        if kw.get("dtype") is torch.uint8:
            time.sleep(0.2)
        return t

    c = fake.cache()
    monkeypatch.setattr(torch, "zeros", slow)
    q, one = torch.ones(1, 2, 64).to(torch.bfloat16), torch.ones(1, dtype=torch.int32)
    threads = [threading.Thread(target=c.attend, args=(q, one[None], one)) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len({work for work, _, _ in fake.calls}) == 1 and len(fake.calls) == 2


@pytest.mark.parametrize("kw", [dict(window=1 << 31), dict(window=1 << 40), dict(window=-1), dict(max_queries=1 << 32),
                                dict(max_queries=0), dict(scale=3.5e38), dict(scale=-1e300)])
def test_numbers_past_their_fields_are_refused(fake, kw):
    from coraanns_b200 import InvalidArgument
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(InvalidArgument):
        fake.cache().attend(torch.zeros(1, 2, 64, dtype=torch.bfloat16), one[None], one, **kw)
    assert not fake.calls


def test_largest_numbers_are_taken(fake):
    one = torch.ones(1, dtype=torch.int32)
    for kw in (dict(window=(1 << 31) - 1), dict(max_queries=(1 << 32) - 1), dict(scale=3.4028234e38)):
        fake.cache().attend(torch.zeros(1, 2, 64, dtype=torch.bfloat16), one[None], one, **kw)
    assert len(fake.calls) == 3
