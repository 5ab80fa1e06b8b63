"""CPU tests of the 4-bit reader operators: what the source has to keep to, host-side logic."""
from __future__ import annotations

import re

from conftest import ROOT

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
