"""Direct global -> LDS loads of the 4-bit tile kernels (CPU: the built library's own code,
disassembled).  A block's rows for round v are loaded rounds ahead, and in front of the
barrier of round v every wave waits until at most N of its loads are in flight, N counted
in the source from the loads of the rounds behind it.  The compiler orders and may move the
loads of weights among them, so this follows every path and counts for itself: at the
barrier of round v none of the direct loads of round v is in flight."""

import os
import re

import pytest

from qllm2_amd import _lib
from tests.test_stage_waits import OBJDUMP, _kernels

LOAD = re.compile(r"^(global_load|buffer_load|flat_load|scratch_load)")
DIRECT = re.compile(r"^global_load_lds_")
STORE = re.compile(r"^(global_store|buffer_store|flat_store|scratch_store)")


def _early_barriers(code, each):
    """Addresses of barriers that are reached with a direct load in flight whose round is at hand: the j-th direct
    load belongs to round j // each.  State of a path: per operation in flight its round relative to the barriers
    passed (None: no direct load), and the same of the next direct load with its place in its round."""
    index = {a: i for i, (a, _) in enumerate(code)}
    todo, seen, bad = [(0, (), 0, 0)], set(), set()
    while todo:
        i, flight, ahead, nth = todo.pop()
        while i < len(code) and (i, flight, ahead, nth) not in seen:
            seen.add((i, flight, ahead, nth))
            at, op = code[i]
            if DIRECT.match(op):
                flight = (*flight, ahead)
                nth += 1
                if nth == each:
                    ahead, nth = ahead + 1, 0
            elif LOAD.match(op) or STORE.match(op):
                flight = (*flight, None)
            elif op.startswith("s_waitcnt"):
                vm = re.search(r"vmcnt\((\d+)\)", op)
                if vm:
                    flight = flight[max(0, len(flight) - int(vm.group(1))):]
            elif op.startswith("s_barrier"):
                if any(f is not None and f <= 0 for f in flight):
                    bad.add(hex(at))
                flight = tuple(None if f is None else f - 1 for f in flight)
                ahead -= 1
            if op.startswith("s_endpgm") or len(flight) > 400:
                break
            jump = re.match(r"s_(c?branch)\w*\s+(\d+)", op)
            if jump:
                off = int(jump.group(2))
                to = index[at + 4 + 4 * (off - 65536 if off >= 32768 else off)]
                if jump.group(1) == "branch":
                    i = to
                    continue
                todo.append((to, flight, ahead, nth))
            i += 1
    return sorted(bad)


def _each(symbol):
    """Direct loads a wave has in a round, from the kernel's template arguments."""
    t = re.search(r"tile_kernelI([tf])Lb[01]ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)E", symbol)
    wn, mt, u = int(t.group(2)), int(t.group(4)), int(t.group(9))
    return -(-(1 if t.group(1) == "t" else 3) * mt * 2 * u // wn)


def test_rounds_have_arrived_at_their_barriers(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip(f"no {OBJDUMP}")
    tiles = {k: c for k, c in _kernels(_lib.lib_path(), str(tmp_path)).items() if "w411tile_kernel" in k}
    assert len(tiles) >= 16
    assert not {k: b for k, b in ((k, _early_barriers(c, _each(k))) for k, c in tiles.items()) if b}


def test_the_check_itself():
    code = lambda *ops: [(4 * i, op) for i, op in enumerate(ops)]  # noqa: E731
    load, other, end = "global_load_lds_dwordx4 v[0:1], off", "global_load_dword v0, v1, s[0:1]", "s_endpgm"
    wait = "s_waitcnt vmcnt({}) lgkmcnt(0)".format
    assert not _early_barriers(code(load, other, load, other, wait(2), "s_barrier", wait(0), "s_barrier", end), 1)
    assert _early_barriers(code(load, other, load, other, wait(3), "s_barrier", end), 1) == []
    assert _early_barriers(code(load, load, other, wait(3), "s_barrier", end), 1) == ["0x10"]
    # a load of weights moved behind the barrier: the count lets the direct load pass
    assert _early_barriers(code(load, load, wait(2), "s_barrier", end), 1) == ["0xc"]
    # two loads a round
    assert _early_barriers(code(load, load, load, load, wait(2), "s_barrier", end), 2) == []
    assert _early_barriers(code(load, load, load, load, wait(3), "s_barrier", end), 2) == ["0x14"]
