"""Pipelines of direct global -> LDS loads (CPU: the built library's own code, disassembled): behind
the barrier of a stage any wave may start loads over what was read in front of it, so no wave
arrives there with LDS reads under way.  The compiler waits for a read where its value is used,
and may move that use behind a barrier that the source has it in front of."""

import os
import re
import shutil
import subprocess

import pytest

from qllm2_amd import _lib

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
TO_LDS = re.compile(r"\b(global|buffer)_load_lds_|\bbuffer_load_\w+ .*\blds\b")
READ = re.compile(r"^ds_(read|load|bpermute|permute|swizzle)")


def _kernels(path, tmp):
    """{symbol: [(address, instruction)]} of the library's device code."""
    copy = shutil.copy(path, tmp)
    subprocess.run([OBJDUMP, "--offloading", copy], cwd=tmp, check=True, capture_output=True)
    out = {}
    for name in os.listdir(tmp):
        if "gfx950" not in name:
            continue
        text = subprocess.run([OBJDUMP, "-d", os.path.join(tmp, name)], check=True, capture_output=True, text=True).stdout
        for block in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            head = re.match(r"[0-9a-f]{16} <(\S+)>:", block)
            if head and TO_LDS.search(block):
                out[head.group(1)] = [(int(m.group(2), 16), m.group(1).strip()) for m in
                                      re.finditer(r"^\t([a-z].*?)\s*// ([0-9A-F]+):", block, re.M)]
    return out


def _reads_at_barriers(code):
    """Addresses of barriers that are reached with LDS reads not waited for, over all paths."""
    index = {a: i for i, (a, _) in enumerate(code)}
    todo, seen, bad = [(0, False)], set(), set()
    while todo:
        i, reads = todo.pop()
        while i < len(code) and (i, reads) not in seen:
            seen.add((i, reads))
            at, op = code[i]
            if READ.match(op):
                reads = True
            elif op.startswith("s_waitcnt"):
                lgkm = re.search(r"lgkmcnt\((\d+)\)", op)
                reads = reads and not (lgkm and lgkm.group(1) == "0")
            elif op.startswith("s_barrier") and reads:
                bad.add(hex(at))
            if op.startswith("s_endpgm"):
                break
            jump = re.match(r"s_(c?branch)\w*\s+(\d+)", op)
            if jump:
                off = int(jump.group(2))
                to = index[at + 4 + 4 * (off - 65536 if off >= 32768 else off)]
                if jump.group(1) == "branch":
                    i = to
                    continue
                todo.append((to, reads))
            i += 1
    return sorted(bad)


def test_no_lds_read_crosses_a_stage_barrier(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip(f"no {OBJDUMP}")
    kernels = _kernels(_lib.lib_path(), str(tmp_path))
    names = " ".join(kernels)
    for known in ("state_pass_f32", "fwd_tile_kernel", "scores_tile_kernel", "scores_grad_kernel", "gemm_kernel", "thin"):
        assert known in names, known
    assert not {k: b for k, b in ((k, _reads_at_barriers(c)) for k, c in kernels.items()) if b}


def test_the_check_itself():
    code = lambda *ops: [(4 * i, op) for i, op in enumerate(ops)]  # noqa: E731
    ok = code("ds_read_b128 v[0:3], v4", "s_waitcnt vmcnt(4) lgkmcnt(0)", "s_barrier", "s_cbranch_scc1 65532", "s_endpgm")
    assert not _reads_at_barriers(ok)
    assert _reads_at_barriers(code("ds_read_b128 v[0:3], v4", "s_waitcnt vmcnt(4)", "s_barrier", "s_endpgm")) == ["0x8"]
    # round a loop: the read behind the barrier meets it again
    assert _reads_at_barriers(code("s_barrier", "ds_read_b32 v0, v1", "s_cbranch_scc1 65533", "s_endpgm")) == ["0x0"]
    assert not _reads_at_barriers(code("ds_read_b32 v0, v1", "s_cbranch_scc1 1", "s_endpgm", "s_waitcnt lgkmcnt(0)", "s_barrier", "s_endpgm"))
