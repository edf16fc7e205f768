"""The paged tile kernel's direct-to-LDS loads, checked in the code the compiler emits for
it (CPU only: hipcc cross-compiles).

The loads are issued from inline assembly, which the compiler does not count: the kernel's
own waits and barriers order them.  That needs two things of the emitted code.  M0, which
holds a load's LDS address, is used by nothing else; and where more than one block of keys
is on its way (four stages), no load of the compiler's own sits among them in the key
loop, since the wait leaves a number of loads outstanding.
"""

import os
import re
import shutil
import subprocess

import pytest

from cutilegpt_amd import build as B

SRC = "paged_tile.hip"


def _kernels(tmp_path):
    out = tmp_path / "k.s"
    cmd = [B.hipcc(), *B.HIPCC_FLAGS, *B.FILE_FLAGS[SRC], "-Wno-inline-asm", "--cuda-device-only", "-S",
           os.path.join(B.CSRC, SRC), "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    kernels = {}
    name = None
    for line in (l.split(";")[0].strip() for l in out.read_text().splitlines()):
        m = re.match(r"(_ZN4cgpt17paged_tile_kernel\S*):", line)
        if m:
            name = m.group(1)
            kernels[name] = []
        elif name and line:
            kernels[name].append(line)
    return kernels


def _loop_of_barrier(lines):
    """The instructions of every basic block on a cycle through the (only) s_barrier."""
    blocks, label = {"": []}, ""
    order = [""]
    for line in lines:
        m = re.match(r"(\.LBB\w+):", line)
        if m or (blocks[label] and blocks[label][-1].startswith(("s_cbranch", "s_branch", "s_endpgm"))):
            label = m.group(1) if m else f"{label}+"
            blocks[label] = []
            order.append(label)
        if not m and not line.startswith("."):
            blocks[label].append(line)
    after = {}
    for i, b in enumerate(order):
        last = blocks[b][-1] if blocks[b] else ""
        nxt = [order[i + 1]] if i + 1 < len(order) and not last.startswith(("s_branch", "s_endpgm")) else []
        after[b] = nxt + ([last.split()[1]] if last.startswith(("s_cbranch", "s_branch")) else [])

    def reach(start, edges):
        seen, todo = set(), [start]
        while todo:
            for n in edges.get(todo.pop(), []):
                if n not in seen:
                    seen.add(n)
                    todo.append(n)
        return seen

    before = {}
    for b, ns in after.items():
        for n in ns:
            before.setdefault(n, []).append(b)
    home = next(b for b in order if any(l.startswith("s_barrier") for l in blocks[b]))
    return [l for b in reach(home, after) & reach(home, before) for l in blocks[b]]


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_loads_to_lds(tmp_path):
    kernels = _kernels(tmp_path)
    deep = {k: v for k, v in kernels.items() if k.split("EEEvNS_")[0].endswith("Li4")}
    assert len(kernels) >= 60 and len(deep) >= 12, (len(kernels), len(deep))
    for name, lines in kernels.items():
        moves = 0
        for i, line in enumerate(lines):
            if re.search(r"\bm0\b", line):
                assert line.startswith("s_mov_b32 m0,"), (name, line)
                assert lines[i + 1] == "s_nop 0" and lines[i + 2].startswith("global_load_lds_dwordx4"), lines[i:i + 3]
                moves += 1
        assert moves > 0, name
    for name, lines in deep.items():
        loop = _loop_of_barrier(lines)
        assert sum(l.startswith("s_barrier") for l in loop) == 1, name
        assert sum(l.startswith("global_load_lds") for l in loop) in (2, 4, 8), name  # K and V of one block
        assert any(re.match(r"s_waitcnt vmcnt\((2|4|8|16)\)", l) for l in loop), name
        loads = [l for l in loop if re.match(r"(global|buffer|scratch|flat)_(load|store)", l) and "lds" not in l]
        assert not loads, (name, loads[:4])
