"""Wait states of the LDS loads written as asm blocks, in the device code as compiled: a
vector instruction's write of a scalar register (v_readfirstlane, v_readlane) must lie five
wait states before a load that reads the register. The compiler counts them for its
own instructions only."""

import concurrent.futures as cf
import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG

from cab_attention import _build

LOAD = re.compile(r"buffer_load\S* .* lds$")
WRITE = re.compile(r"v_read(?:first)?lane_b32 (s\d+)")


def scalars(text):
    out = set()
    for m in re.finditer(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", text):
        out |= set(range(int(m[1]), int(m[2]) + 1)) if m[1] else {int(m[3])}
    return out


def short_waits(lines):
    """(load, write, wait states between) of loads too near a vector instruction's write
    of one of their scalars."""
    code = [x.strip() for x in lines]
    code = [x for x in code if x and not x.startswith((";", "."))]
    out = []
    for i, line in enumerate(code):
        if not LOAD.match(line):
            continue
        reads, wait = scalars(line), 0
        for before in reversed(code[max(0, i - 8):i]):
            if wait >= 5 or before.endswith(":"):
                break
            m = WRITE.match(before)
            if m and scalars(m[1]) & reads:
                out.append((line, before, wait))
                break
            nop = re.match(r"s_nop (\d+)", before)
            wait += int(nop[1]) + 1 if nop else 1
    return out


def test_the_check_itself():
    load = "buffer_load_dwordx4 v0, s[0:3], s14 offen lds"
    assert short_waits(["v_readfirstlane_b32 s0, v1", "s_mov_b32 m0, s9", "s_nop 2", load])
    assert short_waits(["v_readlane_b32 s14, v1, 3", "s_nop 3", load])
    assert not short_waits(["v_readlane_b32 s14, v1, 3", "s_nop 4", load])
    assert not short_waits(["v_readfirstlane_b32 s0, v1", "s_mov_b32 m0, s9", "s_nop 3", load])
    assert not short_waits(["v_readlane_b32 s15, v1, 3", load])


def test_compiled_loads_wait(tmp_path):
    if not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")):
        pytest.skip("hipcc not available")
    sources = [p for p in sorted((PKG / "csrc").glob("*.hip"))
               if re.search(r"bdma16_untracked\(|buffer_load_dword", p.read_text())]
    assert {p.name for p in sources} >= {"sparse_attn.hip", "tree_attn.hip"}

    def compile_one(src):
        out = tmp_path / (src.stem + ".s")
        cmd = [_build._hipcc(), *_build.HIPCC_FLAGS, *_build.EXTRA_FLAGS.get(src.name, []),
               "--cuda-device-only", "-S", str(src), "-o", str(out)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        assert res.returncode == 0, res.stderr[-2000:]
        return src.name, out.read_text().splitlines()

    with cf.ThreadPoolExecutor(4) as pool:
        for name, lines in pool.map(compile_one, sources):
            assert sum(bool(LOAD.match(x.strip())) for x in lines) > 0, name
            bad = short_waits(lines)
            assert not bad, (name, len(bad), bad[:4])
