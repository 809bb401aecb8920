"""Every LDS load written as an asm block holds all of the wait states a vector instruction's
write of one of its scalars needs, five, inside the block: the compiler counts none there, and
what precedes a block (a label, another block's end, an M0 write or none) is its choice."""

import concurrent.futures as cf
import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG

from cab_attention import _build


def short_blocks(lines):
    """(loads in asm blocks, those before which the block waits less than five states)."""
    loads, short, wait = 0, [], None
    for line in (x.strip() for x in lines):
        if "#ASMSTART" in line:
            wait = 0
        elif "#ASMEND" in line:
            wait = None
        elif wait is not None and line and not line.startswith((";", ".")):
            nop = re.match(r"s_nop (\d+)", line)
            if re.match(r"buffer_load\S* .* lds$", line):
                loads += 1
                if wait < 5:
                    short.append((line, wait))
            wait += int(nop[1]) + 1 if nop else 1
    return loads, short


def test_the_check_itself():
    load = "buffer_load_dwordx4 v0, s[0:3], s14 offen lds"
    assert short_blocks(["\ts_nop 4", "\t;;#ASMSTART", "\t" + load, "\t;;#ASMEND"]) == (1, [(load, 0)])
    assert short_blocks([";;#ASMSTART", "s_nop 3", load, ";;#ASMEND"]) == (1, [(load, 4)])
    assert short_blocks([";;#ASMSTART", "s_nop 4", load, ";;#ASMEND", load]) == (1, [])


def test_compiled_blocks_wait(tmp_path):
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
            loads, short = short_blocks(lines)
            assert loads > 0, name
            assert not short, (name, len(short), short[:4])
