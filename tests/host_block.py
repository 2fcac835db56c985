"""Compiles a kernel's headers for the host, with host_block.h in place of the
helpers that are inline PTX."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from conftest import PKG_DIR, ROOT

# Helpers that host_block.h has a version of (the rest of a file is taken as it is).
HELPERS = {
    "serve.cuh": ("cluster_sync", "cluster_map", "ld_cluster"),
    "attn_rows.cuh": ("exp2_fast", "mma_act", "ldsm4", "ldsm4_t", "cp_async16_or_zero", "cp_async_commit",
                      "cp_async_wait"),
    "attn_tiles.cuh": ("max3", "pair2", "unpair2", "fma2", "add2"),
}


def without(text: str, name: str) -> str:
    """`text` without the definition of function `name`."""
    m = re.search(r"^(template <[^\n]*>\n)?__device__ __forceinline__ \w+ " + name + r"\(", text, re.M)
    at = text.index("{", m.end())
    depth = 1
    while depth:
        at += 1
        depth += {"{": 1, "}": -1}.get(text[at], 0)
    return text[:m.start()] + text[at + 1:]


def compile_blocks(tmp: Path, program: str, sources=(), change=lambda name, text: text) -> Path:
    """The program's path; `sources` are copied beside it, cut by `change`."""
    cuda = Path("/usr/local/cuda/include")
    if shutil.which("g++") is None or not cuda.exists():
        pytest.skip("no g++ or no CUDA headers")
    src = tmp / "src" / "csrc"
    src.mkdir(parents=True)
    (tmp / "include").mkdir()
    shutil.copy(ROOT / "include" / "b200gemv.h", tmp / "include")
    for name in ("serve.h", *HELPERS, *sources):
        text = change(name, (PKG_DIR / "csrc" / name).read_text())
        for h in HELPERS.get(name, ()):
            text = without(text, h)
        text = re.sub(r"extern __shared__ (?:__align__\(1024\) )?uint8_t (\w+)\[\];", r"uint8_t* \1 = emu::smem;", text)
        assert "asm" not in re.findall(r"\w+", text), name
        (src / name).write_text(text)
    for name in ("device.cuh", "tc.cuh"):
        (src / name).write_text("#pragma once\n")
    (src / "program.cpp").write_text('#include "host_block.h"\n' + program)
    exe = tmp / "program"
    subprocess.run(["g++", "-std=c++17", "-O2", "-w", "-I", str(src), "-I", str(Path(__file__).parent), "-I", str(cuda),
                    "-o", str(exe), str(src / "program.cpp")], check=True)
    return exe
