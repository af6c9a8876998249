"""The lists of blocks in LDS and their union, on the CPU."""

import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_the_union_of_lists_holds_their_blocks_only(tmp_path):
    exe = tmp_path / "kv_lists_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror",
                    f"-I{ROOT / 'mlxvs_amd' / 'csrc'}",
                    str(ROOT / "tests" / "c" / "kv_lists_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and "all tests passed" in r.stdout, r.stdout + r.stderr
