"""Static check of the built gfx950 code: results of the products that kv_weigh.hip
writes out itself.

The compiler counts the wait states between an MFMA and a vector instruction that
reads its result, but not for one in inline assembly.  On every path from a
v_mfma_f32_32x32x16 (8 passes: 12 wait states, as test_mfma_barrier_waits finds the
compiler to apply) to the first such read this test counts the wait states that
surely pass, as that one does: an instruction one, s_nop N N + 1, s_barrier and
s_waitcnt none.  Nor does it count them between a vector instruction and an MFMA that
reads what that one wrote (2).  CPU only.
"""

import re

import pytest

from mlxvs_amd import build as B
from test_mfma_barrier_waits import REG, _regs, disassemble, parse

NEED = 12
NEED_BEFORE = 2
KIND = "v_mfma_f32_32x32x16"


def short_reads(insts):
    """(function, wait states) of the reads that come too soon."""
    bad = []

    def walk(j, dst, waits, seen):
        while j < len(insts) and waits < NEED:
            if seen.get(j, 1 << 30) <= waits:
                return
            seen[j] = waits
            func, op, text, tgt = insts[j]
            j += 1
            if op == "s_endpgm":
                return
            toks = re.findall(REG, text)
            if op.startswith("v_") and toks:
                srcs = set().union(*(_regs(t) for t in toks[1:])) if len(toks) > 1 else set()
                if op.startswith("v_mfma"):
                    # (the next one of a sum waits by itself, and replaces it)
                    if _regs(toks[0]) & dst:
                        return
                elif srcs & dst:
                    bad.append((func, waits, text))
                    return
                elif _regs(toks[0]) & dst:
                    bad.append((func, waits, text))  # (written over while it is made)
                    return
            if op == "s_nop":
                waits += int(text.split()[1], 0) + 1
            elif op not in ("s_barrier", "s_waitcnt"):
                waits += 1
            if op.startswith("s_cbranch") or op == "s_branch":
                if tgt is not None:
                    walk(tgt, dst, waits, seen)
                if op == "s_branch":
                    return

    for i, (func, op, text, _) in enumerate(insts):
        if op.startswith(KIND):
            walk(i + 1, _regs(text.split()[1].rstrip(",")), 0, {})
    return bad


def short_writes(insts):
    """... and of the operands that are written too late, straight before a product."""
    bad = []
    for i, (func, op, text, _) in enumerate(insts):
        if not op.startswith(KIND):
            continue
        srcs = set().union(*(_regs(t) for t in re.findall(REG, text)[1:]))
        waits = 0
        while i > 0 and waits < NEED_BEFORE:
            i -= 1
            _, op, text, _ = insts[i]
            toks = re.findall(REG, text)
            if op.startswith("v_") and not op.startswith("v_mfma") and toks and _regs(toks[0]) & srcs:
                bad.append((func, waits, text))
            if op == "s_nop":
                waits += int(text.split()[1], 0) + 1
            elif op not in ("s_barrier", "s_waitcnt"):
                waits += 1
    return bad


def test_results_of_written_out_products(tmp_path):
    obj = B.BUILD / "kv_weigh.o"
    if not obj.exists():
        pytest.skip("no built objects (run python -m mlxvs_amd.build)")
    insts = parse(disassemble(obj, tmp_path))
    assert sum(i[1].startswith(KIND) for i in insts) > 100
    assert short_reads(insts) == []
    assert short_writes(insts) == []


def test_the_check_finds_a_short_read():
    listing = """0000000000000000 <_ZShort>:
\tv_mfma_f32_32x32x16_bf16 v[0:15], a[0:3], v[20:23], v[0:15]  // 000000000000: 0
\tv_mfma_f32_32x32x16_bf16 v[32:47], a[0:3], v[20:23], 0       // 000000000008: 0
\ts_nop 7                                                      // 000000000010: 0
\ts_nop 0                                                      // 000000000014: 0
\tv_mov_b32_e32 v60, v61                                       // 000000000018: 0
\tv_add_f32_e32 v50, v15, v15                                  // 00000000001C: 0
\tv_add_f32_e32 v51, v47, v50                                  // 000000000020: 0
\ts_endpgm                                                     // 000000000024: 0
""".split("\n")
    # the first sum is read after 1 + 8 + 1 + 1 = 11, the second after 11, too
    assert [w for _, w, _ in short_reads(parse(listing))] == [11, 11]


def test_the_check_finds_a_late_write():
    listing = """0000000000000000 <_ZLate>:
\tv_accvgpr_read_b32 v23, a9                                    // 000000000000: 0
\tv_accvgpr_read_b32 v20, a8                                    // 000000000008: 0
\ts_nop 0                                                      // 000000000010: 0
\tv_mfma_f32_32x32x16_bf16 v[0:15], a[0:3], v[20:23], v[0:15]  // 000000000014: 0
\ts_endpgm                                                     // 00000000001C: 0
""".split("\n")
    assert [w for _, w, _ in short_writes(parse(listing))] == [1]
