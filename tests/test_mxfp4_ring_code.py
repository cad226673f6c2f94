"""The ring's matrix instructions that stand in asm, in the machine code of the built library (no kernel runs): the compiler does not know
them for what they are, so nothing but the next product may touch a sum until its instruction has written it."""
import os
import re

import pytest

from tests.test_w3_ring_waits import OBJDUMP, _kernels

WAIT_STATES = 19  # of a vector instruction behind a matrix instruction of sixteen passes that writes what it reads or writes
SUM = re.compile(r"v_mfma_scale_f32_32x32x64_f8f6f4 a\[(\d+):(\d+)\]")
TOUCHED = re.compile(r"\ba(?:\[(\d+):(\d+)\]|(\d+)\b)")


def _touches(ins, lo, hi):
    return any(int(m[1] or m[3]) <= hi and int(m[2] or m[3]) >= lo for m in TOUCHED.finditer(ins))


def _too_early(code):
    """(matrix instruction, what touches its sum, wait states between) of every way that is too short."""
    place = {at: i for i, (at, _) in enumerate(code)}
    for i, (_, ins) in enumerate(code):
        sums = SUM.match(ins)
        if not sums:
            continue
        lo, hi = int(sums[1]), int(sums[2])
        todo, seen = [(i, 0)], set()
        while todo:
            j, states = todo.pop()
            at, here = code[j]
            if j != i or states:
                if not here.startswith("v_mfma") and _touches(here, lo, hi):
                    yield ins, here, states
                    continue
                states += int(here.split()[1]) + 1 if here.startswith("s_nop") else 1
            if states >= WAIT_STATES or here.startswith("s_endpgm") or (j, states) in seen:
                continue
            seen.add((j, states))
            ahead = [] if here.startswith("s_branch") else [j + 1]
            if here.startswith(("s_branch", "s_cbranch")):
                words = int(here.split()[1])
                ahead.append(place[at + 4 + 4 * (words - 65536 if words >= 32768 else words)])
            todo += [(h, max(states, 1) if j == i else states) for h in ahead if h < len(code)]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_nothing_touches_a_sum_before_it_is_written(tmp_path):
    checked = 0
    for name, code in _kernels(tmp_path, r"mx_ring_kernelI.*Li2ELi2ELi4ELi4E"):
        assert sum(bool(SUM.match(ins)) for _, ins in code) >= 128, name
        assert not list(_too_early(code)), name
        checked += 1
    assert checked == 3, checked


def test_the_check_finds_a_sum_read_early():
    nops = [(8, "s_nop 15"), (12, "s_nop 3")]
    product = (0, "v_mfma_scale_f32_32x32x64_f8f6f4 a[16:31], v[0:7], v[8:15], a[16:31], v16, v17 op_sel_hi:[0,0,0] cbsz:4 blgp:4")
    assert list(_too_early([product, (8, "v_accvgpr_read_b32 v1, a31"), (12, "s_endpgm")]))
    assert list(_too_early([product, (8, "s_cbranch_scc0 1"), (12, "s_endpgm"), (16, "v_accvgpr_mov_b32 a0, a16"), (20, "s_endpgm")]))
    assert not list(_too_early([product, *nops, (16, "v_accvgpr_read_b32 v1, a31"), (20, "s_endpgm")]))
    assert not list(_too_early([product, (8, "v_accvgpr_read_b32 v1, a32"), (12, "s_endpgm")]))
