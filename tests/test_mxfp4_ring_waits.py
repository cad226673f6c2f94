"""The waits of the ring of steps in the machine code of the built library (no kernel runs). A step ends with a wait and a barrier; behind them a
wavefront reads the next step's tiles and the first chunk of the one behind it. What the wait may leave on its way is therefore the youngest step's loads
into LDS and, of the step's before, those that are of its second chunk alone. The wait counts every load of the step, the scales too, so it rests on
the compiler making them all: it drops one whose result nothing uses."""
import os
import re

import pytest

from tests.test_w3_ring_waits import OBJDUMP, REQUEST, _kernels

WAIT = re.compile(r"s_waitcnt\b.*vmcnt\((\d+)\)")


def _allowed(name):
    """Loads into LDS that a wait may leave outstanding, from the kernel's tiling: wavefronts along rows and columns, tiles a wavefront."""
    tiling = re.search(r"mx_ring_kernelI\w*?Li(\d)ELi(\d)ELi(\d)ELi(\d)E", name)
    wm, wn, mt, nt = map(int, tiling.groups()) if tiling else (2, 2, 2, 2)
    waves, of_a, of_b = wm * wn, wm * mt, wn * nt
    asks_a, asks_b = -(-2 * of_a // waves), 2 * of_b // waves
    second = asks_b // 2 + (asks_a // 2 if of_a % waves == 0 else 0)
    return asks_a + asks_b + second


def _ways_back(code):
    place = {at: i for i, (at, _) in enumerate(code)}
    before = [[] for _ in code]
    for i, (at, ins) in enumerate(code):
        if ins.startswith(("s_branch", "s_cbranch")):
            words = int(ins.split()[1])
            before[place[at + 4 + 4 * (words - 65536 if words >= 32768 else words)]].append(i)
        if not ins.startswith(("s_branch", "s_endpgm", "s_setpc")) and i + 1 < len(code):
            before[i + 1].append(i)
    return before


def _left_at_barriers(code):
    """For every barrier the most loads into LDS among the youngest requests that the wait ahead of it leaves outstanding, over all ways there."""
    before = _ways_back(code)
    for i, (_, ins) in enumerate(code):
        if not ins.startswith("s_barrier"):
            continue
        j = i - 1  # the nearest wait ahead: the step's own
        while j >= 0 and not WAIT.match(code[j][1]) and not REQUEST.match(code[j][1]) and not code[j][1].startswith(("s_branch", "s_cbranch", "s_barrier")):
            j -= 1
        wait = WAIT.match(code[j][1])
        assert wait, (i, "no wait ahead of the barrier")
        left = int(wait[1])
        most, seen, todo = 0, set(), [(h, left, 0) for h in before[i]]
        while todo:
            state = todo.pop()
            if state in seen:
                continue
            seen.add(state)
            at, room, into_lds = state
            if room and REQUEST.match(code[at][1]):
                room, into_lds = room - 1, into_lds + code[at][1].endswith(" lds")
                most = max(most, into_lds)
            if room:
                todo += [(h, room, into_lds) for h in before[at]]
        yield most


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_a_step_ends_when_the_next_ones_tiles_are_there(tmp_path):
    checked = 0
    for name, code in _kernels(tmp_path, r"mx_(ring|fc1_ring|fc2_ring)_kernel"):
        left = list(_left_at_barriers(code))
        assert len(left) >= 8, (name, left)  # the beginning, four steps, the last one or two quads' two, the end
        assert max(left) <= _allowed(name), (name, _allowed(name), left)
        checked += 1
    assert checked >= 22, checked  # three types of six tilings, and the experts' four


def test_the_check_finds_a_wait_that_counts_a_load_nobody_makes():
    lds, scale = "buffer_load_dwordx4 v1, s[0:3], 0 offen lds", "buffer_load_dword v2, v1, s[0:3], 0 offen"
    def left(*body):
        return list(_left_at_barriers([(4 * i, ins) for i, ins in enumerate((*body, "s_barrier", "s_endpgm"))]))
    assert left(lds, lds, scale, lds, "s_waitcnt vmcnt(3)") == [2]
    assert left(lds, lds, lds, "s_waitcnt vmcnt(3)") == [3]
    assert left(lds, lds, "s_waitcnt vmcnt(0)") == [0]
