"""CPU walks through the order of waits, hand-overs and products of the attention kernels (csrc/phases.h): every
interleaving of a small model, whose barriers answer by parity as an mbarrier does."""
import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe_stream_b200", "csrc")


@pytest.fixture(scope="module")
def phases(tmp_path_factory):
    at = tmp_path_factory.mktemp("phases")
    src, so = at / "p.cpp", at / "p.so"
    src.write_text('#include "phases.h"\nextern "C" {'
                   'int waits_before_handover(int j, int n) { return ms::waits_before_handover(j, n); }'
                   'int fill_phase(int k, int n) { return ms::fill_phase(k, n); }'
                   'int first_under_way(int k, int n) { return ms::first_under_way(k, n); }'
                   '}\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I" + CSRC, str(src), "-o", str(so)], check=True)
    return C.CDLL(str(so))


def softmax_programs(tiles, before, behind):
    """What a softmax warp of one query tile does: waits ("s" or "o", phase), arrivals ("p", tile).  With and without
    the wait of a rescaling at each tile.  before(j): it waits for product j - 1 in front of hand-over j; behind: the
    products that it waits for at the end."""
    out = []
    for raises in range(1 << max(0, tiles - 1)):
        prog = []
        for j in range(tiles):
            prog.append(("s", j))
            if j and raises >> (j - 1) & 1:
                prog.append(("o", j - 1))
            if before(j):
                prog.append(("o", j - 1))
            prog.append(("p", j))
        out.append(tuple(prog + [("o", j) for j in behind]))
    return out


def explore(tiles, programs):
    """All interleavings of two warps with these programs, the thread that issues the products, and the products'
    completions (in their order).  Returns what went wrong: "early" (a wait passed before its phase was over) or
    "stuck"."""
    issue = [("s", 0)] + ([("s", 1)] if tiles > 1 else [])
    for j in range(tiles):
        issue += [("wait", j), ("o", j)] + ([("s", j + 2)] if j + 2 < tiles else [])
    wrong, seen, todo = set(), set(), [(0, 0, (0, 0))]      # issued, completed, the warps' places
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        issued, completed, at = state
        done = [x for x in issue[:issued] if x[0] != "wait"]
        ended = done[:completed]
        products = sum(x[0] == "o" for x in ended)
        scores = [sum(x[0] == "s" and x[1] % 2 == b for x in ended) for b in (0, 1)]
        handed = [sum(x[0] == "p" for x in p[:a]) for p, a in zip(programs, at)]
        before = len(todo)
        if completed < len(done):
            todo.append((issued, completed + 1, at))
        if issued < len(issue) and (issue[issued][0] != "wait" or min(handed) > issue[issued][1]):
            todo.append((issued + 1, completed, at))
        for w, (prog, a) in enumerate(zip(programs, at)):
            if a == len(prog):
                continue
            kind, j = prog[a]
            if kind != "p":
                count, phase = (products, j) if kind == "o" else (scores[j % 2], j // 2)
                if count % 2 == phase % 2:                  # the phase of that parity is not over
                    continue
                if count <= phase:
                    wrong.add("early")
            todo.append((issued, completed, at[:w] + (a + 1,) + at[w + 1:]))
        if len(todo) == before and (issued < len(issue) or any(a < len(p) for p, a in zip(programs, at))):
            wrong.add("stuck")
    return wrong


@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5])
def test_softmax_waits_always_pass(phases, tiles):
    progs = softmax_programs(tiles, lambda j: phases.waits_before_handover(j, tiles), [tiles - 1])
    for a in progs:
        for b in progs:
            assert not explore(tiles, (a, b)), (a, b)


def test_the_model_sees_a_wait_that_comes_too_late():
    """Waiting for the last product but one behind the last hand-over: the last one may be over by then."""
    late = softmax_programs(3, lambda j: False, [1, 2])[0]
    assert "stuck" in explore(3, (late, late))
    none = softmax_programs(3, lambda j: False, [2])[0]     # and without it the last one's wait may pass early
    assert "early" in explore(3, (none, none))


@pytest.mark.parametrize("stages", [1, 2, 4])
def test_a_ring_waits_for_every_fill(phases, stages):
    """After any number of fills of which any of the last `stages` have not landed, a wait for one passes exactly when it
    has landed (a wait for parity 0 would pass at once where the fill under way is an odd one)."""
    for issued in range(1, 4 * stages + 1):
        assert phases.first_under_way(issued, stages) == max(0, issued - stages)
        for k in range(phases.first_under_way(issued, stages), issued):
            for landed in (False, True):
                count = sum(i % stages == k % stages for i in range(k)) + landed   # phases of that stage that are over
                assert (count % 2 != phases.fill_phase(k, stages) % 2) == landed
