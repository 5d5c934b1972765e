"""The counted waits of the 8-bit product's tiles, followed through the built code on the CPU.

A workgroup of matmul_tiles (kernels/matmul_fp8.hip) loads steps of the sum into LDS and waits for them by the number of
its later accesses that may still be under way. A wave's accesses are followed here from the kernel's entry along every
branch, and at each barrier the loads that the reads after it need have to be covered by a wait, in a workgroup's first
tile as in those that follow one. Timing hides a wait that is too weak, so no result can show it."""
import re

import pytest

import built_code

# Kernels by the tiles of a wave, TM x TN: a step's loads are TM of X and TN of Y; X and the first half of Y are read after
# a step's second barrier, the rest of Y after the next step's first.
KERNELS = {"helix_matmul_fp8_t88": (8, 8), "helix_matmul_fp8_t86": (8, 6), "helix_matmul_fp8_t84": (8, 4),
           "helix_matmul_fp8_t44": (4, 4), "helix_matmul_fp8_t42": (4, 2), "helix_matmul_fp8_t44p": (4, 4),
           "helix_matmul_fp8_t42p": (4, 2)}
COUNTED = 63   # the counter's largest value: an access that would pass it is not issued before the oldest is done


def accesses(code):
    """[(what, argument)] of a kernel's instructions, in order: ("load",) into LDS of a step's rows, ("other",) access,
    ("wait", n), ("barrier",), ("go", index) and ("maybe", index) branches, ("end",), ("",) for all else."""
    ops = []
    for name, rest, target in code:
        if name.startswith("s_branch"):
            ops.append(("go", target))
        elif name.startswith("s_cbranch"):
            ops.append(("maybe", target))
        elif name == "s_barrier":
            ops.append(("barrier",))
        elif name == "s_endpgm":
            ops.append(("end",))
        elif name == "s_waitcnt" and "vmcnt" in rest:
            ops.append(("wait", int(re.search(r"vmcnt\((\d+)\)", rest).group(1))))
        elif re.match(r"(buffer|global|flat|scratch)_(load|store|atomic)", name):
            ops.append(("load",) if name == "buffer_load_dwordx4" and rest.endswith("lds") else ("other",))
        else:
            ops.append(("",))
    return ops


def uncovered(ops, tm, tn):
    """Barriers after which LDS is read that a load may not have reached yet: {(place, loads that are missing)}.

    A path's state is where it is, which of a step's two barriers comes next, the accesses that may be under way (the
    loads among them are the last ones issued) and the loads issued beyond the steps begun; the latter two return to
    what they were, so that loops end."""
    each, first = tm + tn, tm + tn // 2
    seen, found = set(), set()
    todo = [(0, -1, "", 0)]
    while todo:
        pc, turn, queue, issued = todo.pop()
        while True:
            what = ops[pc]
            if what[0] in ("maybe", "barrier"):
                if (pc, turn, queue, issued) in seen:
                    break
                seen.add((pc, turn, queue, issued))
            if what[0] == "end":
                break
            if what[0] == "go":
                pc = what[1]
                continue
            if what[0] == "maybe":
                todo.append((what[1], turn, queue, issued))
            elif what[0] == "load":
                queue, issued = (queue + "l")[-COUNTED:], issued + 1
            elif what[0] == "other":
                queue = (queue + "o")[-COUNTED:]
            elif what[0] == "wait":
                queue = queue[max(0, len(queue) - what[1]):]
            elif what[0] == "barrier":
                # Turn -1, the prologue's barrier: the first step's X and half of Y; 0: the rest of this step's Y;
                # 1: the next step's X and half of Y.
                needed = (first, each, each + first)[turn + 1]
                missing = needed - (issued - queue.count("l"))
                if missing > 0:
                    found.add((pc, missing))
                if turn == 1:
                    issued -= each
                turn = 0 if turn != 0 else 1
                assert abs(issued) < 8 * each, "the path lost count of the steps"
            pc += 1
    return found


def test_a_weak_wait_is_seen():
    # Two steps loaded ahead, then steps of two barriers without end: one load too many allowed under way at any of them.
    tm, tn = 4, 2
    load, barrier = ("load",), ("barrier",)

    def steps(prologue, one, two):
        head = [load] * 12 + [("wait", prologue), barrier]
        return head + [("wait", one), barrier, *[load] * 5, ("wait", two), barrier, load, ("maybe", len(head)), ("end",)]

    assert not uncovered(steps(6, 6, 6), tm, tn) and not uncovered(steps(0, 6, 6), tm, tn)
    assert uncovered(steps(8, 6, 6), tm, tn) and uncovered(steps(6, 7, 6), tm, tn) and uncovered(steps(6, 6, 7), tm, tn)

    # Two stores before a wait that allows for them: right where they were issued, and not on a path past them.
    def stored(*before):
        return [load] * 12 + [("wait", 6), barrier, ("wait", 6), barrier, *before, ("wait", 3), barrier, ("end",)]

    assert not uncovered(stored(("other",), ("other",)), tm, tn)
    assert uncovered(stored(("maybe", 19), ("other",), ("other",)), tm, tn)
    assert uncovered(stored(), tm, tn)


@pytest.fixture(scope="module")
def built():
    return built_code.kernels("|".join(KERNELS))


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_tiles_wait_for_what_they_read(built, name):
    tm, tn = KERNELS[name]
    ops = accesses(built[name])
    assert sum(op[0] == "load" for op in ops) >= 4 * (tm + tn) and sum(op[0] == "barrier" for op in ops) >= 9
    assert uncovered(ops, tm, tn) == set()
