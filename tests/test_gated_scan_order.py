"""The gated recurrence's reads of the state that comes in, followed through the built code on the CPU: the state that
goes out may take its place, so they are done before a chunk is published (kernels/gated_scan.hip, entering). Whether a
late read meets the new state is a matter of timing, which no result shows reliably."""
import re

import pytest

import built_code


def late_reads(code):
    """Places of a workgroup's joining, from a publishing store (eight bytes past the caches) to the next barrier, where a
    plain load of a word begins, or where one may not have come back at the store. Along every branch."""
    seen, found, published = set(), set(), set()
    todo = [(0, "", False)]
    while todo:
        pc, queue, after = todo.pop()
        while True:
            name, rest, target = code[pc]
            if name.startswith("s_cbranch") or name == "s_barrier":
                if (pc, queue, after) in seen:
                    break
                seen.add((pc, queue, after))
            if name == "s_endpgm":
                break
            if name.startswith("s_branch"):
                pc = target
                continue
            if name.startswith("s_cbranch"):
                todo.append((target, queue, after))
            elif name == "s_barrier":
                after = False
            elif name == "s_waitcnt":
                m = re.search(r"vmcnt\((\d+)\)", rest)
                if m:
                    queue = queue[max(0, len(queue) - int(m.group(1))):]
            elif re.match(r"(buffer|global|flat|scratch)_(load|store|atomic)", name):
                plain = name == "global_load_dword" and "sc1" not in rest
                if name == "global_store_dwordx2" and "sc1" in rest:
                    published.add(pc)
                    after = True
                    if "p" in queue:
                        found.add((pc, "under way"))
                elif plain and after:
                    found.add((pc, "begins"))
                queue = (queue + ("p" if plain else "o"))[-63:]
            pc += 1
    assert published
    return found


def test_a_late_read_is_seen():
    read, publish, barrier, end = (("global_load_dword", "v1, v2, s[0:1]", None),
                                   ("global_store_dwordx2", "v0, v[4:5], s[4:5] sc1", None), ("s_barrier", "", None),
                                   ("s_endpgm", "", None))
    wait = ("s_waitcnt", "vmcnt(0)", None)
    assert not late_reads([read, wait, publish, barrier, end]) and not late_reads([publish, barrier, read, end])
    assert late_reads([read, publish, wait, end]) and late_reads([publish, read, end])
    assert late_reads([("s_cbranch_scc0", "", 3), read, wait, publish, ("s_cbranch_scc1", "", 6), read, barrier, end])


@pytest.fixture(scope="module")
def built():
    return built_code.kernels(r"helix_gated_scan_\w+_w[48]")


def test_the_state_is_read_before_a_chunk_is_published(built):
    assert len(built) == 24
    for name, code in built.items():
        assert late_reads(code) == set(), name
