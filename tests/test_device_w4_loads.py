"""The waits of the 4-bit product kernels that load into LDS, in the gfx950 code.

A wave of those kernels loads the next operands into LDS by itself, and at a barrier waits until so many of its newest
memory operations alone are outstanding ("s_waitcnt vmcnt(n)", written out with the barrier).  That n counts what the source
issues behind the operands that the barrier publishes: fewer, and the wait would end before they have landed.  Loads return
in order, so it is enough to count them on every path."""
import re

import pytest

from tests.test_device_barriers import _device_code, _functions

MEMORY = re.compile(r"(global|buffer|flat|scratch)_(load|store|atomic)")


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    asm = _device_code("w4_gemm.hip", tmp_path_factory.mktemp("w4"))
    return asm, _functions(asm)


def _into_lds(line):
    return MEMORY.match(line) and "lds" in line.split()[0] or re.search(r"\blds\b", line) is not None and MEMORY.match(line)


def behind(lines, behind_lds):
    """[(n of the wait, fewest memory operations on a path from the last barrier, or from the last load into LDS behind that, ...)]
    for every hand-written wait but those that no barrier comes before."""
    at = {l[:-1]: i for i, l in enumerate(lines) if l.endswith(":")}
    seen, todo, found = set(), [(0, None)], {}
    while todo:
        i, count = todo.pop()  # count: None before the first barrier
        while i < len(lines) and (i, count) not in seen:
            seen.add((i, count))
            line = lines[i]
            op, _, args = line.partition(" ")
            wait = re.match(r"vmcnt\((\d+)\) lgkmcnt\(0\)$", args) if op == "s_waitcnt" else None
            if wait and i + 1 < len(lines) and lines[i + 1] == "s_barrier":
                if count is not None:
                    n = int(wait.group(1))
                    found[i] = (n, min(count, found.get(i, (n, count))[1]))
            i += 1
            if op == "s_barrier":
                count = 0
            elif count is not None and MEMORY.match(op):
                count = 0 if behind_lds and _into_lds(line) else min(count + 1, 64)
            elif op == "s_branch":
                i = at[args.strip()]
            elif op.startswith("s_cbranch"):
                todo.append((at[args.strip()], count))
            elif op == "s_endpgm":
                break
    return list(found.values())


def test_the_count_sees_a_missing_load():
    loop = [".a:", "s_waitcnt vmcnt(2) lgkmcnt(0)", "s_barrier", "global_load_lds_dwordx4 v[0:1], off", "global_load_dwordx4 v[0:3], v[4:5], off",
            "s_cbranch_scc1 .a", "s_endpgm"]
    assert behind(loop, False) == [(2, 2)]
    assert behind(loop, True) == [(2, 1)]
    loop[4] = "v_mov_b32_e32 v0, v1"
    assert behind(loop, False) == [(2, 1)]


@pytest.mark.parametrize("kernel,count,behind_lds", [("w4_tile_kernel", 24, False), ("w4_batch_kernel", 0, True)])
def test_waits_leave_only_later_loads(code, kernel, count, behind_lds):
    kernels = {n: l for n, l in code[1].items() if kernel in n}
    assert len(kernels) >= max(count, 6)
    for name, lines in kernels.items():
        waits = behind(lines, behind_lds)
        assert waits, name
        for n, fewest in waits:
            assert n <= fewest, (name, n, fewest)


def test_first_barrier_of_the_tiles(code):
    """Ahead of the loop: stage 0's loads into LDS, then stage 1's; what the first wait leaves outstanding is stage 1's."""
    for name, lines in code[1].items():
        if "w4_tile_kernel" not in name:
            continue
        first = next(i for i, l in enumerate(lines) if l == "s_barrier")
        n = int(re.match(r"s_waitcnt vmcnt\((\d+)\) lgkmcnt\(0\)", lines[first - 1]).group(1))
        ops = [l for l in lines[:first] if MEMORY.match(l)]
        into = [i for i, l in enumerate(ops) if _into_lds(l)]
        stage = len(into) // 2  # of each half
        assert len(into) % 2 == 0 and stage >= 3
        assert len(ops) - n > into[stage - 1], name


def test_first_barrier_of_the_batches(code):
    for name, lines in code[1].items():
        if "w4_batch_kernel" not in name:
            continue
        first = next(i for i, l in enumerate(lines) if l == "s_barrier")
        n = int(re.match(r"s_waitcnt vmcnt\((\d+)\) lgkmcnt\(0\)", lines[first - 1]).group(1))
        ops = [l for l in lines[:first] if MEMORY.match(l)]
        last = max(i for i, l in enumerate(ops) if _into_lds(l))
        assert len(ops) - n > last, name


def test_operands_stay_in_registers(code):
    sizes = re.findall(r"\.amdhsa_kernel (\S+).*?\.amdhsa_private_segment_fixed_size (\d+)", code[0], re.S)
    assert sizes and all(int(n) == 0 for _, n in sizes), [k for k, n in sizes if int(n)]
