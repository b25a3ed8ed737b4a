"""The matrix instructions that the prompt attention writes as instructions, in the gfx950 code.

The compiler keeps the wait states between the matrix instructions that it makes and their
neighbours, but not for those in inline assembly: an operand that a vector instruction wrote is
read two wait states later at the earliest, and eight passes' results by anything but another matrix
instruction that adds to them eleven states later.  The source places waits where it knows of such
neighbours; this looks for the ones that the compiler put there (moves of operands, spills)."""
import re
import subprocess

import pytest

from inferno_amd.build import COMMON_FLAGS, CSRC, hipcc

OPERAND_STATES, RESULT_STATES = 2, 11


def _registers(text):
    out = set()
    for kind, one in re.findall(r"\b([va])(\d+)\b", text):
        out.add((kind, int(one)))
    for kind, first, last in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        out |= {(kind, i) for i in range(int(first), int(last) + 1)}
    return out


def _functions(asm):
    """{name: [(instruction or label, written by hand), ...]}."""
    out, lines, by_hand = {}, None, False
    for raw in asm.splitlines():
        by_hand = "#ASMSTART" in raw or (by_hand and "#ASMEND" not in raw)
        line = raw.split(";")[0].strip()
        label = re.match(r"^([.\w$]+):$", line)
        if label and label.group(1).startswith("_Z"):
            lines = out.setdefault(label.group(1), [])
        elif lines is not None and line and (label or not line.startswith(".")):
            lines.append((line, by_hand))
        if line.startswith(".Lfunc_end"):
            lines = None
    return out


def _ahead(lines, labels, start, states):
    """The instructions that follow start, on any path, with fewer than `states` between."""
    todo, seen = [(start + 1, 0)], set()
    while todo:
        i, n = todo.pop()
        while i < len(lines) and n < states and (i, n) not in seen:
            seen.add((i, n))
            line, by_hand = lines[i]
            op, _, rest = line.partition(" ")
            i += 1
            if line.endswith(":"):
                continue
            yield op, rest, by_hand
            n += int(rest) + 1 if op == "s_nop" else 1
            if op.startswith("s_cbranch"):
                todo.append((labels[rest.strip()], n))
            elif op == "s_branch":
                i = labels[rest.strip()]
            elif op == "s_endpgm":
                break


def too_close(lines):
    labels = {l[:-1]: i for i, (l, _) in enumerate(lines) if l.endswith(":")}
    found = []
    for i, (line, by_hand) in enumerate(lines):
        op, _, rest = line.partition(" ")
        operands = re.split(r",\s*(?![^\[]*\])", rest)
        if op.startswith("v_mfma"):
            if not by_hand:
                continue
            result = _registers(operands[0])
            for other, args, _ in _ahead(lines, labels, i, RESULT_STATES):
                fields = re.split(r",\s*(?![^\[]*\])", args)
                used = _registers(",".join(fields[1:3])) if other.startswith("v_mfma") else _registers(args)
                if used & result:
                    found.append((line, other + " " + args))
        elif op.startswith("v_") and not op.startswith("v_cmp"):
            written = _registers(operands[0])
            for other, args, hand in _ahead(lines, labels, i, OPERAND_STATES):
                if hand and other.startswith("v_mfma") and written & _registers(",".join(
                        re.split(r",\s*(?![^\[]*\])", args)[1:])):
                    found.append((line, other + " " + args))
    return found


def test_a_near_neighbour_is_found():
    def lines(*text):
        return [(t.lstrip("*"), t.startswith("*")) for t in text]

    product = "*v_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], a[0:15]"
    assert too_close(lines("v_mov_b32_e32 v3, v9", "s_nop 0", product, "s_endpgm"))
    assert not too_close(lines("v_mov_b32_e32 v3, v9", "s_nop 1", product, "s_endpgm"))
    assert too_close(lines(product, "s_nop 9", "v_accvgpr_read_b32 v8, a15", "s_endpgm"))
    assert not too_close(lines(product, "s_nop 10", "v_accvgpr_read_b32 v8, a15", "s_endpgm"))
    assert not too_close(lines(product, product, "s_endpgm"))
    assert too_close(lines("x:", "v_mov_b32_e32 v8, a1", product, "s_cbranch_vccnz x", "s_endpgm"))


def test_prompt_attention(tmp_path):
    out = tmp_path / "window_prefill.s"
    subprocess.run([hipcc(), *COMMON_FLAGS, "--cuda-device-only", "-S", str(CSRC / "window_prefill.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    kernels = {n: l for n, l in _functions(out.read_text()).items()
               if any(hand and t.startswith("v_mfma") for t, hand in l)}
    assert len(kernels) == 9  # three head_dims, three formats
    for name, lines in kernels.items():
        assert not too_close(lines), name
