"""The code that the library's own flags give for the int8 product: what the kernels rely
on and no language rule or compiler check holds. Needs hipcc, no GPU.

* The one row of x that a workgroup quantizes lies in dynamic LDS, which begins where
  the static LDS ends, and is read 16 bytes at a time: that end is a multiple of 16.
* Loads to LDS are written as statements, in which the compiler looks for no hazards. A
  memory instruction that reads a scalar register needs five wait states behind a vector
  instruction that wrote it; so none of their scalar operands may come from one closer.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from crosslane_amd import _build

WAIT_STATES = 5


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    if not shutil.which(_build.HIPCC):
        pytest.skip("no hipcc")
    out = str(tmp_path_factory.mktemp("lin8") / "lin8.s")
    subprocess.run([_build.HIPCC, *_build.CFLAGS, "-S", "--cuda-device-only", os.path.join(_build.CSRC, "xl_lin8.hip"), "-o", out],
                   check=True, capture_output=True)
    return open(out).read()


def test_the_quantized_row_is_aligned(code):
    # the type of x is the kernel's fourth template argument; int8 (3) has no such row
    sizes = re.findall(r"\.amdhsa_kernel (\S*lin8_rows_kernelILi\d+ELi\d+ELb[01]ELi([0-3])E\S*)\n\s*\.amdhsa_group_segment_fixed_size (\d+)", code)
    assert sorted(t for _, t, _ in sizes if t != "3") == ["0", "0", "1", "1", "2", "2"]
    for name, kind, size in sizes:
        assert kind == "3" or int(size) % 16 == 0, (name, size)


def scalars(text):
    """The scalar registers that an operand list names."""
    out = {int(n) for n in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        out |= set(range(int(a), int(b) + 1))
    return out


def written_by_vector(line):
    """The scalar registers that a vector instruction writes: its first operand, and a carry's or scale's second."""
    op, _, rest = line.partition(" ")
    if not op.startswith("v_"):
        return set()
    operands = [o.strip() for o in rest.split(",")]
    return scalars(" ".join(operands[:2] if "_co_" in op or "div_scale" in op else operands[:1]))


def too_close(lines):
    """Loads to LDS with a scalar operand that a vector instruction wrote less than WAIT_STATES before, on any
    path within a kernel; and their number. `lines`: one kernel's instructions and labels."""
    labels = {l[:-1]: i for i, l in enumerate(lines) if l.endswith(":")}
    from_ = {}   # label's place -> the branches that go there
    for i, l in enumerate(lines):
        m = re.match(r"s_c?branch\S*\s+(\S+)$", l)
        if m:
            from_.setdefault(labels[m.group(1)], []).append(i)
    bad, loads = [], 0
    for i, l in enumerate(lines):
        if not re.match(r"buffer_load_dwordx4 .*\blds\b", l):
            continue
        loads += 1
        reads, seen, todo = scalars(l), {}, [(i, 0)]
        while todo:
            at, states = todo.pop()
            before = [] if at == 0 or re.match(r"s_branch|s_endpgm|s_setpc", lines[at - 1]) else [at - 1]
            for j in before + from_.get(at, []):
                p = lines[j]
                if written_by_vector(p) & reads:
                    bad.append((p, l, states))
                    continue
                n = states + (0 if p.endswith(":") else int(p.split()[1]) + 1 if p.startswith("s_nop") else 1)
                if n < WAIT_STATES and seen.get(j, WAIT_STATES) > n:
                    seen[j] = n
                    todo.append((j, n))
    return bad, loads


def kernels(code):
    for body in re.findall(r"\n_Z\S*lin8_\w*kernel\S*:[^\n]*\n(.*?)\n\.Lfunc_end", code, re.S):
        lines = [re.split(r"[;#]|//", l)[0].strip() for l in body.split("\n")]
        yield [re.sub(r"\s+", " ", l) for l in lines if l and (l.endswith(":") or not l.startswith("."))]


def test_the_scan_finds_what_it_looks_for():
    load = "buffer_load_dwordx4 v1, s[4:7], s9 offen lds"
    assert too_close(["v_readfirstlane_b32 s9, v0", "s_mov_b32 m0, s2", "s_nop 0", load]) == ([("v_readfirstlane_b32 s9, v0", load, 2)], 1)
    assert too_close(["v_readfirstlane_b32 s6, v0", "s_nop 4", load]) == ([], 1)
    assert len(too_close(["v_readfirstlane_b32 s6, v0", "s_nop 3", load])[0]) == 1
    assert too_close(["v_readfirstlane_b32 s10, v0", "v_add_u32_e32 v2, s9, v2", load]) == ([], 1)
    assert len(too_close([".L:", load, "v_add_co_u32_e64 v2, s[4:5], v0, v1", "s_cbranch_scc1 .L"])[0]) == 1   # round a loop
    assert too_close(["v_cmp_lt_i32_e64 s[4:5], v0, v1", "s_branch .M", ".L:", load, ".M:", "s_endpgm"]) == ([], 1)


def test_loads_to_lds_read_no_scalar_that_a_vector_instruction_just_wrote(code):
    loads = 0
    for lines in kernels(code):
        bad, n = too_close(lines)
        assert not bad, bad[:3]
        loads += n
    assert loads == len(re.findall(r"\n\s*buffer_load_dwordx4 [^\n]*\blds\b", code)) > 1000
