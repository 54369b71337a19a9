"""A barrier hands what a wave stored to LDS to the workgroup's other waves only if the wave's LDS instructions are
done: on this chip a barrier waits for waves, not for their memory. The compiler puts that wait (lgkmcnt) before
__syncthreads() and takes it out again where it finds nothing outstanding, and round a loop it has done so
where the path into the loop has nothing outstanding and the path round it has. So the built
code is walked: on every path, loops' back edges included, no LDS instruction may be outstanding at a barrier.
Needs the ROCm tools, no GPU."""
from __future__ import annotations

import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from crosslane_amd import _build

TOOLS = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(shutil.which(_build.HIPCC) or _build.HIPCC))), "llvm", "bin")
MANY = 64   # LDS instructions behind one, as far as they are counted (lgkmcnt counts to 15)


def outstanding(lines):
    """For each barrier of one kernel (its instructions, and labels that end in a colon): whether an LDS store, and whether an
    LDS load, may be outstanding there. LDS instructions end in order, so one is done once a wait leaves no more
    outstanding than were issued behind it; scalar loads in the same counter make that a wait for more, not for less."""
    labels = {l[:-1]: i for i, l in enumerate(lines) if l.endswith(":")}
    # of the last store and the last load: how many LDS instructions at least came behind it (None: done)
    state, todo, found = {0: (None, None)}, [0], {}
    while todo:
        i = todo.pop()
        if i >= len(lines):
            continue
        last, line = list(state[i]), lines[i]
        op = line.split()[0]
        after = [i + 1]
        if re.match(r"(ds|flat)_", op) and not re.match(r"ds_(bpermute|permute|swizzle|nop)", op):
            last = [None if n is None else min(n + 1, MANY) for n in last]
            last[1 if re.match(r"(ds|flat)_(read|load)", op) else 0] = 0
        elif op == "s_waitcnt":
            m = re.search(r"lgkmcnt\((\d+)\)", line)
            if m:
                last = [None if n is not None and n >= int(m.group(1)) else n for n in last]
        elif op == "s_barrier":
            found[i] = tuple(n is not None for n in last)
        elif op == "s_branch":
            after = [labels[line.split()[1]]]
        elif op.startswith("s_cbranch"):
            after.append(labels[line.split()[1]])
        elif op == "s_endpgm":
            after = []
        else:
            assert not re.match(r"s_(setpc|swappc|call|rfe)", op), line
        for j in after:
            old = state.get(j)
            new = tuple(last) if old is None else tuple(b if a is None else a if b is None else min(a, b) for a, b in zip(old, last))
            if new != old:
                state[j] = new
                todo.append(j)
    return [found[i] for i in sorted(found)]


def test_the_walk_finds_what_it_looks_for():
    wait, barrier = "s_waitcnt lgkmcnt(0)", "s_barrier"
    assert outstanding(["ds_write_b64 v0, v1", barrier]) == [(True, False)]
    assert outstanding(["ds_write_b64 v0, v1", wait, barrier]) == [(False, False)]
    assert outstanding(["ds_read_b128 v[0:3], v4", barrier]) == [(False, True)]
    assert outstanding(["ds_write_b64 v0, v1", "s_waitcnt vmcnt(0)", barrier]) == [(True, False)]
    # a wait that leaves one outstanding covers all but the last
    assert outstanding(["ds_write_b64 v0, v1", "ds_read_b32 v2, v3", "s_waitcnt vmcnt(3) lgkmcnt(1)", barrier]) == [(False, True)]
    assert outstanding(["ds_write_b64 v0, v1", "s_waitcnt lgkmcnt(1)", barrier]) == [(True, False)]
    # round a loop: nothing outstanding on the way in
    loop = ["L0:", barrier, "ds_read_b32 v2, v3", wait, "ds_write_b32 v0, v1", "s_cbranch_scc1 L0", "s_endpgm"]
    assert outstanding(loop) == [(True, False)]
    assert outstanding(loop[:1] + [wait] + loop[1:]) == [(False, False)]
    # one of two ways to a barrier
    assert outstanding(["s_cbranch_execz L1", "ds_write_b32 v0, v1", "s_branch L2", "L1:", wait, "L2:", barrier]) == [(True, False)]


SOURCES = [s for s in _build.SOURCES if s.endswith(".hip")]


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    """Each source's object: the library's, or, where that is older than the source, a new one."""
    if not os.path.exists(os.path.join(TOOLS, "llvm-objdump")) or not shutil.which(_build.HIPCC):
        pytest.skip("no ROCm tools")
    tmp = tmp_path_factory.mktemp("objects")

    def of(src):
        obj = os.path.join(_build.OBJDIR, src.replace(".hip", ".o"))
        inputs = [os.path.join(_build.CSRC, f) for f in (src, *_build.HEADERS)]
        if not os.path.exists(obj) or os.path.getmtime(obj) < max(map(os.path.getmtime, inputs)):
            obj = str(tmp / os.path.basename(obj))
            subprocess.run([_build.HIPCC, *_build.CFLAGS, "-w", "-c", inputs[0], "-o", obj], check=True, capture_output=True)
        return obj

    with ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        return dict(zip(SOURCES, pool.map(of, SOURCES)))


def kernels(obj, tmp):
    """Names and instructions of an object's kernels."""
    run = lambda tool, *args: subprocess.run([os.path.join(TOOLS, tool), *map(str, args)], check=True, capture_output=True, text=True)  # noqa: E731
    run("llvm-objcopy", f"--dump-section=.hip_fatbin={tmp / 'fat'}", obj, tmp / "copy.o")
    run("clang-offload-bundler", "--unbundle", "--type=o", f"--input={tmp / 'fat'}", f"--targets=hipv4-amdgcn-amd-amdhsa--{_build.ARCH}",
        f"--output={tmp / 'code'}")
    name, lines = None, []
    for line in run("llvm-objdump", "-d", "--no-show-raw-insn", "--symbolize-operands", tmp / "code").stdout.split("\n"):
        m = re.match(r"([0-9a-f]+) <(\w+)>:$", line)
        if m and not re.match(r"L\d+$", m.group(2)):
            if name:
                yield name, with_far_branches(lines)
            name, lines = m.group(2), []
        elif m:
            lines.append((int(m.group(1), 16), m.group(2) + ":"))
        elif line.startswith("\t") and "//" in line:   # (padding behind a kernel has no address)
            text, _, at = line.partition("//")
            lines.append((int(at.split(":")[0], 16), text.strip()))
    if name:
        yield name, with_far_branches(lines)


def with_far_branches(lines):
    """(address, instruction or label) as instructions and labels; a branch past what s_branch reaches (the program counter
    plus a constant) as an s_branch."""
    out, targets = [], {}
    for i, (at, text) in enumerate(lines):
        if text.startswith("s_setpc_b64"):
            get, low, high = (t for _, t in lines[i - 3:i])
            assert get.split()[0] == "s_getpc_b64" and low.split()[0] == "s_add_u32" and high.split()[0] == "s_addc_u32", (get, low, high)
            step = (int(low.split()[-1], 0) & 0xffffffff) + (int(high.split()[-1], 0) << 32)
            target = lines[i - 3][0] + 4 + step
            targets[target] = text = f"s_branch J{target:x}"
        out.append((at, text))
    assert set(targets) <= {at for at, _ in out}
    done = set()
    for i, (at, text) in enumerate(out):
        if at in targets and at not in done:
            done.add(at)
            yield f"J{at:x}:"
        yield text


@pytest.mark.parametrize("src", SOURCES)
def test_no_barrier_with_lds_outstanding(src, objects, tmp_path):
    barriers, bad = 0, []
    for name, lines in kernels(objects[src], tmp_path):
        found = outstanding(list(lines))
        barriers += len(found)
        bad += [name] * sum(any(f) for f in found)
    # (counted in the text too: none was lost on the way)
    text = re.sub(r"//[^\n]*", "", open(os.path.join(_build.CSRC, src)).read())
    assert barriers >= len(re.findall(r"__syncthreads\(\)|s_barrier", text)) and not bad, bad
