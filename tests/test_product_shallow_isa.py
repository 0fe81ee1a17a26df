"""product_shallow_kernel sends a tile's first copies into LDS out before the last tile's stores, and then waits with
a count: `s_waitcnt vmcnt(n)` covers the copies only if at least n memory operations were issued behind them. This test
compiles the kernel for gfx950 with the library's own flags and follows every path from those copies to the next
barrier: each has its n stores, and a wait that covers the copies. The walk itself keeps to the same rule, and neither
touches scratch memory.

Runs on the CPU: hipcc cross-compiles; no GPU is used.
"""
import os
import re
import shutil
import subprocess

import pytest

from ae_amd import build as libbuild

STORES = {0: 16, 1: 8, 2: 8}  # of a wave and tile: fp32, fp16, bf16


def _instructions(lines):
    """{function: [instruction, or "label:"]}"""
    out, name = {}, None
    for line in lines:
        line = line.split(";")[0].strip()
        m = re.match(r"^(_Z\w+):", line)
        if m:
            name = m.group(1)
            out[name] = []
        elif name and (re.match(r"^\.LBB\w+:", line) or (line and not line.startswith("."))):
            out[name].append(line)
    return out


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc is not installed")
    path = str(tmp_path_factory.mktemp("isa") / "tile.s")
    cmd = [hipcc, *libbuild.HIPCC_FLAGS, "--cuda-device-only", "-S", os.path.join(libbuild.CSRC, "product_tile.hip"), "-o", path]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    with open(path) as f:
        found = {n: i for n, i in _instructions(f.read().split("\n")).items() if "product_shallow_kernel" in n}
    assert len(found) == 6
    return found


def _next(ins, at, labels):
    """Where control may go behind instruction `at`."""
    op = ins[at]
    if op.startswith("s_endpgm"):
        return []
    if op.startswith("s_cbranch_execz"):
        # without lanes only where the block has turned some off (a block is never entered without any)
        block = next(i for i in range(at, -1, -1) if ins[i].endswith(":") or i == 0)
        if not any("saveexec" in o or re.match(r"(s_\w+_b64 exec|v_cmpx)", o) for o in ins[block:at]):
            return [at + 1]
    m = re.match(r"s_(c?branch)\w*\s+(\.LBB\w+)", op)
    to = [] if m and m.group(1) == "branch" else [at + 1]
    return to + ([labels[m.group(2)]] if m else [])


def _copy(op):
    return op.endswith(" lds")


def _memory(op):
    return re.match(r"(buffer|global|flat|scratch)_(load|store|atomic)", op) is not None


def _to_barriers(ins, start):
    """Over the paths from behind `start` to the next barrier or copy: (least memory operations before each place, the
    barriers that are reached before a wait has covered the copies, the buffer stores and scratch operations met)."""
    labels = {op[:-1]: i for i, op in enumerate(ins) if op.endswith(":")}
    least, todo = {}, [(t, 0) for t in _next(ins, start, labels)]
    uncovered, stores, scratch = set(), set(), set()
    while todo:
        at, count = todo.pop()
        if at >= len(ins) or least.get(at, 1 << 30) <= count:
            continue
        least[at] = count
        op = ins[at]
        if _copy(op):
            continue
        if op.startswith("s_barrier"):
            uncovered.add((at, count))
            continue
        m = re.match(r"s_waitcnt.*vmcnt\((\d+)\)", op)
        if m and int(m.group(1)) <= count:
            continue
        if _memory(op):
            count += 1
            if op.startswith("buffer_store"):
                stores.add(at)
            if op.startswith("scratch"):
                scratch.add(at)
        todo += [(t, count) for t in _next(ins, at, labels)]
    return least, uncovered, stores, scratch


def _groups(ins):
    """The last copies of the runs of copies (between which no barrier, label or branch lies)."""
    last, out = None, []
    for i, op in enumerate(ins):
        if _copy(op):
            last = i
        elif last is not None and (op.startswith(("s_barrier", "s_branch", "s_cbranch")) or op.endswith(":")):
            out.append(last)
            last = None
    return out + ([last] if last is not None else [])


@pytest.mark.parametrize("dtype", STORES)
def test_the_next_tiles_copies_are_waited_for(kernels, dtype):
    (ins,) = (i for n, i in kernels.items() if f"ILi{dtype}ELb1E" in n)
    counts = [int(m.group(1)) for op in ins if (m := re.match(r"s_waitcnt vmcnt\((\d+)\)$", op))]
    assert STORES[dtype] in counts  # the counted wait is there
    checked = 0
    for start in _groups(ins)[1:]:  # (the first tile's copies have no stores behind them: they are waited for alone)
        least, uncovered, stores, scratch = _to_barriers(ins, start)
        if not stores:
            continue
        checked += 1
        # (a tile's first wait is one of two, for the counted copies or, without stores, for everything; each may be
        # skipped for the other: what is left is the path past both, which has all of its stores)
        for at, count in uncovered:
            waits = [int(m.group(1)) for op in ins[at - 12:at] if (m := re.match(r"s_waitcnt vmcnt\((\d+)\)$", op))]
            assert sorted(waits) == [0, STORES[dtype]] and count == STORES[dtype], (start, at, count, waits)
        assert not scratch, [ins[i] for i in scratch]
        # past the caches and through them: as many each
        past = {i for i in stores if re.search(r"\bnt\b", ins[i])}
        assert len(past) == STORES[dtype] and len(stores - past) == STORES[dtype], (start, len(past), len(stores))
    assert checked


@pytest.mark.parametrize("dtype", STORES)
@pytest.mark.parametrize("slots", [0, 1])
def test_the_walk_waits_for_all_copies(kernels, dtype, slots):
    """Between the barrier behind which a step's fragments are read and the copies before it stands vmcnt(0), and no
    scratch memory is used beside the products."""
    (ins,) = (i for n, i in kernels.items() if f"ILi{dtype}ELb{slots}E" in n)
    products = [i for i, op in enumerate(ins) if op.startswith("v_mfma")]
    assert not any(op.startswith("scratch") for op in ins[products[0]:products[-1]])
    for i, op in enumerate(ins):
        if not op.startswith("s_barrier"):
            continue
        behind = next((o for o in ins[i + 1:] if o.startswith(("ds_read", "ds_write", "s_barrier")) or _copy(o)), "")
        if behind.startswith("ds_read") and any(p > i for p in products):
            waits = [int(m.group(1)) for o in ins[max(0, i - 12):i] if (m := re.match(r"s_waitcnt.*vmcnt\((\d+)\)", o))]
            assert 0 in waits, (i, ins[max(0, i - 12):i + 1])


def test_a_dropped_store_would_be_found():
    """The follower itself, on a made-up walk."""
    def walk(n, wait):
        return ["buffer_load_dwordx4 v1, s[0:3], 0 offen lds", "s_cbranch_scc1 .LBB0_2", ".LBB0_1:",
                *["buffer_store_dwordx4 v[0:3], v4, s[0:3], 0 offen nt"] * 8, "s_branch .LBB0_3", ".LBB0_2:",
                *["buffer_store_dwordx4 v[0:3], v4, s[0:3], 0 offen"] * n, ".LBB0_3:", f"s_waitcnt vmcnt({wait})",
                "s_barrier", "s_endpgm"]

    assert not _to_barriers(walk(8, 8), 0)[1]
    assert not _to_barriers(walk(7, 0), 0)[1]
    assert _to_barriers(walk(7, 8), 0)[1]
    assert _to_barriers(walk(8, 9), 0)[1]
