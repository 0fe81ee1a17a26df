"""The product kernels fill LDS stages by copies (buffer loads with `lds`) and hand them to the other waves with a
plain workgroup barrier behind a counted `s_waitcnt vmcnt(n)`. This test compiles them for gfx950 with the
library's own flags and checks the compiled walks (loops of MFMAs):

  - wide tiles: each of a pair of steps has one barrier, right behind a wait for all copies;
  - copied tiles: each step has two barriers, the first behind a wait that leaves at most the next step's copies
    under way, and all of a step's copies are issued behind its second barrier;
  - rows tiles: no barrier at all (a wave reads only what it copied), and a wait for the step's copies before its reads;
  - none of them touches scratch memory.

Runs on the CPU: hipcc cross-compiles; no GPU is used.
"""
import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from ae_amd import build as libbuild

SOURCES = ("product_wide.hip", "product_tile.hip", "product_rows.hip")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc is not installed")
    out = tmp_path_factory.mktemp("isa")

    def compile_one(src):
        path = str(out / (src + ".s"))
        cmd = [hipcc, *libbuild.HIPCC_FLAGS, "--cuda-device-only", "-S", os.path.join(libbuild.CSRC, src), "-o", path]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        assert proc.returncode == 0, proc.stderr
        with open(path) as f:
            return f.read().split("\n")

    with ThreadPoolExecutor(3) as ex:
        return dict(zip(SOURCES, ex.map(compile_one, SOURCES)))


def _walks(lines, kernel):
    """(function, instructions) of the innermost loops with MFMAs and copies in functions of that name."""
    name, start, found = None, {}, []
    for i, line in enumerate(lines):
        m = re.match(r"^(_Z\w+):", line)
        if m:
            name, start, found = m.group(1), {}, []
        m = re.match(r"^(\.LBB\w+):", line)
        if m:
            start[m.group(1)] = i
        m = re.search(r"s_c?branch\w*\s+(\.LBB\w+)", line)
        if not m or m.group(1) not in start or kernel not in (name or ""):
            continue
        first = start[m.group(1)]
        if any(first <= f for f in found):
            continue  # it holds another one
        body = lines[first + 1:i]
        ins = [b.split(";")[0].strip() for b in body]
        ins = [b for b in ins if b and not b.startswith(".")]  # (no labels: a walk may have branches inside)
        if any("v_mfma" in b for b in ins) and any(b.endswith(" lds") for b in ins):
            found.append(first)
            yield name, ins


def _events(ins):
    for b in ins:
        if b.startswith("s_barrier"):
            yield "B"
        elif b.endswith(" lds"):
            yield "C"
        elif b.startswith("ds_read"):
            yield "R"
        elif "v_mfma" in b:
            yield "M"
        elif b.startswith("s_waitcnt"):
            m = re.search(r"vmcnt\((\d+)\)", b)
            if m:
                yield int(m.group(1))
        assert not b.startswith("scratch_"), b


def test_wide_walk(asm):
    walks = list(_walks(asm["product_wide.hip"], "product_wide_kernel"))
    assert len(walks) >= 2 * (4 + 4 + 1)  # types; row tiles 2, 4, 6, 8 of the forward and input gradients; weight gradient
    for name, ins in walks:
        ev = [e for e in _events(ins) if e in ("B",) or isinstance(e, int)]
        assert ev.count("B") == 2, name
        for i, e in enumerate(ev):
            if e == "B":
                assert i > 0 and ev[i - 1] == 0, (name, ev)


def test_copied_walk(asm):
    walks = list(_walks(asm["product_tile.hip"], "product_copied_kernel"))
    seen = 0
    for name, ins in walks:
        bm, bn = map(int, re.search(r"ILi\dELi(\d+)ELi(\d+)E", name).groups())
        copies = (bm + bn) // 32
        ev = [e for e in _events(ins) if e in ("B", "C") or isinstance(e, int)]
        if "B" not in ev:
            continue
        seen += 1
        # rotate to the first wait; then per step: wait, barrier, barrier, copies
        steps = ev.count("B") // 2
        assert ev.count("B") == 2 * steps and steps == 2, name
        want = [copies, "B", "B"] + ["C"] * copies
        assert ev == want * steps, (name, ev)
    assert seen >= 3 * 3


def test_rows_walk(asm):
    walks = list(_walks(asm["product_rows.hip"], "product_rows_kernel"))
    assert len(walks) >= 3 * 5
    for name, ins in walks:
        np_, nj, stages = map(int, re.search(r"ILi\dELi(\d+)ELi(\d+)ELi(\d+)E", name).groups())
        copies = 2 * (np_ + nj)
        ev = list(_events(ins))
        assert "B" not in ev, name
        waits = [i for i, e in enumerate(ev) if isinstance(e, int)]
        assert len(waits) == stages and all(ev[i] == (stages - 1) * copies for i in waits), (name, ev)
        for i, w in enumerate(waits):  # the step's reads, then the copies that reuse its stage
            part = ev[w + 1:waits[i + 1] if i + 1 < len(waits) else len(ev)]
            assert part.count("C") == copies and part.count("R") == 2 * (np_ + nj), (name, part)
            assert max(j for j, e in enumerate(part) if e == "R") < min(j for j, e in enumerate(part) if e == "C"), name
