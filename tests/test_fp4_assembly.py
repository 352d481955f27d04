"""What the fp4 kernels' sources and the compiler's assembly of them have to keep, where correctness depends on it."""
import os
import re
import subprocess

import pytest

from kubernetes_amd.native import build as nb

SOURCE = os.path.join(nb.SRC_DIR, "hip", "kamd_mxfp4.hip")


def test_lds_arrays_state_their_alignment():
    """Arrays of bytes in LDS are read and written by words, 8 and 16 bytes: their declarations have to say so, the type
    does not."""
    with open(SOURCE) as f:
        arrays = [line.strip() for line in f if re.search(r"__shared__.*\[.*\];", line)]
    assert len(arrays) >= 4
    for line in arrays:
        m = re.search(r"aligned\((\d+)\)", line)
        assert m and int(m.group(1)) >= 8, line


def overtaken(text):
    """LDS reads from which a way leads to a load into LDS with no wait for the reads between."""
    lines = [line.split(";")[0].strip() for line in text.splitlines()]
    lines = [line for line in lines if re.match(r"\.LBB\S+:$", line) or (line and line[0] not in "._" and not line.endswith(":"))]
    labels = {line[:-1]: i for i, line in enumerate(lines) if line.endswith(":")}
    bad = []
    for i, line in enumerate(lines):
        if not line.startswith("ds_read"):
            continue
        todo, seen = [i + 1], set()
        while todo:
            at = todo.pop()
            if at in seen or at == len(lines):
                continue
            seen.add(at)
            here = lines[at]
            if here.startswith(("global_load_lds", "buffer_load")) and "lds" in here:
                bad.append((i, at))
                break
            if here.startswith("s_endpgm") or (here.startswith("s_waitcnt") and "lgkmcnt(0)" in here):
                continue
            if here.startswith(("s_branch", "s_cbranch")):
                todo.append(labels[here.split()[1]])
            if not here.startswith("s_branch"):
                todo.append(at + 1)
    return bad


LOOP = """
.LBB0_1:
    s_waitcnt lgkmcnt(0)
    global_load_lds_dwordx4 v[4:5], off
    s_waitcnt vmcnt(4)
    ds_read_b128 v[6:9], v45
    v_mfma_x v[6:9], v[50:53]
    s_cbranch_scc1 .LBB0_1
    s_endpgm
"""


def test_the_check_finds_what_it_looks_for():
    assert overtaken(LOOP) == []
    assert overtaken(LOOP.replace("    s_waitcnt lgkmcnt(0)\n", ""))
    assert overtaken(LOOP.replace("lgkmcnt(0)", "lgkmcnt(1)"))
    assert overtaken(LOOP.replace("    s_waitcnt lgkmcnt(0)\n", "").replace("v_mfma_x", "s_waitcnt vmcnt(0) lgkmcnt(0)\n v_mfma_x")) == []


def test_few_rows_load_no_buffer_that_is_being_read(tmp_path):
    """A wave of the product of few rows has two buffers and no barrier: it loads one again once what it read of it has come."""
    if not os.path.exists(nb.HIPCC):
        pytest.skip("no hipcc")
    cmd = [c for c in nb.targets()["kamd_hip"][2] if not c.endswith(".hip") and c not in ("-shared", "-fPIC")]
    out = tmp_path / "mxfp4.s"
    r = subprocess.run(cmd + ["-S", "--cuda-device-only", SOURCE, "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    kernels = re.findall(r"\n(_ZN5mxfp416gemm_rows_kernel\w+):[^\n]*\n(.*?)\.Lfunc_end", out.read_text(), re.S)
    assert len(kernels) == 16
    for name, text in kernels:
        assert text.count("global_load_lds") >= 8, name
        assert overtaken(text) == [], name
