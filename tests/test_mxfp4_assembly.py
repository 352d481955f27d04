"""The large fp4 product issues its matrix instructions from inline assembly, which the compiler's own hazard
recogniser does not look into. Two rules of the hardware are checked in the assembly that the build's flags give:
  * an ordinary vector instruction's write of a register and a matrix instruction's read of it are 2 wait states
    apart (every instruction is one, `s_nop N` is N + 1);
  * a matrix instruction's sum is read by an ordinary instruction, a store or an LDS write 18 wait states later at
    the earliest.
"""
import os
import re
import subprocess

import pytest

from kubernetes_amd.native import build as nb


def _regs(op):
    """Registers of an operand: v12, v[10:13], a[0:3]."""
    m = re.fullmatch(r"([va])(\d+)", op) or re.fullmatch(r"([va])\[(\d+):(\d+)\]", op)
    if not m:
        return set()
    first, last = int(m.group(2)), int(m.group(m.lastindex))
    return {(m.group(1), i) for i in range(first, last + 1)}


def _is_valu(op):
    return op.startswith("v_") and not op.startswith("v_mfma")


def hazards(instructions):
    """Places where a rule is broken, on any path into them."""
    labels = {name: i for i, (op, name) in enumerate(instructions) if op is None}
    into = {}
    for i, (op, args) in enumerate(instructions):
        if op and (op.startswith("s_cbranch") or op == "s_branch"):
            into.setdefault(labels[_target[i]], []).append(i)

    def before(i, states):
        """(instruction, wait states between it and i) of those at most `states` away, on every path."""
        todo, seen = [(i, 0)], set()
        while todo:
            at, gone = todo.pop()
            if gone >= states or (at, gone) in seen:
                continue
            seen.add((at, gone))
            here = instructions[at]
            back = []
            if here[0] is None:
                back += into.get(at, [])
            if at > 0 and instructions[at - 1][0] not in ("s_branch", "s_endpgm"):
                back.append(at - 1)
            for b in back:
                op, args = instructions[b]
                if op is None:
                    todo.append((b, gone))
                    continue
                yield b, gone
                todo.append((b, gone + (int(args[0]) + 1 if op == "s_nop" else 1)))

    bad = []
    for i, (op, args) in enumerate(instructions):
        if op is None:
            continue
        if op.startswith("v_mfma"):
            reads = set().union(*(_regs(a) for a in args[1:6]))
            for b, _ in before(i, 2):
                wop, wargs = instructions[b]
                if wop and _is_valu(wop) and wargs and _regs(wargs[0]) & reads:
                    bad.append(f"{wop} {wargs} .. {op} {args}")
        elif _is_valu(op) or op.startswith(("global_store", "ds_write", "buffer_store", "scratch_store")):
            reads = set().union(set(), *(_regs(a) for a in (args[1:] if _is_valu(op) else args)))
            if not reads:
                continue
            for b, _ in before(i, 18):
                wop, wargs = instructions[b]
                if wop and wop.startswith("v_mfma") and _regs(wargs[0]) & reads:
                    bad.append(f"{wop} {wargs} .. {op} {args}")
    return bad


_target = {}


def _load(text, symbol):
    """As _instructions, with the branches' targets remembered by place."""
    _target.clear()
    out = []
    body = text[text.index("\n" + symbol):]
    body = body[:body.index(".Lfunc_end")]
    for line in body.splitlines()[2:]:
        line = line.split(";")[0].strip()
        m = re.fullmatch(r"(\.LBB\S+):", line)
        if m:
            out.append((None, m.group(1)))
        elif line and not line.startswith("."):
            op, rest = (line.split(None, 1) + [""])[:2]
            if op.startswith("s_cbranch") or op == "s_branch":
                _target[len(out)] = rest.strip()
            out.append((op, re.findall(r"\b[va]\[\d+:\d+\]|\b[va]\d+\b|\b\d+\b", rest)))
    return out


CLEAN = """
f:
f_begin:
    v_mov_b32_e32 v1, v2
    s_nop 1
    v_mfma_x a[0:3], v[0:3], v[4:7], a[0:3], v8, v9
    s_nop 15
    s_nop 1
    v_accvgpr_read_b32 v10, a0
.Lfunc_end0:
"""


def test_the_check_finds_what_it_looks_for():
    assert hazards(_load(CLEAN, "f:")) == []
    assert hazards(_load(CLEAN.replace("s_nop 1\n    v_mfma", "s_nop 0\n    v_mfma"), "f:"))
    assert hazards(_load(CLEAN.replace("s_nop 15\n", "s_nop 8\n"), "f:"))
    loop = CLEAN.replace("    v_mov_b32_e32 v1, v2\n    s_nop 1\n", "    s_nop 1\n.LBB0_1:\n").replace(
        "    s_nop 15\n", "    v_mov_b32_e32 v9, v2\n    s_cbranch_scc1 .LBB0_1\n    s_nop 15\n")
    assert hazards(_load(loop, "f:"))          # over the back edge: one wait state, the branch
    assert hazards(_load(loop.replace("v_mov_b32_e32 v9", "v_mov_b32_e32 v20"), "f:")) == []


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    if not os.path.exists(nb.HIPCC):
        pytest.skip("no hipcc")
    cmd = [c for c in nb.targets()["kamd_hip"][2] if not c.endswith(".hip") and c not in ("-shared", "-fPIC")]
    out = str(tmp_path_factory.mktemp("asm") / "mxfp4.s")
    src = os.path.join(nb.SRC_DIR, "hip", "kamd_mxfp4.hip")
    r = subprocess.run(cmd + ["-S", "--cuda-device-only", src, "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    with open(out) as f:
        return f.read()


@pytest.mark.parametrize("kernel", ["_ZN5mxfp417gemm_large_kernelIfEE", "_ZN5mxfp417gemm_large_kernelIDF16bEE"])
def test_large_product_keeps_its_distances(assembly, kernel):
    instructions = _load(assembly, kernel)
    products = [a for op, a in instructions if op and op.startswith("v_mfma")]
    assert len(products) >= 4 * 128                                  # 2 tiles in the loop, 2 behind it
    assert all(a[0] == a[3] and a[0].startswith("a[") for a in products)   # in place
    assert not [op for op, _ in instructions if op and op.startswith("scratch_")]   # no register in memory
    assert hazards(instructions) == []


def test_no_packed_fp32(assembly):
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", assembly)
