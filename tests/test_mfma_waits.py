"""The attention kernels' assembly leaves the wait states that a vector
instruction needs before it reads a matrix instruction's result, on every path:
across branches the compiler does not always insert them (the kernels do)."""
import importlib.util
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def build_module():
    spec = importlib.util.spec_from_file_location("_ormi_build", ROOT / "ormi_amd" / "_build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def registers(text):
    out = set()
    for m in re.finditer(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        lo, hi = (int(m[2]), int(m[3])) if m[2] else (int(m[4]), int(m[4]))
        out |= {(m[1], i) for i in range(lo, hi + 1)}
    return out


def passes(op):
    return {"32x32x16": 8, "32x32x2": 16}[re.search(r"\d+x\d+x\d+", op)[0]]


def early_reads(function):
    """(matrix instruction, reader, wait states between) that are too close."""
    code, labels = [], {}
    for line in function.splitlines()[1:]:
        line = line.split(";")[0].strip()
        if m := re.match(r"(\.L\w+):", line):
            labels[m[1]] = len(code)
        elif line and not line.startswith((".", "#")):
            code.append(line)
    found = []
    for i, line in enumerate(code):
        if not line.startswith("v_mfma"):
            continue
        result, need = registers(line.split(None, 1)[1].split(",")[0]), passes(line) + 2
        least, todo = {}, [(i + 1, 0)]
        while todo:
            j, waited = todo.pop()
            if j >= len(code) or waited >= need or least.get(j, need) <= waited:
                continue
            least[j] = waited
            op, *rest = code[j].split(None, 1)
            if op == "s_nop":
                todo.append((j + 1, waited + 1 + int(rest[0], 0)))
                continue
            if op == "s_endpgm":
                continue
            if op.startswith(("s_branch", "s_cbranch")):
                todo.append((labels[rest[0]], waited + 1))
                if op == "s_branch":
                    continue
            reads = op.startswith("v_") and not op.startswith("v_mfma") or op.startswith(("ds_", "global_", "scratch_"))
            if reads and rest and registers(rest[0]) & result:
                found.append((line, code[j], waited))
                continue
            todo.append((j + 1, waited + 1))
    return found


def test_finds_an_early_read():
    text = "f:\n\tv_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], v[0:15]\n\ts_cbranch_scc1 .LBB0_1\n\ts_nop 9\n.LBB0_1:\n\tv_add_f32 v30, v3, v3\n"
    assert early_reads(text) == [("v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], v[0:15]", "v_add_f32 v30, v3, v3", 1)]
    assert not early_reads(text.replace("s_cbranch_scc1", "s_nop 15\n\ts_cbranch_scc1"))


@pytest.mark.parametrize("name", ["attention_bf16", "attention_f16", "attention_f32"])
def test_matrix_results_are_waited_for(name, tmp_path):
    b = build_module()
    out = tmp_path / "a.s"
    subprocess.run([b.HIPCC, *b.HIP_FLAGS, f"-I{b.INCLUDE}", f"-I{b.CSRC / 'hip'}", "-S", "--cuda-device-only",
                    str(b.CSRC / "hip" / f"{name}.hip"), "-o", str(out)], check=True, stderr=subprocess.DEVNULL)
    functions = [f.split(".Lfunc_end")[0] for f in re.split(r"\n(?=_ZN\S+:)", out.read_text())[1:]]
    assert sum("v_mfma" in f for f in functions) >= 18
    for f in functions:
        assert not early_reads(f), f.split(":")[0]
