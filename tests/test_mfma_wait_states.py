"""How many wait states lie between a matrix instruction and a vector instruction
that reads its result: what the installed compiler inserts in straight-line code
of each kind, which the attention kernels' assembly has to keep on every path
(the scan is test_mfma_waits.py's, with these counts)."""
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

import test_mfma_waits as scan

KINDS = {"bf16": ("__bf16", 8, "32x32x16_bf16"), "f16": ("_Float16", 8, "32x32x16_f16"), "f32": ("float", 1, "32x32x2f32")}
STATES = {"bf16": 12, "f16": 12, "f32": 18}


def assembly(source, out):
    b = scan.build_module()
    subprocess.run([b.HIPCC, *b.HIP_FLAGS, f"-I{b.INCLUDE}", f"-I{b.CSRC / 'hip'}", "-S", "--cuda-device-only", str(source), "-o", str(out)],
                   check=True, stderr=subprocess.DEVNULL)
    return out.read_text()


def need(op):
    return STATES["f32" if "x2_f32" in op else "bf16"]


def early(function, monkeypatch):
    monkeypatch.setattr(scan, "passes", lambda op: need(op) - 2)  # the scan adds two
    return scan.early_reads(function)


@pytest.mark.parametrize("kind", list(KINDS))
def test_what_the_compiler_waits(kind, tmp_path):
    elem, n, name = KINDS[kind]
    vec = f"typedef {elem} v __attribute__((ext_vector_type({n})));" if n > 1 else f"typedef {elem} v;"
    src = tmp_path / "k.hip"
    src.write_text("#include <hip/hip_runtime.h>\ntypedef float acc __attribute__((ext_vector_type(16)));\n" + vec + f"""
__global__ void k(const v* a, const v* b, acc* c) {{
    acc x = {{0}};
    x = __builtin_amdgcn_mfma_f32_{name}(a[threadIdx.x], b[threadIdx.x], x, 0, 0, 0);
    for (int i = 0; i < 16; ++i) x[i] = x[i] * 2.5f + 1.0f;
    c[threadIdx.x] = x;
}}
""")
    after = assembly(src, tmp_path / "k.s").split("v_mfma", 1)[1].splitlines()[1:]
    waited = 0
    for line in after:
        m = re.match(r"\s*s_nop (\d+)", line)
        if not m:
            break
        waited += int(m[1]) + 1
    assert waited == STATES[kind]


@pytest.mark.parametrize("waits,enough", [("s_nop 9", False), ("s_nop 10", False), ("s_nop 11", True), ("s_nop 9\n\ts_nop 1", True)])
def test_the_scan_counts_16_bit_products(waits, enough, monkeypatch):
    mfma = "v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], v[0:15]"
    found = early(f"f:\n\t{mfma}\n\t{waits}\n\tv_add_f32 v30, v3, v3\n", monkeypatch)
    assert [] == found if enough else [(mfma, "v_add_f32 v30, v3, v3")] == [f[:2] for f in found]


@pytest.mark.parametrize("waits,enough", [("s_nop 15\n\ts_nop 0", False), ("s_nop 15\n\ts_nop 1", True)])
def test_the_scan_counts_32_bit_products(waits, enough, monkeypatch):
    text = f"f:\n\tv_mfma_f32_32x32x2_f32 v[0:15], v16, v20, v[0:15]\n\t{waits}\n\tv_add_f32 v30, v3, v3\n"
    assert (not early(text, monkeypatch)) == enough


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_the_kernels_wait_by_themselves(kind, tmp_path):
    """settle() alone waits long enough, whatever the compiler adds."""
    traits = {"bf16": "TrBF16", "f16": "TrF16", "f32": "TrF32"}[kind]
    src = tmp_path / "k.hip"
    src.write_text(f"""#include "attention_kernels.h"
__global__ void k(ormi_hip::f32x16_t* c) {{
    ormi_hip::f32x16_t x = c[threadIdx.x];
    ormi_hip::settle<ormi_hip::{traits}>(x);
    c[threadIdx.x] = x;
}}
""")
    inside = assembly(src, tmp_path / "k.s").split(";;#ASMSTART", 1)[1].split(";;#ASMEND", 1)[0]
    assert sum(int(n) + 1 for n in re.findall(r"s_nop (\d+)", inside)) == STATES[kind]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """The attention sources' assembly by name, compiled side by side."""
    names, out = ["attention_bf16", "attention_f16", "attention_f32"], tmp_path_factory.mktemp("asm")
    hip = scan.build_module().CSRC / "hip"
    with ThreadPoolExecutor(len(names)) as pool:
        return dict(zip(names, pool.map(lambda n: assembly(hip / f"{n}.hip", out / f"{n}.s"), names)))


@pytest.mark.parametrize("name", ["attention_bf16", "attention_f16", "attention_f32"])
def test_the_kernels_wait_on_every_path(name, kernels, monkeypatch):
    functions = [f.split(".Lfunc_end")[0] for f in re.split(r"\n(?=_ZN\S+:)", kernels[name])[1:]]
    assert sum("v_mfma" in f for f in functions) >= 18
    for f in functions:
        assert not early(f, monkeypatch), f.split(":")[0]
