"""The generated gfx950 code of the products with packed weights (matmul_type.hip, matmul.hip): no packed-f32 arithmetic, no scratch
memory.  CPU only: hipcc cross-compiles."""
import os
import re
import shutil
import subprocess

import pytest

import isa_checks as c

pytestmark = pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"),
                                reason="needs make and hipcc")


@pytest.mark.parametrize("ty", ["Q4K", "Q6K", "Q8_0", "IQ4NL", "WF16"])
def test_no_packed_f32_and_no_scratch(tmp_path, ty):
    out = str(tmp_path / "matmul.s")
    r = subprocess.run(["make", "-s", "-C", c.CSRC, "asm_matmul", f"ASM_TYPE={ty}", f"ASM_OUT={out}", "EXTRA=-Rpass-analysis=kernel-resource-usage"],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    funcs = c.functions(open(out).read())
    names = c.demangle(sorted(funcs))
    for kernel in ("matvec_dense", "moe_up_dense", "moe_down_dense", "get_rows"):
        assert any(kernel in n for n in names.values())
    packed = [(names[n], i) for n, body in funcs.items() for i in body if re.match(r"v_pk_(add|mul|fma)_f32\b", i)]
    assert packed == []
    scratch = re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", r.stderr)
    assert len(scratch) >= 20 and set(scratch) == {"0"}
