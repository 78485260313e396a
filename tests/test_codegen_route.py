"""The generated gfx950 code of the products' kernels that are the same for all block types (matmul.hip): in what `make asm_matmul`
writes, without packed-f32 arithmetic or scratch memory.  CPU only: hipcc cross-compiles."""
import os
import re
import shutil
import subprocess

import pytest

import isa_checks as c

pytestmark = pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"),
                                reason="needs make and hipcc")


def test_kernels_of_no_block_type(tmp_path):
    out = str(tmp_path / "matmul.s")
    r = subprocess.run(["make", "-s", "-C", c.CSRC, "asm_matmul", "ASM_TYPE=Q8_0", f"ASM_OUT={out}", "EXTRA=-Rpass-analysis=kernel-resource-usage"],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    funcs = c.functions(open(out).read())
    names = c.demangle(sorted(funcs))
    for kernel in ("moe_logits<1", "moe_logits<4", "moe_route", "moe_sum", "fill_zero", "matvec_tiles"):
        mine = [n for n, full in names.items() if kernel in full]
        assert mine, kernel
        assert not [i for n in mine for i in funcs[n] if re.match(r"v_pk_(add|mul|fma)_f32\b", i)]
    of = dict(re.findall(r"Function Name: (\S+)(?:.|\n)*?ScratchSize \[bytes/lane\]: (\d+)", r.stderr))
    assert {n for n in of if "moe_route" in n or "fill_zero" in n} and set(of.values()) == {"0"}
