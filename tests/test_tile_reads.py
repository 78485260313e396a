"""The reads of the products with packed weights stay in the tensor.  Followed on the host through the kernels' own address
arithmetic (tests/native/tile_reads.hip, compiled for the host alone): every 16-byte piece of every lane, for all block types,
rows of 8 to 4104 16-bit floats or 1 to 72 blocks, one row to some tiles of them, and waves that have no tile."""
import os
import shutil
import subprocess

import pytest

HIPCC = "/opt/rocm/bin/hipcc"
SRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "tile_reads.hip")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and shutil.which("hipcc") is None, reason="needs hipcc")


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("tiles") / "tile_reads")
    subprocess.check_call([HIPCC if os.path.exists(HIPCC) else "hipcc", "--offload-arch=gfx950", "--cuda-host-only", "-O2", "-std=c++17", "-o", exe, SRC])
    return exe


def run(exe, *args):
    out = subprocess.run([exe, *args], capture_output=True, text=True, check=True, timeout=600).stdout
    return {(n, k): (int(bad), int(of)) for n, k, bad, of in (line.split() for line in out.splitlines())}


def test_every_piece_lies_in_the_tensor(checker):
    got = run(checker)
    assert len(got) == 32 and all(of > 0 for _, of in got.values())
    assert {k: bad for k, (bad, _) in got.items() if bad} == {}


def test_the_check_can_fail(checker):
    """Where a row's last turn holds less than a piece, an end that wraps round is seen: float rows only."""
    got = run(checker, "plant")
    assert {k for k, (bad, _) in got.items() if bad} == {(n, k) for n in ("f16", "bf16") for k in ("one", "several")}
