"""Products with packed weights on the GPU, at the ends of their ranges: rows that end a few elements into a turn, one token's
activations of every size, codes that are small beside their range, non-finite values, and long lists of ids."""
import numpy as np
import pytest

import matmul_ref as ref
from test_gpu_matmul import Moe, activations, dtype, on_device, output, run_matvec, untouched, weights
from util import same_bits

pytestmark = pytest.mark.gpu


# ---- rows whose last turn is shorter than 16 bytes (tests/test_tile_reads.py follows the addresses on the CPU) ----------------

@pytest.mark.parametrize("ty", [1, 30])
@pytest.mark.parametrize("rows,cols,tokens", [(5, 1025, 1), (8, 1031, 1), (9, 2049, 1), (1, 1026, 1), (33, 3078, 1), (1, 257, 2), (1, 263, 16), (1, 513, 3),
                                              (17, 257, 2), (2, 2055, 7)])
def test_rows_that_end_a_few_elements_into_a_turn(oracle, ty, rows, cols, tokens):
    for xk in ("f32", "bf16"):
        run_matvec(oracle, ty, rows, cols, tokens, xk, "f32", rows + cols)


@pytest.mark.parametrize("ty", [1, 30])
@pytest.mark.parametrize("tokens", [1, 3])
def test_moe_rows_that_end_a_few_elements_into_a_turn(oracle, ty, tokens):
    for hidden, ff in ((257, 1), (259, 9), (1, 513), (9, 262)):
        m = Moe(oracle, 3, hidden, ff, ty, ty, seed=hidden + tokens)
        x, _ = activations(tokens, hidden, "f32", tokens)
        m.check(x, "f32", pad=1)
