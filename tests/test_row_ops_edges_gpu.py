"""rmsnorm_quant and silu_mul_quant at the ends of fp32 and of what the arguments allow."""

import pytest
import torch

from flydsl_b200 import silu_mul_quant
from tests.test_row_ops_gpu import FP8, SILU_REL, TYPES, check, make, silu64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vectors", [1025, 1536, 1537, 2048, 2552, 2561, 3067, 3100, 3584, 3585, 4096])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("quant", [FP8, torch.int8], ids=["fp8", "int8"])
def test_many_wide_gated_rows_of_every_type(vectors, dtype, quant):
    """Three to eight vectors of a row per thread, in every type; chunks that end inside; more rows than SMs, in strides."""
    inter = vectors * (16 // dtype.itemsize)
    x = make(301, 2 * inter + 16, dtype, vectors)[:, : 2 * inter]
    x[5] = 0.0
    y, s = silu_mul_quant(x, quant_dtype=quant)
    check(y, s, silu64(x), quant, SILU_REL)
    for i in (0, 5, 300):
        ys, ss = silu_mul_quant(x[i : i + 1], quant_dtype=quant)  # one row takes the other kernel
        assert torch.equal(y[i : i + 1].view(torch.uint8), ys.view(torch.uint8)) and torch.equal(s[i : i + 1], ss)
