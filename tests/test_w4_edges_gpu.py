"""The products on 4-bit weights at the ends of what their types and arguments allow."""

import pytest
import torch

from flydsl_b200 import compile_w4a16_gemv
from tests.test_w4_gemv_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 4, 5, 40])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("size,scale", [(2.0**-90, 2.0**118), (2.0**-90, 2.0**126), (2.0**-110, 2.0**90), (2.0**-118, 2.0**100), (2.0**-124, 2.0**110)])
def test_scales_and_activations_at_opposite_ends(m, group, size, scale):
    """Products in range of large scales and small activations; bf16 as the range of fp16 has neither."""
    a, q, s, z, _ = make(m, 64, 512, group, "bf16", True, 11)
    x = ((1.0 + a.float().abs().clamp(max=0.9)) * size * torch.sign(a.float() + 1e-3)).to(torch.bfloat16)
    t = torch.full_like(s, scale)
    c = torch.empty(m, 64, dtype=torch.bfloat16, device="cuda")
    compile_w4a16_gemv(N=64, K=512, group_size=group, zero_points=True)(c, x, q, t, z, None, m, 64)
    check(c, x, q, t, z, None, group)


def test_more_tokens_than_a_grid_has_rows():
    """Any number of tokens, in blocks of 64; the last one of 5."""
    m, n, k = 8 * 65535 + 13, 1, 32
    a, q, s, z, _ = make(m, n, k, 32, "bf16", True, 12)
    c = torch.full((m + 1, n), -77.0, dtype=torch.bfloat16, device="cuda")
    compile_w4a16_gemv(N=n, K=k, group_size=32, zero_points=True)(c, a, q, s, z, None, m, n)
    assert bool((c[m:] == -77.0).all())
    check(c[:m], a, q, s, z, None, 32)


@pytest.mark.parametrize("m", [1, 4, 8, 40])
def test_weights_past_four_gigabytes(m):
    n, k = 140001, 65536
    a, q, s, z, _ = make(m, n, k, 128, "bf16", True, 13)
    assert q.numel() > 2**32
    c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    compile_w4a16_gemv(N=n, K=k, zero_points=True)(c, a, q, s, z, None, m, n)
    for part in (slice(0, 200), slice(n // 2, n // 2 + 200), slice(n - 200, n)):
        check(c[:, part], a, q[part], s[part], z[part], None, 128)
