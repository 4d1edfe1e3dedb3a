"""rmsnorm_quant and silu_mul_quant at the ends of fp32 and of what the arguments allow."""

import pytest
import torch

from flydsl_b200 import rmsnorm_quant, silu_mul_quant
from tests.test_row_ops_gpu import FP8, IDS, QUANTS, SILU_REL, TYPES, check, half_step, make, norm64, norm_rel, silu64

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


@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("k", [4096, 1003, 40000])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("quant", [FP8, torch.int8], ids=["fp8", "int8"])
def test_zero_rows_without_eps(quant, dtype, k, eps):
    """A row of zeros is 0 / 0 in every place, that is NaN, that is 0 with scale 1.  Squares below fp32 are 0: the values are infinite
    then, so qmax with scale 1 (to the rounding of qmax * (1 / qmax)), or NaN and so 0 where the weight is 0."""
    x = make(8, k, dtype, 40)
    w = make(1, k, dtype, 41)[0].abs() + 0.5
    x[2] = 0.0
    qmax = 448.0 if quant == FP8 else 127.0
    if dtype != torch.float16:  # 1e-25 is 0 in fp16
        x[5] = 1e-25
    y, s, _ = rmsnorm_quant(x, w, eps, quant_dtype=quant)
    assert not bool(y[2].float().any()) and float(s[2]) == 1.0
    if dtype != torch.float16:
        assert bool((y[5].float() == qmax).all()) and abs(float(s[5]) - 1.0) <= 2.0**-23
    good = [0, 1, 3, 4, 6, 7]
    check(y[good], s[good], norm64(x, w, 0.0)[0][good], quant, norm_rel(k))
    y, s, h = rmsnorm_quant(x, torch.zeros_like(w), eps, residual=torch.zeros_like(x), quant_dtype=quant)
    assert not bool(y.float().any()) and bool((s == 1.0).all()) and torch.equal(h, x)


# The gated value, by the kernel's steps: 2^t within 2^-22, and rounded once more where it is below 2^-126; its correction, 1 + exp and the
# products round once each, the reciprocal is good to its last place: 11 units of 2^-24, and the next power of two is SILU_REL.  Below 2^-126 an
# exponential is off by up to two steps of 2^-149: |g u| times that.  A result below 2^-126 is off by a step itself.
def gated_bound(x, v):
    g, u = x.double().chunk(2, dim=-1)
    return SILU_REL * v.abs() + (g * u).abs() * 2.0**-148 + 2.0**-149


@pytest.mark.parametrize("lo,hi", [(-1.0, 1.0), (-20.0, 20.0), (-87.0, -60.0), (-89.0, -86.0), (-104.0, -88.0), (-300.0, -100.0), (60.0, 300.0)])
@pytest.mark.parametrize("up", [1.0, 1e38, 1e-6])
def test_gated_values_hold_fp32(lo, hi, up):
    """Without a floor: between -88 and -104 exp(g) is below 2^-126, but a product with a large `up` is not."""
    k = 65536
    g = torch.linspace(lo, hi, k, device="cuda")
    u = torch.full_like(g, up) * torch.where(torch.arange(k, device="cuda") % 3 == 0, -1.0, 0.75)
    x = torch.cat([g, u])[None]
    y, none = silu_mul_quant(x, quant_dtype=None)
    v = silu64(x)
    keep = v.abs() < 3.4e38
    assert none is None and bool(torch.isinf(y[~keep & (v.abs() > 3.41e38)]).all())
    err = (y.double() - v).abs()
    assert bool((err <= gated_bound(x, v))[keep].all()), float((err / gated_bound(x, v))[keep].max())


@pytest.mark.parametrize("inter,rows", [(96, 5), (1003, 5), (5120, 300)])
@pytest.mark.parametrize("quant", [FP8, torch.int8, "mxfp8"], ids=["fp8", "int8", "mxfp8"])
def test_rows_of_gates_far_below_zero(quant, inter, rows):
    """What such gates leave is all that a row has."""
    if quant == "mxfp8":
        inter = -(-inter // 32) * 32
    g = torch.Generator(device="cuda").manual_seed(42)
    gate = -87.0 - 3.0 * torch.rand(rows, inter, generator=g, device="cuda")
    x = torch.cat([gate, 1e35 * torch.randn(rows, inter, generator=g, device="cuda")], dim=-1)
    y, s = silu_mul_quant(x, quant_dtype=quant)
    # exp(g) is at least 2^-130 there: two steps of 2^-149 are 2^-18 of it
    check(y, s, silu64(x), quant, SILU_REL + 2.0**-18)


@pytest.mark.parametrize("k", [4096, 1003, 40000])
@pytest.mark.parametrize("dtype,size,weight,eps", [(torch.float32, 1e15, 1e25, 1e-6), (torch.bfloat16, 1e15, 1e25, 1e-6), (torch.float16, 100.0, 1e38, 1e-6),
                                                   (torch.float32, 1e-15, 1e-27, 0.0), (torch.bfloat16, 1e-15, 1e-27, 0.0)],
                         ids=["large32", "largebf16", "largefp16", "small32", "smallbf16"])
@pytest.mark.parametrize("quant", QUANTS, ids=IDS)
def test_norm_where_input_times_weight_leaves_fp32(quant, dtype, size, weight, eps, k):
    """h w is out of range while h w / rms(h) is not."""
    if quant == "mxfp8":
        k = -(-k // 32) * 32
    if quant is None and dtype == torch.float16:
        dtype = torch.bfloat16  # values of 1e38 are none of fp16
    x = (torch.randn(6, k, generator=torch.Generator(device="cuda").manual_seed(43), device="cuda") * size).to(dtype)
    w = (1.0 + torch.rand(k, generator=torch.Generator(device="cuda").manual_seed(44), device="cuda")) * weight / 4
    w = w if dtype == torch.float16 else w.to(dtype)
    x[3] *= 1e-3
    r = (x * 0.25).to(dtype)
    for residual in (None, r):
        y, s, h = rmsnorm_quant(x, w, eps, residual=residual, quant_dtype=quant)
        v, h64 = norm64(x, w, eps, residual)
        assert residual is None or torch.equal(h, h64)
        if quant != "mxfp8":
            check(y, s, v, quant, norm_rel(k))
            continue
        # the quantiser divides by at least 1e-30, also where the scale byte says less
        b, unit = v.reshape(6, -1, 32), torch.pow(2.0, s.double() - 127)[..., None]
        q = (b / unit.clamp_min(1e-30)).clamp(-448, 448)
        top = b.abs().amax(-1, keepdim=True)
        assert bool((top <= 448 * 1.5 * unit * (1 + 2**-16)).all() and (top >= 448 * 0.75 * unit * (1 - 2**-16)).all())
        assert bool(((y.reshape(b.shape).double() - q).abs() <= half_step(q, FP8) + norm_rel(k) * q.abs()).all())


def test_sums_beside_the_inputs_in_one_buffer():
    """residual_out in other columns of the buffer that x lies in: their address ranges cross, their elements do not."""
    k = 256
    buf, r = make(20, 3 * k, torch.bfloat16, 45), make(20, k, torch.bfloat16, 46)
    w = make(1, k, torch.bfloat16, 47)[0]
    x = buf[:, :k]
    want = rmsnorm_quant(x.clone(), w, residual=r)
    kept = buf.clone()
    y, s, h = rmsnorm_quant(x, w, residual=r, residual_out=buf[:, 2 * k :])
    assert torch.equal(h, want[2]) and torch.equal(y.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])
    assert torch.equal(buf[:, : 2 * k], kept[:, : 2 * k]) and h.data_ptr() == buf[:, 2 * k :].data_ptr()
    for at in (1, k - 1):
        with pytest.raises(ValueError, match="overlaps x"):
            rmsnorm_quant(x, w, residual=r, residual_out=buf[:, at : at + k])
    # one row: its distance to the next one says nothing
    one = buf[:1, :k]
    want = rmsnorm_quant(one.clone(), w, residual=r[:1])
    same = one.as_strided((1, k), (7 * k, 1))
    assert torch.equal(rmsnorm_quant(one, w, residual=r[:1], residual_out=same)[2], want[2]) and torch.equal(one, want[2])


@pytest.mark.parametrize("k", [4096, 4095])
def test_rows_past_four_gigabytes(k):
    """Inputs beyond 2^32 bytes and outputs beyond 2^31 elements, of rows that repeat after 61: an offset that wraps meets another row.  Whole
    vectors, and odd rows.  Other numbers of rows sum in another order."""
    rows = (1 << 31) // k + 70
    tail = torch.arange(rows - 122, rows, device="cuda") % 61
    w = make(1, k, torch.bfloat16, 48)[0]
    base = make(61, k, torch.bfloat16, 49)
    x = base.repeat(-(-rows // 61), 1)[:rows]
    y, s, h = rmsnorm_quant(x, w, 1e-5, residual=x, quant_dtype=torch.int8)
    v, h64 = norm64(base, w, 1e-5, base)
    assert torch.equal(h[-122:], h64[tail])
    check(y[-122:], s[-122:], v[tail], torch.int8, norm_rel(k))
    del x, y, s, h
    base = make(61, 2 * k, torch.bfloat16, 50)
    x = base.repeat(-(-rows // 61), 1)[:rows]
    assert x.numel() > 2**32 and rows * k > 2**31
    for quant in (FP8, None):
        y, s = silu_mul_quant(x, quant_dtype=quant)
        check(y[-122:], None if s is None else s[-122:], silu64(base)[tail], quant, SILU_REL)
        del y, s
