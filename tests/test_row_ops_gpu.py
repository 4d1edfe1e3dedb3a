"""rmsnorm_quant and silu_mul_quant against their formulas in float64.

Tolerances, from the kernels' arithmetic (u = 2^-24, half a unit of fp32):

* codes per row: code = nearest(h w (qmax / m)) with m the row's maximum of |h w|.  The product, the quotient and its product
  round once each, so the number that is rounded to a code is within 2^-21 of the exact quotient; a code is then at most half a
  step plus 2^-21 |q| away from the exact q.
* norm statistics: a sum of non-negative terms is off by at most u per addition on a term's way, `L` + 12 of them with L elements
  per thread; the root halves that, and the quotient, eps, root and products add six roundings.
* gated values: exp is within 2 ulp, the fast quotient within 2, three more roundings: 2^-20.  Below g = -87 the quotient may
  be 0 where the exact one is below 2^-118.
* 16-bit results: half a step of the type on top."""

import pytest
import torch

from flydsl_b200 import pertoken_quant, rmsnorm_quant, silu_mul_quant
from flydsl_b200.kernels.gemm.mxfp8_preshuffle import per_1x32_f8_quant_torch

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
U = 2.0**-24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
QUANTS = [FP8, torch.int8, "mxfp8", None]
IDS = ["fp8", "int8", "mxfp8", "none"]


def norm64(x, weight, eps, residual=None):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = h.double()
    return d * weight.double() / torch.sqrt(d.square().mean(-1, keepdim=True) + eps), h


def silu64(x):
    g, u = x.double().chunk(2, dim=-1)
    return g * torch.sigmoid(g) * u


def half_step(q, kind):
    if kind == torch.int8:
        return torch.full_like(q, 0.5)
    e = torch.floor(torch.log2(q.abs().clamp_min(2.0**-6)))
    return torch.pow(2.0, e - 4)


def check(y, s, v, quant, rel, floor=0.0):
    """Codes and scales of float64 values v [rows, K] that the kernel knows up to `rel` of their size (and `floor`)."""
    if quant is None:
        eps = torch.finfo(y.dtype)
        half = 0.0 if y.dtype == torch.float32 else eps.eps / 2
        err = (y.double() - v).abs()
        assert bool((err <= v.abs() * (half * (1 + 2**-8) + rel) + eps.tiny * eps.eps + floor).all()), float((err / v.abs().clamp_min(1e-30)).max())
        return
    assert not bool(torch.isnan(y.float()).any())
    if quant == "mxfp8":
        b = v.reshape(v.shape[0], -1, 32)
        top = b.abs().amax(-1).clamp_min(1e-30) / 448.0
        e = torch.floor(torch.log2(top))
        m = top / torch.pow(2.0, e)
        e = e + (m >= 1.5)
        got = s.double() - 127
        near = ((m - 1.5).abs() <= 4 * rel + 2**-20) | (m >= 2 - 2**-20) | (m <= 1 + 2**-20)  # on a border of the exponent rule
        assert bool(((got == e) | (near & ((got - e).abs() <= 1))).all())
        q = (b / torch.pow(2.0, got)[..., None]).clamp(-448, 448)
        err = (y.reshape(b.shape).double() - q).abs()
        assert bool((err <= half_step(q, FP8) + rel * q.abs() + floor / torch.pow(2.0, got)[..., None]).all())
        return
    qmax = 448.0 if quant == FP8 else 127.0
    amax = v.abs().amax(-1, keepdim=True)
    want = torch.where(amax == 0, 1.0, amax / qmax)
    assert s.shape == want.shape and s.dtype == torch.float32
    assert bool(((s.double() - want).abs() <= rel * want).all()), float(((s.double() - want).abs() / want).max())
    q = v / want
    err = (y.double() - q).abs()
    assert bool((err <= half_step(q, quant) + (2**-21 + 2 * rel) * q.abs() + floor / want).all()), float(err.max())


def norm_rel(k):
    per_thread = max(64, -(-k // 256))
    return (per_thread / 2 + 6 + 8) * U


SILU_REL = 2.0**-20


def make(rows, k, dtype, seed, spread=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda") * torch.exp(spread * torch.randn(k, generator=g, device="cuda"))
    return x.to(dtype)


# one element; less than a vector; odd; a vector; one to eight vectors per thread; one to thirty-two warps per row; beyond registers
SHAPES = [(1, 1), (3, 7), (5, 8), (2, 32), (33, 96), (7, 257), (1, 8192), (300, 1024), (2500, 136), (40, 5120), (9, 16384), (4, 32800), (3, 65544),
          (2, 80000)]


@pytest.mark.parametrize("quant", QUANTS, ids=IDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SHAPES)
def test_norm(rows, k, dtype, quant):
    if quant == "mxfp8" and k % 32:
        k = -(-k // 32) * 32
    x, r = make(rows, k, dtype, rows + k), make(rows, k, dtype, rows + k + 1, 1.0)
    w = make(1, k, dtype, 3)[0]
    for residual, weight in ((None, w), (r, w), (r, w.float() * 1.01)):
        y, s, h = rmsnorm_quant(x, weight, 1e-5, residual=residual, quant_dtype=quant)
        v, h64 = norm64(x, weight, 1e-5, residual)
        if residual is None:
            assert h is None
        else:
            assert h.dtype == dtype and torch.equal(h, h64)
        assert y.shape == x.shape and y.dtype == (dtype if quant is None else torch.int8 if quant == torch.int8 else FP8)
        check(y, s, v, quant, norm_rel(k))


@pytest.mark.parametrize("quant", QUANTS, ids=IDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SHAPES)
def test_silu(rows, k, dtype, quant):
    if quant == "mxfp8" and k % 32:
        k = -(-k // 32) * 32
    x = make(rows, 2 * k, dtype, rows + k)
    x[0, 0] = -200.0
    x[-1, k // 2] = 60.0
    y, s = silu_mul_quant(x, quant_dtype=quant)
    assert y.shape == (rows, k)
    check(y, s, silu64(x), quant, SILU_REL, floor=2.0**-115)


@pytest.mark.parametrize("dtype", TYPES)
def test_silu_over_the_range_of_the_gate(dtype):
    """Every gate value of a 16-bit type (of fp32: as many, over the same range), times 1 and -1; infinities and NaN as the formula has them."""
    g = torch.arange(-32768, 32768, device="cuda").to(torch.int16).view(torch.bfloat16 if dtype == torch.float32 else dtype).to(dtype)
    x = torch.stack([torch.cat([g, torch.ones_like(g)]), torch.cat([g, -torch.ones_like(g)])])
    y, none = silu_mul_quant(x, quant_dtype=None)
    want = silu64(x)
    assert none is None
    want = torch.where(torch.isneginf(x[:, : len(g)].double()), torch.nan, want)  # -Inf times 0
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    keep = torch.isfinite(want) & (want.abs() < torch.finfo(dtype).max)
    assert torch.equal(y[~keep & ~torch.isnan(want)].double(), want[~keep & ~torch.isnan(want)])
    check(torch.where(keep, y, 0.0), None, torch.where(keep, want, 0.0), None, SILU_REL, floor=2.0**-115)


@pytest.mark.parametrize("inter", [8200, 12288, 16384, 28672, 32768, 32776])
@pytest.mark.parametrize("quant", [FP8, torch.int8], ids=["fp8", "int8"])
def test_many_wide_gated_rows(inter, quant):
    """More rows than SMs, wider than a row's registers allow two of; strided rows; a row of zeros, NaN and Inf among them."""
    x = make(300, 2 * inter + 8, torch.bfloat16, inter)[:, : 2 * inter]
    x[7] = 0.0
    x[8, 3], x[9, 5], x[9, 6] = float("nan"), float("inf"), float("-inf")
    y, s = silu_mul_quant(x, quant_dtype=quant)
    rows = [i for i in range(300) if i not in (8, 9)]
    check(y[rows], s[rows], silu64(x)[rows], quant, SILU_REL, floor=2.0**-115)
    for i in (8, 9):
        ys, ss = silu_mul_quant(x[i : i + 1], quant_dtype=quant)  # one row takes the other kernel
        assert torch.equal(y[i : i + 1].view(torch.uint8), ys.view(torch.uint8)) and torch.equal(s[i : i + 1], ss)


@pytest.mark.parametrize("k", [4096, 1000, 1003])
@pytest.mark.parametrize("quant", [FP8, torch.int8], ids=["fp8", "int8"])
def test_rows_of_zeros_nan_inf_and_the_ends_of_the_range(quant, k):
    """Row by row what the per-token quantiser makes of the fp32 values: NaN -> 0, Inf -> qmax, zero rows scale 1; a row's
    neighbours in its block do not notice."""
    x = make(16, k, torch.float32, 5)
    w = torch.ones(k, device="cuda")
    x[1] = 0.0
    x[2, 3] = float("nan")
    x[3, 5] = float("inf")
    x[4] *= 1e25  # squares beyond fp32: every value is 0
    x[5] *= 1e-30  # below eps
    x[6] = 0.0
    x[6, k - 1] = -1e-12
    y, s, _ = rmsnorm_quant(x, w, 1e-6, quant_dtype=quant)
    for row in (1, 2, 3, 4):
        assert not bool(y[row].float().any()) and float(s[row]) == 1.0, row
    v, _ = norm64(x, w, 1e-6)
    good = torch.tensor([0] + list(range(6, 16)), device="cuda")
    check(y[good], s[good], v[good], quant, norm_rel(k))
    # a scale near the bottom of fp32: the codes are those of the stored scale
    assert bool((s[5] > 0).all())
    err = (y[5].double() - v[5] / s[5].double()).abs()
    assert bool((err <= half_step(v[5] / s[5].double(), quant) * 1.01).all())
    # gated activation: rows with Inf and NaN go the same way
    z = make(9, 2 * k, torch.float32, 6)
    z[1] = 0.0
    z[2, k + 4] = float("inf")
    z[2, 4] = 1.0
    z[3, 7] = float("nan")
    z[4, 2] = float("-inf")  # -inf / inf
    y, s = silu_mul_quant(z, quant_dtype=quant)
    g, u = z.chunk(2, -1)
    want, ws = pertoken_quant(g / (1 + torch.exp(-g)) * u, quant_dtype=quant, use_kernel=False)
    assert torch.allclose(s, ws, rtol=SILU_REL * 2)
    step = 1.0 if quant == torch.int8 else 32.0  # torch's int8 truncates
    assert bool(((y.float() - want.float()).abs() <= step).all())
    assert not bool(y[1].float().any()) and float(s[1]) == 1.0 and float(y[3, 7]) == 0.0 and float(y[2, 4]) == (127.0 if quant == torch.int8 else 448.0)


def test_mxfp8_matches_the_quantiser_of_the_block_scaled_gemm():
    """Codes and scales of values that fp32 holds exactly are those of per_1x32_f8_quant, NaN and Inf blocks and zeros too."""
    k = 4096
    x = make(64, k, torch.float32, 8) * 100
    x[3, 40] = float("nan")
    x[4, 70] = float("inf")
    x[5, 128:192] = 0.0
    x[6, :32] = 1e-33
    up = torch.cat([torch.full_like(x, 200.0), x], dim=-1)  # silu(200) is 200 in fp32
    y, s = silu_mul_quant(up, quant_dtype="mxfp8")
    want, ws = per_1x32_f8_quant_torch(200.0 * x)
    assert torch.equal(s, ws)
    nan = torch.isnan(want.float())
    assert torch.equal(nan, torch.isnan(y.float())) and torch.equal(y[~nan].view(torch.uint8), want[~nan].view(torch.uint8))


@pytest.mark.parametrize("k", [512, 500, 501])
def test_rows_that_lie_apart_and_in_place_updates(k):
    """Slices of wider tensors, aligned to 16 bytes and not; outputs and residuals where the caller wants them."""
    wide = make(50, 3 * k + 11, torch.bfloat16, 9)
    res = make(50, 2 * k, torch.bfloat16, 10)
    w = make(1, k, torch.bfloat16, 11)[0]
    for at in (0, 8, 3):
        x, r = wide[:, at : at + k], res[:, k:]
        want = rmsnorm_quant(x.contiguous(), w, 1e-5, residual=r.contiguous())
        got = rmsnorm_quant(x, w, 1e-5, residual=r)
        # other vector widths sum in another order: scales to rounding, residuals to the bit
        assert torch.equal(got[2], want[2]) and torch.allclose(got[1], want[1], rtol=2 * norm_rel(k), atol=0)
        kept = res.clone()
        target = res.clone()
        y, s, h = rmsnorm_quant(x, w, 1e-5, residual=target[:, k:], residual_out=target[:, k:])
        assert h.data_ptr() == target[:, k:].data_ptr()
        assert torch.equal(target[:, k:], want[2]) and torch.equal(target[:, :k], kept[:, :k]) and torch.equal(y.view(torch.uint8), got[0].view(torch.uint8))
    x = wide[:, :k].contiguous()
    r, x2 = res[:, :k].contiguous(), x.clone()
    want = rmsnorm_quant(x, w, 1e-5, residual=r, quant_dtype=None)
    out = rmsnorm_quant(x2, w, 1e-5, residual=r, quant_dtype=None, residual_out=x2)  # over x
    assert out[2] is x2 and torch.equal(x2, want[2]) and torch.equal(out[0], want[0])
    out = rmsnorm_quant(x, w, 1e-5, residual=r, quant_dtype=None, residual_out=r)  # over the residual
    assert out[2].data_ptr() == r.data_ptr() and torch.equal(r, want[2]) and torch.equal(out[0], want[0])
    gu = wide[:, : 2 * k]
    for t, q in ((gu, FP8), (gu, None)):
        a, b = silu_mul_quant(t, quant_dtype=q), silu_mul_quant(t.contiguous(), quant_dtype=q)
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and (q is None or torch.equal(a[1], b[1]))


def test_leading_dimensions_and_empty_batches():
    x = make(24, 256, torch.float16, 12)
    w = make(1, 256, torch.float16, 13)[0]
    want = rmsnorm_quant(x, w)
    got = rmsnorm_quant(x.view(2, 3, 4, 256), w)
    assert got[0].shape == (2, 3, 4, 256) and got[1].shape == (2, 3, 4, 1) and torch.equal(got[1].view(-1), want[1].view(-1))
    got = rmsnorm_quant(x[0], w, quant_dtype="mxfp8")
    assert got[0].shape == (256,) and got[1].shape == (8,)
    heads = x.view(24, 2, 128)[:, 1]  # every second head
    assert torch.equal(rmsnorm_quant(heads, w[:128], quant_dtype=None)[0], rmsnorm_quant(heads.contiguous(), w[:128], quant_dtype=None)[0])
    for q in QUANTS:
        y, s, h = rmsnorm_quant(x[:0], w, residual=x[:0], quant_dtype=q)
        assert y.shape == (0, 256) and h.shape == (0, 256)
        y, s = silu_mul_quant(x[:0], quant_dtype=q)
        assert y.shape == (0, 128)


def test_captured_replayed_and_on_another_stream():
    x, r = make(64, 2048, torch.bfloat16, 14), make(64, 2048, torch.bfloat16, 15)
    w = make(1, 2048, torch.bfloat16, 16)[0]
    want = [rmsnorm_quant(x, w, residual=r), silu_mul_quant(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [rmsnorm_quant(x, w, residual=r), silu_mul_quant(x)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = [rmsnorm_quant(x, w, residual=r), silu_mul_quant(x)]
        graph.replay()
    side.synchronize()
    for a, b, c in zip(want, got, kept):
        for i in range(2):
            assert torch.equal(a[i].view(torch.uint8), b[i].view(torch.uint8)) and torch.equal(a[i].view(torch.uint8), c[i].view(torch.uint8))
    x.copy_(make(64, 2048, torch.bfloat16, 17))  # new inputs in the captured buffers
    want = rmsnorm_quant(x, w, residual=r)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept[0][0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(kept[0][1], want[1])


def test_rows_past_two_gigabytes():
    """Offsets beyond 2^31 bytes and elements: the last rows of a tall tensor are those of a short one."""
    rows, k = (1 << 31) // 4096 + 5, 4096
    x = make(64, k, torch.bfloat16, 18).repeat(-(-rows // 64), 1)[:rows]
    w = make(1, k, torch.bfloat16, 19)[0]
    y, s, _ = rmsnorm_quant(x, w)
    want = rmsnorm_quant(x[-64:].contiguous(), w)
    assert bool((y[-64:].float() - want[0].float()).abs().max() <= 32) and torch.allclose(s[-64:], want[1], rtol=2 * norm_rel(k), atol=0)
    del y, s
    y, s = silu_mul_quant(x)
    want = silu_mul_quant(x[-64:].contiguous())
    assert torch.equal(y[-64:].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s[-64:], want[1])


def test_the_same_without_the_host_extension(monkeypatch):
    from flydsl_b200 import _lib, host_statements

    x, r = make(20, 640, torch.float16, 20), make(20, 640, torch.float16, 21)
    w = make(1, 640, torch.float16, 22)[0]
    want = [t for q in QUANTS for t in (*rmsnorm_quant(x, w, residual=r, quant_dtype=q), *silu_mul_quant(x, quant_dtype=q))]
    monkeypatch.setattr(_lib, "_ops", host_statements)
    got = [t for q in QUANTS for t in (*rmsnorm_quant(x, w, residual=r, quant_dtype=q), *silu_mul_quant(x, quant_dtype=q))]
    assert all((a is None and b is None) or torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, got))


def test_a_layer_of_them(monkeypatch):
    """norm -> fp8 gate-up GEMM -> gated activation -> fp8 down GEMM, each step against its formula on what the step before
    wrote, the way a layer uses them."""
    from flydsl_b200 import compile_preshuffle_gemm, shuffle_weight
    from flydsl_b200 import compiler as flyc

    m, d, i = 70, 1024, 768
    st = torch.cuda.current_stream()
    none = torch.empty(0, dtype=torch.bfloat16, device="cuda")

    def linear(w):
        wq, sw = pertoken_quant(w, quant_dtype=FP8)
        n, k = w.shape
        launch = compile_preshuffle_gemm(N=n, K=k, tile_m=64, tile_n=128, tile_k=128, in_dtype="fp8")
        img = shuffle_weight(wq).view(torch.int8).view(-1)
        c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")

        def run(a, sa):
            args = (c.view(-1), a.view(torch.int8).view(-1), img, sa.view(-1), sw.view(-1), none, m, n, st)
            flyc.compile(launch, *args)(*args)
            return c, (a.double() * sa.double()) @ (wq.double() * sw.double()).t()

        return run

    x, r, w = make(m, d, torch.bfloat16, 23), make(m, d, torch.bfloat16, 24), make(1, d, torch.bfloat16, 25)[0]
    up, down = linear(make(2 * i, d, torch.bfloat16, 26) * 0.03), linear(make(d, i, torch.bfloat16, 27) * 0.03)
    for _ in range(2):  # two layers on one residual stream
        y, s, r = rmsnorm_quant(x, w, 1e-5, residual=r)
        v, _ = norm64(r, w, 1e-5)
        check(y, s, v, FP8, norm_rel(d))
        c, c64 = up(y, s)
        assert bool(((c.double() - c64).abs() <= 1e-2 * c64.abs() + 1e-2).all())
        a, sa = silu_mul_quant(c)
        check(a, sa, silu64(c), FP8, SILU_REL, floor=2.0**-115)
        x, x64 = down(a, sa)
        assert bool(((x.double() - x64).abs() <= 1e-2 * x64.abs() + 1e-2).all())
        x = x.clone()


def test_a_tensor_of_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    x = make(8, 512, torch.bfloat16, 28).to("cuda:1")
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda:1")
    with torch.cuda.device(0):
        y, s, _ = rmsnorm_quant(x, w)
        a, sa = silu_mul_quant(x)
    check(y, s, norm64(x, w, 1e-6)[0], FP8, norm_rel(512))
    check(a, sa, silu64(x), FP8, SILU_REL, floor=2.0**-115)
