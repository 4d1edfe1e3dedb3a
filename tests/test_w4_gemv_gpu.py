"""The products on 4-bit weights against their formula in float64.

Tolerance: codes minus zero points and their products with 16-bit activations are exact; what rounds is the fp32 sums.  A term
passes at most G / 16 tensor-core additions (each off by at most 2^-22 of the terms so far: its aligned sum keeps 24 bits and
cuts), then the scale and the sum over the groups (K / G fused additions at most, in one chain), the sum of two such chains and
over the blocks of a cluster (up to 8): c is off by at most (G / 16 * 4 + K / G + 10) 2^-24 of the sum of the magnitudes, plus half a
step of its own type.  Up to 4 tokens the activations of a group are rounded to multiples of 2^-21 of the power of two at
or below its largest magnitude, by half a multiple at most: the weights of the group times 2^-22 of that magnitude come on top."""

import pytest
import torch

from flydsl_b200 import compile_w4a16_gemv, per_group_w4_quant
from flydsl_b200 import compiler as flyc
from flydsl_b200.kernels.gemm.w4_gemv import w4_to_f32

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(m, n, k, group, x, zeros, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[x]
    a = torch.randn(m, k, generator=g, device="cuda").to(t)
    q = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = (0.02 * torch.exp(torch.randn(n, k // group, generator=g, device="cuda"))).to(t)
    z = torch.randint(0, 16, (n, k // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    bias = torch.randn(n, generator=g, device="cuda").to(t)
    return a, q, s, z, bias


def weights64(q, s, z):
    n, groups = s.shape
    codes = torch.stack([q & 15, q >> 4], dim=-1).reshape(n, groups, -1).double()
    return ((codes - (8.0 if z is None else z.double()[..., None])) * s.double()[..., None]).reshape(n, -1)


ACT = {"none": lambda v: v, "bias": lambda v: v, "bias_relu": torch.relu, "bias_silu": torch.nn.functional.silu,
       "bias_gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}


def check(c, a, q, s, z, bias, group, epilogue="none"):
    w = weights64(q, s, z)
    k = w.shape[1]
    c64, mag = a.double() @ w.t(), a.double().abs() @ w.abs().t()
    if epilogue != "none":
        c64, mag = c64 + bias.double(), mag + bias.double().abs()
    sums = (group / 16 * 4 + k / group + 10) * 2.0**-24 * mag
    if len(a) <= 4:
        top = a.double().abs().reshape(len(a), -1, group).amax(-1)
        sums = sums + 2.0**-22 * top @ w.abs().reshape(len(w), -1, group).sum(-1).t()
    c64 = ACT[epilogue](c64)
    # relu, silu and gelu change a value by at most 1.13 of what its argument changes; exp and the quotients: 2^-20
    err, info = (c.double() - c64).abs(), torch.finfo(c.dtype)
    tol = info.eps / 2 * 1.01 * c64.abs() + 1.2 * sums + 2.0**-20 * c64.abs() + info.tiny * info.eps
    if epilogue == "bias_gelu":
        tol = tol + 2.0**-20 * mag  # 1 + tanh loses leading digits where the result is small
    assert bool((err <= tol).all()), float((err / tol).max())


def run(m, n, k, group, x="bf16", zeros=False, epilogue="none", seed=0):
    a, q, s, z, bias = make(m, n, k, group, x, zeros, seed)
    c = torch.full((m + 3, n), -77.0, dtype=TYPES[x], device="cuda")
    fn = compile_w4a16_gemv(N=n, K=k, group_size=group, in_dtype=x, zero_points=zeros, epilogue=epilogue)
    fn(c, a, q, s, z, bias, m, n, torch.cuda.current_stream())
    assert bool((c[m:] == -77.0).all())  # rows behind the last token
    check(c[:m], a, q, s, z, bias, group, epilogue)
    return c[:m]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True], ids=["signed", "zeros"])
@pytest.mark.parametrize("x", ["bf16", "fp16"])
@pytest.mark.parametrize("m", [1, 2, 8, 9, 16, 17, 31, 33, 64, 65, 100])
def test_tokens(m, x, zeros, group):
    run(m, 320, 1024, group, x, zeros, seed=m)


# one group; chunks that end inside; fewer groups than warps; odd numbers of rows; rows fewer than a tile; long inputs
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (7, 64, 64), (16, 128, 128), (33, 96, 32), (63, 1088, 64), (65, 1184, 32), (129, 2176, 128),
                                       (1000, 704, 64), (17, 28672, 128), (64, 16384, 32), (2561, 512, 128), (9473, 256, 64)])
@pytest.mark.parametrize("m", [1, 5, 13, 40])
def test_shapes(m, n, k, group):
    run(m, n, k, group, "bf16", True, seed=n + k)
    run(m, n, k, group, "fp16", False, seed=n + k + 1)


@pytest.mark.parametrize("epilogue", ["none", "bias", "bias_relu", "bias_silu", "bias_gelu"])
@pytest.mark.parametrize("x", ["bf16", "fp16"])
def test_epilogues(x, epilogue):
    run(3, 200, 512, 128, x, True, epilogue)
    run(20, 72, 256, 32, x, False, epilogue)


@pytest.mark.parametrize("x", ["bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_code_and_place_is_exact(group, x):
    """Integer activations, scales that are powers of two, sums below 2^24: the result is the exact sum, rounded once.  A one-hot
    activation reads back each weight."""
    n, k = 48, 512
    a, q, s, z, _ = make(k, n, k, group, x, True, 5)
    s = torch.pow(2.0, torch.randint(-3, 4, s.shape, device="cuda").float()).to(TYPES[x])
    fn = compile_w4a16_gemv(N=n, K=k, group_size=group, in_dtype=x, zero_points=True)
    eye = torch.eye(k, device="cuda", dtype=TYPES[x])
    c = torch.empty(k, n, dtype=TYPES[x], device="cuda")
    fn(c, eye, q, s, z, None, k, n, torch.cuda.current_stream())
    assert torch.equal(c.double(), weights64(q, s, z).t())
    ints = torch.randint(-20, 21, (6, k), device="cuda").to(TYPES[x])
    fn(c, ints, q, s, z, None, 6, n, torch.cuda.current_stream())
    assert torch.equal(c[:6], (ints.double() @ weights64(q, s, z).t()).to(TYPES[x]))


def test_deterministic_and_independent_of_the_batch():
    """Of up to 4 tokens (integers), and of 5 to 64."""
    a, q, s, z, bias = make(40, 4100, 4096, 128, "bf16", True, 6)
    fn = compile_w4a16_gemv(N=4100, K=4096, group_size=128, zero_points=True)

    def product(x):
        c = torch.empty(len(x), 4100, dtype=torch.bfloat16, device="cuda")
        fn(c, x, q, s, z, None, len(x), 4100, torch.cuda.current_stream())
        return c

    few, many = product(a[:4]), product(a)
    assert all(torch.equal(few, product(a[:4])) and torch.equal(many, product(a)) for _ in range(2))
    assert torch.equal(product(a[3:4].contiguous())[0], few[3])
    assert torch.equal(product(a[30:38].contiguous()), many[30:38])


def test_infinities_and_nan_stay_in_their_token():
    a, q, s, z, _ = make(4, 100, 512, 64, "bf16", True, 7)
    a[1, 5], a[2, 300] = float("nan"), float("inf")
    fn = compile_w4a16_gemv(N=100, K=512, group_size=64, zero_points=True)
    c = torch.empty(4, 100, dtype=torch.bfloat16, device="cuda")
    fn(c, a, q, s, z, None, 4, 100, torch.cuda.current_stream())
    assert bool(torch.isnan(c[1]).all()) and not bool(torch.isfinite(c[2]).any())
    check(c[[0, 3]], a[[0, 3]], q, s, z, None, 64)


@pytest.mark.parametrize("m", [4, 8, 16, 32, 64])
@pytest.mark.parametrize("n,k,group", [(28672, 2048, 128), (1024, 16384, 64), (19000, 4096, 32)])
def test_many_launches_in_a_row(n, k, group, m):
    """Without a pause between them, more blocks than SMs, weights that come from memory: every one gives the same result."""
    a, q, s, z, _ = make(m, n, k, group, "fp16", True, 12)
    fn = compile_w4a16_gemv(N=n, K=k, group_size=group, in_dtype="fp16", zero_points=True)
    others = [q.clone() for _ in range(4)]
    outs = [torch.empty(m, n, dtype=torch.float16, device="cuda") for _ in range(40)]
    for i, c in enumerate(outs):
        fn(c, a, others[i % 4], s, z, None, m, n, torch.cuda.current_stream())
    check(outs[0], a, q, s, z, None, group)
    assert all(torch.equal(outs[0], c) for c in outs)


@pytest.mark.parametrize("m", [1, 4, 5, 40])
def test_largest_and_smallest_activations(m):
    """bf16 activations at both ends of its range; the weights bring the sums back into it."""
    a, q, s, z, _ = make(m, 64, 256, 32, "bf16", True, 11)
    fn = compile_w4a16_gemv(N=64, K=256, group_size=32, zero_points=True)
    for size, scale in ((2.0**127, 2.0**-40), (2.0**-100, 2.0**60)):
        x = (a.float().clamp(-1.9, 1.9) * size).to(torch.bfloat16)
        t = torch.full_like(s, scale)
        c = torch.empty(m, 64, dtype=torch.bfloat16, device="cuda")
        fn(c, x, q, t, z, None, m, 64, torch.cuda.current_stream())
        check(c, x, q, t, z, None, 32)


def test_quantiser_and_product():
    w = torch.randn(256, 1024, device="cuda") * 0.02
    a = torch.randn(5, 1024, device="cuda").to(torch.bfloat16)
    for zeros in (False, True):
        for group in (32, 64, 128):
            q, s, z = per_group_w4_quant(w, group, zero_points=zeros)
            back = w4_to_f32(q, s, z)
            # half a step of the group's scale; with zero points the zero point rounds too, and the end of the range may clip by half a step
            step = s.float().repeat_interleave(group, dim=1)
            assert bool(((back - w).abs() <= step * (1.01 if zeros else 0.52)).all())
            c = torch.empty(5, 256, dtype=torch.bfloat16, device="cuda")
            fn = flyc.compile(compile_w4a16_gemv(N=256, K=1024, group_size=group, zero_points=zeros))
            fn(c, a, q, s, z, None, 5, 256, torch.cuda.current_stream())
            check(c, a, q, s, z, None, group)


def test_captured_replayed_and_on_another_stream():
    m, n, k = 4, 1000, 2048
    a, q, s, z, bias = make(m, n, k, 128, "fp16", True, 8)
    fn = compile_w4a16_gemv(N=n, K=k, in_dtype="fp16", zero_points=True, epilogue="bias_silu")
    want, c = torch.empty(m, n, dtype=torch.float16, device="cuda"), torch.empty(m, n, dtype=torch.float16, device="cuda")
    fn(want, a, q, s, z, bias, m, n, torch.cuda.current_stream())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):  # two graphs, replayed at the same time below
            out = torch.empty_like(c)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                fn(out, a, q, s, z, bias, m, n, side)
            graphs.append((graph, out))
    side.synchronize()
    other = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out in graphs)


def test_without_the_host_extension(monkeypatch):
    from flydsl_b200 import _lib, host_statements

    want = run(5, 100, 256, 64, "bf16", True, "bias")
    monkeypatch.setattr(_lib, "_ops", host_statements)
    assert torch.equal(run(5, 100, 256, 64, "bf16", True, "bias"), want)


def test_decode_layer_on_four_bit_weights():
    """norm -> gate-up product -> gated activation -> down product with 16-bit activations, as a decode step runs them."""
    from flydsl_b200 import rmsnorm_quant, silu_mul_quant
    from tests.test_row_ops_gpu import SILU_REL, norm64, norm_rel, silu64
    from tests.test_row_ops_gpu import check as check_rows

    m, d, i = 3, 1024, 1536
    st = torch.cuda.current_stream()
    a, q1, s1, z1, _ = make(m, 2 * i, d, 128, "bf16", True, 9)
    _, q2, s2, z2, _ = make(m, d, i, 64, "bf16", False, 10)
    up, down = compile_w4a16_gemv(N=2 * i, K=d, zero_points=True), compile_w4a16_gemv(N=d, K=i, group_size=64)
    w, r = torch.ones(d, dtype=torch.bfloat16, device="cuda"), torch.randn(m, d, device="cuda").to(torch.bfloat16)
    c, x = torch.empty(m, 2 * i, dtype=torch.bfloat16, device="cuda"), torch.empty(m, d, dtype=torch.bfloat16, device="cuda")
    y, none, r = rmsnorm_quant(a, w, 1e-5, residual=r, quant_dtype=None, residual_out=r)
    assert none is None
    check_rows(y, None, norm64(r, w, 1e-5)[0], None, norm_rel(d))
    up(c, y, q1, s1, z1, None, m, 2 * i, st)
    check(c, y, q1, s1, z1, None, 128)
    h, _ = silu_mul_quant(c, quant_dtype=None)
    check_rows(h, None, silu64(c), None, SILU_REL, floor=2.0**-115)
    down(x, h, q2, s2, None, None, m, d, st)
    check(x, h, q2, s2, None, None, 64)
