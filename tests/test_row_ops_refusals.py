"""What rmsnorm_quant, silu_mul_quant and the 4-bit products refuse, by message, and what the library's entry points refuse
by code: no GPU work is started by any of it."""

import ctypes

import pytest
import torch

from flydsl_b200 import _lib, compile_w4a16_gemv, per_group_w4_quant, rmsnorm_quant, silu_mul_quant
from flydsl_b200.kernels.gemm.w4_gemv import w4_to_f32

BF16 = torch.bfloat16


def test_cpu_tensors_and_arguments():
    x, w = torch.zeros(4, 64, dtype=BF16), torch.ones(64, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        rmsnorm_quant(x, w)
    with pytest.raises(ValueError, match="CUDA tensor"):
        silu_mul_quant(x)
    with pytest.raises(ValueError, match="quant_dtype"):
        rmsnorm_quant(x, w, quant_dtype=torch.float8_e5m2)
    with pytest.raises(ValueError, match="quant_dtype"):
        silu_mul_quant(x, quant_dtype="mxfp4")
    with pytest.raises(ValueError, match="eps"):
        rmsnorm_quant(x, w, -1e-6)
    with pytest.raises(ValueError, match="eps"):
        rmsnorm_quant(x, w, float("nan"))
    with pytest.raises(ValueError, match="without a residual"):
        rmsnorm_quant(x, w, residual_out=x)


def test_library_codes_need_no_gpu():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) & ~15

    def norm(y=p, scale=p, h=None, x=p, r=None, w=p, rows=1, k=64, xs=64, rs=0, hs=0, eps=1e-6, dt=2, wf=0, q=1):
        return lib.flyb200_rmsnorm_quant(y, scale, h, x, r, w, rows, k, xs, rs, hs, eps, dt, wf, q, None)

    assert norm(rows=0) == 0
    for bad in (dict(y=None), dict(x=None), dict(w=None), dict(scale=None), dict(rows=-1), dict(k=0), dict(dt=3), dict(dt=-1), dict(q=4), dict(q=0),
                dict(r=p), dict(h=p), dict(xs=63), dict(r=p, h=p, rs=63, hs=64), dict(eps=-1.0), dict(eps=float("nan")), dict(k=1 << 30, xs=1 << 30)):
        assert norm(**bad) == _lib.E_BAD_ARG, bad
    assert norm(k=40, q=3) == _lib.E_UNSUPPORTED
    for bad in (dict(x=p + 1), dict(w=p + 1), dict(w=p + 2, wf=1), dict(scale=p + 2), dict(y=p + 1, scale=None, q=0), dict(r=p + 1, h=p, rs=64, hs=64)):
        assert norm(**bad) == _lib.E_BAD_ALIGN, bad

    def silu(y=p, scale=p, x=p, rows=1, i=64, xs=128, dt=2, q=1):
        return lib.flyb200_silu_mul_quant(y, scale, x, rows, i, xs, dt, q, None)

    assert silu(rows=0) == 0
    for bad in (dict(y=None), dict(x=None), dict(scale=None), dict(rows=-1), dict(i=0), dict(i=1 << 30), dict(dt=3), dict(q=-1), dict(q=0), dict(xs=127)):
        assert silu(**bad) == _lib.E_BAD_ARG, bad
    assert silu(i=40, q=3) == _lib.E_UNSUPPORTED
    assert silu(rows=2**31 - 1, i=4096, xs=8192, q=3) == _lib.E_UNSUPPORTED  # more blocks than a grid has
    assert silu(x=p + 1) == _lib.E_BAD_ALIGN

    def w4(c=p, a=p, q=p, s=p, z=None, b=None, m=1, n=16, k=128, g=128, dt=_lib.DT_BF16, e=0):
        return lib.flyb200_gemv_w4a16(c, a, q, s, z, b, m, n, k, g, dt, e, None)

    assert w4(m=0) == 0
    for bad in (dict(c=None), dict(a=None), dict(q=None), dict(s=None), dict(m=-1), dict(n=0), dict(k=0), dict(g=16), dict(g=256), dict(dt=_lib.DT_FP8),
                dict(e=1), dict(e=5), dict(e=-1)):
        assert w4(**bad) == _lib.E_BAD_ARG, bad
    assert w4(k=192) == _lib.E_UNSUPPORTED
    for bad in (dict(a=p + 8), dict(q=p + 8), dict(c=p + 1), dict(s=p + 1), dict(b=p + 1, e=1)):
        assert w4(**bad) == _lib.E_BAD_ALIGN, bad


def test_builder_and_launcher_of_the_four_bit_products():
    for bad in (dict(in_dtype="fp8"), dict(epilogue="relu"), dict(group_size=16), dict(group_size=96), dict(N=0), dict(K=0), dict(K=200), dict(K=-128)):
        with pytest.raises(ValueError):
            compile_w4a16_gemv(**(dict(N=64, K=256) | bad))
    fn = compile_w4a16_gemv(N=64, K=256, zero_points=True, epilogue="bias")
    t = torch.zeros(64, 256, dtype=BF16)
    with pytest.raises(ValueError, match="differs"):
        fn(t, t, t, t, t, t, 1, 32)
    with pytest.raises(ValueError, match="non-negative"):
        fn(t, t, t, t, t, t, -1, 64)
    assert fn(t, t, t, t, t, t, 0, 64) is None
    with pytest.raises(ValueError, match="CUDA tensor"):
        fn(t, t, t, t, t, t, 1, 64)


def test_compile_only_launches_nothing(monkeypatch):
    monkeypatch.setenv("COMPILE_ONLY", "1")
    t = torch.zeros(64, 256, dtype=BF16)
    assert compile_w4a16_gemv(N=64, K=256)(t, t, t, t, None, None, 1, 64) is None


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantiser_on_the_cpu(group, zeros):
    g = torch.Generator().manual_seed(1)
    w = torch.randn(24, 256, generator=g) * 0.05
    w[3] = 0.0
    w[4, :group] = 0.3  # one sign
    w[5, 0] = -1.0
    q, s, z = per_group_w4_quant(w, group, zero_points=zeros)
    assert q.shape == (24, 128) and q.dtype == torch.uint8 and s.shape == (24, 256 // group) and s.dtype == BF16 and (z is None) == (not zeros)
    back = w4_to_f32(q, s, z)
    step = s.float().repeat_interleave(group, dim=1)
    assert bool(((back - w).abs() <= step * (1.01 if zeros else 0.52)).all()) and not bool(back[3].any())
    # nibble order: input 0 in the low half of byte 0
    first = (q[:, 0] & 15).float() - (8.0 if z is None else z[:, 0].float())
    assert torch.equal(first * s[:, 0].float(), back[:, 0])
    for bad in (dict(group_size=48), dict(group_size=16), dict(scale_dtype=torch.float32)):
        with pytest.raises(ValueError):
            per_group_w4_quant(w, **bad)
    with pytest.raises(ValueError):
        per_group_w4_quant(w[0], group)


@pytest.mark.gpu
def test_refusals_of_cuda_tensors():
    x, w = torch.zeros(4, 64, dtype=BF16, device="cuda"), torch.ones(64, dtype=BF16, device="cuda")
    cases = [
        (lambda: rmsnorm_quant(x.t(), w[:4]), "last dimension"),
        (lambda: rmsnorm_quant(x.double(), w), "fp32, fp16 or bf16"),
        (lambda: rmsnorm_quant(x, w.half()), "weight must be"),
        (lambda: rmsnorm_quant(x, w[:32]), "weight must be"),
        (lambda: rmsnorm_quant(x, w.cpu()), "weight must be"),
        (lambda: rmsnorm_quant(x, w, residual=x.half()), "residual must have"),
        (lambda: rmsnorm_quant(x, w, residual=x[:2]), "residual must have"),
        (lambda: rmsnorm_quant(x[:, :40], w[:40], quant_dtype="mxfp8"), "multiple of 32"),
        (lambda: rmsnorm_quant(x[:1].expand(4, 64), w), "overlap"),
        (lambda: rmsnorm_quant(x.view(2, 2, 64).transpose(0, 1), w), "equal distances"),
        (lambda: rmsnorm_quant(x[:, :0], w[:0]), "without elements"),
        (lambda: rmsnorm_quant(x.requires_grad_(False).clone().requires_grad_(), w), "no backward"),
        (lambda: rmsnorm_quant(x, w.clone().requires_grad_()), "no backward"),
        (lambda: rmsnorm_quant(x[:2], w, residual=x[1:3], residual_out=x[2:4]), "overlaps residual"),
        (lambda: rmsnorm_quant(x, w, residual=x.clone(), residual_out=x[:2]), "residual_out must have"),
        (lambda: silu_mul_quant(x[:, :63]), "even last dimension"),
        (lambda: silu_mul_quant(x[:, :48], quant_dtype="mxfp8"), "multiple of 32"),
        (lambda: silu_mul_quant(x.clone().requires_grad_()), "no backward"),
    ]
    for call, words in cases:
        with pytest.raises(ValueError, match=words):
            call()
    with torch.no_grad():
        rmsnorm_quant(x.clone().requires_grad_(), w)
    c, q, s = torch.zeros(4, 32, dtype=BF16, device="cuda"), torch.zeros(32, 32, dtype=torch.uint8, device="cuda"), torch.ones(32, 1, dtype=BF16, device="cuda")
    fn = compile_w4a16_gemv(N=32, K=64, group_size=64)
    z = torch.zeros(32, 1, dtype=torch.uint8, device="cuda")
    fnz = compile_w4a16_gemv(N=32, K=64, group_size=64, zero_points=True)
    fn(c, x, q, s, None, None, 4, 32)
    for args, words in (((c.half(), x, q, s, None, None), "c must be"), ((c, x.half(), q, s, None, None), "a must be"), ((c, x, q, s.float(), None, None), "scale_b must be"),
                        ((c[:2], x, q, s, None, None), "c holds"), ((c, x[:, ::2], q, s, None, None), "contiguous"), ((c, x, q[:16], s, None, None), "b holds"),
                        ((c, x, s, s, None, None), "one-byte")):
        with pytest.raises(ValueError, match=words):
            fn(*args, 4, 32)
    for zero in (None, z.int(), z[:8]):
        with pytest.raises(ValueError, match="zero_b"):
            fnz(c, x, q, s, zero, None, 4, 32)
    with pytest.raises(ValueError, match="bias"):
        compile_w4a16_gemv(N=32, K=64, group_size=64, epilogue="bias")(c, x, q, s, None, None, 4, 32)
    with pytest.raises(_lib.FlyB200Error):
        fn(c, torch.zeros(264, dtype=BF16, device="cuda")[4:260], q, s, None, None, 4, 32)  # not on a 16-byte address
    torch.cuda.synchronize()
