"""The products on 4-bit weights where torch has to see the operations: the launch becomes torch operations on its output."""

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from flydsl_b200 import _lib, compile_w4a16_gemv, host_statements

BF16 = torch.bfloat16


def test_fake_cuda_tensors_and_their_trace():
    fn = compile_w4a16_gemv(N=32, K=128, group_size=64, zero_points=True, epilogue="bias_silu")
    with FakeTensorMode(allow_non_fake_inputs=True):
        c, a = torch.empty(5, 32, device="cuda", dtype=BF16), torch.empty(4, 128, device="cuda", dtype=BF16)
        q, z = torch.empty(32, 64, device="cuda", dtype=torch.int8), torch.empty(32, 2, device="cuda", dtype=torch.uint8)
        s, b = torch.empty(32, 2, device="cuda", dtype=BF16), torch.empty(32, device="cuda", dtype=BF16)
        assert fn(c, a, q, s, z, b, 4, 32) is None
        with pytest.raises(ValueError, match="a holds"):
            fn(c, a, q, s, z, b, 5, 32)

        def step(c, a, q, s, z, b):
            fn(c, a, q, s, z, b, 4, 32)
            return c

        graph = make_fx(step)(c, a, q, s, z, b)
    written = next(n for n in graph.graph.nodes if "copy_" in str(n.target))
    reached, todo = set(), [written]
    while todo:
        n = todo.pop()
        if n not in reached:
            reached.add(n)
            todo += n.all_input_nodes
    assert all(n in reached for n in graph.graph.nodes if n.op == "placeholder")


@pytest.mark.gpu
@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("m", [3, 20])
def test_lazy_negation(m, extension, monkeypatch):
    from tests.test_w4_gemv_gpu import check, make

    if not extension:
        monkeypatch.setattr(_lib, "_ops", host_statements)
    a, q, s, z, bias = make(m, 72, 256, 64, "bf16", True, 1)
    fn = compile_w4a16_gemv(N=72, K=256, group_size=64, zero_points=True, epilogue="bias_silu")
    neg = torch._neg_view
    for args, plain in (((neg(a), q, s, z, bias), (-a, q, s, z, bias)), ((a, q, neg(s), z, bias), (a, q, -s, z, bias)), ((a, q, s, z, neg(bias)), (a, q, s, z, -bias))):
        c = torch.full((m + 1, 72), -77.0, dtype=BF16, device="cuda")
        fn(c, *args, m, 72)
        assert bool((c[m:] == -77.0).all())
        check(c[:m], *plain, 64, "bias_silu")
    c = torch.empty(m, 72, dtype=BF16, device="cuda")
    fn(neg(c), a, q, s, z, bias, m, 72)
    check(-c, a, q, s, z, bias, 64, "bias_silu")


@pytest.mark.gpu
@pytest.mark.parametrize("extension", [True, False])
def test_subclasses_stay_on_the_kernel(extension, monkeypatch):
    """A parameter class of a program's own has its values at its address."""
    from flydsl_b200.kernels.gemm.w4_gemv import W4Gemv
    from tests.test_w4_gemv_gpu import check, make

    class Weight(torch.nn.Parameter):
        pass

    if not extension:
        monkeypatch.setattr(_lib, "_ops", host_statements)
    monkeypatch.setattr(W4Gemv, "_statements", None)  # not called
    a, q, s, z, _ = make(4, 72, 256, 64, "bf16", True, 6)
    own = [t.as_subclass(Weight) for t in (q, s, z)]
    c = torch.empty(4, 72, dtype=BF16, device="cuda")
    compile_w4a16_gemv(N=72, K=256, group_size=64, zero_points=True)(c, a, *own, None, 4, 72)
    check(c, a, q, s, z, None, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("epilogue", ["none", "bias", "bias_relu", "bias_silu", "bias_gelu"])
def test_traced_and_compiled(epilogue):
    from tests.test_w4_gemv_gpu import check, make

    a, q, s, z, bias = make(4, 72, 256, 64, "fp16", False, 2)
    other = make(4, 72, 256, 64, "fp16", False, 3)[0]
    fn = compile_w4a16_gemv(N=72, K=256, group_size=64, in_dtype="fp16", epilogue=epilogue)

    def step(x):
        c = torch.empty(4, 72, dtype=torch.float16, device="cuda")
        fn(c, x, q, s, None, bias, 4, 72)
        return c

    for form in (lambda: make_fx(step)(a), lambda: torch.compile(step, backend="eager", fullgraph=True)):
        check(form()(other), other, q, s, None, bias, 64, epilogue)


@pytest.mark.gpu
def test_tangents_travel():
    from tests.test_w4_gemv_gpu import make, weights64

    a, q, s, z, _ = make(3, 40, 128, 32, "bf16", True, 4)
    t = make(3, 40, 128, 32, "bf16", True, 5)[0]
    fn = compile_w4a16_gemv(N=40, K=128, group_size=32, zero_points=True)
    with fw.dual_level():
        c = torch.zeros(3, 40, dtype=BF16, device="cuda")
        fn(c, fw.make_dual(a, t), q, s, z, None, 3, 40)
        got = fw.unpack_dual(c).tangent.double()
    want, mag = t.double() @ weights64(q, s, z).t(), t.double().abs() @ weights64(q, s, z).abs().t()
    assert bool(((got - want).abs() <= 2.0**-8 * 1.01 * want.abs() + 128 * 2.0**-24 * mag).all())  # half a step of bf16, and fp32 sums of 128 terms
