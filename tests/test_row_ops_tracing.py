"""rmsnorm_quant and silu_mul_quant where torch has to see the operations: fake tensors, tracing, compilation, subclasses and lazily negated
tensors give what the formulas give; tangents are refused, as gradients are."""

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from flydsl_b200 import _lib, host_statements, rmsnorm_quant, silu_mul_quant

FP8 = torch.float8_e4m3fn
QUANTS = [FP8, torch.int8, "mxfp8", None]
IDS = ["fp8", "int8", "mxfp8", "none"]


def expect(quant, rows, k, dtype):
    scale = {None: None, "mxfp8": ((rows, k // 32), torch.uint8)}.get(quant, ((rows, 1), torch.float32))
    return ((rows, k), {None: dtype, torch.int8: torch.int8}.get(quant, FP8)), scale


@pytest.mark.parametrize("quant", QUANTS, ids=IDS)
def test_fake_cuda_tensors(quant):
    with FakeTensorMode():
        x = torch.empty(8, 256, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(256, device="cuda", dtype=torch.float32)
        out = torch.empty_like(x)
        got = [rmsnorm_quant(x, w, residual=x, quant_dtype=quant), rmsnorm_quant(x, w, residual=x, residual_out=out, quant_dtype=quant)]
        gated = silu_mul_quant(x, quant_dtype=quant)
        assert got[1][2] is out and rmsnorm_quant(x, w, quant_dtype=quant)[2] is None
        with pytest.raises(ValueError, match="weight must be"):
            rmsnorm_quant(x, w[:8], quant_dtype=quant)
    describe = lambda t: None if t is None else (tuple(t.shape), t.dtype)  # noqa: E731
    for y, s, h in got:
        assert (describe(y), describe(s)) == expect(quant, 8, 256, torch.bfloat16) and describe(h) == ((8, 256), torch.bfloat16)
    assert tuple(map(describe, gated)) == expect(quant, 8, 128, torch.bfloat16)


@pytest.mark.parametrize("quant", QUANTS, ids=IDS)
def test_a_trace_holds_operations(quant):
    """Of fake CUDA tensors, on any machine: what the graph returns is computed from its inputs."""
    with FakeTensorMode(allow_non_fake_inputs=True):
        x, r, w = torch.empty(8, 256, device="cuda"), torch.empty(8, 256, device="cuda"), torch.empty(256, device="cuda")
        graphs = [make_fx(lambda x, w, r: rmsnorm_quant(x, w, residual=r, quant_dtype=quant))(x, w, r), make_fx(lambda x: silu_mul_quant(x, quant_dtype=quant))(x)]
    for graph in graphs:
        inputs = [n for n in graph.graph.nodes if n.op == "placeholder"]
        reached, todo = set(), list(next(n for n in graph.graph.nodes if n.op == "output").all_input_nodes)
        assert not any("empty" in str(n.target) for n in todo)
        while todo:
            n = todo.pop()
            if n not in reached:
                reached.add(n)
                todo += n.all_input_nodes
        assert all(n in reached for n in inputs)


def test_eagerness_without_the_host_extension():
    """The Python statement of the question agrees with the extension's."""

    class Sub(torch.Tensor):
        pass

    ops, x = _lib.ops(), torch.zeros(4, 4)
    for t in (x, torch.nn.Parameter(x), x.as_subclass(Sub), torch._neg_view(x), torch.zeros(2, dtype=torch.complex64).conj(), 3, None):
        assert ops.eager(t) == host_statements.eager(t)
    assert host_statements.eager(x) and not host_statements.eager(torch._neg_view(x))
    seen = []

    def look(t):
        seen.append((ops.eager(t), host_statements.eager(t)))
        return t + 1

    make_fx(look)(x)
    torch.jit.trace(look, (x,), check_trace=False)
    torch.func.vmap(look)(x)
    torch.func.functionalize(look)(x)
    with FakeTensorMode():
        look(torch.empty(3))
    assert seen and not any(a or b for a, b in seen)




@pytest.mark.gpu
@pytest.mark.parametrize("quant", QUANTS, ids=IDS)
def test_traced_and_compiled(quant):
    from tests.test_row_ops_gpu import SILU_REL, check, make, norm64, norm_rel, silu64

    x, other, r = (make(16, 256, torch.bfloat16, i) for i in range(3))
    w = make(1, 256, torch.bfloat16, 4)[0]
    norm, gated = (lambda x, r: rmsnorm_quant(x, w, 1e-5, residual=r, quant_dtype=quant)), (lambda x: silu_mul_quant(x, quant_dtype=quant))
    if quant is None:  # a trace holds tensors only
        norm, gated = (lambda x, r: rmsnorm_quant(x, w, 1e-5, residual=r, quant_dtype=None)[::2]), (lambda x: silu_mul_quant(x, quant_dtype=None)[0])
    forms = [lambda f, *a: make_fx(f)(*a), lambda f, *a: torch.compile(f, backend="eager", fullgraph=True)]
    if quant != "mxfp8":  # torch.jit.trace cannot record a view of another type, which the scale bytes need: it raises
        forms.append(lambda f, *a: torch.jit.trace(f, a, check_trace=False))
    for form in forms:
        got = form(norm, x, r)(other, r)
        v, h = norm64(other, w, 1e-5, r)
        assert torch.equal(got[-1], h)
        check(got[0], None if quant is None else got[1], v, quant, norm_rel(256))
        got = form(gated, x)(other)
        check(*((got, None) if quant is None else got), silu64(other), quant, SILU_REL)


@pytest.mark.gpu
@pytest.mark.parametrize("quant", QUANTS, ids=IDS)
@pytest.mark.parametrize("extension", [True, False])
def test_lazy_negation_and_subclasses(quant, extension, monkeypatch):
    from tests.test_row_ops_gpu import SILU_REL, check, make, norm64, norm_rel, silu64

    class Sub(torch.Tensor):
        pass

    if not extension:
        monkeypatch.setattr(_lib, "_ops", host_statements)
    x, r, w = make(16, 256, torch.float16, 5), make(16, 256, torch.float16, 6), make(1, 256, torch.float16, 7)[0]
    neg = torch._neg_view
    for args, plain in (((neg(x), w, r), (-x, w, r)), ((x, neg(w), r), (x, -w, r)), ((x, w, neg(r)), (x, w, -r)), ((x.as_subclass(Sub), w, r), (x, w, r))):
        y, s, h = rmsnorm_quant(args[0], args[1], 1e-5, residual=args[2], quant_dtype=quant)
        v, h64 = norm64(plain[0], plain[1], 1e-5, plain[2])
        assert torch.equal(h, h64) and type(y) is type(args[0])
        check(y, s, v, quant, norm_rel(256))
    kept = r.clone()
    y, s, h = rmsnorm_quant(x, w, 1e-5, residual=neg(kept), residual_out=neg(kept), quant_dtype=quant)  # the negated view receives the sum
    assert torch.equal(-kept, norm64(x, w, 1e-5, -r)[1]) and torch.equal(h, -kept)
    check(y, s, norm64(x, w, 1e-5, -r)[0], quant, norm_rel(256))
    y, s = silu_mul_quant(neg(x), quant_dtype=quant)
    check(y, s, silu64(-x), quant, SILU_REL)


@pytest.mark.gpu
@pytest.mark.parametrize("extension", [True, False])
def test_weights_of_a_class_of_their_own_stay_on_the_kernel(extension, monkeypatch):
    from flydsl_b200 import row_ops
    from tests.test_row_ops_gpu import make

    class Weight(torch.nn.Parameter):
        pass

    if not extension:
        monkeypatch.setattr(_lib, "_ops", host_statements)
    x, w = make(16, 256, torch.bfloat16, 9), make(1, 256, torch.bfloat16, 10)[0]
    want = rmsnorm_quant(x, w)
    monkeypatch.setattr(row_ops, "_quantised", None)  # not called
    got = rmsnorm_quant(x, w.as_subclass(Weight))
    assert type(got[0]) is torch.Tensor and torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_tangents_are_refused():
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with fw.dual_level():
        dual, dual_w = fw.make_dual(x, x), fw.make_dual(w, w)
        for call in (lambda: rmsnorm_quant(dual, w), lambda: rmsnorm_quant(x, dual_w), lambda: rmsnorm_quant(x, w, residual=dual), lambda: silu_mul_quant(dual)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        rmsnorm_quant(x, w)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda t: silu_mul_quant(t, quant_dtype=None)[0], (x,), (x,))
    with pytest.raises(ValueError, match="gradient"):
        torch.func.grad(lambda t: silu_mul_quant(t, quant_dtype=None)[0].sum())(x)


@pytest.mark.gpu
@pytest.mark.parametrize("quant", QUANTS, ids=IDS)
def test_over_a_batch_of_a_transform(quant):
    from tests.test_row_ops_gpu import SILU_REL, check, make, silu64

    x = make(24, 256, torch.bfloat16, 8)
    f = (lambda t: silu_mul_quant(t, quant_dtype=None)[0]) if quant is None else (lambda t: silu_mul_quant(t, quant_dtype=quant))
    if quant == "mxfp8":  # vmap has no rule for the view of another type that the scale bytes need
        with pytest.raises(RuntimeError, match="view"):
            torch.func.vmap(f)(x.view(4, 6, 256))
        return
    got = torch.func.vmap(f)(x.view(4, 6, 256))
    y, s = (got, None) if quant is None else got
    check(y.reshape(24, 128), None if s is None else s.reshape(24, -1), silu64(x), quant, SILU_REL)
