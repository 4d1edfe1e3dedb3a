"""Row operators next to the quantised products: what a layer runs between its projections, with the codes and scales
that the products take as the output.

    y, s, h = rmsnorm_quant(x, weight, 1e-5, residual=h)               # ahead of the gate-up (or QKV) projection
    ...                                                                # c = fp8 GEMM of (y, s)
    a, sa = silu_mul_quant(c)                                          # ahead of the down projection

One kernel each, on the current stream of the input's device; nothing is synchronised and nothing is kept between calls,
so they can be captured into a CUDA graph.  ``quant_dtype`` says what comes out:

``torch.float8_e4m3fn``, ``torch.int8``   codes and one fp32 scale per row ([..., 1]), for ``compile_preshuffle_gemm``.
    scale = rowmax|v| * (1 / qmax) (0 -> 1), code = the nearest to v / scale, ties to even; NaN -> 0 and +-Inf -> +-qmax
    beforehand.  The conventions of ``pertoken_quant``, whose int8 codes truncate toward zero as the reference's do.
``"mxfp8"``   E4M3 codes and E8M0 scale bytes [..., K / 32] as ``per_1x32_f8_quant``; ``shuffle_scale`` takes them on to the
    block-scaled GEMM.  K (``inter``) has to be a multiple of 32.
``None``      the values rounded to the type of x, scale ``None``: for projections on 16-bit activations.

Inputs are CUDA tensors of fp32, fp16 or bf16 whose last dimension is contiguous; rows may lie further apart than they are
long (a slice of a wider tensor).  Anything else raises ``ValueError``, as do inputs that carry a gradient, backward or forward: the
operators have no derivative.  Where torch has to see the operations (tracing and compilation, fake tensors and other subclasses, dispatch
modes, functional transforms, lazily negated tensors) they run as torch operations, with the same results up to the last places.
"""

from __future__ import annotations

import torch

from . import _lib
from .kernels.gemm.mxfp8_preshuffle import per_1x32_f8_quant_torch
from .utils import has_tangent, readable, torch_watches

_X_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_QUANT = {None: _lib.ROWQ_NONE, torch.float8_e4m3fn: _lib.ROWQ_FP8, torch.int8: _lib.ROWQ_INT8, "mxfp8": _lib.ROWQ_MXFP8}


def _code(quant_dtype) -> int:
    q = _QUANT.get(quant_dtype)
    if q is None:
        raise ValueError(f"quant_dtype must be torch.float8_e4m3fn, torch.int8, 'mxfp8' or None, got {quant_dtype!r}")
    return q


def _no_tangent(name: str, t: torch.Tensor) -> None:
    if has_tangent(t):
        raise ValueError(f"{name} carries a tangent, and this operator has no forward derivative")


def _rows(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> tuple[int, int]:
    """(rows, stride between them in elements) of a tensor [..., K] with rows at equal distances."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.layout != torch.strided or t.dtype not in _X_DTYPES or t.dim() < 1:
        raise ValueError(f"{name} must be a CUDA tensor of fp32, fp16 or bf16 with at least one dimension")
    if like is not None and (t.dtype != like.dtype or t.shape != like.shape or t.device != like.device):
        raise ValueError(f"{name} must have the shape, dtype and device of x")
    if torch.is_grad_enabled() and t.requires_grad:
        raise ValueError(f"{name} requires a gradient, and this operator has no backward pass: call it under torch.no_grad()")
    _no_tangent(name, t)
    k = t.shape[-1]
    if k == 0:
        raise ValueError(f"{name} has rows without elements")
    rows = t.numel() // k
    if rows >= 2**31 or k >= 2**30:
        raise ValueError(f"{name} has 2^31 rows or rows of 2^30 elements, or more")
    if k > 1 and t.stride(-1) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    stride, expect = None, None
    for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):  # leading dimensions that are one run of rows
        if size == 1:
            continue
        if stride is None:
            stride, expect = st, st * size
        elif st != expect:
            raise ValueError(f"the rows of {name} must lie at equal distances (strides {tuple(t.stride())})")
        else:
            expect = st * size
    if stride is None or rows == 0:
        stride = k
    if stride < k:
        raise ValueError(f"the rows of {name} overlap (strides {tuple(t.stride())})")
    return rows, stride


def _outputs(x: torch.Tensor, width: int, quant: int):
    shape = x.shape[:-1]
    y_dtype = x.dtype if quant == _lib.ROWQ_NONE else torch.int8 if quant == _lib.ROWQ_INT8 else torch.float8_e4m3fn
    y = torch.empty(*shape, width, dtype=y_dtype, device=x.device)
    if quant == _lib.ROWQ_NONE:
        return y, None
    if quant == _lib.ROWQ_MXFP8:
        if width % 32 != 0:
            raise ValueError(f"MXFP8 blocks need rows of a multiple of 32 values, got {width}")
        return y, torch.empty(*shape, width // 32, dtype=torch.uint8, device=x.device)
    return y, torch.empty(*shape, 1, dtype=torch.float32, device=x.device)


def _span(t: torch.Tensor, rows: int, stride: int) -> tuple[int, int, int, int]:
    """(address, rows, distance, width) in bytes; one row has no distance."""
    e = t.element_size()
    return t.data_ptr(), rows, stride * e if rows > 1 else 0, t.shape[-1] * e


def _share(a, b) -> bool:
    """Whether two runs of rows (`_span`) share memory.  At one distance, or where one is a single row, that is decided row by row: other columns
    of one buffer are apart.  At two distances the address ranges decide."""
    (a0, ra, sa, wa), (b0, rb, sb, wb) = a, b
    if ra == 0 or rb == 0 or b0 >= a0 + (ra - 1) * sa + wa or a0 >= b0 + (rb - 1) * sb + wb:
        return False
    step = sa or sb
    if not step or (sa and sb and sa != sb):
        return True
    d = (b0 - a0) % step  # from a row of a to the next start of a row of b
    return d < wa or d + wb > step


def _quantised(v: torch.Tensor, dtype: torch.dtype, quant: int):
    """The outputs of fp32 values as torch operations."""
    if quant == _lib.ROWQ_NONE:
        return v.to(dtype), None
    if quant == _lib.ROWQ_MXFP8:
        return per_1x32_f8_quant_torch(v)
    qmax = 127.0 if quant == _lib.ROWQ_INT8 else 448.0
    v = torch.nan_to_num(v, nan=0.0, posinf=qmax, neginf=-qmax)
    s = v.abs().amax(dim=-1, keepdim=True) * (1.0 / qmax)
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (v / s).clamp(-qmax, qmax)
    return (q.round().to(torch.int8) if quant == _lib.ROWQ_INT8 else q.to(torch.float8_e4m3fn)), s


def rmsnorm_quant(x, weight, eps=1e-6, *, residual=None, quant_dtype=torch.float8_e4m3fn, residual_out=None):
    """``(y, scale, h)``: ``h = x + residual`` rounded to x's type, and the codes and scales of
    ``h * weight / sqrt(mean(h^2) + eps)`` over the last dimension, statistics and values in fp32 (squares beyond its range
    are infinite, and such a row is all zeros; squares below it are 0, and without ``eps`` the values of such a row are infinite, or NaN where
    they are 0).  ``weight`` [K] is of x's type or fp32.  Without a residual ``h`` is None.
    ``residual_out`` receives ``h`` instead of a new tensor; it may be ``residual`` (or ``x``) itself, for an update in place,
    and must not overlap them otherwise."""
    quant = _code(quant_dtype)
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if residual is None and residual_out is not None:
        raise ValueError("residual_out without a residual")
    if not torch.compiler.is_compiling():
        r = _lib.ops().rmsnorm_quant(x, weight, residual, residual_out, eps, quant)
        if type(r) is tuple:
            return r
        if type(r) is int:
            _lib.check(r, "rmsnorm_quant")
    # not the common form: the same step by step, with what is wrong by name
    rows, stride = _rows("x", x)
    k = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.device != x.device or weight.dim() != 1 or weight.numel() != k or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous tensor [{k}] on the device of x")
    if weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"weight must be {x.dtype} or fp32, got {weight.dtype}")
    if torch.is_grad_enabled() and weight.requires_grad:
        raise ValueError("weight requires a gradient, and this operator has no backward pass: call it under torch.no_grad()")
    _no_tangent("weight", weight)
    watched = torch_watches(x, residual, residual_out) or not readable(weight)
    r_stride = h_stride = 0
    h = None
    if residual is not None:
        r_stride = _rows("residual", residual, x)[1]
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual_out is None else residual_out
        h_stride = _rows("residual_out", h, x)[1]
        if residual_out is not None and not watched:
            out = _span(h, rows, h_stride)
            for name, span in (("x", _span(x, rows, stride)), ("residual", _span(residual, rows, r_stride))):
                if span != out and _share(out, span):
                    raise ValueError(f"residual_out overlaps {name} without being the same tensor")
            if _share(out, _span(weight, 1, k)):
                raise ValueError("residual_out overlaps weight")
    y, scale = _outputs(x, k, quant)
    if rows == 0:
        return y, scale, h
    if watched:
        if residual is not None:
            x = (x.float() + residual.float()).to(x.dtype)
            h = x if residual_out is None else residual_out.copy_(x)
        v = x.float()
        v = v * torch.rsqrt(v.square().mean(dim=-1, keepdim=True) + eps) * weight.float()
        return *_quantised(v, x.dtype, quant), h
    with _lib.on_device(x.device):
        rc = _lib.load().flyb200_rmsnorm_quant(
            y.data_ptr(), None if scale is None else scale.data_ptr(), None if h is None else h.data_ptr(), x.data_ptr(),
            None if residual is None else residual.data_ptr(), weight.data_ptr(), rows, k, stride, r_stride, h_stride, eps,
            _X_DTYPES[x.dtype], int(weight.dtype == torch.float32), quant, _lib.current_stream(x.device),
        )  # fmt: skip
    _lib.check(rc, "rmsnorm_quant")
    return y, scale, h


def silu_mul_quant(x, *, quant_dtype=torch.float8_e4m3fn):
    """``(y, scale)``: codes and scales of ``silu(gate) * up`` for ``x = [..., 2 * inter]``, of every row the gate values
    first (the row order of a gate-up projection's weights), values in fp32 (to 2^-20 of themselves, for every gate)."""
    quant = _code(quant_dtype)
    if not torch.compiler.is_compiling():
        r = _lib.ops().silu_mul_quant(x, quant)
        if type(r) is tuple:
            return r
        if type(r) is int:
            _lib.check(r, "silu_mul_quant")
    rows, stride = _rows("x", x)
    if x.shape[-1] % 2 != 0:
        raise ValueError(f"x needs an even last dimension (gate and up values), got {x.shape[-1]}")
    inter = x.shape[-1] // 2
    y, scale = _outputs(x, inter, quant)
    if rows == 0:
        return y, scale
    if torch_watches(x):
        g, u = x.float().chunk(2, dim=-1)
        return _quantised(g / (1.0 + torch.exp(-g)) * u, x.dtype, quant)
    with _lib.on_device(x.device):
        rc = _lib.load().flyb200_silu_mul_quant(y.data_ptr(), None if scale is None else scale.data_ptr(), x.data_ptr(), rows, inter, stride,
                                                _X_DTYPES[x.dtype], quant, _lib.current_stream(x.device))
    _lib.check(rc, "silu_mul_quant")
    return y, scale


__all__ = ["rmsnorm_quant", "silu_mul_quant"]
