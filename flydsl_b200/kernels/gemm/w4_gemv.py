"""Products of few tokens on 4-bit weights with a scale (and, if wanted, a zero point) per group of inputs: the weight
stream of a decode step at a quarter of its 16-bit size, with 16-bit activations.

    q, s, z = per_group_w4_quant(w, group_size=128, zero_points=True)      # w [N, K]; once
    launch = compile_w4a16_gemv(N=N, K=K, group_size=128, in_dtype="bf16", zero_points=True)
    launch(c, a, q, s, z, bias, M, N, stream)                              # c [>= M, N], a [M, K]; -> None, writes c

    c[m, n] = epilogue(sum_g s[n, g] * sum_{k in g} (q[n, k] - z[n, g]) * a[m, k])

The weights are read as they are stored: ``q`` uint8 [N, K / 2], two codes 0..15 per byte with the even input in the low
half (the packing of ``per_1x32_f4_quant``), ``s`` [N, K / group_size] in the type of the activations, ``z`` uint8
[N, K / group_size] with zero points 0..15; without zero points the codes are signed numbers plus 8.  Group sizes 32, 64
and 128.  ``epilogue``, ``bias`` [N] and ``stream`` are those of ``compile_preshuffle_gemm``; the output has the type of the
activations.  Sums are fp32 and no weight is rounded on the way: code minus zero point is exact, and the scale multiplies the
sum of its group.  Up to 4 tokens the activations of a group are rounded to within 2^-22 of the group's largest magnitude (exact
products and sums of integers); a token that holds an infinity or a NaN gives no finite number, and which of the two
may depend on the number of tokens.  So may the last places of a token's results: up to 4 tokens and from 5 on the sums differ in order.

Any number of tokens runs, in blocks of 64 that each stream the weights; for more than that the 8-bit products
on the tensor core (``compile_preshuffle_gemm``) are the faster ones.  Weights, activations and scales are read in place, on
the stream given; nothing is kept between calls, so a launch can be captured into a CUDA graph.  ``c`` must not overlap the inputs.
As with the other launchers no gradient is recorded.  Where torch has to see the operations (tracing and compilation, dispatch modes, functional
transforms, fake tensors, lazily negated tensors, subclasses with a dispatch of their own, tangents) the launch runs as torch operations on torch's
current stream, with the weights in fp32.
"""

from __future__ import annotations

import os

import torch

from ... import _lib
from ...utils import has_tangent, readable
from .preshuffle_gemm import _stream_handle

_TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP_SIZES = (32, 64, 128)
_ACTIVATIONS = {
    "bias": lambda v: v,
    "bias_relu": torch.relu,
    "bias_silu": torch.nn.functional.silu,
    "bias_gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh"),
}


def per_group_w4_quant(w: torch.Tensor, group_size: int = 128, *, zero_points: bool = False, scale_dtype: torch.dtype | None = None):
    """``(codes, scale, zero)`` of weights [N, K] as torch operations on their device.  Without zero points scale =
    max|w| / 7 over a group and zero is None; with them the group's range, which always holds 0, is spread over 0..15.  The
    codes are the nearest ones under the scale as it is stored (``scale_dtype``, by default w's own 16-bit type, bf16 for
    fp32; it has to hold the scales: fp16 none beyond 65504).  A group of zeros gets scale 1."""
    if not isinstance(w, torch.Tensor) or w.dim() != 2 or not w.dtype.is_floating_point:
        raise ValueError("w must be a two-dimensional tensor of floating-point weights")
    if group_size not in GROUP_SIZES or w.shape[1] % group_size != 0 or w.numel() == 0:
        raise ValueError(f"group_size must be one of {GROUP_SIZES} and divide K = {w.shape[1]}, got {group_size}")
    if scale_dtype is None:
        scale_dtype = w.dtype if w.dtype in _TORCH.values() else torch.bfloat16
    if scale_dtype not in _TORCH.values():
        raise ValueError(f"scale_dtype must be bf16 or fp16, got {scale_dtype}")
    n, k = w.shape
    g = w.detach().float().reshape(n, k // group_size, group_size)
    if zero_points:
        lo, hi = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
        s = ((hi - lo) / 15.0).to(scale_dtype)
    else:
        s = (g.abs().amax(-1) / 7.0).to(scale_dtype)
    s = torch.where(s == 0, torch.ones_like(s), s)
    sf = s.float()
    zero = torch.round(-lo / sf).clamp(0, 15).to(torch.uint8) if zero_points else None
    z = 8.0 if zero is None else zero.float()[..., None]
    q = (torch.round(g / sf[..., None]) + z).clamp(0, 15).to(torch.uint8).reshape(n, k // 2, 2)
    return q[..., 0] | (q[..., 1] << 4), s, zero


def w4_to_f32(codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None) -> torch.Tensor:
    """The weights [N, K] in fp32 that codes, scales and zero points stand for."""
    n, groups = scale.shape
    q = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(n, groups, -1).float()
    return ((q - (8.0 if zero is None else zero.float()[..., None])) * scale.float()[..., None]).reshape(n, -1)


class W4Gemv:
    """The callable returned by :func:`compile_w4a16_gemv`."""

    def __init__(self, N, K, group_size, in_dtype, zero_points, epilogue):
        self.N, self.K, self.group_size, self.in_dtype, self.zero_points, self.epilogue = N, K, group_size, in_dtype, zero_points, epilogue
        self._dt, self._epi = _lib.IN_DTYPES[in_dtype], _lib.EPILOGUES[epilogue]

    def __call__(self, arg_c, arg_a, arg_b, arg_scale_b, arg_zero_b, arg_bias, i32_m, i32_n, stream=None):
        M, n_rt = int(i32_m), int(i32_n)
        if n_rt != self.N:
            raise ValueError(f"N passed at call time ({n_rt}) differs from the N the launcher was built for ({self.N})")
        if M < 0:
            raise ValueError("M must be non-negative")
        if os.environ.get("COMPILE_ONLY") == "1":
            return None  # every variant is built ahead of time
        if M == 0:
            return None
        if self.zero_points and arg_zero_b is None:
            raise ValueError("zero_b is missing: the launcher was built with zero_points=True")
        zero = arg_zero_b if self.zero_points else None
        bias = arg_bias if self._epi else None
        rc = None
        if not torch.compiler.is_compiling():
            s = _stream_handle(stream)
            rc = _lib.ops().w4_gemv(arg_c, arg_a, arg_b, arg_scale_b, zero, bias, M, self.N, self.K, self.group_size, self._dt, self._epi, s)
        if rc is None:
            tensors = (arg_c, arg_a, arg_b, arg_scale_b, zero, bias)
            self._check(*tensors, M)
            if not readable(*tensors) or any(has_tangent(t) for t in tensors if t is not None):
                return self._statements(*tensors, M)
            with _lib.on_device(arg_c.device):
                rc = _lib.load().flyb200_gemv_w4a16(
                    arg_c.data_ptr(), arg_a.data_ptr(), arg_b.data_ptr(), arg_scale_b.data_ptr(), None if zero is None else zero.data_ptr(),
                    None if bias is None else bias.data_ptr(), M, self.N, self.K, self.group_size, self._dt, self._epi, s or None,
                )  # fmt: skip
        if rc:
            _lib.check(rc, "w4a16_gemv")
        return None

    def _statements(self, c, a, b, scale, zero, bias, M):
        groups = self.K // self.group_size
        codes = b.reshape(-1)[: self.N * self.K // 2].view(torch.uint8).reshape(self.N, self.K // 2)
        z = None if zero is None else zero.reshape(-1)[: self.N * groups].reshape(self.N, groups)
        w = w4_to_f32(codes, scale.reshape(-1)[: self.N * groups].reshape(self.N, groups), z)
        v = a.reshape(-1)[: M * self.K].reshape(M, self.K).float() @ w.t()
        if self._epi:
            v = _ACTIVATIONS[self.epilogue](v + bias.reshape(-1)[: self.N].float())
        c.view(-1)[: M * self.N].copy_(v.reshape(-1))

    def _check(self, c, a, b, scale, zero, bias, M):
        t16, groups = _TORCH[self.in_dtype], self.K // self.group_size
        need = [("c", c, M * self.N, t16), ("a", a, M * self.K, t16), ("b", b, self.N * self.K // 2, None), ("scale_b", scale, self.N * groups, t16)]
        if self.zero_points:
            need.append(("zero_b", zero, self.N * groups, torch.uint8))
        if self._epi:
            need.append(("bias", bias, self.N, t16))
        for name, t, n, dtype in need:
            if not isinstance(t, torch.Tensor) or not t.is_cuda or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous CUDA tensor")
            if dtype is None and t.element_size() != 1:
                raise ValueError(f"{name} must be a one-byte tensor, two codes per byte")
            if dtype is not None and t.dtype != dtype:
                raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
            if t.numel() < n:
                raise ValueError(f"{name} holds {t.numel()} elements, the launch needs {n}")
            if t.device != c.device:
                raise ValueError("all tensors must live on the same device")


def compile_w4a16_gemv(*, N, K, group_size=128, in_dtype="bf16", zero_points=False, epilogue="none"):
    """Builder of the launcher ``fn(c, a, b, scale_b, zero_b, bias, M, N, stream)``; ``zero_b`` is ignored without
    ``zero_points``, ``bias`` with epilogue "none"."""
    if in_dtype not in _TORCH:
        raise ValueError(f"in_dtype must be 'bf16' or 'fp16', got {in_dtype!r}")
    if epilogue not in _lib.EPILOGUES:
        raise ValueError(f"epilogue must be none/bias/bias_relu/bias_silu/bias_gelu, got {epilogue!r}")
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size!r}")
    if int(N) <= 0 or int(K) <= 0 or int(K) % group_size != 0:
        raise ValueError(f"N must be positive and K a positive multiple of group_size; got N={N}, K={K}, group_size={group_size}")
    return W4Gemv(int(N), int(K), int(group_size), in_dtype, bool(zero_points), epilogue)


__all__ = ["compile_w4a16_gemv", "per_group_w4_quant", "w4_to_f32"]
