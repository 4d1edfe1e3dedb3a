"""The operators around the quantised products of a dense layer, as cases that can be timed and compared.

``norm``  residual addition, root-mean-square norm and the quantisation of its output in one call (``rmsnorm_quant``):
          what a layer runs ahead of its first projection.  Codes per token (fp8, int8), in MXFP8 blocks, or no
          quantisation for a projection on 16-bit activations.
``silu``  the gated activation ``silu(gate) * up`` and the quantisation of its output (``silu_mul_quant``): what a layer
          runs between its gate-up and down projections.
``w4``    a projection of few tokens on 4-bit weights with a scale (and zero point) per group of inputs
          (``compile_w4a16_gemv``).

``run`` computes them as plain torch operations, or, where ``own`` is true, through the package's entry points.
Sizes are those of the benchmark's configurations and of the tests, and ragged ones.
"""

import math

import torch

own = False

EPS = 1e-5
X_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = torch.float8_e4m3fn
QMAX = {"fp8": 448.0, "int8": 127.0}


def _norm(name, rows, k, x="bf16", quant="fp8", residual=True):
    return dict(name=name, kind="norm", rows=rows, k=k, x=x, quant=quant, residual=residual)


def _silu(name, rows, inter, x="bf16", quant="fp8"):
    return dict(name=name, kind="silu", rows=rows, inter=inter, x=x, quant=quant)


def _w4(name, m, n, k, x="bf16", group=128, zeros=False, epilogue="none"):
    return dict(name=name, kind="w4", m=m, n=n, k=k, x=x, group=group, zeros=zeros, epilogue=epilogue)


def listed():
    return [
        # one token of a decode step, ahead of an fp8 projection: the smallest call
        _norm("norm_fp8_1x8192_residual", 1, 8192),
        # a decode batch ahead of a projection on 4-bit weights, which takes 16-bit activations
        _norm("norm_bf16_32x8192_residual", 32, 8192, quant="none"),
        # the first norm of a ragged prefill chunk, which has no residual yet, ahead of int8 projections
        _norm("norm_int8_997x5120", 997, 5120, "fp16", "int8", False),
        # ahead of a block-scaled projection at the size of the tests
        _norm("norm_mxfp8_1024x8192_residual", 1024, 8192, quant="mxfp8"),
        # prefill of the widest configuration
        _norm("norm_fp8_16384x8192_residual", 16384, 8192),
        # a decode batch between the gate-up and down projections
        _silu("silu_fp8_32x28672", 32, 28672),
        # a ragged batch, no size a multiple of a tile
        _silu("silu_int8_515x1408", 515, 1408, "fp16", "int8"),
        # prefill of the widest configuration: the largest pass over memory
        _silu("silu_fp8_8192x28672", 8192, 28672),
        # one token through a square projection
        _w4("w4_bf16_1x8192x8192", 1, 8192, 8192),
        # a ragged output, few rows, the finest groups, fused bias
        _w4("w4_bf16_7x1040x2048_g32_bias", 7, 1040, 2048, "bf16", 32, True, "bias"),
        # a decode batch through the wide up-projection, weights with zero points
        _w4("w4_fp16_16x28672x8192_zeros", 16, 28672, 8192, "fp16", 128, True),
        # the largest decode batch through the down-projection
        _w4("w4_bf16_64x8192x28672_g64", 64, 8192, 28672, "bf16", 64),
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(-(-lo // step) * step, min(hi // step * step, int(round(v / step)) * step))


MOST_VALUES = 16384 * 8192  # of a norm; of an activation's output 8192 * 28672


def draw(rng):
    kind = rng.choice(["norm", "silu", "w4"])
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        return {k: v for k, v in _w4("", _log_int(rng, 1, 64), _log_int(rng, 256, 28672, rng.choice([1, 8, 64])),
                                     _log_int(rng, 512, 8192, group), rng.choice(["bf16", "fp16"]), group, rng.choice([True, False]),
                                     rng.choice(["none", "none", "bias", "bias_silu"])).items() if k != "name"}
    x = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    quant = rng.choice(["fp8", "int8", "mxfp8", "none"])
    width = _log_int(rng, 256, 16384, 32 if quant == "mxfp8" else rng.choice([1, 8, 128]))
    most = MOST_VALUES // 2 if x == "fp32" else MOST_VALUES
    rows = _log_int(rng, 1, max(1, min(16384, most // width)))
    case = _norm("", rows, width, x, quant, rng.choice([True, False])) if kind == "norm" else _silu("", rows, width, x, quant)
    return {k: v for k, v in case.items() if k != "name"}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    t = X_TYPES[case["x"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    if case["kind"] == "norm":
        rows, k = case["rows"], case["k"]
        # a residual stream has a few channels that are much larger than the others
        channel = torch.exp(0.5 * normal(k))
        return dict(case=case, x=normal(rows, k).to(t), weight=(1.0 + 0.2 * normal(k)).to(t),
                    residual=(normal(rows, k) * channel * 4.0).to(t) if case["residual"] else None)
    if case["kind"] == "silu":
        return dict(case=case, x=(normal(case["rows"], 2 * case["inter"]) * 1.5).to(t))
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8)  # two codes a byte, the even input in the low half
    scale = (0.01 * torch.exp(0.3 * normal(n, k // group))).to(t)
    zero = torch.randint(4, 12, (n, k // group), generator=g, device=dev, dtype=torch.uint8) if case["zeros"] else None
    bias = normal(n).to(t) if case["epilogue"] != "none" else None
    return dict(case=case, a=normal(m, k).to(t), codes=codes, scale=scale, zero=zero, bias=bias, c=torch.empty(m, n, dtype=t, device=dev))


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["kind"] == "norm":
        return _plain_norm(state, case)
    if case["kind"] == "silu":
        g, u = state["x"].float().chunk(2, dim=-1)
        return _plain_quant(g / (1.0 + torch.exp(-g)) * u, case["quant"], state["x"].dtype)
    return _plain_w4(state, case)


def _own(state):
    from flydsl_b200 import compile_w4a16_gemv, rmsnorm_quant, silu_mul_quant

    case = state["case"]
    if case["kind"] == "w4":
        fn = state.get("launch")
        if fn is None:  # built once, as a program does
            fn = state["launch"] = compile_w4a16_gemv(N=case["n"], K=case["k"], group_size=case["group"], in_dtype=case["x"],
                                                      zero_points=case["zeros"], epilogue=case["epilogue"])
        fn(state["c"], state["a"], state["codes"], state["scale"], state["zero"], state["bias"], case["m"], case["n"],
           torch.cuda.current_stream())
        return {"c": state["c"]}
    quant = {"fp8": FP8, "int8": torch.int8, "mxfp8": "mxfp8", "none": None}[case["quant"]]
    if case["kind"] == "norm":
        y, s, h = rmsnorm_quant(state["x"], state["weight"], EPS, residual=state["residual"], quant_dtype=quant)
        return _values(y, s) | ({"residual": h} if case["residual"] else {})
    return _values(*silu_mul_quant(state["x"], quant_dtype=quant))


def _values(y, s):
    """Codes and scales as the values they stand for: integer codes as exact bf16 numbers, E8M0 bytes as powers of two."""
    out = {"y": y.to(torch.bfloat16) if y.dtype == torch.int8 else y}
    if s is not None:
        out["scale"] = s.view(torch.float8_e8m0fnu) if s.dtype == torch.uint8 else s
    return out


def _plain_norm(state, case):
    x, out = state["x"], {}
    if case["residual"]:
        x = (x.float() + state["residual"].float()).to(x.dtype)
        out["residual"] = x
    h = x.float()
    n = h * torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + EPS) * state["weight"].float()
    return _plain_quant(n, case["quant"], x.dtype) | out


def _plain_quant(v, quant, dtype):
    """fp32 values [rows, K] as codes and scales; a code is the nearest one, ties to the even one."""
    if quant == "none":
        return {"y": v.to(dtype)}
    if quant == "mxfp8":  # a power of two per 32 values: the exponent of max / 448, one higher from a mantissa of 1.5 on
        b = v.reshape(v.shape[0], -1, 32)
        mantissa, e = torch.frexp(b.abs().amax(dim=-1).clamp_min(1e-30) * (1.0 / 448.0))
        e = e - 1 + (mantissa >= 0.75).int()
        y = (b * torch.exp2(-e.float())[..., None]).clamp(-448.0, 448.0).to(FP8).reshape(v.shape)
        return {"y": y, "scale": (e + 127).clamp(0, 254).to(torch.uint8).view(torch.float8_e8m0fnu)}
    s = v.abs().amax(dim=-1, keepdim=True) * (1.0 / QMAX[quant])
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (v / s).clamp(-QMAX[quant], QMAX[quant])
    return {"y": q.to(FP8) if quant == "fp8" else torch.round(q).to(torch.bfloat16), "scale": s}


def _plain_w4(state, case):
    codes, n, k = state["codes"], case["n"], case["k"]
    q = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(n, k // case["group"], case["group"]).float()
    zero = 8.0 if state["zero"] is None else state["zero"].float()[..., None]
    w = ((q - zero) * state["scale"].float()[..., None]).reshape(n, k)
    c = state["a"].float() @ w.t()
    if state["bias"] is not None:
        c = c + state["bias"].float()
    if case["epilogue"] == "bias_silu":
        c = c / (1.0 + torch.exp(-c))
    return {"c": c.to(state["c"].dtype)}


def work(case):
    """Inputs read once and outputs written once."""
    e = X_TYPES[case["x"]].itemsize
    if case["kind"] == "w4":
        m, n, k, groups = case["m"], case["n"], case["k"], case["k"] // case["group"]
        return {"bytes": n * k // 2 + n * groups * (e + (1 if case["zeros"] else 0)) + e * m * (n + k) + (e * n if case["epilogue"] != "none" else 0),
                "flops": 2.0 * m * n * k}
    rows = case["rows"]
    width = case["k"] if case["kind"] == "norm" else case["inter"]
    code = {"none": e, "fp8": 1, "int8": 1, "mxfp8": 1}[case["quant"]]
    scales = {"none": 0, "fp8": 4 * rows, "int8": 4 * rows, "mxfp8": rows * width // 32}[case["quant"]]
    if case["kind"] == "norm":
        return {"bytes": rows * width * (e * (3 if case["residual"] else 1) + code) + scales + e * width, "flops": 6.0 * rows * width}
    return {"bytes": rows * width * (2 * e + code) + scales, "flops": 8.0 * rows * width}


def exact(case, seed):
    """The operators by their definition in float64: codes are the nearest ones to the float64 quotients."""
    state = prepare(case, seed)
    if case["kind"] == "w4":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        w = torch.empty(n, k, dtype=torch.float64, device=state["a"].device)
        w[:, 0::2], w[:, 1::2] = state["codes"] % 16, state["codes"] // 16
        w = w.view(n, k // group, group)
        w -= 8 if state["zero"] is None else state["zero"].unsqueeze(2)
        w *= state["scale"].unsqueeze(2)
        c = torch.matmul(w.view(n, k), state["a"].double().t()).t()
        if case["epilogue"] != "none":
            c = c + state["bias"].double()
        return {"c": c * torch.sigmoid(c) if case["epilogue"] == "bias_silu" else c}
    x, out = state["x"], {}
    if case["kind"] == "norm":
        if case["residual"]:
            x = torch.add(x.double(), state["residual"].double()).to(x.dtype)  # the sum of two such numbers, rounded once
            out["residual"] = x.double()
        h = x.double()
        v = h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / case["k"] + EPS) * state["weight"].double()
    else:
        v = x[:, : case["inter"]].double()
        v = v * torch.sigmoid(v) * x[:, case["inter"] :].double()
    quant = case["quant"]
    if quant == "none":
        return {"y": v} | out
    if quant == "mxfp8":
        blocks = v.view(case["rows"], -1, 32)
        top = blocks.abs().max(dim=2).values.clamp(min=1e-30) / 448
        e = torch.floor(torch.log2(top))
        e += top >= 1.5 * torch.pow(2.0, e)
        scale = torch.pow(2.0, e)
        return {"y": _nearest_e4m3(blocks / scale.unsqueeze(2)).view(v.shape), "scale": scale} | out
    scale = v.abs().max(dim=1, keepdim=True).values / QMAX[quant]
    scale[scale == 0] = 1
    q = v / scale
    return {"y": _nearest_e4m3(q) if quant == "fp8" else torch.round(q), "scale": scale} | out


def _nearest_e4m3(q):
    """Nearest e4m3 number of each float64 value, ties to even: steps of 2^(exponent - 3), from 2^-9 on."""
    step = torch.pow(2.0, torch.floor(torch.log2(q.abs().clamp(min=2.0**-6))) - 3)
    return (torch.round(q / step) * step).clamp(-448, 448)
