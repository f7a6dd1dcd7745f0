"""Linear layers in 8-bit floating point, as timed cases.

Activations are held as e4m3 codes with a scale for each row's 128 columns, a
weight as e4m3 codes with a scale for each block of 128 x 128.  Scales are powers
of two, the smallest s >= 2^-110 with amax <= 448 s, kept as their biased exponent
(one byte, the e8m0 format); codes and scales of the cases are returned as the
numbers that they stand for.  The kinds:

  quantize  activations to codes and scales: what attention gives, before its
            output projection
  weight    a weight to codes and scales, when a model is loaded
  norm      root-mean-square norm of x, or of the residual stream with x added to
            it, as codes and scales for the projections behind it
  linear    x weight^T of the two, with a bias or the residual's addition
  gate      silu(x gate^T) (x up^T), as codes and scales for the down projection

Tensors live on the "gcu" device; the plain forms see the same memory through
torch's own device.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
GROUP = 128
LEAST = -110  # the smallest scale is 2 ** LEAST
EPS = 1e-6


def listed():
    named = {
        # a decode step of one sequence, before the output projection: latency
        "quantize_token": {"kind": "quantize", "m": 1, "k": 4096, "dtype": "bf16", "wide": 0},
        # a long prompt's FFN activations, columns of a wider tensor
        "quantize_prompt": {"kind": "quantize", "m": 6011, "k": 11008, "dtype": "f16", "wide": 11008},
        # a small projection when a model is loaded, its sizes no multiples of a block
        "weight_odd": {"kind": "weight", "n": 1000, "k": 1500, "dtype": "f32"},
        # an FFN weight
        "weight_ffn": {"kind": "weight", "n": 11008, "k": 4096, "dtype": "bf16"},
        # a decode step of 8 sequences
        "norm_decode": {"kind": "norm", "m": 8, "k": 4096, "dtype": "bf16", "residual": True},
        # four prompts of 2048 tokens
        "norm_prompt": {"kind": "norm", "m": 8192, "k": 4096, "dtype": "bf16", "residual": True},
        # one token through an attention projection: the smallest product
        "linear_token": {"kind": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16",
                         "bias": False, "residual": False},
        # the down projection of a decode step of 24 sequences
        "linear_decode": {"kind": "linear", "m": 24, "n": 4096, "k": 11008, "dtype": "bf16",
                          "bias": False, "residual": True},
        # a piece of a prompt, with a bias, in f16
        "linear_chunk": {"kind": "linear", "m": 777, "n": 4096, "k": 4096, "dtype": "f16",
                         "bias": True, "residual": False},
        # the down projection of four prompts
        "linear_prompt": {"kind": "linear", "m": 8192, "n": 4096, "k": 11008, "dtype": "bf16",
                          "bias": False, "residual": True},
        # the gate and up projections of a decode step of 8 sequences
        "gate_decode": {"kind": "gate", "m": 8, "n": 11008, "k": 4096},
        # the same of two prompts
        "gate_prompt": {"kind": "gate", "m": 4096, "n": 11008, "k": 4096},
    }
    return [{"name": n, **c} for n, c in named.items()]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi):
    """A feature count: of a model (a multiple of 128 or 16), or any."""
    n, step = _log(rng, lo, hi), rng.choice([128, 128, 16, 1])
    return max(step, n // step * step)


def draw(rng):
    kind = rng.choice(["quantize", "quantize", "weight", "norm", "norm", "linear", "linear",
                       "linear", "linear", "gate", "gate"])
    c, k = {"kind": kind}, _width(rng, 64, 11008)
    if kind in ("linear", "gate"):
        m = rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192)])
        n = _width(rng, 64, 32000 if kind == "linear" else 11008)
        most = 3.6e11 if kind == "linear" else 1.8e11
        c.update(m=max(1, min(m, int(most / n / k))), n=n, k=k)
        if kind == "linear":
            c.update(dtype=rng.choice(["bf16", "bf16", "f16"]), bias=rng.random() < 0.3,
                     residual=rng.random() < 0.4)
    elif kind == "weight":
        c.update(n=_width(rng, 64, 11008), k=k, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    else:
        c.update(m=_log(rng, 1, 8192), k=k, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
        if kind == "norm":
            c["residual"] = rng.random() < 0.7
        else:
            c["wide"] = rng.choice([0, 0, c["k"]])
    return c


def _scale_byte(amax):
    """The exponent byte of the smallest power of two s >= 2^LEAST with amax <= 448 s."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=LEAST)
    return (torch.where(amax > 0, e, torch.full_like(e, LEAST)) + 127).to(torch.uint8)


def _two_to(byte, dtype):
    return torch.ldexp(torch.ones((), dtype=dtype, device=byte.device), byte.int() - 127)


def _blocks(n):
    return -(-n // GROUP)


def _fill(x, rows, columns):
    """x with zeros behind it up to whole multiples."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % columns, 0, -x.shape[0] % rows))


def _quantized(x, rows):
    """Codes and scale bytes of x [m, k], a scale for each `rows` x GROUP of it."""
    m, k = x.shape
    parts = _fill(x, rows, GROUP)
    parts = parts.view(-1, rows, parts.shape[1] // GROUP, GROUP)
    byte = _scale_byte(parts.abs().amax((1, 3)))
    codes = (parts / _two_to(byte, x.dtype)[:, None, :, None]).to(E4M3)
    return codes.view(torch.uint8).flatten(2).flatten(0, 1)[:m, :k], byte


def _value(codes, byte, rows, dtype=torch.float32):
    """The numbers that codes [m, k] with these scales stand for."""
    scale = _two_to(byte, dtype).repeat_interleave(rows, 0).repeat_interleave(GROUP, 1)
    return codes.view(E4M3).to(dtype) * scale[: codes.shape[0], : codes.shape[1]]


def _inputs(c, seed):
    """The case's inputs on torch's own device."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def tokens(m, k):
        """Some channels are larger than others, and a batch ends with empty rows."""
        x = normal(m, k) * torch.exp(0.7 * normal(k))
        x[m - m // 50:] = 0
        return x

    dt, s = DTYPES.get(c.get("dtype")), {}
    if c["kind"] == "quantize":
        s["x"] = torch.cat([tokens(c["m"], c["k"]), tokens(c["m"], c["wide"])], 1).to(dt)
    elif c["kind"] == "weight":
        s["w"] = (0.02 * normal(c["n"], c["k"])).to(dt)
    elif c["kind"] == "norm":
        s["x"] = tokens(c["m"], c["k"]).to(dt)
        s["weight"] = (1 + 0.1 * normal(c["k"])).to(dt)
        if c["residual"]:
            s["residual"] = (3 * tokens(c["m"], c["k"])).to(dt)
    else:
        s["x"], s["x_scale"] = _quantized(tokens(c["m"], c["k"]), 1)
        for n in ("w",) if c["kind"] == "linear" else ("w_gate", "w_up"):
            s[n], s[n + "_scale"] = _quantized(0.02 * normal(c["n"], c["k"]), GROUP)
        if c.get("bias"):
            s["bias"] = normal(c["n"]).to(dt)
        if c.get("residual"):
            s["residual"] = (3 * tokens(c["m"], c["n"])).to(dt)
    return s


class _Memory:
    """A gcu tensor's memory, for torch's own device to take up."""

    def __init__(self, t):
        kind = {torch.float32: "<f4", torch.uint8: "|u1"}.get(t.dtype, "<i2")
        self.t, self.__cuda_array_interface__ = t, {
            "shape": tuple(t.shape), "typestr": kind, "data": (t.data_ptr(), False), "version": 2}
        if not t.is_contiguous():
            self.__cuda_array_interface__["strides"] = tuple(n * t.itemsize for n in t.stride())


def _seen(t):
    x = torch.as_tensor(_Memory(t), device="cuda")
    return x if x.dtype == t.dtype else x.view(t.dtype)


def prepare(case, seed):
    root = os.path.join(os.getcwd(), "torch-gcu_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import torch_gcu  # noqa: F401  (registers the device)

    state = {"case": dict(case), "gcu": {}, "seen": {}}
    for n, x in _inputs(case, seed).items():
        codes = case["kind"] in ("linear", "gate") and n in ("x", "w", "w_gate", "w_up")
        # rows of codes begin at multiples of 16 bytes, as the quantising operators leave them
        width = -(-x.shape[-1] // 16) * 16 if codes else x.shape[-1]
        t = torch.empty(x.shape[:-1] + (width,), dtype=x.dtype, device="gcu")
        t = t[..., : x.shape[-1]]
        state["gcu"][n], state["seen"][n] = t, _seen(t)
        state["seen"][n].copy_(x)
    if case["kind"] == "quantize":
        for side in ("gcu", "seen"):
            state[side]["x"] = state[side]["x"][:, : case["k"]]
    torch.cuda.synchronize()
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    c, s = state["case"], state["gcu"]
    eff = torch.gcu.efficient
    if c["kind"] == "quantize":
        return _held(*eff.fp8_quantize(s["x"]))
    if c["kind"] == "weight":
        return _held(*eff.fp8_quantize_weight(s["w"]))
    if c["kind"] == "norm":
        y, total = eff.rms_norm_fp8(s["x"], s["weight"], EPS, residual=s.get("residual"))
        return {**_held(*y), **({"sum": total} if c["residual"] else {})}
    x = eff.FP8Rows(s["x"], s["x_scale"])
    if c["kind"] == "linear":
        return eff.fp8_linear(x, eff.FP8Weight(s["w"], s["w_scale"]), bias=s.get("bias"),
                              residual=s.get("residual"), dtype=DTYPES[c["dtype"]])
    return _held(*eff.fp8_linear_silu_mul(x, eff.FP8Weight(s["w_gate"], s["w_gate_scale"]),
                                          eff.FP8Weight(s["w_up"], s["w_up_scale"])))


def _held(codes, byte):
    return _numbers(_seen(codes), _seen(byte))


def _numbers(codes, byte):
    return {"codes": codes.view(E4M3), "scale": byte.view(E8M0)}


def _plain(state):
    c, s = state["case"], state["seen"]
    if c["kind"] == "quantize":
        return _numbers(*_quantized(s["x"].float(), 1))
    if c["kind"] == "weight":
        return _numbers(*_quantized(s["w"].float(), GROUP))
    if c["kind"] == "norm":
        total = s["x"]
        if c["residual"]:
            total = (total.float() + s["residual"].float()).to(total.dtype)
        y = total.double()  # (a group's amax may lie next to the border between two scales)
        y = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * s["weight"].double()
        return {**_numbers(*_quantized(y, 1)), **({"sum": total} if c["residual"] else {})}
    x = _value(s["x"], s["x_scale"], 1)

    def product(n):
        return torch.matmul(x, _value(s[n], s[n + "_scale"], GROUP).t())

    if c["kind"] == "linear":
        out = product("w")
        for n in ("bias", "residual"):
            if c[n]:
                out = out + s[n].float()
        return out.to(DTYPES[c["dtype"]])
    gate = product("w_gate")
    return _numbers(*_quantized(gate / (1 + torch.exp(-gate)) * product("w_up"), 1))


def work(case):
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4}.get(c.get("dtype"))
    k, kb = c["k"], _blocks(c["k"])
    if c["kind"] == "quantize":
        return {"bytes": c["m"] * ((size + 1) * k + kb), "flops": 3 * c["m"] * k}
    if c["kind"] == "weight":
        return {"bytes": (size + 1) * c["n"] * k + _blocks(c["n"]) * kb, "flops": 3 * c["n"] * k}
    if c["kind"] == "norm":
        passes = 3 if c["residual"] else 1  # x, the residual and their sum
        return {"bytes": c["m"] * (size * passes * k + k + kb) + size * k, "flops": 8 * c["m"] * k}
    m, n, nb = c["m"], c["n"], _blocks(c["n"])
    if c["kind"] == "linear":
        ends = size * (m * n * (1 + c["residual"]) + n * c["bias"])
        return {"bytes": m * (k + kb) + n * k + nb * kb + ends, "flops": 2 * m * n * k}
    return {"bytes": m * (k + kb) + 2 * (n * k + nb * kb) + m * (n + nb), "flops": 4 * m * n * k}


# ---- the operators' definitions in 64 bits --------------------------------------


def _exact_quantized(x, rows):
    """Codes and scales as numbers: a power of two by comparison, a code by its own step."""
    m, k = x.shape
    whole = torch.zeros((-(-m // rows) * rows, _blocks(k) * GROUP), dtype=torch.float64, device="cuda")
    whole[:m, :k] = x
    most = whole.abs().view(-1, rows, _blocks(k), GROUP).amax(3).amax(1)
    s = torch.exp2(torch.ceil(torch.log2(most.clamp(min=1e-300) / 448)).clamp(min=LEAST))
    s = torch.where(most > 448 * s, 2 * s, s)
    s = torch.where((most <= 224 * s) & (s > 2.0 ** LEAST), s / 2, s)
    for i in range(s.shape[1]):  # a column of groups at a time
        part = whole[:, i * GROUP : (i + 1) * GROUP]
        part /= s[:, i].repeat_interleave(rows)[:, None]
        step = torch.exp2(torch.floor(torch.log2(part.abs().clamp(min=2.0 ** -6))) - 3)
        part.copy_(torch.round(part / step) * step)
    return {"codes": whole[:m, :k], "scale": s}


def _exact_value(codes, byte, rows):
    x = codes.view(E4M3).double()
    for i in range(byte.shape[1]):
        x[:, i * GROUP : (i + 1) * GROUP] *= torch.exp2(byte[:, i].double() - 127).repeat_interleave(
            rows)[: x.shape[0], None]
    return x


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "quantize":
        return _exact_quantized(s["x"][:, : c["k"]].double(), 1)
    if c["kind"] == "weight":
        return _exact_quantized(s["w"].double(), GROUP)
    if c["kind"] == "norm":
        total = s["x"].double()
        if c["residual"]:  # (exact, so that one rounding gives the stream the norm is taken of)
            total = (total + s["residual"].double()).to(s["x"].dtype).double()
        power = total.square().sum(1) / c["k"] + EPS
        got = _exact_quantized(total * power.rsqrt()[:, None] * s["weight"].double(), 1)
        return {**got, **({"sum": total} if c["residual"] else {})}
    x = _exact_value(s["x"], s["x_scale"], 1)
    products = [x @ _exact_value(s[n], s[n + "_scale"], GROUP).t().contiguous()
                for n in (("w",) if c["kind"] == "linear" else ("w_gate", "w_up"))]
    if c["kind"] == "gate":
        return _exact_quantized(products[0] * torch.sigmoid(products[0]) * products[1], 1)
    return products[0] + (s["bias"].double() if c["bias"] else 0) + (
        s["residual"].double() if c["residual"] else 0)
