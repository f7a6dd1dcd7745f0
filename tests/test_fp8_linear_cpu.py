"""Linear layers in 8-bit floating point without a GPU: what the entry points refuse,
and the oracle against independent statements of its definition."""
import pytest
import torch

from oracle import fp8 as oracle
from torch_gcu import _abi

INVALID, UNSUPPORTED, TOO_LARGE = 1, 2, 5
U8, BF16 = torch.uint8, torch.bfloat16


def call(m=5, n=200, k=300):
    """Valid arguments of all calls, by name; a pair is codes and scales (of the
    default sizes)."""
    z = lambda *s: torch.zeros(s, dtype=U8)  # noqa: E731
    return {
        "wide": torch.zeros(m, k, dtype=BF16), "residual": torch.zeros(m, k, dtype=BF16),
        "total": torch.zeros(m, k, dtype=BF16), "norm": torch.zeros(k, dtype=BF16),
        "rows": z(m, k), "rows_scale": z(m, 3), "w": z(n, k), "w_scale": z(2, 3),
        "up": z(n, k), "up_scale": z(2, 3), "wide_w": torch.zeros(n, k, dtype=BF16),
        "x": z(m, k), "x_scale": z(m, 3), "out": torch.zeros(m, n, dtype=BF16),
        "bias": torch.zeros(n, dtype=BF16), "add": torch.zeros(m, n, dtype=BF16),
        "gated": z(m, n), "gated_scale": z(m, 2), "eps": 1e-6,
    }


ORDER = {
    "fp8_quantize": ["/rows", "wide"],
    "fp8_quantize_weight": ["/w", "wide_w"],
    "rms_norm_fp8": ["/rows", "total", "wide", "residual", "norm", "eps"],
    "fp8_linear": ["out", "/x", "/w", "bias", "add"],
    "fp8_linear_silu_mul": ["/gated", "/x", "/w", "/up"],
}


def run(op, a):
    def arg(n):
        if n[0] == "/":
            return _abi.MiFp8(_abi.desc(a[n[1:]]), _abi.desc(a[n[1:] + "_scale"]))
        return _abi.desc(a[n]) if isinstance(a[n], torch.Tensor) or a[n] is None else a[n]

    st = getattr(_abi.lib(), "mi_" + op)(*(arg(n) for n in ORDER[op]), None)
    return st, _abi.lib().mi_last_error().decode()


QUANTIZE, WEIGHT, NORM, LINEAR, GATE = ORDER
PRODUCTS = (LINEAR, GATE)
REFUSED = [
    # (ops, changed argument, its new value, status, words of the message)
    ((QUANTIZE, NORM), "wide", lambda t: t.double(), INVALID, "float16 or float32"),
    ((QUANTIZE, NORM), "wide", lambda t: t[:3], INVALID, "codes are"),
    ((QUANTIZE, NORM), "wide", lambda t: t.t().contiguous().t(), INVALID, "dense rows"),
    ((QUANTIZE, NORM), "wide", lambda t: t[None], INVALID, "dense rows"),
    ((QUANTIZE, NORM), "rows", lambda t: t.to(torch.int8), INVALID, "uint8"),
    ((QUANTIZE, NORM), "rows", lambda t: t[:1].expand(5, 300), INVALID, "overlap"),
    ((QUANTIZE, NORM), "rows", lambda t: t.as_strided((5, 300), (150, 1)), INVALID, "overlap"),
    ((QUANTIZE, NORM), "rows_scale", lambda t: t[:, :2], INVALID, "[5, 3]"),
    ((QUANTIZE, NORM), "rows_scale", lambda t: t[:4], INVALID, "[5, 3]"),
    ((QUANTIZE, NORM), "rows_scale", lambda t: t.t().contiguous().t(), INVALID, "dense"),
    ((WEIGHT,), "wide_w", lambda t: t[:, :299], INVALID, "codes are"),
    ((WEIGHT,), "wide_w", lambda t: t.long(), INVALID, "float32"),
    ((WEIGHT, LINEAR, GATE), "w_scale", lambda t: t[:1], INVALID, "128 x 128"),
    ((WEIGHT,), "w_scale", lambda t: t[:1].expand(2, 3), INVALID, "overlap"),
    ((NORM,), "residual", lambda t: t.half(), INVALID, "x's shape and type"),
    ((NORM,), "residual", lambda t: t[:4], INVALID, "x's shape and type"),
    ((NORM,), "total", lambda t: t.half(), INVALID, "x's shape and type"),
    ((NORM,), "total", lambda t: t[:1].expand(5, 300), INVALID, "overlap"),
    ((NORM,), "norm", lambda t: t.float(), INVALID, "dense vector"),
    ((NORM,), "norm", lambda t: t[:299], INVALID, "dense vector"),
    ((NORM,), "norm", lambda t: torch.zeros(600, dtype=BF16)[::2], INVALID, "dense vector"),
    (PRODUCTS, "x", lambda t: t[:, :200], INVALID, "x must be"),
    (PRODUCTS, "x", lambda t: t.float(), INVALID, "uint8"),
    (PRODUCTS, "x", lambda t: t.t().contiguous().t(), INVALID, "dense"),
    (PRODUCTS, "x_scale", lambda t: t.float(), INVALID, "uint8"),
    (PRODUCTS, "x_scale", lambda t: t[:4], INVALID, "[5, 3]"),
    ((LINEAR,), "out", lambda t: t.float(), INVALID, "bfloat16 or float16"),
    ((LINEAR,), "out", lambda t: t[:, :199], INVALID, "out is"),
    ((LINEAR,), "out", lambda t: t[:1].expand(5, 200), INVALID, "overlap"),
    ((LINEAR,), "bias", lambda t: t.half(), INVALID, "bias"),
    ((LINEAR,), "bias", lambda t: t[:100], INVALID, "bias"),
    ((LINEAR,), "bias", lambda t: t[None], INVALID, "bias"),
    ((LINEAR,), "add", lambda t: t.half(), INVALID, "residual must have"),
    ((LINEAR,), "add", lambda t: t[:4], INVALID, "residual must have"),
    ((GATE,), "up", lambda t: t[:150], INVALID, "different shapes"),
    ((GATE,), "gated", lambda t: t[:, :128], INVALID, "gated"),
    ((GATE,), "gated", lambda t: t[:1].expand(5, 200), INVALID, "overlap"),
]


@pytest.mark.parametrize("ops,name,change,status,words", REFUSED)
def test_refuses(ops, name, change, status, words):
    for op in ops:
        a = call()
        a[name] = change(a[name])
        if name == "x" and a[name].shape == (5, 200):  # columns that differ from the weight's
            a["x_scale"] = a["x_scale"][:, :2]
            words = "x has 200 columns"
        if name == "up":
            a["up_scale"] = a["up_scale"][:2]
        if name == "gated" and words == "gated":
            a["gated_scale"] = a["gated_scale"][:, :1]
            words = "expected [5, 200]"
        st, text = run(op, a)
        assert st == status and words in text and op in text, (op, st, text)


OVERLAPS = [
    (QUANTIZE, "rows", "wide"), (QUANTIZE, "rows_scale", "wide"), (QUANTIZE, "rows", "rows_scale"),
    (WEIGHT, "w", "wide_w"), (WEIGHT, "w_scale", "wide_w"), (WEIGHT, "w", "w_scale"),
    (NORM, "rows", "wide"), (NORM, "rows", "residual"), (NORM, "rows", "total"), (NORM, "rows", "norm"),
    (NORM, "rows_scale", "total"), (NORM, "total", "norm"), (NORM, "total", "wide"), (NORM, "total", "residual"),
    (LINEAR, "out", "x"), (LINEAR, "out", "w"), (LINEAR, "out", "x_scale"), (LINEAR, "out", "w_scale"),
    (LINEAR, "out", "bias"), (LINEAR, "out", "add"),
    (GATE, "gated", "x"), (GATE, "gated", "w"), (GATE, "gated", "up"), (GATE, "gated_scale", "x_scale"),
    (GATE, "gated", "gated_scale"), (GATE, "gated_scale", "up_scale"),
]


@pytest.mark.parametrize("op,one,other", OVERLAPS)
def test_refuses_outputs_that_share_memory(op, one, other):
    a = call()
    pool = torch.zeros(1 << 20, dtype=U8)

    def at(t, byte):
        return pool[byte: byte + t.numel() * t.element_size()].view(t.dtype).view(t.shape)

    a[one], a[other] = at(a[one], 1024), at(a[other], 1024 + 64)  # its end in the other's beginning
    if a[one].numel() * a[one].element_size() <= 64:
        a[one] = at(a[one], 1024 + 80)
    if a[other].numel() * a[other].element_size() < 16:
        a[other] = at(a[other], 1024 + 2)
        a[one] = at(a[one], 1024)
    st, text = run(op, a)
    assert st == INVALID and "shares memory" in text, text


def test_null_operands_are_refused():
    for op in ORDER:
        a = call()
        a.update({ORDER[op][0].strip("/"): None})
        st, text = run(op, a)
        assert st != 0 and text, op


def test_sizes_past_the_limits_are_refused():
    a = call(1, 1, 1)
    a["x"] = a["x_scale"] = torch.zeros(1, dtype=U8).as_strided((1 << 32, 1), (0, 1))
    for op in PRODUCTS:
        st, text = run(op, a)
        assert st == TOO_LARGE, text
    for k, groups in (((1 << 30) + 1, (1 << 23) + 1),):  # columns are counted in 31 bits
        wide = torch.zeros(1, dtype=BF16).as_strided((0, k), (0, 1))
        a = {"wide": wide, "rows": torch.zeros(1, dtype=U8).as_strided((0, k), (0, 1)),
             "rows_scale": torch.zeros(1, dtype=U8).as_strided((0, groups), (0, 1))}
        st, text = run(QUANTIZE, a)
        assert st == TOO_LARGE and "2^30" in text, text
    k = (1 << 22) - 15
    a = {**call(1, 1, 1), "x": torch.zeros(1, k, dtype=U8), "x_scale": torch.zeros(1, 1 << 15, dtype=U8),
         "w": torch.zeros(1, k, dtype=U8), "w_scale": torch.zeros(1, 1 << 15, dtype=U8)}
    for op in PRODUCTS:
        st, text = run(op, {**a, "up": a["w"], "up_scale": a["w_scale"], "gated_scale": a["gated_scale"][:, :1]})
        assert st == TOO_LARGE, text


def test_more_outputs_than_a_grid_holds_are_refused():
    n = 1 << 28  # columns, 16 of them a block
    w, scale = torch.zeros(1, 1, dtype=U8).expand(n, 1), torch.zeros(1, 1, dtype=U8).expand(n // 128, 1)
    a = {**call(1, 1, 1), "w": w, "w_scale": scale, "up": w, "up_scale": scale, "bias": None, "add": None,
         "x_scale": torch.zeros(1, 1, dtype=U8), "out": torch.empty(1, n, dtype=BF16),
         "gated": torch.empty(1, n, dtype=U8), "gated_scale": torch.empty(1, n // 128, dtype=U8)}
    for op in PRODUCTS:
        st, text = run(op, a)
        assert st == TOO_LARGE and "too many outputs" in text, text


def test_empty_calls_do_nothing():
    for op in ORDER:
        for shape in ((0, 200, 300), (5, 0, 300)):
            a = call(*shape)
            a["w_scale"] = a["up_scale"] = torch.zeros(-(-shape[1] // 128), 3, dtype=U8)
            a["gated_scale"] = torch.zeros(shape[0], -(-shape[1] // 128), dtype=U8)
            if shape[0] == 0 or op in (WEIGHT, LINEAR, GATE):
                if op == WEIGHT and shape[1]:
                    continue
                st, text = run(op, a)
                assert st == 0, (op, shape, text)


# ---- the oracle -------------------------------------------------------------------


def test_oracle_scales_are_the_smallest():
    amax = torch.tensor([0.0, 1e-40, 448.0, 448.0001, 224.0, 224.1, 1.0, 3e38, 2.0 ** -110 * 448, 2.0 ** -101],
                        dtype=torch.float64)
    s = oracle.value(oracle.scale_byte(amax))
    assert bool((amax <= 448 * s).all())
    assert bool(((amax > 224 * s) | (s == 2.0 ** -110)).all())
    assert s[2] == 1 and s[3] == 2 and s[4] == 0.5


def test_oracle_codes_are_torchs():
    """Codes by arithmetic against torch's own conversion."""
    x = torch.randn(37, 300, generator=torch.Generator().manual_seed(1)) * 3
    code, byte = oracle.quantize(x)
    s = oracle.spread(byte, 1, x.shape)
    assert torch.equal(code, (x.double() / s).float().to(torch.float8_e4m3fn).view(U8))
    assert float((oracle.numbers(code, byte) - x).abs().max()) <= float((x.abs() * 2.0 ** -4).max())


def test_oracle_weight_blocks():
    w = torch.zeros(200, 300)
    w[150, 270] = 448.0 * 8
    w[3, 3] = -1.0
    code, byte = oracle.quantize(w, 128)
    assert byte.tolist()[1][2] == 130 and byte.tolist()[0][0] == 127 - 8 and byte.tolist()[0][1] == 17
    assert torch.equal(oracle.numbers(code, byte, 128), w.double())


def test_oracle_marks_what_is_not_finite():
    x = torch.ones(1, 130)
    x[0, 5], x[0, 129] = float("inf"), float("nan")
    code, byte = oracle.quantize(x)
    got = oracle.numbers(code, byte)
    assert got[0, [5, 129]].isnan().all() and got.isnan().sum() == 2 and byte[0].tolist() == [127 - 8, 127 - 8]


def test_oracle_product_against_a_loop():
    g = torch.Generator().manual_seed(2)
    x = oracle.quantize(torch.randn(3, 200, generator=g))
    w = oracle.quantize(torch.randn(130, 200, generator=g), 128)
    out, mass, power = oracle.product(x, w)
    a = x[0].view(torch.float8_e4m3fn).double()
    b = w[0].view(torch.float8_e4m3fn).double()
    for m, n in ((0, 0), (2, 129), (1, 127)):
        s = sum(float(a[m, k] * b[n, k]) * 2.0 ** (int(x[1][m, k // 128]) + int(w[1][n // 128, k // 128]) - 254)
                for k in range(200))
        assert abs(s - float(out[m, n])) <= 1e-12 * float(mass[m, n])
    assert bool((out.abs() <= mass).all()) and bool((power <= mass.square()).all())
