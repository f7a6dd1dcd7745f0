"""Linear layers in 8-bit floating point on the GPU against their definition in 64
bits.

Codes and scales.  Quantising is exact.  Where y is computed first, it is off by at
most `d` (below), and the code has to be that of some number within d of y: rounding
is monotonic, so it lies between the codes of the two ends, under the scale that was
chosen, which has to be that of an amax within d.

Sums.  A matrix instruction adds 8 neighbours of K at a time and keeps 13 bits below
the largest: each of the other seven loses at most 2^-13 of it, which the sum of the
magnitudes (`mass`) bounds; the sums of those are fp32 (K / 8 of them and the slices).
For the whole output the losses are independent: a seventh of their variances, at most
(2^-13 p)^2 / 3 for each, with p^2 bounded by the sum of squares (`power`); twice
their root is allowed.  Products of small whole numbers are exact, and so has to be
every output, up to its one rounding."""
import math

import pytest
import torch

import torch_gcu  # noqa: F401
from oracle import fp8 as oracle
from torch_gcu import _abi
from torch_gcu.utils import decoder_layer as dl

pytestmark = pytest.mark.gpu
eff = torch.gcu.efficient if hasattr(torch, "gcu") else None
F = 2.0 ** -24
BF16, F16, F32, U8 = torch.bfloat16, torch.float16, torch.float32, torch.uint8


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tokens(m, k, dtype, seed=0, empty=True):
    """Channels of different size, a row of zeros and one of tiny numbers."""
    g = gen(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))
    if m > 2 and empty:
        x[m // 2] = 0
        x[m // 3] *= 2.0 ** -14
    return x.to(dtype)


def cpu(pair):
    return tuple(t.cpu() for t in pair)


def gcu(pair, kind=None):
    kind = kind or eff.FP8Rows
    return kind(*(t.to("gcu") for t in pair))


def check_codes(got, y, d, rows=1):
    """got (codes, scales) of y, whose elements are off by at most d (relative) or
    2^-140."""
    code, byte = cpu(got)
    code, byte = code.reshape(-1, code.shape[-1]), byte.reshape(-1, byte.shape[-1])
    y = y.reshape(-1, y.shape[-1]).double()
    d = torch.as_tensor(d, dtype=torch.float64).expand(y.shape)
    fine = torch.isfinite(y)
    lo = torch.where(fine, y - d * y.abs() - 2.0 ** -140, y)
    hi = torch.where(fine, y + d * y.abs() + 2.0 ** -140, y)
    size = [torch.where(fine, x, 0.0).clamp(min=0) for x in
            (y.abs() - d * y.abs() - 2.0 ** -140, y.abs() + d * y.abs() + 2.0 ** -140)]
    least, most = (oracle.scale_byte(oracle.blocks(x, rows).amax((1, 3))) for x in size)
    assert bool(((byte >= least) & (byte <= most)).all()), "scales"
    # (the scale holds what was computed, so a code's number ends at 448 of it)
    end = 448 * oracle.spread(byte, rows, y.shape)
    want = [oracle.numbers(oracle.quantize(torch.where(fine, x.clamp(-end, end), x), rows, byte)[0], byte, rows)
            for x in (lo, hi)]
    v = oracle.numbers(code, byte, rows)
    assert torch.equal(v.isnan(), ~fine), "NaN codes"
    off = ~((v >= want[0]) & (v <= want[1])) & fine
    assert not off.any(), f"{int(off.sum())} of {off.numel()} codes, first at {off.nonzero()[0].tolist()}"


# ---- quantising -------------------------------------------------------------------

SIZES = [(1, 1), (1, 128), (2, 129), (3, 7), (5, 127), (4, 640), (65, 512), (17, 513), (9, 1024), (3, 1500),
         (33, 2048), (7, 2056), (8, 4096), (2, 4100), (3, 8192), (2, 11008), (1, 16384), (2, 20000), (300, 384)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k", SIZES)
def test_quantize(m, k, dtype):
    x = tokens(m, k, dtype, seed=m + k)
    code, byte = cpu(eff.fp8_quantize(x.to("gcu")))
    want = oracle.quantize(x)
    assert torch.equal(byte, want[1])
    assert torch.equal(code & 0x7F, want[0] & 0x7F)  # (a zero keeps its sign)
    assert torch.equal(oracle.numbers(code, byte), oracle.numbers(*want))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 130), (127, 64), (128, 128), (129, 300), (200, 1000), (1000, 129), (640, 4104)])
def test_quantize_weight(n, k, dtype):
    w = tokens(n, k, dtype, seed=n + k)
    code, byte = cpu(eff.fp8_quantize_weight(w.to("gcu")))
    want = oracle.quantize(w, 128)
    assert torch.equal(byte, want[1])
    assert torch.equal(oracle.numbers(code, byte, 128), oracle.numbers(*want, rows=128))


@pytest.mark.parametrize("k", [128, 2048, 20000, 1001])
def test_quantize_what_is_not_finite(k):
    x = tokens(40, k, F32, seed=3)
    x[1, 5], x[2, k - 1], x[3] = math.inf, math.nan, math.nan
    x[4, 0], x[4, k - 1], x[5] = -math.inf, math.inf, math.inf
    x[6, 7] = 3.3e38
    check_codes(eff.fp8_quantize(x.to("gcu")), x, 0.0)
    check_codes(eff.fp8_quantize_weight(x.to("gcu")), x, 0.0, rows=128)


@pytest.mark.parametrize("fill", [448.0, 448.5, 1.75, 1.7578125, 2.0 ** -110, 1e-38, 1e-44, 3.3e38, 0.0, -0.0])
def test_quantize_scales_at_their_borders(fill):
    x = torch.full((3, 256), fill)
    x[1, 1:] = 0
    code, byte = cpu(eff.fp8_quantize(x.to("gcu")))
    want = oracle.quantize(x)
    assert torch.equal(byte, want[1]) and torch.equal(oracle.numbers(code, byte), oracle.numbers(*want))


def test_quantize_views():
    wide = tokens(40, 3000, BF16, seed=5).to("gcu")
    for x in (wide[:, 100:612], wide[:, 3:260], wide[::3, :1000], wide.view(4, 10, 3000)[:, :, 8:1032],
              wide.view(4, 10, 3000)[1:3, 2:7], wide.t()[:300], wide.view(5, 8, 3000).transpose(0, 1)[:, :, :256],
              wide[:1, 1:2], wide[0], wide[:, :257].unsqueeze(1)):
        got = eff.fp8_quantize(x)
        assert got.codes.shape == x.shape and got.scales.shape == x.shape[:-1] + (-(-x.shape[-1] // 128),)
        want = oracle.quantize(x.cpu().reshape(-1, x.shape[-1]))
        code, byte = cpu(got)
        assert torch.equal(byte.reshape(want[1].shape), want[1])
        assert torch.equal(code.reshape(want[0].shape) & 0x7F, want[0] & 0x7F)


def test_expanded_rows():
    """Rows that are the same memory are read like any."""
    row = tokens(1, 300, BF16, seed=6, empty=False)
    wide = row.to("gcu").expand(9, 300)
    q, one = eff.fp8_quantize(wide), oracle.quantize(row)
    assert torch.equal(q.codes.cpu(), one[0].expand(9, 300)) and torch.equal(q.scales.cpu(), one[1].expand(9, 3))
    y, total = eff.rms_norm_fp8(wide, None, residual=wide)
    assert torch.equal(total.cpu(), (2 * row).expand(9, 300))
    x = eff.FP8Rows(q.codes[:1].expand(70, 300), q.scales[:1].expand(70, 3))
    w = eff.fp8_quantize_weight(torch.randn(200, 300, generator=gen(1)).to("gcu"))
    got = eff.fp8_linear(x, w).cpu()
    assert torch.equal(got, got[:1].expand(70, 200))


@pytest.mark.parametrize("k", [8, 1032])
def test_more_rows_than_a_grids_first_dimension(k):
    """2^20 blocks of 4 rows (of one, above 1024 columns), and a few more."""
    m = (1 << 22) + 7 if k == 8 else (1 << 20) + 7
    x = (torch.arange(m, device="cuda")[:, None] % 251 + torch.arange(k, device="cuda")).to(BF16)
    got = torch.zeros(m, k, dtype=U8, device="cuda"), torch.zeros(m, -(-k // 128), dtype=U8, device="cuda")
    for call in (lambda o, x: _abi.fp8_quantize(o, x), lambda o, x: _abi.rms_norm_fp8(o, None, x, None, None, 1e-6)):
        few = tuple(torch.zeros_like(t[:251]) for t in got)
        call(got, x), call(few, x[:251])
        for t, f in zip(got, few):
            assert torch.equal(t[: m // 251 * 251].view(-1, *f.shape), f.expand(m // 251, *f.shape))
            assert torch.equal(t[m // 251 * 251:], f[: m % 251])
            t.zero_()


def test_quantize_empty():
    for shape in ((0, 128), (3, 0), (2, 0, 5)):
        got = eff.fp8_quantize(torch.empty(shape, dtype=BF16, device="gcu"))
        assert got.codes.shape == torch.Size(shape)
    assert eff.fp8_quantize_weight(torch.empty(0, 4, device="gcu")).scales.shape == (0, 1)


# ---- norm -------------------------------------------------------------------------


def norm_error(k):
    """fp32: sums of squares by chains of at most k / 256 + 64 terms and 12 joins, halved by
    the root; mean, eps, root, quotient, two products."""
    return ((k / 256 + 64 + 12) / 2 + 6) * F


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", SIZES)
def test_rms_norm(m, k, dtype, residual):
    x, r = tokens(m, k, dtype, seed=m + k), 3 * tokens(m, k, dtype, seed=1) if residual else None
    w = (1 + 0.2 * torch.randn(k, generator=gen(2))).to(dtype) if k % 3 else None
    got, total = eff.rms_norm_fp8(x.to("gcu"), None if w is None else w.to("gcu"), 1e-6,
                                  residual=None if r is None else r.to("gcu"))
    y, t = oracle.rms_norm(x, w, 1e-6, r)
    assert torch.equal(total.cpu(), t)
    check_codes(got, y, norm_error(k))


def test_rms_norm_views_and_leading_dims():
    wide = tokens(60, 2100, BF16, seed=8).to("gcu")
    w = torch.ones(520, dtype=BF16, device="gcu")
    for x, r in ((wide.view(3, 20, 2100)[:, :, 8:528], wide.view(3, 20, 2100)[:, :, 1000:1520]),
                 (wide[::2, 3:523], wide[1::2, :520]), (wide[0, :520], wide[1, 1:521])):
        got, total = eff.rms_norm_fp8(x, w[: x.shape[-1]], 1e-5, residual=r)
        y, t = oracle.rms_norm(x.cpu(), w.cpu(), 1e-5, r.cpu())
        assert torch.equal(total.cpu(), t) and got.codes.shape == x.shape
        check_codes(got, y, norm_error(520))
    got, total = eff.rms_norm_fp8(wide, None)
    assert total is wide


def test_rms_norm_in_place_and_untouched_surroundings():
    for k in (1000, 4096, 20000, 1001):
        x, r = tokens(6, k, F16, seed=k), tokens(6, k, F16, seed=k + 1)
        pool = torch.full((8, k + 50), 9.0, dtype=F16, device="cuda")
        pool[1:7, 10: 10 + k] = r.cuda()
        total = pool[1:7, 10: 10 + k]
        code = torch.full((8, k + 30), 77, dtype=U8, device="cuda")
        byte = torch.full((8, -(-k // 128) + 5), 77, dtype=U8, device="cuda")
        out = (code[1:7, 7: 7 + k], byte[1:7, 2:-3])
        _abi.rms_norm_fp8(out, total, x.cuda(), total, None, 1e-6)
        torch.cuda.synchronize()
        y, t = oracle.rms_norm(x, None, 1e-6, r)
        assert torch.equal(total.cpu(), t)
        check_codes(out, y, norm_error(k))
        total.fill_(9.0), out[0].fill_(77), out[1].fill_(77)
        assert bool((pool == 9).all()) and bool((code == 77).all()) and bool((byte == 77).all())


def test_rms_norm_of_what_is_not_finite():
    x = tokens(8, 640, BF16, seed=4)
    x[1, 3], x[2, 600], x[3, 5] = math.inf, math.nan, -math.inf
    w = torch.ones(640, dtype=BF16)
    got, _ = eff.rms_norm_fp8(x.to("gcu"), w.to("gcu"))
    code, byte = cpu(got)
    v = oracle.numbers(code, byte)
    y, _ = oracle.rms_norm(x, w, 1e-6)
    assert torch.equal(v.isnan(), y.isnan())
    keep = [0, 4, 5, 6, 7]
    check_codes((code[keep], byte[keep]), y[keep], norm_error(640))
    w[9] = math.inf
    got, _ = eff.rms_norm_fp8(x[keep].to("gcu"), w.to("gcu"))
    v = oracle.numbers(*cpu(got))
    assert bool(v[:, 9].isnan().all()) and int(v.isnan().sum()) == len(keep)


# ---- products ---------------------------------------------------------------------

SHAPES = [
    (1, 1, 1), (1, 16, 16), (3, 5, 7), (2, 130, 15), (16, 128, 128), (17, 129, 130), (1, 4096, 512), (33, 200, 1000),
    (64, 256, 384), (5, 3000, 2050), (24, 640, 4096), (65, 300, 1000), (128, 128, 4096), (130, 500, 2051),
    (200, 1030, 260), (256, 256, 512), (300, 1000, 1104), (513, 2300, 129), (777, 640, 1500), (1030, 1100, 640),
    (260, 4500, 400), (2100, 2050, 272), (4100, 4099, 136), (40, 33000, 144),
]


def whole_numbers(m, n, k, seed):
    """Operands of -2 .. 2 under scales of 1/2, 1 or 2 a row or block: products and
    their sums are whole multiples of 1/4 below 2^24, so every sum is exact."""
    g = gen(seed)
    x = torch.randint(-2, 3, (m, k), generator=g).float().to(torch.float8_e4m3fn).view(U8)
    w = torch.randint(-2, 3, (n, k), generator=g).float().to(torch.float8_e4m3fn).view(U8)
    kb = -(-k // 128)
    xs = torch.randint(126, 129, (m, kb), generator=g).to(U8)
    ws = torch.randint(126, 129, (-(-n // 128), kb), generator=g).to(U8)
    return (x, xs), (w, ws)


def exact_product(x, w):
    """In float32 matmuls of whole numbers, which are exact too, and quicker."""
    return oracle.numbers(*x).float() @ oracle.numbers(*w, rows=128).float().t()


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("ends", ["", "bias", "residual", "bias residual f16", "bias32"])
def test_linear_is_exact_on_whole_numbers(m, n, k, ends):
    x, w = whole_numbers(m, n, k, m + n + k)
    g, dtype = gen(7), F16 if "f16" in ends else BF16
    out = exact_product(x, w).double()
    args = {}
    if "bias" in ends:
        args["bias"] = torch.randint(-8, 9, (n,), generator=g).to(F32 if "32" in ends else dtype)
        out = out + args["bias"].double()
    if "residual" in ends:
        args["residual"] = torch.randint(-64, 65, (m, n), generator=g).to(dtype)
        out = out + args["residual"].double()
    got = eff.fp8_linear(gcu(x), gcu(w, eff.FP8Weight), dtype=dtype,
                         **{a: t.to("gcu") for a, t in args.items()})
    assert got.dtype == dtype and torch.equal(got.cpu(), out.float().to(dtype))


# the largest sizes of each tile shape and cut of K that stay quick on the CPU, with and
# without whole groups (what runs: 256 x 256, 256 x 128, 128 x 128, 64 x 128, then 64 x 64
# whole, in two and in four)
LARGE = [(4778, 2992, 1111), (1804, 7699, 640), (909, 8018, 1110), (1523, 5177, 256), (259, 6711, 1131),
         (4991, 407, 1152), (2456, 3229, 1102), (265, 6681, 128), (777, 4096, 512), (2655, 68, 4231),
         (70, 3238, 4608), (25, 64, 7072), (42, 65, 4608), (65, 66, 64), (128, 4096, 1024),
         (2183, 6916, 768), (1922, 7104, 896), (4742, 3242, 700), (1935, 7097, 776), (4688, 838, 131),
         (5979, 652, 265), (577, 6619, 393), (5784, 642, 514), (331, 6085, 133), (389, 4938, 257),
         (352, 5695, 512), (3757, 514, 385), (2750, 781, 384)]


@pytest.mark.parametrize("m,n,k", LARGE)
def test_linear_of_every_tile_shape(m, n, k):
    x, w = whole_numbers(m, n, k, m + n + k)
    res = torch.randint(-64, 65, (m, n), generator=gen(5)).to(BF16)
    got = eff.fp8_linear(gcu(x), gcu(w, eff.FP8Weight), residual=res.to("gcu"))
    assert torch.equal(got.cpu(), (exact_product(x, w) + res.float()).to(BF16))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_of_the_largest_and_smallest_scales(m):
    """2^-127 and 2^127, alone and against each other, in every way of the product."""
    n, k = 140, 300
    (x, _), (w, _) = whole_numbers(m, n, k, 23)
    base = exact_product((x, torch.full((m, 3), 127, dtype=U8)), (w, torch.full((2, 3), 127, dtype=U8))).double()
    for a, b in ((0, 254), (254, 0), (0, 127), (254, 127), (1, 1), (127, 0)):
        got = eff.fp8_linear(gcu((x, torch.full((m, 3), a, dtype=U8))),
                             gcu((w, torch.full((2, 3), b, dtype=U8)), eff.FP8Weight)).cpu()
        want = (base * 2.0 ** (a + b - 254)).float().to(BF16)
        if a + b > 370:  # (a term of 2 x 2^127 is float32's infinity, and two of them a NaN)
            assert bool(((got == want) | ~got.isfinite()).all())
        elif a + b < 128:  # (results under float32's normal range may be 0)
            assert bool(((got.double() - want.double()).abs() <= 2.0 ** -126).all())
        else:
            assert torch.equal(got, want), (a, b)


def test_offsets_past_32_bits():
    """Weights and activations of more than 4 GiB: the first and last rows count."""
    k, rows = 4096, (1 << 20) + 4096 + 5
    big = torch.zeros(rows, k, dtype=U8, device="gcu")
    scale = torch.full((rows, 32), 127, dtype=U8, device="gcu")
    few, _ = whole_numbers(7, 1, k, 29)
    few = (few[0], torch.full((7, 32), 127, dtype=U8))
    at = [0, 1, rows - 2, rows - 1]
    lines = whole_numbers(4, 1, k, 31)[0][0]
    for i, r in enumerate(at):
        big[r].copy_(lines[i].to("gcu"))
    want = exact_product(few, (lines, torch.full((1, 32), 127, dtype=U8)))
    blocks = scale[: -(-rows // 128)]
    for m in (7, 70):  # few rows, and tiles
        x = gcu((few[0].repeat(10, 1)[:m], few[1].repeat(10, 1)[:m]))
        got = eff.fp8_linear(x, eff.FP8Weight(big, blocks))
        assert torch.equal(got[:7, at].cpu(), want.to(BF16)) and float(got[:, 4: rows - 4].cpu().float().abs().max()) == 0
        del got
    got = eff.fp8_linear(eff.FP8Rows(big, scale), gcu((few[0], few[1][:1]), eff.FP8Weight))
    assert torch.equal(got[at].cpu(), want.t().to(BF16))
    wide = torch.zeros(rows, k, dtype=BF16, device="gcu")
    wide[rows - 1].fill_(3.0)
    q = eff.fp8_quantize(wide)
    assert oracle.numbers(q.codes[rows - 2:].cpu(), q.scales[rows - 2:].cpu()).tolist() == [[0.0] * k, [3.0] * k]
    q, _ = eff.rms_norm_fp8(wide, None, 0.0)
    check_codes((q.codes[rows - 1:], q.scales[rows - 1:]), torch.ones(1, k), norm_error(k))


def rounding_of(x, w):
    """(sum, bound, deviation) of a product: 64 bits, what an output can be off by, and
    the root of the variance of that."""
    out, mass, power = oracle.product(x, w)
    k = x[0].shape[1]
    fp32 = (k / 8 + 16) * F
    return out, (7 * 2.0 ** -13 + fp32) * mass, (7 / 3 * power).sqrt() * 2.0 ** -13 + F * math.sqrt(k / 8) * mass


def quantized(m, n, k, seed=0):
    x = oracle.quantize(tokens(m, k, F32, seed))
    w = oracle.quantize(0.05 * torch.randn(n, k, generator=gen(seed + 1)), 128)
    return x, w


@pytest.mark.parametrize("m,n,k", [(1, 300, 500), (24, 640, 4096), (100, 1500, 1000), (300, 520, 2100), (1030, 1100, 640)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_of_ordinary_numbers(m, n, k, dtype):
    x, w = quantized(m, n, k)
    got = eff.fp8_linear(gcu(x), gcu(w, eff.FP8Weight), dtype=dtype).cpu().double()
    want, bound, dev = rounding_of(x, w)
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    assert bool(((got - want).abs() <= bound * (1 + u) + u * want.abs() + tiny).all())
    assert float((got - want).norm()) <= 2 * float(dev.norm()) + u * float(want.norm()) + tiny * math.sqrt(m * n)


def test_linear_reads_every_scale():
    """One operand's scales differ by row and group over the whole range that a sum holds."""
    m, n, k = 150, 400, 700
    (x, _), (w, _) = whole_numbers(m, n, k, 3)
    g = gen(9)
    xs = torch.randint(107, 148, (m, 6), generator=g).to(U8)
    ws = torch.randint(107, 148, (4, 6), generator=g).to(U8)
    got = eff.fp8_linear(gcu((x, xs)), gcu((w, ws), eff.FP8Weight)).cpu().double()
    want, bound, _ = rounding_of((x, xs), (w, ws))
    assert bool(((got - want).abs() <= bound * 1.01 + 2.0 ** -9 * want.abs() + 1e-30).all())


@pytest.mark.parametrize("m,n,k", [(5, 300, 260), (70, 300, 640), (300, 700, 500), (1100, 1200, 384)])
def test_linear_of_what_is_not_finite(m, n, k):
    x, w = whole_numbers(m, n, k, 11)
    want = exact_product(x, w).to(BF16)
    x[0][1, 3] = x[0][4, k - 1] = w[0][7, 0] = w[0][n - 1, k - 1] = 0x7F
    x[1][2, 1] = 255
    want[[1, 2, 4]] = math.nan
    want[:, [7, n - 1]] = math.nan
    got = eff.fp8_linear(gcu(x), gcu(w, eff.FP8Weight)).cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


def test_linear_rows_past_k_are_not_read_as_numbers():
    """What lies behind a row's end (NaN codes here) is of no account, aligned or not."""
    for m, n, k in ((20, 200, 130), (300, 600, 200), (20, 200, 133), (3, 40, 9)):
        for off, pitch in ((0, 256), (0, 260), (5, 256), (16, 416)):
            x, w = whole_numbers(m, n, k, k)
            pool = [torch.full((r + 1, pitch), 0x7F, dtype=U8) for r in (m, n)]
            a, b = (p.to("gcu") for p in pool)
            a.view(-1)[off:][: m * pitch].view(m, pitch)[:, :k].copy_(x[0].to("gcu"))
            b.view(-1)[off:][: n * pitch].view(n, pitch)[:, :k].copy_(w[0].to("gcu"))
            xr = eff.FP8Rows(a.view(-1)[off:][: m * pitch].view(m, pitch)[:, :k], x[1].to("gcu"))
            wr = eff.FP8Weight(b.view(-1)[off:][: n * pitch].view(n, pitch)[:, :k], w[1].to("gcu"))
            assert torch.equal(eff.fp8_linear(xr, wr).cpu(), exact_product(x, w).to(BF16)), (m, n, k, off, pitch)


def test_linear_of_rows_far_apart():
    x, w = whole_numbers(3, 140, 200, 21)
    far = torch.zeros(3, 1 << 22, dtype=U8, device="gcu")
    far[:, 64:264].copy_(x[0].to("gcu"))
    got = eff.fp8_linear(eff.FP8Rows(far[:, 64:264], x[1].to("gcu")), gcu(w, eff.FP8Weight))
    assert torch.equal(got.cpu(), exact_product(x, w).to(BF16))


def test_linear_views_and_leading_dims():
    x, w = whole_numbers(24, 300, 384, 13)
    want = exact_product(x, w).to(BF16)
    wg = gcu(w, eff.FP8Weight)
    a = eff.FP8Rows(x[0].to("gcu").view(2, 3, 4, 384), x[1].to("gcu").view(2, 3, 4, 3))
    assert torch.equal(eff.fp8_linear(a, wg).cpu(), want.view(2, 3, 4, 300))
    part = eff.FP8Rows(a.codes[:, 1:, ::2], a.scales[:, 1:, ::2])
    assert torch.equal(eff.fp8_linear(part, wg).cpu(), want.view(2, 3, 4, 300)[:, 1:, ::2])
    last = eff.FP8Rows(a.codes[..., 256:], a.scales[..., 2:])  # groups of wider rows
    got = eff.fp8_linear(last, eff.FP8Weight(wg.codes[:, 256:], wg.scales[:, 2:]))
    assert torch.equal(got.cpu().view(24, 300), exact_product((x[0][:, 256:], x[1][:, 2:]), (w[0][:, 256:], w[1][:, 2:])).to(BF16))
    rows = eff.fp8_linear(a, eff.FP8Weight(wg.codes[128:256], wg.scales[1:2]))
    assert torch.equal(rows.cpu(), want.view(2, 3, 4, 300)[..., 128:256])
    one = eff.FP8Rows(a.codes[0, 0, 0], a.scales[0, 0, 0])
    assert torch.equal(eff.fp8_linear(one, wg).cpu(), want[0])
    res = torch.randint(-9, 9, (300, 24), generator=gen(1)).to(BF16).to("gcu").t()  # not dense along columns
    got = eff.fp8_linear(eff.FP8Rows(a.codes.view(24, 384), a.scales.view(24, 3)), wg, residual=res)
    assert torch.equal(got.cpu(), (exact_product(x, w) + res.cpu().float()).to(BF16))


@pytest.mark.parametrize("m,n,k", [(7, 200, 300), (40, 4096, 2048), (90, 500, 640), (300, 700, 256), (1500, 1100, 128),
                                   (333, 640, 260), (1000, 6784, 128), (1922, 7104, 896)])
def test_linear_in_place_and_untouched_surroundings(m, n, k):
    x, w = whole_numbers(m, n, k, 17)
    for left, pitch in ((8, n + 24), (3, n + 13)):
        pool = torch.full((m + 2, pitch), 5.0, dtype=F16, device="cuda")
        out = pool[1: m + 1, left: left + n]
        res = torch.randint(-9, 10, (m, n), generator=gen(3)).half()
        out.copy_(res)
        _abi.fp8_linear(out, tuple(t.cuda() for t in x), tuple(t.cuda() for t in w), residual=out)
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), (exact_product(x, w) + res.float()).half())
        out.fill_(5.0)
        assert bool((pool == 5).all())


def test_linear_without_columns():
    x = eff.FP8Rows(torch.empty(3, 0, dtype=U8, device="gcu"), torch.empty(3, 0, dtype=U8, device="gcu"))
    w = eff.FP8Weight(torch.empty(5, 0, dtype=U8, device="gcu"), torch.empty(1, 0, dtype=U8, device="gcu"))
    b = torch.arange(5.0).to(BF16).to("gcu")
    assert torch.equal(eff.fp8_linear(x, w, bias=b).cpu(), torch.arange(5.0).to(BF16).expand(3, 5))
    assert int((eff.fp8_linear_silu_mul(x, w, w).codes.cpu() & 0x7F).sum()) == 0
    x = eff.FP8Rows(torch.empty(200, 0, dtype=U8, device="gcu"), torch.empty(200, 0, dtype=U8, device="gcu"))
    assert torch.equal(eff.fp8_linear(x, w, bias=b).cpu(), torch.arange(5.0).to(BF16).expand(200, 5))
    assert int((eff.fp8_linear_silu_mul(x, w, w).codes.cpu() & 0x7F).sum()) == 0
    none = eff.FP8Rows(torch.empty(0, 16, dtype=U8, device="gcu"), torch.empty(0, 1, dtype=U8, device="gcu"))
    w = eff.FP8Weight(torch.zeros(5, 16, dtype=U8, device="gcu"), torch.zeros(1, 1, dtype=U8, device="gcu"))
    assert eff.fp8_linear(none, w).shape == (0, 5) and eff.fp8_linear_silu_mul(none, w, w).codes.shape == (0, 5)


# ---- gate -------------------------------------------------------------------------

GATES = [(1, 1, 1), (1, 128, 128), (3, 5, 7), (2, 300, 130), (16, 640, 512), (33, 129, 1000), (64, 1000, 384),
         (24, 2000, 4096), (65, 300, 1000), (130, 500, 2051), (200, 1030, 260), (300, 1000, 1104), (1030, 1100, 640),
         (2100, 2050, 272), (2, 11008, 256)]


def small_gates(m, n, k, seed):
    """Whole-number operands with sums of a few units for the gate, so that silu is in
    its curved range."""
    x, wg = whole_numbers(m, n, k, seed)
    _, wu = whole_numbers(m, n, k, seed + 1)
    return x, (wg[0], wg[1] - min(5, int(math.log2(k) / 2))), wu


GATES_LARGE = [(669, 8246, 1185), (3236, 2016, 640), (4869, 404, 1153), (470, 8372, 64), (4800, 137, 4545),
               (81, 2404, 2193), (25, 69, 2528), (147, 207, 1137), (65, 70, 912), (17, 65, 305), (33, 67, 272),
               (3765, 2118, 512), (980, 7194, 640), (5586, 1309, 386), (2188, 2971, 513), (2389, 1667, 128),
               (2968, 1292, 133), (5729, 523, 519), (5959, 561, 395), (80, 4030, 2953), (696, 896, 5120)]


def check_gate(got, gate, up, gate_off=0.0, up_off=0.0):
    y = oracle.silu_mul(gate, up)
    # exp2's argument is rounded (|g| 2^-24 of the exponential) and two fast functions of about
    # an ulp, two products; slope of silu is at most 1.1
    d = (8 + 2 * gate.abs()) * 2.0 ** -23
    extra = 1.1 * gate_off * up.abs() + oracle.silu_mul(gate, torch.ones_like(gate)).abs() * up_off + 1.1 * gate_off * up_off
    check_codes(got, y, d + extra / y.abs().clamp(min=1e-300))


@pytest.mark.parametrize("m,n,k", GATES + GATES_LARGE)
def test_gate_on_whole_numbers(m, n, k):
    x, wg, wu = small_gates(m, n, k, m + n + k)
    got = eff.fp8_linear_silu_mul(gcu(x), gcu(wg, eff.FP8Weight), gcu(wu, eff.FP8Weight))
    assert got.codes.shape == (m, n) and got.scales.shape == (m, -(-n // 128))
    check_gate(got, exact_product(x, wg).double(), exact_product(x, wu).double())


@pytest.mark.parametrize("m,n,k", [(24, 640, 4096), (300, 520, 2100)])
def test_gate_of_ordinary_numbers(m, n, k):
    x, wg = quantized(m, n, k)
    _, wu = quantized(1, n, k, seed=4)
    got = eff.fp8_linear_silu_mul(gcu(x), gcu(wg, eff.FP8Weight), gcu(wu, eff.FP8Weight))
    (g, goff, _), (u, uoff, _) = rounding_of(x, wg), rounding_of(x, wu)
    check_gate(got, g, u, goff, uoff)
    v, y = oracle.numbers(*cpu(got)), oracle.silu_mul(g, u)
    assert float((v - y).norm()) <= 2.0 ** -4 * float(y.norm())  # a code's rounding, at most


def test_gate_of_what_is_not_finite():
    for m, n, k in ((5, 300, 260), (200, 520, 384), (1500, 1200, 128)):
        x, wg, wu = small_gates(m, n, k, 19)
        want = oracle.silu_mul(exact_product(x, wg).double(), exact_product(x, wu).double())
        x[0][1, 3] = wg[0][7, 0] = wu[0][n - 1, k - 1] = 0x7F
        want[1] = want[:, 7] = want[:, n - 1] = math.nan
        got = cpu(eff.fp8_linear_silu_mul(gcu(x), gcu(wg, eff.FP8Weight), gcu(wu, eff.FP8Weight)))
        v = oracle.numbers(*got)
        assert torch.equal(v.isnan(), want.isnan())
        fine = ~want.isnan()
        assert bool(((v - want)[fine].abs() <= 2.0 ** -4 * 1.01 * want[fine].abs() + 2.0 ** -9 * want[fine].abs().max()).all())


def test_gate_overflow_is_nan():
    """A product past float32's range has no code; its neighbours keep theirs."""
    x = (torch.full((1, 16), 0x7E, dtype=U8), torch.full((1, 1), 250, dtype=U8))
    w = (torch.full((3, 16), 0x38, dtype=U8), torch.full((1, 1), 127, dtype=U8))
    w[0][1], w[0][2] = 0, 0x01
    got = eff.fp8_linear_silu_mul(gcu(x), gcu(w, eff.FP8Weight), gcu(w, eff.FP8Weight))
    v = oracle.numbers(*cpu(got))
    assert v.isnan().tolist() == [[True, False, True]] and v[0, 1] == 0


# ---- together ---------------------------------------------------------------------


def layer(cfg, seed=3):
    return {n: w.to("gcu") for n, w in dl.init_weights(cfg, seed).items()}


def serving(cfg, lens, dtype=BF16):
    """An empty cache and index tensors for prompts of these lengths."""
    cache = eff.kv8_cache(pages=4 * len(lens), heads=cfg.heads, head_dim=cfg.head_dim, page=64)
    table = torch.arange(4 * len(lens), dtype=torch.int32).view(len(lens), 4).to("gcu")
    starts = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).to("gcu")
    pos = torch.cat([torch.arange(n) for n in lens]).to("gcu")
    return cache, table, torch.tensor(lens, dtype=torch.int32).to("gcu"), starts, pos


def test_decoder_layer_in_8_bits():
    """The layer on quantised weights: what its operators give one by one, and near the
    layer in 16 bits.  A code is off by 2^-4 at most, uniformly, so by 2^-4 / sqrt(3) of
    a row in the 2-norm; a product of two such by 0.051 of what it is, and the longest
    chain (norm, gate and up, their product's codes, down) by 0.12 of the branch, which is
    a part of the stream it is added to."""
    cfg = dl.LayerConfig(vocab=500, hidden=256, heads=4, head_dim=64, ffn=700)
    weights, lens = layer(cfg), [70, 1, 33]
    quantized = dl.quantize_weights(weights)
    ids = torch.randint(0, 500, (sum(lens),), generator=gen(1)).to("gcu")
    got, q, lse = dl.forward_cached(quantized, ids, cfg, *serving(cfg, lens))
    want, _, _ = dl.forward_cached(weights, ids, cfg, *serving(cfg, lens))
    off = (got.cpu().double() - want.cpu().double()).norm() / want.cpu().double().norm()
    assert got.dtype == BF16 and float(off) <= 0.12
    cache, table, lengths, starts, pos = serving(cfg, lens)
    x = torch.nn.functional.embedding(ids, weights["embed"])
    h, _ = eff.rms_norm_fp8(x, weights["attn_norm"], cfg.eps)
    qkv = [eff.fp8_linear(h, quantized[n]).view(len(ids), 4, 64) for n in ("wq", "wk", "wv")]
    eff.rope_(qkv[0], qkv[1], pos, cfg.theta)
    assert torch.equal(qkv[0].cpu(), q.cpu())
    eff.kv8_append(qkv[1], qkv[2], cache, table, lengths, starts)
    a, lse2 = eff.kv8_attention(qkv[0], cache, table, lengths, starts)
    assert torch.equal(lse2.cpu(), lse.cpu())
    o = eff.fp8_linear(eff.fp8_quantize(a.view(-1, 256)), quantized["wo"])
    h, total = eff.rms_norm_fp8(o, weights["ffn_norm"], cfg.eps, residual=x)
    assert torch.equal(total.cpu(), (o.cpu().float() + x.cpu().float()).to(BF16))
    m = eff.fp8_linear_silu_mul(h, quantized["w_gate"], quantized["w_up"])
    assert torch.equal(eff.fp8_linear(m, quantized["w_down"], residual=total).cpu(), got.cpu())


def chain(x, r, w, wide):
    h, total = eff.rms_norm_fp8(x, None, residual=r)
    m = eff.fp8_linear_silu_mul(h, wide, wide)
    return eff.fp8_linear(m, w, residual=total), eff.fp8_quantize(total)


def chain_inputs(m, k, n, seed):
    x, r = tokens(m, k, BF16, seed).to("gcu"), tokens(m, k, BF16, seed + 1).to("gcu")
    wide = eff.fp8_quantize_weight((0.05 * torch.randn(n, k, generator=gen(seed + 2))).to("gcu"))
    w = eff.fp8_quantize_weight((0.05 * torch.randn(k, n, generator=gen(seed + 3))).to("gcu"))
    return x, r, w, wide


def same(a, b):
    return torch.equal(a[0].cpu(), b[0].cpu()) and all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(a[1], b[1]))


@pytest.mark.parametrize("m", [1, 24, 100, 700])
def test_two_graphs_that_take_turns(m):
    """Captured calls, replayed with new inputs between eager calls of the same operators;
    the two graphs' workspaces (slices of K) are their own."""
    sets = [chain_inputs(m, 1024, 1500, s) for s in (1, 20)]
    graphs, outs = [], []
    for s in sets:
        chain(*s)
        torch.gcu.synchronize()
        g = torch.gcu.GCUGraph()
        with torch.gcu.graph(g):
            outs.append(chain(*s))
        graphs.append(g)
    for turn in range(4):
        for s in sets:
            s[0].copy_(tokens(m, 1024, BF16, 50 + turn).to("gcu"))
        want = [chain(*s) for s in sets]
        torch.gcu.synchronize()
        graphs[0].replay(), graphs[1].replay()
        torch.gcu.synchronize()
        assert same(outs[0], want[0]) and same(outs[1], want[1])


@pytest.mark.parametrize("m", [5, 60, 300])
def test_graph_of_calls_that_copy_their_rows(m):
    """Codes that begin at odd bytes are copied to workspace inside the captured call."""
    k, n = 517, 300
    w = whole_numbers(1, n, k, 4)[1]
    wide = torch.zeros(m, k + 40, dtype=U8, device="gcu")
    rows = eff.FP8Rows(wide[:, 3: 3 + k], torch.full((m, 5), 127, dtype=U8, device="gcu"))
    weight = gcu(w, eff.FP8Weight)

    def calls():
        y = eff.fp8_linear(rows, weight)
        return (y, *eff.fp8_linear_silu_mul(rows, weight, weight))

    def fill(seed):
        code = whole_numbers(m, 1, k, seed)[0][0]
        wide.copy_(torch.nn.functional.pad(code, (3, 37)).to("gcu"))

    fill(1)
    calls()
    torch.gcu.synchronize()
    g = torch.gcu.GCUGraph()
    with torch.gcu.graph(g):
        outs = calls()
    for seed in range(2, 6):
        fill(seed)
        want = calls()
        torch.gcu.synchronize()
        g.replay()
        torch.gcu.synchronize()
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(outs, want))


@pytest.mark.parametrize("m", [1, 9, 70])
def test_linear_of_the_most_columns(m):
    """Longer rows than the few-row kernel has room for scales; offsets near 2^30 bytes."""
    k, n = (1 << 22) - 16, 70
    at = torch.cat([torch.randint(0, k, (500,), generator=gen(2)), torch.tensor([0, k - 1, k - 17])])
    x, w = torch.zeros(m, k, dtype=U8), torch.zeros(n, k, dtype=U8)
    xs, ws = whole_numbers(m, n, len(at), 5)
    x[:, at], w[:, at] = xs[0], ws[0]
    scale = lambda r: torch.full((r, -(-k // 128)), 127, dtype=U8)  # noqa: E731
    got = eff.fp8_linear(gcu((x, scale(m))), gcu((w, scale(1)), eff.FP8Weight))
    value = lambda t: t.view(torch.float8_e4m3fn).double()  # noqa: E731
    assert torch.equal(got.cpu().double(), (value(x) @ value(w).t()).to(BF16).double())


def test_two_streams_at_once():
    sets = [chain_inputs(24, 2048, 1500, s) for s in (1, 20)]
    want = [chain(*s) for s in sets]
    torch.gcu.synchronize()
    streams = [torch.gcu.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.gcu.stream(st):
                got[i].append(chain(*sets[i]))
    torch.gcu.synchronize()
    assert all(same(g, want[i]) for i in range(2) for g in got[i])


def test_results_do_not_depend_on_the_run():
    s = chain_inputs(24, 4096, 3000, 2)
    first = chain(*s)
    assert all(same(chain(*s), first) for _ in range(5))


def test_refusals_through_the_public_entry_points():
    x = torch.zeros(4, 256, dtype=BF16, device="gcu")
    r, w = eff.fp8_quantize(x), eff.fp8_quantize_weight(x)
    for call, words in (
            (lambda: eff.fp8_quantize(x.cpu()), "PrivateUse1|gcu|CPU"),
            (lambda: eff.fp8_quantize(x.double()), "float32"),
            (lambda: eff.fp8_quantize_weight(x[0]), "2-D"),
            (lambda: eff.rms_norm_fp8(x, x[0, :5]), "weight must be"),
            (lambda: eff.rms_norm_fp8(x, None, residual=x[:2]), "residual must have"),
            (lambda: eff.rms_norm_fp8(x, x[0].cpu()), "gcu"),
            (lambda: eff.fp8_linear(r, w, dtype=torch.float32), "bfloat16 or float16"),
            (lambda: eff.fp8_linear(r, eff.FP8Weight(w.codes[:, :128], w.scales[:, :1])), "columns"),
            (lambda: eff.fp8_linear(eff.FP8Rows(r.codes, r.scales[:2]), w), "scales"),
            (lambda: eff.fp8_linear(r, w, residual=x), "residual has shape"),
            (lambda: eff.fp8_linear(r, w, bias=x[0]), "bias"),
            (lambda: eff.fp8_linear_silu_mul(r, w, eff.FP8Weight(w.codes[:3], w.scales)), "different shapes"),
    ):
        with pytest.raises((RuntimeError, NotImplementedError), match=words):
            call()
