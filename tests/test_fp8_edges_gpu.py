"""Edges of the 8-bit linear layers on the GPU."""
import math

import pytest
import torch

import torch_gcu  # noqa: F401
from oracle import fp8 as oracle
from test_fp8_linear_gpu import check_gate, cpu, eff, exact_product, gcu, gen, layer, small_gates, tokens, whole_numbers
from test_fp8_rule_cpu import GATE, LINEAR
from torch_gcu import _abi
from torch_gcu.utils import decoder_layer as dl

pytestmark = pytest.mark.gpu
BF16, F16, U8 = torch.bfloat16, torch.float16, torch.uint8


# ---- the decoder layer --------------------------------------------------------------


@pytest.mark.parametrize("kv_heads", [4, 1])
@pytest.mark.parametrize("tokens", [0, 3])
def test_decoder_layer_of_no_and_few_tokens(tokens, kv_heads):
    """A step in which no sequence has a new token gives empty results, and shapes are
    those of the layer in 16 bits."""
    cfg = dl.LayerConfig(vocab=100, hidden=256, heads=4, head_dim=64, ffn=300)
    weights = layer(cfg)
    for n in ("wk", "wv"):
        weights[n] = weights[n][: kv_heads * 64].contiguous()
    cache = eff.kv8_cache(pages=2, heads=kv_heads, head_dim=64, page=64)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).to("gcu")  # noqa: E731
    ids = torch.arange(tokens).to("gcu")
    args = (ids, cfg, cache, i32([[0, 1]]), i32([5]), i32([0, tokens]), ids)
    want = dl.forward_cached(weights, *args)
    got = dl.forward_cached(dl.quantize_weights(weights), *args)
    for g, w in zip(got, want):
        assert g.shape == w.shape and g.dtype == w.dtype
    torch.gcu.synchronize()


# ---- every kernel of a product --------------------------------------------------------


def ids_of(ways):
    return [(way, *size) for way, sizes in ways.items() for size in sizes]


def one_of(ways):
    """The first size of each way."""
    return [(way, *sizes[0]) for way, sizes in ways.items()]


@pytest.mark.parametrize("way,m,n,k", ids_of(LINEAR))
def test_linear_in_place_by_every_way(way, m, n, k):
    """Bias and a residual that is the output itself, in rows of odd pitch between others."""
    x, w = whole_numbers(m, n, k, m + n + k)
    bias = torch.randint(-8, 9, (n,), generator=gen(1)).to(F16)
    res = torch.randint(-64, 65, (m, n), generator=gen(2)).to(F16)
    want = (exact_product(x, w) + bias.float() + res.float()).to(F16)
    pool = torch.full((m + 2, n + 13), 5.0, dtype=F16, device="cuda")
    out = pool[1: m + 1, 3: 3 + n]
    out.copy_(res)
    xc, wc = (tuple(t.cuda() for t in p) for p in (x, w))
    _abi.fp8_linear(out, xc, wc, bias=bias.cuda(), residual=out)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want)
    out.fill_(5.0)
    assert bool((pool == 5).all())


@pytest.mark.parametrize("way,m,n,k", one_of(LINEAR))
def test_linear_of_what_is_not_finite_by_every_way(way, m, n, k):
    """NaN codes at the first and last K of rows and columns, and NaN scales of a row's and
    a block's first and last groups: they make NaN there and nowhere else."""
    x, w = whole_numbers(m, n, k, 11)
    want = exact_product(x, w).to(BF16)
    x[0][1, 3] = x[0][4, k - 1] = w[0][7, 0] = w[0][n - 1, k - 1] = 0x7F
    x[1][2, -1] = x[1][6, 0] = 255
    want[[1, 2, 4, 6]] = math.nan
    want[:, [7, n - 1]] = math.nan
    got = eff.fp8_linear(gcu(x), gcu(w, eff.FP8Weight)).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    if n > 128:  # the second block of the weight
        w[1][1, -1] = 255
        want[:, 128:256] = math.nan
        got = eff.fp8_linear(gcu(x), gcu(w, eff.FP8Weight)).cpu()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("way,m,n,k", one_of(LINEAR))
def test_linear_of_the_largest_and_smallest_scales_by_every_way(way, m, n, k):
    """2^-127 and 2^127 against each other give what 1 and 1 do; alone, sums under float32's
    normal range may be 0 and those above it are not finite."""
    (x, xs), (w, ws) = whole_numbers(m, n, k, 23)
    base = exact_product((x, torch.full_like(xs, 127)), (w, torch.full_like(ws, 127))).double()
    for a, b in ((0, 254), (254, 0), (0, 127), (254, 127), (1, 1)):
        got = eff.fp8_linear(gcu((x, torch.full_like(xs, a))),
                             gcu((w, torch.full_like(ws, b)), eff.FP8Weight)).cpu()
        want = (base * 2.0 ** (a + b - 254)).float().to(BF16)
        if a + b > 370:
            assert bool(((got == want) | ~got.isfinite()).all()), (a, b)
        elif a + b < 128:
            assert bool(((got.double() - want.double()).abs() <= 2.0 ** -126).all()), (a, b)
        else:
            assert torch.equal(got, want), (a, b)


@pytest.mark.parametrize("way,m,n,k", ids_of(GATE))
def test_gate_by_every_way(way, m, n, k):
    """Codes and scales into rows of odd pitch between others."""
    x, wg, wu = small_gates(m, n, k, m + n + k)
    groups = -(-n // 128)
    code = torch.full((m + 2, n + 13), 77, dtype=U8, device="cuda")
    byte = torch.full((m + 2, groups + 3), 77, dtype=U8, device="cuda")
    out = code[1: m + 1, 3: 3 + n], byte[1: m + 1, 1: 1 + groups]
    _abi.fp8_linear_silu_mul(out, *(tuple(t.cuda() for t in p) for p in (x, wg, wu)))
    torch.cuda.synchronize()
    check_gate(out, exact_product(x, wg).double(), exact_product(x, wu).double())
    out[0].fill_(77), out[1].fill_(77)
    assert bool((code == 77).all()) and bool((byte == 77).all())


@pytest.mark.parametrize("way,m,n,k", one_of(GATE))
def test_gate_of_what_is_not_finite_by_every_way(way, m, n, k):
    x, wg, wu = small_gates(m, n, k, 19)
    want = oracle.silu_mul(exact_product(x, wg).double(), exact_product(x, wu).double())
    x[0][1, 3] = x[0][4, k - 1] = wg[0][7, 0] = wu[0][n - 1, k - 1] = 0x7F
    x[1][2, -1] = 255
    want[[1, 2, 4]] = want[:, [7, n - 1]] = math.nan
    got = cpu(eff.fp8_linear_silu_mul(gcu(x), gcu(wg, eff.FP8Weight), gcu(wu, eff.FP8Weight)))
    v = oracle.numbers(*got)
    assert torch.equal(v.isnan(), want.isnan())
    # what is left is rounded to codes alone: by 2^-4 of a value at most, or half the least
    # step under the scale of its group, which is at most 2 amax / 448: 2^-10 of that
    fine = ~want.isnan()
    amax = oracle.blocks(want.nan_to_num().abs(), 1).amax((1, 3)).repeat_interleave(128, 1)[:, :n]
    assert bool(((v - want).abs()[fine] <= (2.0 ** -4 * 1.01 * want.abs() + 2.0 ** -10 * amax / 224)[fine]).all())


# ---- workspaces: captured, on two streams, again and again ------------------------------

# a product and a gate of the same x: slices of K in two and four, the few-row kernels
# whose gates go through memory, tiles
TOGETHER = [((8, 101, 266), (8, 101, 269)), ((56, 4201, 3871), (65, 4313, 2683)), ((65, 115, 2056), (69, 101, 1293)),
            ((32, 1003, 1037), (40, 101, 135)), ((211, 8347, 391), (67, 105, 514))]


def operands(sizes, seed):
    """For each size activations, two weights and a residual, of ordinary numbers."""
    made = []
    for m, n, k in sizes:
        x = eff.fp8_quantize(tokens(m, k, BF16, seed).to("gcu"))
        w = [eff.fp8_quantize_weight((0.05 * torch.randn(n, k, generator=gen(seed + i))).to("gcu")) for i in (1, 2)]
        made.append((x, *w, torch.randn(m, n, generator=gen(seed + 3)).to(BF16).to("gcu")))
    return made


def calls(linear, gate):
    y = eff.fp8_linear(linear[0], linear[1], residual=linear[3])
    return [y, *eff.fp8_linear_silu_mul(gate[0], gate[1], gate[2])]


def equal(a, b):
    return all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(a, b))


def refill(made, seed):
    for (x, *_), i in zip(made, range(2)):
        new = eff.fp8_quantize(tokens(*x.codes.shape, BF16, seed + i).to("gcu"))
        x.codes.copy_(new.codes)
        x.scales.copy_(new.scales)


@pytest.mark.parametrize("sizes", TOGETHER)
def test_two_graphs_by_ways_with_workspaces(sizes):
    """Two captured graphs of the same sizes, replayed with new inputs in turn, between eager
    calls and over each other's freed memory."""
    sets = [operands(sizes, s) for s in (1, 20)]
    graphs, outs = [], []
    for s in sets:
        calls(*s)
        torch.gcu.synchronize()
        g = torch.gcu.GCUGraph()
        with torch.gcu.graph(g):
            outs.append(calls(*s))
        graphs.append(g)
    for turn in range(4):
        for i, s in enumerate(sets):
            refill(s, 50 + 10 * turn + i)
        want = [calls(*s) for s in sets]
        torch.gcu.synchronize()
        for i in ((0, 1), (1, 0))[turn % 2]:
            graphs[i].replay()
        torch.gcu.synchronize()
        assert equal(outs[0], want[0]) and equal(outs[1], want[1]), turn


@pytest.mark.parametrize("sizes", TOGETHER)
def test_two_streams_at_once_by_ways_with_workspaces(sizes):
    sets = [operands(sizes, s) for s in (1, 20)]
    want = [calls(*s) for s in sets]
    torch.gcu.synchronize()
    streams, got = [torch.gcu.Stream() for _ in sets], [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.gcu.stream(st):
                got[i].append(calls(*sets[i]))
    torch.gcu.synchronize()
    assert all(equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.parametrize("way,m,n,k", one_of(LINEAR) + one_of(GATE))
def test_results_of_every_way_do_not_depend_on_the_run(way, m, n, k):
    s = operands([(m, n, k), (m, n, k)], 2)
    first = calls(*s)
    assert all(equal(calls(*s), first) for _ in range(3))
