"""The 8-bit key/value cache on the GPU against its definition in 64 bits.

Tolerances are sums of what the kernels round.  With u = eps / 2 of the queries'
type and f = 2^-24: scores are fp32 sums of exact products, off by at most
(D + 8) f times the row's largest sum of |q k| scale (`reach`), which moves a
softmax weight by that share, twice over (the weight and the sum); each weight
is rounded to q's type (u, and under f16's normal range 2^-25 of the largest
value) and the output once more (u).  Codes, scales and kept positions are exact."""
import math
import os
import subprocess
import sys

import pytest
import torch

import torch_gcu  # noqa: F401
from oracle import kv8 as oracle
from torch_gcu import _abi
from torch_gcu.utils import decoder_layer as dl

pytestmark = pytest.mark.gpu
eff = torch.gcu.efficient if hasattr(torch, "gcu") else None
F = 2.0 ** -24


def gen(seed):
    return torch.Generator().manual_seed(seed)


class Setup:
    """Sequences over a shuffled pool: `new` tokens behind `past` cached ones of
    each.  Slots that no token of a sequence occupies hold NaN codes."""

    def __init__(self, new, past, h, hk, d, page, dtype=torch.bfloat16, pad=0, seed=0, spare=3, width=0):
        g = gen(seed)
        self.new, self.h, self.hk, self.d, self.page, self.dtype = new, h, hk, d, page, dtype
        self.lens = [n + p for n, p in zip(new, past)]
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1] + pad
        need = [-(-n // page) for n in self.lens]
        self.pages = max(1, sum(need) + spare)
        order = torch.randperm(self.pages, generator=g).tolist()
        self.width = max([1, width] + need)
        self.table = [[order.pop() for _ in range(n)] for n in need]
        self.free = order
        self.q = (1.5 * torch.randn(self.tokens, h, d, generator=g)).to(dtype)
        self.k = torch.randn(self.tokens, hk, d, generator=g).to(dtype)
        self.v = torch.randn(self.tokens, hk, d, generator=g).to(dtype)
        codes = [torch.full((self.pages, hk, page, d), 0x7F, dtype=torch.uint8) for _ in range(2)]
        scales = [torch.full((self.pages, hk), math.nan) for _ in range(2)]
        self.cache = (*codes, *scales)
        # the past, written by the oracle
        old = torch.randn(2, sum(past), hk, d, generator=g).to(dtype)
        at = [0]
        for n in past:
            at.append(at[-1] + n)
        oracle.append(self.cache, old[0], old[1], self.table, past, at)

    def index(self, lens=None, table=None):
        rows = [t + [-1] * (self.width - len(t)) for t in (table or self.table)]
        return [torch.tensor(x, dtype=torch.int32).reshape(shape).to("gcu") for x, shape in
                ((rows, (len(rows), self.width)), (lens or self.lens, (-1,)), (self.starts, (-1,)))]

    def fill(self):
        """The new tokens into the CPU cache too."""
        oracle.append(self.cache, self.k, self.v, self.table, self.lens, self.starts)
        return self

    def gcu(self):
        return eff.KV8Cache(*(t.to("gcu") for t in self.cache))


def check_attention(s, out, lse, scale=None, rows=None):
    scale = s.d ** -0.5 if scale is None else scale
    want, log, (mass, reach) = oracle.attention(s.q, s.cache, s.table, s.lens, s.starts, scale)
    u = torch.finfo(s.dtype).eps / 2
    err = (s.d + 8) * F * reach + 2.0 ** -21  # the exp2 unit, the log2(e) factor
    tol = mass * (u + 2 * err[..., None]) + u * want.abs() + 1e-30
    if s.dtype == torch.float16:
        tol = tol + max(s.lens) * 2.0 ** -25 * 2 * mass.nan_to_num(nan=0.0).amax() + 2.0 ** -25
    got = out.cpu().double()
    rows = slice(None) if rows is None else rows
    off = ((got - want).abs() / tol)[rows]
    assert not off.isnan().any(), "NaN"
    assert off.numel() == 0 or off.max() <= 1, f"out {off.max()} of the tolerance"
    got, log, err = lse.cpu().double()[rows], log[rows], err[rows]
    assert torch.equal(got.isinf(), log.isinf())
    fine = log.isfinite()
    off = (got - log).abs()[fine] / (err + 4 * F * log.abs())[fine]
    assert off.numel() == 0 or off.max() <= 1, f"lse {off.max()} of the tolerance"


SHAPES = [
    # new, past, h, hk, d, page
    ([1], [0], 4, 4, 128, 64),                       # one token, its own first
    ([1], [300], 32, 8, 128, 64),
    ([1, 1, 1], [63, 64, 65], 8, 2, 128, 64),        # around a page's end
    ([1, 1, 1, 1], [15, 16, 31, 32], 5, 1, 64, 16),  # small pages, five heads to one
    ([1, 0, 1, 0], [500, 77, 0, 0], 8, 8, 64, 32),   # sequences without new tokens, without any
    ([1] * 70, [3 * i for i in range(70)], 2, 1, 64, 16),  # more than a wave of sequences
    ([5, 1, 3], [1000, 9, 255], 16, 4, 128, 16),
    ([1, 1], [4000, 1], 32, 4, 128, 256),            # cut in parts, beside one that is not
    ([2, 7], [3000, 2222], 6, 2, 64, 128),
    ([17, 40], [0, 100], 4, 4, 128, 32),
    ([33, 130, 1], [70, 0, 500], 8, 2, 128, 64),     # pieces of prompts beside a decode step
    ([257], [129], 24, 8, 64, 64),
    ([300, 5], [1500, 2000], 8, 8, 128, 16),
    ([600], [0], 3, 1, 128, 128),
    ([64, 64], [64, 0], 16, 2, 64, 256),
    ([1024], [3700], 64, 8, 64, 256),                # 256 blocks of 256 rows
    ([515, 500], [4000, 3333], 32, 32, 128, 64),     # and rows that do not fill them
    ([40, 1], [100, 33], 80, 1, 128, 64),            # more heads to one than a tile has rows
    ([70, 33], [200, 0], 14, 2, 64, 32),             # seven heads to one
    ([90, 70], [1500, 1000], 16, 8, 64, 32),         # blocks of 128 keys for most of the CUs
    ([40], [9000], 80, 1, 64, 256),                  # the same, of more heads to one than a tile has rows
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new,past,h,hk,d,page", SHAPES)
def test_append_and_attention(new, past, h, hk, d, page, dtype):
    s = Setup(new, past, h, hk, d, page, dtype, seed=len(new) + h)
    cache, index = s.gcu(), s.index()
    eff.kv8_append(s.k.to("gcu"), s.v.to("gcu"), cache, *index)
    s.fill()
    for got, want in zip(cache, s.cache):
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))
    out, lse = eff.kv8_attention(s.q.to("gcu"), cache, *index)
    assert out.dtype == dtype and lse.dtype == torch.float32
    check_attention(s, out, lse)


def wide_table(rows, heads, page):
    """Columns of a block table with which a call of few tokens counts as one of
    prompts (rows: new tokens x heads of a group, over 64 a sequence)."""
    return (1 << 23) // (rows * heads * page) + 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new,past,h,hk,d,page", [
    ([17, 40], [0, 100], 16, 4, 128, 32),
    ([33, 130, 1], [70, 0, 500], 8, 2, 128, 64),
    ([257], [129], 24, 8, 64, 64),
    ([300, 5], [1500, 2000], 8, 8, 128, 16),
    ([300, 0, 70], [100, 700, 1], 14, 2, 64, 16),  # seven heads to one, a sequence without new tokens
    ([600], [0], 3, 1, 128, 128),
    ([40, 1], [100, 33], 80, 1, 128, 64),
    ([1, 90, 64], [300, 0, 64], 16, 2, 64, 256),
    ([3] * 67, [5 * i for i in range(67)], 23, 1, 64, 16),  # more than a wave of sequences
])
def test_prompts_of_few_tokens(new, past, h, hk, d, page, dtype):
    s = Setup(new, past, h, hk, d, page, dtype, seed=len(new) + h,
              width=wide_table(sum(new) * h // hk, hk, page)).fill()
    out, lse = eff.kv8_attention(s.q.to("gcu"), s.gcu(), *s.index())
    check_attention(s, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new,past,h,hk,d,page", SHAPES)
def test_weigh(new, past, h, hk, d, page, dtype):
    s = Setup(new, past, h, hk, d, page, dtype, seed=3 + len(new)).fill()
    scale = d ** -0.5
    _, log, (_, reach) = oracle.attention(s.q, s.cache, s.table, s.lens, s.starts, scale)
    lse = log.float()
    before = torch.rand(len(new), hk, s.width * page + 5, generator=gen(1))
    want, added = before.double(), torch.zeros(before.shape, dtype=torch.float64)
    oracle.attention(s.q, s.cache, s.table, s.lens, s.starts, scale, added, lse)
    w = before.to("gcu")
    got = eff.kv8_weigh_(w, s.q.to("gcu"), lse.to("gcu"), s.gcu(), *s.index())
    assert got is w
    # per weight the score's error, lse's and exp2's; then an fp32 sum of at most rows terms
    rows = max(new + [1]) * h // hk
    fine = torch.where(log.isfinite(), log.abs(), 0.0)
    err = (d + 8) * F * float(reach.max()) + 4 * F * float(fine.max()) + 2.0 ** -21 + rows * F
    want += added
    off = (w.cpu().double() - want).abs() / (added * err + F * want)
    assert off.max() <= 1, f"{off.max()} of the tolerance"
    for b, n in enumerate(s.lens):
        assert torch.equal(w[b, :, n:].cpu(), before[b, :, n:])


EVICT = [
    # lens, keep, recent, sink, hk, d, page
    ([1000], 250, 64, 4, 8, 128, 64),
    ([1], 1, 0, 0, 1, 64, 16),
    ([5, 0, 16, 17], 16, 4, 2, 2, 64, 16),            # shorter than, as long as, one over
    ([100, 333, 64], 64, 64, 0, 3, 128, 32),          # the last ones only
    ([100, 333], 40, 0, 40, 2, 64, 64),               # the first ones only
    ([700, 2500, 1025], 600, 0, 0, 2, 128, 16),       # by weight alone
    ([3000], 1, 0, 0, 4, 64, 256),
    ([4097, 2048, 1024], 1023, 100, 1, 2, 128, 128),
    ([40000, 16385, 16384], 9000, 300, 4, 1, 64, 256),  # longer than what a block holds
]


@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("lens,keep,recent,sink,hk,d,page", EVICT)
def test_evict(lens, keep, recent, sink, hk, d, page, kind):
    need = -(-keep // page)
    s = Setup([0] * len(lens), lens, hk, hk, d, page, seed=keep, spare=need * len(lens) + 1)
    fresh = [[s.free.pop() for _ in range(need)] for _ in lens]
    g = gen(keep)
    w = torch.rand(len(lens), hk, s.width * page + 3, generator=g) ** 4
    if kind == "ties":
        w = (w * 3).round() - 0.0
        w[w == 1] = -0.0
    elif kind == "odd":
        bad = torch.randint(0, 5, w.shape, generator=g)
        w = torch.where(bad == 0, math.nan, torch.where(bad == 1, math.inf, torch.where(bad == 2, -w, w)))
    cache, index = s.gcu(), s.index()
    new_table = torch.tensor(fresh, dtype=torch.int32).to("gcu")
    kept, left, moved = eff.kv8_evict(cache, w.to("gcu"), index[0], new_table, index[1], keep, recent, sink)
    k, n, m = oracle.evict(s.cache, w, s.table, fresh, lens, keep, recent, sink)
    assert left.cpu().tolist() == n
    assert torch.equal(kept.cpu(), k)
    assert torch.equal(moved.cpu().nan_to_num(nan=7e30), m.nan_to_num(nan=7e30))
    for got, want in zip(cache, s.cache):
        got = got.cpu()
        if got.dtype == torch.uint8:  # 0 and -0 are one number
            got, want = (torch.where(x == 0x80, 0, x.int()) for x in (got, want))
        assert torch.equal(got.nan_to_num(nan=-1.0) if got.is_floating_point() else got,
                           want.nan_to_num(nan=-1.0) if want.is_floating_point() else want)


def test_a_run_of_them_together():
    """A prompt in two pieces, decode steps with the weights added up, eviction,
    and more decode steps on what is left, with another sequence beside it."""
    h, hk, d, page, keep = 8, 2, 128, 32, 100
    g = gen(5)
    lens, W = [0, 0], 16
    pages = list(range(64))
    tables = [[pages.pop() for _ in range(W)] for _ in lens]
    cache = eff.kv8_cache(64, hk, d, page)
    cpu = tuple(t.cpu() for t in cache)
    weights = torch.zeros(2, hk, W * page).to("gcu")
    expect = torch.zeros(2, hk, W * page, dtype=torch.float64)
    for step, new in enumerate([[200, 33], [100, 20], [1, 1], [1, 1], "evict", [1, 1], [1, 0], [40, 2]]):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32).to("gcu")  # noqa: E731
        if new == "evict":
            fresh = [[pages.pop() for _ in range(4)] for _ in lens]
            kept, left, weights = eff.kv8_evict(cache, weights, i32(tables), i32(fresh), i32(lens), keep, 16, 2)
            # by the device's weights: the oracle's could tell near ties otherwise
            k, n, m = oracle.evict(cpu, before, tables, fresh, lens, keep, 16, 2)
            assert torch.equal(kept.cpu(), k) and left.cpu().tolist() == n
            expect, lens = m.double(), n
            tables = [f + [pages.pop() for _ in range(2)] + [0] * (W - 6) for f in fresh]
            continue
        lens = [a + b for a, b in zip(lens, new)]
        starts = [0, new[0], sum(new)]
        q = torch.randn(sum(new), h, d, generator=g).bfloat16()
        k, v = (torch.randn(sum(new), hk, d, generator=g).bfloat16() * (1 + step) for _ in range(2))
        index = [i32(tables), i32(lens), i32(starts)]
        eff.kv8_append(k.to("gcu"), v.to("gcu"), cache, *index)
        out, lse = eff.kv8_attention(q.to("gcu"), cache, *index)
        eff.kv8_weigh_(weights, q.to("gcu"), lse, cache, *index)
        oracle.append(cpu, k, v, tables, lens, starts)
        s = Setup.__new__(Setup)
        s.q, s.cache, s.table, s.lens, s.starts, s.d, s.dtype = q, cpu, tables, lens, starts, d, q.dtype
        check_attention(s, out, lse)
        oracle.attention(q, cpu, tables, lens, starts, d ** -0.5, expect, lse.cpu())
        before = weights.cpu()
        assert torch.allclose(before.double(), expect, rtol=1e-4, atol=1e-6)
    for got, want in zip(cache, cpu):
        assert torch.equal(got.cpu(), want)


def test_tokens_one_by_one_as_together():
    """Page scales that grow token by token end where they would have begun."""
    s = Setup([100], [0], 4, 2, 64, 32, seed=9)
    s.k *= torch.logspace(-2, 2, 100)[:, None, None].to(s.dtype)
    together, single = s.gcu(), s.gcu()
    eff.kv8_append(s.k.to("gcu"), s.v.to("gcu"), together, *s.index())
    for i in range(100):
        lens, starts = (torch.tensor(x, dtype=torch.int32).to("gcu") for x in ([i + 1], [0, 1]))
        eff.kv8_append(s.k[i: i + 1].to("gcu"), s.v[i: i + 1].to("gcu"), single, s.index()[0], lens, starts)
    pages = s.table[0]
    for a, b in zip(together[2:], single[2:]):
        assert torch.equal(a.cpu()[pages], b.cpu()[pages])
    for a, b, scale in zip(together[:2], single[:2], together[2:]):
        x, y = (oracle.values(t.cpu()[pages]) for t in (a, b))
        x, y = (t.flatten(0, 0).transpose(1, 2).reshape(-1, 2, 64) for t in (x, y))
        # a code that became subnormal on the way was rounded there: up to half
        # a step of 2^-9, and again when the scale grew further (a geometric sum)
        assert (x[:100] - y[:100]).abs().max() <= 2.0 ** -9


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("wide", [False, True])
def test_non_finite_tokens_reach_only_who_sees_them(bad, dtype, wide):
    """Token 50 of 70 has a bad key, token 60 a bad value element: the queries
    before them stay what they were, those after are NaN."""
    s = Setup([70, 1], [0, 40], 4, 2, 128, 32, dtype, seed=2, width=wide_table(142, 2, 32) if wide else 0)
    s.k[50, 1, 3], s.v[60, 0, 100] = bad, bad
    cache, index = s.gcu(), s.index()
    eff.kv8_append(s.k.to("gcu"), s.v.to("gcu"), cache, *index)
    s.fill()
    for got, want in zip(cache, s.cache):
        assert torch.equal(got.cpu().view(torch.uint8) & 0x7F, want.view(torch.uint8) & 0x7F)
    out, lse = eff.kv8_attention(s.q.to("gcu"), cache, *index)
    o, e = out.cpu(), lse.cpu()
    group0, group1 = slice(0, 2), slice(2, 4)
    assert o[60:70, group0].isnan().all() and e[60:70, group0].isnan().all()
    assert o[50:70, group1].isnan().all() and e[50:70, group1].isnan().all()
    for h, until in ((group0, 60), (group1, 50)):
        assert o[:until, h].isfinite().all() and o[70:, h].isfinite().all()
    check_attention(s, out, lse, rows=slice(0, 50))
    check_attention(s, out, lse, rows=slice(70, 71))


def test_queries_without_keys_and_rows_of_no_sequence():
    """More new tokens than the cache holds: the first see nothing.  Rows behind
    the last sequence get 0 and -inf, or are left alone through the C ABI."""
    s = Setup([6, 3], [0, 20], 4, 2, 64, 16, pad=5, seed=4)
    s.fill()
    s.lens[0] = 4  # tokens 0 and 1 of sequence 0 come before position 0
    cache, index = s.gcu(), s.index()
    out, lse = eff.kv8_attention(s.q.to("gcu"), cache, *index)
    assert (out[:2] == 0).all().item() and (lse[:2] == -math.inf).all().item()
    assert (out[9:] == 0).all().item() and (lse[9:] == -math.inf).all().item()
    check_attention(s, out, lse)
    dev = [t.cuda() for t in (s.q, *s.cache)]
    o, e = torch.full(s.q.shape, 7.0, dtype=s.dtype, device="cuda"), torch.full((14, 4), 7.0, device="cuda")
    _abi.install_workspace()
    _abi.kv8_attention(o, e, dev[0], dev[1:], *(t.cpu().cuda() for t in index))
    assert (o[9:] == 7).all() and (e[9:] == 7).all()
    assert torch.equal(o[:9].cpu(), out[:9].cpu()) and torch.equal(e[:9].cpu(), lse[:9].cpu())
    w = torch.zeros(2, 2, s.width * 16).to("gcu")
    eff.kv8_weigh_(w, s.q.to("gcu"), lse, cache, *index)
    want = torch.zeros(w.shape, dtype=torch.float64)
    oracle.attention(s.q, s.cache, s.table, s.lens, s.starts, s.d ** -0.5, want, lse.cpu())
    assert torch.allclose(w.cpu().double(), want, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("new,width", [(1, 40), (200, 40), (200, 2000)])
def test_scales_of_pages_that_are_not_there(new, width):
    """Table entries behind a sequence's last page name none; page 0, whose
    scales are NaN, is not the sequence's and must not come in for them."""
    s = Setup([new], [33], 8, 2, 64, 16, width=width, seed=3)
    at = s.table[0].index(0) if 0 in s.table[0] else None
    if at is not None:  # page 0 to the free ones
        s.table[0][at] = s.free.pop()
    s.cache = tuple(torch.full_like(t, 0x7F if t.dtype == torch.uint8 else math.nan) for t in s.cache)
    old = torch.randn(2, 33, 2, 64, generator=gen(4)).to(s.dtype)
    oracle.append(s.cache, old[0], old[1], s.table, [33], [0, 33])
    s.fill()
    assert s.cache[2][0].isnan().all() and s.cache[3][0].isnan().all()
    out, lse = eff.kv8_attention(s.q.to("gcu"), s.gcu(), *s.index())
    check_attention(s, out, lse)
    w = torch.zeros(1, 2, s.width * 16).to("gcu")
    eff.kv8_weigh_(w, s.q.to("gcu"), lse, s.gcu(), *s.index())
    assert w.isfinite().all().item()


def test_prompts_without_keys_bad_pages_and_starts():
    """The same of a call of prompts: tokens before position 0, rows of no
    sequence, a page outside the pool, lengths and starts out of range."""
    s = Setup([200, 130], [0, 20], 4, 2, 64, 16, pad=5, seed=4, width=wide_table(670, 2, 16)).fill()
    s.lens[0] = 150  # tokens 0 .. 49 of sequence 0 come before position 0
    cache, index = s.gcu(), s.index()
    out, lse = eff.kv8_attention(s.q.to("gcu"), cache, *index)
    for empty in (slice(0, 50), slice(330, 335)):
        assert (out[empty] == 0).all().item() and (lse[empty] == -math.inf).all().item()
    check_attention(s, out, lse)
    w = torch.zeros(2, 2, s.width * 16).to("gcu")
    eff.kv8_weigh_(w, s.q.to("gcu"), lse, cache, *index)
    want = torch.zeros(2, 2, s.width * 16, dtype=torch.float64)
    oracle.attention(s.q, s.cache, s.table, s.lens, s.starts, s.d ** -0.5, want, lse.cpu())
    assert torch.allclose(w.cpu().double(), want, rtol=1e-4, atol=1e-6)
    torch.gcu.synchronize()

    bad = [list(t) for t in s.table]
    bad[1][2] = s.pages
    index[0] = s.index(table=bad)[0]
    got, log = eff.kv8_attention(s.q.to("gcu"), cache, *index)
    with pytest.raises(IndexError, match=f"index {s.pages} is out of bounds"):
        torch.gcu.synchronize()
    assert torch.equal(got[:200].cpu(), out[:200].cpu()) and torch.equal(log[:200].cpu(), lse[:200].cpu())
    assert got.cpu().isfinite().all()
    # as if the page's 16 positions did not exist
    keys = oracle.tokens(s.cache[0][:, 0], s.cache[2][:, 0], s.table[1], s.lens[1])
    scores = torch.cat([keys[:32], keys[48:]]) @ s.q[329, 0].double() * s.d ** -0.5
    assert abs(float(log[329, 0]) - float(scores.logsumexp(0))) < 1e-4
    index = s.index(lens=[s.lens[0], -7])
    got, log = eff.kv8_attention(s.q.to("gcu"), cache, *index)
    with pytest.raises(IndexError, match="index -7 is out of bounds"):
        torch.gcu.synchronize()
    assert torch.equal(got[:200].cpu(), out[:200].cpu())
    assert (got[200:] == 0).all().item() and (log[200:] == -math.inf).all().item()
    index = s.index()
    for starts in ([5, 2, 335], [0, 1000, 8], [-3, 4, 2 ** 31 - 1], [335, 335, 0], [0, 335, -2 ** 31]):
        index[2] = torch.tensor(starts, dtype=torch.int32).to("gcu")
        got, log = eff.kv8_attention(s.q.to("gcu"), cache, *index)
        torch.gcu.synchronize()
        assert got.shape == s.q.shape
        eff.kv8_weigh_(w, s.q.to("gcu"), log, cache, *index)
        torch.gcu.synchronize()


def test_no_sequences_and_no_tokens():
    cache = eff.kv8_cache(2, 2, 64, 16)
    none = torch.zeros(0, dtype=torch.int32).to("gcu")
    table, one = torch.zeros(0, 1, dtype=torch.int32).to("gcu"), torch.zeros(1, dtype=torch.int32).to("gcu")
    q = torch.randn(3, 4, 64).bfloat16().to("gcu")
    out, lse = eff.kv8_attention(q, cache, table, none, one)
    assert (out == 0).all().item() and (lse == -math.inf).all().item()
    out, lse = eff.kv8_attention(q[:0], cache, table, none, one)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    eff.kv8_append(q[:0, :2], q[:0, :2], cache, table, none, one)
    kept, left, moved = eff.kv8_evict(cache, torch.zeros(0, 2, 16).to("gcu"), table, table, none, 4, 1)
    assert kept.shape == (0, 2, 4) and left.shape == (0,) and moved.shape == (0, 2, 16)


def test_strided_inputs_and_cache():
    """q, k, v as slices of one projection, k and v pages side by side in one
    pool, heads outside pages, transposed scales."""
    s = Setup([3, 50], [30, 100], 8, 2, 128, 32, seed=6)
    pool = torch.zeros(2, s.hk, s.pages, s.page, s.d, dtype=torch.uint8)
    views = [pool[i].transpose(0, 1) for i in range(2)]
    scales = [torch.zeros(s.hk, s.pages).t() for _ in range(2)]
    for view, t in zip((*views, *scales), s.cache):
        view.copy_(t)
    pool_g, scale_g = pool.to("gcu"), [t.t().contiguous().to("gcu") for t in scales]
    cache = eff.KV8Cache(pool_g[0].transpose(0, 1), pool_g[1].transpose(0, 1), *(t.t() for t in scale_g))
    qkv = torch.cat([s.q, s.k, s.v], 1).to("gcu")
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    index = s.index()
    eff.kv8_append(k, v, cache, *index)
    s.fill()
    for got, want in zip(cache, s.cache):
        assert torch.equal(got.cpu().contiguous().view(torch.uint8), want.view(torch.uint8))
    out, lse = eff.kv8_attention(q, cache, *index)
    check_attention(s, out, lse)
    odd = torch.empty(s.q.numel() + 1, dtype=s.dtype).to("gcu")[1:].view(s.q.shape)  # 2-byte aligned
    odd.copy_(q)
    assert torch.equal(eff.kv8_attention(odd, cache, *index)[0].cpu(), out.cpu())


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("scale", [0.3, 0.0, -0.2])
def test_scales(scale, wide):
    s = Setup([1, 40], [300, 100], 8, 2, 64, 16, seed=7, width=wide_table(164, 2, 16) if wide else 0).fill()
    out, lse = torch.ops.torch_gcu.kv8_attention(s.q.to("gcu"), *s.gcu(), *s.index(), scale)
    check_attention(s, out, lse, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("new,wide", [(1, False), (40, False), (40, True)])
def test_blocks_of_very_different_scales(new, wide, dtype):
    """Values of 2^-20 in most pages, of 1 in one that the softmax hardly sees, then
    of 2^9: sums stay relative to what they hold."""
    s = Setup([new], [400], 4, 2, 128, 16, dtype, seed=8, width=wide_table(80, 2, 16) if wide else 0).fill()
    for i, p in enumerate(s.table[0]):
        s.cache[3][p] *= 2.0 ** (-20 if i < 12 else -6 if i < 20 else 9 if i == 22 else -20)
        s.cache[2][p] *= 2.0 ** (i % 3)
    out, lse = eff.kv8_attention(s.q.to("gcu"), s.gcu(), *s.index())
    check_attention(s, out, lse)
    s.cache[3][:] *= 2.0 ** -9  # small alone: nothing may vanish
    out, lse = eff.kv8_attention(s.q.to("gcu"), s.gcu(), *s.index())
    check_attention(s, out, lse)


def test_far_pages_of_a_large_pool():
    """Byte offsets past 2^31 and 2^32."""
    hk, d, page, pages = 8, 128, 64, 70000  # 4.6 GB of key codes, as many of values
    s = Setup([1, 30], [100, 70], 16, hk, d, page, seed=11, spare=1)
    names = [0, 33000, 65535, 69999, 35000]
    table = [[names[i] for i in t] if max(t) < len(names) else None for t in s.table]
    assert all(table)
    big = eff.KV8Cache(*(torch.empty((pages, hk, page, d), dtype=torch.uint8, device="gcu") for _ in range(2)),
                       *(torch.empty((pages, hk), device="gcu") for _ in range(2)))
    for i, p in enumerate(names[: s.pages]):
        for t, c in zip(big, s.cache):
            t[p].copy_(c[i].to("gcu"))
    index = s.index(table=table)
    eff.kv8_append(s.k.to("gcu"), s.v.to("gcu"), big, *index)
    s.fill()
    for t, c in zip(big, s.cache):
        for i, p in enumerate(names[: s.pages]):
            assert torch.equal(t[p].cpu().view(torch.uint8), c[i].view(torch.uint8))
    out, lse = eff.kv8_attention(s.q.to("gcu"), big, *index)
    check_attention(s, out, lse)
    w = torch.rand(2, hk, s.width * page, generator=gen(3))
    used = {p for t in table for p in t}
    new = [[69998, 69990], [69997, 69980]]
    kept, _, _ = eff.kv8_evict(big, w.to("gcu"), index[0], torch.tensor(new, dtype=torch.int32).to("gcu"), index[1],
                               70, 5, 1)
    assert not used & {p for t in new for p in t}
    s2 = Setup([0, 0], s.lens, hk, hk, d, page, seed=1, spare=8)
    s2.cache, s2.table = tuple(torch.cat([c, c[:4]]) for c in s.cache), s.table
    k, _, _ = oracle.evict(s2.cache, w, s.table, [[s.pages, s.pages + 1], [s.pages + 2, s.pages + 3]], s.lens, 70, 5, 1)
    assert torch.equal(kept.cpu(), k)
    for t, c in zip(big, s2.cache):
        for j, p in enumerate(sum(new, [])):
            got, want = t[p].cpu(), c[s.pages + j]
            if got.dtype == torch.uint8:
                n = 70 - 64 if j % 2 else 64
                got, want = (torch.where(x == 0x80, 0, x.int())[:, :n] for x in (got, want))
            assert torch.equal(got, want)


def test_graphs_follow_lengths_and_share_nothing():
    """Two captured steps replayed in turn, with lengths, tables and tokens changed
    between replays and eager work beside them: each replay equals the eager call."""
    def step(new, past, seed):
        s = Setup([new] * 3, past, 8, 2, 128, 32, seed=seed, width=40, spare=60)
        for t in s.table:
            t += [s.free.pop() for _ in range(6)]
        return s, s.gcu(), s.index(), [t.to("gcu") for t in (s.q, s.k, s.v)]

    runs = []
    for new, past, seed in ((1, [900, 30, 500], 1), (20, [600, 0, 64], 2)):
        s, cache, index, qkv = step(new, past, seed)
        weights = torch.zeros(3, 2, 40 * 32).to("gcu")

        def work(cache=cache, index=index, qkv=qkv, weights=weights):
            eff.kv8_append(qkv[1], qkv[2], cache, *index)
            out, lse = eff.kv8_attention(qkv[0], cache, *index)
            eff.kv8_weigh_(weights, qkv[0], lse, cache, *index)
            return out, lse

        first = [t.clone() for t in cache]
        side = torch.gcu.Stream()
        with torch.gcu.stream(side):
            work()
        torch.gcu.synchronize()
        graph = torch.gcu.GCUGraph()
        with torch.gcu.graph(graph):
            res = work()
        for t, x in zip(cache, first):
            t.copy_(x)
        weights.zero_()
        runs.append((s, cache, index, qkv, weights, graph, res, first))
    for rnd in range(4):
        for s, cache, index, qkv, weights, graph, res, first in runs:
            n = s.new[0]
            lens = [p + 3 * rnd + n for p in (s.lens[i] - n for i in range(3))]
            index[1].copy_(torch.tensor(lens, dtype=torch.int32))
            qkv[0].copy_((s.q.float() * (1 + rnd)).to(s.dtype))
            before = [t.cpu() for t in (*cache, weights)]
            graph.replay()
            torch.gcu.synchronize()
            again = eff.KV8Cache(*(t.to("gcu") for t in before[:4]))
            w = before[4].to("gcu")
            eff.kv8_append(qkv[1], qkv[2], again, *index)
            out, lse = eff.kv8_attention(qkv[0], again, *index)
            eff.kv8_weigh_(w, qkv[0], lse, again, *index)
            for a, b in zip((*cache, weights, *res), (*again, w, out, lse)):
                a, b = a.cpu(), b.cpu()
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_side_stream():
    s = Setup([1, 200], [2000, 50], 16, 4, 128, 64, seed=12).fill()
    cache, index, q = s.gcu(), s.index(), s.q.to("gcu")
    want = eff.kv8_attention(q, cache, *index)
    torch.gcu.synchronize()
    side = torch.gcu.Stream()
    with torch.gcu.stream(side):
        got = eff.kv8_attention(q, cache, *index)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b.cpu())


def test_same_bits_every_time():
    s = Setup([1, 60], [3000, 900], 16, 4, 128, 64, seed=13).fill()
    cache, index, q = s.gcu(), s.index(), s.q.to("gcu")
    out, lse = eff.kv8_attention(q, cache, *index)
    w = eff.kv8_weigh_(torch.zeros(2, 4, s.width * 64).to("gcu"), q, lse, cache, *index)
    for _ in range(3):
        o, e = eff.kv8_attention(q, cache, *index)
        x = eff.kv8_weigh_(torch.zeros(2, 4, s.width * 64).to("gcu"), q, e, cache, *index)
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in ((o, out), (e, lse), (x, w)))


def test_without_workspace_sequences_stay_whole(tmp_path):
    """In a process of its own, where no workspace allocator is registered."""
    s = Setup([1, 40], [3000, 2000], 8, 2, 128, 32, seed=17).fill()
    args, got = tmp_path / "args.pt", tmp_path / "got.pt"
    torch.save([s.q, *s.cache, *(t.cpu() for t in s.index())], args)
    code = ("import sys, torch\n"
            "from torch_gcu import _abi\n"
            "q, *rest = [t.cuda() for t in torch.load(sys.argv[1], weights_only=True)]\n"
            "out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device='cuda')\n"
            "_abi.lib().mi_set_workspace_allocator(_abi._ALLOC_FN(), _abi._FREE_FN(), None)\n"
            "_abi.kv8_attention(out, lse, q, rest[:4], *rest[4:])\n"
            "torch.save([out.cpu(), lse.cpu()], sys.argv[2])\n")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path))
    r = subprocess.run([sys.executable, "-c", code, str(args), str(got)], env=env, capture_output=True,
                       text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]
    check_attention(s, *torch.load(got, weights_only=True))


def test_bad_pages_and_lengths_raise_and_touch_nothing():
    """A page outside the pool is not seen (nor written); a length outside the table
    makes the sequence empty; both raise IndexError at the next synchronisation."""
    s = Setup([1, 1, 30], [100, 70, 60], 4, 2, 64, 32, seed=14)
    before = [t.clone() for t in s.cache]
    cache, index = s.gcu(), s.index()
    bad = [list(t) for t in s.table]
    bad[0][3], bad[2][0] = s.pages, -5  # where sequence 0's new token goes; seen by sequence 2
    index[0] = s.index(table=bad)[0]
    eff.kv8_append(s.k.to("gcu"), s.v.to("gcu"), cache, *index)
    with pytest.raises(IndexError, match=f"index {s.pages} is out of bounds"):
        torch.gcu.synchronize()
    s.fill()
    page = s.table[0][3]
    for got, want, old in zip(cache, s.cache, before):
        want = want.clone()
        want[page] = old[page]
        assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))
    out, lse = eff.kv8_attention(s.q.to("gcu"), cache, *index)
    with pytest.raises(IndexError):
        torch.gcu.synchronize()
    assert out.cpu().isfinite().all()
    check_attention(s, out, lse, rows=slice(1, 2))
    w = torch.zeros(3, 2, s.width * 32).to("gcu")
    eff.kv8_weigh_(w, s.q.to("gcu"), lse, cache, *index)
    with pytest.raises(IndexError):
        torch.gcu.synchronize()
    assert (w[0, :, 96:] == 0).all().item() and (w[2, :, :32] == 0).all().item()

    for wrong in (-1, s.width * 32 + 1, 2 ** 31 - 1):
        index = s.index(lens=[s.lens[0], wrong, s.lens[2]])
        held = [t.cpu() for t in cache]
        eff.kv8_append(s.k.to("gcu")[1:2].expand(31, 2, 64).contiguous(), s.v.to("gcu")[:31], cache, index[0][1:2],
                       index[1][1:2], torch.tensor([0, 1], dtype=torch.int32).to("gcu"))
        with pytest.raises(IndexError, match=f"index {wrong} is out of bounds"):
            torch.gcu.synchronize()
        assert all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, held))
        out, lse = eff.kv8_attention(s.q.to("gcu"), cache, *index)
        with pytest.raises(IndexError):
            torch.gcu.synchronize()
        assert (out[1] == 0).all().item() and (lse[1] == -math.inf).all().item()
        kept, left, _ = eff.kv8_evict(cache, w, index[0], torch.tensor([[s.free[0]], [s.free[1]], [s.free[2]]], dtype=torch.int32).to("gcu"),
                                      index[1], 8, 2)
        with pytest.raises(IndexError):
            torch.gcu.synchronize()
        assert left.cpu().tolist() == [8, 0, 8] and (kept[1] == -1).all().item()


def test_starts_that_run_backwards_stay_in_bounds():
    s = Setup([4, 4], [50, 60], 4, 2, 64, 32, seed=15).fill()
    cache, index = s.gcu(), s.index()
    for starts in ([5, 2, 8], [0, 100, 8], [-3, 4, 2 ** 31 - 1], [8, 8, 0], [0, 8, -2 ** 31]):
        index[2] = torch.tensor(starts, dtype=torch.int32).to("gcu")
        out, lse = eff.kv8_attention(s.q.to("gcu"), cache, *index)
        torch.gcu.synchronize()
        assert out.shape == s.q.shape
        eff.kv8_weigh_(torch.zeros(2, 2, s.width * 32).to("gcu"), s.q.to("gcu"), lse, cache, *index)
        torch.gcu.synchronize()


def test_refusals_on_the_device():
    s = Setup([1], [10], 4, 2, 64, 16, seed=16)
    cache, index = s.gcu(), s.index()
    with pytest.raises(RuntimeError, match="must be a gcu tensor"):
        eff.kv8_attention(s.q.to("gcu"), cache, index[0].cpu(), *index[1:])
    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        eff.kv8_attention(s.q.float().to("gcu"), cache, *index)
    with pytest.raises(RuntimeError, match="heads"):
        eff.kv8_attention(s.q[:, :3].to("gcu"), cache, *index)
    with pytest.raises(RuntimeError, match="int32"):
        eff.kv8_append(s.k.to("gcu"), s.v.to("gcu"), cache, index[0], index[1].long(), index[2])
    with pytest.raises(RuntimeError, match="positions"):
        eff.kv8_weigh_(torch.zeros(1, 2, 8).to("gcu"), s.q.to("gcu"), torch.zeros(1, 4).to("gcu"), cache, *index)


def test_decoder_layer_over_the_cache():
    """Prompts in two pieces, then captured decode steps: the layer is what its ops
    give one by one, its attention what the definition says, and a replay with new
    lengths is the eager call, bit for bit."""
    cfg = dl.LayerConfig(vocab=100, hidden=256, heads=4, head_dim=64, ffn=512)
    w = {n: t.to("gcu") for n, t in dl.init_weights(cfg, 3).items()}
    for n in ("wk", "wv"):  # two k/v heads
        w[n] = w[n][:128].contiguous()
    g = gen(1)
    tables = [[5, 2, 9, 1], [0, 7, 3, 4]]
    table = torch.tensor(tables, dtype=torch.int32).to("gcu")
    cache, mine = eff.kv8_cache(10, 2, 64, 32), eff.kv8_cache(10, 2, 64, 32)
    lens = [0, 0]

    def call(new):
        for b in range(2):
            lens[b] += new[b]
        ids = torch.randint(0, 100, (sum(new),), generator=g)
        pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)])
        i32 = [torch.tensor(x, dtype=torch.int32) for x in (lens, [0, new[0], sum(new)])]
        return [t.to("gcu") for t in (ids, *i32, pos)]

    def by_hand(ids, lengths, starts, pos):
        e, T = eff, ids.shape[0]
        x = torch.nn.functional.embedding(ids, w["embed"])
        h = e.rms_norm(x, w["attn_norm"], cfg.eps)
        q, k, v = (torch.nn.functional.linear(h, w[n]).view(T, -1, 64) for n in ("wq", "wk", "wv"))
        q, k = e.rope(q, k, pos, cfg.theta)
        e.kv8_append(k, v, mine, table, lengths, starts)
        a, lse = e.kv8_attention(q, mine, table, lengths, starts)
        s = Setup.__new__(Setup)
        s.q, s.cache, s.table, s.lens = q.cpu(), [t.cpu() for t in mine], tables, list(lens)
        s.starts, s.d, s.dtype = starts.cpu().tolist(), 64, q.dtype
        check_attention(s, a, lse)
        x = x + torch.nn.functional.linear(a.view(T, -1), w["wo"])
        h = e.rms_norm(x, w["ffn_norm"], cfg.eps)
        m = e.silu_mul(torch.nn.functional.linear(h, w["w_gate"]), torch.nn.functional.linear(h, w["w_up"]))
        return x + torch.nn.functional.linear(m, w["w_down"])

    for new in ([40, 3], [20, 30], [1, 1]):
        ids, lengths, starts, pos = call(new)
        out, _, _ = dl.forward_cached(w, ids, cfg, cache, table, lengths, starts, pos)
        assert torch.equal(out.cpu(), by_hand(ids, lengths, starts, pos).cpu())
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(cache, mine))
    # a captured decode step: its inputs are updated in place between replays (the
    # last eager step is done again by the capture, which runs nothing)
    static = [ids, lengths, starts, pos]
    graph = torch.gcu.GCUGraph()
    with torch.gcu.graph(graph):
        out, _, _ = dl.forward_cached(w, ids, cfg, cache, table, lengths, starts, pos)
    for _ in range(4):
        new = call([1, 1])
        for t, x in zip(static, new):
            t.copy_(x)
        graph.replay()
        torch.gcu.synchronize()
        assert torch.equal(out.cpu(), by_hand(*new).cpu())
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(cache, mine))
