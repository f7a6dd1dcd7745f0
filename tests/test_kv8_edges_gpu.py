"""Edges of the 8-bit key/value cache on the GPU: queries that are not finite beside
rows that pad a tile, pages of very different scales, tokens that are zero, and
tolerances that go by each row's own values."""
import math

import pytest
import torch

import torch_gcu  # noqa: F401
from oracle import kv8 as oracle
from test_kv8_gpu import F, SHAPES, Setup, wide_table
from torch_gcu.utils import decoder_layer as dl

pytestmark = pytest.mark.gpu
eff = torch.gcu.efficient if hasattr(torch, "gcu") else None
DTYPES = [torch.bfloat16, torch.float16]
IDS = ["bf16", "f16"]


def i32(x):
    return torch.tensor(x, dtype=torch.int32).to("gcu")


# ---- accumulated weights ------------------------------------------------------


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("blocks", [1, 200, 400])  # of 128 keys: four, two waves to 32 keys, one
@pytest.mark.parametrize("group", [1, 3, 4])
def test_a_bad_query_weighs_on_the_keys_that_it_sees(group, blocks, bad):
    """The first query of a tile that rows do not fill: a key behind the query's own
    position gets the weight that it gets with any other query there."""
    hk, n, past, page = 2, 100, 60, 16
    s = Setup([n], [past], hk * group, hk, 64, page, seed=group, width=max(1, blocks // hk * 128 // page)).fill()
    cache, index = s.gcu(), s.index()
    for rt in (64, 128):  # rows of a tile: whole tokens of the group's heads
        token = (n - 1) // (rt // group) * (rt // group)
        got = []
        for value in (1.0, bad):
            s.q[token, 0, 5] = value
            q = s.q.to("gcu")
            _, lse = eff.kv8_attention(q, cache, *index)
            w = torch.zeros(1, hk, s.width * page).to("gcu")
            got.append(eff.kv8_weigh_(w, q, lse, cache, *index).cpu())
        s.q[token, 0, 5] = 1.0
        at = past + token + 1
        assert got[0].isfinite().all()
        assert torch.equal(got[1][0, 0, at:], got[0][0, 0, at:])
        assert torch.equal(got[1][0, 1], got[0][0, 1])  # the other k/v head


# ---- eviction -----------------------------------------------------------------


def same_pages(cache, want, pages):
    for got, want in zip(cache, want):
        got, want = got.cpu()[pages], want[pages]
        if got.dtype == torch.uint8:  # 0 and -0 are one number
            got, want = (torch.where(x == 0x80, 0, x.int()) for x in (got, want))
        assert torch.equal(got, want)


@pytest.mark.parametrize("small", [0.0, 1e-30])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 256)])
def test_zero_tokens_of_a_page_with_a_large_scale(d, page, small):
    """Tokens of zeros, kept from a page whose other tokens are large, alone or with
    tokens of another page that are very small."""
    n, hk, keep = page + 8, 2, 10
    s = Setup([0], [n], hk, hk, d, page, seed=1, spare=3)
    x = torch.zeros(2, n, hk, d, dtype=torch.bfloat16)
    x[:, 8:page] = 1e9  # the first 8 tokens of page 0 are zero
    x[:, page:] = small
    s.cache = tuple(torch.zeros_like(t) for t in s.cache)
    oracle.append(s.cache, x[0], x[1], s.table, [n], [0, n])
    w = torch.zeros(1, hk, s.width * page)
    w[..., :7], w[..., page: page + 3] = 2.0, 1.0
    fresh = [[s.free[0]]]
    cache, index = s.gcu(), s.index()
    kept, left, _ = eff.kv8_evict(cache, w.to("gcu"), index[0], i32(fresh), index[1], keep, 0, 0)
    k, m, _ = oracle.evict(s.cache, w, s.table, fresh, [n], keep, 0, 0)
    assert torch.equal(kept.cpu(), k) and left.cpu().tolist() == m
    same_pages(cache, s.cache, list(range(s.pages)))


def test_kept_tokens_of_a_page_that_is_not_there_are_zeros():
    """Whatever the scale of the page that is read in its stead."""
    d, page, hk = 64, 16, 2
    s = Setup([0], [40], hk, hk, d, page, seed=2, spare=6)
    if 0 in s.table[0]:
        s.table[0][s.table[0].index(0)] = s.free.pop()
    s.cache = tuple(torch.zeros_like(t) for t in s.cache)
    x = torch.randn(2, 40, hk, d, generator=torch.Generator().manual_seed(3)).bfloat16()
    oracle.append(s.cache, x[0], x[1], s.table, [40], [0, 40])
    for t in s.cache[2:]:
        t[0] = math.nan
    bad = [list(s.table[0])]
    bad[0][1] = s.pages
    w = torch.zeros(1, hk, s.width * page)
    w[..., 10:30] = 1.0  # six of page 0, and 14 of the page that is not there
    fresh = [[p for p in s.free if p][:2]]
    cache = s.gcu()
    eff.kv8_evict(cache, w.to("gcu"), s.index(table=bad)[0], i32(fresh), i32([40]), 20, 0, 0)
    with pytest.raises(IndexError, match=f"index {s.pages} is out of bounds"):
        torch.gcu.synchronize()
    gone = s.table[0][1]
    for t in s.cache[:2]:
        t[gone] = 0
    for t in s.cache[2:]:
        t[gone] = 1.0
    oracle.evict(s.cache, w, s.table, fresh, [40], 20, 0, 0)
    same_pages(cache, s.cache, fresh[0])


# ---- attention ----------------------------------------------------------------


def bounds(s, scale):
    """(want, tolerance) of the output: each row by its own keys.  With u = eps / 2 of
    the type: a score is an fp32 sum of exact products, off by at most e_j = (D + 8) F
    times its sum of |q k| scale, and 2^-21 for the exp2 unit and log2(e); so a weight
    p_j by p_j (e_j + sum_i p_i e_i).  A weight is rounded to the type: by u, or in f16
    under its normal range by 2^-25 of the row's largest weight (and never by more than
    itself).  The sum over n keys
    is off by n F of the sum of magnitudes, the output rounded by u (2^-25 in f16)."""
    f16, u = s.dtype == torch.float16, torch.finfo(s.dtype).eps / 2
    hk = s.cache[0].shape[1]
    T, H, D = s.q.shape
    want, tol = (torch.zeros(T, H, D, dtype=torch.float64) for _ in range(2))
    for b, total in enumerate(s.lens):
        span = slice(s.starts[b], s.starts[b + 1])
        n = span.stop - span.start
        if n == 0 or total == 0:
            continue
        see = torch.arange(total)[None] <= torch.arange(total - n, total)[:, None]
        for h in range(H):
            g = h // (H // hk)
            k, v = (oracle.tokens(s.cache[i][:, g], s.cache[i + 2][:, g], s.table[b], total) for i in (0, 1))
            q = s.q[span, h].double()
            x = torch.where(see, (q @ k.t()) * scale, -math.inf)
            p = torch.softmax(x, 1).nan_to_num(nan=0.0)  # a row that sees nothing: 0
            e = (D + 8) * F * (q.abs() @ k.abs().t()) * abs(scale) + 2.0 ** -21
            off = p * (e + (p * e).sum(1, keepdim=True) + u + see.sum(1, keepdim=True) * F)
            if f16:
                off = off + torch.minimum(2.0 ** -25 * p.amax(1, keepdim=True), p)
            want[span, h] = p @ v
            tol[span, h] = off @ v.abs() + u * want[span, h].abs()
    tol += 2.0 ** -25 if f16 else 1e-37
    return want, tol


def check(s, out):
    want, tol = bounds(s, s.d ** -0.5)
    off = (out.cpu().double() - want).abs() / tol
    assert not off.isnan().any(), "NaN"
    assert off.max() <= 1, f"{off.max()} of the tolerance, in row {int(off.amax((1, 2)).argmax())}"


def attend(s):
    out, _ = eff.kv8_attention(s.q.to("gcu"), s.gcu(), *s.index())
    return out


def larger(s, page, ratio):
    for _ in range(2):  # 2^130 is no float32
        s.cache[3][page] *= 2.0 ** (ratio // 2)


def width_for(s_new, group, hk, page, wide):
    return wide_table(sum(s_new) * group, hk, page) if wide else 0


BY_ROW = [(False, *SHAPES[i]) for i in (1, 3, 6, 8, 10, 12, 13, 17)]  # by the kernel of few rows
BY_ROW += [(True, *SHAPES[i]) for i in (10, 12, 13, 17)]  # by that of prompts


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("wide,new,past,h,hk,d,page", BY_ROW)
def test_each_row_by_its_own_values(wide, new, past, h, hk, d, page, dtype):
    s = Setup(new, past, h, hk, d, page, dtype, seed=5, width=width_for(new, h // hk, hk, page, wide)).fill()
    check(s, attend(s))
    for i in range(s.pages):
        s.cache[3][i] *= 2.0 ** (i % 5)
    check(s, attend(s))


@pytest.mark.parametrize("dtype,ratio", [(torch.float16, 4), (torch.float16, 14), (torch.float16, 20),
                                         (torch.float16, 30), (torch.bfloat16, 20), (torch.bfloat16, 130)])
@pytest.mark.parametrize("new,wide", [(1, False), (8, False), (90, False), (90, True)])
@pytest.mark.parametrize("d", [64, 128])
def test_a_large_page_of_no_weight(d, new, wide, dtype, ratio):
    """A page whose values are larger by 2^ratio, and whose scores are so low that the
    softmax gives it nothing: the others' weights keep their bits."""
    s = Setup([new], [600], 4, 2, d, 16, dtype, seed=d + new, width=width_for([new], 2, 2, 16, wide))
    s.q[..., 0] = 1024.0
    s.fill()
    low = [s.table[0][10], s.table[0][27]]
    for p in s.table[0]:  # channel 0 of the keys decides alone
        s.cache[0][p, ..., 0] = 0xFE if p in low else 0  # -448
    s.cache[3][:] *= 2.0 ** (-60 if dtype == torch.bfloat16 else 0)
    for p in low:
        larger(s, p, ratio)
    check(s, attend(s))


@pytest.mark.parametrize("dtype,ratio", [(torch.float16, 10), (torch.float16, 20), (torch.float16, 28),
                                         (torch.bfloat16, 20), (torch.bfloat16, 130)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_in_front_of_a_large_page(d, wide, dtype, ratio):
    """Queries that end before a page of large values, in the same tile of keys."""
    s = Setup([100], [100], 4, 2, d, 16, dtype, seed=d, width=width_for([100], 2, 2, 16, wide)).fill()
    large = 12 if dtype == torch.float16 else 70  # times 2^large, the others 2^ratio less
    s.cache[3][:] *= 2.0 ** (large - ratio)
    larger(s, s.table[0][9], ratio)
    check(s, attend(s))


# ---- the decoder layer ----------------------------------------------------------


def test_decoder_layer_without_new_tokens():
    cfg = dl.LayerConfig(vocab=100, hidden=256, heads=4, head_dim=64, ffn=512)
    w = {n: t.to("gcu") for n, t in dl.init_weights(cfg, 3).items()}
    for n in ("wk", "wv"):
        w[n] = w[n][:128].contiguous()
    cache = eff.kv8_cache(4, 2, 64, 32)
    ids = torch.zeros(0, dtype=torch.int64).to("gcu")
    out, q, lse = dl.forward_cached(w, ids, cfg, cache, i32([[0, 1]]), i32([5]), i32([0, 0]), ids)
    assert out.shape == (0, 256) and q.shape == (0, 4, 64) and lse.shape == (0, 4)
    assert all((t.cpu() == 0).all() for t in cache)
