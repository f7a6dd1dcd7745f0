"""Edges of the 8-bit key/value cache on the GPU."""
import math

import pytest
import torch

import torch_gcu  # noqa: F401
from oracle import kv8 as oracle
from test_kv8_gpu import Setup
from torch_gcu.utils import decoder_layer as dl

pytestmark = pytest.mark.gpu
eff = torch.gcu.efficient if hasattr(torch, "gcu") else None


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
