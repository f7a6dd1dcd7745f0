"""Edges of the 8-bit key/value cache on the GPU."""
import math

import pytest
import torch

import torch_gcu  # noqa: F401
from test_kv8_gpu import Setup

pytestmark = pytest.mark.gpu
eff = torch.gcu.efficient if hasattr(torch, "gcu") else None


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
