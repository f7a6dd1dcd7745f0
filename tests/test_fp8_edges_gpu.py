"""Edges of the 8-bit linear layers on the GPU."""
import pytest
import torch

import torch_gcu  # noqa: F401
from test_fp8_linear_gpu import eff, layer
from torch_gcu.utils import decoder_layer as dl

pytestmark = pytest.mark.gpu


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
