"""Fused efficient ops of the gcu device.

``gcu_index`` keeps the reference's one efficient op
(torch_gcu/gcu/efficient/op.py:8-16 -> torch_gcu/csrc/efficient_ops/ops.cpp:335-342);
``rms_norm``, ``rope``, ``rope_`` and ``silu_mul`` are new fused kernels, and
``linear_residual`` / ``linear_silu_mul`` are matmuls with the residual add or
the SwiGLU product fused into their epilogue.  The ``kv8_*`` ops serve from a
key/value cache held in 8 bits.
All are dispatcher ops (``torch.ops.torch_gcu.*``) with gcu kernels only.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from ... import _C  # noqa: F401  (registers torch.ops.torch_gcu)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-6) -> torch.Tensor:
    """x * rsqrt(mean(x^2, -1) + eps) * weight, fp32 math, one rounding."""
    return torch.ops.torch_gcu.rms_norm(x, weight, eps)


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
         theta: float = 10000.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotate-half RoPE of [tokens, heads, head_dim] q and k."""
    return torch.ops.torch_gcu.rope(q, k, positions, theta)


def rope_(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
          theta: float = 10000.0) -> None:
    """In-place RoPE of q (and k)."""
    torch.ops.torch_gcu.rope_(q, k, positions, theta)


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up with one rounding."""
    return torch.ops.torch_gcu.silu_mul(gate, up)


def linear_residual(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
    """residual + F.linear(x, weight), bit for bit as the two ops (the product
    rounded to the input dtype first)."""
    return torch.ops.torch_gcu.linear_residual(x, weight, residual)


def linear_silu_mul(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor) -> torch.Tensor:
    """silu_mul(F.linear(x, w_gate), F.linear(x, w_up)), bit for bit as the
    three ops (both products rounded to the input dtype first)."""
    return torch.ops.torch_gcu.linear_silu_mul(x, w_gate, w_up)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(x @ weight^T) * scales (+ bias): int8 [N, K] weight, fp32 [N] scales,
    widened exactly to bf16/fp16 and multiplied on MFMA with fp32 accumulation."""
    return torch.ops.torch_gcu.int8_linear(x, weight, scales, bias)


def gcu_index(self: torch.Tensor, indices: Sequence[Optional[torch.Tensor]]) -> torch.Tensor:
    """self[indices] with int32 index tensors (no int64 upcast on device)."""
    return torch.ops.torch_gcu.int32_indices_index(self, list(indices))


class KV8Cache(NamedTuple):
    """A pool of pages of e4m3 codes, with a scale per page and k/v head:
    ``value = code * scale``.  ``k`` and ``v`` are uint8 ``[pages, heads, page,
    head_dim]`` (``.view(torch.float8_e4m3fn)`` on another device reads the
    codes), ``k_scale`` and ``v_scale`` float32 ``[pages, heads]``."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def kv8_cache(pages: int, heads: int, head_dim: int, page: int = 64, device="gcu") -> KV8Cache:
    """An empty pool: head_dim 64 or 128, page a power of two from 16 to 256
    tokens.  Pages belong to no one: the caller hands them to sequences by
    block tables."""
    codes = [torch.zeros((pages, heads, page, head_dim), dtype=torch.uint8, device=device)
             for _ in range(2)]
    scales = [torch.zeros((pages, heads), dtype=torch.float32, device=device) for _ in range(2)]
    return KV8Cache(*codes, *scales)


def kv8_append(k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor,
               lengths: torch.Tensor, starts: torch.Tensor) -> None:
    """Write new tokens' keys and values (bf16 or f16 [tokens, heads, head_dim])
    into the cache.

    block_table int32 [sequences, pages of one], lengths int32 [sequences] (the
    tokens that the cache holds, the new ones among them) and starts int32
    [sequences + 1]: tokens starts[b] .. starts[b + 1] - 1 are sequence b's
    last ones.  All three stay on the device, so a captured call follows them.
    A length or page out of range raises IndexError at the next
    synchronisation, and the sequence or page is left alone."""
    torch.ops.torch_gcu.kv8_append(*cache, k, v, block_table, lengths, starts)


def kv8_attention(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor,
                  lengths: torch.Tensor, starts: torch.Tensor,
                  scale: Optional[float] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of new tokens' queries [tokens, heads, head_dim] over the cache,
    each up to its own position (append first): (out, logsumexp float32 [tokens,
    heads]), without gradients.  scale defaults to head_dim ** -0.5.  Tokens of no sequence, and
    tokens that see nothing, get 0 and -inf."""
    return torch.ops.torch_gcu.kv8_attention(q, *cache, block_table, lengths, starts, scale)


def kv8_weigh_(weights: torch.Tensor, q: torch.Tensor, lse: torch.Tensor, cache: KV8Cache,
               block_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
               scale: Optional[float] = None) -> torch.Tensor:
    """Add the softmax weights of these queries (lse from kv8_attention), summed
    over queries and the heads of a group, to weights float32 [sequences, k/v
    heads, positions of the block table or more], in place."""
    torch.ops.torch_gcu.kv8_weigh_(weights, q, lse, *cache, block_table, lengths, starts, scale)
    return weights


def kv8_evict(cache: KV8Cache, weights: torch.Tensor, block_table: torch.Tensor,
              new_table: torch.Tensor, lengths: torch.Tensor, keep: int, recent: int,
              sink: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence to `keep` tokens per k/v head: the first `sink`, the
    last `recent` and the others of largest weight (ties: the lower position),
    moved in their order to the pages of new_table (int32 [sequences, ceil(keep /
    page) or more]), none named twice and none in block_table.  Returns the kept
    positions int32 [sequences, heads, keep] (then -1), the new lengths and the
    kept tokens' weights (shape of weights, then 0).  The old pages are the
    caller's again; queries keep using their true positions for RoPE."""
    return torch.ops.torch_gcu.kv8_evict(*cache, weights, block_table, new_table, lengths, keep,
                                         recent, sink)
