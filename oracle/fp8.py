"""Linear layers in 8-bit floating point in 64 bits, from their definition (torch
on the CPU)."""
from __future__ import annotations

import torch

from .kv8 import codes, e4m3

GROUP = 128
NAN = 0x7F


def value(byte: torch.Tensor) -> torch.Tensor:
    """Scale bytes as the powers of two that they are; 255 is NaN."""
    s = torch.exp2(byte.double() - 127)
    return torch.where(byte == 255, torch.nan, s)


def scale_byte(amax: torch.Tensor) -> torch.Tensor:
    """The byte of the smallest power of two s >= 2^-110 with amax <= 448 s."""
    e = torch.full(amax.shape, -110, dtype=torch.int64)
    for k in range(-110, 128):
        e = torch.where(amax > 448 * 2.0 ** k, k + 1, e)
    return (e + 127).to(torch.uint8)


def blocks(x: torch.Tensor, rows: int) -> torch.Tensor:
    """x [m, k] as [m blocks, rows, k blocks, 128] with zeros behind its end."""
    m, k = x.shape
    whole = torch.zeros(-(-m // rows) * rows, -(-k // GROUP) * GROUP, dtype=torch.float64)
    whole[:m, :k] = x
    return whole.view(-1, rows, whole.shape[1] // GROUP, GROUP)


def spread(byte: torch.Tensor, rows: int, shape) -> torch.Tensor:
    """The scale of each element of a matrix of this shape."""
    s = value(byte).repeat_interleave(rows, 0).repeat_interleave(GROUP, 1)
    return s[: shape[0], : shape[1]]


def quantize(x: torch.Tensor, rows: int = 1, byte=None):
    """(codes as bytes, scale bytes) of x [m, k]; rows 128 for a weight."""
    x = x.double()
    fine = torch.isfinite(x)
    if byte is None:
        byte = scale_byte(blocks(torch.where(fine, x.abs(), 0.0), rows).amax((1, 3)))
    y = torch.where(fine, x, 0.0) / spread(byte, rows, x.shape)
    return torch.where(fine, codes(e4m3(y)), NAN).to(torch.uint8), byte


def numbers(code: torch.Tensor, byte: torch.Tensor, rows: int = 1) -> torch.Tensor:
    """What codes and scales stand for."""
    return code.view(torch.float8_e4m3fn).double() * spread(byte, rows, code.shape)


def product(x, w):
    """(x w^T, mass, power) of quantised x and w: mass the sums of |products|, power
    those of their squares, by which a bound on the sum's rounding goes."""
    a, b = numbers(*x), numbers(*w, rows=GROUP)
    return a @ b.t(), a.abs() @ b.abs().t(), a.square() @ b.square().t()


def rms_norm(x, weight, eps, residual=None):
    """(norm, total): the total in the inputs' type."""
    total = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    t = total.double()
    y = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight.double()), total


def silu_mul(gate, up):
    return gate * torch.sigmoid(gate) * up
