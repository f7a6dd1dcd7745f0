"""8-bit linear layers without a GPU: descriptors that are no tensors."""
import ctypes

import pytest
import torch

from torch_gcu import _abi

INVALID, UNSUPPORTED = 1, 2
U8, BF16 = torch.uint8, torch.bfloat16


@pytest.mark.parametrize("name", ["total", "residual"])
@pytest.mark.parametrize("field,value,status,words",
                         [("ndim", 12, INVALID, "ndim"), ("ndim", -1, INVALID, "ndim"),
                          ("dtype", 99, UNSUPPORTED, "dtype"), ("ndim", 1, INVALID, "rows, columns")])
def test_norm_looks_at_no_more_than_a_descriptor_holds(name, field, value, status, words):
    """A sum or residual of more dims than a descriptor has room for is refused for that,
    before its sizes are read.  (Behind the descriptor lie numbers that, taken for its
    strides, make it reach over every other tensor of the call.)"""
    pool = torch.zeros(8192, dtype=U8)
    at = lambda byte, *s: pool[byte: byte + 2 * 5 * 64].view(BF16).view(s)  # noqa: E731
    tensors = {"total": at(0, 5, 64), "residual": at(1024, 5, 64)}
    x = at(2048, 5, 64)
    out = _abi.MiFp8(_abi.desc(pool[4096: 4096 + 320].view(5, 64)), _abi.desc(pool[5120: 5125].view(5, 1)))
    held = (_abi.MiTensor * 3)()
    ctypes.memset(held, 0x01, ctypes.sizeof(held))
    held[0] = _abi.desc(tensors[name])
    for d in range(2, 8):
        held[0].sizes[d], held[0].strides[d] = 1 << 20, 1 << 20
    setattr(held[0], field, value)
    args = {n: _abi.desc(t) for n, t in tensors.items()}
    args[name] = held[0]
    st = _abi.lib().mi_rms_norm_fp8(out, ctypes.byref(args["total"]), _abi.desc(x),
                                    ctypes.byref(args["residual"]), None, 1e-6, None)
    text = _abi.lib().mi_last_error().decode()
    assert st == status and words in text and name in text, (st, text)
