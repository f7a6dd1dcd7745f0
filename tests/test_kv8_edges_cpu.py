"""Edges of the 8-bit key/value cache that show without a GPU: the places that
its kernels load keys from, and memory that two tensors of a call share."""
import os
import subprocess

import pytest
import torch

from test_kv8_cpu import call, run
from torch_gcu import _abi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KERNELS = os.path.join(REPO, "torch-gcu_amd", "csrc", "kernels")

PLACES = r"""
#include <cassert>
#include <cstdio>
#include <initializer_list>
#include "kv8_index.h"
using namespace mi;

int main() {
  long n = 0;
  auto check = [&](int len) {
    for (int shift = 4; shift <= 8; ++shift)
      for (int tile : {32, 64, 128}) {  // keys of a block, 32 a wave
        const int last = (int)(((long)len - 1) / tile);
        for (int j : {0, last > 0 ? last - 1 : 0, last})
          for (int wave = 0; wave < tile / 32; ++wave)
            for (int t = 0; t < 2; ++t) {
              const int pos = j * tile + 32 * wave + 16 * t;
              const int at = kv8_group_at(pos, len), slot = at & ((1 << shift) - 1);
              assert(at >= 0 && at % 16 == 0 && at < len);
              assert(slot + 15 < 1 << shift);                    // 16 rows of one page's head
              assert(at >> shift <= (len - 1) >> shift);         // of a page that the sequence has
              if (pos < len) assert(at == pos);
              ++n;
            }
      }
  };
  for (int len = 1; len <= 5000; ++len) check(len);
  for (int len : {65535, 65536, 65537, (1 << 30) - 17, (1 << 30) - 1, 1 << 30}) check(len);
  printf("%ld places\n", n);
}
"""


def test_keys_are_loaded_from_inside_a_page(tmp_path):
    """Waves whose keys lie behind the end of a sequence too."""
    src, exe = tmp_path / "places.cpp", tmp_path / "places"
    src.write_text(PLACES)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", KERNELS, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_rope_of_no_tokens_is_no_error():
    """Nor is it taken for one where there are positions to rotate by."""
    q, k = torch.zeros(0, 4, 64, dtype=torch.bfloat16), torch.zeros(0, 2, 64, dtype=torch.bfloat16)
    for positions, status in ((torch.zeros(0, dtype=torch.int64), 0), (torch.zeros(3, dtype=torch.int64), 1)):
        a = [_abi.desc(t) for t in (q, k, q, k, positions)]
        assert _abi.lib().mi_rope(*a, 1e4, None) == status, _abi.lib().mi_last_error()


U8, I32 = torch.uint8, torch.int32


def pages_of(shape, offset, strides=None):
    """k and v codes in one buffer, v `offset` bytes behind k."""
    strides = strides or (2048, 1024, 64, 1)
    extent = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
    buf = torch.zeros(extent + offset + 64, dtype=U8)
    buf = buf[-buf.data_ptr() % 16:]
    return [buf[o:].as_strided(shape, strides) for o in (0, offset)]


CACHE = (3, 2, 16, 64)  # a page's head 1024 bytes
SHARED = [
    # offset of v, strides: pages or heads of one on those of the other
    (0, None), (16, None), (1008, None), (1024, None), (2048, None), (3 * 2048 - 16, None),
    (1008, (4096, 2048, 64, 1)), (2048, (4096, 2048, 64, 1)), (4096 + 2048, (4096, 2048, 64, 1)),
    (1040, (6144, 2048, 64, 1)), (1024, (1024, 4096, 64, 1)),
]
APART = [
    (3 * 2048, None), (1024, (4096, 2048, 64, 1)),          # behind, by turns head by head
    (2048, (4096, 1024, 64, 1)),                            # page by page
    (5120, (4096, 2048, 64, 1)),                            # a page later, the odd heads
    (4096, (1024, 8192, 64, 1)),                            # heads outside pages
]


def set_codes(a, pair):
    a["k_cache"], a["v_cache"] = pair


@pytest.mark.parametrize("op", ["append", "evict"])
@pytest.mark.parametrize("offset,strides", SHARED)
def test_keys_and_values_in_the_same_memory(op, offset, strides):
    a = call()
    set_codes(a, pages_of(CACHE, offset, strides))
    st, message = run(op, a)
    assert st == 1 and "same memory" in message, (st, message)


@pytest.mark.parametrize("offset,strides", APART)
def test_keys_and_values_by_turns(offset, strides):
    a = call(tokens=0)  # nothing to do: done behind the checks
    set_codes(a, pages_of(CACHE, offset, strides))
    assert run("append", a)[0] == 0, run("append", a)
    a = call(seqs=0)
    set_codes(a, pages_of(CACHE, offset, strides))
    assert run("evict", a)[0] == 0, run("evict", a)


def test_keys_and_values_of_other_strides_among_each_other():
    a = call()
    buf = torch.zeros(9 * 4096, dtype=U8)
    a["k_cache"], a["v_cache"] = buf.as_strided(CACHE, (4096, 2048, 64, 1)), buf[1024:].as_strided(CACHE, (8192, 2048, 64, 1))
    st, message = run("append", a)
    assert st == 1 and "same memory" in message


@pytest.mark.parametrize("op", ["append", "evict"])
def test_scales_in_the_same_memory(op):
    one = torch.zeros(16)
    for offset, strides, fine in ((1, (2, 1), False), (4, (2, 1), False), (6, (2, 1), True), (2, (4, 1), True),
                                  (3, (4, 1), False), (1, (4, 2), True), (5, (4, 2), True)):
        a = call(tokens=0) if op == "append" else call(seqs=0)
        a["k_scale"], a["v_scale"] = (one[o:].as_strided((3, 2), strides) for o in (0, offset))
        st, message = run(op, a)
        assert (st == 0) == fine and (fine or "same memory" in message), (offset, strides, st, message)


@pytest.mark.parametrize("offset", [1, 31, 32, 64, 127])
def test_new_weights_on_the_old_ones(offset):
    a = call()
    one = torch.zeros(512)
    a["weights"], a["new_weights"] = (one[o:].as_strided((2, 2, 32), (64, 32, 1)) for o in (0, offset))
    st, message = run("evict", a)
    assert st == 1 and "of their own" in message


def test_new_lengths_on_the_old_ones():
    a = call()
    one = torch.zeros(4, dtype=I32)
    a["lengths"], a["new_lengths"] = one[1:3], one[:2]
    st, message = run("evict", a)
    assert st == 1 and "of their own" in message
