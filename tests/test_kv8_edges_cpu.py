"""Edges of the 8-bit key/value cache that show without a GPU: the places that
its kernels load keys from."""
import os
import subprocess

import torch

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
