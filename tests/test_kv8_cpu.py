"""The 8-bit key/value cache without a GPU: what its entry points refuse, and the
index arithmetic that keeps every access in bounds whatever lengths, starts and
page numbers the device tensors hold."""
import os
import subprocess

import pytest
import torch

from oracle import kv8 as oracle
from torch_gcu import _abi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KERNELS = os.path.join(REPO, "torch-gcu_amd", "csrc", "kernels")
INVALID, UNSUPPORTED, TOO_LARGE = 1, 2, 5


def call(pages=3, heads=2, page=16, d=64, seqs=2, width=2, tokens=4, group=2, dtype=torch.bfloat16):
    """Valid arguments of all four calls, by name."""
    u8, f32, i32 = torch.uint8, torch.float32, torch.int32
    return {
        "k_cache": torch.zeros(pages, heads, page, d, dtype=u8),
        "v_cache": torch.zeros(pages, heads, page, d, dtype=u8),
        "k_scale": torch.zeros(pages, heads), "v_scale": torch.zeros(pages, heads),
        "k": torch.zeros(tokens, heads, d, dtype=dtype), "v": torch.zeros(tokens, heads, d, dtype=dtype),
        "q": torch.zeros(tokens, heads * group, d, dtype=dtype),
        "out": torch.zeros(tokens, heads * group, d, dtype=dtype),
        "lse": torch.zeros(tokens, heads * group, dtype=f32),
        "table": torch.zeros(seqs, width, dtype=i32), "lengths": torch.zeros(seqs, dtype=i32),
        "starts": torch.zeros(seqs + 1, dtype=i32),
        "weights": torch.zeros(seqs, heads, width * page), "new_weights": torch.zeros(seqs, heads, width * page),
        "new_table": torch.zeros(seqs, 1, dtype=i32), "kept": torch.zeros(seqs, heads, 5, dtype=i32),
        "new_lengths": torch.zeros(seqs, dtype=i32),
        "keep": 5, "recent": 2, "sink": 1, "scale": 0.1,
    }


ORDER = {
    "append": ["cache", "k", "v", "table", "lengths", "starts", "stream"],
    "attention": ["out", "lse", "q", "cache", "table", "lengths", "starts", "scale", "fill", "stream"],
    "weigh": ["weights", "q", "lse", "cache", "table", "lengths", "starts", "scale", "stream"],
    "evict": ["cache", "weights", "table", "new_table", "lengths", "keep", "recent", "sink", "kept",
              "new_lengths", "new_weights", "stream"],
}


def run(op, a):
    def arg(n):
        if n == "cache":
            return _abi.MiKv8Cache(*(_abi.desc(a[x]) for x in ("k_cache", "v_cache", "k_scale", "v_scale")))
        if n == "stream":
            return None
        if n == "fill":
            return 0
        return _abi.desc(a[n]) if isinstance(a[n], torch.Tensor) else a[n]

    st = getattr(_abi.lib(), "mi_kv8_" + op)(*(arg(n) for n in ORDER[op]))
    return st, _abi.lib().mi_last_error().decode()


ALL = ("append", "attention", "weigh", "evict")
REFUSED = [
    # (ops, changed argument, its new value, status, words of the message)
    (ALL, "k_cache", lambda t: t.to(torch.int8), INVALID, "uint8"),
    (ALL, "k_cache", lambda t: t[0], INVALID, "uint8"),
    (ALL, "v_cache", lambda t: t[:2].contiguous(), INVALID, "different shapes"),
    (ALL, "k_cache", lambda t: torch.zeros(3, 2, 64, 16, dtype=torch.uint8).transpose(2, 3), INVALID, "dense"),
    (ALL, "k_cache", lambda t: torch.zeros(3 * 2 * 16 * 64 + 1, dtype=torch.uint8)[1:].view(t.shape), INVALID, "aligned"),
    (ALL, "k_cache", lambda t: t[:1].expand(3, 2, 16, 64), INVALID, "overlap"),
    (ALL, "k_cache", lambda t: t.as_strided(t.shape, (16 * 64, 16 * 64, 64, 1)), INVALID, "overlap"),
    (ALL, "k_scale", lambda t: t.as_strided((3, 2), (1, 1)), INVALID, "overlap"),
    (ALL, "k_scale", lambda t: t.double(), INVALID, "float32"),
    (ALL, "v_scale", lambda t: t[:, :1], INVALID, "float32 [pages, heads]"),
    (ALL, "k_scale", lambda t: t[:1].expand(3, 2), INVALID, "overlap"),
    (ALL, "table", lambda t: t.long(), INVALID, "int32"),
    (ALL, "table", lambda t: t.t().contiguous().t(), INVALID, "dense rows"),
    (ALL, "lengths", lambda t: t.long(), INVALID, "int32"),
    (ALL, "lengths", lambda t: t[:1], INVALID, "entries"),
    (ALL, "lengths", lambda t: torch.zeros(4, dtype=torch.int32)[::2], INVALID, "dense"),
    (ALL, "table", lambda t: torch.zeros(2, 0, dtype=torch.int32), INVALID, "columns"),
    (ALL[:3], "starts", lambda t: t[:2], INVALID, "entries"),
    (ALL[:3], "starts", lambda t: t.long(), INVALID, "int32"),
    (("append",), "k", lambda t: t.float(), INVALID, "bfloat16 or float16"),
    (("append",), "v", lambda t: t.half(), INVALID, "both"),
    (("append",), "k", lambda t: t[:, :1], INVALID, "heads"),
    (("append",), "v", lambda t: t[:3], INVALID, "numbers of tokens"),
    (("append",), "k", lambda t: torch.zeros(4, 2, 128, dtype=t.dtype)[..., ::2], UNSUPPORTED, "dense"),
    (("append",), "k", lambda t: torch.zeros(4 * 128 + 1, dtype=t.dtype)[1:].view(t.shape), UNSUPPORTED, "aligned"),
    (("attention", "weigh"), "q", lambda t: t.float(), INVALID, "bfloat16 or float16"),
    (("attention", "weigh"), "q", lambda t: t[:, :3], INVALID, "heads"),
    (("attention", "weigh"), "q", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)[..., ::2], INVALID, "heads"),
    (("attention", "weigh"), "lse", lambda t: t.double(), INVALID, "float32"),
    (("attention", "weigh"), "lse", lambda t: t[:, :2], INVALID, "lse"),
    (("attention", "weigh"), "scale", lambda s: float("nan"), INVALID, "finite"),
    (("attention",), "out", lambda t: t.half(), INVALID, "type"),
    (("attention",), "out", lambda t: t[:2], INVALID, "shape"),
    (("weigh", "evict"), "weights", lambda t: t[..., :31].contiguous(), INVALID, "positions"),
    (("weigh", "evict"), "weights", lambda t: t.double(), INVALID, "float32"),
    (("weigh", "evict"), "weights", lambda t: t[:, :1].expand(2, 2, 32), INVALID, "overlap"),
    (("weigh", "evict"), "weights", lambda t: t.as_strided((2, 2, 32), (32, 32, 1)), INVALID, "overlap"),
    (("attention",), "out", lambda t: t[:1].expand(t.shape), INVALID, "overlap"),
    (("attention",), "lse", lambda t: t.as_strided(t.shape, (1, 1)), INVALID, "overlap"),
    (("evict",), "kept", lambda t: t.as_strided(t.shape, (5, 5, 1)), INVALID, "kept"),
    (("evict",), "keep", lambda n: 0, INVALID, "keep"),
    (("evict",), "recent", lambda n: 5, INVALID, "keep"),
    (("evict",), "sink", lambda n: -1, INVALID, "keep"),
    (("evict",), "keep", lambda n: 17, INVALID, "new_table"),
    (("evict",), "kept", lambda t: t[..., :4].contiguous(), INVALID, "kept"),
    (("evict",), "new_lengths", lambda t: t.long(), INVALID, "new_lengths"),
]


@pytest.mark.parametrize("ops,name,change,status,words", REFUSED, ids=[f"{r[1]}-{i}" for i, r in enumerate(REFUSED)])
def test_refusals_come_before_any_device_call(ops, name, change, status, words):
    for op in ops:
        a = call()
        a[name] = change(a[name])
        st, message = run(op, a)
        assert st == status and words in message, (op, st, message)


@pytest.mark.parametrize("op", ALL)
@pytest.mark.parametrize("d,status", [(32, UNSUPPORTED), (96, UNSUPPORTED), (256, UNSUPPORTED)])
def test_head_dims_that_have_no_kernel(op, d, status):
    st, message = run(op, call(d=d))
    assert st == status and "head_dim" in message


@pytest.mark.parametrize("op", ALL)
@pytest.mark.parametrize("page", [8, 48, 512])
def test_page_sizes(op, page):
    st, message = run(op, call(page=page))
    assert st == INVALID and "page size" in message


@pytest.mark.parametrize("ops,one,other,words", [
    (("append", "evict"), "v_cache", "k_cache", "same memory"),
    (("append", "evict"), "v_scale", "k_scale", "same memory"),
    (("evict",), "new_lengths", "lengths", "of their own"),
    (("evict",), "new_weights", "weights", "of their own"),
])
def test_what_is_written_has_memory_of_its_own(ops, one, other, words):
    for op in ops:
        a = call()
        a[one] = a[other]
        st, message = run(op, a)
        assert st == INVALID and words in message, (op, st, message)


def test_null_cache():
    a = call()
    st = _abi.lib().mi_kv8_append(None, *(_abi.desc(a[n]) for n in ORDER["append"][1:-1]), None)
    assert st == INVALID and b"cache is NULL" in _abi.lib().mi_last_error()


def test_nothing_to_do_is_no_error():
    """No tokens, no sequences: done before any device call."""
    for op in ("append", "attention", "weigh"):
        a = call(tokens=0)
        assert run(op, a)[0] == 0
    assert run("evict", call(seqs=0))[0] == 0


def test_ops_refuse_cpu_tensors():
    import torch_gcu  # noqa: F401

    a = call()
    cache = torch.gcu.efficient.KV8Cache(a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.gcu.efficient.kv8_attention(a["q"], cache, a["table"], a["lengths"], a["starts"])


PROGRAM = r"""
#include <cassert>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <climits>
#include <initializer_list>
#include "kv8_index.h"
using namespace mi;

int main() {
  const int odd[] = {INT_MIN, -70000, -1, 0, 1, 2, 15, 16, 17, 63, 64, 65, 4095, 4096, 70000, INT_MAX - 1, INT_MAX};
  const int caps[] = {16, 64, 4096, 1 << 30}, sizes[] = {0, 1, 5, 4096};
  long n = 0;
  for (int start : odd) for (int next : odd) for (int length : odd) for (int cap : caps) for (int tokens : sizes) {
    const Kv8Seq s = kv8_seq(start, next, length, tokens, cap);
    assert(s.first >= 0 && s.n >= 0 && s.first + s.n <= tokens);
    assert(s.len >= 0 && s.len <= cap);
    assert(s.bad == (length < 0 || length > cap));
    for (int i : {0, s.n / 2, s.n - 1}) if (i >= 0 && i < s.n) {
      const int lim = kv8_limit(s, i);
      assert(lim >= 0 && lim <= s.len);
      assert((long)lim == (((long)s.len - s.n + i + 1) < 0 ? 0 : (long)s.len - s.n + i + 1));
    }
    for (int shift = 4; shift <= 8; ++shift) {
      const int t = kv8_touched(s, shift), size = 1 << shift;
      assert(t >= 0 && t <= kv8_touched_most(s.n, 1, shift));
      if (t > 0) {  // the pages touched lie in the table, and hold exactly the new positions
        const int old = s.len - s.n;
        long slots = 0;
        for (int k : {0, t - 1}) {
          const int index = (old >> shift) + k;
          assert(index >= 0 && (long)index < ((long)cap + size - 1) / size);
        }
        if (t < 300) {
          for (int k = 0; k < t; ++k) {
            const int index = (old >> shift) + k;
            const int lo = old - (index << shift) > 0 ? old - (index << shift) : 0;
            const int hi = s.len - (index << shift) < size ? s.len - (index << shift) : size;
            assert(lo >= 0 && lo < hi && hi <= size);
            slots += hi - lo;
          }
          assert(slots == s.n);
        }
      }
    }
    for (int group : {1, 3, 8}) for (int rt : {16, 32, 128, 256}) for (int kt : {32, 64}) {
      const Kv8Cut c = kv8_cut(s, group, rt, kt);
      assert((long)c.row_tiles * rt >= c.rows && (long)(c.row_tiles - 1) * rt < c.rows);
      assert((long)c.key_tiles * kt >= s.len && ((long)c.key_tiles - 1) * kt < s.len);
      assert(c.row_tiles <= kv8_row_tiles_most(s.n, 1, group, rt));
      for (int target : {1, 256, 512}) for (int wide : {0, 24}) {
        const Kv8Plan plan{target, wide, 8, 2 * target};
        const int chunk = plan.chunk(c.work() * 8), parts = c.parts(chunk);
        assert(parts >= 1 && chunk >= 8);
        assert(8L * c.row_tiles * parts <= plan.many + 8L * c.row_tiles);
      }
    }
    ++n;
  }
  for (int entry : odd) for (int pages : {1, 7, 70000}) {
    const int p = kv8_page(entry, pages);
    assert(p >= -1 && p < pages && (p == entry || entry < 0 || entry >= pages));
  }
  // many sequences of any lengths: the parts fit the room that the host gives them
  srand(7);
  for (int round = 0; round < 2000; ++round) {
    const int seqs = 1 + rand() % 200, heads = 1 + rand() % 16, group = 1 + rand() % 8;
    const int rt = rand() % 2 ? 16 : 128, kt = rt == 16 ? 32 : 64;
    const Kv8Plan plan{256, rand() % 2 ? 0 : 24, 8, 512};
    long tokens = 0, items = 0, touched = 0;
    float work = 0;
    static Kv8Seq all[200];
    for (int b = 0; b < seqs; ++b) {
      const int m = rand() % 4 ? rand() % 3 : rand() % 500;
      all[b] = Kv8Seq{0, m, m + rand() % (1 << (rand() % 18 + 1)), false};
      tokens += m;
      work += kv8_cut(all[b], group, rt, kt).work();
      touched += kv8_touched(all[b], 4);
    }
    const int chunk = plan.chunk(work * heads);
    for (int b = 0; b < seqs; ++b) {
      const Kv8Cut c = kv8_cut(all[b], group, rt, kt);
      items += (long)heads * c.row_tiles * c.parts(chunk);
    }
    assert(items <= plan.many + heads * kv8_row_tiles_most(tokens, seqs, group, rt));
    assert(touched <= kv8_touched_most(tokens, seqs, 4));
    // rounds hold each tile of each sequence once, the farthest-seeing ones first
    int longest = 0;
    for (int b = 0; b < seqs; ++b) if (all[b].n > 0 && all[b].len > longest) longest = all[b].len;
    for (int b = 0; b < seqs && b < 64; ++b) {
      const Kv8Cut c = kv8_cut(all[b], group, rt, kt);
      const Kv8Rounds r(all[b], c, longest, group, rt);
      assert(r.off >= 0 && r.tiles == c.row_tiles && !r.in(-1) && r.before(0) == 0);
      int seen = 0;
      for (int k = r.off > 3 ? r.off - 3 : 0; k < r.off + r.tiles + 3; ++k) {
        assert(r.before(k) == seen);
        seen += r.in(k);
        if (r.in(k)) assert(k - r.off >= 0 && k - r.off < c.row_tiles);
      }
      assert(seen == c.row_tiles);
    }
  }
  for (unsigned u = 0; u < 0x7f800000u; u += 12345) {
    float x;
    memcpy(&x, &u, 4);
    const float s = kv8_scale_of(x);
    assert((double)x <= 448.0 * s && (s == 0x1p-110f || (double)x > 224.0 * s));
  }
  assert(kv8_scale_of(448.f) == 1.f && kv8_scale_of(449.f) == 2.f && kv8_scale_of(0.f) == 0x1p-110f);
  printf("%ld sequences\n", n);
}
"""


def test_index_arithmetic_stays_in_bounds(tmp_path):
    src, exe = tmp_path / "index.cpp", tmp_path / "index"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", KERNELS, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_oracle_codes_round_as_the_type_does():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.logspace(-12, 2.6, 20001), torch.zeros(1)])
    want = x.to(torch.float8_e4m3fn).double()
    assert torch.equal(oracle.e4m3(x.double()), want)
