"""The rule that chooses a kernel for a product of 8-bit floating point, against times of
the ways that a product has, taken on an MI355X."""
import os
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KERNELS = os.path.join(REPO, "torch-gcu_amd", "csrc", "kernels")

TIMES = {  # us by (way, its index in the rule, slices of K)
    ("linear", 777, 4096, 4096): {
        ("tile", 0, 1): 43.3, ("tile", 1, 1): 21.0, ("tile", 2, 1): 23.5, ("tile", 3, 1): 29.4,
        ("tile", 3, 2): 39.1, ("tile", 3, 4): 47.2,
    },
    ("linear", 355, 7616, 10880): {
        ("tile", 0, 1): 105.1, ("tile", 1, 1): 48.4, ("tile", 2, 1): 55.7, ("tile", 3, 1): 59.4,
        ("tile", 3, 2): 72.7, ("tile", 3, 4): 81.2,
    },
    ("linear", 48, 4096, 11008): {
        ("few", 4, 1): 15.8, ("tile", 0, 1): 101.8, ("tile", 1, 1): 43.8, ("tile", 2, 1): 36.6,
        ("tile", 3, 1): 24.9, ("tile", 3, 2): 18.2, ("tile", 3, 4): 14.7,
    },
    ("linear", 32, 4096, 4096): {
        ("few", 3, 1): 6.8, ("tile", 0, 1): 42.1, ("tile", 1, 1): 19.1, ("tile", 2, 1): 15.8,
        ("tile", 3, 1): 11.3, ("tile", 3, 2): 10.4, ("tile", 3, 4): 9.8,
    },
    ("linear", 64, 4096, 4096): {
        ("few", 5, 1): 9.1, ("tile", 0, 1): 42.2, ("tile", 1, 1): 19.1, ("tile", 2, 1): 16.2,
        ("tile", 3, 1): 11.6, ("tile", 3, 2): 11.2, ("tile", 3, 4): 11.0,
    },
    ("linear", 128, 4096, 4096): {
        ("tile", 0, 1): 42.2, ("tile", 1, 1): 19.9, ("tile", 2, 1): 16.2, ("tile", 3, 1): 11.7,
        ("tile", 3, 2): 12.6, ("tile", 3, 4): 15.3,
    },
    ("linear", 512, 4096, 4096): {
        ("tile", 0, 1): 43.2, ("tile", 1, 1): 20.7, ("tile", 2, 1): 17.1, ("tile", 3, 1): 17.4,
        ("tile", 3, 2): 26.0, ("tile", 3, 4): 32.3,
    },
    ("linear", 2048, 4096, 11008): {
        ("tile", 0, 1): 107.0, ("tile", 1, 1): 89.5, ("tile", 2, 1): 121.2, ("tile", 3, 1): 152.0,
    },
    ("linear", 8192, 4096, 11008): {
        ("tile", 0, 1): 260.7, ("tile", 1, 1): 346.7, ("tile", 2, 1): 469.4, ("tile", 3, 1): 581.0,
    },
    ("linear", 60, 14272, 256): {
        ("few", 5, 1): 8.6, ("tile", 0, 1): 11.0, ("tile", 1, 1): 5.6, ("tile", 2, 1): 4.4,
        ("tile", 3, 1): 3.8, ("tile", 3, 2): 9.9, ("tile", 3, 4): 14.8,
    },
    ("linear", 50, 12848, 384): {
        ("few", 5, 1): 8.5, ("tile", 0, 1): 12.3, ("tile", 1, 1): 5.9, ("tile", 2, 1): 4.9,
        ("tile", 3, 1): 4.2, ("tile", 3, 2): 9.0, ("tile", 3, 4): 13.0,
    },
    ("linear", 30, 496, 10880): {
        ("few", 3, 1): 8.4, ("tile", 0, 1): 96.8, ("tile", 1, 1): 39.2, ("tile", 2, 1): 30.1,
        ("tile", 3, 1): 21.9, ("tile", 3, 2): 15.4, ("tile", 3, 4): 10.9,
    },
    ("linear", 5019, 352, 10112): {
        ("tile", 0, 1): 97.0, ("tile", 1, 1): 39.5, ("tile", 2, 1): 31.2, ("tile", 3, 1): 33.9,
    },
    ("linear", 59, 4768, 5120): {
        ("few", 5, 1): 17.1, ("tile", 0, 1): 52.7, ("tile", 1, 1): 23.9, ("tile", 2, 1): 20.7,
        ("tile", 3, 1): 14.7, ("tile", 3, 2): 13.0, ("tile", 3, 4): 14.5,
    },
    ("linear", 17, 1024, 4096): {
        ("few", 2, 1): 4.4, ("few", 3, 1): 5.1, ("tile", 0, 1): 40.7, ("tile", 1, 1): 17.0,
        ("tile", 2, 1): 13.1, ("tile", 3, 1): 10.0, ("tile", 3, 2): 8.9, ("tile", 3, 4): 7.6,
    },
    ("gate", 64, 11008, 4096): {
        ("few", 3, 1): 32.3, ("tile", 0, 1): 48.9, ("tile", 1, 1): 32.5, ("tile", 2, 1): 29.9,
        ("tile", 2, 2): 25.7, ("tile", 2, 4): 34.8,
    },
    ("gate", 32, 11008, 4096): {
        ("few", 2, 1): 22.9, ("tile", 0, 1): 47.7, ("tile", 1, 1): 31.5, ("tile", 2, 1): 28.3,
        ("tile", 2, 2): 22.8, ("tile", 2, 4): 29.2,
    },
    ("gate", 128, 11008, 4096): {
        ("tile", 0, 1): 48.3, ("tile", 1, 1): 35.4, ("tile", 2, 1): 29.8, ("tile", 2, 2): 43.5,
        ("tile", 2, 4): 48.6,
    },
    ("gate", 256, 11008, 4096): {
        ("tile", 0, 1): 49.3, ("tile", 1, 1): 35.7, ("tile", 2, 1): 51.9, ("tile", 2, 2): 63.1,
        ("tile", 2, 4): 84.6,
    },
    ("gate", 384, 11008, 4096): {
        ("tile", 0, 1): 49.5, ("tile", 1, 1): 59.5, ("tile", 2, 1): 64.2, ("tile", 2, 2): 90.3,
        ("tile", 2, 4): 123.8,
    },
    ("gate", 512, 11008, 4096): {
        ("tile", 0, 1): 50.5, ("tile", 1, 1): 64.9, ("tile", 2, 1): 74.6, ("tile", 2, 2): 115.1,
        ("tile", 2, 4): 157.8,
    },
    ("gate", 640, 6784, 4096): {
        ("tile", 0, 1): 47.2, ("tile", 1, 1): 59.2, ("tile", 2, 1): 62.3, ("tile", 2, 2): 79.7,
        ("tile", 2, 4): 113.3,
    },
    ("gate", 1024, 4224, 4096): {
        ("tile", 0, 1): 46.5, ("tile", 1, 1): 59.4, ("tile", 2, 1): 61.1, ("tile", 2, 2): 81.1,
        ("tile", 2, 4): 105.0,
    },
    ("gate", 1024, 11008, 4096): {
        ("tile", 0, 1): 101.5, ("tile", 1, 1): 98.6, ("tile", 2, 1): 142.5, ("tile", 2, 2): 221.2,
        ("tile", 2, 4): 333.0,
    },
    ("gate", 4096, 11008, 4096): {
        ("tile", 0, 1): 311.5, ("tile", 1, 1): 357.7, ("tile", 2, 1): 531.5,
    },
    ("gate", 1510, 2704, 5376): {
        ("tile", 0, 1): 56.7, ("tile", 1, 1): 74.2, ("tile", 2, 1): 74.6,
    },
    ("gate", 1227, 2752, 640): {
        ("tile", 0, 1): 17.5, ("tile", 1, 1): 9.9, ("tile", 2, 1): 12.8,
    },
    ("gate", 539, 4096, 4352): {
        ("tile", 0, 1): 49.2, ("tile", 1, 1): 31.5, ("tile", 2, 1): 47.5, ("tile", 2, 2): 52.5,
        ("tile", 2, 4): 62.3,
    },
    ("gate", 182, 12016, 4608): {
        ("tile", 0, 1): 55.2, ("tile", 1, 1): 38.8, ("tile", 2, 1): 60.8, ("tile", 2, 2): 64.7,
        ("tile", 2, 4): 72.8,
    },
    ("gate", 51, 4848, 640): {
        ("few", 3, 1): 9.3, ("tile", 0, 1): 16.6, ("tile", 1, 1): 9.1, ("tile", 2, 1): 6.8,
        ("tile", 2, 2): 10.4, ("tile", 2, 4): 12.2,
    },
}

# sizes by the way that they go (256 CUs): K of odd and even steps of 128, with and without a
# rest, few steps
LINEAR = {
    ("few", 0, 1): [(8, 101, 266), (7, 333, 2051)],
    ("few", 1, 1): [(16, 107, 137), (13, 1030, 1290)],
    ("few", 2, 1): [(24, 103, 262), (17, 1111, 901)],
    ("few", 3, 1): [(25, 111, 283), (31, 4090, 131), (32, 1003, 1037)],
    ("few", 4, 1): [(48, 121, 145), (41, 1107, 1153)],
    ("few", 5, 1): [(64, 109, 294), (49, 1115, 1027)],
    ("tile", 0, 1): [(3202, 4831, 1648), (2998, 5043, 1717)],
    ("tile", 1, 1): [(777, 5113, 30), (2706, 1409, 128), (1170, 3360, 256), (6533, 517, 386), (602, 6649, 385)],
    ("tile", 2, 1): [(5514, 357, 128), (130, 11641, 260), (211, 8347, 391), (134, 11249, 523)],
    ("tile", 3, 1): [(71, 73, 31), (65, 63, 128), (68, 63, 258), (65, 61, 411), (84, 87, 512), (65, 61, 660)],
    ("tile", 3, 2): [(56, 4201, 3871), (50, 4105, 3522)],
    ("tile", 3, 4): [(65, 115, 2056), (66, 105, 2015)],
}
GATE = {
    ("few", 0, 1): [(8, 101, 269), (7, 333, 2051)],
    ("few", 1, 1): [(16, 103, 257), (13, 1030, 1290)],
    ("few", 2, 1): [(32, 109, 276), (17, 101, 151)],
    ("few", 3, 1): [(64, 109, 272), (40, 101, 135)],
    ("tile", 0, 1): [(2717, 1419, 525), (5533, 653, 411), (4238, 914, 512)],
    ("tile", 1, 1): [(8853, 133, 34), (5888, 301, 128), (8385, 131, 267), (5883, 277, 526)],
    ("tile", 2, 1): [(72, 67, 30), (77, 65, 128), (71, 63, 261), (65, 61, 419), (70, 91, 512), (67, 105, 514)],
    ("tile", 2, 2): [(65, 4313, 2683), (72, 4241, 2484)],
    ("tile", 2, 4): [(69, 101, 1293), (65, 103, 1497)],
}


PICKS = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "fp8_rule.h"
using namespace mi;

int main(int n, char** a) {
  for (int i = 1; i + 3 < n; i += 4) {
    const int m = atoi(a[i + 1]), cols = atoi(a[i + 2]), k = atoi(a[i + 3]);
    const Fp8Way w = strcmp(a[i], "gate") ? fp8_pick_linear(m, cols, k, 256) : fp8_pick_gate(m, cols, k, 256);
    printf("%d %d %d\n", w.few, w.shape, w.slices);
  }
}
"""


def picks(tmp_path, sizes):
    """(way, index, slices) of each (op, M, N, K), on 256 CUs."""
    src, exe = tmp_path / "picks.cpp", tmp_path / "picks"
    src.write_text(PICKS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover=all", "-I", KERNELS, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe), *(str(x) for size in sizes for x in size)], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr
    found = [tuple(int(x) for x in line.split()) for line in r.stdout.splitlines()]
    return [("few", few, 1) if few >= 0 else ("tile", shape, slices) for few, shape, slices in found]


def test_picks_are_near_the_fastest_way(tmp_path):
    """Within a quarter of it everywhere, and on average within 3 %."""
    worse = []
    for (size, times), way in zip(TIMES.items(), picks(tmp_path, TIMES)):
        worse.append(times[way] / min(times.values()))
        assert worse[-1] <= 1.25, f"{size}: {way} takes {times[way]}, {min(times, key=times.get)} {min(times.values())}"
    assert sum(worse) / len(worse) <= 1.03


def test_picks_of_the_least_and_largest_sizes(tmp_path):
    """Any size has a way, and slices of K have whole groups."""
    sizes = [(op, m, n, k) for op in ("linear", "gate") for m in (1, 16, 17, 64, 65, 5000, 0x7FFF0000)
             for n in (1, 15, 129, 33000, 0x7FFF0000) for k in (0, 1, 127, 129, 600, (1 << 22) - 16)]
    for (_, m, _, k), (way, i, slices) in zip(sizes, picks(tmp_path, sizes)):
        assert slices in (1, 2, 4) and (slices == 1 or -(-k // 128) >= 2 * slices)
        assert way == "tile" or m <= 64


def test_few_rows_have_room_for_their_scales(tmp_path):
    """A few-row kernel holds every scale of its rows in LDS: longer rows go to tiles."""
    sizes = [(op, m, 4096, k) for op in ("linear", "gate") for m in (1, 9, 33, 64) for k in (4096, 1 << 21)]
    for (_, _, _, k), (way, _, _) in zip(sizes, picks(tmp_path, sizes)):
        assert way == "tile" or k == 4096


def test_every_way_has_sizes_that_go_it(tmp_path):
    """What the kernels are tested at reaches all of them."""
    named = [(op, *size, way) for op, ways in (("linear", LINEAR), ("gate", GATE))
             for way, sizes in ways.items() for size in sizes]
    for size, way in zip(named, picks(tmp_path, [n[:4] for n in named])):
        assert way == size[4], size


def test_more_columns_than_small_tiles_have_a_grid_for(tmp_path):
    """Go to the largest tiles."""
    sizes = [(op, m, 1 << 30, 16) for op in ("linear", "gate") for m in (17, 64, 65)]
    assert picks(tmp_path, sizes) == [("tile", 0, 1)] * 6
