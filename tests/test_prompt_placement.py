"""Which die works on which tiles of a prompt, computed on the host from the function that the kernels use."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "r2-omni_amd", "csrc")
ROWS, KEYS = 128, 64  # packed rows and keys of a tile

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "r2o_place.hpp"
int main(int, char** v) {
    const int tiles = atoi(v[1]), splits = atoi(v[2]), batch = atoi(v[3]), hkv = atoi(v[4]);
    for (int64_t b = 0; b < r2o_place_blocks(tiles, splits, batch, hkv); ++b) {
        const R2oPlace p = r2o_place((int)b, tiles, splits, batch, hkv);
        if (p.valid) printf("%d %d %d %d\n", (int)(b & 7), p.pair, p.tile, p.split);
    }
}
"""


@pytest.fixture(scope="module")
def places(tmp_path_factory):
    """(die, pair, tile, split) of every block with work."""
    folder = tmp_path_factory.mktemp("place")
    (folder / "place.cpp").write_text(PROGRAM)
    exe = folder / "place"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(folder / "place.cpp"), "-o", str(exe)], check=True)

    def run(*numbers):
        text = subprocess.run([str(exe), *map(str, numbers)], capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in text.splitlines()]

    return run


@pytest.mark.parametrize("hkv", [1, 2, 3, 4, 5, 6, 8, 12, 16])
@pytest.mark.parametrize("tiles,splits,batch", [(1, 1, 1), (7, 1, 2), (3, 4, 3), (34, 7, 1), (11, 2, 8)])
def test_every_item_has_one_block(places, tiles, splits, batch, hkv):
    got = [p[1:] for p in places(tiles, splits, batch, hkv)]
    assert sorted(got) == [(p, t, s) for p in range(batch * hkv) for t in range(tiles) for s in range(splits)]


@pytest.mark.parametrize("hq,hkv", [(28, 4), (16, 2), (32, 8), (12, 1), (8, 8)])
@pytest.mark.parametrize("rows", [(8192,), (8192, 5003, 1231), (8192, 1024), (8192, 4000, 4000, 4000), (8192, 2048, 1024, 512), (300, 8192)])
def test_dies_share_the_key_tiles_of_uneven_requests(places, rows, hq, hkv):
    """Causal prompts of their own lengths in one padded batch, as prompt_attention places it: the busiest die has at most a
    tenth over the mean."""
    group = hq // hkv
    tiles, load = -(-max(rows) * group // ROWS), [0] * 8
    for die, pair, tile, _ in places(tiles, 1, len(rows), hkv):
        n, first = rows[pair // hkv], (tiles - 1 - tile) * ROWS // group
        last = min(((tiles - 1 - tile) * ROWS + ROWS - 1) // group, max(rows) - 1)
        load[die] += -(-(min(last, n - 1) + 1) // KEYS) if first < n else 0
    assert max(load) <= 1.1 * sum(load) / 8
