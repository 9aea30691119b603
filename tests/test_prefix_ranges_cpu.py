"""How the blocks of the product over a shared prefix share its work, compiled for the host."""
from __future__ import annotations

import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include "prefix_ranges.h"
int main() {
    unsigned items, length, tile, blocks;
    while (std::scanf("%u %u %u %u", &items, &length, &tile, &blocks) == 4) {
        const PrefixRanges r = prefix_ranges(items, length, tile, blocks);
        std::printf("%u %u %u\n", r.tiles, r.parts, r.blocks);
        for (unsigned b = 0; b < r.blocks; ++b) {
            const PrefixPiece x = prefix_piece(r, b);
            std::printf("%u %u %u\n", x.item, x.tile, x.units);
        }
        for (unsigned i = 0; r.tiles && i < items; ++i) {
            unsigned first, last;
            prefix_holders(r, i, &first, &last);
            std::printf("%u %u\n", first, last);
        }
    }
}
"""


def prefix_ranges(folder, items, length, tile, blocks):
    """(tiles of an item, item's parts, [(item, tile, units) of a block], [(first, last) block of an item])."""
    src, exe = folder / "ranges.cpp", folder / "ranges"
    if not exe.exists():
        src.write_text(PROGRAM)
        subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{ROOT}/sapphire_b200/csrc", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], input=f"{items} {length} {tile} {blocks}", capture_output=True, text=True, check=True).stdout
    rows = [[int(x) for x in line.split()] for line in out.splitlines()]
    tiles, parts, used = rows[0]
    return tiles, parts, [tuple(x) for x in rows[1:1 + used]], [tuple(x) for x in rows[1 + used:]]


def items_of_blocks(folder, items, length, tile, blocks):
    """The items that each block takes, in its order."""
    tiles, _, pieces, _ = prefix_ranges(folder, items, length, tile, blocks)
    return [list(range(item, item + (first + units - 1) // tiles + 1)) for item, first, units in pieces]


@pytest.mark.parametrize("blocks", [148, 132, 4])
@pytest.mark.parametrize("items,length,tile", [(1, 0, 128), (1, 1, 128), (8, 4099, 80), (12, 2100, 128), (40, 2100, 128), (64, 32768, 80),
                                               (100, 2100, 128), (148, 300, 64), (149, 5, 80), (200, 2100, 128), (999, 30011, 48), (3, 2000001, 96)])
def test_blocks_take_every_tile_once(tmp_path, items, length, tile, blocks):
    tiles, parts, pieces, holders = prefix_ranges(tmp_path, items, length, tile, blocks)
    assert tiles == -(-length // tile) and len(pieces) <= blocks and len(pieces) >= min(blocks, items * tiles) - (items if parts else 0)
    at, seen = 0, [[] for _ in range(items)]
    for b, (item, first, units) in enumerate(pieces):
        assert units > 0 and item * tiles + first == at
        for i in range(item, (at + units - 1) // tiles + 1):
            seen[i].append(b)
        at += units
    assert at == items * tiles
    assert holders == ([(s[0], s[-1]) for s in seen] if tiles else [])
    if parts:
        assert all(first + units <= tiles for _, first, units in pieces)


def test_where_blocks_take_two_items(tmp_path):
    def shared(*a):
        return sum(len(x) > 1 for x in items_of_blocks(tmp_path, *a))
    assert shared(8, 4099, 80, 148) == 0 and shared(40, 2100, 128, 148) == 0
    assert shared(100, 2100, 128, 148) > 60 and shared(200, 2100, 128, 148) > 120
