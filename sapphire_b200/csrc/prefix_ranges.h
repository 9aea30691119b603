// prefix_ranges.h - how the blocks of prefix_kernel.cuh share its work, on the host and the GPU.
#pragma once

#ifdef __CUDACC__
#define PREFIX_FN __host__ __device__ inline
#else
#define PREFIX_FN inline
#endif

// How the blocks share the units (a tile of tokens of one item): each item cut into
// `parts` equal pieces, a block each; or, where that would leave blocks without work for
// longer than a block's second item costs it (its queries, and results of its own: about
// kItemUnits units), all units in a row into equal ranges, item by item.
constexpr int kItemUnits = 5;
struct PrefixRanges {
    unsigned tiles;                // of an item
    unsigned parts;                // of an item, or 0: ranges
    unsigned total, blocks, each, longer;      // of an item's tiles where it has parts, of all units else: `longer` pieces of each + 1, then pieces of each
};
PREFIX_FN PrefixRanges prefix_ranges(unsigned items, unsigned length, unsigned tile, unsigned blocks) {
    PrefixRanges r;
    r.tiles = (length + tile - 1) / tile;
    r.total = items * r.tiles;
    r.blocks = r.total < blocks ? r.total : blocks;
    r.parts = 0;
    r.each = r.blocks ? r.total / r.blocks : 0;
    r.longer = r.total - r.each * r.blocks;
    if (r.blocks && items <= blocks) {
        const unsigned most = blocks / items, parts = most < r.tiles ? most : r.tiles, each = r.tiles / parts, longer = r.tiles - each * parts;
        if (each + (longer ? 1 : 0) <= r.each + kItemUnits) {
            r.parts = parts;
            r.blocks = items * parts;
            r.each = each;
            r.longer = longer;
        }
    }
    return r;
}
// A block's item, and the first of its tiles there and its units.
struct PrefixPiece {
    unsigned item, tile, units;
};
PREFIX_FN PrefixPiece prefix_piece(const PrefixRanges &r, unsigned block) {
    PrefixPiece x;
    const unsigned item = r.parts ? block / r.parts : 0, piece = block - item * r.parts;       // (parts 0: the block)
    const unsigned first = piece * r.each + (piece < r.longer ? piece : r.longer);
    x.units = r.each + (piece < r.longer ? 1 : 0);
    x.item = r.parts ? item : first / r.tiles;
    x.tile = r.parts ? first : first - x.item * r.tiles;
    return x;
}
// The blocks that hold an item.
PREFIX_FN void prefix_holders(const PrefixRanges &r, unsigned item, unsigned *first, unsigned *last) {
    if (r.parts) {
        *first = item * r.parts;
        *last = *first + r.parts - 1;
        return;
    }
    const unsigned split = r.longer * (r.each + 1), a = item * r.tiles, b = a + r.tiles - 1;
    *first = a < split ? a / (r.each + 1) : r.longer + (a - split) / r.each;
    *last = b < split ? b / (r.each + 1) : r.longer + (b - split) / r.each;
}
