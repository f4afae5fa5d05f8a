// Where a block of the prompt kernels works.  Plain C++: the launch, the kernels and a test on the host use it.
#pragma once

#include <cstdint>

struct R2oPlace {
    int pair, tile, split;  // pair: batch number heads + head
    bool valid;             // false for a block that only fills the grid up
};

// Dies (of 8) that share a head where heads are 1, 2 or 4; otherwise a block's head goes by its number.
constexpr int r2o_dies_of_head(int64_t heads) { return heads == 1 || heads == 2 || heads == 4 ? (int)(8 / heads) : 1; }

// Blocks go to the 8 dies (XCDs) in turn, and a die's L2 is its own: where the heads allow it, a die works through the
// tiles of one pair after the other (or shares a pair with some), so that its workgroups read the same rows.  Each die works
// on all `batches`; a caller whose requests are of one length may call their heads one batch's.  Tile by tile, a tile's
// splits together: the caller's first tiles are the longest.
constexpr R2oPlace r2o_place(int block, int tiles, int splits, int batches, int heads) {
    const int items = tiles * splits, die = block & 7, i = block >> 3, dies = r2o_dies_of_head(heads);
    int pair = 0, rank = 0;
    bool valid = true;
    if (heads % 8 == 0) {
        pair = die + 8 * (i / items);
        rank = i % items;
    } else if (dies > 1) {
        const int at = i * dies + die % dies, batch = at / items;
        pair = batch * heads + die / dies;
        rank = at - batch * items;
        valid = batch < batches;
    } else {
        pair = block / items;
        rank = block % items;
    }
    const int tile = rank / splits;
    return {pair, tile, rank - tile * splits, valid};
}

// Blocks of a launch: a head's items in whole turns of the dies that share it.
constexpr int64_t r2o_place_blocks(int64_t tiles, int64_t splits, int64_t batches, int64_t heads) {
    const int64_t dies = r2o_dies_of_head(heads);
    return (batches * tiles * splits + dies - 1) / dies * dies * heads;
}
