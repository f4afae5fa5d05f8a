// Where a block of the prompt kernels works.  Plain C++: the launch, the kernels and a test on the host use it.
#pragma once

#include <algorithm>
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

// Whether the prefix attention may make one list of the rows of all requests of a prefix, whose states need room.
// packed: a request's rows of a KV head; all_rows: the call's.
constexpr bool r2o_prefix_room(int64_t packed, int64_t all_rows) { return packed < 512 && (packed < 128 || all_rows <= 1 << 18); }

// A key tile of a row list, in microseconds of a compute unit: 256 rows are bound by their products, up to 128 by the loads.  Measured
// where the keys come from memory (1 GB of them): 28 and 63 rows 1.4, 112 and 126 1.6, 133 2.05, 168 2.2, 224 2.4, 252 2.5; where they lie
// in the 256 MB behind the L2s 1.1, 1.2, 1.8, 1.85, 1.95 and 2.05 (63, 112, 133, 168, 224 and 252).
constexpr double r2o_prefix_tile_cost(int64_t rows) {
    const int64_t left = rows % 256;
    return 2.3 * (double)(rows / 256) + (left > 128 ? 2.3 : left > 0 ? 1.5 : 0.0);
}

// Whether it does: one list of a prefix's rows wastes row tiles once a prefix and not once a request, but leaves each row's state to a
// join.  Priced, in microseconds of a compute unit a request and head, by the prefixes' slots that the tables hold, for the lengths are
// on the device; with counts, as if they were a quarter to all of the rows.  Measured, in us apart and in one list, heads 28 over 4, 16
// requests over 32000 slots and 2000 own: 7 rows a request and KV head 173 and 41, 84: 191 and 134, 280: 572 and 340, 448: 572 and 524;
// over 8000 and 8000 own 7: 91 and 58, 56: 101 and 81, 280: 281 and 223; 64 requests over 2100 and 2000 own 84: 101 and 91, 126: 107 and
// 115, 280: 236 and 246.  Without a prefix one list wins by its join: one request of 126 rows over 32000 slots 42 and 32, 16 over 8000 71
// and 64; but for 25 to 32 rows, which single waves take: 28 rows 33 and 37, and 55 and 59.
// Requests a prefix are taken to be alike, and the table's rows to be used: 16 requests of 84 rows that all share one of 16 table rows
// are kept apart and take 199 us, one of two 135.
constexpr bool r2o_prefix_merged(int64_t batch, int64_t prefixes, int64_t packed, int64_t all_rows, int64_t shared, bool some_count) {
    if (!r2o_prefix_room(packed, all_rows)) return false;
    if (!prefixes) return packed <= 24 || packed > 32;
    if (packed <= 32) return true;
    const int64_t members = std::max<int64_t>(1, batch / prefixes), rows = some_count ? (5 * packed + 7) / 8 : packed, parts = some_count ? 4 : 1;
    double tile = 0.0;
    for (int64_t i = 1; i <= parts; ++i) tile += r2o_prefix_tile_cost((i * packed + parts - 1) / parts) / (double)parts;
    return (double)shared / 64 * (tile - r2o_prefix_tile_cost(rows * members) / (double)members) > 0.2 * (double)rows;
}

// What a segment's start and end cost beside its tiles, in tiles: of a workgroup about nine microseconds beside 2.3 a tile of 256
// rows, of one wave among eight five beside four.
constexpr int kR2oSegment = 4, kR2oWaveSegment = 1;

// Units (tiles, and what segments cost) of the longest list of such a call, at most: whatever the lengths on the device say.
// slots: the requests' own; shared: the prefixes'.
constexpr int64_t r2o_prefix_units(bool merged, int64_t batch, int64_t hkv, int64_t packed, int64_t slots, int64_t prefixes, int64_t shared) {
    const int64_t own = (slots + 63) / 64, keys = prefixes ? (shared + 63) / 64 : 0;
    return merged ? std::max(hkv * (batch * packed / 256 + prefixes) * (keys + kR2oSegment), hkv * batch * ((packed + 31) / 32) * (2 * own + kR2oWaveSegment))
                  : hkv * batch * ((packed + 255) / 256) * (1 + keys + own + kR2oSegment);
}

// Scratch of such a call, in floats: states of 130, two tiles of 256 rows a workgroup and, merged, two of each row, then eight words
// for each request or workgroup and for all.
constexpr int64_t r2o_prefix_states(int64_t workers, bool merged, int64_t all_rows) { return 512 * workers + (merged ? 2 * all_rows : 0); }
constexpr int64_t r2o_prefix_scratch(int64_t workers, bool merged, int64_t all_rows, int64_t batch) {
    return 130 * r2o_prefix_states(workers, merged, all_rows) + 8 * (1 + std::max(batch, workers));
}
