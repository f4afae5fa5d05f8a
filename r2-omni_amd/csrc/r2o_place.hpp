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

// Whether the prefix attention may make one list of the rows of all requests of a prefix, and so needs room for their states.
// packed: a request's rows of a KV head; all_rows: the call's.
constexpr bool r2o_prefix_room(bool prefixes, int64_t packed, int64_t all_rows) {
    return prefixes && packed < 512 && (packed < 128 || all_rows <= 1 << 18);
}

// Whether it does.  Row tiles have 256 rows: a list wastes them once a prefix and not once a request, but leaves each row's state
// to a join, which takes as long as some hundred slots of a prefix.  Measured, in us apart and in one list, heads 28 over 4, 16
// requests of one prefix of 32641 slots: 168 rows a request 274 and 220, 252: 307 and 313, 280: 563 and 343, 448: 566 and 533, 511: 593 and
// 607; query_lengths that count five eighths of them: 270 and 132, 275 and 193, 303 and 219, 443 and 327, 414 and 376; eights of
// requests over 700 slots, heads 16 over 2, 288 rows: 45 and 53, 320: 44 and 58.
constexpr bool r2o_prefix_merged(bool prefixes, int64_t packed, int64_t all_rows, int64_t slots, bool some_count) {
    return r2o_prefix_room(prefixes, packed, all_rows) && (packed < 128 || (slots >= 2048 && (some_count || 4 * ((packed + 255) / 256 * 256 - packed) >= packed)));
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

// Scratch of such a call, in floats: states of 130, two tiles of 256 rows a workgroup and two of each row, then eight words for each
// request or workgroup and for all.
constexpr int64_t r2o_prefix_states(int64_t workers, bool room, int64_t all_rows) { return 512 * workers + (room ? 2 * all_rows : 0); }
constexpr int64_t r2o_prefix_scratch(int64_t workers, bool room, int64_t all_rows, int64_t batch) {
    return 130 * r2o_prefix_states(workers, room, all_rows) + 8 * (1 + std::max(batch, workers));
}
