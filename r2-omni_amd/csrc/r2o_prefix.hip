// Attention over a prefix that many requests share, and over each request's own slots of the paged cache, for gfx950.
//
// Requests of one prefix stand side by side; row i of request b (q of its rows count, n slots are its own) sees every
// slot of its prefix and its own slots j <= n - q + i:
//     out = sum_j softmax_j(c q . k_j) v_j,     lse = log sum_j exp(c q . k_j)
// over both.  Rows of a KV head's query heads and, where a request has few, of all requests of a prefix are one list, in
// tiles of 256: a wave's 32 rows are one operand of its products, eight waves share a key tile in LDS, and the prefix's rows are
// read once for all of them.  The (row tile, key tile) pairs of a call are one list too, shared evenly over the workgroups,
// whatever the lengths; where a row tile's keys fall to several, or to a prefix and a request of its own, each leaves (maximum,
// sum, products) in scratch for the join.  Beside them, where rows are merged, the requests' own slots, which no two share.
//
// What bounds it: a tile of 256 rows and 64 keys takes 2.3 to 2.7 us (790 to 930 TFLOP/s; a large library product of these types
// reaches 1220), 2.06 without its loads: exponentials beside products.  One of 129 to 224 rows takes 2.05 to 2.4 (1.8 to 1.95 where its
// keys lie in the 256 MB behind the L2s), one of up to 128 1.6, the rows' bytes at 5.3 TB/s.  A call has 22 to 27 us beside its
// tiles: lengths and shares 2, the first tile's pages and rows 5.5, a state's way out 4, the join's launch and way 6 to 13, and the
// uneven end.  64 requests over 65409 slots, heads 32 over 8: 113 us (105 to 118 card to card); 24 over 32641, 28 over 4: 43; 16 questions of 13
// to 58 rows over 16257: 165 to 174 (760 to 800 TFLOP/s).  With 128 rows a workgroup and two of them a compute unit 229, 73 and 345.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "r2o_cache_check.hpp"
#include "r2o_common.hpp"
#include "r2o_place.hpp"
#include "r2o_tiles.hpp"

namespace {

using namespace r2o_tiles;

constexpr int kWaves = 8;    // of a workgroup, which fills a compute unit
constexpr int kRows = 256;   // rows of a workgroup: a wave's 32 each; 128 or fewer: 32 for two waves, which share their keys
constexpr int kWaveRows = 32, kWaveKeys = 32;  // of a wave that works by itself
constexpr int kSegment = kR2oSegment, kWaveSegment = kR2oWaveSegment;
constexpr int kAhead = 4;    // tiles in LDS or on their way there, the one in use among them

// One cache's rows, in the kernels' widths (the host has checked that they fit).
struct Source {
    const uint16_t *key, *value;
    const int32_t *table, *lengths;
    int k_page, k_head, k_slot, v_page, v_head, v_slot, table_stride, pages, last_page, shift;
};

struct PrefixArgs {
    Source own, shared;
    const int32_t *members, *query_lengths;
    const uint16_t* query;
    uint16_t* out;
    float *lse, *partial_out, *partial_ml;
    int* notes;  // for the join
    int64_t q_batch, q_head, o_batch, o_head;
    int q_row, o_row, batch, prefixes, hkv, hq, group, rows, packed, workers;  // packed: rows * group
    float c2;  // scale, in log2 units
};

// The arguments where the hardware put them: each place that asks anew loads what it uses again, instead of holding them
// all in scalar registers.
typedef const __attribute__((address_space(4))) PrefixArgs Args;
typedef const __attribute__((address_space(4))) Source SourceArgs;

__device__ __forceinline__ Args& kernel_args() {
    auto p = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}

// A word at an address that the whole wave shares and that nothing writes meanwhile.
__device__ __forceinline__ int load_uniform(const int32_t* p) { return *(const __attribute__((address_space(4))) int32_t*)p; }

// Sums up to each lane of the wave: shifts within rows of 16 lanes, then the rows' last lanes handed on.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 to rows 2 and 3
    return x;
}

// A number that all lanes share, in a scalar register: compared where it is asked, not held as a mask of lanes.
__device__ __forceinline__ int opaque(int x) {
    asm("" : "+v"(x));
    return __builtin_amdgcn_readfirstlane(x);
}

__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }

__device__ __forceinline__ int filled(SourceArgs& s, int length) { return min(max(length, 0), (s.last_page + 1) << s.shift); }

// ------------------------------------------------------------------------------------- the work
// Where rows are merged there are two lists: the prefixes' (with the rows of all their requests), whose row tiles workgroups
// take as a whole, and the requests' own slots.  Those go to single waves, 32 rows and 32 keys at a time, where that costs less: a
// workgroup's eight have eight requests' latencies under way; or to workgroups in row tiles too.  Otherwise there is one list, of the
// requests, a prefix's slots before the own ones.  The wave goes through prefixes and requests 64 at a time, one a lane; what the
// first 64 hold is loaded at once and kept.
enum List { kPrefixes, kOwn, kRequests };  // whose row tiles a workgroup works on

struct Lane {
    int members, shared, own, rows;  // as the tensors have them: a prefix's, a request's
};

__device__ __forceinline__ Lane lane_of(int i0) {
    Args& a = kernel_args();
    const int i = i0 + (threadIdx.x & 63);
    Lane x{0, 0, 0, a.rows};
    if (i < a.prefixes) {
        x.members = a.members ? r2o_ldg(a.members + i) : a.batch;
        x.shared = r2o_ldg(a.shared.lengths + i);
    }
    if (i < a.batch) {
        x.own = r2o_ldg(a.own.lengths + i);
        if (a.query_lengths) x.rows = r2o_ldg(a.query_lengths + i);
    }
    return x;
}

__device__ __forceinline__ Lane lane_at(const Lane& first, int i0) { return i0 ? lane_of(i0) : first; }

struct Members {
    int first, count;  // requests of this lane's prefix
};

// Counts are cut off where the batch ends, so that whatever they hold no request has two prefixes.
__device__ __forceinline__ Members lane_members(const Lane& x, int& before) {
    Args& a = kernel_args();
    const int m = min(max(x.members, 0), a.batch), upto = wave_scan(m);
    Members r;
    r.first = min(before + upto - m, a.batch);
    r.count = min(m, a.batch - r.first);
    before = min(before + last_lane(upto), a.batch);
    return r;
}

__device__ __forceinline__ int div_up(int x, int by) { return (x + by - 1) / by; }

// The rows that count of the requests before b, one query head's: where query_lengths say so, summed up in LDS.
__device__ __forceinline__ int rows_before(const int* sums, int b) {
    Args& a = kernel_args();
    return a.query_lengths ? sums[b] : b * a.rows;
}

// Rows of a lane's prefix, of all query heads of a KV head.
__device__ __forceinline__ int member_rows(const int* sums, const Members& m) {
    return (rows_before(sums, m.first + m.count) - rows_before(sums, m.first)) * kernel_args().group;
}

__device__ __forceinline__ int counted_rows(int rows) {
    Args& a = kernel_args();
    return min(max(rows, 0), a.rows);
}

// A list's unit is a tile, or what a segment costs before its first one: kSegment or kWaveSegment units.
__device__ __forceinline__ int units(int segments, int tiles, int more) { return tiles ? segments * (tiles + more) : 0; }

// Of this lane's prefix (merged rows): heads x row tiles segments of its key tiles.
__device__ __forceinline__ int prefix_work(const Lane& x, int rows) {
    Args& a = kernel_args();
    return units(a.hkv * div_up(rows, kRows), div_up(filled(a.shared, x.shared), kTile), kSegment);
}

// Of this lane's request's own slots (merged rows), in tiles of 32 rows and 32 keys.
__device__ __forceinline__ int own_work(const Lane& x, int b0) {
    Args& a = kernel_args();
    const int b = b0 + (threadIdx.x & 63);
    return b < a.batch ? units(a.hkv * div_up(counted_rows(x.rows) * a.group, kWaveRows), div_up(filled(a.own, x.own), kWaveKeys), kWaveSegment) : 0;
}

// The same in row tiles and key tiles of workgroups.
__device__ __forceinline__ int own_row_work(const Lane& x, int b0) {
    Args& a = kernel_args();
    const int b = b0 + (threadIdx.x & 63);
    return b < a.batch ? units(a.hkv * div_up(counted_rows(x.rows) * a.group, kRows), div_up(filled(a.own, x.own), kTile), kSegment) : 0;
}

// What a request has to know of its prefix, in LDS: looked up by bisection.  One step a prefix, in every wave and for 64 requests
// at a time, took 17.9 ms where 1024 requests of 5 rows have a prefix each, of 64 slots, and 0.51 like this.
struct Prefixes {
    int units[R2O_PAGED_MAX_BATCH], slots[R2O_PAGED_MAX_BATCH];  // units: of the prefixes before it (merged rows)
    uint16_t ends[R2O_PAGED_MAX_BATCH];                          // its last request, and one
};

// By one wave; sums: merged rows, else nullptr.
__device__ __forceinline__ void write_prefixes(const Lane& first, const int* sums, Prefixes& p) {
    Args& a = kernel_args();
    int before = 0, at = 0;
#pragma unroll 1
    for (int g0 = 0; g0 < a.prefixes; g0 += 64) {
        const Lane x = lane_at(first, g0);
        const Members m = lane_members(x, before);
        const int g = g0 + (int)(threadIdx.x & 63), work = sums ? prefix_work(x, member_rows(sums, m)) : 0, upto = wave_scan(work);
        if (g < a.prefixes) {
            p.units[g] = at + upto - work;
            p.slots[g] = filled(a.shared, x.shared);
            p.ends[g] = (uint16_t)(m.first + m.count);
        }
        at += last_lane(upto);
    }
}

// The prefix of request b, the first that ends behind it; -1 for none.
__device__ __forceinline__ int prefix_of(const Prefixes& p, int b) {
    const int n = kernel_args().prefixes;
    if (!n) return -1;
    int g = 0;
    for (int step = 1 << (31 - __builtin_clz(n)); step; step >>= 1)
        if (g + step <= n && p.ends[g + step - 1] <= b) g += step;
    return g < n ? g : -1;
}

// Of this lane's request with its prefix (rows that are not merged).  A row tile without a key has one tile, of none: its
// rows are written there.
__device__ __forceinline__ int request_work(const Prefixes& p, const Lane& x, int b0) {
    Args& a = kernel_args();
    const int b = b0 + (threadIdx.x & 63), of = prefix_of(p, b);
    const int tiles = div_up(filled(a.own, x.own), kTile) + (of < 0 ? 0 : div_up(p.slots[of], kTile));
    return b < a.batch ? units(a.hkv * div_up(counted_rows(x.rows) * a.group, kRows), max(tiles, 1), kSegment) : 0;
}

// A list shared evenly: worker i takes `each` units from begin(i) on, the first `more` workers one more.
struct Share {
    int total, workers, each, more;
    __device__ __forceinline__ int begin(int i) const { return i * each + min(i, more); }
    __device__ __forceinline__ int worker(int at) const {  // the one that takes unit `at`
        const int u = min(at, total - 1), wide = more * (each + 1);
        return u < wide ? (int)((uint32_t)u / (uint32_t)(each + 1)) : more + (int)((uint32_t)(u - wide) / (uint32_t)each);
    }
};

__device__ __forceinline__ Share share_of(int total, int workers) {
    Share s;
    s.total = total;
    s.workers = max(1, min(workers, total));
    s.each = (int)((uint32_t)total / (uint32_t)s.workers);
    s.more = total - s.each * s.workers;
    return s;
}

// Both lists of merged rows.  Workgroups 0 .. n - 1 take the prefixes', those from `own_first` on the requests', their number by
// what the lists cost.
struct Plan {
    Share shared, own;  // own: waves, or workgroups
    int own_first, by_tiles;
};

// What a list's entry costs, in microseconds of a compute unit: a tile of 256 rows is bound by its products, one of up to 128 by its
// loads; a unit of one wave among eight takes 0.6.  A request's own slots go to waves or to workgroups by these costs: 16 requests of
// 126 rows and 8000 own slots, heads 28 over 4, take 173 us by waves and 71 by workgroups; of 28 rows 59 by either, of 7: 50 and 56.
constexpr float kOwnCost = 0.6f;
__device__ __forceinline__ float tiles_cost(int rows, int keys) {
    Args& a = kernel_args();
    const int left = rows % kRows;
    const float tile = 2.3f * (rows / kRows) + (left > kRows / 2 ? 2.3f : (left ? 1.5f : 0.f));
    return keys ? a.hkv * (keys * tile + 9.f * div_up(rows, kRows)) : 0.f;
}

__device__ __forceinline__ float prefix_cost(const Lane& x, int rows) { return tiles_cost(rows, div_up(filled(kernel_args().shared, x.shared), kTile)); }

__device__ __forceinline__ float wave_total(float x) {
    x += r2o_lane_xor<1>(x);
    x += r2o_lane_xor<2>(x);
    x += r2o_lane_xor<4>(x);
    x += r2o_lane_xor<8>(x);
    return r2o_sum_lane_pair<32>(r2o_sum_lane_pair<16>(x));
}

// An entry of a list: its place there, and what it is.
struct Entry {
    int base;             // tiles before it
    int prefix, request;  // request -1: all of a prefix's; -2: no entry
    int first, members;   // of the prefix: its requests
    int n_shared, n_own, rows, before;  // before: rows of the requests before the prefix's, as many as `rows` are of its own
};

// The units of the lists of merged rows.
struct Sums {
    int shared, own, own_tiles;  // own_tiles: as row tiles; 0 where waves have all rows of a request
    float shared_cost, tiles_cost;
};

__device__ __forceinline__ Sums sums_of(const Lane& first, const int* sums) {
    Args& a = kernel_args();
    Sums s{};
    int before = 0;
#pragma unroll 1
    for (int g0 = 0; g0 < a.prefixes; g0 += 64) {
        const Lane x = lane_at(first, g0);
        const int rows = member_rows(sums, lane_members(x, before));
        s.shared += last_lane(wave_scan(prefix_work(x, rows)));
        s.shared_cost += wave_total(prefix_cost(x, rows));
    }
#pragma unroll 1
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const Lane x = lane_at(first, b0);
        s.own += last_lane(wave_scan(own_work(x, b0)));
        if (a.packed > kWaveRows) {
            const int work = own_row_work(x, b0);
            s.own_tiles += last_lane(wave_scan(work));
            s.tiles_cost += wave_total(work ? tiles_cost(counted_rows(x.rows) * a.group, div_up(filled(a.own, x.own), kTile)) : 0.f);
        }
    }
    return s;
}

__device__ __forceinline__ Plan plan_of(const Sums& s) {
    Args& a = kernel_args();
    Plan p;
    const float waves = kOwnCost * s.own;
    p.by_tiles = __builtin_amdgcn_readfirstlane(s.own_tiles > 0 && s.tiles_cost < 1.25f * waves);  // waves' last ones end unevenly
    const float own = p.by_tiles ? s.tiles_cost : waves;
    int n = s.shared > 0 ? __builtin_amdgcn_readfirstlane((int)(a.workers * (s.shared_cost / (s.shared_cost + own)) + 0.5f)) : 0;
    n = max(min(n, a.workers - (s.own > 0)), (int)(s.shared > 0));
    p.own_first = min(n, a.workers - 1);  // of one workgroup, which does both
    p.shared = share_of(s.shared, n);
    p.own = p.by_tiles ? share_of(s.own_tiles, a.workers - p.own_first) : share_of(s.own, kWaves * (a.workers - p.own_first));
    return p;
}

// What the join has to know, left by one wave: it would take longer to find it out again than to read it.  The shares, then of
// each request the units before its prefix and its own slots and their tiles, the rows before its prefix's requests', theirs, its own
// that count, and those before it.
constexpr int kNote = 8;
__device__ __forceinline__ void write_notes(const Lane& first, const int* sums, const Plan& plan, Prefixes& prefixes) {
    Args& a = kernel_args();
    const int lane = threadIdx.x & 63;
    if (lane == 0) {
        int* to = a.notes;
        to[0] = plan.shared.total;
        to[1] = plan.shared.each;
        to[2] = plan.shared.more;
        to[3] = plan.own_first;
        to[4] = plan.own.total;
        to[5] = plan.own.each;
        to[6] = plan.own.more;
        to[7] = plan.by_tiles;
    }
    write_prefixes(first, sums, prefixes);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    int own = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const Lane x = lane_at(first, b0);
        const int b = b0 + lane, work = plan.by_tiles ? own_row_work(x, b0) : own_work(x, b0), upto = wave_scan(work);
        const int of = prefix_of(prefixes, b);
        if (b < a.batch) {
            int* to = a.notes + kNote * (1 + b);
            const int from = of > 0 ? prefixes.ends[of - 1] : 0;
            to[0] = of < 0 ? 0 : prefixes.units[of];
            to[1] = of < 0 ? 0 : div_up(prefixes.slots[of], kTile);
            to[2] = rows_before(sums, from) * a.group;
            to[3] = of < 0 ? 0 : member_rows(sums, {from, prefixes.ends[of] - from});
            to[4] = own + upto - work;
            to[5] = div_up(filled(a.own, x.own), plan.by_tiles ? kTile : kWaveKeys);
            to[6] = counted_rows(x.rows);
            to[7] = rows_before(sums, b) * a.group;
        }
        own += last_lane(upto);
    }
}

// Merged rows: the prefix that holds tile u of the prefixes' list.
__device__ __forceinline__ Entry find_prefix(const Lane& first, const int* sums, int u) {
    Args& a = kernel_args();
    Entry e{};
    e.request = -2;
    int at = 0, before = 0;
#pragma unroll 1
    for (int g0 = 0; g0 < a.prefixes; g0 += 64) {
        const Lane x = lane_at(first, g0);
        const Members m = lane_members(x, before);
        const int rows = member_rows(sums, m), work = prefix_work(x, rows), upto = wave_scan(work), all = last_lane(upto);
        if ((uint32_t)(u - at) < (uint32_t)all) {
            const int i = __builtin_ctzll(__ballot(at + upto > u));
            e.base = at + __builtin_amdgcn_readlane(upto - work, i);
            e.prefix = g0 + i;
            e.request = -1;
            e.first = __builtin_amdgcn_readlane(m.first, i);
            e.members = __builtin_amdgcn_readlane(m.count, i);
            e.n_shared = filled(a.shared, __builtin_amdgcn_readlane(x.shared, i));
            e.rows = __builtin_amdgcn_readlane(rows, i);
            e.before = __builtin_amdgcn_readfirstlane(rows_before(sums, e.first)) * a.group;
        }
        at += all;
    }
    return e;
}

// Merged rows: the request that holds unit u of the requests' list, of waves or of workgroups (rows: of all query heads of a KV head).
template <bool TILES>
__device__ __forceinline__ Entry find_own(const Lane& first, int u) {
    Args& a = kernel_args();
    Entry e{};
    e.request = -2;
    e.prefix = -1;
    int at = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const Lane x = lane_at(first, b0);
        const int work = TILES ? own_row_work(x, b0) : own_work(x, b0), upto = wave_scan(work), all = last_lane(upto);
        if ((uint32_t)(u - at) < (uint32_t)all) {
            const int i = __builtin_ctzll(__ballot(at + upto > u));
            e.base = at + __builtin_amdgcn_readlane(upto - work, i);
            e.request = b0 + i;
            e.n_own = filled(a.own, __builtin_amdgcn_readlane(x.own, i));
            e.rows = counted_rows(__builtin_amdgcn_readlane(x.rows, i)) * (TILES ? a.group : 1);
        }
        at += all;
    }
    return e;
}

// Rows that are not merged: the request that holds tile u (-1: none), and the tiles of all.
__device__ __forceinline__ Entry find_request(const Lane& first, const Prefixes& prefixes, int u, int& total) {
    Args& a = kernel_args();
    Entry e{};
    e.request = -2;
    e.prefix = -1;
    int at = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const Lane x = lane_at(first, b0);
        const int work = request_work(prefixes, x, b0), upto = wave_scan(work), all = last_lane(upto);
        if ((uint32_t)(u - at) < (uint32_t)all) {
            const int i = __builtin_ctzll(__ballot(at + upto > u));
            e.base = at + __builtin_amdgcn_readlane(upto - work, i);
            e.request = b0 + i;
            e.prefix = __builtin_amdgcn_readfirstlane(prefix_of(prefixes, e.request));
            e.n_shared = e.prefix < 0 ? 0 : __builtin_amdgcn_readfirstlane(prefixes.slots[e.prefix]);
            e.n_own = filled(a.own, __builtin_amdgcn_readlane(x.own, i));
            e.rows = counted_rows(__builtin_amdgcn_readlane(x.rows, i)) * a.group;
        }
        at += all;
    }
    total = at;
    return e;
}

// One row tile of an entry and head, and its key tiles: of a workgroup, `shared` ones of the prefix, then its own; of a
// wave, own ones.
struct Segment {
    int base, tiles;         // the first tile's unit, their number
    int head, row0, shared;  // row0: in the entry's rows
};

__device__ __forceinline__ Segment segment_at(const Entry& e, int u, int tiles, int more, int row_tiles, int rows) {
    Segment s{};
    s.tiles = max(1, tiles);
    const int per_head = max(1, row_tiles), at = (int)((uint32_t)(u - e.base) / (uint32_t)(s.tiles + more));
    s.head = (int)((uint32_t)at / (uint32_t)per_head);
    s.row0 = (at - s.head * per_head) * rows;
    s.base = e.base + at * (s.tiles + more) + more;
    return s;
}

__device__ __forceinline__ Segment segment_of(const Entry& e, int u) {
    const int shared = div_up(e.n_shared, kTile);
    Segment s = segment_at(e, u, shared + div_up(e.n_own, kTile), kSegment, div_up(e.rows, kRows), kRows);
    s.shared = shared;
    return s;
}

// Where partial states lie: two tiles of rows for each workgroup, or for each of its waves, for the segments that it does not
// have alone (the one that another began, and the one that it leaves to others), then, where rows are merged, a place for
// each row of the prefixes' segments and of the requests'.
__device__ __forceinline__ uint32_t split_rows(int worker, bool begins) { return (2u * worker + begins) * kRows; }
__device__ __forceinline__ uint32_t split_wave_rows(int own_first, int wave, bool begins) {  // wave: of all that take requests
    return 2u * kRows * own_first + (2u * wave + begins) * kWaveRows;
}
__device__ __forceinline__ uint32_t whole_prefix_rows(Args& a, int before, int rows, int head) {
    return 2u * kRows * a.workers + (uint32_t)before * a.hkv + (uint32_t)head * rows;
}
__device__ __forceinline__ uint32_t whole_own_rows(Args& a, int b, int head) {
    return 2u * kRows * a.workers + ((uint32_t)(a.batch + b) * a.hkv + head) * a.packed;
}
constexpr uint32_t kNoRow = 0xffffffffu, kResult = 0xfffffffeu;  // no row, and one whose result is written at once

// ------------------------------------------------------------------------------------- the rows
// A cache's rows of one table and head.
struct Side {
    const uint16_t *k, *v;
    const int32_t* table;
    int k_page, k_slot, v_page, v_slot, shift, last_page, pages, n;
};

__device__ __forceinline__ Side side_of(SourceArgs& s, int row, int head, int n) {
    Side x;
    x.k = s.key + (int64_t)head * s.k_head;
    x.v = s.value + (int64_t)head * s.v_head;
    x.table = s.table + (int64_t)row * s.table_stride;
    x.k_page = s.k_page;
    x.k_slot = s.k_slot;
    x.v_page = s.v_page;
    x.v_slot = s.v_slot;
    x.shift = s.shift;
    x.last_page = s.last_page;
    x.pages = s.pages;
    x.n = n;
    return x;
}

// The page of slot j, -1 if it has none or is not filled.
__device__ __forceinline__ int page_of(const Side& x, int j) {
    const int id = load_uniform(x.table + min(j >> x.shift, x.last_page));
    return j < x.n && (uint32_t)id < (uint32_t)x.pages ? id : -1;
}

// 64 neighbouring pages of a table, one a lane, -1 for one outside the pool, and a bit for each inside it.  Scalar loads of a
// tile's pages, one after the other, took longer than the tile.
struct Window {
    int first, ids;
    uint64_t ok;
};

__device__ __forceinline__ Window window_of(SourceArgs& s, const int32_t* table, int first, int lane) {
    const int id = r2o_ldg(table + min(first + lane, s.last_page));
    const bool ok = (uint32_t)id < (uint32_t)s.pages;
    return {first, ok ? id : -1, __ballot(ok)};
}

// Which of the four groups of 16 slots from j0 (a multiple of 64) on, each within a page, have a page and a filled slot.
__device__ __forceinline__ int groups_of(const Window& w, int j0, int shift, int n) {
    const int bits = (int)(w.ok >> ((j0 >> shift) - w.first));
    const int in_pages = shift == 4 ? bits & 15 : (shift == 5 ? (bits & 1) * 3 | (bits >> 1 & 1) * 12 : (bits & 1) * 15);
    return n - j0 >= kTile ? in_pages : in_pages & (1 << (max(n - j0, 0) + 15) / 16) - 1;
}

// Four rows (of 16 from `base` on, the i-th four of them) straight into LDS.
template <int SWZ>
__device__ __forceinline__ void stage_four(const uint16_t* base, int stride, int i, unsigned char* lds, int lane) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)row_chunk<SWZ>(base, stride, 4 * i, 15, i, lane),
                                     (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// Waits for this wave's loads but the last N.
template <int N>
__device__ __forceinline__ void wait_all_but() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 << 14) | 0xF70);
    asm volatile("" ::: "memory");
}

// 16 keys from 16 kb on, transposed, as the A operands of channels 32 db ..: lane half h holds keys 4 h + 0..3 and 8 + 4 h
// + 0..3, the order in which the products' C registers hold the probabilities.  In assembly, with its wait, as K's.
__device__ __forceinline__ void read_value_rows(const unsigned char* tile, int kb, int lane, r2o_u4 (&v)[4]) {
    const int i = lane & 15, r = i >> 2;
    const uint32_t a = lds_address(tile) + (16 * kb + 4 * (lane >> 5) + r) * 256 + 64 * r + 16 * (2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) + 8 * (i & 1);
    r2o_u2 lo[4], hi[4];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9\n\tds_read_b64_tr_b16 %2, %10\n\tds_read_b64_tr_b16 %3, %11\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:2048\n\tds_read_b64_tr_b16 %5, %9 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %10 offset:2048\n\tds_read_b64_tr_b16 %7, %11 offset:2048\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
        : "v"(a), "v"(a ^ 64), "v"(a ^ 128), "v"(a ^ 192)
        : "memory");
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = r2o_u4{lo[x][0], lo[x][1], hi[x][0], hi[x][1]};
}

// A wave's 32 rows: their query rows, and the state of their softmax and products.
struct Rows {
    r2o_u4 q[8];
    f16v acc[4];
    float m, l;
};

__device__ __forceinline__ void start_rows(Rows& w, const uint16_t* src) {
#pragma unroll
    for (int t = 0; t < 8; ++t) w.q[t] = r2o_ldg(reinterpret_cast<const r2o_u4*>(src + 16 * t));
#pragma unroll
    for (int i = 0; i < 4; ++i) w.acc[i] = f16v{};
    w.m = -INFINITY;
    w.l = 0.f;
}

// The query rows, which went out before any tile: waited for here, so that nothing but tiles is counted from here on.
__device__ __forceinline__ void wait_rows(Rows& w) {
#pragma unroll
    for (int t = 0; t < 8; ++t) asm volatile("" : "+v"(w.q[t]));
}

// S^T of 32 keys x 32 rows
template <int RF>
__device__ __forceinline__ f16v products(const Rows& w, const unsigned char* kl, int sub, int lane) {
    f16v x = f16v{};
    r2o_u4 k[8];
    read_all_rows(kl, sub, lane, k);
#pragma unroll
    for (int t = 0; t < 8; ++t) x = mfma32<RF>(k[t], w.q[t], x);
    return x;
}

// The larger of two numbers, by the median of them and infinity: fmaxf makes each operand quiet first, one more instruction for
// each product.  Of NaN and a number the number; of two NaN, in a row that is NaN anyhow, infinity.
__device__ __forceinline__ float larger(float x, float y) { return __builtin_amdgcn_fmed3f(x, y, INFINITY); }

// Masks of 32 keys from `from` on, of which `groups` (a bit for 16) have a page and which a row sees up to `seen`; and the running
// maximum raised where it has to be.
__device__ __forceinline__ void top_of(Rows& w, f16v& x, int from, int seen, int groups, int lane, float c2) {
    if (groups != 3 || __any(from + 31 > seen)) {
        const int back = seen - from - 4 * (lane >> 5), back0 = groups & 1 ? back : -1, back1 = groups & 2 ? back : -1;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = (i < 8 ? back0 : back1) >= 8 * (i >> 2) + (i & 3) ? x[i] : -INFINITY;
    }
    float tmax = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) tmax = larger(tmax, x[i]);
    float y, z;
    r2o_row_swap<32>(tmax, y, z);
    tmax = larger(y, z) * c2;  // -inf stays (c2 > 0)
    if (__any(tmax > w.m + kSlack)) {
        // of the rows that exceed it alone: a row's result does not depend on its neighbours
        const float m_new = tmax > w.m + kSlack ? tmax : w.m;
        const float alpha = m_new == w.m ? 1.f : __builtin_amdgcn_exp2f(w.m - m_new);
        w.l *= alpha;
#pragma unroll
        for (int db = 0; db < 4; ++db) w.acc[db] *= alpha;
        w.m = m_new;
    }
}

template <int RF>
__device__ __forceinline__ void probabilities(Rows& w, const f16v& x, r2o_u4 (&pk)[2], float c2) {
    const float mm = w.m == -INFINITY ? 0.f : w.m;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c2, -mm));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i + 1], c2, -mm));
        w.l += e0 + e1;
        pk[i >> 3][(i & 7) >> 1] = pack2<RF>(e0, e1);
    }
}

template <int RF>
__device__ __forceinline__ void values(Rows& w, const unsigned char* vl, int sub, const r2o_u4 (&pk)[2], int lane) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        r2o_u4 v[4];
        read_value_rows(vl, 2 * sub + kb, lane, v);
#pragma unroll
        for (int db = 0; db < 4; ++db) w.acc[db] = mfma32<RF>(v[db], pk[kb], w.acc[db]);
    }
}

// Whether a channel's sum is infinite or NaN in a row of this wave that counts; a NaN sum of the softmax, of a NaN logit,
// makes the whole row NaN anyhow.
__device__ __forceinline__ bool met_not_finite(const Rows& w, bool counts) {
    float odd[4] = {};
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int db = 0; db < 4; ++db) odd[db] = __builtin_fmaf(w.acc[db][i], 0.f, odd[db]);  // NaN where one is not finite
    const float any = odd[0] + odd[1] + odd[2] + odd[3];
    return __any(any != any && w.l == w.l && counts);
}

// All bits for a finite number, none for an infinite one or NaN: by arithmetic, for 64 conditions at a time do not fit.
__device__ __forceinline__ uint32_t finite_mask(uint32_t bits) { return (uint32_t)((int)((bits & 0x7f800000u) - 0x7f800000u) >> 31); }

// A row's channel is infinite or NaN where a key that it sees is, however small that key's weight: not NaN where the weight is
// rounded to 0 on its way to the product.  Those channels are formed again from the values alone, 32 channels (block db) at a
// time: slots j0 .. j1 - 1 of a side added here, till every row has NaN alone.
template <int RF>
__device__ __forceinline__ void add_not_finite(f16v& extra, int db, const Side& x, int j0, int j1, int seen, bool counts, int lane) {
    bool more = true;
#pragma unroll 1
    for (int j16 = j0; j16 < j1 && more; j16 += 16) {
        const int page = page_of(x, j16);
        if (page < 0) continue;
        const uint16_t* rows = x.v + (int64_t)page * x.v_page + (int64_t)(j16 & ((1 << x.shift) - 1)) * x.v_slot;
        r2o_u4 chunk[4];  // of four rows each
#pragma unroll
        for (int n = 0; n < 4; ++n)
            chunk[n] = r2o_ldg(reinterpret_cast<const r2o_u4*>(rows + (int64_t)(4 * n + (lane >> 4)) * x.v_slot) + (lane & 15));
        if (!__any(zero_not_finite<RF>(chunk))) continue;
        for (int j = 0; j < min(16, x.n - j16); ++j) {
            if (j16 + j > seen) continue;
            const uint16_t* value = rows + (int64_t)j * x.v_slot + 32 * db + 4 * (lane >> 5);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const r2o_u2 y = r2o_ldg(reinterpret_cast<const r2o_u2*>(value + 8 * g));
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t bits = y[k >> 1] >> 16 * (k & 1) & 0xffffu, z = __float_as_uint(RF == 0 ? r2o_bf16_to_f32(bits) : r2o_f16_to_f32(bits));
                    extra[4 * g + k] += __uint_as_float(z & ~finite_mask(z));
                }
            }
        }
        float number = extra[0];  // the largest that is no NaN, or NaN
#pragma unroll
        for (int i = 0; i < 16; ++i) number = fmaxf(number, extra[i]);
        more = !__all(number != number || !counts);
    }
}

__device__ __forceinline__ void take_not_finite(f16v& acc, const f16v& extra) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t x = __float_as_uint(extra[i]), keep = finite_mask(x);
        acc[i] = __uint_as_float((__float_as_uint(acc[i]) & keep) | (x & ~keep));
    }
}

__device__ __forceinline__ void store_state(Args& a, const Rows& w, uint32_t to, bool counts, int lane) {
    if (to == kNoRow) return;
    const int half = lane >> 5;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<R2O_GLOBAL r2o_f4*>((R2O_GLOBAL float*)(a.partial_out + (int64_t)to * 128 + 32 * db + 8 * g + 4 * half)) =
                r2o_f4{w.acc[db][4 * g], w.acc[db][4 * g + 1], w.acc[db][4 * g + 2], w.acc[db][4 * g + 3]};
    if (half == 0) {
        a.partial_ml[2 * (int64_t)to] = counts ? w.m : -INFINITY;
        a.partial_ml[2 * (int64_t)to + 1] = counts ? w.l : 0.f;
    }
}

constexpr unsigned kKeyTiles = kAhead, kValueTiles = kAhead + 1;
typedef unsigned char Lds[kKeyTiles + kValueTiles][kTileBytes];

__device__ __forceinline__ void lds_barrier() {  // of LDS alone: stores to memory are not waited for
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A workgroup's part of a list of row tiles, its own slots behind a prefix's where rows are not merged.  S^T = K Q^T (32 keys x 32
// rows a product), O^T += V^T P^T; three tiles ahead go into LDS while one is computed on.  A tile is two halves of 32 keys: the
// products of the half that follows run beside the exponentials of the one before it.
template <int RF, List LIST>
__device__ __forceinline__ void work_on_row_tiles(Lds& lds, int* flags, const int* sums, const Prefixes& prefixes, const Lane& first, int u, int u_end) {
    while (u < u_end) {
        Args& a = kernel_args();
        int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), worker = blockIdx.x;
        asm("" : "+v"(lane), "+s"(wave), "+s"(worker));  // or what depends on them alone would be held from one segment to the next
        int total;
        const Entry e = LIST == kPrefixes ? find_prefix(first, sums, u) : LIST == kOwn ? find_own<true>(first, u) : find_request(first, prefixes, u, total);
        if (e.request == -2) return;  // lengths that change meanwhile
        const Segment s = segment_of(e, u);
        const int begin = max(0, u - s.base), stop = min(s.tiles, u_end - s.base);
        if (stop <= begin || s.head >= a.hkv) return;  // nothing but a start that is the next one's, or lengths that change meanwhile

        // this lane's row, and the last key of its own that it sees
        const int two = opaque(e.rows - s.row0 <= kRows / 2);  // waves share the keys of 32 rows, a half of each tile each
        const int part = two ? wave >> 2 : 0, in_tile = 32 * (two ? wave & 3 : wave) + (lane & 31);
        const int at = min(s.row0 + in_tile, e.rows - 1), group = a.group;
        int row = at / group, b = e.request;
        const int head = s.head * group + at - row * group;
        if constexpr (LIST == kPrefixes) {  // the request that row `row` of the prefix's is of, and which of its rows that is
            if (a.query_lengths) {
                row += e.before / group;
                b = e.first;
                for (int step = 512; step; step >>= 1)
                    if (b + step < e.first + e.members && sums[b + step] <= row) b += step;
                row -= sums[b];
            } else {
                b = e.first + row / a.rows;
                row -= (b - e.first) * a.rows;
            }
        }
        const int busy = opaque(s.row0 + in_tile - (lane & 31) < e.rows);  // this wave
        uint32_t to = kNoRow;
        if (s.row0 + in_tile < e.rows && part == 0) {
            if (begin > 0 || stop < s.tiles) to = split_rows(worker, begin == 0) + in_tile;
            else if (LIST == kPrefixes) to = whole_prefix_rows(a, e.before, e.rows, s.head) + s.row0 + in_tile;
            else if (LIST == kOwn) to = whole_own_rows(a, e.request, s.head) + s.row0 + in_tile;
            else to = kResult;
        }
        Rows w;
        start_rows(w, a.query + (int64_t)b * a.q_batch + (int64_t)head * a.q_head + (int64_t)row * a.q_row + 8 * (lane >> 5));
        int counted = a.rows;
        if (LIST != kPrefixes && a.query_lengths) counted = counted_rows(r2o_ldg(a.query_lengths + b));
        const int see_own = min(e.n_own - counted + row, e.n_own - 1);
        // the least and the most that a row of the workgroup sees of them; no row of a prefix's segment has any
        const int base_row = e.n_own - __builtin_amdgcn_readfirstlane(counted);
        const int least = LIST == kPrefixes ? 0 : min(base_row + s.row0 / group, e.n_own - 1);
        const int most = LIST == kPrefixes ? -1 : min(base_row + min(s.row0 + kRows - 1, e.rows - 1) / group, e.n_own - 1);
        const int last = min(stop, s.shared + (most >= 0 ? most / kTile + 1 : 0));  // tiles behind it are seen by no row
        const float c2 = a.c2;
        bool bad = false;

        auto of_prefix = [&](int it) { return LIST == kPrefixes || (LIST == kRequests && it < s.shared); };
        auto side_at = [&](int it) {
            Args& x = kernel_args();
            return of_prefix(it) ? side_of(x.shared, e.prefix, s.head, e.n_shared) : side_of(x.own, e.request, s.head, e.n_own);
        };
        auto slot_of = [&](int it) { return (LIST != kRequests || it < s.shared ? it : it - s.shared) * kTile; };
        auto last_seen = [&](int it) { return of_prefix(it) ? e.n_shared - 1 : see_own; };
        // The side and the pages of the next tile to be staged, and its buffers.
        Side side = side_at(begin);
        auto window_at = [&](int it) {
            Args& x = kernel_args();
            return window_of(of_prefix(it) ? x.shared : x.own, side.table, slot_of(it) >> side.shift, lane);
        };
        Window window = window_at(begin);
        unsigned v_at = kKeyTiles;
        asm("" : "+s"(v_at));  // or every wave's place in each would be held in a register
        auto keys_of = [&](int it) { return lds[(it - begin) % kKeyTiles]; };
        // Waves 0 to 3 bring tiles begin, begin + 2, .., waves 4 to 7 the others, 16 rows of K and V a wave: half of the addresses,
        // and the two waves of a SIMD come out of step, one's products beside the other's exponentials.  Returned for every wave:
        // which of the tile's four groups of 16 slots count.
        auto stage = [&](int it) {
            const int j0 = slot_of(it);
            if (LIST == kRequests && it == s.shared && it > begin) {
                side = side_at(it);
                window = window_at(it);
            } else if ((j0 >> side.shift) - window.first > 63) {
                window = window_at(it);
            }
            if (((it - begin) & 1) == wave >> 2) {
                const int j1 = j0 + 16 * (wave & 3), j = j1 & ((1 << side.shift) - 1);
                const int id = max(__builtin_amdgcn_readlane(window.ids, (j1 >> side.shift) - window.first), 0);
                const uint16_t* k = side.k + (int64_t)id * side.k_page + (int64_t)j * side.k_slot;
                const uint16_t* v = side.v + (int64_t)id * side.v_page + (int64_t)j * side.v_slot;
#pragma unroll
                for (int i = 0; i < 4; ++i) stage_four<0>(k, side.k_slot, i, keys_of(it) + (16 * (wave & 3) + 4 * i) * 256, lane);
#pragma unroll
                for (int i = 0; i < 4; ++i) stage_four<1>(v, side.v_slot, i, lds[v_at] + (16 * (wave & 3) + 4 * i) * 256, lane);
            }
            v_at = v_at == kKeyTiles + kValueTiles - 1 ? kKeyTiles : v_at + 1;
            return groups_of(window, j0, side.shift, side.n);
        };
        // This wave's eight value rows of a staged tile.  Rows that no row of the workgroup sees may hold anything: zero.  Where some
        // see a row that others do not, 0 times an infinite or NaN value would be NaN: those become zero before any product.
        auto clean = [&](int it, int v_buffer, int valid) {
            const int n = of_prefix(it) ? e.n_shared : e.n_own, j0 = slot_of(it);
            const bool some = !of_prefix(it) && j0 + kTile - 1 > least && least < n - 1;
            if (valid == 15 && j0 + kTile <= n && !some) return;  // the same for all waves
            r2o_u4* at_lds = reinterpret_cast<r2o_u4*>(lds[v_buffer] + 8 * wave * 256) + lane;
            r2o_u4 x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x[i] = at_lds[64 * i];
                if (!(valid >> (wave >> 1) & 1) || j0 + 8 * wave + 4 * i + (lane >> 4) >= n) x[i] = r2o_u4{};
            }
            bad |= some && zero_not_finite<RF>(x);
#pragma unroll
            for (int i = 0; i < 2; ++i) at_lds[64 * i] = x[i];
            lds_barrier();
        };
        // Tile `it`, behind which `behind` more are on their way (at most three), is there for every wave.  Behind the barrier no wave
        // reads the keys of the tile before it, nor the values of the one before that.
        auto arrive = [&](int it, int behind) {
            if (((it - begin) & 1) == wave >> 2) {  // this wave's: but for the tile after next
                if (behind >= 2) wait_all_but<8>();
                else wait_all_but<0>();
            }
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        int valid = 0;  // four bits a tile, from the current one on
        wait_rows(w);
        if (begin < last) {
            int staged = begin;
#pragma unroll 1
            for (int i = 0; i < 4 * kAhead && staged < last; i += 4) {
                valid |= stage(staged) << i;
                ++staged;
            }
            arrive(begin, staged - begin - 1);
            unsigned v_now = kKeyTiles;
            clean(begin, v_now, valid & 15);
            // From tile `it` to the next one: v_last is left for the values that are still to be read.
            unsigned v_last = 0;
            auto next = [&](int it) __attribute__((always_inline)) {
                v_last = v_now;
                v_now = v_now == kKeyTiles + kValueTiles - 1 ? kKeyTiles : v_now + 1;
                if (it + 1 < last) {
                    arrive(it + 1, staged - it - 2);
                    if (staged < last) {
                        valid |= stage(staged) << 4 * kAhead;
                        ++staged;
                    }
                    clean(it + 1, v_now, valid >> 4 & 15);
                }
                valid >>= 4;
            };
            // Behind the last tile the products are of what lies there, and not used.
            if (!busy) {  // brings its rows of the tiles alone
                for (int it = begin; it < last; ++it) next(it);
            } else if (two) {
                f16v now = products<RF>(w, lds[0], part, lane);
                for (int it = begin; it < last; ++it) {
                    r2o_u4 pk[2];
                    top_of(w, now, slot_of(it) + 32 * part, last_seen(it), valid >> 2 * part & 3, lane, c2);
                    probabilities<RF>(w, now, pk, c2);
                    next(it);
                    now = products<RF>(w, keys_of(it + 1), part, lane);
                    values<RF>(w, lds[v_last], part, pk, lane);
                }
            } else {
                f16v even = products<RF>(w, lds[0], 0, lane);
                for (int it = begin; it < last; ++it) {
                    r2o_u4 pk[2];
                    top_of(w, even, slot_of(it), last_seen(it), valid & 3, lane, c2);
                    f16v odd = products<RF>(w, keys_of(it), 1, lane);
                    probabilities<RF>(w, even, pk, c2);
                    values<RF>(w, lds[v_now], 0, pk, lane);
                    top_of(w, odd, slot_of(it) + 32, last_seen(it), valid >> 2 & 3, lane, c2);
                    next(it);
                    even = products<RF>(w, keys_of(it + 1), 0, lane);
                    probabilities<RF>(w, odd, pk, c2);
                    values<RF>(w, lds[v_last], 1, pk, lane);
                }
            }
        }
        {
            float x, y;
            r2o_row_swap<32>(w.l, x, y);
            w.l = x + y;
        }
        const bool wave_bad = __any(bad);
        if (lane == 0) flags[wave] = wave_bad;
        lds_barrier();  // no wave reads a tile any more
        if (two && part) {
            r2o_f4* to_lds = reinterpret_cast<r2o_f4*>(lds[wave & 3]) + lane;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                to_lds[64 * i] = r2o_f4{w.acc[i >> 2][4 * (i & 3)], w.acc[i >> 2][4 * (i & 3) + 1], w.acc[i >> 2][4 * (i & 3) + 2], w.acc[i >> 2][4 * (i & 3) + 3]};
            float* ml = reinterpret_cast<float*>(lds[4]) + 128 * (wave & 3) + lane;
            ml[0] = w.m;
            ml[64] = w.l;
        }
        lds_barrier();
        if (two && !part) {
            const float* ml = reinterpret_cast<const float*>(lds[4]) + 128 * wave + lane;
            const float m2 = ml[0], l2 = ml[64], mn = fmaxf(w.m, m2), ms = mn == -INFINITY ? 0.f : mn;
            const float f = __builtin_amdgcn_exp2f(w.m - ms), f2 = __builtin_amdgcn_exp2f(m2 - ms);
            const r2o_f4* from_lds = reinterpret_cast<const r2o_f4*>(lds[wave]) + lane;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const r2o_f4 o = from_lds[64 * i];
#pragma unroll
                for (int k = 0; k < 4; ++k) w.acc[i >> 2][4 * (i & 3) + k] = w.acc[i >> 2][4 * (i & 3) + k] * f + o[k] * f2;
            }
            w.l = w.l * f + l2 * f2;
            w.m = mn;
        }
        int any_bad = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) any_bad |= flags[i];
        const bool counts = row < counted;
        if (busy && part == 0 && (any_bad || met_not_finite(w, counts))) {
#pragma unroll
            for (int db = 0; db < 4; ++db) {
                f16v extra = f16v{};
#pragma unroll 1
                for (int from = begin, to_tile; from < last; from = to_tile) {  // the prefix's, then its own
                    to_tile = LIST != kRequests || from >= s.shared ? last : min(last, s.shared);
                    add_not_finite<RF>(extra, db, side_at(from), slot_of(from), slot_of(from) + (to_tile - from) * kTile, last_seen(from), counts, lane);
                }
                take_not_finite(w.acc[db], extra);
            }
        }
        if (LIST == kRequests && to == kResult) {
            Args& x = kernel_args();
            const bool live = counts && !(w.l == 0.f);  // no key seen; NaN logits leave m, and a NaN sum
            const float inv = live ? 1.f / w.l : 0.f;
            uint16_t* dst = x.out + (int64_t)b * x.o_batch + (int64_t)head * x.o_head + (int64_t)row * x.o_row;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    r2o_u2 y;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        y[k] = live ? pack2<RF>(w.acc[db][4 * g + 2 * k] * inv, w.acc[db][4 * g + 2 * k + 1] * inv) : 0u;
                    *reinterpret_cast<R2O_GLOBAL r2o_u2*>((R2O_GLOBAL uint16_t*)(dst + 32 * db + 8 * g + 4 * (lane >> 5))) = y;
                }
            if (lane < 32) x.lse[((int64_t)b * x.hq + head) * x.rows + row] = live ? (w.m + __builtin_amdgcn_logf(w.l)) * kLn2 : -INFINITY;
        } else {
            store_state(kernel_args(), w, to, counts, lane);
        }
        u = s.base + stop;
        lds_barrier();  // flags and states lie where the next segment's go
    }
}

// A wave's part of the requests' own slots (merged rows), in tiles of 32 rows and 32 keys, without a barrier: the next tile's
// keys go out when this one's products have read theirs, its values when these have been.
template <int RF>
__device__ __forceinline__ void work_on_own(Lds& lds, const Lane& first, int own_first, int index, int u, int u_end) {
    while (u < u_end) {
        Args& a = kernel_args();
        int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        asm("" : "+v"(lane), "+s"(wave));
        const Entry e = find_own<false>(first, u);
        if (e.request == -2) return;  // lengths that change meanwhile
        const Segment s = segment_at(e, u, div_up(e.n_own, kWaveKeys), kWaveSegment, div_up(e.rows * a.group, kWaveRows), kWaveRows);
        const int begin = max(0, u - s.base), stop = min(s.tiles, u_end - s.base);
        if (stop <= begin || s.head >= a.hkv) return;
        const int end = e.rows * a.group, p = min(s.row0 + (lane & 31), end - 1), row = p / a.group, head = s.head * a.group + p - row * a.group;
        uint32_t to = kNoRow;
        if (s.row0 + (lane & 31) < end)
            to = (begin > 0 || stop < s.tiles ? split_wave_rows(own_first, index, begin == 0) : whole_own_rows(a, e.request, s.head) + s.row0) + (lane & 31);
        Rows w;
        start_rows(w, a.query + (int64_t)e.request * a.q_batch + (int64_t)head * a.q_head + (int64_t)row * a.q_row + 8 * (lane >> 5));
        const int off = e.n_own - e.rows, seen = min(off + row, e.n_own - 1);
        const int least = min(off + s.row0 / a.group, e.n_own - 1), most = min(off + min(s.row0 + kWaveRows - 1, end - 1) / a.group, e.n_own - 1);
        const int last = min(stop, most >= 0 ? most / kWaveKeys + 1 : 0);  // tiles behind it are seen by no row
        const float c2 = a.c2;
        const Side side = side_of(a.own, e.request, s.head, e.n_own);
        Window window = window_of(a.own, side.table, begin * kWaveKeys >> side.shift, lane);
        unsigned char *const kl = lds[wave], *const vl = kl + kTileBytes / 2;
        bool bad = false;
        // The page of a tile's group of 16 slots, -1 for none; windows are as wide as whole tiles.
        auto page_at = [&](int j) {
            if ((j >> side.shift) - window.first > 63) window = window_of(kernel_args().own, side.table, j >> side.shift, lane);
            const int id = __builtin_amdgcn_readlane(window.ids, (j >> side.shift) - window.first);
            return j < side.n ? id : -1;
        };
        auto stage = [&](const uint16_t* base, int page_stride, int slot_stride, int id, int j, auto swizzle, unsigned char* to_lds) {
            const uint16_t* rows = base + (int64_t)max(id, 0) * page_stride + (int64_t)(j & ((1 << side.shift) - 1)) * slot_stride;
#pragma unroll
            for (int i = 0; i < 4; ++i) stage_four<decltype(swizzle)::value>(rows, slot_stride, i, to_lds + 4 * i * 256, lane);
        };
        auto stage_keys = [&](int j, int id0, int id1) {
            stage(side.k, side.k_page, side.k_slot, id0, j, std::integral_constant<int, 0>(), kl);
            stage(side.k, side.k_page, side.k_slot, id1, j + 16, std::integral_constant<int, 0>(), kl + 4096);
        };
        auto stage_values = [&](int j, int id0, int id1) {
            stage(side.v, side.v_page, side.v_slot, id0, j, std::integral_constant<int, 1>(), vl);
            stage(side.v, side.v_page, side.v_slot, id1, j + 16, std::integral_constant<int, 1>(), vl + 4096);
        };
        wait_rows(w);
        if (begin < last) {
            int id0 = page_at(begin * kWaveKeys), id1 = page_at(begin * kWaveKeys + 16);
            stage_keys(begin * kWaveKeys, id0, id1);
            stage_values(begin * kWaveKeys, id0, id1);
            for (int it = begin; it < last; ++it) {
                const int j0 = it * kWaveKeys;
                const bool more = it + 1 < last;
                int next0 = -1, next1 = -1;
                if (more) {
                    next0 = page_at(j0 + kWaveKeys);
                    next1 = page_at(j0 + kWaveKeys + 16);
                }
                wait_all_but<8>();
                f16v x = products<RF>(w, kl, 0, lane);
                if (more) stage_keys(j0 + kWaveKeys, next0, next1);
                top_of(w, x, j0, seen, (id0 >= 0) | (id1 >= 0) << 1, lane, c2);
                r2o_u4 pk[2];
                probabilities<RF>(w, x, pk, c2);
                if (more) wait_all_but<8>();
                else wait_all_but<0>();
                // rows that no row of the wave sees, or some do and others do not, as a workgroup has it
                const bool some = j0 + kWaveKeys - 1 > least && least < side.n - 1;
                if (some || id0 < 0 || id1 < 0 || j0 + kWaveKeys > side.n) {
                    r2o_u4* at_lds = reinterpret_cast<r2o_u4*>(vl) + lane;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        r2o_u4 y[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            y[i] = at_lds[256 * g + 64 * i];
                            if ((g ? id1 : id0) < 0 || j0 + 16 * g + 4 * i + (lane >> 4) >= side.n) y[i] = r2o_u4{};
                        }
                        bad |= some && zero_not_finite<RF>(y);
#pragma unroll
                        for (int i = 0; i < 4; ++i) at_lds[256 * g + 64 * i] = y[i];
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                }
                values<RF>(w, vl, 0, pk, lane);
                if (more) stage_values(j0 + kWaveKeys, next0, next1);
                id0 = next0;
                id1 = next1;
            }
        }
        {
            float x, y;
            r2o_row_swap<32>(w.l, x, y);
            w.l = x + y;
        }
        const bool counts = row < e.rows;
        if (__any(bad) || met_not_finite(w, counts)) {
            const Side x = side_of(kernel_args().own, e.request, s.head, e.n_own);
#pragma unroll
            for (int db = 0; db < 4; ++db) {
                f16v extra = f16v{};
                add_not_finite<RF>(extra, db, x, begin * kWaveKeys, last * kWaveKeys, seen, counts, lane);
                take_not_finite(w.acc[db], extra);
            }
        }
        store_state(kernel_args(), w, to, counts, lane);
        u = s.base + stop;
    }
}

// The probabilities are rounded to the rows' 16 bits for the product with V, whose two operands are of one type; their sum
// takes them unrounded.  Results differ from those of 32-bit probabilities by 1.5e-4 to 3.6e-4 of their size in bf16 and 4e-5 in fp16,
// where both are 1.6e-3 and 2.1e-4 off 64 bits by their own rounding.
template <int RF, bool MERGED>
__global__ __launch_bounds__(64 * kWaves, 2) void prefix_partial_kernel(PrefixArgs) {
    __shared__ __align__(1024) Lds lds;
    __shared__ int flags[kWaves], sums_lds[R2O_PAGED_MAX_BATCH + 1];
    __shared__ Prefixes prefixes;
    Args& a = kernel_args();
    const Lane first = lane_of(0);
    int u = 0, u_end = 0;
    if constexpr (MERGED) {
        int own_first, by_tiles, index, v = 0, v_end = 0;
        if (a.query_lengths) {
            if (threadIdx.x < 64) {
                int before = 0;
#pragma unroll 1
                for (int b0 = 0; b0 <= a.batch; b0 += 64) {
                    const int b = b0 + (int)threadIdx.x, rows = b < a.batch ? counted_rows(lane_at(first, b0).rows) : 0, upto = wave_scan(rows);
                    if (b <= a.batch) sums_lds[b] = before + upto - rows;
                    before += last_lane(upto);
                }
            }
            __syncthreads();
        }
        {
            const Sums sums = sums_of(first, sums_lds);
            const Plan plan = plan_of(sums);
            if (sums.shared > 0 && (int)blockIdx.x < plan.shared.workers) {
                u = plan.shared.begin(blockIdx.x);
                u_end = plan.shared.begin(blockIdx.x + 1);
            }
            own_first = plan.own_first;
            if (blockIdx.x == gridDim.x - 1 && threadIdx.x >= 64 * (kWaves - 1)) write_notes(first, sums_lds, plan, prefixes);
            by_tiles = plan.by_tiles;
            index = (int)blockIdx.x - own_first;
            if (!by_tiles) index = kWaves * index + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
            if (sums.own > 0 && index >= 0 && index < plan.own.workers) {
                v = plan.own.begin(index);
                v_end = plan.own.begin(index + 1);
            }
        }
        work_on_row_tiles<RF, kPrefixes>(lds, flags, sums_lds, prefixes, first, u, u_end);
        if (by_tiles) work_on_row_tiles<RF, kOwn>(lds, flags, sums_lds, prefixes, first, v, v_end);
        else work_on_own<RF>(lds, first, own_first, index, v, v_end);
    } else {
        if (a.prefixes) {
            if (threadIdx.x < 64) write_prefixes(first, nullptr, prefixes);
            __syncthreads();
        }
        int total;
        find_request(first, prefixes, -1, total);
        const Share share = share_of(total, a.workers);
        int request = -1, place[4] = {};
        if (total > 0 && (int)blockIdx.x < share.workers) {
            u = share.begin(blockIdx.x);
            u_end = share.begin(blockIdx.x + 1);
            const Entry e = find_request(first, prefixes, u, total);
            const Segment s = segment_of(e, u);
            // the segment that this workgroup is the second to work on is joined by the note's reader
            if (e.request >= 0 && s.base < u && s.base >= share.begin((int)blockIdx.x - 1)) {
                request = e.request;
                place[0] = s.head;
                place[1] = s.row0;
                place[2] = e.rows;
                place[3] = share.worker(s.base + s.tiles - 1) - (int)blockIdx.x + 2;
            }
        }
        if (threadIdx.x == 0) {
            int* to = a.notes + kNote * (int)blockIdx.x;
            to[0] = request;
#pragma unroll
            for (int i = 0; i < 4; ++i) to[1 + i] = place[i];
        }
        work_on_row_tiles<RF, kRequests>(lds, flags, sums_lds, prefixes, first, u, u_end);
    }
}

// ---------------------------------------------------------------------------------------- joining
struct State {
    float m, l;
    r2o_f4 o;  // four channels
};

__device__ __forceinline__ void join_state(State& s, float m2, float l2, const r2o_f4& o2) {
    const float mn = fmaxf(s.m, m2), ms = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(s.m - ms), f2 = __builtin_amdgcn_exp2f(m2 - ms);
    s.l = s.l * f + l2 * f2;
#pragma unroll
    for (int k = 0; k < 4; ++k) s.o[k] = weighed(s.o[k], f) + weighed(o2[k], f2);
    s.m = mn;
}

__device__ __forceinline__ void join_partial(Args& a, State& s, uint32_t row, int d4) {
    const int64_t at = row;
    const float m2 = r2o_ldg(a.partial_ml + 2 * at), l2 = r2o_ldg(a.partial_ml + 2 * at + 1);
    join_state(s, m2, l2, r2o_ldg(reinterpret_cast<const r2o_f4*>(a.partial_out + at * 128) + d4));
}

template <int RF>
__device__ __forceinline__ void write_row(Args& a, const State& s, int b, int head, int row, int d4) {
    const bool live = !(s.l == 0.f);
    const float inv = live ? 1.f / s.l : 0.f;
    r2o_u2 w{};
    if (live) w = r2o_u2{pack2<RF>(s.o[0] * inv, s.o[1] * inv), pack2<RF>(s.o[2] * inv, s.o[3] * inv)};
    *reinterpret_cast<R2O_GLOBAL r2o_u2*>((R2O_GLOBAL uint16_t*)(a.out + (int64_t)b * a.o_batch + (int64_t)head * a.o_head + (int64_t)row * a.o_row + 4 * d4)) = w;
    if (d4 == 0) a.lse[((int64_t)b * a.hq + head) * a.rows + row] = live ? (s.m + __builtin_amdgcn_logf(s.l)) * kLn2 : -INFINITY;
}

// Rows that are not merged.  Workgroups (w, .) join the segment that worker w + 1 is the second to work on, eight rows each; those
// behind the workers' write the rows that their requests do not count.  A row's states are added by 32 lanes where they are few;
// where they are more the eight groups of 32 lanes share them, for all eight rows at a time: one request of 126 rows over 32000 slots,
// 64 states a row, takes 42 us so and 72 by 32 lanes a row.
constexpr int kJoinRows = 8, kFewStates = 4;

template <int RF>
__global__ __launch_bounds__(256) void prefix_join_split_kernel(PrefixArgs) {
    __shared__ __align__(16) float red[8][kJoinRows][128];
    __shared__ float red_ml[8][kJoinRows][2];
    Args& a = kernel_args();
    const int d4 = threadIdx.x & 31, part = threadIdx.x >> 5, r0 = blockIdx.y * kJoinRows;
    if ((int)blockIdx.x >= a.workers - 1) {
        const int b = (int)blockIdx.x - (a.workers - 1), counted = counted_rows(load_uniform(a.query_lengths + b)), each = a.rows - counted;
        const int64_t rows = (int64_t)a.hq * each;
        for (int64_t i = r0 + part; i < rows; i += gridDim.y * kJoinRows) {
            const int head = (int)(i / each), row = counted + (int)(i - (int64_t)head * each);
            write_row<RF>(a, State{-INFINITY, 0.f, r2o_f4{}}, b, head, row, d4);
        }
        return;
    }
    const int w = (int)blockIdx.x + 1;
    const int* note = a.notes + kNote * w;
    const int request = load_uniform(note), head = load_uniform(note + 1), row0 = load_uniform(note + 2), rows = load_uniform(note + 3), count = load_uniform(note + 4);
    const int here = min(kJoinRows, min(kRows, rows - row0) - r0);
    if (request < 0 || here <= 0) return;
    auto states_at = [&](int i) { return (i == 0 ? split_rows(w - 1, true) : split_rows(w - 1 + i, false)) + r0; };
    State x{-INFINITY, 0.f, r2o_f4{}};
    if (count <= kFewStates) {
        if (part >= here) return;
#pragma unroll 4
        for (int i = 0; i < count; ++i) join_partial(a, x, states_at(i) + part, d4);
    } else {
        State s[kJoinRows];
#pragma unroll
        for (int k = 0; k < kJoinRows; ++k) s[k] = x;
        for (int i = part; i < count; i += 8) {
            const uint32_t at0 = states_at(i);
            float m2[kJoinRows], l2[kJoinRows];
            r2o_f4 o2[kJoinRows];
#pragma unroll
            for (int k = 0; k < kJoinRows; ++k) {
                const int64_t at = at0 + min(k, here - 1);
                m2[k] = r2o_ldg(a.partial_ml + 2 * at);
                l2[k] = r2o_ldg(a.partial_ml + 2 * at + 1);
                o2[k] = r2o_ldg(reinterpret_cast<const r2o_f4*>(a.partial_out + at * 128) + d4);
            }
#pragma unroll
            for (int k = 0; k < kJoinRows; ++k) join_state(s[k], m2[k], l2[k], o2[k]);
        }
#pragma unroll
        for (int k = 0; k < kJoinRows; ++k) {
            *reinterpret_cast<r2o_f4*>(&red[part][k][4 * d4]) = s[k].o;
            if (d4 == 0) {
                red_ml[part][k][0] = s[k].m;
                red_ml[part][k][1] = s[k].l;
            }
        }
        __syncthreads();
        if (part >= here) return;
#pragma unroll
        for (int i = 0; i < 8; ++i) join_state(x, red_ml[i][part][0], red_ml[i][part][1], *reinterpret_cast<const r2o_f4*>(&red[i][part][4 * d4]));
    }
    const int p = row0 + r0 + part, row = p / a.group;
    write_row<RF>(a, x, request, head * a.group + p - row * a.group, row, d4);
}

// Rows of a call from which on 128 lanes join a row, and 32: fewer rows have the states of more workgroups each.  A whole call of 32
// rows takes 16.3 us by 256 lanes a row and 17.3 by 128; 672: 41.7, 41.6 and by 32 49.3; 1792: 57.6, 57.7, 58.6; 3584: 35.3, 33.5,
// 33.3; 7168: 49.8, 44.1, 41.7; 16128: 85.0, 72.7, 63.3.
constexpr int64_t kJoinBy128 = 512, kJoinBy32 = 4096;

// Merged rows: PARTS groups of 32 lanes share a row's partial states of the prefix's segment and of its own.
template <int RF, int PARTS>
__global__ __launch_bounds__(256) void prefix_join_merged_kernel(PrefixArgs) {
    constexpr int kRowsHere = 8 / PARTS;
    __shared__ __align__(16) float red[8][128];
    __shared__ float red_ml[8][2];
    Args& a = kernel_args();
    const int d4 = threadIdx.x & 31, group = threadIdx.x >> 5, part = group % PARTS;
    const int per_request = a.hkv * a.packed, all_rows = a.batch * per_request;
    int at_row = kRowsHere * (int)blockIdx.x + group / PARTS;
    if (PARTS > 1) at_row = __builtin_amdgcn_readfirstlane(at_row);  // of both groups of a wave
    const bool live = at_row < all_rows;
    at_row = min(at_row, all_rows - 1);
    const int b = at_row / per_request, in_request = at_row - b * per_request, h = in_request / a.packed, p = in_request - h * a.packed;
    const int row = p / a.group, head = h * a.group + p - row * a.group;
    const int *all = a.notes, *note = a.notes + kNote * (1 + b);
    auto load = [](const int* from) { return PARTS == 1 ? r2o_ldg(from) : load_uniform(from); };
    const Share shared{load_uniform(all), 0, load_uniform(all + 1), load_uniform(all + 2)}, own{load_uniform(all + 4), 0, load_uniform(all + 5), load_uniform(all + 6)};
    const int own_first = load_uniform(all + 3), shared_base = load(note), shared_tiles = load(note + 1), before = load(note + 2), rows = load(note + 3),
              own_base = load(note + 4), own_tiles = load(note + 5), counted = load(note + 6), place = load(note + 7), by_tiles = load_uniform(all + 7);
    State s{-INFINITY, 0.f, r2o_f4{}};
    if (live && row < counted) {
        // the states of one segment, of `tiles` tiles from unit `base` on: shared by the groups, four loads of each under way
        auto add = [&](const Share& share, int base, int tiles, uint32_t whole, auto split) {
            const int w0 = share.worker(base), count = share.worker(base + tiles - 1) - w0 + 1;
            for (int i0 = part; i0 < count; i0 += 4 * PARTS) {
                float m2[4], l2[4];
                r2o_f4 o2[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = min(i0 + PARTS * k, count - 1);
                    const int64_t at = count == 1 ? whole : split(w0 + i, i == 0);
                    m2[k] = r2o_ldg(a.partial_ml + 2 * at);
                    l2[k] = r2o_ldg(a.partial_ml + 2 * at + 1);
                    o2[k] = r2o_ldg(reinterpret_cast<const r2o_f4*>(a.partial_out + at * 128) + d4);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i0 + PARTS * k < count) join_state(s, m2[k], l2[k], o2[k]);
            }
        };
        if (shared_tiles > 0 && shared.total > 0) {  // a list without units: lengths that changed meanwhile
            const int r = place - before + p, tile = r / kRows;
            add(shared, shared_base + (h * div_up(rows, kRows) + tile) * (shared_tiles + kSegment) + kSegment, shared_tiles,
                whole_prefix_rows(a, before, rows, h) + r, [&](int w, bool begins) { return split_rows(w, begins) + r - tile * kRows; });
        }
        if (own_tiles > 0 && own.total > 0) {
            if (by_tiles) {
                const int tile = p / kRows;
                add(own, own_base + (h * div_up(counted * a.group, kRows) + tile) * (own_tiles + kSegment) + kSegment, own_tiles,
                    whole_own_rows(a, b, h) + p, [&](int w, bool begins) { return split_rows(own_first + w, begins) + p - tile * kRows; });
            } else {
                const int chunk = p / kWaveRows;
                add(own, own_base + (h * div_up(counted * a.group, kWaveRows) + chunk) * (own_tiles + kWaveSegment) + kWaveSegment, own_tiles,
                    whole_own_rows(a, b, h) + p, [&](int w, bool begins) { return split_wave_rows(own_first, w, begins) + p - chunk * kWaveRows; });
            }
        }
    }
    if constexpr (PARTS > 1) {
        *reinterpret_cast<r2o_f4*>(&red[group][4 * d4]) = s.o;
        if (d4 == 0) {
            red_ml[group][0] = s.m;
            red_ml[group][1] = s.l;
        }
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int i = 1; i < PARTS; ++i) join_state(s, red_ml[group + i][0], red_ml[group + i][1], *reinterpret_cast<const r2o_f4*>(&red[group + i][4 * d4]));
    }
    if (live) write_row<RF>(a, s, b, head, row, d4);
}

// ------------------------------------------------------------------------------------ host checks
Source source_of(const r2o_paged_cache& c) {
    Source s{};
    s.key = c.key_pages;
    s.value = c.value_pages;
    s.table = c.page_table;
    s.lengths = c.lengths;
    s.k_page = (int)c.key_strides[0];
    s.k_head = (int)c.key_strides[1];
    s.k_slot = (int)c.key_strides[2];
    s.v_page = (int)c.value_strides[0];
    s.v_head = (int)c.value_strides[1];
    s.v_slot = (int)c.value_strides[2];
    s.table_stride = (int)c.table_stride;
    s.pages = (int)c.pages;
    s.last_page = (int)c.max_pages - 1;
    s.shift = 31 - __builtin_clz((unsigned)c.page_size);
    return s;
}

}  // namespace

extern "C" {

int r2o_paged_prefix_attention(const r2o_paged_prefix_params* p, void* stream) {
    if (!p || !r2o_paged_cache_ok(p->cache) || p->cache.weight_pages) return R2O_EINVAL;
    const r2o_paged_cache &c = p->cache, &f = p->prefix;
    const bool any = f.batch != 0;  // of the prefixes; without one their fields are not looked at
    if (any && (!r2o_paged_cache_ok(f) || f.weight_pages || f.hkv != c.hkv || f.dtype != c.dtype || (f.batch > 1 && !p->members))) return R2O_EINVAL;
    if (p->hq < c.hkv || p->hq > (1 << 30) || p->hq % c.hkv || p->rows < 1 || p->rows > (1 << 29) || !r2o_aligned(p->query, 16) || !r2o_aligned(p->out, 16) ||
        !r2o_aligned(p->lse, 4) || !r2o_strides_ok(p->q_strides, 3, INT64_MAX) || !r2o_strides_ok(p->o_strides, 3, INT64_MAX) ||
        p->q_strides[2] > R2O_MAX_ROW_STRIDE || p->o_strides[2] > R2O_MAX_ROW_STRIDE || reinterpret_cast<uintptr_t>(p->members) % 4 ||
        reinterpret_cast<uintptr_t>(p->query_lengths) % 4 || !(p->sm_scale > 0.f) || !(p->sm_scale < INFINITY) || p->workers < 1 ||
        p->workers > R2O_PAGED_MAX_WORKERS || !r2o_aligned(p->scratch, 16))
        return R2O_EINVAL;
    const int64_t group = p->hq / c.hkv, packed = group * p->rows;
    if (packed > (1 << 30)) return R2O_EINVAL;
    const int64_t all_rows = c.batch * c.hkv * packed;
    if (all_rows > (1 << 30)) return R2O_EINVAL;
    const int64_t shared = any ? f.max_pages * f.page_size : 0;
    const int64_t slots = c.max_pages * c.page_size;
    const bool merged = r2o_prefix_merged(c.batch, f.batch, packed, all_rows, shared, p->query_lengths);
    if (p->scratch_floats < r2o_prefix_scratch(p->workers, merged, all_rows, c.batch)) return R2O_EINVAL;
    const int64_t states = r2o_prefix_states(p->workers, merged, all_rows);
    if (r2o_prefix_units(merged, c.batch, c.hkv, packed, slots, f.batch, shared) > 0x7fffffff - kWaves * R2O_PAGED_MAX_WORKERS)
        return R2O_EINVAL;
    PrefixArgs a{};
    a.own = source_of(c);
    a.shared = any ? source_of(f) : a.own;
    a.members = p->members;
    a.query_lengths = p->query_lengths;
    a.query = p->query;
    a.out = p->out;
    a.lse = p->lse;
    a.partial_out = p->scratch;
    a.partial_ml = p->scratch + 128 * states;
    a.notes = reinterpret_cast<int*>(p->scratch + 130 * states);
    a.q_batch = p->q_strides[0];
    a.q_head = p->q_strides[1];
    a.q_row = (int)p->q_strides[2];
    a.o_batch = p->o_strides[0];
    a.o_head = p->o_strides[1];
    a.o_row = (int)p->o_strides[2];
    a.batch = (int)c.batch;
    a.prefixes = (int)f.batch;
    a.hkv = (int)c.hkv;
    a.hq = (int)p->hq;
    a.group = (int)group;
    a.rows = (int)p->rows;
    a.packed = (int)packed;
    a.workers = (int)p->workers;
    a.c2 = p->sm_scale * kLog2e;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)p->workers);
    auto launch = [&](auto partial, auto join_kernel, const dim3& join) {
        hipLaunchKernelGGL(partial, grid, dim3(64 * kWaves), 0, st, a);
        if (hipGetLastError() != hipSuccess) return R2O_ELAUNCH;
        if (join.x == 0) return R2O_OK;
        hipLaunchKernelGGL(join_kernel, join, dim3(256), 0, st, a);
        return hipGetLastError() == hipSuccess ? R2O_OK : R2O_ELAUNCH;
    };
    if (merged) {
        auto join = [&](auto parts) {
            constexpr int kParts = decltype(parts)::value;
            const dim3 blocks((unsigned)((all_rows * kParts + 7) / 8));
            return c.dtype == 0 ? launch(prefix_partial_kernel<0, true>, prefix_join_merged_kernel<0, kParts>, blocks)
                                : launch(prefix_partial_kernel<1, true>, prefix_join_merged_kernel<1, kParts>, blocks);
        };
        if (all_rows < kJoinBy128) return join(std::integral_constant<int, 8>());
        if (all_rows < kJoinBy32) return join(std::integral_constant<int, 4>());
        return join(std::integral_constant<int, 1>());
    }
    const dim3 join((unsigned)(p->workers - 1 + (p->query_lengths ? c.batch : 0)), kRows / kJoinRows);
    return c.dtype == 0 ? launch(prefix_partial_kernel<0, false>, prefix_join_split_kernel<0>, join)
                        : launch(prefix_partial_kernel<1, false>, prefix_join_split_kernel<1>, join);
}

}  // extern "C"
