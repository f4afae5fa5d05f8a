// Attention over a prefix that many requests share, and over each request's own slots of the paged cache, for gfx950.
//
// Requests of one prefix stand side by side; row i of request b (q of its rows count, n slots are its own) sees every
// slot of its prefix and its own slots j <= n - q + i:
//     out = sum_j softmax_j(c q . k_j) v_j,     lse = log sum_j exp(c q . k_j)
// over both.  Rows of a KV head's query heads and, where a request has few, of all requests of a prefix are one list, in
// tiles of 128: the prefix's rows are read once for all of them.  The (row tile, key tile) pairs of a call are one list too,
// shared evenly over the workgroups, whatever the lengths; where a row tile's keys fall to several, or to a prefix and a
// request of its own, each leaves (maximum, sum, products) in scratch for the join.
#include <algorithm>
#include <initializer_list>

#include "r2o_cache_check.hpp"
#include "r2o_common.hpp"
#include "r2o_tiles.hpp"

namespace {

using namespace r2o_tiles;

constexpr int kRows = 128;   // rows of a workgroup: 4 waves of 32
constexpr int kMinTiles = 2; // key tiles that a workgroup takes at least

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
    int64_t q_batch, q_head, o_batch, o_head;
    int q_row, o_row, batch, prefixes, hkv, hq, group, rows, packed, workers, merged;  // packed: rows * group
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

__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }

__device__ __forceinline__ int filled(SourceArgs& s, int length) { return min(max(length, 0), (s.last_page + 1) << s.shift); }
__device__ __forceinline__ int key_tiles(SourceArgs& s, int length) { return (filled(s, length) + kTile - 1) / kTile; }

// ------------------------------------------------------------------------------------- the list
// Entries: where rows are merged, each prefix (with the rows of all its requests) and then each request (its own slots);
// otherwise each request, its prefix's slots before its own.  An entry has `heads` times its row tiles times its key tiles
// of work.  The wave goes through them 64 at a time, one a lane.
struct Members {
    int first, count;  // requests of this lane's prefix
};

// Counts are cut off where the batch ends, so that whatever they hold no request has two prefixes.
__device__ __forceinline__ Members lane_members(Args& a, int g0, int& before) {
    const int g = g0 + (threadIdx.x & 63);
    int m = 0;
    if (g < a.prefixes) m = a.members ? min(max(r2o_ldg(a.members + g), 0), a.batch) : a.batch;
    const int upto = wave_scan(m);
    Members x;
    x.first = min(before + upto - m, a.batch);
    x.count = min(m, a.batch - x.first);
    before = min(before + last_lane(upto), a.batch);
    return x;
}

__device__ __forceinline__ int row_tiles(int rows) { return (rows + kRows - 1) / kRows; }

// Work of this lane's prefix (merged rows).
__device__ __forceinline__ int lane_prefix_work(Args& a, int g0, const Members& x) {
    const int g = g0 + (threadIdx.x & 63);
    return g < a.prefixes && x.count ? a.hkv * row_tiles(x.count * a.packed) * key_tiles(a.shared, r2o_ldg(a.shared.lengths + g)) : 0;
}

// The prefix of this lane's request, -1 for none, and all lanes' members are looked at: one step a prefix.
__device__ __forceinline__ int prefix_of(Args& a, int b) {
    int of = -1, before = 0;
    for (int g0 = 0; g0 < a.prefixes; g0 += 64) {
        const Members x = lane_members(a, g0, before);
        const int here = min(64, a.prefixes - g0);
        for (int i = 0; i < here; ++i) {
            const int first = __builtin_amdgcn_readlane(x.first, i), count = __builtin_amdgcn_readlane(x.count, i);
            of = (uint32_t)(b - first) < (uint32_t)count ? g0 + i : of;
        }
    }
    return of;
}

// Work of this lane's request.  Not merged, a row tile without a key has one tile, of none: its rows are written there.
__device__ __forceinline__ int lane_request_work(Args& a, int b0) {
    const int b = b0 + (threadIdx.x & 63);
    int tiles = b < a.batch ? key_tiles(a.own, r2o_ldg(a.own.lengths + b)) : 0;
    if (a.merged) return a.hkv * tiles;
    const int g = prefix_of(a, b);
    if (g >= 0 && b < a.batch) tiles += key_tiles(a.shared, r2o_ldg(a.shared.lengths + g));
    return b < a.batch ? a.hkv * row_tiles(a.packed) * max(tiles, 1) : 0;
}

// The list shared evenly: worker i takes `each` tiles from begin(i) on, the first `more` workers one more.
struct Share {
    int total, workers, each, more;
    __device__ __forceinline__ int begin(int i) const { return i * each + min(i, more); }
    __device__ __forceinline__ int worker(int at) const {  // the one that takes tile `at`
        const int u = min(at, total - 1), wide = more * (each + 1);
        return u < wide ? (int)((uint32_t)u / (uint32_t)(each + 1)) : more + (int)((uint32_t)(u - wide) / (uint32_t)each);
    }
};

__device__ __forceinline__ Share share_of(Args& a, int total) {
    Share s;
    s.total = total;
    s.workers = max(1, min(a.workers, (total + kMinTiles - 1) / kMinTiles));
    s.each = (int)((uint32_t)total / (uint32_t)s.workers);
    s.more = total - s.each * s.workers;
    return s;
}

// An entry: its place in the list, and what it is.
struct Entry {
    int base, work;      // tiles before it, its own
    int prefix, request; // request -1: all of a prefix's
    int first, members;  // of the prefix
};

// The entry that holds tile u; the tiles of all entries, if `all`.  u = -1: none.
__device__ __forceinline__ Entry find(Args& a, int u, int& total) {
    Entry e{};
    e.request = -2;
    int at = 0;
    const int lane = threadIdx.x & 63;
    if (a.merged) {
        int before = 0;
        for (int g0 = 0; g0 < a.prefixes; g0 += 64) {
            const Members x = lane_members(a, g0, before);
            const int work = lane_prefix_work(a, g0, x), upto = wave_scan(work), all = last_lane(upto);
            if ((uint32_t)(u - at) < (uint32_t)all) {
                const int i = __builtin_ctzll(__ballot(at + upto > u));
                e.base = at + __builtin_amdgcn_readlane(upto - work, i);
                e.work = __builtin_amdgcn_readlane(work, i);
                e.prefix = g0 + i;
                e.request = -1;
                e.first = __builtin_amdgcn_readlane(x.first, i);
                e.members = __builtin_amdgcn_readlane(x.count, i);
            }
            at += all;
        }
    }
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int work = lane_request_work(a, b0), upto = wave_scan(work), all = last_lane(upto);
        if ((uint32_t)(u - at) < (uint32_t)all) {
            const int i = __builtin_ctzll(__ballot(at + upto > u));
            e.base = at + __builtin_amdgcn_readlane(upto - work, i);
            e.work = __builtin_amdgcn_readlane(work, i);
            e.request = b0 + i;
            e.prefix = a.merged ? -1 : __builtin_amdgcn_readlane(prefix_of(a, b0 + lane), i);
        }
        at += all;
    }
    total = at;
    return e;
}

// One row tile of an entry and head, and the keys that it may see: `shared` tiles of the prefix, then `own` ones.
struct Segment {
    int base, tiles;         // in the list
    int head, row0, rows;    // first row in the entry's list of them, and that list's end
    int shared, n_shared, n_own;
};

__device__ __forceinline__ Segment segment_of(Args& a, const Entry& e, int u) {
    Segment s;
    s.n_shared = e.prefix >= 0 ? filled(a.shared, load_uniform(a.shared.lengths + e.prefix)) : 0;
    s.n_own = e.request >= 0 ? filled(a.own, load_uniform(a.own.lengths + e.request)) : 0;
    s.shared = (s.n_shared + kTile - 1) / kTile;
    s.tiles = max(1, s.shared + (s.n_own + kTile - 1) / kTile);
    s.rows = e.request < 0 ? e.members * a.packed : a.packed;
    const int per_head = row_tiles(s.rows), at = (int)((uint32_t)(u - e.base) / (uint32_t)s.tiles);
    s.head = (int)((uint32_t)at / (uint32_t)per_head);
    s.row0 = (at - s.head * per_head) * kRows;
    s.base = e.base + at * s.tiles;
    return s;
}

// Where partial states lie: two tiles of rows for each worker, for the segments that it does not have alone (the one that
// another began, and the one that it leaves to others), then, where rows are merged, a place for each row of the prefixes'
// segments and of the requests'.
__device__ __forceinline__ int64_t split_rows(int worker, bool begins) { return ((int64_t)2 * worker + begins) * kRows; }
__device__ __forceinline__ int64_t whole_rows(Args& a, bool shared, int first, int members, int b, int head) {
    const int64_t packed = a.packed, base = (int64_t)2 * a.workers * kRows;
    return base + (shared ? ((int64_t)first * a.hkv + (int64_t)head * members) * packed : ((int64_t)(a.batch + b) * a.hkv + head) * packed);
}

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

// The page of slot j, -1 if it has none.
__device__ __forceinline__ int page_of(const Side& x, int j) {
    const int id = load_uniform(x.table + min(j >> x.shift, x.last_page));
    return j < x.n && (uint32_t)id < (uint32_t)x.pages ? id : -1;
}

// Four groups of 16 slots, each within a page: bit i for one that has a page and a filled slot.
__device__ __forceinline__ int tile_valid(const Side& x, int j0, int wave, int& page) {
    int valid = 0;
    page = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int id = page_of(x, j0 + 16 * i);
        valid |= (id >= 0) << i;
        page = i == wave ? max(id, 0) : page;
    }
    return valid;
}

// This wave's 16 rows of K and V, straight into LDS.
template <int SWZ>
__device__ __forceinline__ void stage_group(const uint16_t* base, int stride, unsigned char* lds, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)row_chunk<SWZ>(base, stride, 4 * i, 15, i, lane),
            (__attribute__((address_space(3))) void*)(lds + (16 * wave + 4 * i) * 256), 16, 0, 0);
}

// One workgroup: its share of the list.  S^T = K Q^T (32 keys x 32 rows a product), O^T += V^T P^T; two tiles ahead go into LDS
// while one is computed on.
// The probabilities are rounded to the rows' 16 bits for the product with V, whose two operands are of one type; their sum
// takes them unrounded.
template <int RF>
__global__ __launch_bounds__(256, 2) void prefix_partial_kernel(PrefixArgs) {
    __shared__ __align__(16) unsigned char k_lds[2][kTileBytes], v_lds[3][kTileBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int worker = blockIdx.x;
    int u, u_end;
    {
        Args& a = kernel_args();
        int total;
        find(a, -1, total);
        const Share share = share_of(a, total);
        if (worker >= share.workers || total == 0) return;
        u = share.begin(worker);
        u_end = share.begin(worker + 1);
    }
    while (u < u_end) {
        Args& a = kernel_args();
        int total;
        const Entry e = find(a, u, total);
        if (e.request == -2) return;  // lengths that change meanwhile
        const Segment s = segment_of(a, e, u);
        const int begin = u - s.base, stop = min(s.tiles, u_end - s.base);
        if (begin < 0 || stop <= begin || s.head >= a.hkv) return;

        // this lane's row, and the last key of its own that it sees
        const int at = min(s.row0 + 32 * wave + col, s.rows - 1), group = a.group;
        const int rank = e.request < 0 ? at / a.packed : 0, p = at - rank * a.packed, row = p / group, head = s.head * group + p - row * group;
        const int b = e.request < 0 ? e.first + rank : e.request;
        const bool busy = s.row0 + 32 * wave < s.rows;  // of this wave
        // where its partial state goes; -1 for no row, -2 for a row that is written here
        uint32_t to = 0xffffffffu;
        if (s.row0 + 32 * wave + col < s.rows) {
            if (begin > 0 || stop < s.tiles) to = (uint32_t)split_rows(worker, begin == 0) + 32 * wave + col;
            else if (a.merged) to = (uint32_t)whole_rows(a, e.request < 0, e.first, e.members, e.request, s.head) + s.row0 + 32 * wave + col;
            else to = 0xfffffffeu;
        }
        int counted = a.rows;
        if (a.query_lengths) counted = min(max(r2o_ldg(a.query_lengths + b), 0), a.rows);
        const int off = s.n_own - counted;
        const int see_own = min(off + row, s.n_own - 1);
        // the least that a row of the workgroup, and of this wave, sees of them; no row of a prefix's segment has any
        const int wg_least = __builtin_amdgcn_readfirstlane(e.request < 0 ? 0 : min(s.n_own - counted + s.row0 / group, s.n_own - 1));
        const int most = __builtin_amdgcn_readfirstlane(
            e.request < 0 ? -1 : min(s.n_own - counted + min(s.row0 + kRows - 1, s.rows - 1) / group, s.n_own - 1));
        const int last = min(stop, s.shared + max(most, -1) / kTile + (most >= 0));  // tiles behind it are seen by no row

        r2o_u4 q[8];
        {
            const uint16_t* src = a.query + (int64_t)b * a.q_batch + (int64_t)head * a.q_head + (int64_t)row * a.q_row + 8 * half;
#pragma unroll
            for (int t = 0; t < 8; ++t) q[t] = r2o_ldg(reinterpret_cast<const r2o_u4*>(src + 16 * t));
        }
        float m = -INFINITY, l = 0.f;
        f16v acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = f16v{};
        const float c2 = a.c2;
        bool bad = false;

        auto side_at = [&](int it) {
            Args& x = kernel_args();
            return it < s.shared ? side_of(x.shared, e.prefix, s.head, s.n_shared) : side_of(x.own, e.request, s.head, s.n_own);
        };
        auto slot_of = [&](int it) { return (it < s.shared ? it : it - s.shared) * kTile; };
        // Loads of a tile; which groups of 16 slots count.
        auto stage = [&](int it, int v_at) {
            const Side x = side_at(it);
            const int j0 = slot_of(it), j = (j0 + 16 * wave) & ((1 << x.shift) - 1);
            int page;
            const int valid = tile_valid(x, j0, wave, page);
            stage_group<0>(x.k + (int64_t)page * x.k_page + (int64_t)j * x.k_slot, x.k_slot, k_lds[it & 1], wave, lane);
            stage_group<1>(x.v + (int64_t)page * x.v_page + (int64_t)j * x.v_slot, x.v_slot, v_lds[v_at], wave, lane);
            return valid;
        };
        auto last_seen = [&](int it) { return it < s.shared ? s.n_shared - 1 : see_own; };
        // This wave's 16 value rows of a staged tile.  Rows that no row of the workgroup sees may hold anything: zero.  Where some see
        // a row that others do not, 0 times an infinite or NaN value would be NaN: those become zero before any product.
        auto clean = [&](int it, int v_at, int valid) {
            const int n = it < s.shared ? s.n_shared : s.n_own, j0 = slot_of(it) + 16 * wave;
            const bool some = it >= s.shared && slot_of(it) + kTile - 1 > wg_least && wg_least < n - 1;
            const bool ends = j0 + 16 > n || !(valid >> wave & 1);
            if (!some && !ends) return;
            r2o_u4* at_lds = reinterpret_cast<r2o_u4*>(v_lds[v_at] + 16 * wave * 256) + lane;
            r2o_u4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = at_lds[64 * i];
                if (!(valid >> wave & 1) || j0 + 4 * i + (lane >> 4) >= n) x[i] = r2o_u4{};
            }
            bad |= some && zero_not_finite<RF>(x);
#pragma unroll
            for (int i = 0; i < 4; ++i) at_lds[64 * i] = x[i];
        };
        auto products = [&](const unsigned char* kl, int sub) __attribute__((always_inline)) {
            f16v x = f16v{};
            r2o_u4 k[8];
            read_all_rows(kl, sub, lane, k);
#pragma unroll
            for (int t = 0; t < 8; ++t) x = mfma32<RF>(k[t], q[t], x);
            return x;
        };
        // masks, and the running maximum raised where it has to be
        auto top_of = [&](f16v& x, int it, int sub, int valid) __attribute__((always_inline)) {
            const int from = slot_of(it) + 32 * sub, seen = last_seen(it);
            if (valid != 15 || __any(from + 31 > seen)) {
                const int back = seen - from - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    x[i] = back >= 8 * (i >> 2) + (i & 3) && (valid >> (2 * sub + (i >> 3)) & 1) ? x[i] : -INFINITY;
            }
            float tmax = fmaxf(x[0], x[1]);
#pragma unroll
            for (int i = 2; i < 16; i += 2) tmax = fmaxf(tmax, fmaxf(x[i], x[i + 1]));
            float y, z;
            r2o_row_swap<32>(tmax, y, z);
            tmax = fmaxf(y, z) * c2;  // -inf stays (c2 > 0)
            if (__any(tmax > m + kSlack)) {
                // of the rows that exceed it alone: a row's result does not depend on its neighbours
                const float m_new = tmax > m + kSlack ? tmax : m;
                const float alpha = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
                l *= alpha;
#pragma unroll
                for (int db = 0; db < 4; ++db) acc[db] *= alpha;
                m = m_new;
            }
        };
        auto probabilities = [&](const f16v& x, r2o_u4 (&pk)[2]) __attribute__((always_inline)) {
            const float mm = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c2, -mm));
                const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i + 1], c2, -mm));
                l += e0 + e1;
                pk[i >> 3][(i & 7) >> 1] = pack2<RF>(e0, e1);
            }
        };
        auto values = [&](const unsigned char* vl, int sub, const r2o_u4 (&pk)[2]) __attribute__((always_inline)) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int db = 0; db < 4; ++db) acc[db] = mfma32<RF>(read_values(vl, 2 * sub + kb, db, lane), pk[kb], acc[db]);
        };
        // A tile is two halves of 32 keys; the products of the half that follows run beside the exponentials of the one
        // before it.  A wave without rows brings its rows of the tiles alone.
        if (begin < last) {
            int valid = stage(begin, 0), next = 0, after = 0;
            if (begin + 1 < last) next = stage(begin + 1, 1);
            wait_staged();
            clean(begin, 0, valid);
            __syncthreads();
            f16v even{};
            if (busy) even = products(k_lds[begin & 1], 0);
            for (int it = begin, v_at = 0; it < last; ++it) {
                const int v_next = v_at == 2 ? 0 : v_at + 1;
                r2o_u4 pk[2];
                f16v odd{};
                if (busy) {
                    top_of(even, it, 0, valid);
                    odd = products(k_lds[it & 1], 1);
                    probabilities(even, pk);
                    values(v_lds[v_at], 0, pk);
                    top_of(odd, it, 1, valid);
                }
                wait_staged();
                if (it + 1 < last) clean(it + 1, v_next, next);
                __syncthreads();  // the next tile is there; this one's V stays till every wave is past the next barrier
                if (busy) {
                    even = products(k_lds[(it + 1) & 1], 0);  // behind the last tile: what lies there, not used
                    probabilities(odd, pk);
                    values(v_lds[v_at], 1, pk);
                }
                if (it + 2 < last) after = stage(it + 2, v_next == 2 ? 0 : v_next + 1);
                valid = next;
                next = after;
                v_at = v_next;
            }
        }
        __syncthreads();
        int* const flags = reinterpret_cast<int*>(k_lds[0]);
        const bool wave_bad = __any(bad);
        if (lane == 0) flags[wave] = wave_bad;
        __syncthreads();
        const bool any_bad = (flags[0] | flags[1] | flags[2] | flags[3]) != 0;
        {
            float x, y;
            r2o_row_swap<32>(l, x, y);
            l = x + y;
        }
        // A row's channel is infinite or NaN where a key that it sees is, however small that key's weight: not NaN where the weight
        // is rounded to 0 on its way to the product.  Those channels are formed again from the values alone.
        float odd_sum[4] = {};
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int db = 0; db < 4; ++db) odd_sum[db] = __builtin_fmaf(acc[db][i], 0.f, odd_sum[db]);  // NaN where one is not finite
        const float any_odd = odd_sum[0] + odd_sum[1] + odd_sum[2] + odd_sum[3];
        const bool met = __any(any_odd != any_odd && l == l && row < counted);  // a NaN sum, of a NaN logit, makes the whole row NaN
        if (busy && (any_bad || met)) {
            f16v extra[4];
#pragma unroll
            for (int db = 0; db < 4; ++db) extra[db] = f16v{};
            bool more = true;  // till every row has NaN alone
            for (int it = begin; it < last && more; ++it) {
                const Side x = side_at(it);
                const int seen = last_seen(it);
                for (int j16 = slot_of(it); j16 < slot_of(it) + kTile && more; j16 += 16) {
                    const int page = page_of(x, j16);
                    if (page < 0) continue;
                    const uint16_t* rows = x.v + (int64_t)page * x.v_page + (int64_t)(j16 & ((1 << x.shift) - 1)) * x.v_slot;
                    r2o_u4 chunk[4];  // of four rows each
                    bool any = false;
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        chunk[n] = r2o_ldg(reinterpret_cast<const r2o_u4*>(rows + (int64_t)(4 * n + (lane >> 4)) * x.v_slot) + (lane & 15));
#pragma unroll
                    for (int n = 0; n < 4; ++n) any |= any_not_finite<RF>(chunk[n]);
                    if (!__any(any)) continue;
                    for (int j = 0; j < min(16, x.n - j16); ++j) {
                        if (j16 + j > seen) continue;
                        const uint16_t* src = rows + (int64_t)j * x.v_slot + 4 * half;
#pragma unroll
                        for (int db = 0; db < 4; ++db)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const uint32_t y = r2o_ldg(src + 32 * db + 8 * (i >> 2) + (i & 3));
                                if (not_finite<RF>(y)) extra[db][i] += RF == 0 ? r2o_bf16_to_f32(y) : r2o_f16_to_f32(y);
                            }
                    }
                    bool all_nan = true;
#pragma unroll
                    for (int db = 0; db < 4; ++db)
#pragma unroll
                        for (int i = 0; i < 16; ++i) all_nan &= extra[db][i] != extra[db][i];
                    more = !__all(all_nan || row >= counted);
                }
            }
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[db][i] = __builtin_isfinite(extra[db][i]) ? acc[db][i] : extra[db][i];
        }
        if (to != 0xffffffffu) {
            Args& x = kernel_args();
            if (to == 0xfffffffeu) {
                const bool live = row < counted && !(l == 0.f);  // no key seen; NaN logits leave m, and a NaN sum
                const float inv = live ? 1.f / l : 0.f;
                uint16_t* dst = x.out + (int64_t)b * x.o_batch + (int64_t)head * x.o_head + (int64_t)row * x.o_row;
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        r2o_u2 w;
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            w[k] = live ? pack2<RF>(acc[db][4 * g + 2 * k] * inv, acc[db][4 * g + 2 * k + 1] * inv) : 0u;
                        *reinterpret_cast<R2O_GLOBAL r2o_u2*>((R2O_GLOBAL uint16_t*)(dst + 32 * db + 8 * g + 4 * half)) = w;
                    }
                if (half == 0) x.lse[((int64_t)b * x.hq + head) * x.rows + row] = live ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
            } else {
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<R2O_GLOBAL r2o_f4*>((R2O_GLOBAL float*)(x.partial_out + (int64_t)to * 128 + 32 * db + 8 * g + 4 * half)) =
                            r2o_f4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
                if (half == 0) {
                    x.partial_ml[2 * (int64_t)to] = row < counted ? m : -INFINITY;
                    x.partial_ml[2 * (int64_t)to + 1] = row < counted ? l : 0.f;
                }
            }
        }
        u = s.base + stop;
        __syncthreads();  // the flags lie where the next tiles go
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

__device__ __forceinline__ void join_partial(Args& a, State& s, int64_t at, int d4) {
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

// Rows that are not merged: the workgroups (w, .) join the segment that worker w is the second to work on, 32 lanes a row.
template <int RF>
__global__ __launch_bounds__(256) void prefix_join_split_kernel(PrefixArgs) {
    Args& a = kernel_args();
    int total;
    find(a, -1, total);
    const Share share = share_of(a, total);
    const int w = (int)blockIdx.x + 1;
    if (w >= share.workers) return;
    const int u = share.begin(w);
    const Entry e = find(a, u, total);
    if (e.request < 0) return;
    const Segment s = segment_of(a, e, u);
    if (s.base == u || s.base < share.begin(w - 1) || s.head >= a.hkv) return;  // begun here, or by another than the one before
    const int count = share.worker(s.base + s.tiles - 1) - (w - 1) + 1;
    const int r = blockIdx.y * 8 + (threadIdx.x >> 5), d4 = threadIdx.x & 31;
    if (s.row0 + r >= s.rows) return;
    State x{-INFINITY, 0.f, r2o_f4{}};
    join_partial(a, x, split_rows(w - 1, true) + r, d4);
#pragma unroll 4
    for (int i = 1; i < count; ++i) join_partial(a, x, split_rows(w - 1 + i, false) + r, d4);
    const int p = s.row0 + r, row = p / a.group;
    write_row<RF>(a, x, e.request, s.head * a.group + p - row * a.group, row, d4);
}

// Merged rows: a workgroup a row, whose partial states of the prefix's segment and of its own are shared by 8 groups of 32
// lanes.
template <int RF>
__global__ __launch_bounds__(256) void prefix_join_merged_kernel(PrefixArgs) {
    __shared__ __align__(16) float red[8][128];
    __shared__ float red_ml[8][2];
    Args& a = kernel_args();
    const int per_request = a.hkv * a.packed;
    const int b = (int)blockIdx.x / per_request, in_request = (int)blockIdx.x - b * per_request, h = in_request / a.packed, p = in_request - h * a.packed;
    const int row = p / a.group, head = h * a.group + p - row * a.group, d4 = threadIdx.x & 31, part = threadIdx.x >> 5;
    // one pass over the list: its length, and where this row's segments lie
    int at = 0, before = 0, shared_base = 0, first = 0, members = 0, prefix = -1, own_base = 0;
    for (int g0 = 0; g0 < a.prefixes; g0 += 64) {
        const Members x = lane_members(a, g0, before);
        const int work = lane_prefix_work(a, g0, x), upto = wave_scan(work);
        const uint64_t mine = __ballot((uint32_t)(b - x.first) < (uint32_t)x.count);
        if (mine) {
            const int i = __builtin_ctzll(mine);
            prefix = g0 + i;
            shared_base = at + __builtin_amdgcn_readlane(upto - work, i);
            first = __builtin_amdgcn_readlane(x.first, i);
            members = __builtin_amdgcn_readlane(x.count, i);
        }
        at += last_lane(upto);
    }
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int work = lane_request_work(a, b0), upto = wave_scan(work);
        if ((uint32_t)(b - b0) < 64u) own_base = at + __builtin_amdgcn_readlane(upto - work, b - b0);
        at += last_lane(upto);
    }
    const Share share = share_of(a, at);
    const int shared_tiles = prefix >= 0 ? key_tiles(a.shared, load_uniform(a.shared.lengths + prefix)) : 0;
    const int own_tiles = key_tiles(a.own, load_uniform(a.own.lengths + b));
    const int counted = a.query_lengths ? load_uniform(a.query_lengths + b) : a.rows;
    State s{-INFINITY, 0.f, r2o_f4{}};
    auto add = [&](int base, int tiles, int r, int64_t whole) {  // the states of one segment, row r of its tile
        if (tiles == 0 || share.total == 0) return;
        const int w0 = share.worker(base), count = share.worker(base + tiles - 1) - w0 + 1;
        if (count == 1) {
            if (part == 0) join_partial(a, s, whole, d4);
            return;
        }
        for (int i = part; i < count; i += 8) join_partial(a, s, split_rows(w0 + i, i == 0) + r, d4);
    };
    if (row < counted) {
        const int r = (b - first) * a.packed + p, tile = r / kRows;
        if (prefix >= 0)
            add(shared_base + (h * row_tiles(members * a.packed) + tile) * shared_tiles, shared_tiles, r - tile * kRows,
                whole_rows(a, true, first, members, b, h) + r);
        add(own_base + h * own_tiles, own_tiles, p, whole_rows(a, false, 0, 0, b, h) + p);
    }
    *reinterpret_cast<r2o_f4*>(&red[part][4 * d4]) = s.o;
    if (d4 == 0) {
        red_ml[part][0] = s.m;
        red_ml[part][1] = s.l;
    }
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) join_state(s, red_ml[i][0], red_ml[i][1], *reinterpret_cast<const r2o_f4*>(&red[i][4 * d4]));
    write_row<RF>(a, s, b, head, row, d4);
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

int64_t tiles_of(const r2o_paged_cache& c) { return (c.max_pages * c.page_size + kTile - 1) / kTile; }

}  // namespace

extern "C" {

int r2o_paged_prefix_attention(const r2o_paged_prefix_params* p, void* stream) {
    if (!p || !r2o_paged_cache_ok(p->cache) || p->cache.weight_pages) return R2O_EINVAL;
    const r2o_paged_cache &c = p->cache, &f = p->prefix;
    const bool any = f.batch != 0;  // of the prefixes; without one their fields are not looked at
    if (any && (!r2o_paged_cache_ok(f) || f.weight_pages || f.hkv != c.hkv || f.dtype != c.dtype || (f.batch > 1 && !p->members))) return R2O_EINVAL;
    if (p->hq < c.hkv || p->hq % c.hkv || p->rows < 1 || p->rows > (1 << 29) || !r2o_aligned(p->query, 16) || !r2o_aligned(p->out, 16) ||
        !r2o_aligned(p->lse, 4) || !r2o_strides_ok(p->q_strides, 3, INT64_MAX) || !r2o_strides_ok(p->o_strides, 3, INT64_MAX) ||
        p->q_strides[2] > R2O_MAX_ROW_STRIDE || p->o_strides[2] > R2O_MAX_ROW_STRIDE || reinterpret_cast<uintptr_t>(p->members) % 4 ||
        reinterpret_cast<uintptr_t>(p->query_lengths) % 4 || !(p->sm_scale > 0.f) || !(p->sm_scale < INFINITY) || p->workers < 1 ||
        p->workers > R2O_PAGED_MAX_WORKERS || !r2o_aligned(p->scratch, 16))
        return R2O_EINVAL;
    const int64_t group = p->hq / c.hkv, packed = group * p->rows, all_rows = c.batch * c.hkv * packed;
    if (packed > (1 << 30) || all_rows > (1 << 30)) return R2O_EINVAL;
    const bool merged = any && packed < kRows;
    if (p->scratch_floats < 130 * (2 * kRows * p->workers + (merged ? 2 * all_rows : 0))) return R2O_EINVAL;
    // whatever the lengths on the device say
    const int64_t shared = any ? tiles_of(f) : 0, per_request = (packed + kRows - 1) / kRows;
    const int64_t most = merged ? c.hkv * (((c.batch * packed) / kRows + f.batch) * shared + c.batch * tiles_of(c))
                                : c.hkv * c.batch * per_request * (shared + tiles_of(c));
    if (most > 0x7fffffff - R2O_PAGED_MAX_WORKERS) return R2O_EINVAL;
    PrefixArgs a{};
    a.own = source_of(c);
    a.shared = any ? source_of(f) : a.own;
    a.members = p->members;
    a.query_lengths = p->query_lengths;
    a.query = p->query;
    a.out = p->out;
    a.lse = p->lse;
    a.partial_out = p->scratch;
    a.partial_ml = p->scratch + 128 * (p->scratch_floats / 130);
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
    a.merged = merged;
    a.c2 = p->sm_scale * kLog2e;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)p->workers);
    if (c.dtype == 0) hipLaunchKernelGGL(prefix_partial_kernel<0>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(prefix_partial_kernel<1>, grid, dim3(256), 0, st, a);
    R2O_CHECK_LAUNCH();
    if (merged) {
        const dim3 join((unsigned)all_rows);
        if (c.dtype == 0) hipLaunchKernelGGL(prefix_join_merged_kernel<0>, join, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(prefix_join_merged_kernel<1>, join, dim3(256), 0, st, a);
        R2O_CHECK_LAUNCH();
    } else if (p->workers > 1) {
        const dim3 join((unsigned)p->workers - 1, kRows / 8);
        if (c.dtype == 0) hipLaunchKernelGGL(prefix_join_split_kernel<0>, join, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(prefix_join_split_kernel<1>, join, dim3(256), 0, st, a);
        R2O_CHECK_LAUNCH();
    }
    return R2O_OK;
}

}  // extern "C"
