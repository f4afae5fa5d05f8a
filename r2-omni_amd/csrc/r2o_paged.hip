// A paged key-value cache for gfx950: rows written into it, attention of one new token over it, and the
// eviction of the tokens that received the least attention.
//
// K and V rows of 128 channels (bf16 or fp16) live in pages of 16, 32, 64 or 128 slots; a request's slot j is slot
// j % size of page page_table[b][j / size], for every KV head.  A page id outside the pool makes its slots
// invisible and keeps every access in bounds.
#include <algorithm>
#include <cstdlib>
#include <initializer_list>
#include <type_traits>

#include "r2o_common.hpp"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Filled slots of a request, within what its page table can hold.
__device__ __forceinline__ int filled(const r2o_paged_cache& c, int b) {
    return min(max(r2o_ldg(c.lengths + b), 0), (int)(c.max_pages * c.page_size));
}

// A word at an address that the whole wave shares and that nothing writes meanwhile, through the scalar cache: it
// waits for no vector load and no vector load waits for it.
__device__ __forceinline__ int load_uniform(const int32_t* p) {
    return *(const __attribute__((address_space(4))) int32_t*)p;
}

__device__ __forceinline__ int shift_of(const r2o_paged_cache& c) { return 31 - __builtin_clz((int)c.page_size); }

// The page of a request's slot, or -1.
__device__ __forceinline__ int page_of(const r2o_paged_cache& c, int b, int slot, int shift) {
    const int page = r2o_ldg(c.page_table + b * c.table_stride + (slot >> shift));
    return (uint32_t)page < (uint32_t)c.pages ? page : -1;
}

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

// ---------------------------------------------------------------------------------------- extend
// 16 lanes move one K and one V row.  Bound by the rows' bytes for a prompt (32641 rows of 8 heads: 52 us, 5.2 TB/s read and written), by the
// launch for a step (5 us).
__global__ __launch_bounds__(256) void paged_extend_kernel(r2o_paged_extend_params p) {
    const r2o_paged_cache& c = p.cache;
    const int h = blockIdx.y, b = blockIdx.z, l16 = threadIdx.x & 15;
    const int i = blockIdx.x * 16 + (threadIdx.x >> 4);
    const int count = p.counts ? min(max(r2o_ldg(p.counts + b), 0), (int)p.rows) : (int)p.rows;
    const int slot = r2o_ldg(c.lengths + b) - count + i, shift = shift_of(c);
    if (i >= count || slot < 0 || slot >= (int)(c.max_pages * c.page_size)) return;
    const int page = page_of(c, b, slot, shift);
    if (page < 0) return;
    const int at = slot & ((1 << shift) - 1);
    const r2o_u4 k = r2o_ldg(reinterpret_cast<const r2o_u4*>(p.key + b * p.key_strides[0] + h * p.key_strides[1] + (int64_t)i * p.key_strides[2]) + l16);
    const r2o_u4 v = r2o_ldg(reinterpret_cast<const r2o_u4*>(p.value + b * p.value_strides[0] + h * p.value_strides[1] + (int64_t)i * p.value_strides[2]) + l16);
    r2o_store8<true>(c.key_pages + page * c.key_strides[0] + h * c.key_strides[1] + at * c.key_strides[2] + 8 * l16, k);
    r2o_store8<true>(c.value_pages + page * c.value_strides[0] + h * c.value_strides[1] + at * c.value_strides[2] + 8 * l16, v);
    if (c.weight_pages && l16 == 0)
        c.weight_pages[page * c.weight_strides[0] + h * c.weight_strides[1] + at] =
            p.weights ? r2o_ldg(p.weights + b * p.weights_strides[0] + h * p.weights_strides[1] + i) : 0.f;
}

// ------------------------------------------------------------------------------------- attention
constexpr int kWaves = 4;
constexpr int kSlots = 32;                 // slots of a wave's tile
constexpr int kMinTiles = 4;               // tiles a workgroup takes at least: one a wave
constexpr int kNoWindow = 1 << 30;
constexpr float kSlack = 8.f;

// r2o_paged_attention_params in the kernels' widths (the host has checked that they fit): fewer scalar registers.
struct AttentionArgs {
    uint16_t *key, *value;
    float* weight;
    const int32_t *table, *lengths;
    const uint16_t *query, *new_key, *new_value;
    uint16_t* out;
    float *lse, *partial_out, *partial_ml, *logits;
    int k_page, k_head, k_slot, v_page, v_head, v_slot, w_page, w_head, table_stride;
    int q_batch, q_head, nk_batch, nk_head, nv_batch, nv_head;
    int pages, last_page, shift, batch, hkv, group, window, sinks, workers, weight_blocks;
    float c2;  // scale, in log2 units
};

// A kernel's arguments where the hardware put them.  Each place that asks anew loads what it uses again, instead of
// holding 60 words in scalar registers from the first use to the last, which spills.
typedef const __attribute__((address_space(4))) AttentionArgs Args;

__device__ __forceinline__ Args& kernel_args() {
    auto p = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}

template <int RF>
__device__ __forceinline__ r2o_f4 mfma16(r2o_u4 a, r2o_u4 b, r2o_f4 c) {
    return RF == 0 ? r2o_mfma_bf16(a, b, c) : r2o_mfma_f16(a, b, c);
}

template <int RF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return RF == 0 ? r2o_pack_bf2(lo, hi) : r2o_pack_h2(lo, hi);
}

// The visible tiles of one request: those of its sinks, then those of its window.
struct Tiles {
    int n, lo, sink_tiles, first, count;  // filled slots, first slot of the window
    __device__ __forceinline__ int slot(int t) const { return (t < sink_tiles ? t : first + t - sink_tiles) * kSlots; }
    __device__ __forceinline__ bool sees(int j, int sinks) const { return j < n && (j >= lo || j < sinks); }
};

__device__ __forceinline__ Tiles tiles_of(Args& a, int length) {
    Tiles t;
    t.n = min(max(length, 0), (a.last_page + 1) << a.shift);
    t.lo = max(0, t.n - a.window);
    t.first = t.lo / kSlots;
    t.sink_tiles = min((a.sinks + kSlots - 1) / kSlots, t.first);
    t.count = t.sink_tiles + (t.n + kSlots - 1) / kSlots - t.first;
    return t;
}

// The tiles of all (request, head) pairs, in order, shared evenly: worker i takes `each` tiles from begin(i) on, the
// first `more` workers one more.  The partial state of worker i for pair q lies in slot i + q: along the list of
// (worker, pair) one of the two grows by one at a time, so the slots differ.
struct Share {
    int total, workers, each, more;
    __device__ __forceinline__ int begin(int i) const { return i * each + min(i, more); }
    __device__ __forceinline__ int worker(int at) const {  // the one that takes tile `at`, or the last tile
        const int u = min(at, total - 1);
        const int wide = more * (each + 1);
        return u < wide ? (int)((uint32_t)u / (uint32_t)(each + 1)) : more + (int)((uint32_t)(u - wide) / (uint32_t)each);
    }
};

// The wave goes through the batch 64 requests at a time: this lane's request's tiles, and the sum of those up to it.
struct Lane {
    int count, upto;
};

__device__ __forceinline__ Lane lane_tiles(Args& a, int b0) {
    const int lane = threadIdx.x & 63, b = b0 + lane;
    Lane x;
    x.count = b < a.batch ? tiles_of(a, r2o_ldg(a.lengths + b)).count : 0;
    x.upto = wave_scan(x.count);
    return x;
}

__device__ __forceinline__ Share make_share(Args& a) {
    int total = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) total += __builtin_amdgcn_readlane(lane_tiles(a, b0).upto, 63);
    Share s;
    s.total = total * a.hkv;
    s.workers = max(1, min(a.workers, (s.total + kMinTiles - 1) / kMinTiles));
    s.each = (int)((uint32_t)s.total / (uint32_t)s.workers);
    s.more = s.total - s.each * s.workers;
    return s;
}

// The request that holds tile u, and the tiles before it; `batch` if lengths that change meanwhile leave none.
__device__ __forceinline__ int request_of(Args& a, int u, int& before) {
    before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const Lane x = lane_tiles(a, b0);
        const int all = __builtin_amdgcn_readlane(x.upto, 63) * a.hkv;
        if (u < before + all) {
            const int at = __builtin_ctzll(__ballot(before + x.upto * a.hkv > u));
            before += __builtin_amdgcn_readlane(x.upto - x.count, at) * a.hkv;
            return b0 + at;
        }
        before += all;
    }
    return a.batch;
}

// The tiles of the requests before b.
__device__ __forceinline__ int tiles_before(Args& a, int b) {
    int before = 0;
    for (int b0 = 0; b0 <= b; b0 += 64) {
        const Lane x = lane_tiles(a, b0);
        before += b - b0 < 64 ? __builtin_amdgcn_readlane(x.upto - x.count, b - b0) : __builtin_amdgcn_readlane(x.upto, 63);
    }
    return before * a.hkv;
}

// Nontemporal: each row is read once a call.  The ragged decode of 252 MB takes 76 us with plain loads, 68 so.
__device__ __forceinline__ void load_lds16(const void* gsrc, unsigned char* lds) {
    constexpr int kNT = 2;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)gsrc,
                                     (__attribute__((address_space(3))) void*)lds, 16, 0, kNT);
}

constexpr int vmcnt_imm(int n) { return (n & 0xF) | ((n >> 4) << 14) | (0x7 << 4) | (0xF << 8); }

// The pages of a tile's two halves; -1 for one outside the pool.
__device__ __forceinline__ void tile_pages(Args& a, const int32_t* table, int j0, int (&page)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int id = load_uniform(table + min((j0 + 16 * k) >> a.shift, a.last_page));
        page[k] = (uint32_t)id < (uint32_t)a.pages ? id : -1;
    }
}

// One tile of a (request, head): its page ids and the place of its slots in LDS.  A wave's stage holds 32 K rows, then
// 32 V rows, each row 16 chunks of 16 bytes: K row r's chunk c at place c ^ (r & 15), for reads of one chunk by 16 rows;
// V row r's at c ^ 2 (r & 7), for transposing reads of two chunks by eight rows: LDS answers 256 bytes a clock where they
// fall into different banks.
constexpr int kStage = 2 * kSlots * 256;

struct Head {
    const uint16_t *k, *v;   // the head's rows in the pools
    int k_page, v_page;      // strides, elements
    int k_slot, v_slot;
    int shift;
    int k_lane[4], v_lane[2];  // byte offsets of this lane's row and chunk among four rows, by where these lie among 16 (8)
};

// Asynchronous loads of one tile into a stage: 16 of 1 KB, four rows each.
__device__ __forceinline__ void load_tile(const Head& x, int j0, const int (&page)[2], unsigned char* stage) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const int at = (j0 + 16 * m) & ((1 << x.shift) - 1), id = max(page[m], 0);
        const unsigned char* k = reinterpret_cast<const unsigned char*>(x.k + (int64_t)id * x.k_page + (int64_t)at * x.k_slot);
        const unsigned char* v = reinterpret_cast<const unsigned char*>(x.v + (int64_t)id * x.v_page + (int64_t)at * x.v_slot);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            load_lds16(k + (int64_t)(8 * i) * x.k_slot + x.k_lane[i], stage + 4096 * m + 1024 * i);
            load_lds16(v + (int64_t)(8 * i) * x.v_slot + x.v_lane[i & 1], stage + 8192 + 4096 * m + 1024 * i);
        }
    }
}

__device__ __forceinline__ uint32_t lds_address(const unsigned char* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)p;
}

// A stage's K rows l16 and 16 + l16 as A operands: chunks 4 x + g, at `row` + (16 (4 x + g) ^ the row's swizzle).  In
// assembly, with its wait: before a load from LDS that the compiler makes it waits for every asynchronous load into
// LDS, the next tile's among them.
__device__ __forceinline__ void read_keys(uint32_t row, uint32_t chunk, r2o_u4 (&k)[2][4]) {
    const uint32_t a = row + chunk, b = row + (chunk ^ 64), c = row + (chunk ^ 128), e = row + (chunk ^ 192);
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
        "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\tds_read_b128 %6, %10 offset:4096\n\t"
        "ds_read_b128 %7, %11 offset:4096\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(k[1][0]), "=&v"(k[1][1]), "=&v"(k[1][2]), "=&v"(k[1][3])
        : "v"(a), "v"(b), "v"(c), "v"(e)
        : "memory");
}

// V rows 4 g + 0..3 and 16 more, transposed, as the A operands of channels 64 d + 16 x ..
__device__ __forceinline__ void read_values(uint32_t row, uint32_t chunk, int d, r2o_u4 (&v)[4]) {
    const uint32_t at = chunk ^ (128 * d), a = row + at, b = row + (at ^ 32), c = row + (at ^ 64), e = row + (at ^ 96);
    r2o_u2 lo[4], hi[4];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9\n\tds_read_b64_tr_b16 %2, %10\n\tds_read_b64_tr_b16 %3, %11\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:4096\n\tds_read_b64_tr_b16 %5, %9 offset:4096\n\t"
        "ds_read_b64_tr_b16 %6, %10 offset:4096\n\tds_read_b64_tr_b16 %7, %11 offset:4096\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
        : "v"(a), "v"(b), "v"(c), "v"(e)
        : "memory");
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = r2o_u4{lo[x][0], lo[x][1], hi[x][0], hi[x][1]};
}

// One workgroup: its share of the tiles, 4 waves taking a pair's tiles in turn, each with its own softmax state and
// two LDS stages: the next tile's loads go out before this one's products, its page ids one tile earlier still.
// S^T = K Q^T (16 slots x 16 heads a product), O^T += V^T P^T; P^T's operand is the C registers of S^T as they are: the
// slots of a product are summed in that order on both sides.
// Bound by the rows' bytes: a ragged batch of 252 MB takes 51 us, 4.9 TB/s of the 5.9 that a streaming read reaches (52 in
// turn with four other caches, 1.3 GB in all), about 5 of it the first loads and the last join.  One workgroup a compute unit,
// whose LDS it fills: with twice as many, a windowed batch of 251 MB takes 54.3 us instead of 51.2.
// The probabilities are rounded to the rows' 16 bits for the product with V, whose two operands are of one type; their sum
// and the slots' weights take them unrounded.  The results' error against 64 bits is that of their own rounding.
template <int RF, bool WEIGHTS>
__global__ __launch_bounds__(256, 1) void paged_partial_kernel(AttentionArgs) {
    __shared__ __align__(16) unsigned char lds[kWaves][2][kStage];
    __shared__ float ml_lds[kWaves][2][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int worker = blockIdx.x;
    int u, u_end, base, b;
    {
        Args& a = kernel_args();
        const Share share = make_share(a);
        if (worker >= share.workers || share.total == 0) return;
        u = share.begin(worker);
        u_end = share.begin(worker + 1);
        b = request_of(a, u, base);
        if (b >= a.batch) return;
    }
    while (u < u_end) {
        Args& a = kernel_args();
        Tiles t = tiles_of(a, load_uniform(a.lengths + b));
        while (u >= base + t.count * a.hkv) {
            base += t.count * a.hkv;
            if (++b >= a.batch) return;
            t = tiles_of(a, load_uniform(a.lengths + b));
        }
        const int h = (int)((uint32_t)(u - base) / (uint32_t)t.count), pair_base = base + h * t.count;
        const int t0 = u - pair_base, t1 = min(t.count, u_end - pair_base), group = a.group, sinks = min(a.sinks, t.n);
        const int new_slot = a.new_key ? t.n - 1 : -1;
        const float c2 = a.c2;

        r2o_u4 q[4];
        {
            const uint16_t* src = a.query + (int64_t)b * a.q_batch + (int64_t)(h * group + min(l16, group - 1)) * a.q_head + 8 * g;
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = r2o_ldg(reinterpret_cast<const r2o_u4*>(src + 32 * k));
        }
        Head head;
        head.k = a.key + (int64_t)h * a.k_head;
        head.v = a.value + (int64_t)h * a.v_head;
        head.k_page = a.k_page;
        head.v_page = a.v_page;
        head.k_slot = a.k_slot;
        head.v_slot = a.v_slot;
        head.shift = a.shift;
#pragma unroll
        for (int i = 0; i < 4; ++i) head.k_lane[i] = 2 * g * a.k_slot + 16 * (l16 ^ (4 * i + g));
#pragma unroll
        for (int i = 0; i < 2; ++i) head.v_lane[i] = 2 * g * a.v_slot + 16 * (l16 ^ (8 * i + 2 * g));
        const int32_t* table = a.table + (int64_t)b * a.table_stride;
        float* logits = WEIGHTS ? a.logits + (int64_t)pair_base * group * kSlots : nullptr;

        float m = -INFINITY, l = 0.f;
        r2o_f4 acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = r2o_f4{};
        int page[2] = {}, next[2] = {}, after[2] = {};
        int it = t0 + wave;
        if (it < t1) {
            tile_pages(a, table, t.slot(it), page);
            load_tile(head, t.slot(it), page, lds[wave][0]);
            if (it + kWaves < t1) tile_pages(a, table, t.slot(it + kWaves), next);
        }
        for (int buf = 0; it < t1; it += kWaves, buf ^= 1) {
            unsigned char *stage = lds[wave][buf], *other = lds[wave][buf ^ 1];
            const int j0 = t.slot(it);
            if (it + kWaves < t1) {
                load_tile(head, t.slot(it + kWaves), next, other);
                if (it + 2 * kWaves < t1) tile_pages(a, table, t.slot(it + 2 * kWaves), after);
            } else {
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            }
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(16));  // all but the next tile's have landed
            __builtin_amdgcn_wave_barrier();
            unsigned char* vl = stage + 8192;
            const bool has_new = (uint32_t)(new_slot - j0) < (uint32_t)kSlots;
            const bool part = (page[0] | page[1]) < 0 || j0 + kSlots > t.n || (j0 < t.lo && j0 + kSlots > sinks);
            const int lo0 = page[0] < 0 ? 0x7fffffff : t.lo, lo1 = page[1] < 0 ? 0x7fffffff : t.lo;
            const int sink0 = page[0] < 0 ? 0 : sinks, sink1 = page[1] < 0 ? 0 : sinks;
            auto sees = [&](int j, int lo, int sink) { return ((j >= lo) & (j < t.n)) | (j < sink); };
            if (has_new) {  // the appended rows, into the stage and into their page
                Args& e = kernel_args();
                const int r = new_slot - j0, page_new = r < 16 ? page[0] : page[1];
                const int64_t at = new_slot & ((1 << e.shift) - 1);
                const uint16_t* ks = e.new_key + (int64_t)b * e.nk_batch + (int64_t)h * e.nk_head;
                const uint16_t* vs = e.new_value + (int64_t)b * e.nv_batch + (int64_t)h * e.nv_head;
                uint16_t* kd = e.key + (int64_t)h * e.k_head + (int64_t)page_new * e.k_page + at * e.k_slot;
                uint16_t* vd = e.value + (int64_t)h * e.v_head + (int64_t)page_new * e.v_page + at * e.v_slot;
                if (lane < 32) {
                    const r2o_u4 x = r2o_ldg(reinterpret_cast<const r2o_u4*>(lane < 16 ? ks : vs) + l16);
                    *reinterpret_cast<r2o_u4*>(stage + (lane < 16 ? 0 : 8192) + 256 * r + 16 * (l16 ^ (lane < 16 ? r & 15 : 2 * (r & 7)))) = x;
                    if (page_new >= 0) r2o_store8<true>((lane < 16 ? kd : vd) + 8 * l16, x);
                }
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            }
            if (part) {  // V bits of slots that are not seen may be anything: zero
                const int r = lane >> 1;
                if (!sees(j0 + r, r < 16 ? lo0 : lo1, r < 16 ? sink0 : sink1))
#pragma unroll
                    for (int i = 0; i < 8; ++i) reinterpret_cast<r2o_u4*>(vl)[16 * r + 8 * (lane & 1) + i] = r2o_u4{};
            }
            __builtin_amdgcn_wave_barrier();  // LDS operations of a wave stay in order
            r2o_f4 s[2] = {r2o_f4{}, r2o_f4{}};
            {
                r2o_u4 k[2][4];
                read_keys(lds_address(stage) + 256 * l16, 16 * (g ^ l16), k);
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y) s[y] = mfma16<RF>(k[y][x], q[x], s[y]);
            }
            if (part) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + 4 * g + i;
                    s[0][i] = sees(j, lo0, sink0) ? s[0][i] : -INFINITY;
                    s[1][i] = sees(j + 16, lo1, sink1) ? s[1][i] : -INFINITY;
                }
            }
            if (WEIGHTS && l16 < group) {
                float* dst = logits + ((int64_t)it * group + l16) * kSlots + 4 * g;
#pragma unroll
                for (int y = 0; y < 2; ++y) *reinterpret_cast<R2O_GLOBAL r2o_f4*>((R2O_GLOBAL float*)(dst + 16 * y)) = s[y] * c2;
            }
            float tmax = fmaxf(s[0][0], s[1][0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) tmax = fmaxf(tmax, fmaxf(s[0][i], s[1][i]));
            float x, y;
            r2o_row_swap<16>(tmax, x, y);
            tmax = fmaxf(x, y);
            r2o_row_swap<32>(tmax, x, y);
            tmax = fmaxf(x, y) * c2;
            if (__any(tmax > m + kSlack)) {  // of the heads that exceed it alone
                const float m_new = tmax > m + kSlack ? tmax : m;
                const float alpha = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
                l *= alpha;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] *= alpha;
                m = m_new;
            }
            const float ms = m == -INFINITY ? 0.f : m;
            r2o_u4 pk;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][i & 3], c2, -ms));
                const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][(i & 3) + 1], c2, -ms));
                l += e0 + e1;
                pk[i >> 1] = pack2<RF>(e0, e1);
            }
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                r2o_u4 v[4];
                const int r = l16 >> 2;
                read_values(lds_address(vl) + 1024 * g + 256 * r + 8 * (l16 & 1), (16 * ((l16 & 3) >> 1)) ^ (32 * ((4 * g + r) & 7)), d, v);
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[4 * d + x] = mfma16<RF>(v[x], pk, acc[4 * d + x]);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                page[y] = next[y];
                next[y] = after[y];
            }
        }
        {
            float x, y;
            r2o_row_swap<16>(l, x, y);
            l = x + y;
            r2o_row_swap<32>(l, x, y);
            l = x + y;
        }
        // join the waves: lane (l16, g) holds head l16, channels 16 d + 4 g + 0..3
        float* mine = reinterpret_cast<float*>(lds[wave][0]);
#pragma unroll
        for (int d = 0; d < 8; ++d) *reinterpret_cast<r2o_f4*>(mine + l16 * 128 + 16 * d + 4 * g) = acc[d];
        if (g == 0) {
            ml_lds[wave][0][l16] = m;
            ml_lds[wave][1][l16] = l;
        }
        __syncthreads();
        Args& e = kernel_args();
        const int64_t state = ((int64_t)worker + b * e.hkv + h) * group;
        for (int i = threadIdx.x; i < group * 32; i += 256) {
            const int qh = i >> 5, d4 = i & 31;
            float mx = -INFINITY;
#pragma unroll
            for (int x = 0; x < kWaves; ++x) mx = fmaxf(mx, ml_lds[x][0][qh]);
            const float ms = mx == -INFINITY ? 0.f : mx;
            float lt = 0.f;
            r2o_f4 o{};
#pragma unroll
            for (int x = 0; x < kWaves; ++x) {
                const float f = __builtin_amdgcn_exp2f(ml_lds[x][0][qh] - ms);
                lt += f * ml_lds[x][1][qh];
                o += f * *reinterpret_cast<const r2o_f4*>(reinterpret_cast<const float*>(lds[x][0]) + qh * 128 + 4 * d4);
            }
            *reinterpret_cast<r2o_f4*>(e.partial_out + (state + qh) * 128 + 4 * d4) = o;
            if (d4 == 0) {
                e.partial_ml[(state + qh) * 2] = mx;
                e.partial_ml[(state + qh) * 2 + 1] = lt;
            }
        }
        __syncthreads();
        u = pair_base + t1;
    }
}

// The joined maximum and sum of one (pair, head) from its partial states, by a whole wave.
struct Ml {
    float m, l;
};

__device__ __forceinline__ void join_states(float& m, float& l, float m2, float l2) {
    const float mn = fmaxf(m, m2), ms = mn == -INFINITY ? 0.f : mn;
    l = l * __builtin_amdgcn_exp2f(m - ms) + l2 * __builtin_amdgcn_exp2f(m2 - ms);
    m = mn;
}

__device__ __forceinline__ Ml join_ml(const float* ml, int64_t slot0, int count, int group, int head) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < count; i += 64) {
        const float* s = ml + ((slot0 + i) * group + head) * 2;
        join_states(m, l, r2o_ldg(s), r2o_ldg(s + 1));
    }
    join_states(m, l, r2o_lane_xor<1>(m), r2o_lane_xor<1>(l));
    join_states(m, l, r2o_lane_xor<2>(m), r2o_lane_xor<2>(l));
    join_states(m, l, r2o_lane_xor<4>(m), r2o_lane_xor<4>(l));
    join_states(m, l, r2o_lane_xor<8>(m), r2o_lane_xor<8>(l));
    float m2, l2;
    r2o_row_swap<16>(m, m, m2);
    r2o_row_swap<16>(l, l, l2);
    join_states(m, l, m2, l2);
    r2o_row_swap<32>(m, m, m2);
    r2o_row_swap<32>(l, l, l2);
    join_states(m, l, m2, l2);
    return {m, l};
}

// The infinite and NaN values of channels 2 lane and 2 lane + 1 that a request's token sees, added up; 0 where there are
// none.  By one wave, in the tiles of the workers whose products met one (first: the pair's first tile of all, w0 its
// worker, of `count`), 16 rows in flight, till every channel is NaN.
template <int RF>
__device__ __forceinline__ void seen_not_finite(const Tiles& t, const Share& share, int first, int w0, int count, int b, int h, int head, float& x, float& y) {
    Args& a = kernel_args();
    const int lane = threadIdx.x & 63;
    const int32_t* table = a.table + (int64_t)b * a.table_stride;
    const uint16_t* rows = a.value + (int64_t)h * a.v_head + 8 * (lane & 15);
    float sum[8] = {};
    bool more = true;
#pragma unroll 1
    for (int w = w0; w < w0 + count && more; ++w) {
        const float* part = a.partial_out + (((int64_t)w + b * a.hkv + h) * a.group + head) * 128 + 2 * lane;
        if (!__any(!(__builtin_isfinite(r2o_ldg(part)) && __builtin_isfinite(r2o_ldg(part + 1))))) continue;
        const int stop = 2 * (min(share.begin(w + 1), first + t.count) - first);
#pragma unroll 1
        for (int half = 2 * (max(share.begin(w), first) - first); half < stop && more; ++half) {
            r2o_u4 v[4];
            bool seen[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // four rows a load
                const int j = t.slot(half >> 1) + 16 * (half & 1) + 4 * i + (lane >> 4);
                const int page = r2o_ldg(table + min(j >> a.shift, a.last_page));
                seen[i] = t.sees(j, a.sinks) && (uint32_t)page < (uint32_t)a.pages;
                v[i] = r2o_ldg(reinterpret_cast<const r2o_u4*>(rows + (int64_t)(seen[i] ? page : 0) * a.v_page + (int64_t)(j & ((1 << a.shift) - 1)) * a.v_slot));
            }
            bool all_nan = true;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t bits = v[i][k >> 1] >> (16 * (k & 1)) & 0xffffu;
                    const float f = RF == 0 ? r2o_bf16_to_f32(bits) : r2o_f16_to_f32(bits);
                    sum[k] += seen[i] && !__builtin_isfinite(f) ? f : 0.f;
                }
                all_nan &= sum[k] != sum[k];
            }
            more = !__all(all_nan);
        }
    }
    x = y = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        float p, q;
        r2o_row_swap<16>(sum[k], p, q);
        r2o_row_swap<32>(p + q, p, q);
        const float all = __shfl(p + q, lane >> 2);  // chunk lane / 4 holds this lane's channels, its elements 2 (lane % 4) ..
        x = k == 2 * (lane & 3) ? all : x;
        y = k == 2 * (lane & 3) + 1 ? all : y;
    }
}

// Blocks below batch x hq: one (request, query head) each, the partial outputs joined.  Blocks behind them: an even
// share of all tiles each, whose slots' weights grow by their probabilities.  Bound by its launch and its round trips: 5
// us for a call without weights, 10.9 for a ragged batch of 252 MB with them.
template <int RF>
__global__ __launch_bounds__(256) void paged_join_kernel(AttentionArgs) {
    Args& a = kernel_args();
    __shared__ float red[8][128];
    __shared__ float lse2[16];
    const int group = a.group, hkv = a.hkv, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hq = group * hkv;
    const Share share = make_share(a);
    const int heads = a.batch * hq;
    if ((int)blockIdx.x < heads) {
        const int b = blockIdx.x / hq, qh = blockIdx.x % hq, h = qh / group, head = qh % group;
        const int base = tiles_before(a, b);
        const Tiles t = tiles_of(a, load_uniform(a.lengths + b));
        float* lse = a.lse + blockIdx.x;
        uint16_t* dst = a.out + (int64_t)blockIdx.x * 128;
        if (t.count == 0 || share.total == 0) {
            if (threadIdx.x < 64) reinterpret_cast<uint32_t*>(dst)[threadIdx.x] = 0;
            if (threadIdx.x == 0) *lse = -INFINITY;
            return;
        }
        const int u = base + h * t.count, w0 = share.worker(u), count = share.worker(u + t.count - 1) - w0 + 1;
        const int64_t slot0 = (int64_t)w0 + b * hkv + h;
        // the first 32 partial outputs go out with the states that weigh them
        const int row = threadIdx.x >> 5, d4 = threadIdx.x & 31;
        r2o_f4 part[4];
        float part_m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t at = (slot0 + min(row + 8 * k, count - 1)) * group + head;
            part_m[k] = r2o_ldg(a.partial_ml + at * 2);
            part[k] = r2o_ldg(reinterpret_cast<const r2o_f4*>(a.partial_out + at * 128) + d4);
        }
        const Ml ml = join_ml(a.partial_ml, slot0, count, group, head);
        const bool live = !(ml.l == 0.f);  // no slot seen; NaN logits leave m, and a NaN sum
        const float ms = ml.m == -INFINITY ? 0.f : ml.m;
        r2o_f4 o{};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (row + 8 * k < count) o += __builtin_amdgcn_exp2f(part_m[k] - ms) * part[k];
        for (int i = row + 32; i < count; i += 8) {
            const int64_t at = (slot0 + i) * group + head;
            const float f = __builtin_amdgcn_exp2f(r2o_ldg(a.partial_ml + at * 2) - ms);
            o += f * r2o_ldg(reinterpret_cast<const r2o_f4*>(a.partial_out + at * 128) + d4);
        }
        *reinterpret_cast<r2o_f4*>(&red[row][4 * d4]) = o;
        __syncthreads();
        if (threadIdx.x < 64) {
            const float inv = live ? 1.f / ml.l : 0.f;
            float x = 0.f, y = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x += red[i][2 * threadIdx.x];
                y += red[i][2 * threadIdx.x + 1];
            }
            x *= inv;
            y *= inv;
            // A channel is infinite or NaN where a slot that the token sees is, however small that slot's weight: not NaN where
            // the weight is rounded to 0 on its way to a product or a state's factor is 0, which depends on the workers' shares.
            // A NaN sum, of a NaN logit, makes the whole row NaN.
            if (__any(live && ml.l == ml.l && !(__builtin_isfinite(x) && __builtin_isfinite(y)))) {
                float x2, y2;
                seen_not_finite<RF>(t, share, u, w0, count, b, h, head, x2, y2);
                x = __builtin_isfinite(x2) ? x : x2;
                y = __builtin_isfinite(y2) ? y : y2;
            }
            reinterpret_cast<uint32_t*>(dst)[threadIdx.x] = live ? pack2<RF>(x, y) : 0u;
            if (threadIdx.x == 0) *lse = live ? (ml.m + __builtin_amdgcn_logf(ml.l)) * kLn2 : -INFINITY;
        }
        return;
    }
    // weights
    const int block = blockIdx.x - heads;
    int u = (int)((int64_t)share.total * block / a.weight_blocks);
    const int u_end = (int)((int64_t)share.total * (block + 1) / a.weight_blocks);
    if (u >= u_end) return;
    int base;
    int b = request_of(a, u, base);
    if (b >= a.batch) return;
    Tiles t = tiles_of(a, load_uniform(a.lengths + b));
    while (u < u_end) {
        while (u >= base + t.count * hkv) {
            base += t.count * hkv;
            if (++b >= a.batch) return;
            t = tiles_of(a, load_uniform(a.lengths + b));
        }
        const int h = (int)((uint32_t)(u - base) / (uint32_t)t.count), pair_base = base + h * t.count;
        const int stop = min(pair_base + t.count, u_end);
        const int w0 = share.worker(pair_base), count = share.worker(pair_base + t.count - 1) - w0 + 1;
        for (int head = wave; head < group; head += 4) {
            const Ml ml = join_ml(a.partial_ml, (int64_t)w0 + b * hkv + h, count, group, head);
            if (lane == 0) lse2[head] = ml.l == 0.f ? INFINITY : ml.m + __builtin_amdgcn_logf(ml.l);
        }
        __syncthreads();
        const int32_t* table = a.table + (int64_t)b * a.table_stride;
        const int r = threadIdx.x % kSlots;
        for (int tile = u + threadIdx.x / kSlots; tile < stop; tile += 256 / kSlots) {
            const int j = t.slot(tile - pair_base) + r;
            if (!t.sees(j, a.sinks)) continue;
            const int page = r2o_ldg(table + (j >> a.shift));
            if ((uint32_t)page >= (uint32_t)a.pages) continue;
            const float* x = a.logits + (int64_t)tile * group * kSlots + r;
            float sum = 0.f;
            for (int h0 = 0; h0 < group; h0 += 8) {  // eight loads in flight
                float s[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] = r2o_ldg(x + min(h0 + i, group - 1) * kSlots);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += h0 + i < group ? __builtin_amdgcn_exp2f(s[i] - lse2[min(h0 + i, group - 1)]) : 0.f;
            }
            float* w = a.weight + (int64_t)page * a.w_page + (int64_t)h * a.w_head + (j & ((1 << a.shift) - 1));
            *w = a.new_key && j == t.n - 1 ? sum : *w + sum;
        }
        __syncthreads();
        u = stop;
    }
}

// ------------------------------------------------------------------------------------------ evict
constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64, kBins = 4 * kSelectThreads;

// Slots in the order in which they stay, as integers: protected ones, then weights (NaN first, -0 equal to 0), then
// those of no page; 0 behind the filled ones.
constexpr uint32_t kProtected = 0xffffffffu, kNaN = 0xfffffffeu, kNoPage = 1u;

__device__ __forceinline__ uint32_t number_key(float w) {  // -inf: 0x007fffff, inf: 0xff800000, NaN beyond either
    const int u = __float_as_int(w + 0.f);
    return (uint32_t)(u ^ ((u >> 31) | (int)0x80000000));
}

constexpr uint32_t kLeastNumber = 0x007fffffu, kMostNumber = 0xff800000u;

__device__ __forceinline__ uint32_t order_key(float w) { return w != w ? kNaN : number_key(w); }

// Sum over the wave, by moves between lanes through the VALU.
__device__ __forceinline__ int wave_sum(int x) {
    x += __float_as_int(r2o_lane_xor<1>(__int_as_float(x)));
    x += __float_as_int(r2o_lane_xor<2>(__int_as_float(x)));
    x += __float_as_int(r2o_lane_xor<4>(__int_as_float(x)));
    x += __float_as_int(r2o_lane_xor<8>(__int_as_float(x)));
    float a, b;
    r2o_row_swap<16>(__int_as_float(x), a, b);
    x = __float_as_int(a) + __float_as_int(b);
    r2o_row_swap<32>(__int_as_float(x), a, b);
    return __float_as_int(a) + __float_as_int(b);
}

// Least over the wave of unsigned words.
__device__ __forceinline__ uint32_t wave_least(uint32_t x) {
    x = min(x, __float_as_uint(r2o_lane_xor<1>(__uint_as_float(x))));
    x = min(x, __float_as_uint(r2o_lane_xor<2>(__uint_as_float(x))));
    x = min(x, __float_as_uint(r2o_lane_xor<4>(__uint_as_float(x))));
    x = min(x, __float_as_uint(r2o_lane_xor<8>(__uint_as_float(x))));
    float a, b;
    r2o_row_swap<16>(__uint_as_float(x), a, b);
    x = min(__float_as_uint(a), __float_as_uint(b));
    r2o_row_swap<32>(__uint_as_float(x), a, b);
    return min(__float_as_uint(a), __float_as_uint(b));
}

// Of the waves' numbers, one a lane: the sum of those before `wave`, and of all.
__device__ __forceinline__ int waves_before(int x, int wave, int& all) {
    const int upto = wave_scan((threadIdx.x & 63) < kSelectWaves ? x : 0);
    all = __builtin_amdgcn_readlane(upto, kSelectWaves - 1);
    return __builtin_amdgcn_readlane(upto, wave) - __builtin_amdgcn_readlane(x, wave);
}

// One workgroup a (request, head).  A wave holds a run of neighbouring slots as rows of 256, four neighbours a lane, E keys
// a lane in registers (the rows behind are read again when they are needed).  The key of the last slot that stays, the
// largest T that at least `keep` keys reach, is found by counting keys in parts of their range, 4096 a round, at most three
// rounds.  Then every wave knows how many slots before its own stay, and writes its own in order: those above T, and of
// the equal ones the first.  The counts do not depend on the order of their additions.
// Bound by one compute unit's instructions: 8 rows of 65409 slots take 23 us (16 waves a row; loads 1.3 us of it, forming
// the keys 5, three rounds 10, places 6), of 2112 slots 6.6 us.  Rows past 65536 slots are read again in each pass: a call on
// 8 rows of 131072 slots takes 95 us, on 8 of 65409 35.  Comparing all keys with one trial after another, 13 to 20
// times, took 45 us; narrowing by trials and then among 8192 listed ones 43 us.  Rows of one compute unit's registers stay
// within one kernel: counts joined over several would cost a launch, some 4 us, a round.
struct SelectLds {
    int bins[kBins];
    int before[kSelectWaves][2];
    int found[3];
};

template <int E>
__device__ __forceinline__ void select_row(const r2o_paged_evict_params& p, SelectLds& lds, int h, int b, int n) {
    constexpr int kQuads = E / 4;
    int(&bins)[kBins] = lds.bins;
    int(&found)[3] = lds.found;
    int(&before)[kSelectWaves][2] = lds.before;
    const r2o_paged_cache& c = p.source;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), keep = (int)p.keep;
    int32_t* kept = p.kept + (int64_t)blockIdx.x * keep;
    const int quads = max(kQuads, (n + 4 * kSelectThreads - 1) / (4 * kSelectThreads)), first = wave * quads * 256 + 4 * lane;
    const int shift = shift_of(c), mask = (1 << shift) - 1, lo = (int)p.sinks, hi = n - (int)p.recent;  // [lo, hi) may go
    const int32_t* table = c.page_table + b * c.table_stride;
    const float* weights = c.weight_pages + h * c.weight_strides[1];
    const int pages = (int)c.pages, w_page = (int)c.weight_strides[0];
    // four neighbours lie in one page; a quad behind the filled slots reads the last filled one's
    auto page_at = [&](int j) { return r2o_ldg(table + (min(j, n - 1) >> shift)); };
    auto weights_at = [&](int j, int page, float (&w)[4]) {
        const float* src = weights + (int64_t)((uint32_t)page < (uint32_t)pages ? page : 0) * w_page + (min(j, (n - 1) & ~3) & mask);
        typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // slots are unit-strided, rows may start anywhere
        const f4 y = *(const R2O_GLOBAL f4*)src;
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = y[x];
    };
    auto placed = [&](int j, uint32_t k) {  // what a slot's place says over its weight
        k = j < lo || j >= hi ? kProtected : k;
        return j < n ? k : 0u;
    };
    auto quad_at = [&](int j, uint32_t (&k)[4]) {
        float w[4];
        const int page = page_at(j);
        weights_at(j, page, w);
#pragma unroll
        for (int x = 0; x < 4; ++x) k[x] = placed(j + x, (uint32_t)page < (uint32_t)pages ? order_key(w[x]) : kNoPage);
    };
    uint32_t keys[kQuads][4];
    uint32_t most = 0, least = 0xffffffffu;
    int page[kQuads], from = first;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) page[i] = page_at(first + 256 * i);
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
        float w[4];
        weights_at(first + 256 * i, page[i], w);
#pragma unroll
        for (int x = 0; x < 4; ++x) keys[i][x] = __float_as_uint(w[x]);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // what all rows need at once would spill
    }
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
        asm volatile("" : "+v"(from));  // each place forms its slots anew: kept, they would spill
        const int row = wave * quads * 256 + 256 * i;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            keys[i][x] = number_key(__uint_as_float(keys[i][x]));
            asm volatile("" : "+v"(keys[i][x]));  // one key whole before the next
        }
        uint32_t high = max(max(keys[i][0], keys[i][1]), max(keys[i][2], keys[i][3]));
        uint32_t low = min(min(keys[i][0], keys[i][1]), min(keys[i][2], keys[i][3]));
        asm volatile("" : "+v"(page[i]), "+v"(high), "+v"(low));
        const bool mapped = (uint32_t)page[i] < (uint32_t)pages;
        if (row < lo || row + 256 > hi || !__all(mapped && low >= kLeastNumber && high <= kMostNumber)) {
            high = 0;
            low = kProtected;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const bool number = keys[i][x] >= kLeastNumber && keys[i][x] <= kMostNumber;
                keys[i][x] = placed(from + 256 * i + x, !mapped ? kNoPage : number ? keys[i][x] : kNaN);
                high = max(high, keys[i][x] == kProtected ? 0u : keys[i][x]);
                low = min(low, keys[i][x] ? keys[i][x] : kProtected);
            }
        }
        most = max(most, high);
        least = min(least, low);
        asm volatile("" : "+v"(most), "+v"(least));  // now, not when all keys are formed
    }

    auto each = [&](auto&& f) {  // of this thread's keys, four by four
#pragma unroll
        for (int i = 0; i < kQuads; ++i) f(keys[i]);
        for (int i = kQuads; i < quads; ++i) {
            uint32_t k[4];
            quad_at(first + 256 * i, k);
            f(k);
        }
    };
    for (int i = kQuads; i < quads; ++i) {
        uint32_t k[4];
        quad_at(first + 256 * i, k);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            most = max(most, k[x] == kProtected ? 0u : k[x]);
            least = min(least, k[x] ? k[x] : kProtected);
        }
    }
    least = wave_least(least);
    most = ~wave_least(~most);
    if (lane == 0) {
        before[wave][0] = (int)least;
        before[wave][1] = (int)most;
    }
    *reinterpret_cast<int4*>(bins + 4 * tid) = int4{0, 0, 0, 0};
    __syncthreads();
    least = wave_least((uint32_t)before[lane % kSelectWaves][0]);
    most = ~wave_least(~(uint32_t)before[lane % kSelectWaves][1]);
    // The key of the last slot that stays lies in [lo, hi): `reach` keys are at least lo, `keep` or more, and `past` at
    // least hi, fewer.  A round counts the keys above lo in 4096 parts of the range and goes on in the part that holds it.
    // Those equal to lo are not counted but what is left: slots that no query weighs would queue for one counter.
    uint32_t lo_key = (uint32_t)__builtin_amdgcn_readfirstlane((int)least), hi_key = (uint32_t)__builtin_amdgcn_readfirstlane((int)most) + 1;
    int reach = n, past = (int)p.sinks + (int)p.recent;
    if (past == keep) {  // the protected ones alone
        lo_key = kProtected;
        reach = keep;
    }
    while (reach > keep && hi_key - lo_key > 1) {
        const uint32_t span = hi_key - lo_key;
        const int part = max(0, 20 - __builtin_clz(span - 1));  // a part holds 2^part keys
        const uint32_t bottom = lo_key + 1, counted = span - 1;
        __syncthreads();  // the counters are clear, and the waves' words read
        each([&](const uint32_t (&k)[4]) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (k[x] - bottom < counted) atomicAdd(&bins[(k[x] - bottom) >> part], 1);
            __builtin_amdgcn_sched_barrier(0);
        });
        __syncthreads();
        int4* own = reinterpret_cast<int4*>(bins + kBins - 4 - 4 * tid);  // the highest parts are the first thread's
        const int4 c4 = *own;
        *own = int4{0, 0, 0, 0};
        const int upto = wave_scan(c4.x + c4.y + c4.z + c4.w);
        if (lane == 63) before[wave][0] = upto;
        if (tid == 0) found[0] = -1;
        __syncthreads();
        int all;
        int at = past + upto - (c4.x + c4.y + c4.z + c4.w) + waves_before(before[lane % kSelectWaves][0], wave, all);
        all += past;
        const int c[4] = {c4.w, c4.z, c4.y, c4.x};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (at < keep && at + c[x] >= keep) {  // of one thread at most
                found[0] = kBins - 1 - 4 * tid - x;
                found[1] = at;
                found[2] = at + c[x];
            }
            at += c[x];
        }
        __syncthreads();
        const int bin = __builtin_amdgcn_readfirstlane(found[0]);
        if (bin < 0) {  // lo itself
            past = __builtin_amdgcn_readfirstlane(all);
            hi_key = lo_key + 1;
        } else {
            past = __builtin_amdgcn_readfirstlane(found[1]);
            reach = __builtin_amdgcn_readfirstlane(found[2]);
            lo_key = bottom + ((uint32_t)bin << part);
            hi_key = min(hi_key - lo_key, 1u << part) + lo_key;
        }
    }
    __syncthreads();  // the waves' words are read
    uint32_t t = (uint32_t)__builtin_amdgcn_readfirstlane((int)lo_key);
    if (reach == keep) --t;  // all that reach it stay, as those above t - 1
    const uint32_t equal = reach == keep ? 0u : t;  // no key at all, or the key whose first slots fill up
    int sures = 0, equals = 0;
    each([&](const uint32_t (&k)[4]) {
#pragma unroll
        for (int x = 0; x < 4; ++x) sures += k[x] > t ? 1 : 0;
        __builtin_amdgcn_sched_barrier(0);
    });
    if (equal)
        each([&](const uint32_t (&k)[4]) {
#pragma unroll
            for (int x = 0; x < 4; ++x) equals += k[x] == equal ? 1 : 0;
            __builtin_amdgcn_sched_barrier(0);
        });
    sures = wave_sum(sures);
    equals = wave_sum(equals);
    if (lane == 0) {
        before[wave][0] = sures;
        before[wave][1] = equals;
    }
    __syncthreads();
    int sure_all, equal_all;
    int sure_at = waves_before(before[lane % kSelectWaves][0], wave, sure_all);
    int equal_at = waves_before(before[lane % kSelectWaves][1], wave, equal_all);
    const int still = keep - sure_all;  // of the equal ones; 0 where just `keep` reached
    if (still < 0) return;  // rows read again have changed meanwhile: no place is left for the answer
    // values of their own: the comparisons above are made again, not kept
    uint32_t above = (uint32_t)__builtin_amdgcn_readfirstlane((int)t), same = (uint32_t)__builtin_amdgcn_readfirstlane((int)equal);
    asm volatile("" : "+s"(above), "+s"(same), "+v"(from));
    auto write_all = [&](auto ties) {
        auto write = [&](int j, const uint32_t (&k)[4], auto again) {
            int mine = 0;  // sure ones, and equal ones above 16 bits
#pragma unroll
            for (int x = 0; x < 4; ++x) mine += (k[x] > above ? 1 : 0) + (ties && k[x] == same ? 1 << 16 : 0);
            const int upto = wave_scan(mine), all = __builtin_amdgcn_readlane(upto, 63);
            int s = sure_at + ((upto - mine) & 0xffff), e = equal_at + ((upto - mine) >> 16);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const bool sure = k[x] > above, eq = ties && k[x] == same;
                const int to = ties ? s + min(e, still) : s;
                if ((sure || (eq && e < still)) && (!again || to < keep)) kept[to] = j + x;
                s += sure ? 1 : 0;
                e += eq ? 1 : 0;
            }
            sure_at += all & 0xffff;
            equal_at += all >> 16;
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int i = 0; i < kQuads; ++i) write(from + 256 * i, keys[i], std::false_type());
        for (int i = kQuads; i < quads; ++i) {
            uint32_t k[4];
            quad_at(from + 256 * i, k);
            write(from + 256 * i, k, std::true_type());
        }
    };
    if (equal) write_all(std::true_type());
    else write_all(std::false_type());
}

// E: for the longest request that the page table can hold; a shorter one takes as few keys a lane as it needs.
template <int E>
__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(r2o_paged_evict_params p) {
    __shared__ __align__(16) SelectLds lds;
    const r2o_paged_cache& c = p.source;
    const int h = blockIdx.x % (int)c.hkv, b = blockIdx.x / (int)c.hkv, keep = (int)p.keep;
    const int n = __builtin_amdgcn_readfirstlane(filled(c, b));
    if (h == 0 && threadIdx.x == 0) p.target_lengths[b] = min(n, keep);
    if (n <= keep) {
        int32_t* kept = p.kept + (int64_t)blockIdx.x * keep;
        for (int i = threadIdx.x; i < keep; i += kSelectThreads) kept[i] = i < n ? i : -1;
        return;
    }
    if (E == 4 || n <= 4 * kSelectThreads) return select_row<4>(p, lds, h, b, n);
    if (E == 16 || n <= 16 * kSelectThreads) return select_row<16>(p, lds, h, b, n);
    select_row<64>(p, lds, h, b, n);
}

// 16 lanes move one kept slot's K and V row and its weight.  Bound by the rows' bytes: eight requests of 2048 slots and 4
// heads take 13.5 us, 5.0 TB/s read and written, what a large copy reaches.
__global__ __launch_bounds__(256) void paged_compact_kernel(r2o_paged_evict_params p) {
    const r2o_paged_cache &c = p.source, &o = p.target;
    const int h = blockIdx.y, b = blockIdx.z, l16 = threadIdx.x & 15, i = blockIdx.x * 16 + (threadIdx.x >> 4);
    if (i >= (int)p.keep || i >= (int)(o.max_pages * o.page_size)) return;
    const int j = r2o_ldg(p.kept + ((int64_t)b * c.hkv + h) * p.keep + i);
    if ((uint32_t)j >= (uint32_t)(c.max_pages * c.page_size)) return;  // -1 behind the request's length
    const int shift = shift_of(c), to_shift = shift_of(o), at = j & ((1 << shift) - 1), to_at = i & ((1 << to_shift) - 1);
    const int page = page_of(c, b, j, shift), to = page_of(o, b, i, to_shift);
    if (to < 0) return;
    r2o_u4 k{}, v{};
    float w = 0.f;
    if (page >= 0) {
        k = r2o_ldg(reinterpret_cast<const r2o_u4*>(c.key_pages + page * c.key_strides[0] + h * c.key_strides[1] + at * c.key_strides[2]) + l16);
        v = r2o_ldg(reinterpret_cast<const r2o_u4*>(c.value_pages + page * c.value_strides[0] + h * c.value_strides[1] + at * c.value_strides[2]) + l16);
        if (o.weight_pages && l16 == 0) w = r2o_ldg(c.weight_pages + page * c.weight_strides[0] + h * c.weight_strides[1] + at);
    }
    r2o_store8<true>(o.key_pages + to * o.key_strides[0] + h * o.key_strides[1] + to_at * o.key_strides[2] + 8 * l16, k);
    r2o_store8<true>(o.value_pages + to * o.value_strides[0] + h * o.value_strides[1] + to_at * o.value_strides[2] + 8 * l16, v);
    if (o.weight_pages && l16 == 0) o.weight_pages[to * o.weight_strides[0] + h * o.weight_strides[1] + to_at] = w;
}

// ------------------------------------------------------------------------------------ host checks
bool aligned(const void* p, uintptr_t n) { return p && reinterpret_cast<uintptr_t>(p) % n == 0; }

bool rows_ok(const int64_t* st, int n) {  // the kernels hold strides in 32 bits and multiply into 64
    for (int i = 0; i < n; ++i)
        if (st[i] < 0 || st[i] % 8 || st[i] > 0x7fffffff) return false;
    return true;
}

// The extend kernel multiplies in 64 bits: a prompt's requests, heads and rows may lie anywhere.
bool new_rows_ok(const int64_t* st) {
    for (int i = 0; i < 3; ++i)
        if (st[i] < 0 || st[i] % 8) return false;
    return true;
}

// One slot's rows lie within 32-bit offsets of the next ones'.
bool slots_ok(const r2o_paged_cache& c) { return c.key_strides[2] <= R2O_PAGED_MAX_SLOT_STRIDE && c.value_strides[2] <= R2O_PAGED_MAX_SLOT_STRIDE; }

bool cache_ok(const r2o_paged_cache& c) {
    return slots_ok(c) && (c.dtype == 0 || c.dtype == 1) && aligned(c.key_pages, 16) && aligned(c.value_pages, 16) && aligned(c.page_table, 4) &&
           aligned(c.lengths, 4) && reinterpret_cast<uintptr_t>(c.weight_pages) % 4 == 0 && rows_ok(c.key_strides, 3) &&
           rows_ok(c.value_strides, 3) && c.weight_strides[0] >= 0 && c.weight_strides[0] <= 0x7fffffff && c.weight_strides[1] >= 0 &&
           c.weight_strides[1] <= 0x7fffffff && (c.table_stride >= c.max_pages || c.table_stride == 0) && c.table_stride <= 0x7fffffff &&
           c.pages >= 1 && c.pages <= 0x7fffffff && c.max_pages >= 1 && c.batch >= 1 && c.batch <= R2O_PAGED_MAX_BATCH &&
           c.hkv >= 1 && c.hkv <= 1024 &&
           (c.page_size == 16 || c.page_size == 32 || c.page_size == 64 || c.page_size == 128) && c.max_pages <= (1 << 29) / c.page_size;
}

// One row of page ids for all requests: their pages may be read, not written.
bool one_row(const r2o_paged_cache& c) { return c.batch > 1 && c.table_stride == 0; }

}  // namespace

extern "C" {

int r2o_paged_extend(const r2o_paged_extend_params* p, void* stream) {
    if (!p || !cache_ok(p->cache) || one_row(p->cache) || !aligned(p->key, 16) || !aligned(p->value, 16) || !new_rows_ok(p->key_strides) ||
        !new_rows_ok(p->value_strides) || p->rows < 1 || p->rows > (1 << 29) || reinterpret_cast<uintptr_t>(p->counts) % 4 ||
        reinterpret_cast<uintptr_t>(p->weights) % 4 || p->weights_strides[0] < 0 || p->weights_strides[1] < 0 ||
        (p->weights && !p->cache.weight_pages))
        return R2O_EINVAL;
    const dim3 grid((unsigned)((p->rows + 15) / 16), (unsigned)p->cache.hkv, (unsigned)p->cache.batch);
    hipLaunchKernelGGL(paged_extend_kernel, grid, dim3(256), 0, (hipStream_t)stream, *p);
    R2O_CHECK_LAUNCH();
    return R2O_OK;
}

int r2o_paged_attention(const r2o_paged_attention_params* p, void* stream) {
    if (!p || !cache_ok(p->cache)) return R2O_EINVAL;
    const r2o_paged_cache& c = p->cache;
    const int64_t group = p->hq / c.hkv, pairs = c.batch * c.hkv;
    if (p->hq < c.hkv || p->hq % c.hkv || group > R2O_MAX_GQA || !aligned(p->query, 16) || !rows_ok(p->query_strides, 2) ||
        !aligned(p->out, 16) || !aligned(p->lse, 4) || p->window < 0 || p->sinks < 0 || p->sinks > (1 << 29) || !(p->sm_scale > 0.f) ||
        !(p->sm_scale < INFINITY) || p->workers < 1 || p->workers > R2O_PAGED_MAX_WORKERS || !aligned(p->partial_out, 16) ||
        !aligned(p->partial_ml, 8) || p->partial_states < (p->workers + pairs) * group)
        return R2O_EINVAL;
    if ((p->append_key == nullptr) != (p->append_value == nullptr)) return R2O_EINVAL;
    if (one_row(c) && (p->append_key || c.weight_pages)) return R2O_EINVAL;
    if (p->append_key && (!aligned(p->append_key, 16) || !aligned(p->append_value, 16) || !rows_ok(p->append_strides, 4)))
        return R2O_EINVAL;
    // every slot that the page tables can hold has room for its logits, whatever the lengths on the device say
    const int64_t tiles = (c.max_pages * c.page_size + kSlots - 1) / kSlots;
    if (pairs * tiles > 0x7fffffff - R2O_PAGED_MAX_WORKERS) return R2O_EINVAL;
    if (c.weight_pages && (!aligned(p->logits, 16) || p->logits_floats < pairs * tiles * kSlots * group)) return R2O_EINVAL;
    AttentionArgs a{};
    a.key = c.key_pages;
    a.value = c.value_pages;
    a.weight = c.weight_pages;
    a.table = c.page_table;
    a.lengths = c.lengths;
    a.query = p->query;
    a.new_key = p->append_key;
    a.new_value = p->append_value;
    a.out = p->out;
    a.lse = p->lse;
    a.partial_out = p->partial_out;
    a.partial_ml = p->partial_ml;
    a.logits = p->logits;
    a.k_page = (int)c.key_strides[0];
    a.k_head = (int)c.key_strides[1];
    a.k_slot = (int)c.key_strides[2];
    a.v_page = (int)c.value_strides[0];
    a.v_head = (int)c.value_strides[1];
    a.v_slot = (int)c.value_strides[2];
    a.w_page = (int)c.weight_strides[0];
    a.w_head = (int)c.weight_strides[1];
    a.table_stride = (int)c.table_stride;
    a.q_batch = (int)p->query_strides[0];
    a.q_head = (int)p->query_strides[1];
    a.nk_batch = (int)p->append_strides[0];
    a.nk_head = (int)p->append_strides[1];
    a.nv_batch = (int)p->append_strides[2];
    a.nv_head = (int)p->append_strides[3];
    a.pages = (int)c.pages;
    a.last_page = (int)c.max_pages - 1;
    a.shift = 31 - __builtin_clz((unsigned)c.page_size);
    a.batch = (int)c.batch;
    a.hkv = (int)c.hkv;
    a.group = (int)group;
    a.window = p->window ? (int)std::min<int64_t>(p->window, kNoWindow) : kNoWindow;
    a.sinks = p->window ? (int)p->sinks : 0;
    a.workers = (int)p->workers;
    // Short work each, bound by the latency of its loads: the join of a ragged batch of 252 MB takes 15.8 us with one for
    // each worker, 13.1 with two, 11.6 with four, 14.0 with eight.
    a.weight_blocks = 4 * a.workers;
    a.c2 = p->sm_scale * kLog2e;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)p->workers), join((unsigned)(c.batch * p->hq + (c.weight_pages ? a.weight_blocks : 0)));
    auto launch = [&](auto partial, auto join_kernel) {
        hipLaunchKernelGGL(partial, grid, dim3(256), 0, st, a);
        if (hipGetLastError() != hipSuccess) return R2O_ELAUNCH;
        hipLaunchKernelGGL(join_kernel, join, dim3(256), 0, st, a);
        return hipGetLastError() == hipSuccess ? R2O_OK : R2O_ELAUNCH;
    };
    if (c.dtype == 0)
        return c.weight_pages ? launch(paged_partial_kernel<0, true>, paged_join_kernel<0>)
                              : launch(paged_partial_kernel<0, false>, paged_join_kernel<0>);
    return c.weight_pages ? launch(paged_partial_kernel<1, true>, paged_join_kernel<1>)
                          : launch(paged_partial_kernel<1, false>, paged_join_kernel<1>);
}

int r2o_paged_evict(const r2o_paged_evict_params* p, void* stream) {
    if (!p || !cache_ok(p->source) || !cache_ok(p->target)) return R2O_EINVAL;
    const r2o_paged_cache &c = p->source, &o = p->target;
    if (!c.weight_pages || one_row(o) || c.dtype != o.dtype || c.batch != o.batch || c.hkv != o.hkv || p->keep < 1 ||
        p->keep > o.max_pages * o.page_size || p->sinks < 0 || p->recent < 0 || p->sinks > p->keep || p->recent > p->keep - p->sinks ||
        !aligned(p->kept, 4) || !aligned(p->target_lengths, 4) || std::abs(p->target_lengths - c.lengths) < c.batch)
        return R2O_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 rows((unsigned)(c.batch * c.hkv)), threads(kSelectThreads);
    const int64_t most = c.max_pages * c.page_size;  // slots that a lane holds: those of the longest request there can be
    if (most <= 4 * kSelectThreads) hipLaunchKernelGGL(paged_select_kernel<4>, rows, threads, 0, st, *p);
    else if (most <= 16 * kSelectThreads) hipLaunchKernelGGL(paged_select_kernel<16>, rows, threads, 0, st, *p);
    else hipLaunchKernelGGL(paged_select_kernel<64>, rows, threads, 0, st, *p);
    R2O_CHECK_LAUNCH();
    hipLaunchKernelGGL(paged_compact_kernel, dim3((unsigned)((p->keep + 15) / 16), (unsigned)c.hkv, (unsigned)c.batch), dim3(256), 0,
                       st, *p);
    R2O_CHECK_LAUNCH();
    return R2O_OK;
}

}  // extern "C"
