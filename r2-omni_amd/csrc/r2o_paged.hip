// A paged key-value cache for gfx950: rows written into it, attention of one new token over it, and the
// eviction of the tokens that received the least attention.
//
// K and V rows of 128 channels (bf16 or fp16) live in pages of 16, 32, 64 or 128 slots; a request's slot j is slot
// j % size of page page_table[b][j / size], for every KV head.  A page id outside the pool makes its slots
// invisible and keeps every access in bounds.
#include <algorithm>
#include <initializer_list>

#include "r2o_common.hpp"

namespace {

typedef short s4v __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Filled slots of a request, within what its page table can hold.
__device__ __forceinline__ int filled(const r2o_paged_cache& c, int b) {
    return min(max(r2o_ldg(c.lengths + b), 0), (int)(c.max_pages * c.page_size));
}

__device__ __forceinline__ int shift_of(const r2o_paged_cache& c) { return 31 - __builtin_clz((int)c.page_size); }

// The page of a request's slot, or -1.
__device__ __forceinline__ int page_of(const r2o_paged_cache& c, int b, int slot, int shift) {
    const int page = r2o_ldg(c.page_table + b * c.table_stride + (slot >> shift));
    return (uint32_t)page < (uint32_t)c.pages ? page : -1;
}

// ---------------------------------------------------------------------------------------- extend
// 16 lanes move one K and one V row.  Bound by the rows' bytes for a prompt, by the launch for a step.
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
constexpr int kVBytes = kSlots * 256;
constexpr int kMinTiles = 4;               // tiles a workgroup takes at least: one a wave
constexpr float kSlack = 8.f;

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

__device__ __forceinline__ Tiles request_tiles(const r2o_paged_attention_params& p, int b) {
    Tiles t;
    t.n = filled(p.cache, b);
    t.lo = p.window ? max(0, t.n - (int)min(p.window, (int64_t)1 << 30)) : 0;
    t.first = t.lo / kSlots;
    t.sink_tiles = p.window ? min(((int)p.sinks + kSlots - 1) / kSlots, t.first) : 0;
    t.count = t.sink_tiles + (t.n + kSlots - 1) / kSlots - t.first;
    return t;
}

// Sum over the batch of the requests' tiles (one head's), by the whole wave.
__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, R2O_WAVE);
    return x;
}

// How the tiles of all (request, head) pairs, in order, are shared: worker i takes [i total / workers, (i + 1)
// total / workers).  The partial state of worker i for pair q lies in slot i + q: along the list of (worker,
// pair) one of the two grows by one at a time, so the slots differ.
struct Share {
    int64_t total;
    int workers;
    __device__ __forceinline__ int64_t begin(int i) const { return total * i / workers; }
    // the worker that takes tile u
    __device__ __forceinline__ int worker(int64_t u) const {
        int64_t i = u * workers / total;
        while (begin((int)i) > u) --i;
        while (begin((int)i + 1) <= u) ++i;
        return (int)i;
    }
};

__device__ __forceinline__ Share make_share(const r2o_paged_attention_params& p) {
    const int lane = threadIdx.x & 63;
    int64_t total = 0;
    for (int b0 = 0; b0 < (int)p.cache.batch; b0 += 64) {
        const int b = b0 + lane;
        total += wave_sum(b < (int)p.cache.batch ? request_tiles(p, b).count : 0);
    }
    total *= p.cache.hkv;
    Share s;
    s.total = total;
    s.workers = (int)max((int64_t)1, min(p.workers, (total + kMinTiles - 1) / kMinTiles));
    return s;
}

__device__ __forceinline__ void load_lds16(const void* gsrc, unsigned char* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)gsrc,
                                     (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// One workgroup: its share of the tiles, 4 waves taking a pair's tiles in turn.  Per tile of 32 slots a wave loads
// K rows into registers as the A operand of S^T = K Q^T (16 slots x 16 heads a product), V rows into LDS by
// asynchronous loads, from which transposing reads give the A operand of O^T = V^T P^T; P^T's operand is the C
// registers of S^T as they are, the slots of a product being summed in that order on both sides.
template <int RF>
__global__ __launch_bounds__(256, 2) void paged_partial_kernel(r2o_paged_attention_params p) {
    __shared__ __align__(16) unsigned char lds[kWaves][2][kVBytes];
    __shared__ float ml_lds[kWaves][2][16];
    const r2o_paged_cache& c = p.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int group = (int)(p.hq / c.hkv), hkv = (int)c.hkv, shift = shift_of(c);
    const Share share = make_share(p);
    const int worker = blockIdx.x;
    if (worker >= share.workers || share.total == 0) return;
    int64_t u = share.begin(worker);
    const int64_t u_end = share.begin(worker + 1);
    const float c2 = p.sm_scale * kLog2e;
    const int sinks = (int)p.sinks;

    // the request of tile u
    int b = 0;
    int64_t base = 0;
    Tiles t = request_tiles(p, 0);
    while (u >= base + (int64_t)t.count * hkv) {
        base += (int64_t)t.count * hkv;
        t = request_tiles(p, ++b);
    }
    while (u < u_end) {
        while (u >= base + (int64_t)t.count * hkv) {
            base += (int64_t)t.count * hkv;
            t = request_tiles(p, ++b);
        }
        const int h = (int)((u - base) / t.count);
        const int64_t pair_base = base + (int64_t)h * t.count;
        const int t0 = (int)(u - pair_base), t1 = (int)min((int64_t)t.count, u_end - pair_base);

        r2o_u4 q[4];
        {
            const uint16_t* src = p.query + b * p.query_strides[0] + (int64_t)(h * group + min(l16, group - 1)) * p.query_strides[1] + 8 * g;
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = r2o_ldg(reinterpret_cast<const r2o_u4*>(src + 32 * k));
        }
        const uint16_t* kpool = c.key_pages + h * c.key_strides[1];
        const uint16_t* vpool = c.value_pages + h * c.value_strides[1];
        const uint16_t* new_k = p.append_key + b * p.append_strides[0] + h * p.append_strides[1];
        const uint16_t* new_v = p.append_value + b * p.append_strides[2] + h * p.append_strides[3];
        const int new_slot = p.append_key ? t.n - 1 : -1;
        const int32_t* table = c.page_table + b * c.table_stride;
        const int last_page = (int)c.max_pages - 1, in_page = (1 << shift) - 1;
        const int kp = (int)c.key_strides[0], ks = (int)c.key_strides[2], vp0 = (int)c.value_strides[0], vs = (int)c.value_strides[2];

        auto pages_at = [&](int j0, int (&page)[2]) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int id = r2o_ldg(table + min((j0 + 16 * k) >> shift, last_page));
                page[k] = __builtin_amdgcn_readfirstlane((uint32_t)id < (uint32_t)c.pages ? id : -1);
            }
        };
        auto load = [&](int j0, const int (&page)[2], r2o_u4 (&k)[2][4], unsigned char* vl) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int j = j0 + 16 * m + l16;
                const uint16_t* src = kpool + (int64_t)max(page[m], 0) * kp + (int64_t)(j & in_page) * ks;
                if (j == new_slot) src = new_k;
#pragma unroll
                for (int x = 0; x < 4; ++x) k[m][x] = r2o_ldg(reinterpret_cast<const r2o_u4*>(src + 32 * x + 8 * g));
            }
#pragma unroll
            for (int x = 0; x < 8; ++x) {  // 4 rows at a time; chunk cc of row r lies at cc ^ 2 (r & 3)
                const int j = j0 + 4 * x + g, cc = l16 ^ (2 * g);
                const uint16_t* src = vpool + (int64_t)max(page[x >> 2], 0) * vp0 + (int64_t)(j & in_page) * vs;
                if (j == new_slot) src = new_v;
                load_lds16(src + 8 * cc, vl + 1024 * x);
            }
        };

        float m = -INFINITY, l = 0.f;
        r2o_f4 acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = r2o_f4{};
        for (int it = t0 + wave; it < t1; it += kWaves) {
            unsigned char* vl = lds[wave][0];
            const int j0 = t.slot(it);
            int page[2];
            pages_at(j0, page);
            r2o_u4 k[2][4];
            load(j0, page, k, vl);
            r2o_f4 s[2] = {r2o_f4{}, r2o_f4{}};
#pragma unroll
            for (int mm = 0; mm < 2; ++mm)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[mm] = mfma16<RF>(k[mm][x], q[x], s[mm]);
            __builtin_amdgcn_s_waitcnt(0);
            __builtin_amdgcn_wave_barrier();
            const bool full = page[0] >= 0 && page[1] >= 0 && j0 + kSlots <= t.n && (j0 >= t.lo || j0 + kSlots <= sinks);
            if (!full) {
                // rows that are not seen: their logits leave, and their V bits, which may be anything, become zero
#pragma unroll
                for (int mm = 0; mm < 2; ++mm)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (page[mm] < 0 || !t.sees(j0 + 16 * mm + 4 * g + i, sinks)) s[mm][i] = -INFINITY;
                const int r = lane >> 1;
                if ((r < 16 ? page[0] : page[1]) < 0 || !t.sees(j0 + r, sinks))
#pragma unroll
                    for (int i = 0; i < 8; ++i) reinterpret_cast<r2o_u4*>(vl)[16 * r + 8 * (lane & 1) + i] = r2o_u4{};
                __builtin_amdgcn_s_waitcnt(0);
                __builtin_amdgcn_wave_barrier();
            }
            if (new_slot >= j0 && new_slot < j0 + kSlots && lane < 32) {  // the appended rows into their page
                const int page_new = new_slot - j0 < 16 ? page[0] : page[1], at = new_slot & in_page;
                if (page_new >= 0) {
                    const uint16_t* src = lane < 16 ? new_k : new_v;
                    uint16_t* dst = lane < 16 ? c.key_pages + h * c.key_strides[1] + (int64_t)page_new * kp + (int64_t)at * ks
                                              : c.value_pages + h * c.value_strides[1] + (int64_t)page_new * vp0 + (int64_t)at * vs;
                    r2o_store8<true>(dst + 8 * l16, r2o_ldg(reinterpret_cast<const r2o_u4*>(src) + l16));
                }
            }
            if (c.weight_pages && l16 < group) {
                float* dst = p.logits + ((pair_base + it) * group + l16) * kSlots;
#pragma unroll
                for (int mm = 0; mm < 2; ++mm) *reinterpret_cast<r2o_f4*>(dst + 16 * mm + 4 * g) = s[mm] * c2;
            }
            float tmax = s[0][0];
#pragma unroll
            for (int mm = 0; mm < 2; ++mm)
#pragma unroll
                for (int i = 0; i < 4; ++i) tmax = fmaxf(tmax, s[mm][i]);
            float x, y;
            r2o_row_swap<16>(tmax, x, y);
            tmax = fmaxf(x, y);
            r2o_row_swap<32>(tmax, x, y);
            tmax = fmaxf(x, y) * c2;
            if (__any(tmax > m + kSlack)) {
                const float m_new = fmaxf(m, tmax);
                const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
                l *= alpha;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] *= alpha;
                m = m_new;
            }
            const float mm_ = m == -INFINITY ? 0.f : m;
            r2o_u4 pk;
#pragma unroll
            for (int mm = 0; mm < 2; ++mm)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mm][i], c2, -mm_));
                    const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mm][i + 1], c2, -mm_));
                    l += e0 + e1;
                    pk[2 * mm + (i >> 1)] = pack2<RF>(e0, e1);
                }
            typedef __attribute__((address_space(3))) s4v lds4;
            const int r = l16 >> 2;
            const unsigned char* vp = vl + (4 * g + r) * 256 + 8 * (l16 & 1);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                const int cc = (2 * d + ((l16 & 3) >> 1)) ^ (2 * r);
                const r2o_u2 lo = __builtin_bit_cast(r2o_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vp + 16 * cc)));
                const r2o_u2 hi = __builtin_bit_cast(r2o_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vp + 16 * 256 + 16 * cc)));
                acc[d] = mfma16<RF>(r2o_u4{lo[0], lo[1], hi[0], hi[1]}, pk, acc[d]);
            }
            __builtin_amdgcn_s_waitcnt(0);
            __builtin_amdgcn_wave_barrier();
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
        const int64_t slot = (int64_t)worker + (int64_t)b * hkv + h;
        for (int e = threadIdx.x; e < group * 32; e += 256) {
            const int head = e >> 5, d4 = e & 31;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, ml_lds[w][0][head]);
            const float ms = mx == -INFINITY ? 0.f : mx;
            float lt = 0.f;
            r2o_f4 o{};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(ml_lds[w][0][head] - ms);
                lt += f * ml_lds[w][1][head];
                o += f * *reinterpret_cast<const r2o_f4*>(reinterpret_cast<const float*>(lds[w][0]) + head * 128 + 4 * d4);
            }
            *reinterpret_cast<r2o_f4*>(p.partial_out + (slot * group + head) * 128 + 4 * d4) = o;
            if (d4 == 0) {
                p.partial_ml[(slot * group + head) * 2] = mx;
                p.partial_ml[(slot * group + head) * 2 + 1] = lt;
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

__device__ __forceinline__ Ml join_ml(const float* ml, int64_t slot0, int count, int group, int head) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < count; i += 64) {
        const float* s = ml + ((slot0 + i) * group + head) * 2;
        const float m2 = r2o_ldg(s), l2 = r2o_ldg(s + 1);
        const float mn = fmaxf(m, m2), ms = mn == -INFINITY ? 0.f : mn;
        l = l * __builtin_amdgcn_exp2f(m - ms) + l2 * __builtin_amdgcn_exp2f(m2 - ms);
        m = mn;
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float m2 = __shfl_xor(m, x, R2O_WAVE), l2 = __shfl_xor(l, x, R2O_WAVE);
        const float mn = fmaxf(m, m2), ms = mn == -INFINITY ? 0.f : mn;
        l = l * __builtin_amdgcn_exp2f(m - ms) + l2 * __builtin_amdgcn_exp2f(m2 - ms);
        m = mn;
    }
    return {m, l};
}

// Blocks below batch x hq: one (request, query head) each, the partial outputs joined.  Blocks behind them: the
// share of one worker again, whose slots' weights grow by their probabilities.
template <int RF>
__global__ __launch_bounds__(256) void paged_join_kernel(r2o_paged_attention_params p) {
    __shared__ float red[8][128];
    __shared__ float lse2[16];
    const r2o_paged_cache& c = p.cache;
    const int group = (int)(p.hq / c.hkv), hkv = (int)c.hkv, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Share share = make_share(p);
    const int heads = (int)(c.batch * p.hq);
    if ((int)blockIdx.x < heads) {
        const int b = blockIdx.x / (int)p.hq, hq = blockIdx.x % (int)p.hq, h = hq / group, head = hq % group;
        int64_t base = 0;
        for (int i = 0; i < b; ++i) base += (int64_t)request_tiles(p, i).count * hkv;
        const Tiles t = request_tiles(p, b);
        const int64_t u = base + (int64_t)h * t.count;
        float* lse = p.lse + (int64_t)b * p.hq + hq;
        uint16_t* dst = p.out + ((int64_t)b * p.hq + hq) * 128;
        if (t.count == 0) {
            if (threadIdx.x < 64) reinterpret_cast<uint32_t*>(dst)[threadIdx.x] = 0;
            if (threadIdx.x == 0) *lse = -INFINITY;
            return;
        }
        const int w0 = share.worker(u), w1 = share.worker(u + t.count - 1), count = w1 - w0 + 1;
        const int64_t slot0 = (int64_t)w0 + (int64_t)b * hkv + h;
        const Ml ml = join_ml(p.partial_ml, slot0, count, group, head);
        const bool live = ml.m != -INFINITY;
        const float ms = live ? ml.m : 0.f;
        const int row = threadIdx.x >> 5, d4 = threadIdx.x & 31;
        r2o_f4 o{};
        for (int i = row; i < count; i += 8) {
            const int64_t at = (slot0 + i) * group + head;
            const float f = __builtin_amdgcn_exp2f(r2o_ldg(p.partial_ml + at * 2) - ms);
            o += f * r2o_ldg(reinterpret_cast<const r2o_f4*>(p.partial_out + at * 128) + d4);
        }
        *reinterpret_cast<r2o_f4*>(&red[row][4 * d4]) = o;
        __syncthreads();
        if (threadIdx.x < 64) {
            const float inv = live ? 1.f / ml.l : 0.f;
            float a = 0.f, e = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a += red[i][2 * threadIdx.x];
                e += red[i][2 * threadIdx.x + 1];
            }
            reinterpret_cast<uint32_t*>(dst)[threadIdx.x] = live ? pack2<RF>(a * inv, e * inv) : 0u;
            if (threadIdx.x == 0) *lse = live ? (ml.m + __builtin_amdgcn_logf(ml.l)) * kLn2 : -INFINITY;
        }
        return;
    }
    // weights
    const int worker = blockIdx.x - heads, shift = shift_of(c);
    if (worker >= share.workers || share.total == 0) return;
    int64_t u = share.begin(worker);
    const int64_t u_end = share.begin(worker + 1);
    int b = 0;
    int64_t base = 0;
    Tiles t = request_tiles(p, 0);
    while (u < u_end) {
        while (u >= base + (int64_t)t.count * hkv) {
            base += (int64_t)t.count * hkv;
            t = request_tiles(p, ++b);
        }
        const int h = (int)((u - base) / t.count);
        const int64_t pair_base = base + (int64_t)h * t.count;
        const int64_t stop = min(pair_base + t.count, u_end);
        const int w0 = share.worker(pair_base), w1 = share.worker(pair_base + t.count - 1);
        for (int head = wave; head < group; head += 4) {
            const Ml ml = join_ml(p.partial_ml, (int64_t)w0 + (int64_t)b * hkv + h, w1 - w0 + 1, group, head);
            if (lane == 0) lse2[head] = ml.m == -INFINITY ? INFINITY : ml.m + __builtin_amdgcn_logf(ml.l);
        }
        __syncthreads();
        for (int64_t e = u * kSlots + threadIdx.x; e < stop * kSlots; e += 256) {
            const int64_t tile = e / kSlots;
            const int r = (int)(e % kSlots), j = t.slot((int)(tile - pair_base)) + r;
            if (!t.sees(j, (int)p.sinks)) continue;
            const int page = page_of(c, b, j, shift);
            if (page < 0) continue;
            float sum = 0.f;
            for (int head = 0; head < group; ++head)
                sum += __builtin_amdgcn_exp2f(r2o_ldg(p.logits + (tile * group + head) * kSlots + r) - lse2[head]);
            float* w = c.weight_pages + page * c.weight_strides[0] + h * c.weight_strides[1] + (j & ((1 << shift) - 1));
            *w = p.append_key && j == t.n - 1 ? sum : *w + sum;
        }
        __syncthreads();
        u = stop;
    }
}

// ------------------------------------------------------------------------------------------ evict
constexpr int kSelectThreads = 1024;

// A total order of fp32 weights as integers: NaN above everything, -0 equal to 0.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup a (request, head): the weight that the last kept slot has is found digit by digit (8 bits a pass,
// counts in LDS), then the kept slots are written in order: those above it, and of the equal ones the first.
__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(r2o_paged_evict_params p) {
    __shared__ int hist[256];
    __shared__ int scan[kSelectThreads / 64][2];
    __shared__ int found[2];
    const r2o_paged_cache& c = p.source;
    const int h = blockIdx.x % (int)c.hkv, b = blockIdx.x / (int)c.hkv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = filled(c, b), keep = (int)p.keep, shift = shift_of(c), mask = (1 << shift) - 1;
    int32_t* kept = p.kept + (int64_t)blockIdx.x * keep;
    if (h == 0 && tid == 0) p.target_lengths[b] = min(n, keep);
    if (n <= keep) {
        for (int i = tid; i < keep; i += kSelectThreads) kept[i] = i < n ? i : -1;
        return;
    }
    const int lo = (int)p.sinks, hi = n - (int)p.recent;  // what may go
    auto key_at = [&](int j) {
        const int page = page_of(c, b, j, shift);
        return page < 0 ? 0u : order_key(r2o_ldg(c.weight_pages + page * c.weight_strides[0] + h * c.weight_strides[1] + (j & mask)));
    };
    int need = keep - (int)p.sinks - (int)p.recent;  // of [lo, hi)
    uint32_t prefix = 0;
    for (int d = 24; d >= 0; d -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = lo + tid; j < hi; j += kSelectThreads) {
            const uint32_t k = key_at(j);
            if (d == 24 || (k >> (d + 8)) == (prefix >> (d + 8))) atomicAdd(&hist[(k >> d) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {  // the digit with which the count from above first reaches `need`
            int above = 0, x = 255;
            while (x > 0 && above + hist[x] < need) above += hist[x--];
            found[0] = x;
            found[1] = need - above;
        }
        __syncthreads();
        prefix |= (uint32_t)found[0] << d;
        need = found[1];
        __syncthreads();
    }
    // `need` of those equal to prefix stay
    int at = 0, equal = 0;  // kept and equal ones before this chunk
    for (int j0 = 0; j0 < n; j0 += kSelectThreads) {
        const int j = j0 + tid;
        const bool inside = j >= lo && j < hi;
        const uint32_t k = inside ? key_at(j) : 0u;
        const bool eq = inside && k == prefix, sure = j < n && (!inside || k > prefix);
        const uint64_t eq_mask = __ballot(eq), sure_mask = __ballot(sure);
        if (lane == 0) {
            scan[wave][0] = __popcll(eq_mask);
            scan[wave][1] = __popcll(sure_mask);
        }
        __syncthreads();
        int eq_before = equal, sure_before = 0, eq_all = 0, sure_all = 0;
        for (int w = 0; w < kSelectThreads / 64; ++w) {
            if (w < wave) {
                eq_before += scan[w][0];
                sure_before += scan[w][1];
            }
            eq_all += scan[w][0];
            sure_all += scan[w][1];
        }
        const uint64_t below = ((uint64_t)1 << lane) - 1;
        eq_before += __popcll(eq_mask & below);
        sure_before += __popcll(sure_mask & below);
        const int eq_kept_before = min(eq_before, need) - min(equal, need);
        if (sure || (eq && eq_before < need)) kept[at + sure_before + eq_kept_before] = j;
        at += sure_all + min(equal + eq_all, need) - min(equal, need);
        equal += eq_all;
        __syncthreads();
    }
}

// 16 lanes move one kept slot's K and V row and its weight.
__global__ __launch_bounds__(256) void paged_compact_kernel(r2o_paged_evict_params p) {
    const r2o_paged_cache &c = p.source, &o = p.target;
    const int h = blockIdx.y, b = blockIdx.z, l16 = threadIdx.x & 15, i = blockIdx.x * 16 + (threadIdx.x >> 4);
    if (i >= (int)p.keep || i >= (int)(o.max_pages * o.page_size)) return;
    const int j = r2o_ldg(p.kept + ((int64_t)b * c.hkv + h) * p.keep + i);
    if (j < 0) return;
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

bool cache_ok(const r2o_paged_cache& c) {
    return (c.dtype == 0 || c.dtype == 1) && aligned(c.key_pages, 16) && aligned(c.value_pages, 16) && aligned(c.page_table, 4) &&
           aligned(c.lengths, 4) && reinterpret_cast<uintptr_t>(c.weight_pages) % 4 == 0 && rows_ok(c.key_strides, 3) &&
           rows_ok(c.value_strides, 3) && c.weight_strides[0] >= 0 && c.weight_strides[1] >= 0 && c.table_stride >= c.max_pages &&
           c.pages >= 1 && c.pages <= 0x7fffffff && c.max_pages >= 1 && c.batch >= 1 && c.batch <= R2O_PAGED_MAX_BATCH &&
           c.hkv >= 1 && c.hkv <= 1024 &&
           (c.page_size == 16 || c.page_size == 32 || c.page_size == 64 || c.page_size == 128) && c.max_pages <= (1 << 29) / c.page_size;
}

}  // namespace

extern "C" {

int r2o_paged_extend(const r2o_paged_extend_params* p, void* stream) {
    if (!p || !cache_ok(p->cache) || !aligned(p->key, 16) || !aligned(p->value, 16) || !rows_ok(p->key_strides, 3) ||
        !rows_ok(p->value_strides, 3) || p->rows < 1 || p->rows > (1 << 29) || reinterpret_cast<uintptr_t>(p->counts) % 4 ||
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
    if (p->append_key && (!aligned(p->append_key, 16) || !aligned(p->append_value, 16) || !rows_ok(p->append_strides, 4)))
        return R2O_EINVAL;
    // every slot that the page tables can hold has room for its logits, whatever the lengths on the device say
    const int64_t tiles = (c.max_pages * c.page_size + kSlots - 1) / kSlots;
    if (c.weight_pages && (!aligned(p->logits, 16) || p->logits_floats < pairs * tiles * kSlots * group)) return R2O_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)p->workers), join((unsigned)(c.batch * p->hq + (c.weight_pages ? p->workers : 0)));
    if (c.dtype == 0) {
        hipLaunchKernelGGL(paged_partial_kernel<0>, grid, dim3(256), 0, st, *p);
        R2O_CHECK_LAUNCH();
        hipLaunchKernelGGL(paged_join_kernel<0>, join, dim3(256), 0, st, *p);
    } else {
        hipLaunchKernelGGL(paged_partial_kernel<1>, grid, dim3(256), 0, st, *p);
        R2O_CHECK_LAUNCH();
        hipLaunchKernelGGL(paged_join_kernel<1>, join, dim3(256), 0, st, *p);
    }
    R2O_CHECK_LAUNCH();
    return R2O_OK;
}

int r2o_paged_evict(const r2o_paged_evict_params* p, void* stream) {
    if (!p || !cache_ok(p->source) || !cache_ok(p->target)) return R2O_EINVAL;
    const r2o_paged_cache &c = p->source, &o = p->target;
    if (!c.weight_pages || c.dtype != o.dtype || c.batch != o.batch || c.hkv != o.hkv || p->keep < 1 ||
        p->keep > o.max_pages * o.page_size || p->sinks < 0 || p->recent < 0 || p->sinks + p->recent > p->keep ||
        !aligned(p->kept, 4) || !aligned(p->target_lengths, 4) || p->target_lengths == c.lengths)
        return R2O_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)(c.batch * c.hkv)), dim3(kSelectThreads), 0, st, *p);
    R2O_CHECK_LAUNCH();
    hipLaunchKernelGGL(paged_compact_kernel, dim3((unsigned)((p->keep + 15) / 16), (unsigned)c.hkv, (unsigned)c.batch), dim3(256), 0,
                       st, *p);
    R2O_CHECK_LAUNCH();
    return R2O_OK;
}

}  // extern "C"
