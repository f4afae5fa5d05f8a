// Queries and keys rotated by their positions on up to three axes, for gfx950: into tensors, or the keys, with their
// values, into their slots of the paged cache.
//
// Channel pair (i, i + 64) of a token's row turns by the angle a = position[axis of i] * inv_freq[i]:
//     y_i = c x_i - s x_{i+64},  y_{i+64} = c x_{i+64} + s x_i,  c = scaling cos a, s = scaling sin a
// in fp32, with x = w x / sqrt(mean x^2 + eps) before where there are norm weights, and one rounding at the end.
//
// A row (128 channels of one (request, head, token)) is 16 lanes of 8 channels, one 16-byte load and store; a channel's
// partner is lane ^ 8, read by DPP.  A wave takes 4 tokens and walks a run of heads: the 64 angles of a token are formed once
// for all of them, and the rows of four heads, in large calls of sixteen, are in flight at a time.
#include <algorithm>
#include <initializer_list>

#include "r2o_cache_check.hpp"
#include "r2o_common.hpp"

namespace {

struct RotateArgs {
    r2o_rotation rotation;
    const uint16_t *q, *k, *v;
    uint16_t *q_out, *k_out;
    int64_t q_strides[3], k_strides[3], v_strides[3], qo_strides[3], ko_strides[3], weights_strides[2];
    r2o_paged_cache cache;  // of a paged call
    const float* weights;
    const int32_t* counts;
    uint32_t items, tokens;  // items: batch * tokens
    int hq, hkv, heads, heads_per_wave, hadamard;
};

// The position of a token on an axis.
__device__ __forceinline__ int64_t position_at(const r2o_rotation& r, int axis, int64_t b, int64_t token) {
    const int64_t at = axis * r.position_strides[0] + b * r.position_strides[1] + token * r.position_strides[2];
    return r.position_bytes == 8 ? r2o_ldg(reinterpret_cast<const int64_t*>(r.positions) + at)
                                 : (int64_t)r2o_ldg(reinterpret_cast<const int32_t*>(r.positions) + at);
}

// cos and sin of the lane's channels 8 c8 .. 8 c8 + 7, the sine with its channel's sign.  The angle in half turns, position *
// (inv_freq / pi), loses its whole part in 64 bits (a position of 2^31 leaves 2^-22 of one), the rest, at most 1/2, goes to
// the hardware's sine and cosine, which take turns and are off by at most 1.2e-7 (2^-23; looked at for 2^24 arguments).  Polynomials
// instead took 15.3 us where this takes 14.1 (4 padded requests of 1037 rows, 16 + 2 heads).
__device__ __forceinline__ void angles(const r2o_rotation& r, int64_t b, int64_t token, int64_t slot, int c8, float (&c)[8], float (&s)[8]) {
    const int d0 = 8 * (c8 & 7);
    double p0, p1 = 0.0, p2 = 0.0;
    if (r.positions) {
        p0 = (double)position_at(r, 0, b, token);
        if (r.axes > 1) p1 = (double)position_at(r, 1, b, token);
        if (r.axes > 2) p2 = (double)position_at(r, 2, b, token);
    } else {
        p0 = p1 = p2 = (double)slot;
    }
    const uint32_t m1 = (uint32_t)(r.pairs_1 >> d0) & 255u, m2 = (uint32_t)(r.pairs_2 >> d0) & 255u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double f = r.freq_bytes == 8 ? r2o_ldg(reinterpret_cast<const double*>(r.inv_freq) + d0 + i)
                                           : (double)r2o_ldg(reinterpret_cast<const float*>(r.inv_freq) + d0 + i);
        const double p = m1 >> i & 1 ? p1 : (m2 >> i & 1 ? p2 : p0), halves = p * (f * 0.3183098861837907), n = __builtin_rint(halves);
        const float x = 0.5f * (float)(halves - n), sign = __builtin_amdgcn_fract(0.5 * n) != 0.0 ? -r.scaling : r.scaling;
        c[i] = __builtin_amdgcn_cosf(x) * sign;
        s[i] = __builtin_amdgcn_sinf(x) * (c8 < 8 ? -sign : sign);
    }
}

// One row in place; sn carries the sign of its channel.
template <bool NORM>
__device__ __forceinline__ void rotate_row(float (&x)[8], const float (&cs)[8], const float (&sn)[8], const float (&weight)[8], float eps) {
    if constexpr (NORM) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf(x[i], x[i], s);
        s += r2o_lane_xor<8>(s);
        s += r2o_lane_xor<4>(s);
        s += r2o_lane_xor<2>(s);
        s += r2o_lane_xor<1>(s);
        const float inv = __fdiv_rn(1.f, __fsqrt_rn(__builtin_fmaf(s, 1.f / 128.f, eps)));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * weight[i];
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(r2o_lane_xor<8>(x[i]), sn[i], x[i] * cs[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
}

// Rows of a call past what the caches hold (not kThroughCaches) are read and written past them, 16 heads' at a time.  32641 rows of 32 heads take
// 101 us so (5.28 TB/s, as a copy's) and 113 through the caches, four at a time; into pages, 32 + 2 x 8 heads with norms, 153 and
// 189.  With 8 heads at a time 107 and 163, 12: 105 and 154, 24: 104 and 156; with loads alone past the caches 107 and 162, stores
// alone 105 and 157.
// A round of fewer heads loads its last one's rows again in place of the missing ones', without a branch: but not where more than a
// third of a wave's loads would be such (kPastShortRounds), for past the caches they are read again.  100003 rows of 4 heads take 42 us
// so and 62 with them, 32641 of 18 60 and 68, of 20 into pages 66 and 72, 100003 of 24, where a quarter would be, 230 and 227; 32641
// of 48 with norms, where none is, 156 and 153.
enum Caches { kThroughCaches, kPastCaches, kPastShortRounds };

template <Caches CACHES>
constexpr int kHeadsInFlight = CACHES ? 16 : 4;

constexpr bool short_rounds(int64_t heads) {  // of a wave
    const int64_t each = kHeadsInFlight<kPastCaches>, loads = (heads + each - 1) / each * each;
    return 3 * (loads - heads) > loads;
}

template <Caches CACHES>
__device__ __forceinline__ r2o_u4 load_row(const uint16_t* p) {
    if constexpr (CACHES != kThroughCaches) return __builtin_nontemporal_load((const R2O_GLOBAL r2o_u4*)p);
    return r2o_load8<true>(p);
}

template <Caches CACHES>
__device__ __forceinline__ void store_row(uint16_t* p, const r2o_u4& w) {
    if constexpr (CACHES != kThroughCaches) __builtin_nontemporal_store(w, (R2O_GLOBAL r2o_u4*)p);
    else r2o_store8<true>(p, w);
}

// grid (ceil(items / 16), ceil(heads / heads_per_wave)), block 256.  Lanes past the last item work on it again and store
// nothing: the exchanges need every lane of the wave.
template <int DT, bool NORM, bool PAGED, Caches CACHES>
__global__ __launch_bounds__(256) void rotate_by_position_kernel(RotateArgs a) {
    const int lane = threadIdx.x & 63, c8 = lane & 15;
    const uint32_t item = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 4 + (lane >> 4);
    bool live = item < a.items;
    const uint32_t at = live ? item : a.items - 1, b = at / a.tokens, token = at - b * a.tokens;
    // of a paged call: whether the row counts, its slot, and where that lies
    bool counts = true;
    int64_t slot = 0, key_at = -1, value_at = 0, weight_at = 0;
    if constexpr (PAGED) {
        const r2o_paged_cache& c = a.cache;
        const int n = a.counts ? min(max(r2o_ldg(a.counts + b), 0), (int)a.tokens) : (int)a.tokens;
        counts = (int)token < n;
        slot = (int64_t)r2o_ldg(c.lengths + b) - n + token;
        if (live && counts && slot >= 0 && slot < c.max_pages * c.page_size) {
            const int shift = 31 - __builtin_clz((int)c.page_size);
            const int page = r2o_ldg(c.page_table + b * c.table_stride + (slot >> shift));
            if ((uint32_t)page < (uint32_t)c.pages) {
                const int64_t in_page = slot & (c.page_size - 1);
                key_at = page * c.key_strides[0] + in_page * c.key_strides[2] + 8 * c8;
                value_at = page * c.value_strides[0] + in_page * c.value_strides[2] + 8 * c8;
                weight_at = page * c.weight_strides[0] + in_page;
            }
        }
    }
    auto in_head = [&](const int64_t (&st)[3]) { return b * st[0] + token * st[2] + 8 * c8; };
    const int64_t qo0 = in_head(a.qo_strides), ko0 = PAGED ? 0 : in_head(a.ko_strides);
    const int h_end = min(a.heads, (int)(blockIdx.y + 1) * a.heads_per_wave);
    if (PAGED && !__any(live && counts)) {  // of a padded request: zeros
        for (int h = blockIdx.y * a.heads_per_wave; h < min(h_end, a.hq); ++h)
            if (live) r2o_store8<true>(a.q_out + qo0 + h * a.qo_strides[1], r2o_u4{});
        return;
    }
    float cs[8], sn[8], wq[8], wk[8];
    angles(a.rotation, b, token, slot, c8, cs, sn);
    if constexpr (NORM) {
        r2o_unpack8<DT>(r2o_load8<true>(a.rotation.q_weight + 8 * c8), wq);
        r2o_unpack8<DT>(r2o_load8<true>(a.rotation.k_weight + 8 * c8), wk);
    }
    const int64_t q0 = in_head(a.q_strides), k0 = in_head(a.k_strides), v0 = PAGED ? in_head(a.v_strides) : 0;
    for (int h0 = blockIdx.y * a.heads_per_wave; h0 < h_end; h0 += kHeadsInFlight<CACHES>) {
        r2o_u4 raw[kHeadsInFlight<CACHES>];
#pragma unroll
        for (int u = 0; u < kHeadsInFlight<CACHES>; ++u) {  // h is wave-uniform
            if (CACHES == kPastShortRounds && u && h0 + u >= h_end) break;
            const int h = min(h0 + u, h_end - 1);
            if (h < a.hq) raw[u] = load_row<CACHES>(a.q + q0 + h * a.q_strides[1]);
            else if (!PAGED || h < a.hq + a.hkv) raw[u] = load_row<CACHES>(a.k + k0 + (h - a.hq) * a.k_strides[1]);
            else raw[u] = load_row<CACHES>(a.v + v0 + (h - a.hq - a.hkv) * a.v_strides[1]);
        }
#pragma unroll
        for (int u = 0; u < kHeadsInFlight<CACHES>; ++u) {
            const int h = h0 + u;
            if (h >= h_end) break;
            if (PAGED && h >= a.hq + a.hkv) {
                if (key_at >= 0) store_row<CACHES>(a.cache.value_pages + value_at + (h - a.hq - a.hkv) * a.cache.value_strides[1], raw[u]);
                continue;
            }
            float x[8];
            r2o_unpack8<DT>(raw[u], x);
            rotate_row<NORM>(x, cs, sn, h < a.hq ? wq : wk, a.rotation.eps);
            if (!PAGED && a.hadamard) r2o_fwht_row8(x, c8);
            r2o_u4 y = r2o_pack8<DT>(x);
            if (h < a.hq) {
                if (PAGED && !counts) y = r2o_u4{};
                if (live) store_row<CACHES>(a.q_out + qo0 + h * a.qo_strides[1], y);
            } else if constexpr (PAGED) {
                const int64_t kv = h - a.hq;
                if (key_at >= 0) {
                    store_row<CACHES>(a.cache.key_pages + key_at + kv * a.cache.key_strides[1], y);
                    if (a.cache.weight_pages && c8 == 0)
                        a.cache.weight_pages[weight_at + kv * a.cache.weight_strides[1]] =
                            a.weights ? r2o_ldg(a.weights + b * a.weights_strides[0] + kv * a.weights_strides[1] + token) : 0.f;
                }
            } else if (live) {
                store_row<CACHES>(a.k_out + ko0 + (h - a.hq) * a.ko_strides[1], y);
            }
        }
    }
}

// ------------------------------------------------------------------------------------ host checks
bool rows_ok(const void* p, const int64_t (&st)[3]) { return r2o_strides_ok(st, 3, INT64_MAX) && r2o_aligned(p, 16); }

bool rotation_ok(const r2o_rotation& r, bool slots) {
    if (r.axes < 1 || r.axes > 3 || (r.freq_bytes != 4 && r.freq_bytes != 8) || !r2o_aligned(r.inv_freq, r.freq_bytes) || (r.pairs_1 & r.pairs_2) ||
        (r.axes < 2 && r.pairs_1) || (r.axes < 3 && r.pairs_2) || !(r.eps >= 0.f) || !(r.eps < INFINITY) || !(r.scaling > -INFINITY) ||
        !(r.scaling < INFINITY) || (r.q_weight == nullptr) != (r.k_weight == nullptr) || (r.q_weight && (!r2o_aligned(r.q_weight, 16) || !r2o_aligned(r.k_weight, 16))))
        return false;
    if (!r.positions) return slots;
    for (int64_t s : r.position_strides)
        if (s < 0) return false;
    return (r.position_bytes == 4 || r.position_bytes == 8) && r2o_aligned(r.positions, r.position_bytes);
}

// Heads of a wave: all of them share its angles, but a call of few tokens is spread over the chip first.  With kFullWaves waves, 4
// for each SIMD, 4096 rows of 36 heads into their pages take 16.4 us; 19.5 with twice as many, which form the angles twice as often.
constexpr int64_t kFullWaves = 4096;

// Bytes of rows from which on they pass the caches by.  Rows that lie in memory: 16 MB take 13.3 us so and 11.6 through the caches, 33
// MB 18.2 and 19.0, 66 MB 27.4 and 31.6, 197 MB 76 and 85, into pages with norms 49 MB 24.7 and 27.6, 98 MB 44 and 46, 148 MB 61 and
// 73.  Rows that the caches still hold, 45 MB into pages: 22.7 and 19.4, 63 MB: 30.0 and 28.8.
constexpr int64_t kStreamed = (int64_t)1 << 26;

template <bool PAGED, Caches CACHES>
int launch_kernel(const RotateArgs& a, int64_t dtype, dim3 grid, hipStream_t st) {
    const bool norm = a.rotation.q_weight != nullptr;
    if (dtype == 0) {
        if (norm) hipLaunchKernelGGL((rotate_by_position_kernel<0, true, PAGED, CACHES>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((rotate_by_position_kernel<0, false, PAGED, CACHES>), grid, dim3(256), 0, st, a);
    } else {
        if (norm) hipLaunchKernelGGL((rotate_by_position_kernel<1, true, PAGED, CACHES>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((rotate_by_position_kernel<1, false, PAGED, CACHES>), grid, dim3(256), 0, st, a);
    }
    R2O_CHECK_LAUNCH();
    return R2O_OK;
}

template <bool PAGED>
int launch(RotateArgs& a, int64_t dtype, int64_t batch, int64_t tokens, int64_t heads, hipStream_t st) {
    if (heads > 0x7fffffff / 2 || tokens > R2O_POSITION_MAX_TOKENS || batch > R2O_POSITION_MAX_TOKENS / tokens) return R2O_EINVAL;
    const int64_t items = batch * tokens;
    a.items = (uint32_t)items;
    a.tokens = (uint32_t)tokens;
    a.heads = (int)heads;
    const int64_t token_waves = (items + 3) / 4;
    int64_t per = std::max<int64_t>(1, std::min((heads * token_waves + kFullWaves - 1) / kFullWaves, heads));
    per = std::max(per, (heads + 65534) / 65535);  // the grid's second dimension
    a.heads_per_wave = (int)per;
    const dim3 grid((unsigned)((items + 15) / 16), (unsigned)((heads + per - 1) / per));
    if (heads * items <= kStreamed / 256) return launch_kernel<PAGED, kThroughCaches>(a, dtype, grid, st);
    return short_rounds(per) ? launch_kernel<PAGED, kPastShortRounds>(a, dtype, grid, st) : launch_kernel<PAGED, kPastCaches>(a, dtype, grid, st);
}

}  // namespace

extern "C" {

int r2o_position_rope(const r2o_position_rope_params* p, void* stream) {
    if (!p || !rotation_ok(p->rotation, false) || !rows_ok(p->query, p->q_strides) || !rows_ok(p->key, p->k_strides) ||
        !rows_ok(p->query_out, p->qo_strides) || !rows_ok(p->key_out, p->ko_strides) || (p->dtype != 0 && p->dtype != 1) || p->batch < 1 ||
        p->hq < 1 || p->hkv < 1 || p->tokens < 1 || p->hq > 0x3fffffff || p->hkv > 0x3fffffff)
        return R2O_EINVAL;
    RotateArgs a{};
    a.rotation = p->rotation;
    a.q = p->query;
    a.k = p->key;
    a.q_out = p->query_out;
    a.k_out = p->key_out;
    std::copy_n(p->q_strides, 3, a.q_strides);
    std::copy_n(p->k_strides, 3, a.k_strides);
    std::copy_n(p->qo_strides, 3, a.qo_strides);
    std::copy_n(p->ko_strides, 3, a.ko_strides);
    a.hq = (int)p->hq;
    a.hkv = (int)p->hkv;
    a.hadamard = p->hadamard ? 1 : 0;
    return launch<false>(a, p->dtype, p->batch, p->tokens, p->hq + p->hkv, (hipStream_t)stream);
}

int r2o_paged_rope_extend(const r2o_paged_rope_extend_params* p, void* stream) {
    if (!p) return R2O_EINVAL;
    const r2o_paged_cache& c = p->cache;
    if (!r2o_paged_cache_ok(c) || r2o_one_row(c) || !rotation_ok(p->rotation, true) || !rows_ok(p->query, p->q_strides) ||
        !rows_ok(p->key, p->k_strides) || !rows_ok(p->value, p->v_strides) || !rows_ok(p->query_out, p->qo_strides) || p->hq < 1 ||
        p->hq > 0x3fffffff || p->rows < 1 || p->rows > (1 << 29) || reinterpret_cast<uintptr_t>(p->counts) % 4 ||
        reinterpret_cast<uintptr_t>(p->weights) % 4 || p->weights_strides[0] < 0 || p->weights_strides[1] < 0 || (p->weights && !c.weight_pages))
        return R2O_EINVAL;
    RotateArgs a{};
    a.rotation = p->rotation;
    a.cache = c;
    a.q = p->query;
    a.k = p->key;
    a.v = p->value;
    a.q_out = p->query_out;
    a.weights = p->weights;
    a.counts = p->counts;
    std::copy_n(p->q_strides, 3, a.q_strides);
    std::copy_n(p->k_strides, 3, a.k_strides);
    std::copy_n(p->v_strides, 3, a.v_strides);
    std::copy_n(p->qo_strides, 3, a.qo_strides);
    std::copy_n(p->weights_strides, 2, a.weights_strides);
    a.hq = (int)p->hq;
    a.hkv = (int)c.hkv;
    return launch<true>(a, c.dtype, c.batch, p->rows, p->hq + 2 * c.hkv, (hipStream_t)stream);
}

}  // extern "C"
