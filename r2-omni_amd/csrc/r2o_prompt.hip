// Attention of a prompt's rows for gfx950, and the attention weight that each key received.
//
// Row i of a request with q rows and n keys stands at position p = n - q + i.  It sees key j where j <= p and,
// with a window of W, p - j < W or j < sinks.  prompt_attention_kernel:
//     out_i = sum_j softmax_j(c q_i . k_j) v_j,     lse_i = log sum_j exp(c q_i . k_j)
// in one pass over the keys with the running maximum and sum of the softmax.  attention_weights_kernel:
//     w_j = sum over a KV head's query heads and rows of exp(c q_i . k_j - lse_i)
// which needs lse alone, so keys are the outer loop and nothing of size rows x keys is stored.
//
// Both keep the products' operands in the layouts of v_mfma_f32_32x32x16: A holds row m = lane % 32, k = 8
// (lane / 32) + 0..7; B column n = lane % 32, the same k; C column n = lane % 32 and rows 8 (i / 4) + 4 (lane /
// 32) + i % 4 in register i.
#include <algorithm>
#include <initializer_list>

#include "r2o_common.hpp"
#include "r2o_place.hpp"

namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int kRows = 128;      // query rows of a workgroup: 4 waves of 32
constexpr int kTile = 64;       // keys of a tile
constexpr int kTileBytes = kTile * 256;
constexpr int kNoWindow = 1 << 30;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running maximum is raised only when a tile exceeds it by more than this (log2 units): p stays below 2^8
// and most tiles skip the rescaling of 64 accumulators.  Maximum, sum and accumulators refer to one value, so
// the quotient is exact.
constexpr float kSlack = 8.f;

template <int RF>
__device__ __forceinline__ f16v mfma32(r2o_u4 a, r2o_u4 b, f16v c) {
    if constexpr (RF == 0)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(r2o_bf16x8, a), __builtin_bit_cast(r2o_bf16x8, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(r2o_half8, a), __builtin_bit_cast(r2o_half8, b), c,
                                                      0, 0, 0);
}

template <int RF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return RF == 0 ? r2o_pack_bf2(lo, hi) : r2o_pack_h2(lo, hi);
}

// A staged tile's row is 16 chunks of 16 bytes, chunk c of row r at place c ^ swizzle(r).  LDS answers 256 bytes a clock,
// so 16 lanes' 16-byte reads, or 32 lanes' 8-byte ones, have to fall into 256 different ones.  SWZ 0: r & 15, for reads
// of one chunk by 32 rows (4.1 clocks a wave; r & 7 takes 8.1); 1: 4 (r & 3), for transposing reads of four chunks by 4
// rows (3.0 clocks; 2 (r & 3) takes 4.1).  A wave brings 16 rows, four at a time: lane l writes at 16 l, so the swizzle is
// made by which chunk it reads.  This lane's chunk of four rows from r0 on, clamped to `last`:
template <int SWZ>
__device__ __forceinline__ const unsigned char* row_chunk(const uint16_t* base, int stride, int r0, int last, int i, int lane) {
    const int r4 = lane >> 4, place = lane & 15, c = place ^ (SWZ == 0 ? 4 * i + r4 : 4 * r4);
    return reinterpret_cast<const unsigned char*>(base + (int64_t)r0 * stride) + (uint32_t)(2 * min(r4, last - r0) * stride + 16 * c);
}

// Into registers, and from there into LDS.
__device__ __forceinline__ void load_rows(const uint16_t* base, int stride, int row0, int last, r2o_u4 (&x)[4], int wave, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = r2o_ldg(reinterpret_cast<const r2o_u4*>(row_chunk<0>(base, stride, min(row0 + 16 * wave + 4 * i, last), last, i, lane)));
}

__device__ __forceinline__ void store_rows(unsigned char* lds, const r2o_u4 (&x)[4], int wave, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<r2o_u4*>(lds + (16 * wave + 4 * i) * 256 + 16 * lane) = x[i];
}

// 32 rows of a staged tile (SWZ 0) as the A operand of step t (channels 16 t ..).
__device__ __forceinline__ r2o_u4 read_rows(const unsigned char* tile, int block, int t, int lane) {
    const int r = lane & 31, c = 2 * t + (lane >> 5);
    return *reinterpret_cast<const r2o_u4*>(tile + (32 * block + r) * 256 + 16 * (c ^ (r & 15)));
}

// Straight into LDS, asynchronously.
template <int SWZ>
__device__ __forceinline__ void stage_rows(const uint16_t* base, int stride, int row0, int last, unsigned char* lds, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)row_chunk<SWZ>(base, stride, min(row0 + 16 * wave + 4 * i, last), last, i, lane),
            (__attribute__((address_space(3))) void*)(lds + (16 * wave + 4 * i) * 256), 16, 0, 0);
}

__device__ __forceinline__ void wait_staged() { __builtin_amdgcn_s_waitcnt(0xF70); }  // vmcnt(0), the other counters left alone

__device__ __forceinline__ uint32_t lds_address(const unsigned char* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)p;
}

// 32 rows of a staged tile (SWZ 0) as the A operands of all eight steps, in assembly, with its wait: before a load from LDS
// that the compiler makes it waits for every asynchronous load into LDS.
__device__ __forceinline__ void read_all_rows(const unsigned char* tile, int block, int lane, r2o_u4 (&k)[8]) {
    const int r = lane & 31;
    const uint32_t a = lds_address(tile) + (32 * block + r) * 256 + 16 * ((lane >> 5) ^ (r & 15));
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
        "ds_read_b128 %4, %12\n\tds_read_b128 %5, %13\n\tds_read_b128 %6, %14\n\tds_read_b128 %7, %15\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(k[4]), "=&v"(k[5]), "=&v"(k[6]), "=&v"(k[7])
        : "v"(a), "v"(a ^ 32), "v"(a ^ 64), "v"(a ^ 96), "v"(a ^ 128), "v"(a ^ 160), "v"(a ^ 192), "v"(a ^ 224)
        : "memory");
}

// 16 keys from 16 kb on, transposed, as the A operand of channels 32 db ..: lane half h holds keys 4 h + 0..3 and
// 8 + 4 h + 0..3, the order in which the products' C registers hold the probabilities.
__device__ __forceinline__ r2o_u4 read_values(const unsigned char* tile, int kb, int db, int lane) {
    const int i = lane & 15, r = i >> 2;
    const int c = 4 * db + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    const unsigned char* p = tile + (16 * kb + 4 * (lane >> 5) + r) * 256 + 16 * (c ^ (4 * r)) + 8 * (i & 1);
    typedef __attribute__((address_space(3))) s4v lds4;
    const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
    const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 8 * 256));
    const r2o_u2 a = __builtin_bit_cast(r2o_u2, lo), b = __builtin_bit_cast(r2o_u2, hi);
    return r2o_u4{a[0], a[1], b[0], b[1]};
}

__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
    return j <= p && (j > p - window || j < sinks);
}

// The same for key j = first + c by two comparisons, with `back` = p - first and `sink` = min(sinks, p + 1) - 1 - first
// formed once: 0 <= p - j < window, or j at most the last sink.
__device__ __forceinline__ bool sees_from(int back, int sink, int c, uint32_t window) {
    return ((uint32_t)(back - c) < window) | (sink >= c);
}

// Infinite or NaN.
template <int RF>
__device__ __forceinline__ bool not_finite(uint32_t bits16) {
    constexpr uint32_t e = RF == 0 ? 0x7f80u : 0x7c00u;
    return (bits16 & e) == e;
}

template <int RF>
__device__ __forceinline__ bool any_not_finite(r2o_u4 x) {
    bool any = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) any |= not_finite<RF>(x[k]) | not_finite<RF>(x[k] >> 16);
    return any;
}

// A partial output by the factor of its state: infinite and NaN ones stay, where a factor of 0 would make them NaN.
__device__ __forceinline__ float weighed(float x, float f) { return __builtin_isfinite(x) ? x * f : x; }

// In a tile that some row of the workgroup sees in part, a masked key's probability is 0, but 0 times an infinite
// or NaN value is NaN: such elements become zero before any product; true if there was one.
template <int RF>
__device__ __forceinline__ bool zero_not_finite(r2o_u4 (&x)[4]) {
    constexpr uint32_t e = RF == 0 ? 0x7f807f80u : 0x7c007c00u, one = RF == 0 ? 0x00800080u : 0x04000400u;
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t bad = ((x[i][k] & e) + one) & 0x80008000u;  // a full exponent carries into the sign's place
            any |= bad;
            x[i][k] &= ~((bad >> 15) * 0xffffu);
        }
    return any != 0;
}

// The kernels' arguments in their widths (the host has checked that they fit), read where the hardware put them: each
// place that asks anew loads what it uses again, instead of holding them all in scalar registers.
struct PromptArgs {
    const uint16_t *query, *key, *value;
    uint16_t* out;
    float* lse;
    const int32_t *query_lengths, *key_lengths;
    const float* lse_in;
    float *weights, *partial_out, *partial_ml;
    int64_t q_batch, q_head, k_batch, k_head, v_batch, v_head, o_batch, o_head;
    int q_row, k_row, v_row, o_row, batches, hq, hkv, pairs, splits, group, queries, keys, window, sinks;
    float c2;  // scale, in log2 units
};

typedef const __attribute__((address_space(4))) PromptArgs Args;

__device__ __forceinline__ Args& kernel_args() {
    auto p = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}

struct Lengths {
    int q, n, off;  // rows, keys, position of row 0
};

__device__ __forceinline__ Lengths request_lengths(Args& a, int b) {
    Lengths s;
    s.q = a.query_lengths ? min(max(r2o_ldg(a.query_lengths + b), 0), a.queries) : a.queries;
    s.n = a.key_lengths ? min(max(r2o_ldg(a.key_lengths + b), 0), a.keys) : a.keys;
    s.q = __builtin_amdgcn_readfirstlane(s.q);
    s.n = __builtin_amdgcn_readfirstlane(s.n);
    s.off = s.n - s.q;
    return s;
}

// ------------------------------------------------------------------------------ prompt attention
// The rows of a KV head's query heads are one list, packed row r = (row r / group, head r % group): a workgroup's 128
// stand at 128 / group neighbouring positions, so its last tiles are masked in part for few of them, and a chunk of few
// rows fills it.  grid: (row tiles x pairs of request and KV head, splits); with splits each takes a share of the key tiles and
// leaves (maximum, sum, products) in scratch for prompt_join_kernel.
// 16384 rows of 28 heads over 4: 1950 us, 987 TFLOP/s (bf16; a large library product reaches 1270 to 1380); 8192, 5003 and
// 1231 rows of 32 heads with a window of 1024 and four sinks: 366 us (fp16); 257 rows of 16 heads over 4097 keys: 26.5 us in
// 7 splits and 5.2 for the join.  Bound by what runs beside the matrix instructions.  Of 1968 us (one card), it takes without
// its reads of LDS 1810, without the loads into it 1715, without either 1568, without the maximum 1841, without all three
// 1418, without exponentials 1866.  A wave of 64 rows reads half as much from LDS, but its 512 registers leave one wave a
// SIMD: 2693 us; 256 rows a workgroup (8 waves) 1953 against 2009 then, but 386 against 365 for the windowed batch and 39
// against 33 for the 257 rows.  All of a half's V operands read at once, as K's are: 2001 against 1999.
// The probabilities are rounded to the rows' 16 bits, at most half a step each, for the product with V, whose two operands
// are of one type; their sum takes them unrounded.  The results' error against 64 bits is that of their own rounding: 1.7e-3
// (bf16) and 2.1e-4 (fp16), as with probabilities of 32 bits.
template <int RF>
__global__ __launch_bounds__(256, 2) void prompt_attention_kernel(PromptArgs) {
    // K tiles t and t + 1, V tiles t to t + 2: two workgroups fill a compute unit's 160 KB
    __shared__ __align__(16) unsigned char k_lds[2][kTileBytes], v_lds[3][kTileBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    Args& a = kernel_args();
    const int group = a.group, rows = a.queries * group;
    const int row_tiles = (rows + kRows - 1) / kRows, splits = a.splits;
    const R2oPlace at_block = r2o_place(blockIdx.x, row_tiles, splits, a.batches, a.pairs / a.batches);
    if (!at_block.valid) return;
    const int pair = at_block.pair, split = at_block.split;
    const int kvh = pair % a.hkv, b = pair / a.hkv, row0 = (row_tiles - 1 - at_block.tile) * kRows;  // the last rows see most
    const Lengths s = request_lengths(a, b);
    const int window = a.window, sinks = a.sinks;
    const uint16_t* kbase = a.key + b * a.k_batch + kvh * a.k_head;
    const uint16_t* vbase = a.value + b * a.v_batch + kvh * a.v_head;
    const int k_row = a.k_row, v_row = a.v_row;

    const int packed = row0 + 32 * wave + col, row = min(packed, rows - 1) / group, head = min(packed, rows - 1) - row * group;
    r2o_u4 q[8];
    {
        const uint16_t* src = a.query + b * a.q_batch + (kvh * group + head) * a.q_head + (int64_t)row * a.q_row + 8 * half;
#pragma unroll
        for (int t = 0; t < 8; ++t) q[t] = r2o_ldg(reinterpret_cast<const r2o_u4*>(src + 16 * t));
    }

    // positions of the workgroup's rows and of this wave's
    const int wg_first = row0 / group, wg_last = min(row0 + kRows - 1, rows - 1) / group;
    const int wg_min = s.off + wg_first, wg_max = s.off + wg_last;
    const int w0 = min(row0 + 32 * wave, rows - 1), pmin = s.off + w0 / group, pmax = s.off + min(w0 + 31, rows - 1) / group;
    const int p = s.off + row, pv = min(p, s.n - 1);
    // key tiles that any row of the workgroup sees: sink tiles, then the window's
    const int top = min(s.n - 1, wg_max);
    const int first = max(0, wg_min - window + 1) / kTile;
    const int end = wg_first < s.q && top >= 0 ? top / kTile + 1 : 0;
    const int sink_tiles = end ? min((sinks + kTile - 1) / kTile, min(first, end)) : 0;
    const int all = sink_tiles + max(0, end - first);
    const int begin = (int)((int64_t)all * split / splits), tiles = (int)((int64_t)all * (split + 1) / splits);
    const int last = max(s.n - 1, 0);

    const float c2 = a.c2;
    float m = -INFINITY, l = 0.f;
    f16v acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = f16v{};

    auto tile_key = [&](int it) { return (it < sink_tiles ? it : first + it - sink_tiles) * kTile; };
    auto seen_in_part = [&](int kt) { return !(kt + kTile - 1 <= wg_min && (kt > wg_max - window || kt + kTile <= sinks)); };
    // The next tile but one goes straight into LDS while the next one is computed on: K into the buffer that every wave
    // has left behind the last barrier, V into the third one.  The transposing reads that follow wait for it, long after
    // it went out.  16384 rows of 28 heads took 1983 us so, 2057 through registers.
    bool bad = false;
    auto stage = [&](int it, int v_at) {
        stage_rows<0>(kbase, k_row, tile_key(it), last, k_lds[it & 1], wave, lane);
        stage_rows<1>(vbase, v_row, tile_key(it), last, v_lds[v_at], wave, lane);
    };
    // this wave's rows of a staged tile that some row of the workgroup sees in part
    auto clean = [&](int it, int v_at) {
        if (!seen_in_part(tile_key(it))) return;
        r2o_u4* at = reinterpret_cast<r2o_u4*>(v_lds[v_at] + 16 * wave * 256) + lane;
        r2o_u4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = at[64 * i];
        if (zero_not_finite<RF>(x)) {
            bad = true;
#pragma unroll
            for (int i = 0; i < 4; ++i) at[64 * i] = x[i];
        }
    };
    // S^T of 32 keys x 32 rows
    auto products = [&](const unsigned char* kl, int sub) __attribute__((always_inline)) {
        f16v x = f16v{};
        r2o_u4 k[8];
        read_all_rows(kl, sub, lane, k);
#pragma unroll
        for (int t = 0; t < 8; ++t) x = mfma32<RF>(k[t], q[t], x);
        return x;
    };
    // masks, and the running maximum raised where it has to be
    auto top_of = [&](f16v& x, int from_key) __attribute__((always_inline)) {
        if (!(from_key + 31 <= pmin && (from_key > pmax - window || from_key + 32 <= sinks))) {
            const int from = from_key + 4 * half, back = pv - from, sink = min(sinks, pv + 1) - 1 - from;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = sees_from(back, sink, 8 * (i >> 2) + (i & 3), window) ? x[i] : -INFINITY;
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
    // before it.
    if (begin < tiles) {
        stage(begin, 0);
        if (begin + 1 < tiles) stage(begin + 1, 1);
        wait_staged();
        clean(begin, 0);
        __syncthreads();
        f16v even = products(k_lds[begin & 1], 0);
        for (int it = begin, v_at = 0; it < tiles; ++it) {
            const int kt = tile_key(it), v_next = v_at == 2 ? 0 : v_at + 1;
            r2o_u4 pk[2];
            top_of(even, kt);
            f16v odd = products(k_lds[it & 1], 1);
            probabilities(even, pk);
            values(v_lds[v_at], 0, pk);
            top_of(odd, kt + 32);
            wait_staged();
            if (it + 1 < tiles) clean(it + 1, v_next);
            __syncthreads();  // the next tile is there; this one's V stays till every wave is past the next barrier
            even = products(k_lds[(it + 1) & 1], 0);  // behind the last tile: what lies there, not used
            probabilities(odd, pk);
            values(v_lds[v_at], 1, pk);
            if (it + 2 < tiles) stage(it + 2, v_next == 2 ? 0 : v_next + 1);
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
    // A row's channel is infinite or NaN where a key that it sees is, however small that key's weight: not NaN where the
    // weight is rounded to 0 on its way to the product, which depends on the maximum so far.  Those channels are formed
    // again from the values alone: over all tiles where a product has met one, else over those where some were taken out.
    float odd[4] = {};
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int db = 0; db < 4; ++db) odd[db] = __builtin_fmaf(acc[db][i], 0.f, odd[db]);  // NaN where one is not finite
    const float any_odd = odd[0] + odd[1] + odd[2] + odd[3];
    const bool met = __any(any_odd != any_odd && l == l && row < s.q);  // a NaN sum, of a NaN logit, makes the whole row NaN
    if (any_bad || met) {
        f16v extra[4];
#pragma unroll
        for (int db = 0; db < 4; ++db) extra[db] = f16v{};
        bool more = true;  // till every row has NaN alone
        for (int it = begin; it < tiles && more; ++it) {
            const int kt = tile_key(it);
            if (!met && !seen_in_part(kt)) continue;
            for (int j16 = kt; j16 < kt + kTile && more; j16 += 16) {
                r2o_u4 chunk[4];  // of four rows each
                bool any = false;
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    chunk[n] = r2o_ldg(reinterpret_cast<const r2o_u4*>(vbase + (int64_t)min(j16 + 4 * n + (lane >> 4), last) * v_row) + (lane & 15));
#pragma unroll
                for (int n = 0; n < 4; ++n) any |= any_not_finite<RF>(chunk[n]);
                if (!__any(any)) continue;
                for (int j = j16; j < min(j16 + 16, s.n); ++j) {
                    if (!sees(pv, j, window, sinks)) continue;
                    const uint16_t* src = vbase + (int64_t)j * v_row + 4 * half;
#pragma unroll
                    for (int db = 0; db < 4; ++db)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const uint32_t x = r2o_ldg(src + 32 * db + 8 * (i >> 2) + (i & 3));
                            if (not_finite<RF>(x)) extra[db][i] += RF == 0 ? r2o_bf16_to_f32(x) : r2o_f16_to_f32(x);
                        }
                }
                bool all_nan = true;
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) all_nan &= extra[db][i] != extra[db][i];
                more = !__all(all_nan || row >= s.q);
            }
        }
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[db][i] = __builtin_isfinite(extra[db][i]) ? acc[db][i] : extra[db][i];
    }
    if (packed >= rows) return;
    Args& e = kernel_args();
    if (splits > 1) {
        const int64_t at = ((int64_t)split * e.pairs + pair) * rows + packed;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<R2O_GLOBAL r2o_f4*>((R2O_GLOBAL float*)(e.partial_out + at * 128 + 32 * db + 8 * g + 4 * half)) =
                    r2o_f4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
        if (half == 0) {
            e.partial_ml[2 * at] = row < s.q ? m : -INFINITY;
            e.partial_ml[2 * at + 1] = row < s.q ? l : 0.f;
        }
        return;
    }
    const bool live = row < s.q && !(l == 0.f);  // no key seen; NaN logits leave m, and a NaN sum
    const float inv = live ? 1.f / l : 0.f;
    uint16_t* dst = e.out + b * e.o_batch + (kvh * group + head) * e.o_head + (int64_t)row * e.o_row;
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
    if (half == 0)
        e.lse[((int64_t)b * e.hq + kvh * group + head) * e.queries + row] = live ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

// 32 lanes a packed row: its splits' states, joined in order.  Bound by its launch and one round trip to the partial
// states: 257 rows of 16 heads in 7 splits (15 MB) take 5.2 us.
template <int RF>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs, int splits) {
    Args& a = kernel_args();
    const int kvh = (int)blockIdx.y % a.hkv, b = (int)blockIdx.y / a.hkv, group = a.group, rows = a.queries * group;
    const int packed = blockIdx.x * 8 + (threadIdx.x >> 5), d4 = threadIdx.x & 31;
    if (packed >= rows) return;
    const int row = packed / group, head = packed - row * group;
    float m = -INFINITY, l = 0.f;
    r2o_f4 o{};
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
        const int64_t at = ((int64_t)i * gridDim.y + blockIdx.y) * rows + packed;
        const float m2 = r2o_ldg(a.partial_ml + 2 * at), l2 = r2o_ldg(a.partial_ml + 2 * at + 1);
        const r2o_f4 o2 = r2o_ldg(reinterpret_cast<const r2o_f4*>(a.partial_out + at * 128) + d4);
        const float mn = fmaxf(m, m2), ms = mn == -INFINITY ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f(m - ms), f2 = __builtin_amdgcn_exp2f(m2 - ms);
        l = l * f + l2 * f2;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = weighed(o[k], f) + weighed(o2[k], f2);
        m = mn;
    }
    const bool live = !(l == 0.f);
    const float inv = live ? 1.f / l : 0.f;
    r2o_u2 w{};
    if (live) w = r2o_u2{pack2<RF>(o[0] * inv, o[1] * inv), pack2<RF>(o[2] * inv, o[3] * inv)};
    *reinterpret_cast<R2O_GLOBAL r2o_u2*>((R2O_GLOBAL uint16_t*)(a.out + b * a.o_batch + (kvh * group + head) * a.o_head + (int64_t)row * a.o_row + 4 * d4)) = w;
    if (d4 == 0) a.lse[((int64_t)b * a.hq + kvh * group + head) * a.queries + row] = live ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

// ----------------------------------------------------------------------------- attention weights
constexpr int kWeightKeys = 256;  // keys of a workgroup: 4 waves of 64, whose rows stay in registers

// A split takes a share of the (query head, 64-row tile) pairs that see the key tile; its sums go to `weights` ([splits,
// batch, hkv, keys]; the result itself where there is one split).  S = Q K^T: a lane sums its own two keys.  A row tile is two halves of 32; the products of the half that follows run beside the
// exponentials of the one before it.  The sums carry what an addition rounds off along: 8192 terms of very different size.
// Bound by the sum of what each pair needs, no one part of it: 8192 rows of 16 heads over as many keys take 172 us (799
// TFLOP/s of products), without the products 128, without exponentials 153, without their arguments as well 134, without
// the reads of Q from LDS 157, without the load of K 165; with 32 keys a wave, that is twice the reads of Q, 320 against 236
// then.  64 rows of 28 heads over 32641 keys: 30 to 32 us, of which 10.5 are the launch, K's load, the first row tile and the
// sums' way out, 21 the other row tiles; without the products 24.5, without the load of K 28.4.
template <int RF>
__global__ __launch_bounds__(256, 2) void attention_weights_kernel(PromptArgs) {
    __shared__ __align__(16) unsigned char q_lds[2][kTileBytes];
    __shared__ __align__(16) float lse_lds[3][kTile];
    Args& a = kernel_args();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int group = a.group, key_tiles = (a.keys + kWeightKeys - 1) / kWeightKeys;
    const R2oPlace at_block = r2o_place(blockIdx.x, key_tiles, a.splits, 1, a.pairs);
    if (!at_block.valid) return;
    const int pair = at_block.pair, split = at_block.split;
    const int kvh = pair % a.hkv, b = pair / a.hkv, key0 = at_block.tile * kWeightKeys;  // the first keys have most rows
    const Lengths s = request_lengths(a, b);
    const int window = a.window, sinks = a.sinks;
    const int kw = key0 + 64 * wave, j = kw + col;  // this lane's keys: j and j + 32

    // rows that see any of the tile's keys: p >= key0, and without a sink among them p < last key + window
    const int last_key = min(key0 + kWeightKeys, s.n) - 1;
    const int row_lo = max(0, key0 - s.off);
    const int row_hi = key0 < sinks ? s.q : min((int64_t)s.q, (int64_t)last_key + window - s.off);
    const int first = row_lo / kTile, per_head = key0 < s.n ? max(0, (row_hi + kTile - 1) / kTile - first) : 0;
    const int64_t pairs = (int64_t)per_head * group;
    const int begin = (int)(pairs * split / a.splits), end = (int)(pairs * (split + 1) / a.splits);

    float sum[2] = {0.f, 0.f}, lost[2] = {0.f, 0.f};  // of up to hq / hkv * queries terms: what each addition loses is kept
    if (begin < end) {
        const float c2 = a.c2;
        r2o_u4 k[2][8];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint16_t* src = a.key + b * a.k_batch + kvh * a.k_head + (int64_t)min(j + 32 * n, s.n - 1) * a.k_row + 8 * half;
#pragma unroll
            for (int t = 0; t < 8; ++t) k[n][t] = r2o_ldg(reinterpret_cast<const r2o_u4*>(src + 16 * t));
        }
        r2o_u4 qx[4];
        float lse_next = 0.f;
        // the head and row tile of the tile that is loaded next, of the one that is stored and of the one computed on
        int head = begin / per_head, row_tile = begin - head * per_head;
        auto load = [&](int h, int r) {
            lse_next = r2o_ldg(a.lse_in + ((int64_t)b * a.hq + kvh * group + h) * a.queries + min((first + r) * kTile + ((int)threadIdx.x & (kTile - 1)), s.q - 1));
            load_rows(a.query + b * a.q_batch + (kvh * group + h) * a.q_head, a.q_row, (first + r) * kTile, s.q - 1, qx, wave, lane);
        };
        auto store = [&](int r, int q_at, int lse_at) {  // rows behind the request, and those that saw no key, give exp2(-inf)
            store_rows(q_lds[q_at], qx, wave, lane);
            const bool none = (first + r) * kTile + (int)threadIdx.x >= s.q || lse_next == -INFINITY;
            if (threadIdx.x < kTile) lse_lds[lse_at][threadIdx.x] = none ? INFINITY : lse_next * kLog2e;
        };
        auto products = [&](const unsigned char* ql, int rb, f16v (&x)[2]) __attribute__((always_inline)) {
            x[0] = x[1] = f16v{};
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const r2o_u4 q = read_rows(ql, rb, t, lane);
#pragma unroll
                for (int n = 0; n < 2; ++n) x[n] = mfma32<RF>(q, k[n][t], x[n]);
            }
        };
        auto add = [&](const f16v (&x)[2], const float* lse, int p0) __attribute__((always_inline)) {  // p0: position of the half's first row
            const bool full = p0 >= kw + 63 && (kw > p0 + 31 - window || kw + 64 <= sinks);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float part[2] = {0.f, 0.f};
                if (full) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const r2o_f4 y = *reinterpret_cast<const r2o_f4*>(lse + 8 * g + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) part[i & 1] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[n][4 * g + i], c2, -y[i]));
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const r2o_f4 y = *reinterpret_cast<const r2o_f4*>(lse + 8 * g + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[n][4 * g + i], c2, -y[i]));
                            part[i & 1] += sees(p0 + 8 * g + 4 * half + i, j + 32 * n, window, sinks) ? e : 0.f;
                        }
                    }
                }
                const float term = part[0] + part[1] - lost[n], next = sum[n] + term;
                lost[n] = (next - sum[n]) - term;
                sum[n] = next;
            }
        };
        load(head, row_tile);
        store(row_tile, 0, 0);
        __syncthreads();
        f16v even[2], odd[2];
        products(q_lds[0], 0, even);
        for (int it = begin, q_at = 0, lse_at = 0; it < end; ++it, q_at ^= 1) {
            const int p0 = s.off + (first + row_tile) * kTile, lse_to = lse_at == 2 ? 0 : lse_at + 1;
            if (++row_tile == per_head) {
                row_tile = 0;
                ++head;
            }
            if (it + 1 < end) load(head, row_tile);
            products(q_lds[q_at], 1, odd);
            add(even, lse_lds[lse_at], p0);
            if (it + 1 < end) store(row_tile, q_at ^ 1, lse_to);
            __syncthreads();
            products(q_lds[q_at ^ 1], 0, even);  // behind the last tile: what lies there, not used
            add(odd, lse_lds[lse_at] + 32, p0 + 32);
            lse_at = lse_to;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float x, y;
            r2o_row_swap<32>(sum[n], x, y);
            sum[n] = x + y;
        }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
        if (half == n && j + 32 * n < a.keys)
            a.weights[((int64_t)split * a.pairs + pair) * a.keys + j + 32 * n] = j + 32 * n < s.n ? sum[n] : 0.f;
}

__global__ __launch_bounds__(256) void weights_join_kernel(const float* src, float* dst, int64_t n, int splits) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float sum = 0.f;
    for (int k = 0; k < splits; ++k) sum += r2o_ldg(src + k * n + i);
    dst[i] = sum;
}

// Rows lie within 32-bit offsets of the next ones'.
bool strides_ok(const int64_t* st) {
    return st[0] >= 0 && st[1] >= 0 && st[2] >= 0 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0 && st[2] <= R2O_MAX_ROW_STRIDE;
}

bool aligned(std::initializer_list<const void*> ps, uintptr_t n) {
    for (const void* p : ps)
        if (!p || reinterpret_cast<uintptr_t>(p) % n) return false;
    return true;
}

bool shapes_ok(const r2o_prompt_params* p) {
    constexpr int64_t kMost = 1 << 29;
    return p && (p->dtype == 0 || p->dtype == 1) && p->batch >= 1 && p->hkv >= 1 && p->hq >= p->hkv && p->hq % p->hkv == 0 &&
           p->batch * p->hkv <= 65535 && p->batch <= 65535 && p->hq <= 65535 && p->queries >= 1 && p->queries <= kMost &&
           p->keys >= 1 && p->keys <= kMost && p->window >= 0 && p->sinks >= 0 && p->sinks <= kMost && p->sm_scale > 0.f &&
           p->sm_scale < INFINITY && aligned({p->query, p->key}, 16) && strides_ok(p->q_strides) && strides_ok(p->k_strides) &&
           reinterpret_cast<uintptr_t>(p->query_lengths) % 4 == 0 && reinterpret_cast<uintptr_t>(p->key_lengths) % 4 == 0;
}

PromptArgs kernel_arguments(const r2o_prompt_params* p) {
    PromptArgs a{};
    a.query = p->query;
    a.key = p->key;
    a.value = p->value;
    a.out = p->out;
    a.lse = p->lse;
    a.query_lengths = p->query_lengths;
    a.key_lengths = p->key_lengths;
    a.lse_in = p->lse_in;
    a.q_batch = p->q_strides[0];
    a.q_head = p->q_strides[1];
    a.q_row = (int)p->q_strides[2];
    a.k_batch = p->k_strides[0];
    a.k_head = p->k_strides[1];
    a.k_row = (int)p->k_strides[2];
    a.v_batch = p->v_strides[0];
    a.v_head = p->v_strides[1];
    a.v_row = (int)p->v_strides[2];
    a.o_batch = p->o_strides[0];
    a.o_head = p->o_strides[1];
    a.o_row = (int)p->o_strides[2];
    a.hq = (int)p->hq;
    a.hkv = (int)p->hkv;
    a.pairs = (int)(p->batch * p->hkv);
    a.splits = (int)p->splits;
    a.group = (int)(p->hq / p->hkv);
    a.queries = (int)p->queries;
    a.keys = (int)p->keys;
    a.window = p->window ? (int)std::min<int64_t>(p->window, kNoWindow) : kNoWindow;
    a.sinks = p->window ? (int)p->sinks : 0;
    a.c2 = p->sm_scale * kLog2e;
    return a;
}

}  // namespace

extern "C" {

int r2o_prompt_attention(const r2o_prompt_params* p, void* stream) {
    if (!shapes_ok(p) || !aligned({p->value, p->out}, 16) || !aligned({p->lse}, 4) || !strides_ok(p->v_strides) ||
        !strides_ok(p->o_strides))
        return R2O_EINVAL;
    const int64_t rows = p->queries * (p->hq / p->hkv), pairs = p->batch * p->hkv;
    if (rows > (1 << 30) || p->splits < 1 || p->splits > 65535) return R2O_EINVAL;
    if (p->splits > 1 && (!aligned({p->scratch}, 16) || p->scratch_floats < p->splits * pairs * rows * 130)) return R2O_EINVAL;
    // Requests of one length keep their pairs to dies of their own (four of 4096 rows, 16 heads over 2: 292 us, spread 311);
    // of lengths that may differ, each is spread over all dies (8192, 2048, 1024 and 512 rows: 384 us, pinned 1100).
    const int64_t batches = p->query_lengths || p->key_lengths ? p->batch : 1;
    const int64_t blocks = r2o_place_blocks((rows + kRows - 1) / kRows, p->splits, batches, pairs / batches);
    if (blocks > 0x7fffffff) return R2O_EINVAL;
    const dim3 grid((unsigned)blocks);
    const dim3 join((unsigned)((rows + 7) / 8), (unsigned)pairs);
    const hipStream_t st = (hipStream_t)stream;
    PromptArgs a = kernel_arguments(p);
    a.batches = (int)batches;
    a.partial_out = p->scratch;
    a.partial_ml = p->scratch + p->splits * pairs * rows * 128;
    if (p->dtype == 0) hipLaunchKernelGGL(prompt_attention_kernel<0>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(prompt_attention_kernel<1>, grid, dim3(256), 0, st, a);
    R2O_CHECK_LAUNCH();
    if (p->splits > 1) {
        if (p->dtype == 0) hipLaunchKernelGGL(prompt_join_kernel<0>, join, dim3(256), 0, st, a, (int)p->splits);
        else hipLaunchKernelGGL(prompt_join_kernel<1>, join, dim3(256), 0, st, a, (int)p->splits);
        R2O_CHECK_LAUNCH();
    }
    return R2O_OK;
}

int r2o_attention_weights(const r2o_prompt_params* p, void* stream) {
    if (!shapes_ok(p) || !aligned({p->lse_in, p->weights}, 4) || p->splits < 1 || p->splits > 65535) return R2O_EINVAL;
    const int64_t n = p->batch * p->hkv * p->keys;
    if (p->splits > 1 && (!aligned({p->scratch}, 4) || p->scratch_floats < p->splits * n)) return R2O_EINVAL;
    // Pairs keep to dies of their own here, whatever the lengths: 8192 and 1024 rows of 28 heads over 4 take 568 us, spread
    // 563, two requests of 8192 rows 572 and 659.
    const int64_t blocks = r2o_place_blocks((p->keys + kWeightKeys - 1) / kWeightKeys, p->splits, 1, p->batch * p->hkv);
    if ((n + 255) / 256 > 0x7fffffff || blocks > 0x7fffffff) return R2O_EINVAL;
    const dim3 grid((unsigned)blocks);
    const hipStream_t st = (hipStream_t)stream;
    PromptArgs a = kernel_arguments(p);
    a.weights = p->splits > 1 ? p->scratch : p->weights;
    if (p->dtype == 0) hipLaunchKernelGGL(attention_weights_kernel<0>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(attention_weights_kernel<1>, grid, dim3(256), 0, st, a);
    R2O_CHECK_LAUNCH();
    if (p->splits > 1) {
        hipLaunchKernelGGL(weights_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p->scratch, p->weights, n,
                           (int)p->splits);
        R2O_CHECK_LAUNCH();
    }
    return R2O_OK;
}

}  // extern "C"
