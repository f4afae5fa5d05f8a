// Tiles of 64 key and value rows in LDS and the products on them: what the attention kernels that take 32 query rows a
// wave share.
//
// The operands' layouts are those of v_mfma_f32_32x32x16: A holds row m = lane % 32, k = 8 (lane / 32) + 0..7; B column
// n = lane % 32, the same k; C column n = lane % 32 and rows 8 (i / 4) + 4 (lane / 32) + i % 4 in register i.
#pragma once

#include "r2o_common.hpp"

namespace r2o_tiles {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;  // keys of a tile
constexpr int kTileBytes = kTile * 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running maximum is raised only when a tile exceeds it by more than this (log2 units): p stays below 2^8
// and most tiles skip the rescaling of 64 accumulators.  Maximum, sum and accumulators refer to one value, so
// the quotient does not depend on it but by the rounding of p to 16 bits: that of a key which outweighs all others is 1,
// without an error, where the value is its own, and up to 2^8, half a step off, where it is not.  Attention over a prefix,
// bf16, 128 conversations: 1.680e-3 off 64 bits with the slack, 1.670e-3 without, as with p of 32 bits (1.669e-3), but
// 170 us become 183 (questions) and 43 become 47 (24 requests).
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
template <int RF, int N>
__device__ __forceinline__ bool zero_not_finite(r2o_u4 (&x)[N]) {
    constexpr uint32_t e = RF == 0 ? 0x7f807f80u : 0x7c007c00u, one = RF == 0 ? 0x00800080u : 0x04000400u;
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t bad = ((x[i][k] & e) + one) & 0x80008000u;  // a full exponent carries into the sign's place
            any |= bad;
            x[i][k] &= ~((bad >> 15) * 0xffffu);
        }
    return any != 0;
}

}  // namespace r2o_tiles
