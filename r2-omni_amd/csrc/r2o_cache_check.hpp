// What every entry that takes a paged cache checks of it before a launch.
#pragma once

#include <stdint.h>

#include "r2o_sspa.h"

inline bool r2o_aligned(const void* p, uintptr_t n) { return p && reinterpret_cast<uintptr_t>(p) % n == 0; }

// Element strides as the kernels hold them: multiples of 8, none negative, at most `most`.
inline bool r2o_strides_ok(const int64_t* st, int n, int64_t most) {
    for (int i = 0; i < n; ++i)
        if (st[i] < 0 || st[i] % 8 || st[i] > most) return false;
    return true;
}

// The kernels hold page and head strides in 32 bits and multiply into 64; one slot's rows lie within 32-bit offsets of the
// next ones'.
inline bool r2o_paged_cache_ok(const r2o_paged_cache& c) {
    return (c.dtype == 0 || c.dtype == 1) && r2o_aligned(c.key_pages, 16) && r2o_aligned(c.value_pages, 16) && r2o_aligned(c.page_table, 4) &&
           r2o_aligned(c.lengths, 4) && reinterpret_cast<uintptr_t>(c.weight_pages) % 4 == 0 && r2o_strides_ok(c.key_strides, 3, 0x7fffffff) &&
           r2o_strides_ok(c.value_strides, 3, 0x7fffffff) && c.key_strides[2] <= R2O_PAGED_MAX_SLOT_STRIDE &&
           c.value_strides[2] <= R2O_PAGED_MAX_SLOT_STRIDE && c.weight_strides[0] >= 0 && c.weight_strides[0] <= 0x7fffffff &&
           c.weight_strides[1] >= 0 && c.weight_strides[1] <= 0x7fffffff && (c.table_stride >= c.max_pages || c.table_stride == 0) &&
           c.table_stride <= 0x7fffffff && c.pages >= 1 && c.pages <= 0x7fffffff && c.max_pages >= 1 && c.batch >= 1 &&
           c.batch <= R2O_PAGED_MAX_BATCH && c.hkv >= 1 && c.hkv <= 1024 &&
           (c.page_size == 16 || c.page_size == 32 || c.page_size == 64 || c.page_size == 128) && c.max_pages <= (1 << 29) / c.page_size;
}

// One row of page ids for all requests: their pages may be read, not written.
inline bool r2o_one_row(const r2o_paged_cache& c) { return c.batch > 1 && c.table_stride == 0; }
