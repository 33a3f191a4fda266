/* Where a token's keys lie in a paged cache, with every index that device
 * data gives (starts, lengths, page ids) brought into range: no table makes a
 * kernel touch memory outside the tensors that the host has checked. Plain
 * C++, so that the same functions run in a CPU test. */
#pragma once
#include <stdint.h>

#include "../qw_text_args.h"

#ifdef __HIPCC__
#define QW_HD __host__ __device__ __forceinline__
#else
#define QW_HD static inline
#endif

/* New rows [begin, begin + rows) of a sequence of `length` tokens. */
struct qw_span {
    uint32_t begin, rows, length;
};
QW_HD qw_span qw_cache_span(const qw_cache_args &c, uint32_t s, uint32_t all_rows) {
    const uint64_t room = (uint64_t)c.table_ld << c.page_shift;
    uint32_t b = c.starts[s], e = c.starts[s + 1], n = c.lengths[s];
    b = b < all_rows ? b : all_rows;
    e = e < all_rows ? e : all_rows;
    e = e > b ? e : b;
    return {b, e - b, n < room ? n : (uint32_t)room};
}

/* The place of a new token in its sequence; negative for more new tokens than
 * the sequence is long. */
QW_HD int64_t qw_cache_place(const qw_span &s, uint32_t token) {
    return (int64_t)s.length - s.rows + token;
}

/* Table entry of a token's page (t below the span's length, or clamped). */
QW_HD uint64_t qw_cache_entry(const qw_cache_args &c, uint32_t s, uint32_t t) {
    const uint32_t i = t >> c.page_shift;
    return (uint64_t)s * c.table_ld + (i < c.table_ld ? i : c.table_ld - 1);
}

/* First element of a token's K/V head; only for page < c.pages. */
QW_HD uint64_t qw_cache_at(const qw_cache_args &c, uint32_t page, uint32_t t, uint32_t head,
                           uint32_t head_dim) {
    const uint64_t slot = ((uint64_t)page << c.page_shift) + (t & ((1u << c.page_shift) - 1));
    return (slot * c.kv_heads + head) * head_dim;
}

/* Bytes that a load of `n` consecutive tokens (of one page) of a head may
 * read from the first on, when only tokens below `end` exist: the rest reads
 * as zero. */
QW_HD uint32_t qw_cache_bytes(const qw_cache_args &c, uint32_t t, uint32_t n, uint32_t end,
                              uint32_t head_dim) {
    const uint32_t left = end > t ? end - t : 0, there = left < n ? left : n;
    const uint32_t bytes = (there * c.kv_heads - c.kv_heads + 1) * head_dim * 2;
    return there ? bytes : 0;
}
