/* Kernel argument blocks of the text operators (rotary positions, attention
 * over a paged cache, linears on 4-bit weights), shared by the host runtime
 * and qwen_text_kernels.hip. */
#ifndef QW_TEXT_ARGS_H
#define QW_TEXT_ARGS_H

#include <stdint.h>

/* A paged cache: token t of sequence s lies in page table[s * table_ld +
 * (t >> page_shift)], slot t & (page_size - 1), at ((page * page_size + slot)
 * * kv_heads + head) * head_dim of k and v. */
typedef struct {
    uint16_t *k, *v;
    const uint32_t *table, *lengths, *starts;
    uint32_t pages, page_shift, table_ld, sequences, kv_heads;
} qw_cache_args;

typedef struct {
    uint16_t *q_out, *k_out;
    const uint16_t *q, *k, *v;
    const uint16_t *norm_q, *norm_k; /* [head_dim] or NULL */
    const uint32_t *positions;       /* [rows]; NULL: the place in the sequence */
    const uint32_t *turns;           /* [rotary_dim / 2][2] */
    uint32_t ldq, ldk, ldv, ldq_out, ldk_out;
    uint32_t rows, heads, kv_heads, rotary_dim;
    int32_t half, cached;
    float factor, eps;
    qw_cache_args cache;
} qw_rotary_args;

typedef struct {
    uint16_t *out;
    const uint16_t *q;
    uint32_t ldq, ldo, rows, heads, group; /* group: query heads per K/V head */
    uint32_t window;                       /* 0: none */
    float scale_log2;
    /* the grid: row blocks (an upper bound) x K/V heads x pieces of the keys;
     * piece_tiles: tiles a piece takes (r16, r32), or 0 */
    uint32_t blocks, pieces, piece_tiles;
    float *part;
    uint32_t *flag;
    qw_cache_args cache;
} qw_paged_args;

/* Bytes of LDS for x and scales in the linears of few rows: two workgroups a
 * CU, or one. */
#define QW_L4_FEW 65536
#define QW_L4_WIDE 147456
typedef struct {
    uint16_t *out;
    const uint16_t *in;
    const uint8_t *weight;
    const uint16_t *scales, *zeros, *bias;
    uint32_t rows, k, cols, lda, ldc;
    uint32_t pieces; /* ranges of k that meet in part, counted in flag */
    float *part;
    uint32_t *flag;
} qw_linear4_args;

typedef struct {
    uint8_t *q;
    uint16_t *scales, *zeros; /* zeros NULL: symmetric */
    const uint16_t *in;
    uint32_t rows, cols, group;
} qw_quant4_args;

typedef struct {
    uint16_t *out;
    const uint8_t *q;
    const uint16_t *scales, *zeros;
    uint32_t rows, cols, group;
} qw_dequant4_args;

#endif
