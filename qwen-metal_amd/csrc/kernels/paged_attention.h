/* Attention of new tokens over a paged cache, D = 128, grouped K/V heads.
 *
 * Token i of the n new ones of a sequence of `length` has the place p = length
 * - n + i and sees the keys (p - window, p] whose page exists. The rows of one
 * (sequence, K/V head) are its new tokens times the query heads that share
 * the head, row r = token r / group, head r % group, so K and V are read once
 * for the whole group, whatever its size.
 *
 * Two forms. Many rows: blocks of 256 or 128 rows with the loop of the image
 * attention (attention.h: S^T = K Q^T and O^T = V^T P^T on
 * v_mfma_f32_32x32x16_bf16, K and V straight into LDS, QK of the next tile
 * under the softmax), bound by the matrix cores and the softmax's vector work
 * beside them: 32 heads on 8, four prompts of 2324 to 4096 tokens 365 to 390 us
 * by board (0.84 to 0.89 PFLOP/s), 512 tokens at 7937 in 3 pieces 88 us. Few
 * rows (single tokens): 16 or 32 rows on
 * v_mfma_f32_16x16x32_bf16, every wave streaming key tiles of its own through
 * its own part of LDS without a barrier, bound by HBM: 64 users of 4100 to 8192
 * keys 309 us (5.2 TB/s), two of 131000 and 91773 171 us (5.3). One user of
 * 2049 keys takes 10.7 us, an empty launch 3.0 of it, the rest seven latencies
 * one after another: starts, table, keys, the piece's sums, its counter, all
 * pieces' sums, the store.
 *
 * P is rounded to bf16 for its product with V, and its sum is that of the
 * rounded values: the matrix cores have no faster form than bf16 that holds
 * it, and a weighted mean moves by 2^-9 of the mean distance from it.
 *
 * A 1 KB load brings 4 keys, which lie in one page (pages are 8 tokens or
 * more): its base is the page's, in scalar registers, its extent ends at the
 * sequence's last token, so what lies behind it (and all of a page that does
 * not exist) reads as zero, whatever the cache holds there. The base is 64
 * bits wide: a cache may pass 4 GB.
 *
 * What a row must not see gets the score -inf, so P is 0 there; but 0 times an
 * infinity or NaN in V (a key that other rows of the tile do see) would reach
 * the row. Tiles with masked scores therefore look at their V values first,
 * and where one is not finite the products leave it out and what it gives to
 * the rows that see it, an infinity or NaN, is added on the side. */
#pragma once
#include "attention_parts.h"
#include "paged_cache.h"

#define PA_D 128

/* A workgroup's rows: block `blk` of `rows` rows of sequence `seq`. */
struct pa_job {
    uint32_t seq, blk;
    qw_span span;
};
/* The sequence that row block b falls in when each has ceil(rows / BM) of
 * them; all lanes together. False for blocks past the last. */
template <uint32_t BM>
__device__ __forceinline__ bool pa_find(const qw_paged_args &a, uint32_t b, pa_job &job) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t done = 0;
    for (uint32_t s0 = 0; s0 < a.cache.sequences; s0 += 64) {
        uint32_t nb = 0;
        qw_span sp = {0, 0, 0};
        if (s0 + lane < a.cache.sequences) {
            sp = qw_cache_span(a.cache, s0 + lane, a.rows);
            nb = (uint32_t)(((uint64_t)sp.rows * a.group + BM - 1) / BM);
        }
        uint32_t upto = nb; /* inclusive sum over the lanes */
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t t = (uint32_t)__shfl_up((int)upto, o, 64);
            if (lane >= (uint32_t)o) upto += t;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(b < done + upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            job.seq = s0 + l;
            job.blk = b - (done + __builtin_amdgcn_readlane(upto - nb, l));
            job.span = {(uint32_t)__builtin_amdgcn_readlane(sp.begin, l),
                        (uint32_t)__builtin_amdgcn_readlane(sp.rows, l),
                        (uint32_t)__builtin_amdgcn_readlane(sp.length, l)};
            return true;
        }
        done += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

/* Keys [lo, hi) of the new token `token`. */
__device__ __forceinline__ void pa_limits(const qw_paged_args &a, const qw_span &sp,
                                          uint32_t token, uint32_t &lo, uint32_t &hi) {
    const int64_t p = qw_cache_place(sp, token);
    hi = p < 0 ? 0 : (uint32_t)p + 1;
    lo = a.window && hi > a.window ? hi - a.window : 0;
}

/* Buffer of one load's keys: `n` tokens from t on, those below `end`, of the
 * head whose first element is at `base`. */
__device__ __forceinline__ u32x4 pa_rsrc(const qw_cache_args &c, uint64_t base, uint32_t page,
                                         uint32_t t, uint32_t n, uint32_t end) {
    const bool there = page < c.pages;
    const uint64_t at = base + 2 * qw_cache_at(c, there ? page : 0, t, 0, PA_D);
    const uint32_t bytes = qw_cache_bytes(c, t, n, end, PA_D);
    /* the same in every lane: said so, or the compiler keeps it in vector registers */
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) & 0xffffu,
                 (uint32_t)__builtin_amdgcn_readfirstlane(there ? bytes : 0u), 0x00020000u};
}

/* The keys of the 64 from kv0 on, a bit each, that a row with the limits
 * [lo, hi) sees of those in `have`. */
__device__ __forceinline__ uint64_t pa_seen(uint32_t kv0, uint32_t lo, uint32_t hi, uint64_t have) {
    const uint32_t n = hi > kv0 ? min(hi - kv0, 64u) : 0, skip = lo > kv0 ? min(lo - kv0, 64u) : 0;
    const uint64_t below = n < 64 ? (1ull << n) - 1 : ~0ull;
    return skip < 64 ? have & below & (~0ull << skip) : 0;
}
/* v where bit b of m is set, else -inf: two instructions (bit field, insert) */
__device__ __forceinline__ float pa_where(uint32_t m, int b, float v) {
    const uint32_t all = (uint32_t)__builtin_amdgcn_sbfe((int)m, b, 1);
    return __uint_as_float((all & __float_as_uint(v)) | (~all & 0xff800000u));
}
/* Key of s[kbk][v] in a tile: 32 kbk + 8 (v / 4) + 4 h + v % 4; seen: bits of
 * the keys, moved down by 4 h. */
__device__ __forceinline__ void pa_mask(floatx16 (&s)[AKB], uint64_t seen) {
    const uint32_t half[AKB] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
    for (int kbk = 0; kbk < AKB; kbk++)
#pragma unroll
        for (int v = 0; v < 16; v++)
            s[kbk][v] = pa_where(half[kbk], 8 * (v >> 2) + (v & 3), s[kbk][v]);
}

/* The greatest magnitudes, as bit patterns, of 8 bf16 values and those of m, in
 * pairs; 0x7f80 or more in a half: one is infinite or NaN. */
typedef u16 u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 pa_greatest(u16x2 m, bf16x8 v) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; i++)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    return m;
}
__device__ __forceinline__ bool pa_not_finite(u16x2 m) {
    return __builtin_amdgcn_ballot_w64(m[0] >= 0x7f80 || m[1] >= 0x7f80) != 0;
}
/* v with zeros in place of what is not finite */
__device__ __forceinline__ bf16x8 pa_finite(bf16x8 v) {
    u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0xffffu;
        if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
    }
    return __builtin_bit_cast(bf16x8, w);
}
/* ones where v is NaN or the infinity of the sign (0 or 0x8000), else zeros */
__device__ __forceinline__ bf16x8 pa_infinite(bf16x8 v, uint32_t sign) {
    u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t u = 0;
#pragma unroll
        for (int s = 0; s < 32; s += 16) {
            const uint32_t x = w[i] >> s & 0xffffu;
            if ((x & 0x7fffu) > 0x7f80u || x == (0x7f80u | sign)) u |= 0x3F80u << s;
        }
        w[i] = u;
    }
    return __builtin_bit_cast(bf16x8, w);
}

/* ---- many rows ----------------------------------------------------------- */

/* A wave's rows once more, where V held an infinity or NaN in a tile that some
 * of them see only in part: K and V from memory, one tile at a time, with the
 * products taken over V's finite values and what the others give to the rows
 * that see them (an infinity, or NaN) added on the side. Nothing here is made
 * for speed: it costs some 10 us a tile, and no ordinary call comes here. */
__device__ __forceinline__ void pa_again(const qw_paged_args &a, const pa_job &job, uint32_t kvh,
                                         uint32_t r0, uint32_t tile0, uint32_t ntiles,
                                         uint32_t end, floatx16 (&o)[4], float &m_run, float &l_run) {
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid)); /* all anew: nothing is kept over the main loop for this */
    const uint32_t lane = tid & 63, h = lane >> 5, j = lane & 31;
    const uint32_t r = min(r0 + tid / 64 * 32 + j, job.span.rows * a.group - 1);
    const uint32_t token = r / a.group, head = kvh * a.group + r % a.group;
    uint32_t lo, hi;
    pa_limits(a, job.span, token, lo, hi);
    const u16 *qrow = a.q + (size_t)(job.span.begin + token) * a.ldq + head * PA_D;
    const float c = a.scale_log2;
#pragma unroll
    for (int db = 0; db < 4; db++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[db][v] = 0.0f;
    m_run = -INFINITY, l_run = 0.0f;
    for (uint32_t kv0 = tile0 * AKT; kv0 < (tile0 + ntiles) * AKT; kv0 += AKT) {
        /* a key a lane: its page, or none */
        uint32_t page = 0xffffffffu;
        if (kv0 + lane < end) page = a.cache.table[qw_cache_entry(a.cache, job.seq, kv0 + lane)];
        const uint64_t have = __builtin_amdgcn_ballot_w64(page < a.cache.pages);
        floatx16 s[AKB];
#pragma unroll
        for (int kbk = 0; kbk < AKB; kbk++) {
            const uint32_t p = (uint32_t)__shfl((int)page, 32 * kbk + j, 64);
#pragma unroll
            for (int v = 0; v < 16; v++) s[kbk][v] = 0.0f;
#pragma unroll 1
            for (int st = 0; st < 8; st++) {
                bf16x8 kf = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
                if (have >> (32 * kbk + j) & 1)
                    kf = *(const bf16x8 *)(a.cache.k + qw_cache_at(a.cache, p, kv0 + 32 * kbk + j, kvh, PA_D) + 16 * st + 8 * h);
                const bf16x8 qf = *(const bf16x8 *)(qrow + 16 * st + 8 * h);
                s[kbk] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf, s[kbk], 0, 0, 0);
            }
        }
        pa_mask(s, pa_seen(kv0, lo, hi, have) >> 4 * h);
        float mt = -INFINITY;
#pragma unroll
        for (int kbk = 0; kbk < AKB; kbk++)
#pragma unroll
            for (int v = 0; v < 16; v++) mt = fmaxf(mt, s[kbk][v]);
        const float m_to = fmaxf(m_run, fmaxf(mt, __shfl_xor(mt, 32, 64)) * c);
        const float alpha = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_to);
        if (m_to != m_run) {
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < 4; db++)
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (m_run != -INFINITY) o[db][v] *= alpha;
        }
        m_run = m_to;
        bf16x8 pf[2 * AKB], seen[2 * AKB];
        l_run += attn_exp(s, pf, c, m_run == -INFINITY ? 0.0f : m_run);
#pragma unroll
        for (int tk = 0; tk < 2 * AKB; tk++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                seen[tk][e] = s[tk >> 1][8 * (tk & 1) + e] == -INFINITY ? (__bf16)0.0f : (__bf16)1.0f;
#pragma unroll
        for (int db = 0; db < 4; db++) {
            floatx16 up, down; /* how many such values the row sees */
#pragma unroll
            for (int v = 0; v < 16; v++) up[v] = down[v] = 0.0f;
#pragma unroll
            for (int tk = 0; tk < 2 * AKB; tk++) {
                bf16x8 vf;
                /* a step's addresses are made anew, or they would all be kept
                 * over the four blocks of d and registers spilled */
                uint32_t kk = 16 * tk + 4 * h;
                asm volatile("" : "+v"(kk), "+v"(page));
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t k = kk + 8 * (e >> 2) + (e & 3);
                    const uint32_t p = (uint32_t)__shfl((int)page, k, 64);
                    u16 v = 0;
                    if (have >> k & 1) v = a.cache.v[qw_cache_at(a.cache, p, kv0 + k, kvh, PA_D) + 32 * db + j];
                    vf[e] = __builtin_bit_cast(__bf16, v);
                }
                o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa_finite(vf), pf[tk], o[db], 0, 0, 0);
                up = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa_infinite(vf, 0), seen[tk], up, 0, 0, 0);
                down = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa_infinite(vf, 0x8000), seen[tk], down, 0, 0, 0);
                asm volatile("" ::: "memory"); /* one step's loads at a time: registers */
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int v = 0; v < 16; v++) {
                o[db][v] += up[v] > 0.0f ? INFINITY : 0.0f;
                o[db][v] += down[v] > 0.0f ? -INFINITY : 0.0f;
            }
        }
    }
}

/* NW waves of 32 rows. Pieces: a block's key tiles are cut in a.pieces ranges
 * that meet in memory as the image attention's do. PIECES: the most of them, or
 * 1. More than 8 are a kernel of their own, whose longer meeting costs 1 to 2
 * us with few (512 tokens at 7937 in 3 pieces: 87.3 us against 89.8). */
template <int NW, int PIECES>
__device__ __forceinline__ void pa_many(const qw_paged_args &a) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[4 * A_TILE];
    __shared__ uint32_t arrived;
    constexpr uint32_t BM = 32 * NW;
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t h = lane >> 5, j = lane & 31;
    /* ids are dealt round-robin to the 8 XCDs: each takes a contiguous range
     * of (K/V head, block), so the blocks of a head share an L2; the last
     * blocks, which see the most keys, go first */
    const uint32_t pieces = PIECES > 1 ? a.pieces : 1, nwg = a.blocks * a.cache.kv_heads * pieces;
    const uint32_t x = blockIdx.x & 7u;
    const uint32_t pid = x * (nwg >> 3) + min(x, nwg & 7u) + (blockIdx.x >> 3);
    const uint32_t piece = pid % pieces, place = pid / pieces;
    const uint32_t kvh = place / a.blocks, b = a.blocks - 1 - place % a.blocks;
    pa_job job;
    if (!pa_find<BM>(a, b, job)) return;
    const uint32_t R = job.span.rows * a.group; /* rows of this sequence and head */
    const uint32_t r0 = job.blk * BM, r = min(r0 + wave * 32 + j, R - 1);
    const uint32_t token = r / a.group, head = kvh * a.group + r % a.group;

    uint32_t lo, L, lo_first, hi_last, lo_most, hi_least, unused;
    pa_limits(a, job.span, token, lo, L);
    /* over the block and over the wave: limits grow with the row */
    pa_limits(a, job.span, r0 / a.group, lo_first, unused);
    pa_limits(a, job.span, min(r0 + BM - 1, R - 1) / a.group, unused, hi_last);
    pa_limits(a, job.span, min(r0 + wave * 32, R - 1) / a.group, unused, hi_least);
    pa_limits(a, job.span, min(r0 + wave * 32 + 31, R - 1) / a.group, lo_most, unused);
    const uint32_t first = lo_first / AKT, all = (hi_last + AKT - 1) / AKT - min(first, (hi_last + AKT - 1) / AKT);
    const uint32_t tile0 = first + (uint32_t)((uint64_t)piece * all / pieces);
    const uint32_t ntiles = first + (uint32_t)((uint64_t)(piece + 1) * all / pieces) - tile0;

    floatx16 o[4];
#pragma unroll
    for (int db = 0; db < 4; db++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[db][v] = 0.0f;

    constexpr int DPW = AKT / 4 / NW; /* direct loads per wave per tile */
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)lds;
    const uint32_t drow = lane >> 4, dphys = lane & 15, ld = a.cache.kv_heads * PA_D;
    uint32_t kvo[DPW], vvo[DPW];
#pragma unroll
    for (int jj = 0; jj < DPW; jj++) {
        const uint32_t row = (wave * DPW + jj) * 4 + drow;
        kvo[jj] = (drow * ld + ((dphys ^ (row & 15)) * 8)) * 2;
        vvo[jj] = (drow * ld + ((dphys ^ (4 * (row & 3))) * 8)) * 2;
    }
    /* a tile's table entries, one key a lane, and the page ids they give; no
     * page: 0xffffffff */
    const uint32_t *const table = a.cache.table + (size_t)job.seq * a.cache.table_ld;
    auto entry = [&](uint32_t kv0) __attribute__((always_inline)) {
        return table[min((kv0 + lane) >> a.cache.page_shift, a.cache.table_ld - 1)];
    };
    auto page_of = [&](uint32_t p, uint32_t kv0) __attribute__((always_inline)) {
        return kv0 + lane < hi_last && p < a.cache.pages ? p : 0xffffffffu;
    };
    const uint64_t kbase = (uint64_t)(a.cache.k + kvh * PA_D), vbase = (uint64_t)(a.cache.v + kvh * PA_D);
    const uint32_t token_bytes = ld * 2, slots = (1u << a.cache.page_shift) - 1;
    /* a whole tile's loads: byte offsets of their keys in K and V, in a few
     * scalar instructions each */
    auto places = [&](uint64_t (&at)[DPW], uint32_t kv0, uint32_t ids) __attribute__((always_inline)) {
#pragma unroll
        for (int jj = 0; jj < DPW; jj++) {
            const uint32_t blk = wave * DPW + jj, page = __builtin_amdgcn_readlane(ids, blk * 4);
            at[jj] = (uint64_t)((page << a.cache.page_shift) + ((kv0 + 4 * blk) & slots)) * token_bytes;
        }
    };
    auto issue = [&](uint64_t base, uint32_t stage, uint32_t kv0, uint32_t ids, uint64_t have,
                     const uint64_t (&at)[DPW], const uint32_t (&off)[DPW]) __attribute__((always_inline)) {
        if (have == ~0ull) {
#pragma unroll
            for (int jj = 0; jj < DPW; jj++)
                attn_dma(u32x4{(uint32_t)(base + at[jj]), (uint32_t)((base + at[jj]) >> 32) & 0xffffu,
                               3 * token_bytes + 2 * PA_D, 0x00020000u},
                         lds0 + stage * A_TILE + (wave * DPW + jj) * 1024, off[jj], 0);
            return;
        }
#pragma unroll
        for (int jj = 0; jj < DPW; jj++) {
            const uint32_t blk = wave * DPW + jj;
            const uint32_t page = __builtin_amdgcn_readlane(ids, blk * 4);
            attn_dma(pa_rsrc(a.cache, base, page, kv0 + 4 * blk, 4, hi_last),
                     lds0 + stage * A_TILE + blk * 1024, off[jj], 0);
        }
    };
    /* page ids of tiles t and t + 1, which of their keys have one and where
     * their loads are, and tile t + 2's entries, which were asked for a tile
     * ahead */
    uint32_t id1 = 0xffffffffu, next = 0;
    uint64_t have0 = 0, have1 = 0, at1[DPW];
#pragma unroll
    for (int jj = 0; jj < DPW; jj++) at1[jj] = 0;
    if (ntiles) {
        const uint32_t e0 = entry(tile0 * AKT), e1 = entry((tile0 + 1) * AKT);
        next = entry((tile0 + 2) * AKT);
        const uint32_t id0 = page_of(e0, tile0 * AKT);
        id1 = page_of(e1, (tile0 + 1) * AKT);
        have0 = __builtin_amdgcn_ballot_w64(id0 != 0xffffffffu);
        have1 = __builtin_amdgcn_ballot_w64(id1 != 0xffffffffu);
        uint64_t at0[DPW];
        places(at0, tile0 * AKT, id0);
        places(at1, (tile0 + 1) * AKT, id1);
        issue(kbase, 0, tile0 * AKT, id0, have0, at0, kvo);
        issue(vbase, 2, tile0 * AKT, id0, have0, at0, vvo);
        issue(kbase, 1, (tile0 + 1) * AKT, id1, have1, at1, kvo);
    }
    bf16x8 qf[8];
    {
        const u16 *qrow = a.q + (size_t)(job.span.begin + token) * a.ldq + head * PA_D;
#pragma unroll
        for (int s = 0; s < 8; s++) qf[s] = *(const bf16x8 *)(qrow + 16 * s + 8 * h);
    }
    const float c = a.scale_log2;
    auto qk = [&](uint32_t kstage, floatx16 (&s)[AKB], int i0, int i1) __attribute__((always_inline)) {
        const unsigned char *ks = lds + kstage * A_TILE;
#pragma unroll
        for (int i = i0; i < i1; i++) {
            const int kbk = i % AKB, st = i / AKB;
            if (st == 0) {
#pragma unroll
                for (int v = 0; v < 16; v++) s[kbk][v] = 0.0f;
            }
            const bf16x8 kf = *(const bf16x8 *)(ks + (kbk * 32 + j) * 256 +
                                                (((2 * st + h) ^ (j & 15)) << 4));
            s[kbk] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[st], s[kbk], 0, 0, 0);
        }
    };
    const uint32_t tq = lane & 3, te = (lane >> 2) & 3;
    const uint32_t tdb = 16 * ((lane >> 4) & 1) + 4 * tq;
    auto read_v = [&](uint32_t vstage, int tk, int db) __attribute__((always_inline)) {
        const unsigned char *vs = lds + (2 + vstage) * A_TILE;
        const uint32_t d = 32 * db + tdb, cc = d >> 3, half = (d >> 2) & 1;
        const uint32_t r0_ = 16 * tk + 4 * h + te, r1_ = r0_ + 8;
        const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (attn_lds_b4 *)(vs + r0_ * 256 + ((cc ^ (4 * (r0_ & 3))) << 4) + half * 8));
        const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (attn_lds_b4 *)(vs + r1_ * 256 + ((cc ^ (4 * (r1_ & 3))) << 4) + half * 8));
        return bf16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
    };

    float m_run = -INFINITY, l_run = 0.0f;
    bool odd_values = false; /* in the V of a tile with masked scores */
    floatx16 s0[AKB], s1[AKB];
    __builtin_amdgcn_s_waitcnt(0x0F70); /* vmcnt(0) */
    attn_barrier();
    if (ntiles) qk(0, s0, 0, 8 * AKB);
    auto iter = [&](floatx16 (&sc)[AKB], floatx16 (&sn)[AKB], uint32_t t, auto odd)
        __attribute__((always_inline)) {
        constexpr uint32_t st = decltype(odd)::value;
        const uint32_t kv0 = (tile0 + t) * AKT;
        const uint32_t id2 = page_of(next, kv0 + 2 * AKT);
        const uint64_t have2 = __builtin_amdgcn_ballot_w64(id2 != 0xffffffffu);
        uint64_t at2[DPW];
        places(at2, kv0 + 2 * AKT, id2);
        issue(kbase, st, kv0 + 2 * AKT, id2, have2, at2, kvo);
        issue(vbase, 2 + (st ^ 1), kv0 + AKT, id1, have1, at1, vvo);
#pragma unroll
        for (int jj = 0; jj < DPW; jj++) at1[jj] = at2[jj];
        next = entry(kv0 + 3 * AKT);
        const bool masked = kv0 + AKT > hi_least || kv0 < lo_most || have0 != ~0ull;
        if (masked) {
            pa_mask(sc, pa_seen(kv0, lo, L, have0) >> 4 * h);
            const unsigned char *vs = lds + (2 + st) * A_TILE;
            u16x2 most = {0, 0};
#pragma unroll 4
            for (uint32_t n = 0; n < A_TILE / 1024; n++)
                most = pa_greatest(most, *(const bf16x8 *)(vs + n * 1024 + lane * 16));
            odd_values |= pa_not_finite(most);
        }
        bf16x8 vpre[4];
#pragma unroll
        for (int db = 0; db < 4; db++) vpre[db] = read_v(st, 0, db);
        bf16x8 pf[2 * AKB];
        float rs = attn_exp(sc, pf, c, m_run == -INFINITY ? 0.0f : m_run);
        qk(st ^ 1, sn, 0, 8 * AKB);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int i = 0; i < 8 * AKB; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
            if (i + 2 < 8 * AKB) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        /* the running maximum moves lazily, as in attention_kernel.inc */
        if (__builtin_amdgcn_ballot_w64(!(rs < 256.0f) || (m_run == -INFINITY && L != 0))) {
            float mt = -INFINITY;
#pragma unroll
            for (int kbk = 0; kbk < AKB; kbk++)
#pragma unroll
                for (int v = 0; v < 16; v++) mt = fmaxf(mt, sc[kbk][v]);
            const float m_new = fmaxf(mt, __shfl_xor(mt, 32, 64)) * c;
            const bool move = m_new > m_run + 8.0f;
            if (__builtin_amdgcn_ballot_w64(move)) {
                const float m_to = move ? m_new : m_run;
                const float alpha = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_to);
                l_run *= alpha;
#pragma unroll
                for (int db = 0; db < 4; db++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[db][v] *= alpha;
                m_run = m_to;
                rs = attn_exp(sc, pf, c, m_run == -INFINITY ? 0.0f : m_run);
            }
        }
        l_run += rs;
#pragma unroll
        for (int tk = 0; tk < 2 * AKB; tk++)
#pragma unroll
            for (int db = 0; db < 4; db++)
                o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tk ? read_v(st, tk, db) : vpre[db],
                                                                pf[tk], o[db], 0, 0, 0);
        id1 = id2, have0 = have1, have1 = have2;
        __builtin_amdgcn_s_waitcnt(0x0F70); /* vmcnt(0): K(t + 2), V(t + 1) landed */
        attn_barrier();
    };
    uint32_t t = 0;
    for (; t + 1 < ntiles; t += 2) {
        iter(s0, s1, t, std::integral_constant<uint32_t, 0>());
        iter(s1, s0, t + 1, std::integral_constant<uint32_t, 1>());
    }
    if (t < ntiles) iter(s0, s1, t, std::integral_constant<uint32_t, 0>());
    if (odd_values)
        pa_again(a, job, kvh, r0, tile0, ntiles, hi_last, o, m_run, l_run);

    if (PIECES > 1 && pieces > 1) {
        /* a wave's partial as in the image attention: 16 KB of O, m and l */
        constexpr uint32_t WB = 16 * 1024 + 2 * 256, PB = NW * WB;
        const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
            (void *)((unsigned char *)a.part + (size_t)place * pieces * PB), (short)0,
            (int)(pieces * PB), 0x00020000);
        const uint32_t own = piece * PB + wave * WB;
#pragma unroll
        for (int i = 0; i < 16; i++)
            __builtin_amdgcn_raw_buffer_store_b128(
                __builtin_bit_cast(u32x4, floatx4{o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1],
                                                  o[i >> 2][4 * (i & 3) + 2], o[i >> 2][4 * (i & 3) + 3]}),
                pr, own + i * 1024 + lane * 16, 0, 17);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(m_run), pr, own + 16 * 1024 + lane * 4, 0, 17);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l_run), pr, own + 16 * 1024 + 256 + lane * 4, 0, 17);
        __builtin_amdgcn_s_waitcnt(0x0F70); /* vmcnt(0): the partial's stores are done */
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __syncthreads();
        if (tid == 0)
            arrived = __hip_atomic_fetch_add(a.flag + place, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (arrived != pieces - 1) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        /* Every load here takes memory's latency, so m and l of 8 pieces are
         * asked for together, and O of two. A piece in which the row sees no key
         * has m = -inf, O = l = 0; so has a piece past the last, read as it with
         * the factor 0. */
        float f[PIECES], l[PIECES], m_all = -INFINITY;
#pragma unroll
        for (uint32_t p0 = 0; p0 < PIECES; p0 += 8) {
            if (p0 > 0 && p0 >= pieces) {
#pragma unroll
                for (uint32_t pc = p0; pc < p0 + 8; pc++) f[pc] = -INFINITY, l[pc] = 0.0f;
                continue;
            }
#pragma unroll
            for (uint32_t pc = p0; pc < p0 + 8; pc++)
                f[pc] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                    pr, min(pc, pieces - 1) * PB + wave * WB + 16 * 1024 + lane * 4, 0, 17));
#pragma unroll
            for (uint32_t pc = p0; pc < p0 + 8; pc++)
                l[pc] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                    pr, min(pc, pieces - 1) * PB + wave * WB + 16 * 1024 + 256 + lane * 4, 0, 17));
        }
#pragma unroll
        for (uint32_t pc = 0; pc < PIECES; pc++) m_all = fmaxf(m_all, f[pc]);
        l_run = 0.0f;
#pragma unroll
        for (uint32_t pc = 0; pc < PIECES; pc++) {
            f[pc] = f[pc] == -INFINITY || pc >= pieces ? 0.0f : __builtin_amdgcn_exp2f(f[pc] - m_all);
            l_run = __builtin_fmaf(l[pc], f[pc], l_run);
        }
#pragma unroll
        for (int db = 0; db < 4; db++)
#pragma unroll
            for (int v = 0; v < 16; v++) o[db][v] = 0.0f;
#pragma unroll
        for (uint32_t pc = 0; pc < PIECES; pc += 2) {
            if (pc >= pieces) break;
            floatx4 q[2][16];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    q[n][i] = __builtin_bit_cast(
                        floatx4, __builtin_amdgcn_raw_buffer_load_b128(
                                     pr, min(pc + n, pieces - 1) * PB + wave * WB + i * 1024 + lane * 16, 0, 17));
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 16; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        /* not a sum with 0 times an infinity */
                        const float x = q[n][i][e], y = o[i >> 2][4 * (i & 3) + e];
                        o[i >> 2][4 * (i & 3) + e] = f[pc + n] != 0.0f ? __builtin_fmaf(x, f[pc + n], y) : y;
                    }
        }
        if (tid == 0)
            __hip_atomic_store(a.flag + place, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    const float l_all = l_run + __shfl_xor(l_run, 32, 64);
    uint32_t at = r0 + wave * 32 + j; /* anew, as in pa_again */
    asm volatile("" : "+v"(at));
    if (at >= R) return;
    const float inv = l_all == 0.0f ? 0.0f : 1.0f / l_all;
    u16 *orow = a.out + (size_t)(job.span.begin + at / a.group) * a.ldo +
                (kvh * a.group + at % a.group) * PA_D;
#pragma unroll
    for (int db = 0; db < 4; db++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *(u32x2 *)(orow + 32 * db + 8 * g + 4 * h) =
                u32x2{pack_bf(o[db][4 * g] * inv, o[db][4 * g + 1] * inv),
                      pack_bf(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv)};
}
QW_KERNEL void __launch_bounds__(512, 1) qw_paged_attention_q256(qw_paged_args a) { pa_many<8, 1>(a); }
QW_KERNEL void __launch_bounds__(256, 2) qw_paged_attention_q128(qw_paged_args a) { pa_many<4, 1>(a); }
QW_KERNEL void __launch_bounds__(256, 2) qw_paged_attention_q128_split(qw_paged_args a) { pa_many<4, 8>(a); }
QW_KERNEL void __launch_bounds__(256, 2) qw_paged_attention_q128_split32(qw_paged_args a) { pa_many<4, 32>(a); }

/* ---- few rows ------------------------------------------------------------ */

#define PF_KEYS 32            /* keys of a wave's tile */
#define PF_TILE (PF_KEYS * 256)
#define PF_STAGES 2
#define PF_WAVES 4
#define PF_SEGMENT 252        /* tiles whose page ids are in LDS at a time */
#define PF_IDS 1024           /* of pages of 8 tokens, the smallest */

/* RT: tiles of 16 rows */
template <int RT>
__device__ __forceinline__ void pa_few(const qw_paged_args &a) {
    constexpr uint32_t BM = 16 * RT;
    /* the waves' rings of K and V tiles; at the end their sums, 16 RT rows of
     * 128 + m + l */
    constexpr uint32_t SUMS = BM * (PA_D + 4);
    __shared__ __attribute__((aligned(16))) unsigned char lds[PF_WAVES * PF_STAGES * 2 * PF_TILE];
    __shared__ uint32_t ids[PF_IDS];
    __shared__ uint32_t arrived;
    static_assert(PF_WAVES * SUMS * 4 <= sizeof(lds), "the sums lie where the tiles were");
    const uint32_t tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t piece = blockIdx.x % a.pieces, place = blockIdx.x / a.pieces;
    const uint32_t kvh = place % a.cache.kv_heads, b = place / a.cache.kv_heads;
    pa_job job;
    if (!pa_find<BM>(a, b, job)) return;
    const uint32_t R = job.span.rows * a.group, r0 = job.blk * BM, rows = min(BM, R - r0);

    uint32_t lo[RT], L[RT], lo_first, hi_last, lo_most, hi_least, unused;
    pa_limits(a, job.span, r0 / a.group, lo_first, hi_least);
    pa_limits(a, job.span, (r0 + rows - 1) / a.group, lo_most, hi_last);
    const uint32_t first = lo_first / PF_KEYS, end = (hi_last + PF_KEYS - 1) / PF_KEYS;
    const uint32_t all = end - min(first, end);
    /* tiles of a piece: as planned, or more for a longer sequence than that */
    const uint32_t per = max(a.piece_tiles, (all + a.pieces - 1) / a.pieces);
    const uint32_t used = max(1u, (all + per - 1) / per); /* pieces */
    if (piece >= used) return;
    const uint32_t tile0 = first + piece * per, tile1 = first + min((piece + 1) * per, all);

    bf16x8 qf[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const uint32_t r = r0 + min(16 * rt + i, rows - 1);
        const uint32_t token = r / a.group, head = kvh * a.group + r % a.group;
        pa_limits(a, job.span, token, lo[rt], L[rt]);
        const u16 *qrow = a.q + (size_t)(job.span.begin + token) * a.ldq + head * PA_D;
#pragma unroll
        for (int s = 0; s < 4; s++) qf[rt][s] = *(const bf16x8 *)(qrow + 32 * s + 8 * g);
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)lds +
                          wave * (PF_STAGES * 2 * PF_TILE);
    unsigned char *mine = lds + wave * (PF_STAGES * 2 * PF_TILE);
    /* 16-byte chunk c of key row k lies at c ^ (k % 16) in K tiles (a QK
     * fragment pass reads one chunk of 16 rows) and at c ^ 2 (k % 8) in V
     * tiles (a transposing pass reads 2 chunks of 8 rows) */
    const uint32_t drow = lane >> 4, dphys = lane & 15, ld = a.cache.kv_heads * PA_D;
    uint32_t koff[4], voff[2];
#pragma unroll
    for (uint32_t n = 0; n < 4; n++) koff[n] = (drow * ld + ((dphys ^ (4 * n + drow)) * 8)) * 2;
#pragma unroll
    for (uint32_t n = 0; n < 2; n++) voff[n] = (drow * ld + ((dphys ^ (2 * (4 * n + drow))) * 8)) * 2;
    const uint64_t kbase = (uint64_t)(a.cache.k + kvh * PA_D), vbase = (uint64_t)(a.cache.v + kvh * PA_D);
    uint32_t id0 = 0; /* table entry of ids[0] */
    bool gap = false; /* a page of the segment does not exist */
    const uint32_t token_bytes = ld * 2, slots = (1u << a.cache.page_shift) - 1;
    auto issue = [&](uint32_t stage, uint32_t tile) __attribute__((always_inline)) {
        const uint32_t to = lds0 + stage * 2 * PF_TILE;
        /* the ids of the tile's keys, one a lane: one LDS read */
        const uint32_t mine_ = tile * PF_KEYS + (lane & 31);
        const uint32_t page_ = mine_ < hi_last ? ids[(mine_ >> a.cache.page_shift) - id0] : 0xffffffffu;
        if (__builtin_amdgcn_ballot_w64(page_ != 0xffffffffu) == ~0ull) {
#pragma unroll
            for (int n = 0; n < PF_KEYS / 4; n++) {
                const uint32_t page = __builtin_amdgcn_readlane(page_, 4 * n);
                const uint64_t at = (uint64_t)((page << a.cache.page_shift) + ((tile * PF_KEYS + 4 * n) & slots)) * token_bytes;
                const uint64_t k = kbase + at, v = vbase + at;
                attn_dma(u32x4{(uint32_t)k, (uint32_t)(k >> 32) & 0xffffu, 3 * token_bytes + 2 * PA_D, 0x00020000u},
                         to + n * 1024, koff[n & 3], 0);
                attn_dma(u32x4{(uint32_t)v, (uint32_t)(v >> 32) & 0xffffu, 3 * token_bytes + 2 * PA_D, 0x00020000u},
                         to + PF_TILE + n * 1024, voff[n & 1], 0);
            }
            return;
        }
#pragma unroll
        for (int n = 0; n < PF_KEYS / 4; n++) {
            const uint32_t t = tile * PF_KEYS + 4 * n, page = __builtin_amdgcn_readlane(page_, 4 * n);
            attn_dma(pa_rsrc(a.cache, kbase, page, t, 4, hi_last), to + n * 1024, koff[n & 3], 0);
            attn_dma(pa_rsrc(a.cache, vbase, page, t, 4, hi_last), to + PF_TILE + n * 1024, voff[n & 1], 0);
        }
    };
    const uint32_t te = i >> 2, tq = i & 3;
    auto read_v = [&](uint32_t stage, int db) __attribute__((always_inline)) {
        const unsigned char *vs = mine + stage * 2 * PF_TILE + PF_TILE;
        const uint32_t cc = 2 * db + (tq >> 1), half = tq & 1, k0 = 4 * g + te, k1 = k0 + 16;
        const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (attn_lds_b4 *)(vs + k0 * 256 + ((cc ^ (2 * (k0 & 7))) << 4) + half * 8));
        const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (attn_lds_b4 *)(vs + k1 * 256 + ((cc ^ (2 * (k1 & 7))) << 4) + half * 8));
        return bf16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
    };

    floatx4 o[RT][8];
    float m_run[RT], l_run[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m_run[rt] = -INFINITY, l_run[rt] = 0.0f;
#pragma unroll
        for (int db = 0; db < 8; db++) o[rt][db] = floatx4{0, 0, 0, 0};
    }
    const float c = a.scale_log2;
    const qw_b2 ones = {(__bf16)1.0f, (__bf16)1.0f};
    auto step = [&](uint32_t stage, uint32_t tile) __attribute__((always_inline)) {
        const unsigned char *ks = mine + stage * 2 * PF_TILE;
        floatx4 s[RT][2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int st = 0; st < 4; st++) {
                const bf16x8 kf = *(const bf16x8 *)(ks + (16 * kt + i) * 256 + (((4 * st + g) ^ i) << 4));
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    if (st == 0) s[rt][kt] = floatx4{0, 0, 0, 0};
                    s[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[rt][st], s[rt][kt], 0, 0, 0);
                }
            }
        /* key of s[.][kt][v]: kv0 + 16 kt + 4 g + v */
        const uint32_t kv0 = tile * PF_KEYS;
        uint32_t have = ~0u;
        if (gap) {
            const uint32_t t = kv0 + (lane & 31);
            have = (uint32_t)__builtin_amdgcn_ballot_w64(
                t < hi_last && ids[(t >> a.cache.page_shift) - id0] != 0xffffffffu);
        }
        const bool masked = kv0 + PF_KEYS > hi_least || kv0 < lo_most || have != ~0u;
        if (masked) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                const uint32_t seen = (uint32_t)pa_seen(kv0, lo[rt], L[rt], have) >> 4 * g;
#pragma unroll
                for (int n = 0; n < 8; n++)
                    s[rt][n >> 2][n & 3] = pa_where(seen, 16 * (n >> 2) + (n & 3), s[rt][n >> 2][n & 3]);
            }
        }
        bf16x8 pf[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            auto exps = [&]() __attribute__((always_inline)) {
                const float m = m_run[rt] == -INFINITY ? 0.0f : m_run[rt];
                float rs = 0.0f;
#pragma unroll
                for (int n = 0; n < 8; n += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][n >> 2][n & 3], c, -m));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][n >> 2][(n & 3) + 1], c, -m));
                    const qw_b2 pp = __builtin_bit_cast(qw_b2, pack_bf(p0, p1));
                    pf[rt][n] = pp[0], pf[rt][n + 1] = pp[1];
                    rs = __builtin_amdgcn_fdot2_f32_bf16(pp, ones, rs, false);
                }
                return rs;
            };
            float rs = exps();
            /* the maximum moves as in the many-row form, by 2^8 at least */
            if (__builtin_amdgcn_ballot_w64(!(rs < 256.0f) || (m_run[rt] == -INFINITY && L[rt] != 0))) {
                float mt = -INFINITY;
#pragma unroll
                for (int n = 0; n < 8; n++) mt = fmaxf(mt, s[rt][n >> 2][n & 3]);
                mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
                const float m_new = fmaxf(mt, __shfl_xor(mt, 32, 64)) * c;
                const bool move = m_new > m_run[rt] + 8.0f;
                if (__builtin_amdgcn_ballot_w64(move)) {
                    const float m_to = move ? m_new : m_run[rt];
                    const float alpha = m_run[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[rt] - m_to);
                    l_run[rt] *= alpha;
#pragma unroll
                    for (int db = 0; db < 8; db++) o[rt][db] *= alpha;
                    m_run[rt] = m_to;
                    rs = exps();
                }
            }
            l_run[rt] += rs;
        }
        bool odd_values = false;
        if (masked) {
            u16x2 most = {0, 0};
#pragma unroll
            for (int db = 0; db < 8; db++) most = pa_greatest(most, read_v(stage, db));
            odd_values = pa_not_finite(most);
        }
        if (!odd_values) {
#pragma unroll
            for (int db = 0; db < 8; db++) {
                const bf16x8 vf = read_v(stage, db);
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
                    o[rt][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[rt], o[rt][db], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int db = 0; db < 8; db++) {
                const bf16x8 vf = read_v(stage, db);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    bf16x8 seen;
#pragma unroll
                    for (int n = 0; n < 8; n++)
                        seen[n] = s[rt][n >> 2][n & 3] == -INFINITY ? (__bf16)0.0f : (__bf16)1.0f;
                    o[rt][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa_finite(vf), pf[rt], o[rt][db], 0, 0, 0);
#pragma unroll
                    for (int sign = 0; sign < 2; sign++) {
                        const floatx4 n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            pa_infinite(vf, sign << 15), seen, floatx4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                        for (int v = 0; v < 4; v++)
                            o[rt][db][v] += n[v] > 0.0f ? (sign ? -INFINITY : INFINITY) : 0.0f;
                    }
                }
            }
        }
    };
    /* Tiles tile0 + wave, + 4, ...: the next one's loads are out before this
     * one's are waited for (16 loads a tile). The wave alone writes and reads
     * its ring, so the wait is all the order that is needed; the LDS reads of
     * a stage are done before its next loads are issued, for their values
     * have gone into the matrix instructions. */
    for (uint32_t seg = tile0; seg < tile1; seg += PF_SEGMENT) {
        const uint32_t seg1 = min(seg + PF_SEGMENT, tile1);
        id0 = (seg * PF_KEYS) >> a.cache.page_shift;
        const uint32_t n = ((min(seg1 * PF_KEYS, hi_last) - 1) >> a.cache.page_shift) - id0 + 1;
        bool none = false;
        __syncthreads(); /* every wave is through with the segment before */
        for (uint32_t e = tid; e < n; e += 64 * PF_WAVES) {
            const uint32_t p = a.cache.table[(uint64_t)job.seq * a.cache.table_ld + id0 + e];
            ids[e] = p < a.cache.pages ? p : 0xffffffffu;
            none |= p >= a.cache.pages;
        }
        gap = __syncthreads_or(none);
        uint32_t tile = seg + wave, stage = 0;
        if (tile < seg1) issue(0, tile);
        for (; tile < seg1; tile += PF_WAVES, stage ^= 1) {
            const bool more = tile + PF_WAVES < seg1;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); /* the other stage has been read */
            if (more) {
                issue(stage ^ 1, tile + PF_WAVES);
                asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            step(stage, tile);
        }
    }
    /* ---- the waves' sums, then the pieces' ------------------------------- */
    __syncthreads();
    float *sums = (float *)lds; /* [wave][row][128 | m | l], row stride 132 */
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        float l = l_run[rt];
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        float *to = sums + wave * SUMS + (16 * rt + i) * (PA_D + 4);
#pragma unroll
        for (int db = 0; db < 8; db++) *(floatx4 *)(to + 16 * db + 4 * g) = o[rt][db];
        if (g == 0) to[PA_D] = m_run[rt], to[PA_D + 1] = l;
    }
    __syncthreads();
    /* a thread has 8 columns of row tid / 16 (and 16 further for RT 2) */
    float acc[RT][8], m_all[RT], l_all[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const float *row = sums + (16 * rt + tid / 16) * (PA_D + 4);
        m_all[rt] = -INFINITY, l_all[rt] = 0.0f;
#pragma unroll
        for (int w = 0; w < PF_WAVES; w++) m_all[rt] = fmaxf(m_all[rt], row[w * SUMS + PA_D]);
#pragma unroll
        for (int e = 0; e < 8; e++) acc[rt][e] = 0.0f;
#pragma unroll
        for (int w = 0; w < PF_WAVES; w++) {
            const float m = row[w * SUMS + PA_D];
            if (m == -INFINITY) { /* the wave saw no key of the row, or scores that are NaN */
                l_all[rt] += row[w * SUMS + PA_D + 1];
                continue;
            }
            const float f = __builtin_amdgcn_exp2f(m - m_all[rt]);
            l_all[rt] = __builtin_fmaf(row[w * SUMS + PA_D + 1], f, l_all[rt]);
#pragma unroll
            for (int e = 0; e < 8; e++)
                acc[rt][e] = __builtin_fmaf(row[w * SUMS + (tid & 15) * 8 + e], f, acc[rt][e]);
        }
    }
    uint32_t rows_left = rows; /* that this thread stores */
    if (used > 1) {
        /* a piece's rows [row][128 | m | l] in memory, as the waves' in LDS */
        float *part = a.part + (size_t)place * a.pieces * SUMS;
        const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
            (void *)part, (short)0, (int)(a.pieces * SUMS * 4), 0x00020000);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const uint32_t row = 16 * rt + tid / 16;
            const uint32_t at = (piece * SUMS + row * (PA_D + 4)) * 4;
            if (row < rows) {
#pragma unroll
                for (int e = 0; e < 8; e += 4)
                    __builtin_amdgcn_raw_buffer_store_b128(
                        __builtin_bit_cast(u32x4, floatx4{acc[rt][e], acc[rt][e + 1], acc[rt][e + 2], acc[rt][e + 3]}),
                        pr, at + ((tid & 15) * 8 + e) * 4, 0, 17);
                if ((tid & 15) == 0)
                    __builtin_amdgcn_raw_buffer_store_b64(
                        u32x2{__float_as_uint(m_all[rt]), __float_as_uint(l_all[rt])}, pr, at + PA_D * 4, 0, 17);
            }
        }
        __builtin_amdgcn_s_waitcnt(0x0F70); /* vmcnt(0): the piece's stores are done */
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __syncthreads();
        if (tid == 0)
            arrived = __hip_atomic_fetch_add(a.flag + place, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (arrived != used - 1) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        /* `sets` of threads take every sets-th piece of a row's 8 columns each,
         * and meet in LDS. The first four of them, which for a short context
         * are all, are asked for here, with all pieces' m and l: one latency. */
        const uint32_t sets = rows > 8 ? 1 : rows > 4 ? 2 : 4, per = 16 * PF_WAVES / 4 / sets; /* rows a pass */
        const uint32_t set = tid / 16 / per;
        floatx4 q[4][2];
        auto load_o = [&](uint32_t row, uint32_t p0) __attribute__((always_inline)) {
            const uint32_t at = (row * (PA_D + 4) + (tid & 15) * 8) * 4;
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    q[n][e] = __builtin_bit_cast(
                        floatx4, __builtin_amdgcn_raw_buffer_load_b128(
                                     pr, at + min(p0 + n * sets, used - 1) * SUMS * 4 + 16 * e, 0, 17));
        };
        load_o(tid / 16 % per, set);
        float *ml = (float *)lds; /* [row][piece][m | l], then a factor for m */
        for (uint32_t e = tid; e < used * rows; e += 64 * PF_WAVES) {
            const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(
                pr, (e % used * SUMS + e / used * (PA_D + 4) + PA_D) * 4, 0, 17);
            ml[2 * e] = __uint_as_float(v[0]), ml[2 * e + 1] = __uint_as_float(v[1]);
        }
        __syncthreads();
        /* the rows' maxima and sums: 8 threads each */
        float *total = ml + 2 * used * rows; /* [row] */
        for (uint32_t r = tid / 8; r < rows; r += 8 * PF_WAVES) {
            float m = -INFINITY, l = 0.0f;
            for (uint32_t pc = tid & 7; pc < used; pc += 8) m = fmaxf(m, ml[2 * (r * used + pc)]);
#pragma unroll
            for (int o_ = 1; o_ < 8; o_ <<= 1) m = fmaxf(m, __shfl_xor(m, o_, 64));
            for (uint32_t pc = tid & 7; pc < used; pc += 8) {
                const float x = ml[2 * (r * used + pc)];
                const float f = x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - m);
                ml[2 * (r * used + pc)] = f;
                l = __builtin_fmaf(ml[2 * (r * used + pc) + 1], f, l);
            }
#pragma unroll
            for (int o_ = 1; o_ < 8; o_ <<= 1) l += __shfl_xor(l, o_, 64);
            if ((tid & 7) == 0) total[r] = l;
        }
        __syncthreads();
        float *meet = total + BM;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const uint32_t row = 16 * rt + tid / 16 % per;
#pragma unroll
            for (int e = 0; e < 8; e++) acc[rt][e] = 0.0f;
            if (row < rows) {
                for (uint32_t p0 = set; p0 < used; p0 += 4 * sets) {
                    if (rt || p0 != set) load_o(row, p0);
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const uint32_t pc = p0 + n * sets;
                        const float f = pc < used ? ml[2 * (row * used + pc)] : 0.0f;
                        if (f == 0.0f) continue; /* no key of the row, or no such piece */
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            acc[rt][e] = __builtin_fmaf(q[n][e >> 2][e & 3], f, acc[rt][e]);
                    }
                }
                l_all[rt] = total[row];
                if (set) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        meet[((set - 1) * per + row) * PA_D + (tid & 15) * 8 + e] = acc[rt][e];
                }
            }
        }
        if (sets > 1) { /* at most 8 rows: RT's first tile alone */
            __syncthreads();
            if (set == 0 && tid / 16 < rows)
                for (uint32_t n = 1; n < sets; n++)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        acc[0][e] += meet[((n - 1) * per + tid / 16) * PA_D + (tid & 15) * 8 + e];
            if (set) rows_left = 0;
        }
        if (tid == 0)
            __hip_atomic_store(a.flag + place, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const uint32_t row = 16 * rt + tid / 16;
        if (row >= rows_left) continue;
        const uint32_t r = r0 + row, token = r / a.group, head = kvh * a.group + r % a.group;
        const float inv = l_all[rt] == 0.0f ? 0.0f : 1.0f / l_all[rt];
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = pack_bf(acc[rt][2 * e] * inv, acc[rt][2 * e + 1] * inv);
        *(u32x4 *)(a.out + (size_t)(job.span.begin + token) * a.ldo + head * PA_D + (tid & 15) * 8) = w;
    }
}
QW_KERNEL void __launch_bounds__(64 * PF_WAVES, 2) qw_paged_attention_r16(qw_paged_args a) { pa_few<1>(a); }
QW_KERNEL void __launch_bounds__(64 * PF_WAVES, 2) qw_paged_attention_r32(qw_paged_args a) { pa_few<2>(a); }
