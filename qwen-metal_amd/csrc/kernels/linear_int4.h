/* Linears on 4-bit weights with a scale (and a zero point) per group of
 * inputs, for few rows:
 *
 *   y[r][c] = sum over groups g of s[c][g] (sum q[c][k] x[r][k] - z[c][g] sum x[r][k])
 *
 * The weight is streamed once; 16 columns x 32 inputs a step go through
 * v_mfma_f32_16x16x32_bf16 against up to 16 rows of x each. A weight becomes
 * the bf16 number 128 + q by one and-or per pair: 0x4300 is 128, whose last
 * mantissa bit is 1. (q there as an integer would need a conversion each, and
 * q s rounded to bf16 would cost 2^-9 of every weight.) The group's products
 * P = sum (128 + q) x stay in fp32, as does X = sum x, by an MFMA against
 * ones, and s (P - (128 + z) X) is added to the row's sum: what cancels is 128
 * / 4.6 times the result, 2^-19 of it in fp32. A step's nibbles come out in
 * the order 0 4 1 5 2 6 3 7 of each 8 inputs, x is permuted alike.
 *
 * A lane loads 16 bytes, 32 inputs of one column; its 16-lane row takes the
 * inputs 32 g .. 32 g + 31 of 128. With groups of 128 an MFMA may sum over
 * any of them, with smaller ones the four rows' words are exchanged first
 * (4 x 4 transpose by permlane swaps) so that each MFMA has 32 neighbours. */
#pragma once
#include "common.h"

#define L4_WAVES 8

__device__ __forceinline__ bf16x8 l4_widen(uint32_t w) {
    /* one in a vector, one in a scalar register: v_and_or_b32 takes no literal,
     * and the compiler's and, or with one each are two instructions */
    uint32_t m = 0x000F000Fu, c = 0x43004300u;
    asm("" : "+v"(m), "+s"(c));
    return __builtin_bit_cast(bf16x8, u32x4{(w & m) | c, (w >> 4 & m) | c, (w >> 8 & m) | c,
                                            (w >> 12 & m) | c});
}
/* x[0..7] in the order of l4_widen */
__device__ __forceinline__ bf16x8 l4_order(u32x4 x) {
    return __builtin_bit_cast(
        bf16x8, u32x4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u),
                      __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                      __builtin_amdgcn_perm(x[3], x[1], 0x05040100u),
                      __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)});
}

/* w[j] of 16-lane row g <-> w[g] of row j */
__device__ __forceinline__ u32x4 l4_transpose(u32x4 w) {
    auto r = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    auto s = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    auto t = __builtin_amdgcn_permlane16_swap(r[0], s[0], false, false);
    auto u = __builtin_amdgcn_permlane16_swap(r[1], s[1], false, false);
    return u32x4{(uint32_t)t[0], (uint32_t)t[1], (uint32_t)u[0], (uint32_t)u[1]};
}

/* What a step of 128 inputs takes of a column tile: 16 bytes of weights a lane
 * and the groups' scales and zero points (Z: there are some). Steps past the
 * last are read as it: no branch stands between a load and its use, where the
 * compiler would wait for every load. */
template <int GS>
using l4_pack = std::conditional_t<GS == 32, uint64_t, std::conditional_t<GS == 64, uint32_t, u16>>;
template <int GS, bool Z>
struct l4_step {
    u32x4 q;
    l4_pack<GS> s, z; /* 16 bits a group */
};
/* 128 / GS neighbours of t[at], at most `count` in all, in one load (as single
 * ones they took most of the time of small groups: 60 rows, 4096 -> 24576,
 * groups of 32 with zero points 85 us against 50.6). Ones that would pass the end are
 * read from it back and moved down. */
template <int GS>
__device__ __forceinline__ l4_pack<GS> l4_groups(const u16 *t, uint64_t at, uint64_t count) {
    const uint64_t from = GS == 128 ? at : min(at, count - 128 / GS);
    l4_pack<GS> v;
    __builtin_memcpy(&v, t + from, sizeof(v));
    if (GS < 128) v >>= 16 * (uint32_t)(at - from);
    return v;
}
template <int GS, bool Z>
__device__ __forceinline__ void l4_load(const qw_linear4_args &a, l4_step<GS, Z> &w, uint32_t col,
                                        uint32_t st, uint32_t g) {
    const uint32_t groups = a.k / GS, steps = (a.k + 127) / 128, k0 = min(st, steps - 1) * 128;
    uint32_t at = k0 + 32 * g;
    if (GS < 128) at = min(at, a.k - 32);
    w.q = *(const u32x4 *)(a.weight + ((size_t)col * a.k + at) / 2);
    const uint64_t e = (uint64_t)col * groups + k0 / GS, all = (uint64_t)a.cols * groups;
    w.s = l4_groups<GS>(a.scales, e, all);
    w.z = Z ? l4_groups<GS>(a.zeros, e, all) : (l4_pack<GS>)0x4100410041004100ull; /* 8 */
}

/* ---- up to 16 rows that fit LDS ------------------------------------------- */

/* A workgroup takes tiles of 16 columns, its 8 waves every 8th step of them.
 * All of x lies in LDS, in the order that l4_widen gives weights, and a tile's
 * scales and zero points (one block of memory) are copied there a tile ahead:
 * as 2-byte loads, two of each a step at groups of 64, they took as long as
 * the weights (12288 -> 4096, one row: 21.0 us against 10.3 with groups of 128
 * and no zero points). Weights are loaded L4_AHEAD steps before their use,
 * over the end of a tile into the next. Rows past the last are computed as it,
 * and not stored; so are columns.
 *
 * x decides how many workgroups a CU has: two where it takes 64 KB with the
 * scales, one up to 144. Beyond, and for more rows, x goes through LDS in
 * slabs, which costs its pieces' meeting (16 rows, 4096 -> 6144: 8.3 us here,
 * 10.9 there; 4096 -> 24576 15.0 and 19.6; 4 rows, 12288 -> 4096 11.4 and
 * 20.2). Bound by HBM with the way to the first weights: one row 4096 -> 24576
 * 12.5 us (4.2 TB/s), 12288 -> 4096 with zero points 10.1, of which an empty
 * launch is 3. */
#define L4_AHEAD 4
template <int GS, bool Z, int LDS>
__device__ __forceinline__ void linear4_few(const qw_linear4_args &a) {
    /* x, then two buffers of scales and zero points */
    __shared__ __attribute__((aligned(16))) unsigned char lds[LDS];
    __shared__ float part[L4_WAVES][256];
    const uint32_t tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t steps = (a.k + 127) / 128, tiles = (a.cols + 15) / 16, groups = a.k / GS;
    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u,
                                                         0x3F803F80u});
    u32x4 w[L4_AHEAD];
    auto load = [&](int u, uint32_t tile, uint32_t st) __attribute__((always_inline)) {
        const uint32_t col = min(min(tile, tiles - 1) * 16 + i, a.cols - 1);
        uint32_t at = min(st, steps - 1) * 128 + 32 * g;
        if (GS < 128) at = min(at, a.k - 32);
        w[u] = *(const u32x4 *)(a.weight + ((size_t)col * a.k + at) / 2);
    };
    uint32_t tile = blockIdx.x;
#pragma unroll
    for (int u = 0; u < L4_AHEAD; u++) load(u, tile, wave + u * L4_WAVES);
    /* scales of a tile: `groups` of 16 columns; a column's row in LDS is 4
     * bytes longer, so that the lanes' reads hit different banks */
    const uint32_t srow = groups * 2 + (groups & 1 ? 2 : 4), sbytes = 16 * srow;
    unsigned char *const sl = lds + (size_t)a.rows * steps * 256;
    auto copy_scales = [&](uint32_t t, uint32_t buffer) __attribute__((always_inline)) {
        for (uint32_t e = tid * 2; e < 16 * groups; e += 2 * 64 * L4_WAVES) {
            /* two neighbours; a pair may pass from a column to the next */
            const uint64_t at = min((uint64_t)t * 16 * groups + e, (uint64_t)a.cols * groups - 2);
            const uint32_t s = *(const uint32_t *)(a.scales + at);
            const uint32_t z = Z ? *(const uint32_t *)(a.zeros + at) : 0;
            unsigned char *to = sl + buffer * sbytes * (1 + Z);
            const uint32_t c0 = e / groups, c1 = (e + 1) / groups;
            *(u16 *)(to + c0 * srow + (e - c0 * groups) * 2) = (u16)s;
            *(u16 *)(to + c1 * srow + (e + 1 - c1 * groups) * 2) = (u16)(s >> 16);
            if (Z) {
                *(u16 *)(to + sbytes + c0 * srow + (e - c0 * groups) * 2) = (u16)z;
                *(u16 *)(to + sbytes + c1 * srow + (e + 1 - c1 * groups) * 2) = (u16)(z >> 16);
            }
        }
    };
    copy_scales(tile, 0);
    /* 16-byte chunk ch of a row at ch ^ row; zeros behind k. Loads of some rows
     * together: one after another they are a latency each (16 rows, 4096 ->
     * 6144: 12.0 us against 8.3; 16 together 8.7). */
    auto copy_x = [&](auto together) __attribute__((always_inline)) {
        constexpr uint32_t XR = decltype(together)::value;
        for (uint32_t ch = tid; ch < steps * 16; ch += 64 * L4_WAVES)
            for (uint32_t row0 = 0; row0 < a.rows; row0 += XR) {
                u32x4 v[XR];
#pragma unroll
                for (uint32_t n = 0; n < XR; n++)
                    v[n] = *(const u32x4 *)(a.in + (size_t)min(row0 + n, a.rows - 1) * a.lda + min(8 * ch, a.k - 8));
#pragma unroll
                for (uint32_t n = 0; n < XR; n++) {
                    const uint32_t row = row0 + n;
                    if (8 * ch >= a.k) v[n] = u32x4{0, 0, 0, 0};
                    if (row < a.rows) *(bf16x8 *)(lds + row * steps * 256 + ((ch ^ row) << 4)) = l4_order(v[n]);
                }
            }
    };
    if (LDS <= QW_L4_FEW && a.rows == 1)
        copy_x(std::integral_constant<uint32_t, 1>());
    else
        copy_x(std::integral_constant<uint32_t, LDS <= QW_L4_FEW ? 4 : 8>());
    __syncthreads();
    floatx4 sum = {0, 0, 0, 0};
    const uint32_t xrow = min(i, a.rows - 1);
    const unsigned char *const xr = lds + xrow * steps * 256;
    auto step = [&](int u, uint32_t st, const unsigned char *sc) __attribute__((always_inline)) {
        const u32x4 q = GS == 128 ? w[u] : l4_transpose(w[u]);
#pragma unroll
        for (int n = 0; n < 128 / GS; n++) {
            floatx4 xs = {0, 0, 0, 0}, p = {0, 0, 0, 0};
#pragma unroll
            for (int j = n * GS / 32; j < (n + 1) * GS / 32; j++) {
                const uint32_t ch = st * 16 + (GS == 128 ? 4 * g + j : 4 * j + g);
                const bf16x8 xf = *(const bf16x8 *)(xr + ((ch ^ xrow) << 4));
                xs = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, ones, xs, 0, 0, 0);
                p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, l4_widen(q[j]), p, 0, 0, 0);
            }
            const uint32_t gi = min(st * (128 / GS) + n, groups - 1) * 2; /* past k: x is zero */
            const float s = bf2f(*(const u16 *)(sc + gi));
            const float z = Z ? -128.0f - bf2f(*(const u16 *)(sc + sbytes + gi)) : -136.0f;
#pragma unroll
            for (int r = 0; r < 4; r++)
                sum[r] = __builtin_fmaf(s, __builtin_fmaf(z, xs[r], p[r]), sum[r]);
        }
    };
    for (uint32_t buffer = 0; tile < tiles; tile += gridDim.x, buffer ^= 1) {
        const unsigned char *const sc = sl + buffer * sbytes * (1 + Z) + i * srow;
        for (uint32_t base = 0; base < steps; base += L4_AHEAD * L4_WAVES) {
            const bool end = base + L4_AHEAD * L4_WAVES >= steps;
            const uint32_t to = end ? tile + gridDim.x : tile;
            const uint32_t from = wave + (end ? 0 : base + L4_AHEAD * L4_WAVES);
#pragma unroll
            for (int u = 0; u < L4_AHEAD; u++) {
                const uint32_t st = base + u * L4_WAVES + wave;
                if (st < steps) step(u, st, sc);
                load(u, to, from + u * L4_WAVES);
            }
        }
        if (tile + gridDim.x < tiles) copy_scales(tile + gridDim.x, buffer ^ 1);
        /* row 4 g + r, column i: the waves' sums meet in LDS */
        *(floatx4 *)&part[wave][lane * 4] = sum;
        sum = floatx4{0, 0, 0, 0};
        __syncthreads();
        const uint32_t row = tid >> 4, c = tid & 15, col = tile * 16 + c;
        if (tid < 256 && row < a.rows && col < a.cols) {
            float y = 0.0f;
#pragma unroll
            for (int n = 0; n < L4_WAVES; n++) y += part[n][((row >> 2) * 16 + c) * 4 + (row & 3)];
            a.out[(size_t)row * a.ldc + col] = f2bf(y + (a.bias ? bf2f(a.bias[col]) : 0.0f));
        }
        __syncthreads();
    }
}
#define L4_FEW(name, gs, lds, waves)                                                             \
    QW_KERNEL void __launch_bounds__(64 * L4_WAVES, waves) qw_linear4_##name##_g##gs(qw_linear4_args a) { \
        linear4_few<gs, false, lds>(a);                                                          \
    }                                                                                            \
    QW_KERNEL void __launch_bounds__(64 * L4_WAVES, waves) qw_linear4_##name##_g##gs##z(qw_linear4_args a) { \
        linear4_few<gs, true, lds>(a);                                                           \
    }
L4_FEW(few, 32, QW_L4_FEW, 4) L4_FEW(few, 64, QW_L4_FEW, 4) L4_FEW(few, 128, QW_L4_FEW, 4)
L4_FEW(wide, 32, QW_L4_WIDE, 2) L4_FEW(wide, 64, QW_L4_WIDE, 2) L4_FEW(wide, 128, QW_L4_WIDE, 2)

/* ---- up to 64 rows ------------------------------------------------------- */

/* x weighs as much as the weight: 16 columns a workgroup read it from L2
 * 1536 times for 24576 columns (98.8 us at 60 rows, 30.7 here). A workgroup
 * has 128 columns, 32 for each of 4 waves and two such sets of waves, or 96
 * or 64 columns, 48 or 32 for each of two waves and four such sets. A set takes
 * every 2nd or 4th slab of 128 inputs; x's slabs pass through LDS, in the order
 * that l4_widen gives weights, one round of the sets ahead. The widest tile
 * widens the fewest weights and reads the least of x, a narrower one fills the
 * CUs where the widest leaves some idle: the host weighs them by measured
 * times. Few columns are cut along K in a.pieces ranges that meet in memory
 * (the last in adds them in order). NT: tiles of 16 rows.
 *
 * Bound by the issue of vector and matrix instructions: with 128 columns the
 * same loop without any load from memory took 24 us of 32. The sums X, a third
 * of the matrix instructions there, are a quarter with 48 columns a wave. */
template <int NT, int COLS, int GS, bool Z>
__device__ __forceinline__ void linear4_many(const qw_linear4_args &a) {
    constexpr int CW = COLS > 96 ? 4 : 2, SETS = L4_WAVES / CW, CT = COLS / CW / 16;
    constexpr int ROWS = 16 * NT, SLAB = ROWS * 256 /* bytes */, N = CT * NT;
    constexpr int XN = SETS * ROWS * 16 / 512; /* chunks of x of a thread */
    __shared__ __attribute__((aligned(16))) unsigned char lds[2][SETS * SLAB];
    __shared__ uint32_t arrived;
    const uint32_t tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), set = wave / CW, part = wave % CW;
    const uint32_t piece = blockIdx.x % a.pieces, tile = blockIdx.x / a.pieces;
    const uint32_t col0 = tile * COLS + part * (16 * CT);
    const uint32_t slabs = (a.k + 127) / 128;
    const uint32_t first = (uint64_t)slabs * piece / a.pieces;
    const uint32_t last = (uint64_t)slabs * (piece + 1) / a.pieces;
    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u,
                                                         0x3F803F80u});
    uint32_t col[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) col[c] = min(col0 + 16 * c + i, a.cols - 1);
    /* x: chunk n of a thread is 16 bytes of a row of one of the sets' slabs;
     * chunk ch of a row lies at ch ^ (row % 16) */
    u32x4 xv[XN];
    auto load_x = [&](uint32_t slab) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < XN; n++) {
            const uint32_t c = n * 512 + tid, row = (c >> 4) % ROWS;
            const uint32_t k = (slab + c / (ROWS * 16)) * 128 + (c & 15) * 8;
            xv[n] = u32x4{0, 0, 0, 0};
            if (k < a.k) xv[n] = *(const u32x4 *)(a.in + (size_t)min(row, a.rows - 1) * a.lda + k);
        }
    };
    auto store_x = [&](uint32_t buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < XN; n++) {
            const uint32_t c = n * 512 + tid, row = (c >> 4) % ROWS;
            *(bf16x8 *)(lds[buffer] + c / (ROWS * 16) * SLAB + row * 256 +
                        (((c & 15) ^ (row & 15)) << 4)) = l4_order(xv[n]);
        }
    };
    l4_step<GS, Z> w[2][CT];
    auto load_w = [&](int u, uint32_t slab) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < CT; c++) l4_load(a, w[u][c], col[c], slab, g);
    };
    floatx4 sum[CT][NT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int t = 0; t < NT; t++) sum[c][t] = floatx4{0, 0, 0, 0};
    auto step = [&](int u, uint32_t buffer, uint32_t k0) __attribute__((always_inline)) {
        const unsigned char *xs_ = lds[buffer] + set * SLAB;
        u32x4 q[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) q[c] = GS == 128 ? w[u][c].q : l4_transpose(w[u][c].q);
#pragma unroll
        for (int n = 0; n < 128 / GS; n++) {
            if (GS < 128 && k0 + n * GS >= a.k) break;
            floatx4 xs[NT], p[CT][NT];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                xs[t] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < CT; c++) p[c][t] = floatx4{0, 0, 0, 0};
            }
#pragma unroll
            for (int j = n * GS / 32; j < (n + 1) * GS / 32; j++) {
                bf16x8 wf[CT];
#pragma unroll
                for (int c = 0; c < CT; c++) wf[c] = l4_widen(q[c][j]);
                const uint32_t ch = GS == 128 ? 4 * g + j : 4 * j + g;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const bf16x8 xf = *(const bf16x8 *)(xs_ + (16 * t + i) * 256 + ((ch ^ i) << 4));
                    xs[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, ones, xs[t], 0, 0, 0);
#pragma unroll
                    for (int c = 0; c < CT; c++)
                        p[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, wf[c], p[c][t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const float s = bf2f((u16)(w[u][c].s >> 16 * n)), z = -128.0f - bf2f((u16)(w[u][c].z >> 16 * n));
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        sum[c][t][r] = __builtin_fmaf(s, __builtin_fmaf(z, xs[t][r], p[c][t][r]),
                                                      sum[c][t][r]);
            }
        }
    };
    /* slabs at, at + 1, ... (one a set) from buffer, weights of the two rounds
     * after in flight */
    load_x(first);
    load_w(0, first + set);
    load_w(1, first + SETS + set);
    store_x(0);
    load_x(first + SETS);
    __syncthreads();
    uint32_t buffer = 0;
    for (uint32_t at = first; at < last; at += 2 * SETS) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t s = at + SETS * u; /* the same for all waves */
            if (s >= last) break;
            if (s + set < last) step(u, buffer, (s + set) * 128);
            load_w(u, s + 2 * SETS + set);
            if (s + SETS < last) {
                store_x(buffer ^ 1);
                load_x(s + 2 * SETS);
            }
            __syncthreads();
            buffer ^= 1;
        }
    }
    /* the sets' sums meet in LDS: set s adds up every SETS-th block of 16 x
     * 16 from the s-th on, and has it from here on */
    float *const meet = (float *)lds + part * (N * 256) + lane * 4;
    static_assert(L4_WAVES * N * 1024 <= sizeof(lds), "");
#pragma unroll
    for (int n = 0; n < N; n++) *(floatx4 *)(meet + (set * CW * N + n) * 256) = sum[n / NT][n % NT];
    __syncthreads();
    constexpr int OWN = (N + SETS - 1) / SETS;
    floatx4 own[OWN];
#pragma unroll
    for (int m = 0; m < OWN; m++) {
        const uint32_t n = min(m * SETS + set, N - 1);
        own[m] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < SETS; w++) own[m] += *(const floatx4 *)(meet + (w * CW * N + n) * 256);
    }
    if (a.pieces > 1) {
        constexpr uint32_t PB = CW * N * 1024; /* bytes of a piece */
        const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
            (void *)((unsigned char *)a.part + (size_t)tile * a.pieces * PB), (short)0,
            (int)(a.pieces * PB), 0x00020000);
        const uint32_t at = part * (N * 1024) + set * 1024 + lane * 16;
#pragma unroll
        for (int m = 0; m < OWN; m++)
            if (m * SETS + set < N)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, own[m]), pr,
                                                       piece * PB + at + m * SETS * 1024, 0, 17);
        __builtin_amdgcn_s_waitcnt(0x0F70); /* vmcnt(0): the piece's stores are done */
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __syncthreads();
        if (tid == 0)
            arrived = __hip_atomic_fetch_add(a.flag + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (arrived != a.pieces - 1) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
#pragma unroll
        for (int m = 0; m < OWN; m++) own[m] = floatx4{0, 0, 0, 0};
        for (uint32_t pc = 0; pc < a.pieces; pc++)
#pragma unroll
            for (int m = 0; m < OWN; m++)
                own[m] += __builtin_bit_cast(
                    floatx4, __builtin_amdgcn_raw_buffer_load_b128(
                                 pr, pc * PB + at + (min(m * SETS + set, N - 1) - set) * 1024, 0, 17));
        if (tid == 0)
            __hip_atomic_store(a.flag + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int m = 0; m < OWN; m++) {
        const uint32_t n = m * SETS + set, to = col0 + 16 * (n / NT) + i;
        if (n >= N || to >= a.cols) continue;
        const float b = a.bias ? bf2f(a.bias[to]) : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint32_t row = 16 * (n % NT) + 4 * g + r;
            if (row < a.rows) a.out[(size_t)row * a.ldc + to] = f2bf(own[m][r] + b);
        }
    }
}
/* One workgroup a CU is what the host plans, so two waves a SIMD: with a third
 * in mind the compiler asks for x later (60 rows, 4096 -> 32768: 39.0 us
 * against 36.4). */
#define L4_MANY(nt, cols, gs)                                                                           \
    QW_KERNEL void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) qw_linear4_r##nt##_c##cols##_g##gs(qw_linear4_args a) {    \
        linear4_many<nt, cols, gs, false>(a);                                                           \
    }                                                                                                   \
    QW_KERNEL void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) qw_linear4_r##nt##_c##cols##_g##gs##z(qw_linear4_args a) { \
        linear4_many<nt, cols, gs, true>(a);                                                            \
    }
#define L4_GROUPS(nt, cols) L4_MANY(nt, cols, 32) L4_MANY(nt, cols, 64) L4_MANY(nt, cols, 128)
#define L4_TILES(cols) L4_GROUPS(1, cols) L4_GROUPS(2, cols) L4_GROUPS(4, cols)
L4_TILES(64) L4_TILES(96) L4_TILES(128)

/* One wave per 64 groups' worth of weights would waste lanes on short rows, so
 * a lane has a group of its own: two passes over its 32 to 128 weights (the
 * second from cache). Symmetric: s = bf16(max |w| / 7), q = rint(w / s) + 8 in
 * 1 .. 15. With zero points: s = bf16((max - min) / 15) with min <= 0 <= max,
 * z = rint(-min / s), q = rint(w / s) + z, all in 0 .. 15. A group of zeros has
 * s = 0 and q = the zero point. */
QW_KERNEL void __launch_bounds__(256) qw_quantize_int4_rows(qw_quant4_args a) {
#pragma clang fp contract(off)
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t groups = a.cols / a.group;
    if (at >= (uint64_t)a.rows * groups) return;
    const u16 *in = a.in + at * a.group;
    float lo = 0.0f, hi = 0.0f;
    for (uint32_t k = 0; k < a.group; k += 8) {
        const u32x4 v = *(const u32x4 *)(in + k);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            lo = fminf(lo, fminf(lo_bf(v[i]), hi_bf(v[i])));
            hi = fmaxf(hi, fmaxf(lo_bf(v[i]), hi_bf(v[i])));
        }
    }
    const u16 sb = f2bf(a.zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f);
    const float s = bf2f(sb);
    const float z = !a.zeros ? 8.0f : s > 0.0f ? fminf(rintf(-lo / s), 15.0f) : 0.0f;
    a.scales[at] = sb;
    if (a.zeros) a.zeros[at] = f2bf(z);
    for (uint32_t k = 0; k < a.group; k += 8) {
        const u32x4 v = *(const u32x4 *)(in + k);
        uint32_t out = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float w = i & 1 ? hi_bf(v[i / 2]) : lo_bf(v[i / 2]);
            const float q = s > 0.0f ? fminf(fmaxf(rintf(w / s) + z, 0.0f), 15.0f) : z;
            out |= (uint32_t)q << (4 * i);
        }
        *(uint32_t *)(a.q + (at * a.group + k) / 2) = out;
    }
}

/* bf16((q - z) s), 8 weights a thread: the copy that linears of many rows run
 * on. Each weight is rounded once. */
QW_KERNEL void __launch_bounds__(256) qw_dequant_int4_bf16(qw_dequant4_args a) {
    const uint64_t n = (uint64_t)a.rows * a.cols / 8, stride = (uint64_t)gridDim.x * 256;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < n; at += stride) {
        const uint32_t q = *(const uint32_t *)(a.q + 4 * at);
        const uint64_t g = 8 * at / a.group;
        const float s = bf2f(a.scales[g]), z = a.zeros ? bf2f(a.zeros[g]) : 8.0f;
        u32x4 out;
#pragma unroll
        for (int i = 0; i < 4; i++)
            out[i] = pack_bf(((float)(q >> (8 * i) & 15) - z) * s,
                             ((float)(q >> (8 * i + 4) & 15) - z) * s);
        *(u32x4 *)(a.out + 8 * at) = out;
    }
}
