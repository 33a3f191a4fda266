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
    const uint32_t m = 0x000F000Fu, c = 0x43004300u;
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

/* NT: tiles of 16 rows, CT: tiles of 16 columns per workgroup, GS: group */
template <int NT, int CT, int GS>
__device__ __forceinline__ void linear4_impl(const qw_linear4_args &a) {
    __shared__ float part[L4_WAVES / 2][CT * NT * 256];
    const uint32_t lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col0 = blockIdx.x * 16 * CT, groups = a.k / GS, steps = (a.k + 127) / 128;
    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u,
                                                         0x3F803F80u});
    /* columns past the last are computed as it, and not stored; so are rows */
    uint32_t col[CT];
    const uint8_t *w[CT];
    const u16 *x[NT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        col[c] = min(col0 + 16 * c + i, a.cols - 1);
        w[c] = a.weight + (size_t)col[c] * (a.k / 2) + 16 * g;
    }
#pragma unroll
    for (int t = 0; t < NT; t++)
        x[t] = a.in + (size_t)min(16 * t + i, a.rows - 1) * a.lda + (GS == 128 ? 32 : 8) * g;
    floatx4 sum[CT][NT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int t = 0; t < NT; t++) sum[c][t] = floatx4{0, 0, 0, 0};

    for (uint32_t st = wave; st < steps; st += L4_WAVES) {
        const uint32_t k0 = st * 128;
        u32x4 q[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            q[c] = u32x4{0, 0, 0, 0};
            if (GS == 128 || k0 + 32 * g < a.k) q[c] = *(const u32x4 *)(w[c] + k0 / 2);
            if (GS < 128) q[c] = l4_transpose(q[c]);
        }
#pragma unroll
        for (int j0 = 0; j0 < 4; j0 += GS / 32) { /* a group */
            if (GS < 128 && k0 + 32 * j0 >= a.k) break;
            const uint32_t gi = (k0 + 32 * j0) / GS;
            floatx4 xs[NT], p[CT][NT];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                xs[t] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < CT; c++) p[c][t] = floatx4{0, 0, 0, 0};
            }
#pragma unroll
            for (int j = j0; j < j0 + GS / 32; j++) {
                bf16x8 wf[CT];
#pragma unroll
                for (int c = 0; c < CT; c++) wf[c] = l4_widen(q[c][j]);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const bf16x8 xf = l4_order(
                        *(const u32x4 *)(x[t] + k0 + (GS == 128 ? 8 : 32) * j));
                    xs[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, ones, xs[t], 0, 0, 0);
#pragma unroll
                    for (int c = 0; c < CT; c++)
                        p[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, wf[c], p[c][t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const size_t at = (size_t)col[c] * groups + gi;
                const float s = bf2f(a.scales[at]);
                const float z = -128.0f - (a.zeros ? bf2f(a.zeros[at]) : 8.0f);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        sum[c][t][r] = __builtin_fmaf(s, __builtin_fmaf(z, xs[t][r], p[c][t][r]),
                                                      sum[c][t][r]);
            }
        }
    }
    /* the waves' sums meet in halves: rows 4 g + r of tile t, column i */
#pragma unroll
    for (uint32_t h = L4_WAVES / 2; h > 0; h >>= 1) {
        if (wave >= h && wave < 2 * h) {
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int t = 0; t < NT; t++)
                    *(floatx4 *)&part[wave - h][(c * NT + t) * 256 + lane * 4] = sum[c][t];
        }
        __syncthreads();
        if (wave < h) {
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int t = 0; t < NT; t++)
                    sum[c][t] += *(const floatx4 *)&part[wave][(c * NT + t) * 256 + lane * 4];
        }
        __syncthreads();
    }
    if (wave) return;
#pragma unroll
    for (int c = 0; c < CT; c++) {
        if (col0 + 16 * c + i >= a.cols) continue;
        const float b = a.bias ? bf2f(a.bias[col[c]]) : 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t row = 16 * t + 4 * g + r;
                if (row < a.rows) a.out[(size_t)row * a.ldc + col[c]] = f2bf(sum[c][t][r] + b);
            }
    }
}
#define L4_KERNEL(nt, ct, gs)                                                                \
    QW_KERNEL void __launch_bounds__(64 * L4_WAVES, 2) qw_linear4_r##nt##c##ct##g##gs(qw_linear4_args a) { \
        linear4_impl<nt, ct, gs>(a);                                                         \
    }
#define L4_GROUPS(nt, ct) L4_KERNEL(nt, ct, 32) L4_KERNEL(nt, ct, 64) L4_KERNEL(nt, ct, 128)
L4_GROUPS(1, 1)
L4_GROUPS(2, 1)
L4_GROUPS(4, 1)

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
