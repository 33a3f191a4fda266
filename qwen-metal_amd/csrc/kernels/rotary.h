/* Rotary positions of q and k, with the per-head RMS norm ahead of them where
 * there is one, and k and v going into a paged cache.
 *
 * Pair i of a head turns by position * f_i, f_i in turns as a 64-bit
 * fraction: the product modulo one turn is exact in integer arithmetic (its
 * top 32 bits are pos * high + mulhi(pos, low)), however far the position,
 * where a product in fp32 is off by a radian at a position of 2^24. What is
 * left of the turn is brought to an eighth either way and goes into the
 * series of sine and cosine. Norm and rotation stay in fp32 and are rounded
 * once, at the store.
 *
 * Bound by latency for few rows (one row into the cache 3.8 us, an empty launch
 * 3.0: starts and lengths, the table's entry, the store), by HBM and close
 * behind it by the vector unit for many (7724 rows of 32 + 8 heads, normed,
 * into the cache 46.6 us, 4.1 TB/s; a large copy has 4.8). A workgroup has one
 * row and 256 / (head_dim / 8) of its heads (or three times as many), a lane 16
 * bytes of a head: the row's sines are made once per workgroup and shared
 * through LDS (made by every lane for itself they cost 8 pairs for each 16
 * bytes, more than the bytes' time). */
#pragma once
#include "common.h"
#include "paged_cache.h"

/* (cos, sin) of a 32-bit fraction of a turn: a quarter turn's multiple off the
 * top, the rest x in [-pi/4, pi/4] by the Taylor series (remainders x^11/11! <
 * 2e-9 and x^10/10! < 3e-8). */
__device__ __forceinline__ qw_f2 rotary_cos_sin(uint32_t turn) {
    const uint32_t quarter = (turn + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(turn - (quarter << 30)) * 1.46291807926715968e-9f; /* 2 pi / 2^32 */
    const float y = x * x;
    const float s = x * __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
    const float c = __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 1.0f / 40320, -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
    return qw_f2{quarter == 1 || quarter == 2 ? -a : a, quarter >= 2 ? -b : b};
}

/* How many of starts[1..n] are at or below `row`: the sequence of a row, all
 * 64 lanes together. */
__device__ __forceinline__ uint32_t rotary_sequence(const qw_cache_args &c, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t n = 0;
    for (uint32_t s = 0; s < c.sequences; s += 64) {
        const bool below = s + lane < c.sequences && c.starts[s + lane + 1] <= row;
        n += __popcll(__builtin_amdgcn_ballot_w64(below));
    }
    return n;
}

/* Not kept in L2, where the rows to come would have to push it out: 7724 rows
 * of 32 + 8 heads into the cache 50.7 -> 46.6 us, 1000 rows of them beside it
 * 6.2 -> 5.0. An attention that follows at once gains and loses nothing by it:
 * both together 41.9 -> 41.3 us at 1000 rows, 250 -> 251.5 at 7724, 15.4 at
 * one. */
__device__ __forceinline__ void rotary_store(u16 *to, u32x4 v) {
    __builtin_nontemporal_store(v, (u32x4 *)to);
}

/* H heads a lane: 1 for few rows, where the chain of loads to a row's page is
 * the time, 3 for many, where a row's chain, sines and norm weights serve 3
 * times the bytes (the 7724 rows: 60 us with 1, 50 with 3, before the stores
 * went past L2). */
template <int D, int H>
__device__ __forceinline__ void rotary_impl(const qw_rotary_args &a) {
    constexpr uint32_t LPH = D / 8, HPP = 256 / LPH; /* lanes per head, heads per pass */
    __shared__ __attribute__((aligned(16))) qw_f2 turned[D / 2];
    const uint32_t tid = threadIdx.x, row = blockIdx.x, c8 = tid % LPH * 8;
    const uint32_t head0 = blockIdx.y * (HPP * H) + tid / LPH;
    const uint32_t all = a.heads + a.kv_heads * (a.cached ? 2 : 1);
    const uint32_t hn = a.rotary_dim / 2;
    const bool whole = hn % 8 == 0; /* a lane's partners lie in one chunk */
    const bool pairs = a.half && c8 < a.rotary_dim;
    /* each head's own values, and those that they are paired with: element e
     * with e + hn below hn and e - hn from there on */
    u32x4 own[H], other[H];
#pragma unroll
    for (int n = 0; n < H; n++) {
        const uint32_t head = head0 + n * HPP;
        own[n] = other[n] = u32x4{0, 0, 0, 0};
        if (head >= all) continue;
        const bool is_q = head < a.heads, is_k = head < a.heads + a.kv_heads;
        const u16 *src = is_q   ? a.q + (size_t)row * a.ldq + head * D
                         : is_k ? a.k + (size_t)row * a.ldk + (head - a.heads) * D
                                : a.v + (size_t)row * a.ldv + (head - a.heads - a.kv_heads) * D;
        own[n] = *(const u32x4 *)(src + c8);
        if (!pairs || !is_k) continue;
        if (whole) {
            other[n] = *(const u32x4 *)(src + (c8 < hn ? c8 + hn : c8 - hn));
        } else {
            u16 t[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                const uint32_t e = c8 + i;
                t[i] = e < hn ? src[e + hn] : e < a.rotary_dim ? src[e - hn] : 0;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) other[n][i] = t[2 * i] | (uint32_t)t[2 * i + 1] << 16;
        }
    }

    uint32_t pos = 0;
    uint64_t at = ~0ull; /* of the cache's K/V head 0 */
    if (a.cached) {
        const uint32_t s = rotary_sequence(a.cache, row);
        if (s == a.cache.sequences) return; /* behind the last sequence */
        const qw_span sp = qw_cache_span(a.cache, s, a.rows);
        if (row < sp.begin || row - sp.begin >= sp.rows) return;
        const int64_t place = qw_cache_place(sp, row - sp.begin);
        if (place < 0) return; /* a token that its sequence does not have */
        pos = (uint32_t)place;
        const uint32_t page = a.cache.table[qw_cache_entry(a.cache, s, pos)];
        if (page < a.cache.pages) at = qw_cache_at(a.cache, page, pos, 0, D);
    }
    if (a.positions) pos = a.positions[row];
    if (tid < hn) {
        const u32x2 t = *(const u32x2 *)(a.turns + 2 * tid);
        const qw_f2 cs = rotary_cos_sin(pos * t[0] + __umulhi(pos, t[1]));
        turned[tid] = qw_f2{cs[0] * a.factor, cs[1] * a.factor};
    }
    __syncthreads();
    /* the lane's sines, the same for all its heads: y = x c + other s, the sign
     * of s by the side */
    float c[8], s[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
        const uint32_t e = c8 + i;
        c[i] = 1.0f, s[i] = 0.0f;
        if (e >= a.rotary_dim) continue;
        const qw_f2 t = turned[!a.half ? e / 2 : e < hn ? e : e - hn];
        c[i] = t[0];
        s[i] = (a.half ? e < hn : !(e & 1)) ? -t[1] : t[1];
    }
#pragma unroll
    for (int n = 0; n < H; n++) {
        const uint32_t head = head0 + n * HPP;
        if (head >= all) continue;
        const bool is_q = head < a.heads, is_k = !is_q && head < a.heads + a.kv_heads;
        const uint32_t kvh = is_q ? 0 : is_k ? head - a.heads : head - a.heads - a.kv_heads;
        if (is_q || is_k) {
            float x[8], y[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[2 * i] = lo_bf(own[n][i]), x[2 * i + 1] = hi_bf(own[n][i]);
                y[2 * i] = lo_bf(other[n][i]), y[2 * i + 1] = hi_bf(other[n][i]);
            }
            const u16 *w = is_q ? a.norm_q : a.norm_k;
            if (w) {
                float sq = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) sq = __builtin_fmaf(x[i], x[i], sq);
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) sq += __shfl_xor(sq, o, 64);
                const float inv = __builtin_amdgcn_rsqf(__builtin_fmaf(sq, 1.0f / D, a.eps));
                const u32x4 wv = *(const u32x4 *)(w + c8);
#pragma unroll
                for (int i = 0; i < 4; i++) x[2 * i] *= inv * lo_bf(wv[i]), x[2 * i + 1] *= inv * hi_bf(wv[i]);
                if (pairs && whole) {
                    const u32x4 ov = *(const u32x4 *)(w + (c8 < hn ? c8 + hn : c8 - hn));
#pragma unroll
                    for (int i = 0; i < 4; i++) y[2 * i] *= inv * lo_bf(ov[i]), y[2 * i + 1] *= inv * hi_bf(ov[i]);
                } else if (pairs) {
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) {
                        const uint32_t e = c8 + i;
                        if (e < a.rotary_dim) y[i] *= inv * bf2f(w[e < hn ? e + hn : e - hn]);
                    }
                }
            }
            if (!a.half) {
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = x[i ^ 1];
            }
            /* past rotary_dim c = 1, s = 0 and y = 0 or a finite neighbour's:
             * only there could an infinity in y spoil x, so it is left out */
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c8 + i < a.rotary_dim) x[i] = __builtin_fmaf(y[i], s[i], x[i] * c[i]);
#pragma unroll
            for (int i = 0; i < 4; i++) own[n][i] = pack_bf(x[2 * i], x[2 * i + 1]);
        }
        if (is_q) {
            rotary_store(a.q_out + (size_t)row * a.ldq_out + head * D + c8, own[n]);
        } else if (!a.cached) {
            rotary_store(a.k_out + (size_t)row * a.ldk_out + kvh * D + c8, own[n]);
        } else if (at != ~0ull) {
            rotary_store((is_k ? a.cache.k : a.cache.v) + at + kvh * D + c8, own[n]);
        }
    }
}
#define ROTARY(d)                                                                                     \
    QW_KERNEL void __launch_bounds__(256) qw_rotary_d##d(qw_rotary_args a) { rotary_impl<d, 1>(a); }  \
    QW_KERNEL void __launch_bounds__(256) qw_rotary_d##d##_h3(qw_rotary_args a) { rotary_impl<d, 3>(a); }
ROTARY(64) ROTARY(128) ROTARY(256)
