/* Pieces of the flash attention loop that the image kernels (attention.h) and
 * those over a paged cache (paged_attention.h) share. */
#pragma once
#include "common.h"

#define AKB 2                       /* 32-key blocks per tile */
#define AKT (32 * AKB)              /* keys per tile */
#define A_TILE (AKT * 256)          /* one K or V tile: AKT keys x 128 bf16 */

/* P = exp2(S c - m) rounded to bf16 (the B operand of P.V, one bf16x8 per
 * 16-key K-step) and the lane's part of the row sum, which adds the same
 * rounded values (v_dot2 against ones). */
__device__ __forceinline__ float attn_exp(const floatx16 (&s)[AKB], bf16x8 (&pf)[2 * AKB],
                                          float c, float m_use) {
    float rs = 0.0f;
    const qw_b2 ones = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int tk = 0; tk < 2 * AKB; tk++) {
        const int kbk = tk >> 1, v0 = 8 * (tk & 1);
#pragma unroll
        for (int u = 0; u < 8; u += 2) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kbk][v0 + u], c, -m_use));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kbk][v0 + u + 1], c, -m_use));
            const qw_b2 pp = __builtin_bit_cast(qw_b2, pack_bf(p0, p1));
            pf[tk][u] = pp[0];
            pf[tk][u + 1] = pp[1];
            rs = __builtin_amdgcn_fdot2_f32_bf16(pp, ones, rs, false);
        }
    }
    return rs;
}

/* One 16-byte-per-lane direct load into LDS (buffer_load_dwordx4 ... lds):
 * M0 = the wave's LDS base, lane l writes base + 16 l. Issued from inline
 * assembly so the compiler does not treat it as a pending LDS store (it
 * would wait for every one in flight before each LDS read); the kernel
 * waits for them itself (vmcnt) before the barrier that publishes a tile. The
 * load reads M0 one wait state after its write at the earliest, and a scalar
 * register that a vector instruction wrote (a spilled one read back from a
 * lane, a page's address) five after (gfx9 rules; the compiler does not see
 * inside the asm to insert them): the write of M0 and s_nop 3. */
__device__ __forceinline__ void attn_dma(u32x4 rsrc, uint32_t lds_base, uint32_t voff,
                                         uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds_base), "v"(voff), "s"(rsrc), "s"(soff)
                 : "m0");
}

__device__ __forceinline__ void attn_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

typedef __attribute__((address_space(3))) bf16x4 attn_lds_b4;
