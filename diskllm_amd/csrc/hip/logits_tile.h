/*
 * logits_tile.h -- what the LM head's products share: staging in LDS, the soft-cap, the
 * tiles' places.
 */
#ifndef DLK_LOGITS_TILE_H
#define DLK_LOGITS_TILE_H

#include <hip/hip_runtime.h>

#include "dlk_device.h"
#include "../../../include/diskllm_amd.h"

namespace dlk {

typedef int i4 __attribute__((ext_vector_type(4)));

/* Waits until at most N of the wave's loads are in flight and its LDS work is done. */
template <int N>
DLK_DEV void wait_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (N >> 4) << 14);
    asm volatile("" ::: "memory");
}

/* 16-byte chunk c of row r of a staged tile lies at chunk place(r, c): the lanes of a
 * fragment read (16 rows at one or two neighbouring chunks) then meet every bank once. */
template <int BK>
DLK_DEV int place(int r, int c) {
    return BK == 64 ? c ^ ((0x78 >> (2 * ((r >> 2) & 3))) & 3) : BK == 128 ? c ^ (r & 7) : c ^ (r & 15);
}

/* cap * tanh(y / cap) in some 16 instructions (libm's bits, which dlk_softcap gives, take
 * 65: 240 us of the 512 x 262,144 product against 60).  t = |y| / cap: below 0.35 the
 * series of tanh(t) / t to t^10 (what is left out: 2e-9 of it), above (1 - e) / (1 + e)
 * with e = exp(-2t).  At 0.35, the worst place, e is off by 3.4 half-steps, which 2 e / (1
 * + e)^2 / tanh makes 4.5; with t's own two and those of 1 + e, its reciprocal and the
 * products some 10 half-steps of the result at most.  recip: 1 / cap, finite. */
DLK_DEV float capped(float y, float cap, float recip) {
    const float q = y * recip, t = fabsf(q), t2 = t * t;
    float s = fmaf(t2, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    s = fmaf(t2, s, -17.0f / 315.0f);
    s = fmaf(t2, s, 2.0f / 15.0f);
    s = fmaf(t2, s, -1.0f / 3.0f);
    s = fmaf(t * t2, s, t);
    const float e = __builtin_amdgcn_exp2f(-2.88539008177792681f * t);
    const float b = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
    return copysignf(t < 0.35f ? s : b, q) * cap;
}

/* Loads 16 bytes a lane straight into LDS: lane i's to dst + 16 i (dst the same in all lanes). */
DLK_DEV void load_to_lds(const int8_t *src, int8_t *dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                     (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
}

/* One tile's place: workgroups go to the XCDs in turn, so each XCD gets a run of tiles, the
 * tiles of x for one tile of w side by side: w comes from memory once. */
template <int BM, int BN>
DLK_DEV bool tile_of(int rows, int vocab, int &m0, int &v0) {
    const int mtiles = (rows + BM - 1) / BM, vtiles = (vocab + BN - 1) / BN;
    const int tile = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
    m0 = tile % mtiles * BM;
    v0 = tile / mtiles * BN;
    return tile < mtiles * vtiles;
}

}  // namespace dlk

#endif
