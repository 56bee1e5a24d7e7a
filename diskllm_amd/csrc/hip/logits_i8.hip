/*
 * logits_i8.hip -- an LM head in 8-bit integers: logits[r, v] = (x_r . w_v) * x_scale[r] *
 * w_scale[v], the soft-cap as epilogue (dlk_logits_i8).
 */
#include <hip/hip_runtime.h>

#include "softcap4.h"
#include "../../../include/diskllm_amd.h"

namespace dlk {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i4_any __attribute__((ext_vector_type(4), aligned(1)));

struct I8Params {
    const int8_t *x, *w;
    int64_t ldx, ldw, ld;
    const float *x_scale, *w_scale;
    float *logits;
    int rows, vocab, n;
    float cap, recip;
};

/* The 16 bytes at k of a row of n < 16. */
__device__ __noinline__ i4 load16_short(const int8_t *p, int k, int n) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll 1
    for (int c = 0; k + c < n; c++) {
        const uint32_t b = (uint32_t)(uint8_t)p[k + c] << (8 * (c & 3));
        w[0] |= c >> 2 == 0 ? b : 0;
        w[1] |= c >> 2 == 1 ? b : 0;
        w[2] |= c >> 2 == 2 ? b : 0;
        w[3] |= c >> 2 == 3 ? b : 0;
    }
    return i4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
}

/* The 16 bytes at k of a row of n, zeros past its end: no byte outside the row is read
 * (the row's last 16 bytes, shifted down, where k + 16 > n). */
DLK_DEV i4 load16_to(const int8_t *p, int k, int n) {
    if (DLK_COLD(n < 16)) return load16_short(p, k, n);
    const int a = min(k, n - 16), s = k - a;
    const i4 v = *(const i4_any *)(p + a);
    const uint64_t lo = (uint64_t)(uint32_t)v.y << 32 | (uint32_t)v.x, hi = (uint64_t)(uint32_t)v.w << 32 | (uint32_t)v.z;
    const int b = 8 * (s & 7);
    const uint64_t l1 = s < 8 ? (lo >> b) | (b ? hi << (64 - b) : 0) : s < 16 ? hi >> b : 0;
    const uint64_t h1 = s < 8 ? hi >> b : 0;
    return i4{(int)(uint32_t)l1, (int)(uint32_t)(l1 >> 32), (int)(uint32_t)h1, (int)(uint32_t)(h1 >> 32)};
}

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

/* BM rows of x and BN rows of w per workgroup, WGM x WGN waves, steps of BK bytes of n,
 * ST stages in LDS.  DMA: the rows of both are whole 16-byte chunks, loaded straight into
 * LDS; else through registers, any alignment. */
template <int BM, int BN, int WGM, int WGN, int BK, int ST, int OCC, bool DMA, bool CAP>
__global__ __launch_bounds__(WGM * WGN * 64, OCC) void logits_i8_kernel(I8Params p) {
    constexpr int W = WGM * WGN, WM = BM / WGM, WN = BN / WGN, MF = WM / 16, NF = WN / 16;
    constexpr int CPR = BK / 16, RPI = 64 / CPR;   /* chunks of a row; rows that a wave loads at once */
    constexpr int NI = (BM + BN) / RPI / W;        /* loads of a wave per stage */
    constexpr int STAGE = (BM + BN) * BK;
    static_assert((BM + BN) % (RPI * W) == 0 && BM % RPI == 0 && (BK == 64 || BK == 128 || BK == 256), "tiles");
    __shared__ __align__(1024) int8_t lds[ST * STAGE];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    /* workgroups go to the XCDs in turn: each XCD gets a run of tiles, the rows' tiles of one
     * tile of w side by side, so that w comes from memory once */
    const int mtiles = (p.rows + BM - 1) / BM, vtiles = (p.vocab + BN - 1) / BN;
    const int tile = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
    if (tile >= mtiles * vtiles) return;
    const int m0 = tile % mtiles * BM, v0 = tile / mtiles * BN;
    const int8_t *src[NI];                         /* the row of this lane's chunk */
    int at[NI];                                    /* and its place in the row */
#pragma unroll
    for (int j = 0; j < NI; j++) {
        const int r = (j * W + wave) * RPI + lane / CPR;
        at[j] = place<BK>(r, lane % CPR) * 16;
        src[j] = r < BM ? p.x + (int64_t)min(m0 + r, p.rows - 1) * p.ldx
                        : p.w + (int64_t)min(v0 + r - BM, p.vocab - 1) * p.ldw;
    }
    i4 reg[DMA ? 1 : NI];
    auto fetch = [&](int k0, int slot) {
#pragma unroll
        for (int j = 0; j < NI; j++) {
            if (DMA && k0 + BK <= p.n) {
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src[j] + k0 + at[j]),
                                                 (__attribute__((address_space(3))) void *)&lds[slot * STAGE + (j * W + wave) * 1024],
                                                 16, 0, 0);
            } else {
                const i4 v = k0 + BK <= p.n ? (i4)*(const i4_any *)(src[j] + k0 + at[j]) : load16_to(src[j], k0 + at[j], p.n);
                if (DMA) *(i4 *)&lds[slot * STAGE + (j * W + wave) * 1024 + lane * 16] = v;
                else reg[j] = v;
            }
        }
    };
    auto put = [&](int slot) {
        if (!DMA) {
#pragma unroll
            for (int j = 0; j < NI; j++) *(i4 *)&lds[slot * STAGE + (j * W + wave) * 1024 + lane * 16] = reg[j];
        }
    };
    const int lr = lane & 15, lk = lane >> 4, wm = wave % WGM * WM, wn = wave / WGM * WN;
    i4 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int f = 0; f < NF; f++) acc[m][f] = i4{0, 0, 0, 0};
    const int steps = (p.n + BK - 1) / BK;
#pragma unroll
    for (int s = 0; s < ST - 1; s++)
        if (s < steps) { fetch(s * BK, s); put(s); }
    int slot = 0;
    for (int it = 0; it < steps; it++) {
        if (it + ST - 2 < steps) wait_loads<NI *(ST - 2)>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int next = slot == 0 ? ST - 1 : slot - 1;        /* the slot that step it - 1 has left */
        if (it + ST - 1 < steps) fetch((it + ST - 1) * BK, next);
        const int8_t *xs = &lds[slot * STAGE], *ws = xs + BM * BK;
#pragma unroll
        for (int s = 0; s < BK / 64; s++) {
            i4 a[NF], b[MF];
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const int r = wn + f * 16 + lr;
                a[f] = *(const i4 *)&ws[r * BK + place<BK>(BM + r, s * 4 + lk) * 16];
            }
#pragma unroll
            for (int m = 0; m < MF; m++) {
                const int r = wm + m * 16 + lr;
                b[m] = *(const i4 *)&xs[r * BK + place<BK>(r, s * 4 + lk) * 16];
            }
#pragma unroll
            for (int m = 0; m < MF; m++)
#pragma unroll
                for (int f = 0; f < NF; f++)
                    acc[m][f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[f], b[m], acc[m][f], 0, 0, 0);
        }
        if (it + ST - 1 < steps) put(next);
        slot = slot == ST - 1 ? 0 : slot + 1;
    }
#pragma unroll
    for (int f = 0; f < NF; f++) {
        const int v = v0 + wn + f * 16 + lk * 4;
        float ws[4];
#pragma unroll
        for (int c = 0; c < 4; c++) ws[c] = p.w_scale[min(v + c, p.vocab - 1)];
#pragma unroll
        for (int m = 0; m < MF; m++) {
            const int r = m0 + wm + m * 16 + lr;
            const float sx = p.x_scale[min(r, p.rows - 1)];
            float y[4];
#pragma unroll
            for (int c = 0; c < 4; c++) y[c] = (float)acc[m][f][c] * sx * ws[c];
            if (CAP) softcap4<false>(y, p.cap, p.recip);
            if (r < p.rows) {
                float *out = p.logits + (int64_t)r * p.ld + v;
                if (v + 3 < p.vocab) {
                    store4(out, make_float4(y[0], y[1], y[2], y[3]));
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (v + c < p.vocab) out[c] = y[c];
                }
            }
        }
    }
}

template <int BM, int BN, int WGM, int WGN, int BK, int ST, int OCC, bool DMA>
int launch_i8(const I8Params &p, hipStream_t stream) {
    const int64_t tiles = (((int64_t)p.vocab + BN - 1) / BN) * (((int64_t)p.rows + BM - 1) / BM);
    if (tiles > 0x3fffffff) return DLK_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)((tiles + 7) / 8 * 8)), block(WGM * WGN * 64);
    if (p.cap > 0.0f)
        hipLaunchKernelGGL((logits_i8_kernel<BM, BN, WGM, WGN, BK, ST, OCC, DMA, true>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((logits_i8_kernel<BM, BN, WGM, WGN, BK, ST, OCC, DMA, false>), grid, block, 0, stream, p);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

template <bool DMA>
int launch_i8_rows(const I8Params &p, hipStream_t stream) {
    if (p.rows <= 16) return launch_i8<16, 64, 1, 4, 256, 3, 2, DMA>(p, stream);
    if (p.rows <= 32) return launch_i8<32, 64, 1, 4, 128, 4, 2, DMA>(p, stream);
    if (p.rows <= 64) return launch_i8<64, 64, 1, 4, 128, 4, 2, DMA>(p, stream);
    if (p.rows <= 128) return launch_i8<128, 128, 2, 2, 64, 3, 2, DMA>(p, stream);
    return launch_i8<256, 128, 2, 2, 64, 3, 2, DMA>(p, stream);
}

}  // namespace dlk

extern "C" int dlk_logits_i8(const int8_t *x, int64_t ldx, const float *x_scale, const int8_t *w, int64_t ldw,
                             const float *w_scale, int rows, int vocab, int n, float softcap, float *logits, int64_t ld,
                             hipStream_t stream) {
    using namespace dlk;
    if (!x || !x_scale || !w || !w_scale || !logits || rows < 0 || vocab <= 0 || n <= 0) return DLK_ERR_INVALID;
    if (ldx < n || ldw < n || ld < vocab) return DLK_ERR_INVALID;
    if ((((uintptr_t)x_scale | (uintptr_t)w_scale | (uintptr_t)logits) & 3) != 0) return DLK_ERR_INVALID;
    /* |sum| <= 128 * 128 * n in 32 bits; int indices */
    if (n > 131071 || vocab > 0x7fffffff - 65536 || rows > 0x7fffffff - 65536) return DLK_ERR_UNSUPPORTED;
    if (rows == 0) return DLK_OK;
    I8Params p;
    p.x = x; p.w = w; p.ldx = ldx; p.ldw = ldw; p.ld = ld;
    p.x_scale = x_scale; p.w_scale = w_scale; p.logits = logits;
    p.rows = rows; p.vocab = vocab; p.n = n;
    p.cap = softcap > 0.0f ? softcap : 0.0f;
    p.recip = p.cap > 0.0f ? dlk_softcap_recip(p.cap) : 0.0f;
    const bool chunks = (((uintptr_t)x | (uintptr_t)w | (uintptr_t)ldx | (uintptr_t)ldw) & 15) == 0;
    return chunks ? launch_i8_rows<true>(p, stream) : launch_i8_rows<false>(p, stream);
}
