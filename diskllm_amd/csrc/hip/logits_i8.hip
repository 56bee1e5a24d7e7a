/*
 * logits_i8.hip -- an LM head in 8-bit integers: logits[r, v] = (x_r . w_v) * x_scale[r] *
 * w_scale[v], the soft-cap as epilogue (dlk_logits_i8).
 *
 * The sum is exact (v_mfma_i32_16x16x64_i8; 131,071 products of +-128 by +-128 fit in 32 bits), so no order
 * of n matters: no tile or split changes a bit.  w is the instruction's first operand: a
 * lane's four results are then four neighbouring ids of one row, one 16-byte store.
 *
 * Bounds.  Up to 128 rows w's bytes: each is read from memory once (the tiles of x for
 * one tile of w lie side by side on one XCD), and what it takes is loads in flight: both
 * operands go straight into an LDS ring (global_load_lds, 16 bytes a lane), which costs no
 * registers and no waits but one barrier a step.  16 x 151,936 x 4,096 takes 114-116 us,
 * 5.5-5.7 TB/s (a large copy: 5.1); 1 x 32,000 x 2,048 11.5, 5.7 TB/s.  Above that the
 * products and what feeds them: 512 x 262,144 x 4,096 with the cap in 605-639 us (by the box and its
 * clock), 1,720-1,820 TOP/s, of which some 150 cap and write 537 MB of logits after each workgroup's
 * loop; the loop alone runs at 2,440, as a library product of 16,384^3 does.  It has the
 * loads into LDS at about 12 TB/s, where shorter steps, a third stage of w, another order of n
 * and stores that bypass the caches gave nothing; tiles of 256 x 256 ask for the fewest bytes.
 *
 * Between 129 and 511 rows neither is reached: tiles leave rows empty (300 are computed as 384),
 * and 147 KB of stages leave one workgroup a CU, with nothing beside its epilogue: 200 x
 * 151,936 x 4,096 215 us and 300 rows 282, where the bytes are 147 and 159 at a copy's rate.  And
 * tiles go by the rows alone, not by the rounds of the CUs that they make: 512 x 100,000 x 1,200,
 * 3.05 rounds, takes 131 where the operations are 64.
 *
 * Rows that are not 16-byte aligned cannot go that way: they go through registers
 * (logits_i8_any_kernel; 33 x 50,257 x 2,047 33.3-35.9 us, 3.1-3.3 TB/s, in padded rows 27).  Their
 * 16-byte loads are what it waits for: both stages wholly in flight (no branch in the loop) or
 * steps twice as long were no faster, nor was loading the rows' own chunks into LDS and
 * reading fragments at each row's shift (59 us: unaligned LDS reads).
 */
#include <math.h>

#include <hip/hip_runtime.h>

#include "dlk_device.h"
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

/* A wave's MF x NF fragments of sums as logits: rows m0 .., ids v0 ...  A fragment's lane
 * holds four ids of one row; where WIDE, 16 rows at a time go through the wave's own 16 *
 * (NF * 16 + 4) floats of LDS, so that a store writes whole rows of NF * 64 bytes (512 x
 * 262,144 out of n = 512: 252 -> 181 us), else each lane stores its own 16 bytes. */
template <bool CAP, bool WIDE, int MF, int NF>
DLK_DEV void write_logits(const I8Params &p, const i4 (&acc)[MF][NF], int m0, int v0, float *mine) {
    const int lane = lane_id(), lr = lane & 15, lk = lane >> 4;
    constexpr int LD = NF * 16 + 4, LPR = NF * 4, RPS = 64 / LPR;        /* lanes of a row, rows of a store */
    auto store = [&](int r, int v, const float (&y)[4]) {
        if (r >= p.rows) return;
        float *out = p.logits + (int64_t)r * p.ld + v;
        if (v + 3 < p.vocab) {
            store4(out, make_float4(y[0], y[1], y[2], y[3]));
        } else {
#pragma unroll
            for (int c = 0; c < 3; c++)
                if (v + c < p.vocab) out[c] = y[c];
        }
    };
    float ws[NF][4];
#pragma unroll
    for (int f = 0; f < NF; f++)
#pragma unroll
        for (int c = 0; c < 4; c++) ws[f][c] = p.w_scale[min(v0 + f * 16 + lk * 4 + c, p.vocab - 1)];
    float sx[MF];
#pragma unroll
    for (int m = 0; m < MF; m++) sx[m] = p.x_scale[min(m0 + m * 16 + lr, p.rows - 1)];
    /* (here, before the first store: waited for later, a load waits for the stores before it too) */
#pragma unroll
    for (int m = 0; m < MF; m++) asm volatile("" : "+v"(sx[m]));
#pragma unroll
    for (int m = 0; m < MF; m++) {
#pragma unroll
        for (int f = 0; f < NF; f++) {
            float y[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                y[c] = (float)acc[m][f][c] * sx[m] * ws[f][c];
                if (CAP) y[c] = capped(y[c], p.cap, p.recip);
            }
            if (WIDE) *(float4 *)&mine[lr * LD + f * 16 + lk * 4] = make_float4(y[0], y[1], y[2], y[3]);
            else store(m0 + m * 16 + lr, v0 + f * 16 + lk * 4, y);
        }
        if (WIDE) {
#pragma unroll
            for (int i = 0; i < 16 / RPS; i++) {
                const int r = i * RPS + lane / LPR, c = lane % LPR * 4;
                const float4 q = *(const float4 *)&mine[r * LD + c];
                const float y[4] = {q.x, q.y, q.z, q.w};
                store(m0 + m * 16 + r, v0 + c, y);
            }
        }
    }
}

/* Loads 16 bytes a lane straight into LDS: lane i's to dst + 16 i (dst the same in all lanes). */
DLK_DEV void load_to_lds(const int8_t *src, int8_t *dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                     (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
}

/* Of a last, shorter step the chunks past n are copies of the last one (so that all lanes load):
 * this lane's chunk of x at k, once it is in LDS, gets zeros for what is past n.  What w has
 * there does not matter then. */
DLK_DEV void end_row(int8_t *chunk, int k, int n) {
    if (k + 16 <= n) return;
    i4 v = *(const i4 *)chunk;
    const int keep = max(n - k, 0);                /* bytes */
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int b = keep - 4 * c;
        v[c] = b >= 4 ? v[c] : b <= 0 ? 0 : v[c] & ((1 << (8 * b)) - 1);
    }
    *(i4 *)chunk = v;
}

/* One tile's place: workgroups go to the XCDs in turn, so each XCD gets a run of tiles, the
 * tiles of x for one tile of w side by side: w comes from memory once. */
template <int BM, int BN>
DLK_DEV bool tile_of(const I8Params &p, int &m0, int &v0) {
    const int mtiles = (p.rows + BM - 1) / BM, vtiles = (p.vocab + BN - 1) / BN;
    const int tile = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
    m0 = tile % mtiles * BM;
    v0 = tile / mtiles * BN;
    return tile < mtiles * vtiles;
}

/* The products of one staged step: x in xs, w in ws, BK bytes a row, chunks at place(). */
template <int BK, int MF, int NF>
DLK_DEV void multiply_stage(const int8_t *xs, const int8_t *ws, i4 (&acc)[MF][NF]) {
    const int lr = lane_id() & 15, lk = lane_id() >> 4;
#pragma unroll
    for (int s = 0; s < BK / 64; s++) {
        const int at = lr * BK + place<BK>(lr, s * 4 + lk) * 16;      /* (tiles start at multiples of 16 rows) */
        i4 a[NF], b[MF];
#pragma unroll
        for (int f = 0; f < NF; f++) a[f] = *(const i4 *)&ws[f * 16 * BK + at];
#pragma unroll
        for (int m = 0; m < MF; m++) b[m] = *(const i4 *)&xs[m * 16 * BK + at];
#pragma unroll
        for (int m = 0; m < MF; m++)
#pragma unroll
            for (int f = 0; f < NF; f++)
                acc[m][f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[f], b[m], acc[m][f], 0, 0, 0);
    }
}

template <int MF, int NF>
DLK_DEV void clear(i4 (&acc)[MF][NF]) {
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int f = 0; f < NF; f++) acc[m][f] = i4{0, 0, 0, 0};
}

/* Rows of whole 16-byte chunks: BM rows of x and BN of w per workgroup, WGM x WGN waves, steps
 * of BK bytes of n loaded straight into LDS, ST stages in a ring: step it + ST - 1 is asked
 * for while step it is multiplied, one barrier a step.  The loop holds nothing but that: with
 * the last, shorter step in it the compiler waited for every load before each LDS read.  Few
 * rows are bound by w's bytes: two workgroups a CU fill its LDS with loads in flight, long
 * pieces of w's rows at a time (16 x 151,936 x 4,096: 116 us, 5.5 TB/s). */
template <int BM, int BN, int WGM, int WGN, int BK, int ST, bool CAP>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void logits_i8_kernel(I8Params p) {
    constexpr int W = WGM * WGN, WM = BM / WGM, WN = BN / WGN, MF = WM / 16, NF = WN / 16;
    constexpr int CPR = BK / 16, RPI = 64 / CPR;   /* chunks of a row; rows that a wave loads at once */
    constexpr int NI = (BM + BN) / RPI / W;        /* loads of a wave per stage */
    constexpr int STAGE = (BM + BN) * BK;
    static_assert((BM + BN) % (RPI * W) == 0 && BM % (RPI * W) == 0 && BK >= 64 && BK <= 512, "tiles");
    __shared__ __align__(1024) int8_t lds[ST * STAGE];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    int m0, v0;
    if (!tile_of<BM, BN>(p, m0, v0)) return;
    const int8_t *src[NI];                         /* the row of this lane's chunk */
    int at[NI];                                    /* and its place in the row */
#pragma unroll
    for (int j = 0; j < NI; j++) {
        const int r = (j * W + wave) * RPI + lane / CPR;
        at[j] = place<BK>(r, lane % CPR) * 16;
        src[j] = r < BM ? p.x + (int64_t)min(m0 + r, p.rows - 1) * p.ldx
                        : p.w + (int64_t)min(v0 + r - BM, p.vocab - 1) * p.ldw;
    }
    const int last = (p.n - 1) & ~15;              /* (behind a row's end at most the rest of its last chunk is loaded) */
    auto fetch = [&](int it, int slot) {
#pragma unroll
        for (int j = 0; j < NI; j++)
            load_to_lds(src[j] + min(it * BK + at[j], last), &lds[slot * STAGE + (j * W + wave) * 1024]);
    };
    const int wm = wave % WGM * WM, wn = wave / WGM * WN;
    i4 acc[MF][NF];
    clear(acc);
    const int whole = p.n / BK, steps = (p.n + BK - 1) / BK;
#pragma unroll
    for (int s = 0; s < ST - 1; s++)
        if (s < steps) fetch(s, s);
    int slot = 0;
    for (int it = 0; it < whole; it++) {
        if (it + ST - 2 < steps) wait_loads<NI *(ST - 2)>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        /* the slot that step it - 1 has left */
        if (it + ST - 1 < steps) fetch(it + ST - 1, slot == 0 ? ST - 1 : slot - 1);
        multiply_stage<BK>(&lds[slot * STAGE + wm * BK], &lds[slot * STAGE + (BM + wn) * BK], acc);
        slot = slot == ST - 1 ? 0 : slot + 1;
    }
    if (whole < steps) {                           /* a last, shorter step */
        wait_loads<0>();
#pragma unroll
        for (int j = 0; j < BM / (RPI * W); j++)   /* (x's rows are the first loads) */
            end_row(&lds[slot * STAGE + (j * W + wave) * 1024 + lane * 16], whole * BK + at[j], p.n);
        __syncthreads();
        multiply_stage<BK>(&lds[slot * STAGE + wm * BK], &lds[slot * STAGE + (BM + wn) * BK], acc);
    }
    constexpr bool WIDE = NF >= 4;
    static_assert(!WIDE || W * 16 * (WN + 4) * 4 <= ST * STAGE, "room for the output");
    if (WIDE) __syncthreads();
    write_logits<CAP, WIDE>(p, acc, m0 + wm, v0 + wn, (float *)lds + (WIDE ? wave * 16 * (WN + 4) : 0));
}

/* Rows of any alignment: as above through registers, two stages in LDS and two on their
 * way, so that a step's loads have two steps' time. */
template <int BM, int BN, int WGM, int WGN, int BK, bool CAP>
__global__ __launch_bounds__(WGM * WGN * 64, BM == 32 ? 3 : 4) void logits_i8_any_kernel(I8Params p) {
    constexpr int W = WGM * WGN, WM = BM / WGM, WN = BN / WGN, MF = WM / 16, NF = WN / 16;
    constexpr int CPR = BK / 16, RPI = 64 / CPR, NI = (BM + BN) / RPI / W, STAGE = (BM + BN) * BK;
    static_assert((BM + BN) % (RPI * W) == 0 && BM % RPI == 0 && BK >= 64 && BK <= 512, "tiles");
    __shared__ __align__(1024) int8_t lds[2 * STAGE];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    int m0, v0;
    if (!tile_of<BM, BN>(p, m0, v0)) return;
    const int8_t *src[NI];
    int at[NI];
#pragma unroll
    for (int j = 0; j < NI; j++) {
        const int r = (j * W + wave) * RPI + lane / CPR;
        at[j] = place<BK>(r, lane % CPR) * 16;
        src[j] = r < BM ? p.x + (int64_t)min(m0 + r, p.rows - 1) * p.ldx
                        : p.w + (int64_t)min(v0 + r - BM, p.vocab - 1) * p.ldw;
    }
    auto load = [&](i4 (&reg)[NI], int k0) {
        if (k0 + BK <= p.n) {
#pragma unroll
            for (int j = 0; j < NI; j++) reg[j] = *(const i4_any *)(src[j] + k0 + at[j]);
        } else {
#pragma unroll
            for (int j = 0; j < NI; j++) reg[j] = load16_to(src[j], k0 + at[j], p.n);
        }
    };
    auto put = [&](const i4 (&reg)[NI], int slot) {
#pragma unroll
        for (int j = 0; j < NI; j++) *(i4 *)&lds[slot * STAGE + (j * W + wave) * 1024 + lane * 16] = reg[j];
    };
    const int wm = wave % WGM * WM, wn = wave / WGM * WN;
    i4 acc[MF][NF], even[NI], odd[NI];
    clear(acc);
    const int steps = (p.n + BK - 1) / BK;
    load(even, 0);
    if (steps > 1) load(odd, BK);
    put(even, 0);
    for (int it = 0; it < steps; it += 2) {
        __syncthreads();
        if (it + 2 < steps) load(even, (it + 2) * BK);
        multiply_stage<BK>(&lds[wm * BK], &lds[(BM + wn) * BK], acc);
        if (it + 1 >= steps) break;
        put(odd, 1);
        __syncthreads();
        if (it + 3 < steps) load(odd, (it + 3) * BK);
        multiply_stage<BK>(&lds[STAGE + wm * BK], &lds[STAGE + (BM + wn) * BK], acc);
        if (it + 2 < steps) put(even, 0);
    }
    write_logits<CAP, false>(p, acc, m0 + wm, v0 + wn, nullptr);
}

/* The product of many rows: 256 x 256 tiles, eight waves of 128 x 64, steps of 128 bytes (whole
 * cache lines: 64 cost 8% more) in two stages of 64 KB.  Each half-step's fragments are read
 * into registers while the matrix cores work on the half-step before, the reads spread
 * between the products (sched_group_barrier; the compiler alone puts them last), and a stage
 * is loaded again as soon as its second half is in registers. */
template <bool CAP>
__global__ __launch_bounds__(512, 2) void logits_i8_wide_kernel(I8Params p) {
    constexpr int BM = 256, BN = 256, BK = 128, WGM = 2, WM = 128, WN = 64, MF = 8, NF = 4;
    constexpr int W = 8, RPI = 8, NX = BM / RPI / W, NW = BN / RPI / W, XST = BM * BK, WST = BN * BK;
    __shared__ __align__(1024) int8_t lds[2 * (XST + WST)];
    int8_t *const ldw = lds + 2 * XST;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    int m0, v0;
    if (!tile_of<BM, BN>(p, m0, v0)) return;
    const int8_t *sx[NX], *sw[NW];                 /* rows (a wave's loads have one row in eight: one place in all) */
    const int at = place<BK>(lane / 8, lane % 8) * 16;
#pragma unroll
    for (int j = 0; j < NX; j++) sx[j] = p.x + (int64_t)min(m0 + (j * W + wave) * RPI + lane / 8, p.rows - 1) * p.ldx;
#pragma unroll
    for (int j = 0; j < NW; j++) sw[j] = p.w + (int64_t)min(v0 + (j * W + wave) * RPI + lane / 8, p.vocab - 1) * p.ldw;
    const int last = (p.n - 1) & ~15;              /* (behind a row's end at most the rest of its last chunk is loaded) */
    auto fetch = [&](int it, int slot) {
        const int k = min(it * BK + at, last);
#pragma unroll
        for (int j = 0; j < NX; j++) load_to_lds(sx[j] + k, &lds[slot * XST + (j * W + wave) * 1024]);
#pragma unroll
        for (int j = 0; j < NW; j++) load_to_lds(sw[j] + k, &ldw[slot * WST + (j * W + wave) * 1024]);
    };
    auto end_rows = [&](int it) {                  /* of a last, shorter step, once this wave's loads are there */
#pragma unroll
        for (int j = 0; j < NX; j++) end_row(&lds[(it & 1) * XST + (j * W + wave) * 1024 + lane * 16], it * BK + at, p.n);
    };
    const int lr = lane & 15, lk = lane >> 4, wm = wave % WGM * WM, wn = wave / WGM * WN;
    const int half0 = lr * BK + place<BK>(lr, lk) * 16, half1 = lr * BK + place<BK>(lr, 4 + lk) * 16;
    auto take = [&](i4 (&a)[NF], i4 (&b)[MF], int slot, int half) {
        const int8_t *xs = &lds[slot * XST + wm * BK + half], *ws = &ldw[slot * WST + wn * BK + half];
#pragma unroll
        for (int f = 0; f < NF; f++) a[f] = *(const i4 *)&ws[f * 16 * BK];
#pragma unroll
        for (int m = 0; m < MF; m++) b[m] = *(const i4 *)&xs[m * 16 * BK];
    };
    i4 acc[MF][NF];
    clear(acc);
    auto multiply = [&](const i4 (&a)[NF], const i4 (&b)[MF]) {
#pragma unroll
        for (int m = 0; m < MF; m++)
#pragma unroll
            for (int f = 0; f < NF; f++)
                acc[m][f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[f], b[m], acc[m][f], 0, 0, 0);
        /* one LDS read (0x100), two products (0x8), over and over; then the other products */
#pragma unroll
        for (int i = 0; i < MF + NF; i++) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, MF * NF - 2 * (MF + NF), 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    i4 a0[NF], b0[MF], a1[NF], b1[MF];
    const int steps = (p.n + BK - 1) / BK, shorter = p.n % BK != 0 ? steps - 1 : -1;
    fetch(0, 0);
    if (steps > 1) {
        fetch(1, 1);
        wait_loads<NX + NW>();
    } else {
        wait_loads<0>();
        if (shorter == 0) end_rows(0);
        wait_loads<0>();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    take(a0, b0, 0, half0);
    for (int it = 0; it < steps; it++) {
        take(a1, b1, it & 1, half1);
        multiply(a0, b0);
        if (it + 1 < steps) {
            wait_loads<0>();                       /* step it + 1 is there; this wave has read all of step it */
            if (it + 1 == shorter) {
                end_rows(it + 1);
                wait_loads<0>();
            }
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (it + 2 < steps) fetch(it + 2, it & 1);
            take(a0, b0, (it + 1) & 1, half0);
        }
        multiply(a1, b1);
    }
    __syncthreads();
    write_logits<CAP, true>(p, acc, m0 + wm, v0 + wn, (float *)lds + wave * 16 * (WN + 4));
}

/* One launch of `kernel`, tiles of BM x BN; the grid a multiple of the XCDs. */
int launch_tiles(void (*kernel)(I8Params), int bm, int bn, int threads, const I8Params &p, hipStream_t stream) {
    const int64_t tiles = (((int64_t)p.vocab + bn - 1) / bn) * (((int64_t)p.rows + bm - 1) / bm);
    if ((tiles + 7) / 8 * 8 * threads > 0xffffffffLL) return DLK_ERR_UNSUPPORTED;      /* (no launch) */
    hipLaunchKernelGGL(kernel, dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(threads), 0, stream, p);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

template <int BM, int BN, int WGM, int WGN, int BK, int ST>
int launch_i8(const I8Params &p, hipStream_t stream) {
    return launch_tiles(p.cap > 0.0f ? logits_i8_kernel<BM, BN, WGM, WGN, BK, ST, true>
                                     : logits_i8_kernel<BM, BN, WGM, WGN, BK, ST, false>, BM, BN, WGM * WGN * 64, p, stream);
}

template <int BM, int BN, int WGM, int WGN, int BK>
int launch_i8_any(const I8Params &p, hipStream_t stream) {
    return launch_tiles(p.cap > 0.0f ? logits_i8_any_kernel<BM, BN, WGM, WGN, BK, true>
                                     : logits_i8_any_kernel<BM, BN, WGM, WGN, BK, false>, BM, BN, WGM * WGN * 64, p, stream);
}

int launch_i8_wide(const I8Params &p, hipStream_t stream) {
    return launch_tiles(p.cap > 0.0f ? logits_i8_wide_kernel<true> : logits_i8_wide_kernel<false>, 256, 256, 512, p, stream);
}

}  // namespace dlk

extern "C" int dlk_logits_i8(const int8_t *x, int64_t ldx, const float *x_scale, const int8_t *w, int64_t ldw,
                             const float *w_scale, int rows, int vocab, int n, float softcap, float *logits, int64_t ld,
                             hipStream_t stream) {
    using namespace dlk;
    if (!x || !x_scale || !w || !w_scale || !logits || rows < 0 || vocab <= 0 || n <= 0) return DLK_ERR_INVALID;
    if (ldx < n || ldw < n || ld < vocab || !(fabsf(softcap) < INFINITY)) return DLK_ERR_INVALID;
    if ((((uintptr_t)x_scale | (uintptr_t)w_scale | (uintptr_t)logits) & 3) != 0) return DLK_ERR_INVALID;
    /* |sum| <= 128 * 128 * n in 32 bits; int indices */
    if (n > 131071 || vocab > 0x7fffffff - 65536 || rows > 0x7fffffff - 65536) return DLK_ERR_UNSUPPORTED;
    if (rows == 0) return DLK_OK;
    /* a cap below 2^-128 has no reciprocal among the floats: the product without it, then the cap by exact quotients */
    if (softcap > 0.0f && 1.0f / softcap == INFINITY) {
        int rc = dlk_logits_i8(x, ldx, x_scale, w, ldw, w_scale, rows, vocab, n, 0.0f, logits, ld, stream);
        for (int64_t r = 0; rc == DLK_OK && r < rows; r += 65535)
            rc = dlk_softcap(logits + r * ld, ld, (int)(rows - r < 65535 ? rows - r : 65535), vocab, softcap, stream);
        return rc;
    }
    I8Params p;
    p.x = x; p.w = w; p.ldx = ldx; p.ldw = ldw; p.ld = ld;
    p.x_scale = x_scale; p.w_scale = w_scale; p.logits = logits;
    p.rows = rows; p.vocab = vocab; p.n = n;
    p.cap = softcap > 0.0f ? softcap : 0.0f;
    p.recip = p.cap > 0.0f ? 1.0f / p.cap : 0.0f;
    /* Tiles by the rows (us at 32,000 and 151,936 ids of n = 4,096; the smallest tile that holds
     * the rows unless said otherwise):
     *   16 rows     64 ids of 512 bytes a step 27.4, 116; of 256 bytes and 4 stages 28.4, 119
     *   32          64 ids of 256 bytes 30.1, 128; 128 ids of 128 bytes 32.7, 130
     *   64          64 ids of 128 bytes 34.8, 145; of 256 bytes 34.2, 163
     *   128         128 ids of 64 bytes 41.3, 173; of 128 bytes 44.5, 190
     *   200         128 x 256 47.9, 219; 128 x 128 58.1, 234; 256 x 256 62.2, 221
     *   300         128 x 256 76.5, 283; 256 x 256 67.5, 306
     *   512         256 x 256 (262,144 ids) 558; 128 x 256 657; 128 x 128 787 */
    /* (the stride of a single row says nothing) */
    const int64_t strides = (rows > 1 ? ldx : 0) | (vocab > 1 ? ldw : 0);
    const bool chunks = (((uintptr_t)x | (uintptr_t)w | (uintptr_t)strides) & 15) == 0;
    if (!chunks) {
        /* (33 x 50,257 x 2,047: 35.6; 300 x 100,001 x 4,097: 433, in tiles of 128 rows 562) */
        if (rows <= 16) return launch_i8_any<16, 64, 1, 4, 256>(p, stream);
        if (rows <= 32) return launch_i8_any<32, 64, 1, 4, 256>(p, stream);
        return launch_i8_any<64, 128, 2, 4, 128>(p, stream);
    }
    if (rows <= 16) return launch_i8<16, 64, 1, 4, 512, 2>(p, stream);
    if (rows <= 32) return launch_i8<32, 64, 2, 2, 256, 3>(p, stream);
    if (rows <= 64) return launch_i8<64, 64, 2, 2, 128, 4>(p, stream);
    if (rows <= 128) return launch_i8<128, 128, 2, 2, 64, 3>(p, stream);
    /* past that tiles of 256 rows where they leave little empty */
    const int64_t by128 = ((int64_t)rows + 127) / 128 * 128, by256 = ((int64_t)rows + 255) / 256 * 256;
    if (rows <= 384 || by128 * 6 < by256 * 5) return launch_i8<128, 256, 2, 4, 128, 3>(p, stream);
    return launch_i8_wide(p, stream);
}
