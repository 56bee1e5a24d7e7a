/*
 * logits_mx.hip -- an LM head in microscaled 4-bit floating point (dlk_logits_mx):
 *
 *   logits[r, v] = sum over blocks b of 2^(sx[r, b] + sw[v, b] - 254) * (x_r . w_v over the block's 32 values)
 *
 * v_mfma_scale_f32_16x16x128 takes four blocks of 16 rows of each side with their scales as
 * they are stored: nothing is unpacked or multiplied by a scale elsewhere.  Products of 4-bit
 * by 4- or 6-bit values are exact in it and its sums are in 32 bits (8-bit values, which it
 * takes too, it adds eight at a time to 2^-14 of the largest: not offered).  A lane's k-th
 * group of the instruction's four need not be the k-th block as long as both sides agree: of
 * 16 blocks lane group g takes 4 g .. 4 g + 3 in turn, whose four scales are one word of the
 * scales' row, picked by the instruction.  w is its first operand, as in logits_i8.hip.
 *
 * Bounds.  Few rows: w's bytes, as there (16 x 151,936 x 4,096 in 66 us with 6-bit hidden states, 5.1 TB/s; a large
 * copy: 4.9).  Many: the products and what feeds them, 512 x 262,144 x 4,096 in 380 us, 390-412 with the cap (24 such
 * calls one after another 385 to 520), of which some 80 write 537 MB after each workgroup's loop; between n = 4,096 and
 * 8,192 3.56 PFLOP/s (a library product of 16,384^3 in this format, written in 16 bits: 3.32 in all).  The matrix cores
 * are busy for 28 to 33% of a capped call's cycles (40% of the loop's), at a clock that goes from 2.1 down to 1.8 GHz
 * or less as such calls follow one another; the loop's LDS reads met none of the same bank once chunks lay as mx_spot() has
 * them, which changed nothing, nor did more stages of half the length.
 */
#include <math.h>

#include <type_traits>

#include "logit_row.h"
#include "logits_tile.h"

namespace dlk {

typedef int i2 __attribute__((ext_vector_type(2)));
typedef int i8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

struct MxParams {
    const uint8_t *x, *w, *xs, *ws;
    int64_t ldx, ldw, ldxs, ldws, ld;
    float *logits;
    int rows, vocab, blocks;
    float cap, recip;
    bool past;           /* stores go past the caches */
};

/* A wave's sums as logits (write_logits of logits_i8.hip without scales). */
template <bool CAP, bool WIDE, int MF, int NF>
DLK_DEV void write_sums(const MxParams &p, const f4 (&acc)[MF][NF], int m0, int v0, float *mine) {
    const int lane = lane_id(), lr = lane & 15, lk = lane >> 4;
    constexpr int LD = NF * 16 + 4, LPR = NF * 4, RPS = 64 / LPR;        /* lanes of a row, rows of a store */
    auto store = [&](int r, int v, const float (&y)[4]) {
        if (r >= p.rows) return;
        float *out = p.logits + (int64_t)r * p.ld + v;
        if (v + 3 < p.vocab) {
            store_past<4>(out, f4{y[0], y[1], y[2], y[3]}, p.past);
        } else {
#pragma unroll
            for (int c = 0; c < 3; c++)
                if (v + c < p.vocab) out[c] = y[c];
        }
    };
#pragma unroll
    for (int m = 0; m < MF; m++) {
#pragma unroll
        for (int f = 0; f < NF; f++) {
            float y[4];
#pragma unroll
            for (int c = 0; c < 4; c++) y[c] = CAP ? capped(acc[m][f][c], p.cap, p.recip) : acc[m][f][c];
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

/* One instruction: OPW and OPX are the bytes of the scale words, FMT the format of x. */
template <int FMT, int OPW, int OPX>
DLK_DEV f4 mx_mfma(i8 w, i8 x, f4 acc, int sw, int sx) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc, 4, FMT == DLK_MX_FP4 ? 4 : 2, OPW, sw, OPX, sx);
}

/* Chunk c of the PER chunks that each of the four lane groups has of a staged row lies at
 * mx_spot(c): in rows of 128 bytes the groups' chunks of one instruction side by side, else as
 * they come, a group's own: so place() spreads the groups that LDS serves together over the
 * banks (the other way round two of three reads of 512 rows met). mx_chunk: the inverse. */
template <int PER>
DLK_DEV int mx_spot(int c) { return PER == 2 ? c % PER * 4 + c / PER : c; }
template <int PER>
DLK_DEV int mx_chunk(int at) { return PER == 2 ? at % 4 * PER + at / 4 : at; }

/* What a workgroup stages of each step of NB blocks: rows of w and x in 16-byte chunks at
 * place() (an FP6 block's 24 bytes as its first and its last 16), then 16 bytes of scales a row
 * (NB = 8: those of this step and its neighbour). */
template <int FMT, int BM, int BN, int NB>
struct MxStage {
    static constexpr int CX = FMT == DLK_MX_FP4 ? 1 : 2;                 /* chunks of a block of x */
    static constexpr int WROW = NB * 16, XROW = NB * CX * 16;
    static constexpr int X = BN * WROW, SW = X + BM * XROW, SX = SW + BN * 16, END = SX + BM * 16;
    static constexpr int CHUNKS = END / 16;
};

/* The products of one staged step.  LAST: the row may end in it (blocks behind its end count as zeros). */
template <int FMT, int BM, int BN, int NB, bool LAST, int MF, int NF>
DLK_DEV void multiply_mx(const int8_t *lds, int wm, int wn, int it, int blocks, f4 (&acc)[MF][NF]) {
    typedef MxStage<FMT, BM, BN, NB> St;
    constexpr int PER = NB / 4;                    /* blocks of a lane group */
    const int lr = lane_id() & 15, g = lane_id() >> 4;
    const int8_t *const w = lds + (wn + lr) * St::WROW, *const x = lds + St::X + (wm + lr) * St::XROW;
    int sw[NF], sx[MF];
    auto scales = [&](const int8_t *at) {
        int v;
        if (NB == 16) v = *(const int *)(at + g * 4);
        else v = *(const uint16_t *)(at + (it & 1) * 8 + g * 2);
        if (LAST) {
            /* 1 in the place of those behind the row's end (255 among them would be NaN) */
            const int left = min(max(blocks - (it * NB + g * PER), 0), PER);
            const uint32_t keep = left >= 4 ? 0xffffffffu : (1u << (8 * left)) - 1;
            v = (int)(((uint32_t)v & keep) | (0x7f7f7f7fu & ~keep));
        }
        return v;
    };
#pragma unroll
    for (int f = 0; f < NF; f++) sw[f] = scales(lds + St::SW + (wn + f * 16 + lr) * 16);
#pragma unroll
    for (int m = 0; m < MF; m++) sx[m] = scales(lds + St::SX + (wm + m * 16 + lr) * 16);
    auto step = [&](auto number) {
        constexpr int s = decltype(number)::value;
        i8 a[NF], b[MF];
        const int c = g * PER + s;
#pragma unroll
        for (int f = 0; f < NF; f++) {
            const i4 v = *(const i4 *)&w[f * 16 * St::WROW + place<St::WROW>(lr, mx_spot<PER>(c)) * 16];
            a[f] = i8{v.x, v.y, v.z, v.w, 0, 0, 0, 0};
        }
        const bool some = !LAST || it * NB + c < blocks;
#pragma unroll
        for (int m = 0; m < MF; m++) {
            const int8_t *row = &x[m * 16 * St::XROW];
            if (FMT == DLK_MX_FP4) {
                const i4 v = *(const i4 *)&row[place<St::XROW>(lr, mx_spot<PER>(c)) * 16];
                b[m] = some ? i8{v.x, v.y, v.z, v.w, 0, 0, 0, 0} : i8{0, 0, 0, 0, 0, 0, 0, 0};
            } else {
                const i4 v = *(const i4 *)&row[place<St::XROW>(lr, mx_spot<2 * PER>(2 * c)) * 16];
                const i2 u = *(const i2 *)&row[place<St::XROW>(lr, mx_spot<2 * PER>(2 * c + 1)) * 16 + 8];
                b[m] = some ? i8{v.x, v.y, v.z, v.w, u.x, u.y, 0, 0} : i8{0, 0, 0, 0, 0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int m = 0; m < MF; m++)
#pragma unroll
            for (int f = 0; f < NF; f++) acc[m][f] = mx_mfma<FMT, s, s>(a[f], b[m], acc[m][f], sw[f], sx[m]);
    };
    step(std::integral_constant<int, 0>());
    step(std::integral_constant<int, 1>());
    if constexpr (PER == 4) {
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    }
}

/* BM rows of x and BN of w per workgroup, WGM x WGN waves, steps of NB blocks loaded straight
 * into LDS, ST stages in a ring: step it + ST - 1 is asked for while step it is multiplied, one
 * barrier a step. */
template <int FMT, int BM, int BN, int WGM, int WGN, int NB, int ST, bool CAP>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void logits_mx_kernel(MxParams p) {
    typedef MxStage<FMT, BM, BN, NB> St;
    constexpr int W = WGM * WGN, WM = BM / WGM, WN = BN / WGN, MF = WM / 16, NF = WN / 16;
    constexpr int NI = (St::CHUNKS + 64 * W - 1) / (64 * W);             /* loads of a wave per stage */
    constexpr int STAGE = NI * W * 1024;
    __shared__ __align__(1024) int8_t lds[ST * STAGE];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    int m0, v0;
    if (!tile_of<BM, BN>(p.rows, p.vocab, m0, v0)) return;
    const int steps = (p.blocks + NB - 1) / NB, whole = p.blocks / NB;
    /* this lane's chunk of load j: at src + min(it * per + first, last) * size */
    const uint8_t *src[NI];
    int first[NI], size[NI];
#pragma unroll
    for (int j = 0; j < NI; j++) {
        const int c = min(((j * W + wave) * 64 + lane), St::CHUNKS - 1) * 16;
        if (c < St::X) {
            const int r = c / St::WROW, k = place<St::WROW>(r, c % St::WROW / 16);
            src[j] = p.w + (int64_t)min(v0 + r, p.vocab - 1) * p.ldw;
            first[j] = mx_chunk<NB / 4>(k);
            size[j] = 16;
        } else if (c < St::SW) {
            const int r = (c - St::X) / St::XROW, k = place<St::XROW>(r, (c - St::X) % St::XROW / 16);
            const int b = mx_chunk<NB / 4 * St::CX>(k);
            src[j] = p.x + (int64_t)min(m0 + r, p.rows - 1) * p.ldx + (St::CX == 2 ? b % 2 * 8 : 0);
            first[j] = b / St::CX;
            size[j] = St::CX == 2 ? 24 : 16;
        } else {
            const bool of_w = c < St::SX;
            const int r = (c - (of_w ? St::SW : St::SX)) / 16;
            src[j] = of_w ? p.ws + (int64_t)min(v0 + r, p.vocab - 1) * p.ldws : p.xs + (int64_t)min(m0 + r, p.rows - 1) * p.ldxs;
            first[j] = 0;
            size[j] = 1;                           /* (a byte a block) */
        }
    }
    auto fetch = [&](int it, int slot) {
#pragma unroll
        for (int j = 0; j < NI; j++) {
            const int b = it * NB + first[j];
            const int at = size[j] == 1 ? b & ~15 : min(b, p.blocks - 1) * size[j];
            load_to_lds((const int8_t *)src[j] + at, &lds[slot * STAGE + (j * W + wave) * 1024]);
        }
    };
    const int wm = wave % WGM * WM, wn = wave / WGM * WN;
    f4 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int f = 0; f < NF; f++) acc[m][f] = f4{0.0f, 0.0f, 0.0f, 0.0f};
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
        multiply_mx<FMT, BM, BN, NB, false>(&lds[slot * STAGE], wm, wn, it, p.blocks, acc);
        slot = slot == ST - 1 ? 0 : slot + 1;
    }
    if (whole < steps) {                           /* a last, shorter step */
        wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        multiply_mx<FMT, BM, BN, NB, true>(&lds[slot * STAGE], wm, wn, whole, p.blocks, acc);
    }
    constexpr bool WIDE = NF >= 4;
    static_assert(!WIDE || W * 16 * (WN + 4) * 4 <= ST * STAGE, "room for the output");
    if (WIDE) __syncthreads();
    write_sums<CAP, WIDE>(p, acc, m0 + wm, v0 + wn, (float *)lds + (WIDE ? wave * 16 * (WN + 4) : 0));
}

/* The product of many rows in 4 bits: 256 x 256 tiles, eight waves of 128 x 64, steps of eight
 * blocks (128 bytes a row) in two stages of 64 KB, 16 scales a row every other step.  A step is
 * four quarters of 16 products, each with half of a half-step's rows of x; the quarter before
 * reads their fragments (the compiler alone reads two and waits), the last one the next
 * step's first, once that has arrived; the stage that it leaves is loaded again from there on.
 * Two rows' scales of a step share a word.  The last tiles of rows and ids lie over the ones
 * before them (at least 256 of each: the same sums again), so that a lane's rows are one stride
 * apart. */
template <bool CAP>
__global__ __launch_bounds__(512, 2) void logits_mx_wide_kernel(MxParams p) {
    constexpr int BM = 256, BN = 256, WM = 128, WN = 64, MF = 8, NF = 4, HF = MF / 2, W = 8, RPI = 8;
    constexpr int NX = BM / RPI / W, NW = BN / RPI / W;
    constexpr int XST = BM * 128, WST = BN * 128, SST = (BM + BN) * 16;
    __shared__ __align__(1024) int8_t lds[2 * (XST + WST + SST)];
    int8_t *const ldw = lds + 2 * XST, *const sc = ldw + 2 * WST;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    int m0, v0;
    if (!tile_of<BM, BN>(p.rows, p.vocab, m0, v0)) return;
    m0 = min(m0, p.rows - BM);
    v0 = min(v0, p.vocab - BN);
    /* this lane's rows: wave * 8 + lane / 8 of every 64; its block of a row's eight */
    const int block = mx_chunk<2>((lane % 8) ^ (lane / 8));
    const uint32_t row = (uint32_t)(wave * RPI + lane / 8);
    const uint32_t xat = row * (uint32_t)p.ldx, wat = row * (uint32_t)p.ldw;
    const uint8_t *const x0 = p.x + (int64_t)m0 * p.ldx, *const w0 = p.w + (int64_t)v0 * p.ldw;
    /* its row of scales: w's 256 are the first four waves', x's the others' */
    const bool of_w = wave < 4;
    const int srow = wave * 64 + lane;
    const uint8_t *const s0 = of_w ? p.ws + (int64_t)(v0 + wave * 64) * p.ldws : p.xs + (int64_t)(m0 + wave * 64 - BN) * p.ldxs;
    const uint32_t sat = (uint32_t)lane * (uint32_t)(of_w ? p.ldws : p.ldxs);
    const int steps = (p.blocks + 7) / 8;
    auto fetch = [&](int it) __attribute__((always_inline)) {
        const uint32_t k = (uint32_t)min(it * 8 + block, p.blocks - 1) * 16;
        const int slot = it & 1;
#pragma unroll
        for (int j = 0; j < NX; j++)
            load_to_lds((const int8_t *)(x0 + (int64_t)j * (RPI * W) * p.ldx) + (xat + k), &lds[slot * XST + (j * W + wave) * 1024]);
#pragma unroll
        for (int j = 0; j < NW; j++)
            load_to_lds((const int8_t *)(w0 + (int64_t)j * (RPI * W) * p.ldw) + (wat + k), &ldw[slot * WST + (j * W + wave) * 1024]);
        if ((it & 1) == 0) load_to_lds((const int8_t *)s0 + it * 8 + sat, &sc[(it >> 1 & 1) * SST + wave * 1024]);
    };
    /* of a row's last step, once this wave's loads are there: zeros for x's blocks behind its end, and 1 for their
     * scales (255 among them would be NaN) */
    auto end_rows = [&](int it) {
        if (it * 8 + block >= p.blocks) {
#pragma unroll
            for (int j = 0; j < NX; j++) *(i4 *)&lds[(it & 1) * XST + (j * W + wave) * 1024 + lane * 16] = i4{0, 0, 0, 0};
        }
        if ((it & 1) == 0 && it * 8 + 16 > p.blocks) {
            i4 *at = (i4 *)&sc[(it >> 1 & 1) * SST + srow * 16];
            i4 v = *at;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int left = p.blocks - it * 8 - 4 * c;                  /* scales of the word that count */
                const uint32_t keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1;
                v[c] = (int)(((uint32_t)v[c] & keep) | (0x7f7f7f7fu & ~keep));
            }
            *at = v;
        }
    };
    const int lr = lane & 15, g = lane >> 4, wm = wave % 2 * WM, wn = wave / 2 * WN;
    const int half0 = lr * 128 + (mx_spot<2>(2 * g) ^ (lr & 7)) * 16, half1 = lr * 128 + (mx_spot<2>(2 * g + 1) ^ (lr & 7)) * 16;
    auto take_w = [&](i4 (&a)[NF], int slot, int half) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < NF; f++) a[f] = *(const i4 *)&ldw[slot * WST + (wn + f * 16) * 128 + half];
    };
    auto take_x = [&](i4 (&b)[HF], int slot, int half, int from) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < HF; m++) b[m] = *(const i4 *)&lds[slot * XST + (wm + (from + m) * 16) * 128 + half];
    };
    typedef uint16_t h2 __attribute__((ext_vector_type(2)));
    auto take_scales = [&](h2 (&sw)[NF / 2], h2 (&sx)[MF / 2], int it) __attribute__((always_inline)) {
        const int8_t *at = &sc[(it >> 1 & 1) * SST + lr * 16 + (it & 1) * 8 + g * 2];
#pragma unroll
        for (int f = 0; f < NF / 2; f++)
            sw[f] = h2{*(const uint16_t *)(at + (wn + f * 32) * 16), *(const uint16_t *)(at + (wn + f * 32 + 16) * 16)};
#pragma unroll
        for (int m = 0; m < MF / 2; m++)
            sx[m] = h2{*(const uint16_t *)(at + (BN + wm + m * 32) * 16), *(const uint16_t *)(at + (BN + wm + m * 32 + 16) * 16)};
    };
    f4 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int f = 0; f < NF; f++) acc[m][f] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    const std::integral_constant<int, 0> zero;
    const std::integral_constant<int, 1> one;
    /* a quarter: half `half` of a step's blocks, x's fragments from `from` on; READS LDS reads (0x100) among its
     * products (0x8) */
    auto quarter = [&](auto half, auto from, auto reads, const i4 (&a)[NF], const i4 (&b)[HF], const h2 (&sw)[NF / 2],
                       const h2 (&sx)[MF / 2]) __attribute__((always_inline)) {
        constexpr int S = decltype(half)::value, FROM = decltype(from)::value * HF, READS = decltype(reads)::value;
        auto product = [&](auto mo, auto fo, int m2, int f2) __attribute__((always_inline)) {
            constexpr int M = decltype(mo)::value, F = decltype(fo)::value;
            const i4 av = a[2 * f2 + F], bv = b[2 * m2 + M];
            f4 &sum = acc[FROM + 2 * m2 + M][2 * f2 + F];
            sum = mx_mfma<DLK_MX_FP4, 2 * F + S, 2 * M + S>(
                i8{av.x, av.y, av.z, av.w, 0, 0, 0, 0}, i8{bv.x, bv.y, bv.z, bv.w, 0, 0, 0, 0}, sum,
                __builtin_bit_cast(int, sw[f2]), __builtin_bit_cast(int, sx[FROM / 2 + m2]));
        };
#pragma unroll
        for (int m2 = 0; m2 < HF / 2; m2++)
#pragma unroll
            for (int f2 = 0; f2 < NF / 2; f2++) {
                product(zero, zero, m2, f2);
                product(zero, one, m2, f2);
                product(one, zero, m2, f2);
                product(one, one, m2, f2);
            }
        constexpr int EACH = READS > 16 ? 2 : 1, GROUPS = READS / EACH;      /* reads at a time */
#pragma unroll
        for (int i = 0; i < GROUPS; i++) {
            __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, HF * NF - GROUPS, 0);
        __builtin_amdgcn_sched_barrier(0);
        /* (here: the compiler would move the products to the block in which their sums are used next) */
#pragma unroll
        for (int m = 0; m < HF; m++)
#pragma unroll
            for (int f = 0; f < NF; f++) asm volatile("" : "+v"(acc[FROM + m][f]));
    };
    i4 a0[NF], a1[NF], low[HF], high[HF];
    h2 sw[NF / 2], sx[MF / 2], nsw[NF / 2], nsx[MF / 2];
    fetch(0);
    if (steps > 1) {
        fetch(1);
        wait_loads<NX + NW>();
    } else {
        wait_loads<0>();
    }
    if (steps <= 2) {
        end_rows(0);
        wait_loads<0>();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    take_w(a0, 0, half0);
    take_x(low, 0, half0, 0);
    take_scales(sw, sx, 0);
    for (int it = 0; it < steps; it++) {
        const int slot = it & 1;
        take_x(high, slot, half0, HF);
        quarter(zero, zero, std::integral_constant<int, HF>(), a0, low, sw, sx);
        take_w(a1, slot, half1);
        take_x(low, slot, half1, 0);
        quarter(zero, one, std::integral_constant<int, HF + NF>(), a0, high, sw, sx);
        take_x(high, slot, half1, HF);
        quarter(one, zero, std::integral_constant<int, HF>(), a1, low, sw, sx);
        if (it + 1 < steps) {
            wait_loads<0>();                       /* step it + 1 is there; this wave has read all of step it */
            if (it + 3 >= steps) {                 /* (a row's last 16 scales may be two steps') */
                end_rows(it + 1);
                wait_loads<0>();
            }
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (it + 2 < steps) fetch(it + 2);
            take_w(a0, slot ^ 1, half0);
            take_x(low, slot ^ 1, half0, 0);
            take_scales(nsw, nsx, it + 1);
        }
        quarter(one, one, std::integral_constant<int, HF + NF + MF + NF>(), a1, high, sw, sx);
#pragma unroll
        for (int f = 0; f < NF / 2; f++) sw[f] = nsw[f];
#pragma unroll
        for (int m = 0; m < MF / 2; m++) sx[m] = nsx[m];
    }
    __syncthreads();
    write_sums<CAP, true>(p, acc, m0 + wm, v0 + wn, (float *)lds + wave * 16 * (WN + 4));
}

template <int FMT, int BM, int BN, int WGM, int WGN, int NB, int ST>
int launch_mx(const MxParams &p, hipStream_t stream) {
    const int64_t tiles = (((int64_t)p.vocab + BN - 1) / BN) * (((int64_t)p.rows + BM - 1) / BM);
    const int threads = WGM * WGN * 64;
    if ((tiles + 7) / 8 * 8 * threads > 0xffffffffLL) return DLK_ERR_UNSUPPORTED;      /* (no launch) */
    const dim3 grid((unsigned)((tiles + 7) / 8 * 8));
    if (p.cap > 0.0f)
        hipLaunchKernelGGL((logits_mx_kernel<FMT, BM, BN, WGM, WGN, NB, ST, true>), grid, dim3(threads), 0, stream, p);
    else
        hipLaunchKernelGGL((logits_mx_kernel<FMT, BM, BN, WGM, WGN, NB, ST, false>), grid, dim3(threads), 0, stream, p);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

int launch_mx_wide(const MxParams &p, hipStream_t stream) {
    const int64_t tiles = (((int64_t)p.vocab + 255) / 256) * (((int64_t)p.rows + 255) / 256);
    if ((tiles + 7) / 8 * 8 * 512 > 0xffffffffLL) return DLK_ERR_UNSUPPORTED;          /* (no launch) */
    const dim3 grid((unsigned)((tiles + 7) / 8 * 8));
    if (p.cap > 0.0f) hipLaunchKernelGGL(logits_mx_wide_kernel<true>, grid, dim3(512), 0, stream, p);
    else hipLaunchKernelGGL(logits_mx_wide_kernel<false>, grid, dim3(512), 0, stream, p);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

template <int FMT>
int launch_mx_tiles(const MxParams &p, hipStream_t stream) {
    /* Tiles by the rows (us at 151,936 ids of n = 4,096, hidden states of 4 and of 6 bits):
     *   16 rows     64 ids, 16 blocks a step, 2 stages 68, 70; 3 stages 69, 80; 128 ids, 8 blocks, 3 stages 71, 72
     *   32          128 ids, 8 blocks, 3 stages 78, 84; 64 ids, 16 blocks, 2 stages 78-83, 82; 256 ids 91, 99
     *   64          64 ids, 16 blocks, 2 stages 88, 126; 128 ids, 8 blocks, 3 stages 89, 95; 256 ids 93, 98
     *   128         128 x 128 111, 134; 128 x 256 117, 117
     *   200         256 x 256 142, -; 128 x 256 160, 172; 128 x 128 154, 237
     *   300         128 x 128 198, 332; 256 x 256 210, -; 128 x 256 220, 241
     *   512         256 x 256 by quarters 229; at once 234, -; 128 x 256 314, 354; 128 x 128 286, 458
     * (128 x 256 in 6 bits: a wave has 32 rows of 128 ids; with 64 of 64 120, 178, 252, 399.  256 x 256 at once: 64
     * rows of 128 ids; with 128 of 64 as long, and 200 x 50,257 x 1,024 24.2 for 22.5.  In 6 bits two stages of 256 x
     * 256 take 208 KB in steps of eight blocks, more than LDS has; in steps of four 112: not built) */
    if (p.rows <= 16) return launch_mx<FMT, 16, 64, 1, 4, 16, 2>(p, stream);
    if (p.rows <= 32) return launch_mx<FMT, 32, 128, 1, 4, 8, 3>(p, stream);
    if (FMT == DLK_MX_FP6) {
        if (p.rows <= 64) return launch_mx<DLK_MX_FP6, 64, 128, 2, 2, 8, 3>(p, stream);
        return launch_mx<DLK_MX_FP6, 128, 256, 4, 2, 8, 2>(p, stream);
    }
    if (p.rows <= 64) return launch_mx<DLK_MX_FP4, 64, 64, 2, 2, 16, 2>(p, stream);
    if (p.rows <= 128) return launch_mx<DLK_MX_FP4, 128, 128, 2, 2, 8, 2>(p, stream);
    if (p.rows < 256) return launch_mx<DLK_MX_FP4, 256, 256, 4, 2, 8, 2>(p, stream);
    /* past that tiles of 256 rows where they leave little empty (and a lane's offsets in a tile fit 32 bits) */
    const int64_t by128 = ((int64_t)p.rows + 127) / 128 * 128, by256 = ((int64_t)p.rows + 255) / 256 * 256;
    const bool near = ((p.ldx | p.ldw | p.ldxs | p.ldws) >> 22) == 0;
    if (by256 * 5 <= by128 * 6 && p.vocab >= 256 && near) return launch_mx_wide(p, stream);
    return launch_mx<DLK_MX_FP4, 128, 128, 2, 2, 8, 2>(p, stream);
}

}  // namespace dlk

extern "C" int dlk_logits_mx(const uint8_t *x, int x_format, int64_t ldx, const uint8_t *x_scale, int64_t ldxs,
                             const uint8_t *w, int64_t ldw, const uint8_t *w_scale, int64_t ldws, int rows, int vocab,
                             int n, float softcap, float *logits, int64_t ld, hipStream_t stream) {
    using namespace dlk;
    if (!x || !x_scale || !w || !w_scale || !logits || rows < 0 || vocab <= 0 || n <= 0) return DLK_ERR_INVALID;
    if (x_format != DLK_MX_FP4 && x_format != DLK_MX_FP6) return DLK_ERR_INVALID;
    const int64_t blocks = ((int64_t)n + 31) / 32, scales = (blocks + 15) / 16 * 16;
    const int64_t bytes = blocks * (x_format == DLK_MX_FP4 ? 16 : 24);
    /* (the stride of a single row says nothing) */
    if ((rows > 1 && (ldx < bytes || ldxs < scales)) || (vocab > 1 && (ldw < blocks * 16 || ldws < scales)) || ld < vocab)
        return DLK_ERR_INVALID;
    if (!(fabsf(softcap) < INFINITY)) return DLK_ERR_INVALID;
    if ((((uintptr_t)x | (uint64_t)(rows > 1 ? ldx : 0)) & (x_format == DLK_MX_FP4 ? 15 : 7)) != 0) return DLK_ERR_INVALID;
    if ((((uintptr_t)w | (uintptr_t)x_scale | (uintptr_t)w_scale | (uint64_t)(rows > 1 ? ldxs : 0) |
          (uint64_t)(vocab > 1 ? ldw | ldws : 0)) & 15) != 0 || ((uintptr_t)logits & 3) != 0)
        return DLK_ERR_INVALID;
    /* int indices of a row's bytes */
    if (n > 0x3fffffff || vocab > 0x7fffffff - 65536 || rows > 0x7fffffff - 65536) return DLK_ERR_UNSUPPORTED;
    if (rows == 0) return DLK_OK;
    /* a cap below 2^-128 has no reciprocal among the floats: the product without it, then the cap by exact quotients */
    if (softcap > 0.0f && 1.0f / softcap == INFINITY) {
        int rc = dlk_logits_mx(x, x_format, ldx, x_scale, ldxs, w, ldw, w_scale, ldws, rows, vocab, n, 0.0f, logits, ld, stream);
        for (int64_t r = 0; rc == DLK_OK && r < rows; r += 65535)
            rc = dlk_softcap(logits + r * ld, ld, (int)(rows - r < 65535 ? rows - r : 65535), vocab, softcap, stream);
        return rc;
    }
    MxParams p;
    p.x = x; p.w = w; p.xs = x_scale; p.ws = w_scale;
    p.ldx = ldx; p.ldw = ldw; p.ldxs = ldxs; p.ldws = ldws; p.ld = ld;
    p.logits = logits;
    p.rows = rows; p.vocab = vocab; p.blocks = (int)blocks;
    p.cap = softcap > 0.0f ? softcap : 0.0f;
    p.recip = p.cap > 0.0f ? 1.0f / p.cap : 0.0f;
    /* Past the caches where a call that reads the logits next would not find them: more than L2 holds, or much beside
     * the weights that went through it (us of the product and of the scores after it, through / past:
     * 16 x 151,936 x 4,096 76.5 / 75.5, x 1,024 26.7 / 27.8; 64 x 151,936 x 1,024 42.6 / 39.8;
     * 64 x 50,257 x 4,096 35.4 / 36.2; 4 x 151,936 x 4,096 67.7 / 68.2) */
    const int64_t out = (int64_t)rows * vocab * 4, in = (int64_t)vocab * blocks * 17;
    p.past = (out >= 32 << 20 || (out >= 8 << 20 && in + out >= 128 << 20)) && whole_lines(logits, ld * 4);
    return x_format == DLK_MX_FP4 ? launch_mx_tiles<DLK_MX_FP4>(p, stream) : launch_mx_tiles<DLK_MX_FP6>(p, stream);
}
