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

template <int MT, int NT, int WAVES, int BK, bool CAP>
__global__ __launch_bounds__(WAVES * 64) void logits_i8_kernel(I8Params p) {
    constexpr int T = WAVES * 64, KS = BK / 64, NF = NT / 16, MF = MT / 16;
    constexpr int CPR = BK / 16;                   /* 16-byte chunks in a staged row */
    constexpr int XC = MT * CPR / T;               /* chunks a thread stages */
    static_assert(MT * CPR % T == 0 && CPR % 8 == 0, "staging");
    __shared__ __align__(16) int8_t xs[2][MT * BK];
    const int t = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int mtiles = (p.rows + MT - 1) / MT;
    const int vt = blockIdx.x / mtiles, m0 = (blockIdx.x % mtiles) * MT;
    const int v0 = vt * (NT * WAVES) + wave * NT;
    const int lr = lane & 15, lk = lane >> 4;
    const int8_t *wrow[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) wrow[f] = p.w + (int64_t)min(v0 + f * 16 + lr, p.vocab - 1) * p.ldw + lk * 16;
    i4 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int f = 0; f < NF; f++) acc[m][f] = i4{0, 0, 0, 0};
    i4 xr[XC];
    auto load_x = [&](int k0) {
#pragma unroll
        for (int c = 0; c < XC; c++) {
            const int ch = t + c * T, r = ch / CPR, k = k0 + (ch % CPR) * 16;
            const int8_t *row = p.x + (int64_t)min(m0 + r, p.rows - 1) * p.ldx;
            xr[c] = k0 + BK <= p.n ? (i4)*(const i4_any *)(row + k) : load16_to(row, k, p.n);
        }
    };
    auto store_x = [&](int buf) {
#pragma unroll
        for (int c = 0; c < XC; c++) {
            const int ch = t + c * T, r = ch / CPR, cc = ch % CPR;
            *(i4 *)&xs[buf][r * BK + (cc ^ (r & 7)) * 16] = xr[c];
        }
    };
    auto load_w = [&](i4 (&w)[NF][KS], int k0) {
        if (k0 + BK <= p.n) {
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int s = 0; s < KS; s++) w[f][s] = *(const i4_any *)(wrow[f] + k0 + s * 64);
        } else {
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int s = 0; s < KS; s++) w[f][s] = load16_to(wrow[f] - lk * 16, k0 + s * 64 + lk * 16, p.n);
        }
    };
    auto compute = [&](const i4 (&w)[NF][KS], int buf) {
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int m = 0; m < MF; m++) {
                const int r = m * 16 + lr;
                const i4 b = *(const i4 *)&xs[buf][r * BK + ((s * 4 + lk) ^ (r & 7)) * 16];
#pragma unroll
                for (int f = 0; f < NF; f++)
                    acc[m][f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[f][s], b, acc[m][f], 0, 0, 0);
            }
        }
    };
    i4 w0[NF][KS], w1[NF][KS];
    load_x(0);
    load_w(w0, 0);
    store_x(0);
    __syncthreads();
    for (int k = 0; k < p.n; k += 2 * BK) {
        const bool more1 = k + BK < p.n, more2 = k + 2 * BK < p.n;
        if (more1) { load_x(k + BK); load_w(w1, k + BK); }
        compute(w0, 0);
        if (!more1) break;
        store_x(1);
        __syncthreads();
        if (more2) { load_x(k + 2 * BK); load_w(w0, k + 2 * BK); }
        compute(w1, 1);
        if (!more2) break;
        store_x(0);
        __syncthreads();
    }
#pragma unroll
    for (int f = 0; f < NF; f++) {
        const int v = v0 + f * 16 + lk * 4;
        float ws[4];
#pragma unroll
        for (int c = 0; c < 4; c++) ws[c] = p.w_scale[min(v + c, p.vocab - 1)];
#pragma unroll
        for (int m = 0; m < MF; m++) {
            const int r = m0 + m * 16 + lr;
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

template <int MT, int NT, int WAVES, int BK>
int launch_i8(const I8Params &p, hipStream_t stream) {
    const int64_t blocks = (((int64_t)p.vocab + NT * WAVES - 1) / (NT * WAVES)) * (((int64_t)p.rows + MT - 1) / MT);
    if (blocks > 0x7fffffff) return DLK_ERR_UNSUPPORTED;
    if (p.cap > 0.0f)
        hipLaunchKernelGGL((logits_i8_kernel<MT, NT, WAVES, BK, true>), dim3((unsigned)blocks), dim3(WAVES * 64), 0,
                           stream, p);
    else
        hipLaunchKernelGGL((logits_i8_kernel<MT, NT, WAVES, BK, false>), dim3((unsigned)blocks), dim3(WAVES * 64), 0,
                           stream, p);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
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
    if (rows <= 16) return launch_i8<16, 16, 4, 512>(p, stream);
    if (rows <= 32) return launch_i8<32, 16, 4, 512>(p, stream);
    if (rows <= 64) return launch_i8<64, 32, 4, 256>(p, stream);
    return launch_i8<128, 32, 4, 128>(p, stream);
}
