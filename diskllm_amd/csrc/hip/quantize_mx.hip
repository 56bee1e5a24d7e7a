/*
 * quantize_mx.hip -- microscaled blocks of 32 values (dlk_quantize_mx), and the values they
 * stand for (dlk_dequantize_mx).
 *
 *   e = floor(log2(max |x|)) - 2, held as e + 127 in a byte;  element = x / 2^e to the nearest of the format
 *
 * Both formats' largest element has the exponent 2, so the byte is the exponent field of the
 * block's largest float less 2, and nothing is divided.  Elements: the hardware's
 * conversions, which round halves to even and take denormals as they are: FP4 as it is; FP6
 * (E2M3) as 8-bit E4M3 of x / 2^(e + 6), whose codes from 0 to 31, denormals included, are
 * E2M3's, with x held to the largest element first.
 *
 * Bound by memory: eight values a thread (16-byte loads of 16-bit types), four threads a
 * block, a wave's 64 groups side by side over the ends of rows, four such spans a wave.
 * 100,001 x 4,090 bfloat16 to 4 bits 198-226 us, 4.6-5.3 TB/s (a large copy: 4.9), and back 176,
 * 5.8; 8,192 rows of a table of 151,936 x 4,096 by id as float32 23.7, 6.4; one row of 4,096 3.4
 * and 3.1, a launch and a round trip.  Eight spans a wave, or two, were no faster.
 */
#include "logit_row.h"

namespace dlk {

constexpr int kMxThreads = 256;
constexpr int kMxSpans = 4;                        /* groups of eight values a thread */

/* Where group `i` of a wave's span lies: row and group of the row (`per` to a row), found for the wave's first and
 * moved on. */
DLK_DEV void mx_place(uint64_t first, uint32_t per, int lane, int64_t &row, uint32_t &unit) {
    const uint64_t r = first < 0xffffffffull ? (uint64_t)((uint32_t)first / per) : first / per;
    row = (int64_t)r;
    uint32_t u = (uint32_t)(first - r * per) + (uint32_t)lane;
    while (u >= per) {
        u -= per;
        row++;
    }
    unit = u;
}

/* The larger of a and |b|, |c|; NaN where one is NaN. */
DLK_DEV float maximum_abs(float a, float b, float c) {
    float d;
    asm("v_maximum3_f32 %0, %1, |%2|, |%3|" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

/* Lane (lane ^ 1) or (lane ^ 2) of the four of a block; the next of them. */
constexpr int kQuadXor1 = 0xb1, kQuadXor2 = 0x4e, kQuadNext = 0x39;
template <int CTRL>
DLK_DEV uint32_t quad(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}

typedef short s2_t __attribute__((ext_vector_type(2)));
typedef float f2_t __attribute__((ext_vector_type(2)));

/* Eight elements as 32 bits. */
DLK_DEV uint32_t fp4_of(const float (&v)[8], float scale) {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
}

/* Four elements of 6 bits: scale is 2^6 of the block's, v within the largest element. */
DLK_DEV uint32_t fp6_of(float a, float b, float c, float d, float scale) {
    s2_t p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s2_t{0, 0}, a, b, scale, false);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, c, d, scale, true);
    const uint32_t w = __builtin_bit_cast(uint32_t, p);
    const uint32_t k = (w & 0x1f1f1f1fu) | (w >> 2 & 0x20202020u);
    return (k & 0x3f) | (k >> 2 & 0xfc0) | (k >> 4 & 0x3f000) | (k >> 6 & 0xfc0000);
}

template <int DT, int FMT>
__global__ __launch_bounds__(kMxThreads) void quantize_mx_kernel(const typename LogitRow<DT>::T *__restrict__ x,
                                                                 int64_t ldx, int rows, int n, uint32_t per,
                                                                 uint8_t *__restrict__ q, int64_t ldq,
                                                                 uint8_t *__restrict__ scale, int64_t lds, bool past) {
    typedef LogitRow<DT> In;
    const int lane = lane_id();
    const uint64_t first = ((uint64_t)blockIdx.x * (kMxThreads / 64) + __builtin_amdgcn_readfirstlane(wave_id())) * 64 * kMxSpans;
    float v[kMxSpans][8];
    int64_t row[kMxSpans];
    uint32_t unit[kMxSpans];
#pragma unroll
    for (int s = 0; s < kMxSpans; s++) {
        mx_place(first + 64 * s, per, lane, row[s], unit[s]);
        const int i = (int)unit[s] * 8;
        const typename In::T *p = x + row[s] * ldx + i;
        if (row[s] < rows && i + 8 <= n) {
            load8<DT>(p, v[s]);
        } else {
#pragma unroll
            for (int c = 0; c < 8; c++) v[s][c] = row[s] < rows && i + c < n ? In::one(p + c) : 0.0f;
        }
    }
#pragma unroll
    for (int s = 0; s < kMxSpans; s++) {
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; c += 2) top = maximum_abs(top, v[s][c], v[s][c + 1]);
        uint32_t t = f2u(top) & 0x7fffffffu;       /* NaN above infinity above the rest */
        t = max(t, quad<kQuadXor1>(t));
        t = max(t, quad<kQuadXor2>(t));
        const int field = (int)(t >> 23);
        const bool bad = field == 255;
        const int e = max(field - 2, 0);           /* the scale's byte */
        uint32_t w0, w1 = 0;
        if (FMT == DLK_MX_FP4) {
            /* (2^-127 is no normal float: there twice the values over 2^-126) */
            if (DLK_COLD(ballot(e == 0 && t != 0) != 0)) {
#pragma unroll
                for (int c = 0; c < 8; c++) v[s][c] *= e == 0 ? 2.0f : 1.0f;
            }
            w0 = bad ? 0 : fp4_of(v[s], u2f((uint32_t)max(e, 1) << 23));
        } else {
            const float most = u2f((uint32_t)(e + 2) << 23 | 0x700000u);    /* 7.5 of the scale */
            float y[8];
#pragma unroll
            for (int c = 0; c < 8; c++) y[c] = fminf(fmaxf(v[s][c], -most), most);
            int by = e + 6;
            if (DLK_COLD(ballot(by > 254) != 0)) {
#pragma unroll
                for (int c = 0; c < 8; c++) y[c] *= by > 254 ? 0.0009765625f : 1.0f;
                by -= by > 254 ? 10 : 0;
            }
            const float unit_scale = u2f((uint32_t)by << 23);
            const uint32_t a = bad ? 0 : fp6_of(y[0], y[1], y[2], y[3], unit_scale);
            const uint32_t b = bad ? 0 : fp6_of(y[4], y[5], y[6], y[7], unit_scale);
            w0 = a | b << 24;                      /* this thread's six bytes */
            w1 = b >> 8;
        }
        if (row[s] >= rows) continue;
        const int64_t block = unit[s] >> 2;
        const int part = (int)(unit[s] & 3);
        if (FMT == DLK_MX_FP4) {
            store_past<4>(q + row[s] * ldq + block * 16 + part * 4, w0, past);
        } else {
            /* three of a block's four threads store eight bytes each */
            const uint32_t n0 = quad<kQuadNext>(w0), n1 = quad<kQuadNext>(w1);
            uint2 o = make_uint2(w0, w1 | n0 << 16);
            if (part == 1) o = make_uint2(w0 >> 16 | w1 << 16, n0);
            if (part == 2) o = make_uint2(w1 | n0 << 16, n0 >> 16 | n1 << 16);
            if (part < 3) *(uint2 *)(q + row[s] * ldq + block * 24 + part * 8) = o;
        }
        if (part == 0) scale[row[s] * lds + block] = bad ? 255 : (uint8_t)e;
    }
}

typedef uint32_t u1_any __attribute__((aligned(2)));

/* The bits of group `unit` of G values of a row at p. */
template <int FMT, int G>
DLK_DEV uint64_t mx_bits(const uint8_t *p, uint32_t unit) {
    if (FMT == DLK_MX_FP4) {
        p += (uint64_t)unit * (G / 2);
        return G == 8 ? *(const uint32_t *)p : *(const uint16_t *)p;
    }
    p += (uint64_t)unit * (G / 4 * 3);
    if (G == 8) return *(const u1_any *)p | (uint64_t) * (const uint16_t *)(p + 4) << 32;
    return (uint32_t)p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16;
}

/* A group's values: its bits times the scale of byte e. */
template <int FMT, int G>
DLK_DEV void mx_values(uint64_t w, uint32_t e, float (&v)[G]) {
    const float by = u2f(e == 0 ? 0x400000u : e == 255 ? 0x7fc00000u : e << 23);
    if (FMT == DLK_MX_FP4) {
        const f2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)w, 1.0f, 1);
        v[0] = a.x * by; v[1] = a.y * by; v[2] = b.x * by; v[3] = b.y * by;
        if constexpr (G == 8) {
            const f2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)w, 1.0f, 3);
            v[4] = c.x * by; v[5] = c.y * by; v[6] = d.x * by; v[7] = d.y * by;
        }
    } else {
#pragma unroll
        for (int c = 0; c < G; c++) {
            const uint32_t k = (uint32_t)(w >> (6 * c));
            /* the code's five bits as a float's last of the exponent and first of the mantissa: 2^-126 of the element */
            const float m = u2f((k & 31) << 20 | (k & 32) << 26);
            v[c] = m * 8.507059173023462e37f * by;           /* 2^126 */
        }
    }
}

/* 16 bytes of the output a thread and span, so that a wave's store is 1 KB in one piece. */
template <int DT, int FMT>
__global__ __launch_bounds__(kMxThreads) void dequantize_mx_kernel(const uint8_t *__restrict__ q, int64_t ldq,
                                                                   const uint8_t *__restrict__ scale, int64_t lds,
                                                                   int table_rows, const int32_t *__restrict__ ids,
                                                                   int rows, int n, uint32_t per,
                                                                   typename LogitRow<DT>::T *__restrict__ out, int64_t ld, bool past) {
    typedef LogitRow<DT> Out;
    constexpr int G = Out::G;
    const int lane = lane_id();
    const uint64_t first = ((uint64_t)blockIdx.x * (kMxThreads / 64) + __builtin_amdgcn_readfirstlane(wave_id())) * 64 * kMxSpans;
    int64_t row[kMxSpans];
    uint32_t unit[kMxSpans], e[kMxSpans];
    uint64_t w[kMxSpans];
    bool none[kMxSpans];
#pragma unroll
    for (int s = 0; s < kMxSpans; s++) {
        mx_place(first + 64 * s, per, lane, row[s], unit[s]);
        const int64_t r = min(row[s], (int64_t)rows - 1);
        int64_t from = ids ? (int64_t)ids[r] : r;
        none[s] = from < 0 || from >= table_rows;
        from = none[s] ? 0 : from;
        w[s] = mx_bits<FMT, G>(q + from * ldq, unit[s]);
        e[s] = scale[from * lds + unit[s] / (32 / G)];
    }
#pragma unroll
    for (int s = 0; s < kMxSpans; s++) {
        if (row[s] >= rows) continue;
        float v[G];
        mx_values<FMT, G>(w[s], e[s], v);
#pragma unroll
        for (int c = 0; c < G; c++) v[c] = none[s] ? 0.0f : v[c];
        const int i = (int)unit[s] * G;
        typename Out::T *o = out + row[s] * ld + i;
        if (i + G <= n) {
            store_past<sizeof(*o)>(o, Out::pack(v), past);
        } else {
#pragma unroll
            for (int c = 0; c < G; c++)
                if (i + c < n) Out::put(o + c, v[c]);
        }
    }
}

/* Workgroups of `rows` rows of `per` groups; 0: more than a launch holds. */
unsigned mx_blocks(int64_t rows, uint32_t per) {
    const int64_t at_once = (int64_t)kMxThreads * kMxSpans, blocks = (rows * per + at_once - 1) / at_once;
    return blocks * kMxThreads > 0xffffffffLL ? 0 : (unsigned)blocks;
}

template <int DT>
int launch_quantize_mx(const void *x, int64_t ldx, int rows, int n, int format, uint8_t *q, int64_t ldq, uint8_t *scale,
                       int64_t lds, hipStream_t stream) {
    typedef const typename LogitRow<DT>::T *P;
    const uint32_t per = (uint32_t)(((int64_t)n + 31) / 32 * 4);
    const unsigned blocks = mx_blocks(rows, per);
    if (blocks == 0) return DLK_ERR_UNSUPPORTED;
    const bool past = (int64_t)rows * n >= 64 << 20 && whole_lines(q, ldq);
    if (format == DLK_MX_FP4)
        hipLaunchKernelGGL((quantize_mx_kernel<DT, DLK_MX_FP4>), dim3(blocks), dim3(kMxThreads), 0, stream, (P)x, ldx,
                           rows, n, per, q, ldq, scale, lds, past);
    else
        hipLaunchKernelGGL((quantize_mx_kernel<DT, DLK_MX_FP6>), dim3(blocks), dim3(kMxThreads), 0, stream, (P)x, ldx,
                           rows, n, per, q, ldq, scale, lds, past);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

template <int DT>
int launch_dequantize_mx(const uint8_t *q, int64_t ldq, const uint8_t *scale, int64_t lds, int table_rows,
                         const int32_t *ids, int rows, int n, int format, void *out, int64_t ld, hipStream_t stream) {
    typedef typename LogitRow<DT>::T *P;
    constexpr int G = LogitRow<DT>::G;
    /* (more than the L2 caches hold) */
    const int64_t size = DT == DLK_F32 ? 4 : 2;
    const bool past = rows * size * n >= 32 << 20 && whole_lines(out, ld * size);
    const uint32_t per = (uint32_t)(((int64_t)n + G - 1) / G);
    const unsigned blocks = mx_blocks(rows, per);
    if (blocks == 0) return DLK_ERR_UNSUPPORTED;
    if (format == DLK_MX_FP4)
        hipLaunchKernelGGL((dequantize_mx_kernel<DT, DLK_MX_FP4>), dim3(blocks), dim3(kMxThreads), 0, stream, q, ldq,
                           scale, lds, table_rows, ids, rows, n, per, (P)out, ld, past);
    else
        hipLaunchKernelGGL((dequantize_mx_kernel<DT, DLK_MX_FP6>), dim3(blocks), dim3(kMxThreads), 0, stream, q, ldq,
                           scale, lds, table_rows, ids, rows, n, per, (P)out, ld, past);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

}  // namespace dlk

extern "C" int dlk_quantize_mx(const void *x, int dtype, int64_t ldx, int rows, int n, int format, uint8_t *q,
                               int64_t ldq, uint8_t *scale, int64_t ld_scale, hipStream_t stream) {
    if (!x || !q || !scale || rows < 0 || n <= 0 || ldx < n) return DLK_ERR_INVALID;
    if (dtype != DLK_F32 && dtype != DLK_BF16 && dtype != DLK_F16) return DLK_ERR_INVALID;
    if (format != DLK_MX_FP4 && format != DLK_MX_FP6) return DLK_ERR_INVALID;
    const int64_t blocks = ((int64_t)n + 31) / 32;
    if (ldq < blocks * (format == DLK_MX_FP4 ? 16 : 24) || ld_scale < blocks) return DLK_ERR_INVALID;
    if ((((uintptr_t)q | (uintptr_t)ldq) & 7) != 0 || ((uintptr_t)x & (dtype == DLK_F32 ? 3 : 1)) != 0) return DLK_ERR_INVALID;
    if (n > 0x7fffffff - 65536) return DLK_ERR_UNSUPPORTED;
    if (rows == 0) return DLK_OK;
    if (dtype == DLK_F32) return dlk::launch_quantize_mx<DLK_F32>(x, ldx, rows, n, format, q, ldq, scale, ld_scale, stream);
    if (dtype == DLK_BF16) return dlk::launch_quantize_mx<DLK_BF16>(x, ldx, rows, n, format, q, ldq, scale, ld_scale, stream);
    return dlk::launch_quantize_mx<DLK_F16>(x, ldx, rows, n, format, q, ldq, scale, ld_scale, stream);
}

extern "C" int dlk_dequantize_mx(const uint8_t *q, int64_t ldq, const uint8_t *scale, int64_t ld_scale, int table_rows,
                                 const int32_t *ids, int rows, int n, int format, void *out, int dtype, int64_t ld,
                                 hipStream_t stream) {
    if (!q || !scale || !out || rows < 0 || table_rows < 0 || n <= 0 || ld < n) return DLK_ERR_INVALID;
    if (dtype != DLK_F32 && dtype != DLK_BF16 && dtype != DLK_F16) return DLK_ERR_INVALID;
    if (format != DLK_MX_FP4 && format != DLK_MX_FP6) return DLK_ERR_INVALID;
    const int64_t blocks = ((int64_t)n + 31) / 32;
    if (ldq < blocks * (format == DLK_MX_FP4 ? 16 : 24) || ld_scale < blocks) return DLK_ERR_INVALID;
    if ((((uintptr_t)q | (uintptr_t)ldq) & 7) != 0 || ((uintptr_t)out & (dtype == DLK_F32 ? 3 : 1)) != 0 ||
        ((uintptr_t)ids & 3) != 0)
        return DLK_ERR_INVALID;
    /* (ids that no row of an empty table answers still read its first one's place) */
    if (rows > 0 && (table_rows == 0 || (!ids && rows > table_rows))) return DLK_ERR_INVALID;
    if (n > 0x7fffffff - 65536) return DLK_ERR_UNSUPPORTED;
    if (rows == 0) return DLK_OK;
    if (dtype == DLK_F32)
        return dlk::launch_dequantize_mx<DLK_F32>(q, ldq, scale, ld_scale, table_rows, ids, rows, n, format, out, ld, stream);
    if (dtype == DLK_BF16)
        return dlk::launch_dequantize_mx<DLK_BF16>(q, ldq, scale, ld_scale, table_rows, ids, rows, n, format, out, ld, stream);
    return dlk::launch_dequantize_mx<DLK_F16>(q, ldq, scale, ld_scale, table_rows, ids, rows, n, format, out, ld, stream);
}
