/*
 * quantize.hip -- 8-bit values and a scale for each row: hidden states (a scale per
 * token) and an LM head's weights (a scale per channel), for dlk_logits_i8.
 *
 *   scale = max |x| / 127 (rounded once to float),  q = x / scale to the nearest, halves to even.
 *
 * The quotient's rounding is decided exactly, not by a rounded quotient: with
 * n = floor of the approximate one (off by at most 2e-5, so the true value lies
 * between n - 2e-5 and n + 1 + 2e-5), the sign of x - (n + 1/2) * scale, which one
 * FMA gives without error, says whether q is n or n + 1.
 *
 * Bound by memory for many rows, by latency for few: each row is read once into
 * registers (the maximum, then the values), up to 8,192 entries; longer rows are read
 * a second time.  50,257 x 4,096 takes 181-202 us in float32, 5.1-5.7 TB/s read and written (a
 * large copy: 5.1), 131-135 in bfloat16 and float16, 4.6-4.7; 1 x 4,096 bf16 3.3, a launch and one round trip.  A workgroup a row, so
 * that one row has 256 threads' loads in flight; rows of up to 1,024 entries, of which that
 * would leave most threads idle, a wave each.  Rows of any stride: 16-byte loads need no
 * more than the type's own alignment here.
 */
#include <hip/hip_runtime.h>

#include "dlk_device.h"
#include "../../../include/diskllm_amd.h"

namespace dlk {

constexpr int kQuantThreads = 256;
constexpr int kQuantKeep = 4;             /* groups of eight that a thread keeps in registers */

typedef float f8_any __attribute__((ext_vector_type(8), aligned(4)));
typedef uint16_t h8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef uint32_t u2_any __attribute__((ext_vector_type(2), aligned(1)));

template <int DT>
struct QuantIn {
    typedef uint16_t T;
    DLK_DEV static float one(const uint16_t *p) {
        return DT == DLK_BF16 ? u2f((uint32_t)*p << 16) : (float)__builtin_bit_cast(_Float16, *p);
    }
    DLK_DEV static void eight(const uint16_t *p, float (&v)[8]) {
        const h8_any h = *(const h8_any *)p;
#pragma unroll
        for (int c = 0; c < 8; c++)
            v[c] = DT == DLK_BF16 ? u2f((uint32_t)h[c] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h[c]);
    }
};
template <>
struct QuantIn<DLK_F32> {
    typedef float T;
    DLK_DEV static float one(const float *p) { return *p; }
    DLK_DEV static void eight(const float *p, float (&v)[8]) {
        const f8_any x = *(const f8_any *)p;
#pragma unroll
        for (int c = 0; c < 8; c++) v[c] = x[c];
    }
};

/* x / scale to the nearest integer, halves to even, within +-127.  inv: the rounded
 * 1 / scale, 0 where that would leave the range of a float (scale below 1e-30: the
 * quotient then in 64 bits, which tells any quotient of two floats from a half). */
DLK_DEV int quantized(float x, float scale, float inv) {
    float q;
    if (DLK_HOT(inv != 0.0f)) {
        const float n = floorf(x * inv);
        const float d = fmaf(-(n + 0.5f), scale, x);
        const float even = 2.0f * floorf(0.5f * (n + 1.0f));      /* the even one of n, n + 1 */
        q = d > 0.0f ? n + 1.0f : d < 0.0f ? n : even;
    } else {
        q = scale > 0.0f ? (float)rint((double)x / (double)scale) : 0.0f;
    }
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

/* TPR threads to a row. */
template <int DT, int TPR>
__global__ __launch_bounds__(kQuantThreads) void quantize_kernel(const typename QuantIn<DT>::T *__restrict__ x,
                                                                 int64_t ldx, int rows, int n,
                                                                 int8_t *__restrict__ q, int64_t ldq,
                                                                 float *__restrict__ scale) {
    typedef QuantIn<DT> In;
    __shared__ uint32_t part[kQuantThreads / 64];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (kQuantThreads / TPR) + threadIdx.x / TPR;
    if (TPR == 64 && row >= rows) return;          /* (a whole wave) */
    const typename In::T *xr = x + row * ldx;
    int8_t *qr = q + row * ldq;
    float v[kQuantKeep][8];
    uint32_t top = 0;                              /* the largest |x| as bits: NaN above infinity above the rest */
#pragma unroll
    for (int j = 0; j < kQuantKeep; j++) {
        const int i = (t + j * TPR) * 8;
        if (i + 8 <= n) {
            In::eight(xr + i, v[j]);
        } else {
#pragma unroll
            for (int c = 0; c < 8; c++) v[j][c] = i + c < n ? In::one(xr + i + c) : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < kQuantKeep; j++)
#pragma unroll
        for (int c = 0; c < 8; c++) top = max(top, f2u(v[j][c]) & 0x7fffffffu);
    for (int i = (t + kQuantKeep * TPR) * 8; i < n; i += TPR * 8)
        for (int c = 0; c < 8 && i + c < n; c++) top = max(top, f2u(In::one(xr + i + c)) & 0x7fffffffu);
    top = wave_minmax_u32<false>(top);
    if (TPR > 64) {
        if (lane_id() == 0) part[wave_id()] = top;
        __syncthreads();
        top = part[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; w++) top = max(top, part[w]);
    }
    /* a row with NaN or infinity has no scale: NaN, so that its logits show it */
    const bool bad = top >= 0x7f800000u;
    const float s = bad ? u2f(0x7fc00000u) : u2f(top) / 127.0f;
    const float inv = s >= 1e-30f ? 1.0f / s : 0.0f;
    if (t == 0) scale[row] = s;
#pragma unroll
    for (int j = 0; j < kQuantKeep; j++) {
        const int i = (t + j * TPR) * 8;
        if (i >= n) break;
        int b[8];
#pragma unroll
        for (int c = 0; c < 8; c++) b[c] = bad ? 0 : quantized(v[j][c], s, inv);
        if (i + 8 <= n) {
            u2_any w;
            w.x = (uint32_t)(b[0] & 255) | (uint32_t)(b[1] & 255) << 8 | (uint32_t)(b[2] & 255) << 16 | (uint32_t)b[3] << 24;
            w.y = (uint32_t)(b[4] & 255) | (uint32_t)(b[5] & 255) << 8 | (uint32_t)(b[6] & 255) << 16 | (uint32_t)b[7] << 24;
            *(u2_any *)(qr + i) = w;
        } else {
#pragma unroll
            for (int c = 0; c < 8; c++)
                if (i + c < n) qr[i + c] = (int8_t)b[c];
        }
    }
    for (int i = (t + kQuantKeep * TPR) * 8; i < n; i += TPR * 8)
        for (int c = 0; c < 8 && i + c < n; c++) qr[i + c] = (int8_t)(bad ? 0 : quantized(In::one(xr + i + c), s, inv));
}

template <int DT>
int launch_quantize(const void *x, int64_t ldx, int rows, int n, int8_t *q, int64_t ldq, float *scale,
                    hipStream_t stream) {
    typedef const typename QuantIn<DT>::T *P;
    /* short rows: a wave each */
    if (n <= 1024)
        hipLaunchKernelGGL((quantize_kernel<DT, 64>), dim3((unsigned)((rows + 3) / 4)), dim3(kQuantThreads), 0, stream,
                           (P)x, ldx, rows, n, q, ldq, scale);
    else
        hipLaunchKernelGGL((quantize_kernel<DT, 256>), dim3((unsigned)rows), dim3(kQuantThreads), 0, stream, (P)x, ldx,
                           rows, n, q, ldq, scale);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

}  // namespace dlk

extern "C" int dlk_quantize_rows(const void *x, int dtype, int64_t ldx, int rows, int n, int8_t *q, int64_t ldq,
                                 float *scale, hipStream_t stream) {
    if (!x || !q || !scale || rows < 0 || n <= 0 || ldx < n || ldq < n) return DLK_ERR_INVALID;
    if (((uintptr_t)scale & 3) != 0 || ((uintptr_t)x & (dtype == DLK_F32 ? 3 : 1)) != 0) return DLK_ERR_INVALID;
    /* int indices; 2^32 threads and over are no launch */
    const int64_t blocks = n <= 1024 ? ((int64_t)rows + 3) / 4 : rows;
    if (n > 0x7fffffff - 65536 || blocks * dlk::kQuantThreads > 0xffffffffLL) return DLK_ERR_UNSUPPORTED;
    if (dtype != DLK_F32 && dtype != DLK_BF16 && dtype != DLK_F16) return DLK_ERR_INVALID;
    if (rows == 0) return DLK_OK;
    if (dtype == DLK_F32) return dlk::launch_quantize<DLK_F32>(x, ldx, rows, n, q, ldq, scale, stream);
    if (dtype == DLK_BF16) return dlk::launch_quantize<DLK_BF16>(x, ldx, rows, n, q, ldq, scale, stream);
    return dlk::launch_quantize<DLK_F16>(x, ldx, rows, n, q, ldq, scale, stream);
}
