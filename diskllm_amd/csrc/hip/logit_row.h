/*
 * logit_row.h -- rows of logits in float32, bfloat16 or float16, 16 bytes at a time.
 */
#ifndef DLK_LOGIT_ROW_H
#define DLK_LOGIT_ROW_H

#include "dlk_device.h"
#include "../../../include/diskllm_amd.h"

namespace dlk {

template <int DT>
struct LogitRow {
    typedef uint16_t T;
    static constexpr int G = 8;                    /* values of a 16-byte group */
    typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(2)));
    DLK_DEV static float value(uint32_t h) {
        return DT == DLK_BF16 ? u2f(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
    }
    DLK_DEV static float one(const T *p) { return value(*p); }
    DLK_DEV static void unpack(Raw r, float *v) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            v[2 * c] = value(r[c] & 0xffff);
            v[2 * c + 1] = DT == DLK_BF16 ? u2f(r[c] & 0xffff0000u) : value(r[c] >> 16);
        }
    }
    DLK_DEV static uint32_t bits(float v) {        /* rounded to the nearest, halves to even */
        return DT == DLK_BF16 ? (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v)
                              : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v);
    }
    DLK_DEV static Raw pack(const float *v) {
        Raw r;
#pragma unroll
        for (int c = 0; c < 4; c++) r[c] = bits(v[2 * c]) | bits(v[2 * c + 1]) << 16;
        return r;
    }
    DLK_DEV static void put(T *p, float v) { *p = (uint16_t)bits(v); }
};
template <>
struct LogitRow<DLK_F32> {
    typedef float T;
    static constexpr int G = 4;
    typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(4)));
    DLK_DEV static float one(const T *p) { return *p; }
    DLK_DEV static void unpack(Raw r, float *v) {
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = u2f(r[c]);
    }
    DLK_DEV static Raw pack(const float *v) { return Raw{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])}; }
    DLK_DEV static void put(T *p, float v) { *p = v; }
};

/* Whether the mask (null: every one) allows id v. */
DLK_DEV bool mask_allows(const uint32_t *mask, int v) { return !mask || (mask[v >> 5] >> (v & 31) & 1) != 0; }

}  // namespace dlk

#endif
