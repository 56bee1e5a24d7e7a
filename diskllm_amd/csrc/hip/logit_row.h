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

/* Eight values at p. */
template <int DT>
DLK_DEV void load8(const typename LogitRow<DT>::T *p, float (&v)[8]) {
    typedef LogitRow<DT> In;
#pragma unroll
    for (int k = 0; k < 8 / In::G; k++) In::unpack(*(const typename In::Raw *)(p + k * In::G), v + k * In::G);
}

/* Whether rows at p, ld bytes apart, begin with cache lines: past the caches a line that two waves write
 * goes to memory twice (100,001 rows of 4,090 bfloat16: 208 us past them, 183 through). */
inline bool whole_lines(const void *p, int64_t ld) { return (((uintptr_t)p | (uintptr_t)ld) & 127) == 0; }

/* Stores v at p of ALIGN bytes' alignment, past the caches where `past`: what the next call would not find
 * there anyway, as large outputs, is written at the memory's rate (8,192 x 4,096 float32 dequantised: 44 us
 * through the caches, 23.5 past them). */
template <int ALIGN, class V>
DLK_DEV void store_past(void *p, V v, bool past) {
    typedef V Any __attribute__((aligned(ALIGN)));
    if (past) {
        /* (apart from the other store, or the compiler makes one plain store of the two) */
        asm volatile("" ::: "memory");
        __builtin_nontemporal_store(v, (Any *)p);
        asm volatile("" ::: "memory");
    } else {
        *(Any *)p = v;
    }
}

/* Whether the mask (null: every one) allows id v. */
DLK_DEV bool mask_allows(const uint32_t *mask, int v) { return !mask || (mask[v >> 5] >> (v & 31) & 1) != 0; }

}  // namespace dlk

#endif
