/*
 * top_list.h -- lists of a row's largest logits, shared by the beam selection and the
 * scoring of tokens: entries, orders and the exchange of words between workgroups.
 */
#ifndef DLK_TOP_LIST_H
#define DLK_TOP_LIST_H

#include "dlk_device.h"

namespace dlk {

DLK_DEV void bpub64(uint64_t *a, uint64_t v) { __hip_atomic_store(a, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DLK_DEV uint64_t bget64(const uint64_t *a) {
    return __hip_atomic_load((uint64_t *)a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

/* x where bit c of `bits` is set, else -inf (a bit field's sign, a bitwise choice). */
DLK_DEV float allowed_or_ninf(float x, uint32_t bits, int c) {
    const uint32_t m = (uint32_t)((int)(bits << (31 - c)) >> 31);
    return u2f((f2u(x) & m) | (0xff800000u & ~m));
}

/* An entry of a list: larger is better (the logit's ascending key, then the lower id). */
DLK_DEV uint64_t entry_of(float l, int id) { return (uint64_t)~desc_key(l) << 32 | (uint32_t)~id; }
DLK_DEV float entry_logit(uint64_t e) { return key_value(~(uint32_t)(e >> 32)); }
DLK_DEV int entry_id(uint64_t e) { return (int)~(uint32_t)e; }

/* Lane's place among the lanes of `who`, from `first` on. */
DLK_DEV int place_in(uint64_t who, int first) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, (uint32_t)first));
}

/* LDS that only this wave writes and reads: its instructions go in order, the compiler has to keep it. */
DLK_DEV void wave_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

}  // namespace dlk

#endif
