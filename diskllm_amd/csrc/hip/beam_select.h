/*
 * beam_select.h -- parameters of the beam selection kernel, shared by its host side
 * (capi.hip) and the kernel (beam_select.hip).
 */
#ifndef DLK_BEAM_SELECT_H
#define DLK_BEAM_SELECT_H

#include <stdint.h>

namespace dlk {

constexpr int kBeamThreads = 256;
constexpr int kBeamGroups = 8;                                  /* groups of four logits per thread */
constexpr int kBeamSlice = kBeamThreads * kBeamGroups * 4;      /* logits of one workgroup */

/* What a workgroup says of its slice of a row. */
struct BeamSlot {
    uint64_t sum;        /* sum of exp(l - max) over the slice (double) */
    uint64_t max_kept;   /* the slice's maximum (float bits, high word) and the entries it lists (low word) */
};

struct BeamParams {
    const float *logits;
    int64_t ld;
    const int32_t *hist_off, *hist_ids;
    const uint32_t *mask;
    int64_t mask_ld;
    const int32_t *mask_row;
    const float *scores;
    const int32_t *lengths;
    const uint8_t *finished;
    int32_t *out_tokens, *out_parents;
    float *out_scores;
    int32_t *out_lengths;
    uint8_t *out_finished;
    uint32_t *status;
    int V, beams, n, eos, max_hist;
    float alpha;
    uint32_t order;
    float rep, freq, pres;
    int g0;              /* first group of the launch */
    int slices;          /* workgroups per row */
    uint32_t *counters;  /* [groups] zero between launches */
    BeamSlot *slots;     /* [rows][slices] */
    uint64_t *cands;     /* [rows][slices][n] */
};

}  // namespace dlk

#endif
