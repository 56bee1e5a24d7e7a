/*
 * beam_select.h -- parameters of the beam selection kernel, shared by its host side
 * (capi.hip) and the kernel (beam_select.hip).
 */
#ifndef DLK_BEAM_SELECT_H
#define DLK_BEAM_SELECT_H

#include <stdint.h>

namespace dlk {

constexpr int kBeamThreads = 256;
constexpr int kBeamBatch = kBeamThreads * 16;                   /* logits of a batch: four groups of four per thread */

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
    int batches;         /* of each */
    uint32_t *counters;  /* [groups] zero between launches */
    BeamSlot *slots;     /* [rows][slices] */
    uint64_t *cands;     /* [rows][slices][n] */
};

/* Batches of each workgroup for rows of `vocab` logits: about 1,100 workgroups (some four a CU,
 * resident together) where that takes at most six batches each, so that a workgroup's
 * fixed 5 us are paid few times (us by batches of each:
 *   64 x 151,936 with histories   1: 46, 2: 33.4, 3: 32.9, 4: 35, 8: 50
 *   128 x 50,257 in groups of 16  1: 39, 2: 32.5, 3: 31.6, 4: 38 (the merge has become 5 shorter since)
 *   512 x 262,144                 1: 302, 2: 185, 3: 156, 4: 145, 8: 145
 *   4 x 32,000                    1: 11.4, 2: 13.8);
 * more where the merge would meet over 256 lists a group, which it takes in one round trip. */
inline int beam_batches(int64_t rows, int beams, int vocab) {
    const int64_t per_row = ((int64_t)vocab + kBeamBatch - 1) / kBeamBatch;
    int64_t m = (rows * per_row + 1099) / 1100;
    if (m > 6) m = 6;
    if (m < (per_row * beams + 255) / 256) m = (per_row * beams + 255) / 256;
    const int64_t slices = (per_row + m - 1) / m;
    return (int)((per_row + slices - 1) / slices);
}

}  // namespace dlk

#endif
