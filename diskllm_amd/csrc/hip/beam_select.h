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

constexpr int kBeamEntries = kBeamThreads * 16;                  /* entries that a merge takes at once */

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
    int batches;         /* of a row, shared out to them */
    uint32_t *counters;  /* [groups] zero between launches */
    BeamSlot *slots;     /* [rows][slices] */
    uint64_t *cands;     /* [rows][slices][n] */
};

/* Workgroups for each row of `vocab` logits: some 800 in all (three a CU: beyond that the
 * fixed 2.6 us of each cost more than more waves give), where that leaves five batches each
 * at most; but no more than give a group 4,096 entries, which its merge takes in one round
 * trip, unless each had more than eight batches then; and 256 to a group (us by workgroups a row,
 * taken with a shorter exponential that cost some 2% less:
 *   64 x 151,936 with histories        10: 34.4, 12: 34.1, 13: 33.7, 16: 34.9, 20: 36.3
 *   128 x 50,257, groups of 16         4: 25.0, 6: 24.7, 8: 28.1, 10: 29.4
 *   512 x 262,144                      8: 141, 11: 143, 13: 142, 16: 146, 21: 153
 *   512 x 262,144 masked               4: 142, 5: 132, 8: 129, 10: 128, 14: 131
 *   256 x 128,256, 16 beams, 32 out    4: 86.7, 6: 74.6, 8: 65.1, 10: 72.9, 16: 103
 *   48 x 151,936, 12 beams, 24 out     8: 37.1, 10: 36.7, 13: 29.5, 16: 37.8
 *   16 x 128,256, 16 beams, 32 out     4: 62.5, 7: 36.9, 8: 34.7, 16: 39.3
 *   4 x 32,000                         4: 13.8, 8: 11.4). */
inline int beam_slices(int64_t rows, int beams, int n_out, int vocab) {
    const int64_t batches = ((int64_t)vocab + kBeamBatch - 1) / kBeamBatch, least = (batches + 7) / 8;
    const int64_t once = kBeamEntries / (beams * n_out);
    int64_t s = (800 + rows / 2) / rows;
    if (s < (batches + 4) / 5) s = (batches + 4) / 5;
    if (s > once) s = once > least ? once : least;
    if (s > kBeamThreads / beams) s = kBeamThreads / beams;
    return (int)(s < batches ? s : batches);
}

}  // namespace dlk

#endif
