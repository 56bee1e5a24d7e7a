/*
 * token_logprobs.h -- parameters of the scoring kernels, shared by their host side
 * (capi.hip) and the kernels (token_logprobs.hip).
 */
#ifndef DLK_TOKEN_LOGPROBS_H
#define DLK_TOKEN_LOGPROBS_H

#include <stdint.h>

namespace dlk {

constexpr int kLogprobThreads = 256;
constexpr int kLogprobMaxSlices = 64;                            /* of a row (a lane each, as they are joined) */
constexpr int kLogprobEntries = kLogprobThreads * 16;            /* entries that a join takes */

/* Logits of a batch: four 16-byte loads a thread. */
inline int logprob_batch(int dtype) { return dtype == 0 ? kLogprobThreads * 16 : kLogprobThreads * 32; }

/* What a workgroup says of its slice of a row. */
struct LogprobSlot {
    uint64_t sum, dot;   /* sums of e and of e * t over the slice, e = 2^t, t = (l - max) * log2(e) / T (doubles) */
    uint64_t max_kept;   /* the slice's maximum (float bits, high word) and the entries it lists (low word) */
};

struct LogprobParams {
    const void *logits;
    int64_t ld;
    const uint32_t *mask;
    int64_t mask_ld;
    const int32_t *mask_row;
    const int32_t *tokens;
    float *logprobs, *stats;
    int32_t *top_ids;
    float *top_logprobs;
    uint32_t *status;
    int V, given, n;     /* n: alternatives */
    float scale;         /* log2(e) / T */
    double inv_t;
    int r0;              /* first row of the launch */
    int slices;          /* workgroups per row */
    int batches;         /* of a row, shared out to them */
    uint32_t *counters;  /* [rows] zero between launches; none where slices == 1 */
    LogprobSlot *slots;  /* [rows][slices] */
    uint64_t *cands;     /* [rows][slices][n] */
};

/* Workgroups for each row: some 800 in all (three a CU), as the beam selection's slices. */
inline int logprob_slices(int64_t rows, int batches) {
    int64_t s = (800 + rows / 2) / rows;
    if (s < 1) s = 1;
    if (s > kLogprobMaxSlices) s = kLogprobMaxSlices;
    return (int)(s < batches ? s : batches);
}

}  // namespace dlk

#endif
