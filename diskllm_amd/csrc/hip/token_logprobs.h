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
inline int logprob_batch(int dtype) { return kLogprobThreads * (dtype == 0 ? 16 : 32); }

constexpr int kLogprobRecords = 64;                              /* of each thread's maxima in a slice */

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
    int cap;             /* entries that a slice may list for the row's last workgroup */
    float scale;         /* log2(e) / T */
    double inv_t;
    int r0;              /* first row of the launch */
    int slices;          /* workgroups per row */
    int batches;         /* of a row, shared out to them */
    uint32_t *counters;  /* [rows] zero between launches; none where slices == 1 */
    LogprobSlot *slots;  /* [rows][slices] */
    uint64_t *cands;     /* [rows][slices][cap] */
};

/* Workgroups for each row: some 384 in all, two at least up to 256 rows (of more than four rows two thirds of the
 * batches at most); past that one.  What each one adds, its list and the row's joining, is a chain of some 5 us
 * that others of its CU run beside (us by workgroups a row, float32 with 5 alternatives):
 *   1 x 32,000      1: 10.9, 2: 12.0, 4: 12.2, 8: 10.8
 *   8 x 151,936     4: 16.0, 8: 13.8, 18: 12.5, 25: 12.1, 37: 13.7
 *   64 x 151,936    1: 28.7, 2: 21.7, 4: 18.0, 8: 18.2, 13: 19.7, 37: 35.8
 *   128 x 50,257    1: 16.0, 2: 15.5, 4: 16.8, 9: 21.1
 *   256 x 151,936   1: 48.9, 2: 42.7, 4: 42.5, 8: 47.6
 *   300 x 50,257    1: 20.4, 2: 22.7, 4: 29.9
 * without alternatives
 *   1 x 32,000      1: 6.8, 2: 6.0, 4: 5.0, 8: 4.8
 *   8 x 151,936     4: 9.4, 8: 7.0, 18: 6.6, 25: 6.9, 37: 8.0
 *   16 x 151,936    8: 7.7, 12: 7.9, 16: 8.1, 24: 9.3, 37: 11.7
 *   64 x 151,936    1: 23.9, 2: 15.4, 4: 11.4, 6: 11.1, 8: 11.6, 13: 13.5
 *   128 x 50,257    1: 10.9, 2: 9.7, 3: 9.5, 4: 9.8, 9: 11.1
 *   256 x 151,936   1: 37.0, 2: 27.6, 4: 28.8, 8: 30.7
 *   300 x 50,257    1: 13.6, 2: 15.7, 4: 17.4;  x 151,936 39.2, 36.8, 37.4
 * of 64
 *   8 x 151,936     4: 19.5, 8: 17.1, 18: 20.6, 25: 22.3;  64 x 151,936 2: 26.3, 4: 20.9, 6: 21.9, 8: 22.3 */
inline int logprob_slices(int64_t rows, int batches) {
    int64_t s = rows > 256 ? 1 : (384 + rows / 2) / rows;
    if (rows > 4 && s > (batches * 2 + 2) / 3) s = (batches * 2 + 2) / 3;
    if (s > kLogprobMaxSlices) s = kLogprobMaxSlices;
    return (int)(s < batches ? s : batches);
}

}  // namespace dlk

#endif
