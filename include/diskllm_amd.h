/*
 * diskllm_amd.h -- batched, device-resident C ABI of the MI355X sampling and
 * grammar-mask path.
 *
 * The drop-in headers include/sampler.h and include/grammar.h keep DiskLLM's
 * single-row host API; this header adds the batched entry points they are built
 * on.  All pointers below are device pointers unless stated otherwise; every
 * call is asynchronous on `stream` and returns a DLK_* status.
 *
 * Row semantics are those of the reference caller diskllm_sample_grammar()
 * (src/core/sampler_api.c:48-73) with the allow-mask in place of the grammar
 * callback: mask -> penalties (in `penalty_order`) -> sampler_sample()
 * (src/sampler.c:136-234).  Token ids are bit-identical to the reference built
 * as strict ISO C (-std=c11 -O2) on the same inputs and the same xorshift state.
 */
#ifndef DISKLLM_AMD_H
#define DISKLLM_AMD_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DLK_OK 0
#define DLK_ERR_INVALID (-1)      /* bad argument */
#define DLK_ERR_UNSUPPORTED (-2)  /* shape or parameter outside the supported range */
#define DLK_ERR_HIP (-3)          /* a HIP runtime call failed */
#define DLK_ERR_FORMAT (-4)       /* a file that cannot be opened, is truncated or is not in the format read */

/* Device status bits written by the kernels (dlk_batch.status). */
#define DLK_STATUS_HISTORY_TOO_LONG 1u  /* a row's history exceeded max_history: its id is -1 */
#define DLK_STATUS_SYNC_TIMEOUT 2u      /* a cross-workgroup wait gave up: the call's ids are invalid,
                                           though each stays inside [0, vocab) */
#define DLK_STATUS_UNSUPPORTED_ROW 4u   /* reserved: no row kind is refused any more (rows whose
                                           s = (l - max) / T holds NaN with top_k > 4096 are served) */

/* Penalty ops, packed low nibble first into dlk_sample_params.penalty_order. */
#define DLK_OP_REPETITION 1u  /* src/sampler.c:21-33, once per occurrence */
#define DLK_OP_FREQUENCY 2u   /* builder-defined: l -= f * count, once per distinct id */
#define DLK_OP_PRESENCE 3u    /* src/sampler.c:35-52, once per distinct id */
/* Reference caller order: presence then repetition (src/core/sampler_api.c:55-61). */
#define DLK_ORDER_REFERENCE (DLK_OP_PRESENCE | (DLK_OP_REPETITION << 4))
/* repetition -> frequency -> presence. */
#define DLK_ORDER_REP_FREQ_PRES (DLK_OP_REPETITION | (DLK_OP_FREQUENCY << 4) | (DLK_OP_PRESENCE << 8))

typedef struct {
    /* sampler_config (include/sampler.h:10-16) without the seed: */
    float temperature;        /* 0 = greedy; any other value as the reference uses it (1/temperature
                                 negative, zero or infinite included, src/sampler.c:154) */
    int top_k;                /* active when 0 < top_k < vocab */
    float top_p;              /* active when < 1 */
    float min_p;              /* active when > 0 (absolute threshold, src/sampler.c:189) */
    /* penalties (diskllm_sampler_params, include/diskllm.h:48-56, plus frequency): */
    float repeat_penalty;     /* active when > 1 */
    float frequency_penalty;  /* active when != 0 */
    float presence_penalty;   /* active when != 0 */
    uint32_t penalty_order;   /* DLK_ORDER_* or any packing of DLK_OP_* */
    int max_history;          /* upper bound on any row's history length (0 = 1024); above 1024 the
                                 penalties may be applied to a scratch copy of the rows first */
    int n_out;                /* candidate outputs per row (0 = none) */
    int path;                 /* DLK_PATH_AUTO; the others force one implementation (tests) */
    float softcap;            /* > 0: logits = softcap * tanhf(logits / softcap) first, as the
                                 reference's decode step does (src/core/context.c:873-876); else none */
} dlk_sample_params;

#define DLK_PATH_AUTO 0        /* fastest path that covers the configuration */
#define DLK_PATH_ROW 1         /* one workgroup per row, every sum emulated exactly */
#define DLK_PATH_FULL_EXACT 2  /* fused full-vocabulary kernel with every row finished by its exact
                                  fallbacks: the softmax, min-p and top-p sums found by the split exact
                                  sums and the draw walked slice by slice from each slice's exact start,
                                  as for a row whose certified bounds or candidate chains do not decide
                                  them (tests) */
#define DLK_PATH_FULL_NO_WAIT 3  /* fused full-vocabulary kernel whose cross-workgroup waits give up at the
                                   first poll that finds a word not yet written: forces the
                                   DLK_STATUS_SYNC_TIMEOUT path (tests; the ids are then invalid).
                                   Shapes whose slices hold 24 entries per thread, no soft-cap;
                                   others return DLK_ERR_UNSUPPORTED */

typedef struct {
    const float *logits;      /* [rows, ld] fp32, read only */
    int64_t ld;               /* row stride in elements (>= vocab) */
    const int32_t *hist_off;  /* [rows+1] CSR offsets into hist_ids, or NULL */
    const int32_t *hist_ids;  /* previously seen token ids (out-of-range ids are skipped) */
    const uint32_t *mask;     /* packed allow-masks, bit i%32 of word i/32 (1 = allowed), or NULL */
    int64_t mask_ld;          /* words between mask rows */
    const int32_t *mask_row;  /* [rows] mask row used by each row (e.g. a DFA state), or NULL = row */
    uint64_t *rng;            /* [rows] xorshift64 states (non-zero), advanced once per sampled row */
    int32_t *out_ids;         /* [rows] sampled token ids */
    int32_t *out_cand_ids;    /* [rows, n_out] first n_out candidates in buffer order, or NULL */
    float *out_cand_probs;    /* [rows, n_out] their softmax probabilities (src/sampler.c:183-185) */
    float *out_cand_logprobs; /* [rows, n_out] log of their final sampling probability (-inf if cut) */
    uint32_t *status;         /* one word of DLK_STATUS_* bits, OR-ed by the kernels, or NULL */
} dlk_batch;

/* Initial xorshift state for a seed (src/sampler.c:87): seed 0 -> 0xDEADBEEF12345678. */
uint64_t dlk_seed_state(uint64_t seed);

/* Sample one token per row.  Replaces, for a batch of rows, the sequence
 * diskllm_grammar_apply_mask (as a packed mask) -> sampler_apply_*_penalty ->
 * sampler_sample of the reference (src/core/sampler_api.c:48-63). */
int dlk_sample(const dlk_batch *batch, int rows, int vocab, const dlk_sample_params *params,
               hipStream_t stream);

/* Workspace lifetime.  dlk_sample and the calls built on it keep one lazily
 * grown device workspace per (device, stream) they are called on (kernels queued
 * on one stream run in order and share it; calls on different streams never
 * do).  It is held until the process ends or until this call, which waits for
 * the stream's queued work and frees the stream's workspaces on the current
 * device.  Call it before destroying a stream that was passed to dlk_sample; a
 * later call on the stream allocates afresh.  No counterpart in the reference,
 * whose sampler owns a host work buffer freed by sampler_free
 * (src/sampler.c:91-95).
 *
 * HIP graphs: nothing is allocated while `stream` is captured, in any capture
 * mode, so make each call once on that stream before capturing it.  A captured
 * call that finds no workspace is recorded on the row kernel, which needs none
 * and is several times slower (histories past 1,024 ids and top_k above 4,096,
 * which need one, return DLK_ERR_HIP).  A graph uses the workspace its calls were
 * captured with: its replays and the stream's other calls must not overlap,
 * and it is not replayed after this call has released the stream.  A later call
 * that needs a larger workspace leaves the graph's alone.  Where device memory is
 * short a call takes its rows in several launches, at the last on the row
 * kernel. */
int dlk_release_stream(hipStream_t stream);

/* dlk_sample without any allocation.  No counterpart in the reference: it is
 * for callers that cannot allocate device memory (code under HIP graph capture,
 * serving loops and harnesses that forbid hipMalloc).  Same arguments, kernels
 * and results as dlk_sample; its workspace is a fixed 64 MiB scratch array per
 * device (held until the process ends), whose counter words each call clears
 * with a fill kernel on `stream`.  Every call on a device shares that device's
 * array, so calls that overlap on one device race: those over rows of odd length
 * or alignment too, which ran without the array before the fused kernels took
 * such rows.  DLK_ERR_UNSUPPORTED when the
 * call needs more than the array holds or a second buffer: max_history > 1024
 * (the penalties then run on a scratch copy of the rows), or a batch whose
 * kernels' workspace exceeds the array (the fused full-vocabulary kernel takes
 * as many rows per launch as the array holds, about 680 KB per row at a
 * vocabulary of 151,936). */
#define DLK_NOALLOC_SCRATCH_BYTES (64u << 20)
int dlk_sample_noalloc(const dlk_batch *batch, int rows, int vocab, const dlk_sample_params *params,
                       hipStream_t stream);

/* Byte-DFA allow-masks (no reference counterpart; replaces the accept_str
 * callback loop of src/core/grammar.c:284-306 for byte-level automata).
 * Token t = bytes[off[t] .. off[t+1]) is allowed from state s iff s != 0, the
 * token is non-empty and no prefix walk through trans[s*256 + byte] reaches
 * state 0; the EOS id (if >= 0) is allowed iff bit s of accept_mask is set.
 * Writes out_mask[r * mask_ld + w] for the n_rows states in `states`. */
int dlk_dfa_mask(const uint32_t *off, const uint8_t *bytes, int vocab, const uint8_t *trans, int n_states,
                 const int32_t *states, int n_rows, int eos_id, uint64_t accept_mask, uint32_t *out_mask,
                 int64_t mask_ld, hipStream_t stream);

/* y[i] = expf(x[i]) for i < n, bit-identical to the host libm expf that the
 * reference's softmax calls (src/sampler.c:179; glibc 2.35, x86-64 FMA variant). */
int dlk_expf(const float *x, float *y, int64_t n, hipStream_t stream);

/* Penalties in place on device logits [rows, ld], history as in dlk_batch
 * (hist_off [rows+1], hist_ids).  One call replaces, per row,
 * sampler_apply_presence_penalty (src/sampler.c:35-52: `pres` subtracted once
 * per distinct in-range id) and sampler_apply_repetition_penalty (:21-33: once
 * per occurrence, negative logits multiplied, others divided, only when
 * rep > 1), plus the frequency penalty (freq * count once per distinct id), in
 * `order` (DLK_OP_* nibbles, low first). */
int dlk_apply_penalties(float *logits, int64_t ld, int rows, int vocab, const int32_t *hist_off,
                        const int32_t *hist_ids, uint32_t order, float rep, float freq, float pres,
                        hipStream_t stream);

/* ---- grammar masks (src/core/grammar.c) ------------------------------------ */

/* Grammar modes, chosen from the grammar text as diskllm_grammar_init_from_str
 * does (src/core/grammar.c:21-26): receipt when it names bbox_2d (checked
 * first, :240), else JSON when it names object or value, else no constraint. */
#define DLK_GRAMMAR_NONE 0
#define DLK_GRAMMAR_JSON 1
#define DLK_GRAMMAR_RECEIPT 2
#define DLK_GRAMMAR_BUF 8192      /* the reference's buffer: buffer + piece must stay < 8191 bytes */

/* State of one validator after the bytes fed so far (a resumable form of
 * is_valid_receipt_prefix / is_valid_json_prefix, src/core/grammar.c:68-226). */
typedef struct {
    int32_t mode;             /* DLK_GRAMMAR_* */
    int32_t pc;               /* program point; 255 = rejected */
    int32_t n, m;             /* receipt: key / number position; JSON: brace / bracket depth */
    uint8_t prev;             /* previous byte */
    uint8_t flag;             /* receipt: the number had a digit; JSON: inside a string */
    uint8_t pad[2];
} dlk_scan_state;

/* Balance of the whole buffer (diskllm_grammar_is_finished, src/core/grammar.c:258-273). */
typedef struct {
    int32_t braces, brackets;
    int32_t len;              /* bytes in the buffer */
    uint8_t in_str, prev, pad[2];
} dlk_balance_state;

/* One sequence's grammar position: everything the mask needs about its buffer. */
typedef struct {
    dlk_scan_state scan;
    dlk_balance_state bal;
} dlk_grammar_row;

/* Host helpers (plain C, no device work): the mode a grammar text selects, a
 * fresh row, and a row advanced by n appended buffer bytes. */
int dlk_grammar_mode_of(const char *grammar_text);
void dlk_grammar_row_init(dlk_grammar_row *row, int mode);
void dlk_grammar_row_feed(dlk_grammar_row *row, const char *bytes, int n);

/* Grammar allow-masks for `rows` sequences (states: device array of
 * dlk_grammar_row) over one vocabulary of token strings in CSR form, token t =
 * bytes[off[t] .. off[t+1]) read up to its first NUL (strlen).  Per token, as
 * diskllm_grammar_apply_mask (src/core/grammar.c:275-308): the EOS id is
 * allowed iff the buffer is finished; an empty string is not allowed; any other
 * token iff buffer + token fits the buffer and is still a valid prefix.
 * Writes mask[r * mask_ld + w] (bit t%32 of word t/32, 1 = allowed); when
 * `logits` is not NULL sets disallowed logits[r * ld + t] to -inf; when `valid`
 * is not NULL writes each row's allowed count (the reference's return value). */
int dlk_grammar_mask(const uint32_t *off, const uint8_t *bytes, int vocab, const dlk_grammar_row *states,
                     int rows, int eos_id, uint32_t *mask, int64_t mask_ld, float *logits, int64_t ld,
                     int32_t *valid, hipStream_t stream);

/* The device form of diskllm_grammar_advance (src/core/grammar.c:248-256) as
 * diskllm_sample_grammar applies it after the draw (src/core/sampler_api.c:
 * 65-70): for each row whose token (device array) is not eos_id, that token's
 * string (up to its first NUL) is appended to the row's buffer when buffer +
 * string stays below 8191 bytes, i.e. the row's states take those bytes. */
int dlk_grammar_advance(const uint32_t *off, const uint8_t *bytes, int vocab, dlk_grammar_row *states,
                        const int32_t *tokens, int rows, int eos_id, hipStream_t stream);

/* One constrained decoding step for a batch, on the device, replacing
 * diskllm_sample_grammar (src/core/sampler_api.c:48-73) per row: the grammar
 * mask of each row's state (written to batch->mask, which must be a
 * [rows, mask_ld] buffer, and mask_row NULL), penalties and the draw as
 * dlk_sample (params->order DLK_ORDER_REFERENCE gives the reference's order),
 * then the rows' states advanced by the drawn tokens.
 * Unlike the reference it does not write -inf into the caller's logits. */
int dlk_sample_grammar(const dlk_batch *batch, int rows, int vocab, const dlk_sample_params *params,
                       const uint32_t *off, const uint8_t *bytes, dlk_grammar_row *states, int eos_id,
                       hipStream_t stream);

/* The reference's logit soft-cap, in place: logits[r * ld + i] = cap *
 * tanhf(logits[r * ld + i] / cap) for i < vocab (src/core/context.c:604-606
 * after a prefill, :873-876 after a decode step, a host loop there), with tanhf
 * bit-identical to the host libm's.  No-op unless cap > 0, as in the reference. */
int dlk_softcap(float *logits, int64_t ld, int rows, int vocab, float cap, hipStream_t stream);

/* ---- logits from 8-bit weights -------------------------------------------------
 * What stands before the calls above in a decode step: the LM head of a model whose
 * weights are kept in 8 bits, with the soft-cap as its epilogue (the reference's LM
 * head and cap, src/core/context.c:854-876, on block-quantised weights there).  No
 * counterpart of the 8-bit form in the reference. */

/* Element types of dlk_quantize_rows' input. */
#define DLK_F32 0
#define DLK_BF16 1
#define DLK_F16 2

/* Row-wise symmetric quantisation: scale[r] = max_i |x[r * ldx + i]| / 127 (one
 * float rounding), q[r * ldq + i] = x / scale[r] to the nearest integer, halves to
 * even, decided exactly; within +-127.  A row of zeros, or of values so small that the
 * scale rounds to 0: scale 0 and zeros.  A row that holds NaN or infinity: scale NaN and
 * zeros, so its logits are NaN.  Hidden states take it per token, weights [vocab, n] once
 * per channel.  x, q and scale need the alignment of their elements only and may not
 * overlap; strides are in elements. */
int dlk_quantize_rows(const void *x, int dtype, int64_t ldx, int rows, int n, int8_t *q, int64_t ldq, float *scale,
                      hipStream_t stream);

/* logits[r * ld + v] = (sum_i x[r * ldx + i] * w[v * ldw + i]) * x_scale[r] * w_scale[v],
 * the sum exact in 32-bit integers (n <= 131,071, else DLK_ERR_UNSUPPORTED), then
 * three float roundings (the sum's, and one per scale); softcap > 0: then softcap *
 * tanh(logit / softcap) to 2^-20 of it, or to 2^-148 * softcap or 2^-149 (the smallest
 * float) where one of those is more (not libm's bits, which dlk_softcap gives); softcap
 * must be finite.  Any strides and byte alignment of x and w; where both are 16-byte
 * aligned with strides that are multiples of 16, the 16 bytes that hold a row's last entry
 * are read to their end (what stands there does not matter).  Entries past vocab in a
 * row of logits are left as they are; logits may not overlap the inputs. */
int dlk_logits_i8(const int8_t *x, int64_t ldx, const float *x_scale, const int8_t *w, int64_t ldw,
                  const float *w_scale, int rows, int vocab, int n, float softcap, float *logits, int64_t ld,
                  hipStream_t stream);

/* ---- logits from 4-bit weights ---------------------------------------------------
 * The same head with its weights in microscaled 4-bit floating point: half the bytes of
 * the 8-bit one, which a decode step is bound by.  A row of n values is ceil(n / 32) blocks
 * of 32; block b's value i is an element times 2^(scale[b] - 127).  Elements: DLK_MX_FP4, 16
 * bytes a block, value 2 k in the low and 2 k + 1 in the high half of byte k, each a sign and
 * one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (E2M1); DLK_MX_FP6, 24 bytes a block, value i in the 6 bits
 * from 6 i on (the first byte's lowest bit is bit 0), each a sign and one of 0, 0.125 .. 2, 2.25 .. 4,
 * 4.5 .. 7.5 (E2M3): for hidden states, which 4 bits are few for.  Scale 255: NaN.  No counterpart
 * in the reference. */
#define DLK_MX_FP4 0
#define DLK_MX_FP6 1

/* Blocks of each row of x [rows, n] (DLK_F32, DLK_BF16 or DLK_F16; strides in elements).  A
 * block's scale is 2^(floor(log2(max |x|)) - 2), at least 2^-127; its elements are x over that
 * to the nearest, halves to the even code, decided exactly, and at most the largest element.
 * A block of zeros: scale 2^-127 and zeros; one that holds NaN or infinity: scale 255 and
 * zeros.  The last block of a row is filled with zeros.  q takes ceil(n / 32) * 16 (FP6: 24)
 * bytes a row at q + r * ldq, 8-byte aligned (ldq too); scale ceil(n / 32) bytes a row at
 * scale + r * ld_scale, of any alignment.  x needs its elements' alignment; no overlaps. */
int dlk_quantize_mx(const void *x, int dtype, int64_t ldx, int rows, int n, int format, uint8_t *q, int64_t ldq,
                    uint8_t *scale, int64_t ld_scale, hipStream_t stream);

/* The values of rows of blocks, n of each, in `dtype` (rounded to the nearest, halves to even, where
 * it does not hold them): out[r * ld + i] of row ids[r] of the table q, or of row r where ids is
 * NULL: with ids the embedding rows of tokens from a tied table.  An id outside [0,
 * table_rows) gives zeros; rows <= table_rows without ids, and a table without rows is refused
 * (DLK_ERR_INVALID) where rows > 0, with ids too.  Alignment as above; of out its elements'. */
int dlk_dequantize_mx(const uint8_t *q, int64_t ldq, const uint8_t *scale, int64_t ld_scale, int table_rows,
                      const int32_t *ids, int rows, int n, int format, void *out, int dtype, int64_t ld,
                      hipStream_t stream);

/* logits[r * ld + v] = sum over the ceil(n / 32) blocks of x's row r (x_format) and w's row v
 * (FP4) of their values' products; softcap as in dlk_logits_i8.  The products of a block are
 * exact, sums are in 32 bits: off by at most 2^-20 of the sum of the products' sizes for each
 * 512 values or part of them (four sums); products below 2^-149 may count as 0.  A block with
 * scale 255 makes its row's logits NaN.
 * x, w and the scales: 16-byte aligned (x in FP6: 8), strides too (the bytes of a row of
 * scales up to the next multiple of 16 are read; what stands there does not matter).  Entries
 * past vocab in a row of logits are left as they are; logits may not overlap the inputs. */
int dlk_logits_mx(const uint8_t *x, int x_format, int64_t ldx, const uint8_t *x_scale, int64_t ldxs, const uint8_t *w,
                  int64_t ldw, const uint8_t *w_scale, int64_t ldws, int rows, int vocab, int n, float softcap,
                  float *logits, int64_t ld, hipStream_t stream);

/* ---- scores of tokens ----------------------------------------------------------------
 * What a model's logits say of tokens that are known: the log-probabilities that a
 * request asks for beside its sampled tokens, of a prompt's tokens, or of a batch in
 * training, with their gradient.  No counterpart in the reference. */

#define DLK_MAX_GIVEN 64                /* given tokens of a row */
#define DLK_MAX_ALTERNATIVES 64         /* alternatives of a row */

typedef struct {
    const void *logits;       /* [rows, ld] of dtype, read only */
    int dtype;                /* DLK_F32, DLK_BF16 or DLK_F16 */
    int64_t ld;               /* row stride in elements (>= vocab) */
    const uint32_t *mask;     /* packed allow-masks as in dlk_batch, or NULL */
    int64_t mask_ld;
    const int32_t *mask_row;
    const int32_t *tokens;    /* [rows, n_given]; outside [0, vocab): no token */
    float *out_logprobs;      /* [rows, n_given] their log-probabilities; 0 where there is no token */
    float *out_stats;         /* [rows, 4] or NULL: largest allowed logit, sum of exp((l - largest) / T),
                                 entropy, log of the sum of exp(l / T) */
    int32_t *out_top_ids;     /* [rows, n_top] the largest allowed logits' ids, largest first, of equal ones the lower
                                 id; -1 where a row has no more */
    float *out_top_logprobs;  /* [rows, n_top] their log-probabilities; -inf likewise */
    uint32_t *status;         /* one word of DLK_STATUS_* bits, OR-ed, or NULL */
} dlk_logprob_batch;

typedef struct {
    int n_given;              /* tokens of each row, at most DLK_MAX_GIVEN; 0 = none */
    int n_top;                /* alternatives of each row, at most DLK_MAX_ALTERNATIVES; 0 = none */
    float temperature;        /* T: finite, at least 1e-30 */
} dlk_logprob_params;

/* log p_v = l_v / T - log(sum_u exp(l_u / T)) over the ids that the mask allows (-inf for
 * the others); the entropy -sum p log p.  The logits are read once, with alternatives those near them
 * again (where too many are equal, all).  A row without an allowed logit
 * above -inf: log-probabilities -inf, statistics -inf, 0, 0 and -inf, no alternatives.  A
 * row whose allowed logits hold NaN or +inf: NaN (ids -1), and DLK_STATUS_NOT_FINITE; what stands in
 * places that are not allowed does not matter.  Exponentials and sums of up to 32 terms in
 * 32 bits, the rest in 64: at up to 262,144 logits a row log-probabilities are off by their own rounding and
 * 2.2e-5 at most (logits of 16 bits: 1.4e-5; some 2e-7 as measured).  Takes workspace as dlk_sample does
 * where rows are few (dlk_release_stream; one call on the stream before capturing it, else
 * DLK_ERR_HIP).  Outputs may not overlap inputs. */
int dlk_token_logprobs(const dlk_logprob_batch *batch, int rows, int vocab, const dlk_logprob_params *params,
                       hipStream_t stream);

typedef struct {
    const void *logits;       /* these as in the forward call */
    int dtype;
    int64_t ld;
    const uint32_t *mask;
    int64_t mask_ld;
    const int32_t *mask_row;
    const int32_t *tokens;
    const float *stats;       /* [rows, 4] as dlk_token_logprobs has left them */
    const float *grad_logprobs;  /* [rows, n_given] */
    const float *grad_entropy;   /* [rows], or NULL: 0 */
    void *grad;               /* [rows, ld_grad] of dtype: written; the logits themselves (ld_grad == ld) or apart from
                                    them */
    int64_t ld_grad;
} dlk_logprob_grad_batch;

/* The logits' gradient of sum_j grad_logprobs[r, j] * logprob[r, j] + grad_entropy[r] * entropy[r]:
 *   grad_v = (1 / T) * (sum_j g_j [v = token_j] - p_v * (sum_j g_j + h * (log p_v + entropy)))
 * in 32 bits, rounded once to dtype; 0 for ids that are not allowed or whose logit is -inf.  The same
 * token may be given several times.  Places without a token, or whose token the mask does not allow or
 * whose logit is -inf, count for nothing.  A row in which nothing is to be differentiated (every g that
 * counts and h are 0, or no logit is allowed): zeros, whatever its logits hold; else a row whose statistics
 * are NaN gets NaN for its allowed ids, but for those whose logit is -inf.  n_top does not matter.  No
 * workspace. */
int dlk_token_logprobs_grad(const dlk_logprob_grad_batch *batch, int rows, int vocab, const dlk_logprob_params *params,
                            hipStream_t stream);

/* ---- beam search ----------------------------------------------------------------
 * The deterministic counterpart of dlk_sample: the best continuations of each group
 * (request) of `beams` rows over the vocabulary, and the beams' states following
 * their parents.  No counterpart in the reference. */

#define DLK_STATUS_NOT_FINITE 8u        /* dlk_beam_select: a row's allowed logits held NaN or +inf, or its score
                                           was NaN or +inf: it has no continuations */
#define DLK_MAX_BEAMS 64                /* beams and n_out */

typedef struct {
    const float *logits;      /* [groups * beams, ld] fp32, read only; row g * beams + b is beam b of group g */
    int64_t ld;
    const int32_t *hist_off;  /* histories and masks as in dlk_batch, per row; or NULL */
    const int32_t *hist_ids;
    const uint32_t *mask;
    int64_t mask_ld;
    const int32_t *mask_row;
    const float *scores;      /* [groups * beams] sums of log-probabilities, -inf: no such beam; NULL = all 0 */
    const int32_t *lengths;   /* [groups * beams] tokens so far, for the length penalty; NULL = all 0 */
    const uint8_t *finished;  /* [groups * beams] not 0: the beam has ended; NULL = none */
    int32_t *out_tokens;      /* [groups * n_out] the continuations, best first; -1 where a group has no more */
    int32_t *out_parents;     /* [groups * n_out] the row each continues; -1 likewise */
    float *out_scores;        /* [groups * n_out] their scores; -inf likewise */
    int32_t *out_lengths;     /* [groups * n_out] or NULL; 0 likewise */
    uint8_t *out_finished;    /* [groups * n_out] 1 where the token is eos_id, or NULL; 0 likewise */
    uint32_t *status;         /* one word of DLK_STATUS_* bits, OR-ed, or NULL */
} dlk_beam_batch;

typedef struct {
    int beams;                /* rows per group (1 before the first step of a request), at most DLK_MAX_BEAMS */
    int n_out;                /* continuations per group, at most DLK_MAX_BEAMS */
    int eos_id;               /* a continuation by this id has ended; -1 = none (finished is NULL then) */
    float length_penalty;     /* candidates are ordered by score / length^length_penalty; 0 = by score */
    float repeat_penalty;     /* as in dlk_sample_params */
    float frequency_penalty;
    float presence_penalty;
    uint32_t penalty_order;
    int max_history;          /* upper bound on any row's history (0 = 1024; at most 65,535); a row past it has no
                                 continuations and sets DLK_STATUS_HISTORY_TOO_LONG */
} dlk_beam_params;

/* One step of a beam search.  Row r's logits l are masked, then penalised, as
 * dlk_sample does; its continuation by id v has
 *   score = scores[r] + (l_v - max l) - log(sum_u exp(l_u - max l)),  length = lengths[r] + 1,
 * computed in 64 bits (exponentials to 4e-15 of each) and rounded once.  A finished row has one continuation: eos_id,
 * with its score and length as they are (whatever its logits hold).  Ids with logit
 * -inf are no continuations, nor are those of rows with score -inf.
 * Of each group's continuations the n_out with the largest score / max(length,
 * 1)^length_penalty (before rounding) are written, largest first; of equal ones the
 * lower row first, then the larger logit, then the lower id (continuations of two rows
 * whose scores over length^length_penalty differ by no more than what those roundings come
 * to, 2^-42 and 2^-50 of their size at up to 262,144 logits a row, may come in either
 * order, the same in every call of these inputs).  Outputs may not overlap
 * inputs (an output that is its own input is refused).  Takes workspace as dlk_sample
 * does (dlk_release_stream; one call on the stream before capturing it, else
 * DLK_ERR_HIP). */
int dlk_beam_select(const dlk_beam_batch *batch, int groups, int vocab, const dlk_beam_params *params,
                    hipStream_t stream);

/* One buffer whose rows follow the beams: bytes at
 *   base + o * outer + r * row + i * inner,  o < n_outer, i < n_inner,
 * for row r; a cache [layers, rows, heads, room, width] filled up to `length` has outer =
 * layer, inner = head and bytes = length * width * element size.  Strides in bytes,
 * not negative.  src == dst: in place, with equal strides. */
typedef struct {
    const void *src;
    void *dst;
    int64_t bytes;
    int64_t src_row, src_outer, src_inner;
    int64_t dst_row, dst_outer, dst_inner;
    int n_outer, n_inner;
} dlk_beam_state;

/* The rows' histories (CSR, as in dlk_batch) and the tokens to append. */
typedef struct {
    const int32_t *off;       /* [groups * beams + 1] */
    const int32_t *ids;
    const int32_t *tokens;    /* [groups * n_out] appended; a negative one appends nothing; NULL = none */
    int max_history;          /* each new history keeps its last max_history ids */
    int32_t *out_off;         /* [groups * n_out + 1]; no overlap with the inputs */
    int32_t *out_ids;         /* room for groups * n_out * max_history ids; those past out_off's last are left */
} dlk_beam_history;

/* The states of groups * n_out rows from those of groups * beams: row r takes row
 * parents[r] (as dlk_beam_select writes it).  A parent outside its own group's rows
 * (-1 among them) moves nothing: the row's states are left, its history is empty.
 * In-place states need n_out == beams; they move as if all rows were read before
 * any is written, and rows that are their own parents cost nothing.  Destinations of
 * one call may not overlap one another, nor any source but their own in place (states
 * that begin at one address are refused).
 * n_states of any number; history may be NULL. */
int dlk_beam_reorder(const int32_t *parents, int groups, int beams, int n_out, const dlk_beam_state *states,
                     int n_states, const dlk_beam_history *history, hipStream_t stream);

/* The vocabulary table of the calls above (token t = bytes[off[t] .. off[t+1]),
 * read up to its first NUL) from a GGUF file's `tokenizer.ggml.tokens` string
 * array: the strings tokenizer_init loads (src/tokenizer.c:247-300) and
 * tokenizer_decode_raw returns (src/tokenizer.c:377-380).  Host memory, no
 * device work.  The table covers ids 0 .. vocab-1 (vocab <= 0: one id per
 * string); ids past the file's strings get empty entries, which the mask
 * disallows as the reference does the NULL string it gets for them.  A file
 * with no tokens array gives an all-empty table (the reference's tokenizer
 * has vocab_size 0 then).  Call once with off = NULL to get *n_tokens (the
 * array's length) and *n_bytes (bytes the table needs), then with off
 * ([vocab+1] entries) and bytes ([bytes_cap] bytes) to fill them.
 * DLK_ERR_FORMAT: the file cannot be opened, is truncated, is not GGUF, or its
 * tokens array does not hold strings; DLK_ERR_INVALID: bytes_cap too small. */
int dlk_vocab_csr_from_gguf(const char *path, int vocab, uint32_t *off, uint8_t *bytes, int64_t bytes_cap,
                            int32_t *n_tokens, int64_t *n_bytes);

/* The token-string callback of diskllm_grammar_apply_mask (include/grammar.h,
 * src/core/grammar.c:275-308: NUL-terminated strings, NULL for no string) over a
 * table in the form above, for callers that hold the vocabulary as that table
 * rather than as a tokenizer (no counterpart in the reference, whose caller
 * passes tokenizer_decode_raw, src/core/sampler_api.c:42-46).  ctx points to a
 * dlk_csr_vocab; the string is copied into its scratch buffer (scratch_cap
 * bytes; longer entries are cut there), so one ctx serves one thread at a time.
 * NULL for ids outside [0, vocab). */
typedef struct {
    const uint32_t *off;      /* [vocab+1] */
    const uint8_t *bytes;
    int vocab;
    char *scratch;            /* [scratch_cap] */
    int scratch_cap;
} dlk_csr_vocab;
const char *dlk_csr_token_str(void *ctx, int token_id);

#ifdef __cplusplus
}
#endif

#endif
