/*
 * token_logprobs_grad.hip -- the logits' gradient of the given tokens' log-probabilities and
 * of the entropy (dlk_token_logprobs_grad):
 *
 *   dl_v = (1 / T) * (sum_j g_j [v = token_j] - p_v * (sum_j g_j + h * (log p_v + entropy)))
 *
 * over the given tokens whose own logit is above -inf (-inf is a mask as the bits are), with
 * p_v = 2^((l_v - max) * log2(e) / T) / z of the statistics that the forward call left, so that a
 * row is read once and no workgroup waits for another.  Bound by memory: 256 threads, 16-byte
 * groups, a wave's 64 groups side by side, of which it knows by one ballot of the tokens (a lane
 * each) whether any lies there.  2,048 x 151,936 bfloat16 215 us, 5.8 TB/s read and written (a
 * large copy: 4.9); 48 x 50,257 float32 5.9 within a graph, its statistics and tokens, and then the tokens' logits,
 * a round trip each before the first product.  Over the logits the tokens' groups are a launch of their
 * own (48 x 50,257 with four tokens a row 9.6, 2,048 x 151,936 bfloat16 250; in one launch, which could
 * take a stored gradient for a token's logit, 6.5 and 245).
 */
#include "logit_row.h"
#include "../../../include/diskllm_amd.h"

namespace dlk {

constexpr int kGradThreads = 256;

struct GradParams {
    const void *logits;
    int64_t ld;
    const uint32_t *mask;
    int64_t mask_ld;
    const int32_t *mask_row;
    const int32_t *tokens;
    const float *stats, *g, *h;
    void *grad;
    int64_t ld_grad;
    int V, given, pieces;
    float scale, inv_t;  /* log2(e) / T, 1 / T */
    bool past;           /* stores go past the caches */
    int64_t r0;
};

/* Lane k's v, k the same in all lanes. */
DLK_DEV int32_t of_lane(int32_t v, int k) { return __builtin_amdgcn_readlane(v, k); }
DLK_DEV float of_lane(float v, int k) { return u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(v), k)); }

/* What a row's workgroups all know of it. */
struct GradRow {
    int32_t held, token;     /* this lane's given token: that the mask allows, that counts (its logit above -inf); else -1 */
    float g;                 /* its weight, 0 where it does not count */
    float top, by, by_t;     /* p's weight is by + by_t * (the logit's exponent of 2) */
    bool none;               /* no allowed id, or nothing to differentiate (whatever the logits hold): zeros */
};

template <int DT, bool ENTROPY>
DLK_DEV GradRow grad_row(const GradParams &p, int64_t row, const typename LogitRow<DT>::T *lg, const uint32_t *mw) {
    GradRow r;
    const int lane = lane_id();
    const float z = p.stats[row * 4 + 1], entropy = p.stats[row * 4 + 2];
    r.top = p.stats[row * 4];
    r.token = -1;
    r.g = 0.0f;
    if (lane < p.given) {
        r.token = p.tokens[row * p.given + lane];
        r.g = p.g[row * p.given + lane];
    }
    if (r.token < 0 || r.token >= p.V || !mask_allows(mw, r.token)) r.token = -1;
    r.held = r.token;
    if (r.token >= 0 && LogitRow<DT>::one(lg + r.token) == -INFINITY) r.token = -1;
    if (r.token < 0) r.g = 0.0f;
    float h = 0.0f;
    if (ENTROPY) h = p.h[row];
    float total = 0.0f;
#pragma unroll 1
    for (int j = 0; j < p.given; j++) total += of_lane(r.g, j);
    r.none = r.top == -INFINITY || (ballot(r.g != 0.0f) == 0 && h == 0.0f);
    const float per = p.inv_t * (1.0f / z);
    r.by = ENTROPY ? (total + h * (entropy - logf(z))) * per : total * per;
    r.by_t = ENTROPY ? h * 0.693147180559945309f * per : 0.0f;
    return r;
}

/* -p_v * its weight for the group of logits x at i. */
template <int DT, bool ENTROPY>
DLK_DEV void grad_group(const GradParams &p, const GradRow &r, const uint32_t *mw, int i, const float (&x)[LogitRow<DT>::G],
                        float (&y)[LogitRow<DT>::G]) {
    uint32_t bits = 0xffffffffu;
    if (mw) bits = mw[min(i, p.V - 1) >> 5] >> (i & 31);
#pragma unroll
    for (int c = 0; c < LogitRow<DT>::G; c++) {
        const float d = (x[c] - r.top) * p.scale, e = __builtin_amdgcn_exp2f(d);
        y[c] = ENTROPY ? -e * fmaf(r.by_t, fmaxf(d, -200.0f), r.by) : -e * r.by;
        if (mw) y[c] = (bits >> c & 1) != 0 ? y[c] : 0.0f;
        y[c] = r.none || x[c] == -INFINITY ? 0.0f : y[c];
    }
}

/* Row blockIdx.x / pieces, piece blockIdx.x % pieces: four groups a thread.  OVER: the gradient goes over the logits;
 * every workgroup of a row reads its tokens' logits, so their groups are left to the kernel below. */
template <int DT, bool ENTROPY, bool OVER>
__global__ __launch_bounds__(kGradThreads) void token_logprobs_grad_kernel(GradParams p) {
    typedef LogitRow<DT> In;
    constexpr int T = kGradThreads, GR = 4, G = In::G, B = T * GR * G;
    const int t = threadIdx.x;
    const int64_t row = p.r0 + blockIdx.x / p.pieces;
    const int b0 = (int)(blockIdx.x % p.pieces) * B;
    const typename In::T *lg = (const typename In::T *)p.logits + row * p.ld;
    typename In::T *out = (typename In::T *)p.grad + row * p.ld_grad;
    const uint32_t *mw = p.mask ? p.mask + (int64_t)(p.mask_row ? p.mask_row[row] : row) * p.mask_ld : nullptr;
    const int s1 = p.V;
    typename In::Raw raw[GR];
    auto place = [&](int j) { return b0 + (j * T + t) * G; };
#pragma unroll
    for (int j = 0; j < GR; j++)
        if (place(j) + G <= s1) raw[j] = *(const typename In::Raw *)(lg + place(j));
    const GradRow r = grad_row<DT, ENTROPY>(p, row, lg, mw);
#pragma unroll
    for (int j = 0; j < GR; j++) {
        const int i = place(j);
        float x[G], y[G];
        if (i + G <= s1) {
            In::unpack(raw[j], x);
        } else {
#pragma unroll
            for (int c = 0; c < G; c++) x[c] = i + c < s1 ? In::one(lg + i + c) : -INFINITY;
        }
        grad_group<DT, ENTROPY>(p, r, mw, i, x, y);
        /* the wave's 64 groups lie side by side: the tokens among them, in their order */
        const int w0 = b0 + (j * T + (t & ~63)) * G;
        bool mine = true;
        const int32_t of = OVER ? r.held : r.token;
        for (uint64_t who = ballot(of >= w0 && of - w0 < 64 * G); who != 0; who &= who - 1) {
            const int k = __builtin_ctzll(who);
            const int at = shfl(of, k) - i;
            if (OVER) {
                mine &= at < 0 || at >= G;
            } else {
                const float add = shfl(r.g, k) * p.inv_t;
#pragma unroll
                for (int c = 0; c < G; c++) y[c] += at == c && !r.none ? add : 0.0f;
            }
        }
        if (OVER && !mine) continue;
        if (i + G <= s1) {
            store_past<sizeof(*out)>(out + i, In::pack(y), p.past);
        } else {
#pragma unroll
            for (int c = 0; c < G; c++)
                if (i + c < s1) In::put(out + i + c, y[c]);
        }
    }
}

/* The tokens' groups of a gradient over its logits, a wave a row and a lane a token: a wave has read all of its row's
 * before it stores one. */
template <int DT, bool ENTROPY>
__global__ __launch_bounds__(kGradThreads) void token_logprobs_grad_tokens_kernel(GradParams p, int rows) {
    typedef LogitRow<DT> In;
    constexpr int G = In::G;
    const int lane = lane_id(), n = (int)blockIdx.x * (kGradThreads / 64) + wave_id();
    if (n >= rows) return;
    const int64_t row = p.r0 + n;
    typename In::T *lg = (typename In::T *)p.grad + row * p.ld_grad;
    const uint32_t *mw = p.mask ? p.mask + (int64_t)(p.mask_row ? p.mask_row[row] : row) * p.mask_ld : nullptr;
    const GradRow r = grad_row<DT, ENTROPY>(p, row, lg, mw);
    const int i = max(r.held, 0) / G * G;
    float x[G], y[G];
#pragma unroll
    for (int c = 0; c < G; c++) x[c] = i + c < p.V ? In::one(lg + i + c) : -INFINITY;
    grad_group<DT, ENTROPY>(p, r, mw, i, x, y);
    bool mine = r.held >= 0;                       /* no earlier lane has this group */
#pragma unroll 1
    for (int k = 0; k < p.given; k++) {
        const int at = of_lane(r.token, k) - i, first = of_lane(r.held, k);
        const float add = of_lane(r.g, k) * p.inv_t;
        mine &= k >= lane || first < i || first >= i + G;
#pragma unroll
        for (int c = 0; c < G; c++) y[c] += at == c && !r.none ? add : 0.0f;
    }
    __builtin_amdgcn_s_waitcnt(0);
    if (!mine) return;
#pragma unroll
    for (int c = 0; c < G; c++)
        if (i + c < p.V) In::put(lg + i + c, y[c]);
}

template <int DT, bool ENTROPY>
int launch_grad_kernels(const GradParams &p, int64_t rows, hipStream_t stream) {
    const dim3 pieces((unsigned)(rows * p.pieces)), threads(kGradThreads);
    constexpr int waves = kGradThreads / 64;
    if (p.grad != p.logits || p.given == 0) {
        hipLaunchKernelGGL((token_logprobs_grad_kernel<DT, ENTROPY, false>), pieces, threads, 0, stream, p);
    } else {
        hipLaunchKernelGGL((token_logprobs_grad_kernel<DT, ENTROPY, true>), pieces, threads, 0, stream, p);
        hipLaunchKernelGGL((token_logprobs_grad_tokens_kernel<DT, ENTROPY>), dim3((unsigned)((rows + waves - 1) / waves)),
                           threads, 0, stream, p, (int)rows);
    }
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

template <int DT>
int launch_grad(const GradParams &p, int64_t rows, hipStream_t stream) {
    return p.h ? launch_grad_kernels<DT, true>(p, rows, stream) : launch_grad_kernels<DT, false>(p, rows, stream);
}

}  // namespace dlk

extern "C" int dlk_token_logprobs_grad(const dlk_logprob_grad_batch *b, int rows, int vocab,
                                       const dlk_logprob_params *prm, hipStream_t stream) {
    using namespace dlk;
    if (!b || !prm || rows < 0 || vocab <= 0 || !b->logits || !b->stats || !b->grad) return DLK_ERR_INVALID;
    if (b->ld < vocab || b->ld_grad < vocab) return DLK_ERR_INVALID;
    if (b->dtype != DLK_F32 && b->dtype != DLK_BF16 && b->dtype != DLK_F16) return DLK_ERR_INVALID;
    if (prm->n_given < 0 || (prm->n_given > 0 && (!b->tokens || !b->grad_logprobs))) return DLK_ERR_INVALID;
    if (b->mask && b->mask_ld < (vocab + 31) / 32) return DLK_ERR_INVALID;
    if (!(prm->temperature >= 1e-30f && prm->temperature < INFINITY)) return DLK_ERR_INVALID;
    const uintptr_t align = b->dtype == DLK_F32 ? 3 : 1;
    if ((((uintptr_t)b->logits | (uintptr_t)b->grad) & align) != 0) return DLK_ERR_INVALID;
    /* over the logits: place by place only */
    if (b->grad == b->logits && rows > 1 && b->ld_grad != b->ld) return DLK_ERR_INVALID;
    if (prm->n_given > DLK_MAX_GIVEN || vocab > 0x7fffffff - (1 << 20)) return DLK_ERR_UNSUPPORTED;
    if (rows == 0) return DLK_OK;
    GradParams p;
    p.logits = b->logits; p.ld = b->ld; p.mask = b->mask; p.mask_ld = b->mask_ld; p.mask_row = b->mask_row;
    p.tokens = b->tokens; p.stats = b->stats; p.g = b->grad_logprobs; p.h = b->grad_entropy;
    p.grad = b->grad; p.ld_grad = b->ld_grad; p.V = vocab; p.given = prm->n_given;
    p.inv_t = 1.0f / prm->temperature;
    p.scale = (float)(1.4426950408889634 / (double)prm->temperature);
    /* (64 x 151,936 bf16, 19 MB: 9.5 us past the caches, 10.9 through them; 48 x 50,257 float32, 10 MB: 7.9 both) */
    const int64_t size = b->dtype == DLK_F32 ? 4 : 2;
    p.past = rows * size * vocab >= 16 << 20 && whole_lines(b->grad, b->ld_grad * size);
    const int batch = kGradThreads * 4 * (b->dtype == DLK_F32 ? 4 : 8);
    p.pieces = (int)(((int64_t)vocab + batch - 1) / batch);
    /* (2^32 threads and over are no launch) */
    const int64_t most = 0xffffffLL / p.pieces;
    for (p.r0 = 0; p.r0 < rows; p.r0 += most) {
        const int64_t n = rows - p.r0 < most ? rows - p.r0 : most;
        const int rc = b->dtype == DLK_F32 ? launch_grad<DLK_F32>(p, n, stream)
                     : b->dtype == DLK_BF16 ? launch_grad<DLK_BF16>(p, n, stream)
                                            : launch_grad<DLK_F16>(p, n, stream);
        if (rc != DLK_OK) return rc;
    }
    return DLK_OK;
}
