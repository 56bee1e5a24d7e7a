/*
 * token_logprobs.hip -- log-probabilities of given tokens, the entropy and the largest
 * alternatives of each row of logits (dlk_token_logprobs).
 *
 *   t_v = (l_v - max) * log2(e) / T,  z = sum 2^t_v,  u = sum 2^t_v * t_v  (over the allowed ids)
 *   log p_v = (l_v - max) / T - log z,  entropy = log z - ln2 * u / z   (both terms >= 0: nothing cancels)
 *
 * One workgroup reads a slice of a row (logprob_slices() to a row) once, a batch of four
 * 16-byte groups a thread at a time into registers.  Each thread keeps its own maximum and
 * its sums below it: 16 or 32 terms of a batch are added in 32 bits, batches in 64, so that
 * log z of a row that is nearly sure of one token (1 + little) keeps the little: its own
 * roundings, not those of 1, are what such a token's log-probability shows.
 * A wave lists its slice's n largest entries (top_list.h) as the beam selection's do.  The
 * row's last workgroup to finish joins sums and lists; no order of arrival shows.
 */
#include "top_list.h"
#include "logit_row.h"
#include "token_logprobs.h"

namespace dlk {

constexpr int kScoreWaveList = 256;    /* entries that a wave lists */
constexpr int kScoreJoin = 512;        /* entries that a join ranks at once */

/* The largest of three; NaN where one is NaN. */
DLK_DEV float maximum3(float a, float b, float c) {
    float d;
    asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

struct ScoreShared {
    uint64_t list[kLogprobThreads / 64][kScoreWaveList];
    uint64_t joint[kLogprobThreads / 64 * kScoreWaveList];
    double sum[kLogprobThreads / 64], dot[kLogprobThreads / 64];
    double lnz;
    float top[kLogprobThreads / 64];
    uint32_t wave_key[kLogprobThreads / 64];
    int listed[kLogprobThreads / 64], bad[kLogprobThreads / 64];
    float max;
    int last, count, row_bad;
};

/* A bound that n of the threads' keys reach: n / 4 of each wave's do, or, where a wave has too
 * few, n of one wave's.  0: none. */
DLK_DEV uint32_t score_bound(ScoreShared &sh, uint32_t key, int n) {
    uint32_t bound = 0;
#pragma unroll 1
    for (int one = 0; one < 2 && bound == 0; one++) {
        const uint32_t kw = wave_rth(key, one ? n : (n + 3) / 4);
        if (one) __syncthreads();
        if (lane_id() == 0) sh.wave_key[wave_id()] = kw;
        __syncthreads();
        bound = sh.wave_key[0];
#pragma unroll
        for (int w = 1; w < kLogprobThreads / 64; w++) bound = one ? max(bound, sh.wave_key[w]) : min(bound, sh.wave_key[w]);
    }
    return __builtin_amdgcn_readfirstlane(bound);
}

/* Sums over the wave as they are below the maximum `to` (all lanes' own maxima m <= to > -inf). */
DLK_DEV void lower(float m, float to, float scale, double &sum, double &dot) {
    const float d = fmaxf((m - to) * scale, -126.0f);
    const double f = m > -INFINITY ? (double)__builtin_amdgcn_exp2f(d) : 0.0;
    dot = m > -INFINITY ? (dot + sum * (double)d) * f : 0.0;
    sum *= f;
}

DLK_DEV void write_top(const LogprobParams &p, int64_t row, int j, int id, float lp) {
    p.top_ids[row * p.n + j] = id;
    p.top_logprobs[row * p.n + j] = lp;
}

/* The row's outputs: its maximum, sums and n largest entries (ranked among list[0 .. all)) are known. */
template <bool TOP>
DLK_DEV void finish_row(const LogprobParams &p, ScoreShared &sh, int64_t row, float top, double z, double u, bool bad,
                        int32_t token, float logit, const uint64_t *list, int all) {
    const int t = threadIdx.x;
    const bool some = top > -INFINITY;
    double lnz = 0.0;
    if (some && !bad) lnz = log(z);
    if (t < p.given) {
        /* -2: the mask does not allow it, -1: no token */
        float lp = 0.0f;
        if (token != -1) lp = bad ? u2f(0x7fc00000u) : some && token >= 0 ? (float)(((double)logit - (double)top) * p.inv_t - lnz) : -INFINITY;
        p.logprobs[row * p.given + t] = lp;
    }
    if (t == 0 && p.stats) {
        float4 s = make_float4(-INFINITY, 0.0f, 0.0f, -INFINITY);
        if (some) s = make_float4(top, (float)z, (float)(lnz - 0.69314718055994531 * u / z), (float)((double)top * p.inv_t + lnz));
        if (bad) s = make_float4(u2f(0x7fc00000u), u2f(0x7fc00000u), u2f(0x7fc00000u), u2f(0x7fc00000u));
        store4(p.stats + row * 4, s);
    }
    if (bad && t == 0 && p.status) atomicOr(p.status, DLK_STATUS_NOT_FINITE);
    if (TOP) {
        if (bad) all = 0;
        for (int a = t; a < all; a += kLogprobThreads) {
            const uint64_t e = list[a];
            int equal;
            const int rank = rank_in(list, all, e, equal);
            if (rank < p.n) write_top(p, row, rank, entry_id(e), (float)(((double)entry_logit(e) - (double)top) * p.inv_t - lnz));
        }
        for (int j = all + t; j < p.n; j += kLogprobThreads) write_top(p, row, j, -1, bad ? u2f(0x7fc00000u) : -INFINITY);
    }
}

/* The row's slices joined, by its last workgroup. */
template <bool TOP>
DLK_DEV void join_row(const LogprobParams &p, ScoreShared &sh, int rl, int32_t token, float logit) {
    constexpr int T = kLogprobThreads, PRE = kLogprobEntries / T;
    const int t = threadIdx.x, lane = lane_id();
    const LogprobSlot *slots = p.slots + (int64_t)rl * p.slices;
    const uint64_t *cands = p.cands + (int64_t)rl * p.slices * p.n;
    const int E = p.slices * p.n;
    uint64_t ent[PRE];
    /* every wave joins the sums for itself; the entries are asked for at the same time */
    const bool mine = lane < p.slices;
    const LogprobSlot *slot = slots + min(lane, p.slices - 1);
    double z = u2d(bget64(&slot->sum)), u = u2d(bget64(&slot->dot));
    const uint64_t mk = bget64(&slot->max_kept);
    if (TOP) {
#pragma unroll
        for (int q = 0; q < PRE; q++)
            if (q * T < E) ent[q] = bget64(&cands[min(q * T + t, E - 1)]);
        if (lane == 0 && wave_id() == 0) sh.count = 0;
    }
    const float m = mine ? u2f((uint32_t)(mk >> 32)) : -INFINITY;
    const bool bad = ballot(mine && (uint32_t)mk == 0xffffffffu) != 0;
    const float top = wave_max_dpp(m);
    lower(m, fmaxf(top, -3.40282347e38f), p.scale, z, u);
    z = shfl(wave_incl_scan_d(mine ? z : 0.0), 63);
    u = shfl(wave_incl_scan_d(mine ? u : 0.0), 63);
    int all = 0;
    if (TOP && !bad) {
        /* entry i of list s lies at s * n + i; those that a list does not have are 0 */
        uint64_t best = 0;
#pragma unroll
        for (int q = 0; q < PRE; q++) {
            if (q * T >= E) { ent[q] = 0; continue; }
            const int at = q * T + t, s = min(at, E - 1) / p.n;
            const int kept = (int)(uint32_t)shfl((int)(uint32_t)mk, s);
            if (at >= E || at - s * p.n >= kept) ent[q] = 0;
            best = max(best, ent[q]);
        }
        uint32_t bound = 0;
        if (E > 256) bound = score_bound(sh, (uint32_t)(best >> 32), p.n);
        else __syncthreads();
        auto gather = [&](uint64_t least) {
#pragma unroll
            for (int q = 0; q < PRE; q++)
                if (ent[q] != 0 && ent[q] >= least) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < kScoreJoin) sh.joint[at] = ent[q];
                }
        };
        gather((uint64_t)bound << 32);
        __syncthreads();
        all = sh.count;
        if (DLK_COLD(all > kScoreJoin)) {
            /* more than are ranked at once: the n-th largest entry, bit by bit (no two are equal) */
            uint64_t nth = 0;
#pragma unroll 1
            for (uint64_t bit = 1ull << 63; bit; bit >>= 1) {
                __syncthreads();
                if (t == 0) sh.count = 0;
                __syncthreads();
                int c = 0;
#pragma unroll
                for (int q = 0; q < PRE; q++) c += (int)__popcll(ballot(ent[q] >= (nth | bit)));
                if (lane == 0) atomicAdd(&sh.count, c);
                __syncthreads();
                if (sh.count >= p.n) nth |= bit;
            }
            __syncthreads();
            if (t == 0) sh.count = 0;
            __syncthreads();
            gather(nth);
            __syncthreads();
            all = sh.count;
        }
    }
    finish_row<TOP>(p, sh, (int64_t)p.r0 + rl, top, z, u, bad, token, logit, sh.joint, all);
}

/* A slice of a row: its share of the row's p.batches batches (shares differ by one at most). */
template <int DT, bool TOP>
__global__ __launch_bounds__(kLogprobThreads, 4) void token_logprobs_kernel(LogprobParams p) {
    typedef LogitRow<DT> In;
    constexpr int T = kLogprobThreads, GR = 4, G = In::G, E = GR * G, B = T * E;
    __shared__ ScoreShared sh;
    const int t = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int slice = blockIdx.x % p.slices, rl = blockIdx.x / p.slices;      /* rl: row of the launch */
    const int64_t row = (int64_t)p.r0 + rl;
    const typename In::T *lg = (const typename In::T *)p.logits + row * p.ld;
    const uint32_t *mw = p.mask ? p.mask + (int64_t)(p.mask_row ? p.mask_row[row] : row) * p.mask_ld : nullptr;
    const int s0 = (int)((int64_t)slice * p.batches / p.slices) * B;
    const int s1 = (int)min((int64_t)p.V, (int64_t)((int64_t)(slice + 1) * p.batches / p.slices) * B);
    typename In::Raw raw[GR];
    /* the thread's group j of the batch at b0 */
    auto place = [&](int b0, int j) { return b0 + (j * T + t) * G; };
    auto load = [&](int b0) {
#pragma unroll
        for (int j = 0; j < GR; j++)
            if (place(b0, j) + G <= s1) raw[j] = *(const typename In::Raw *)(lg + place(b0, j));
    };
    load(s0);
    /* the given tokens' logits: asked for here, used by the row's last workgroup (-1: no token, -2: not allowed) */
    int32_t token = -1;
    float logit = -INFINITY;
    if (t < p.given) {
        const int32_t id = p.tokens[row * p.given + t];
        if (id >= 0 && id < p.V) {
            token = mask_allows(mw, id) ? id : -2;
            logit = In::one(lg + id);
        }
    }
    float most = -INFINITY;                        /* this thread's maximum and its sums below it */
    double sum = 0.0, dot = 0.0;
    bool bad = false;
    uint64_t *list = sh.list[wave];
    int listed = 0;
    float least = -INFINITY;                       /* bound: n entries of the slice reach it (as a logit, and exactly) */
    uint64_t bound = 0;
    auto put = [&](bool take, uint64_t e) {
        const uint64_t who = ballot(take);
        const int at = place_in(who, listed);
        if (take && at < kScoreWaveList) list[at] = e;
        listed += (int)__popcll(who);
    };
    for (int b0 = s0; b0 < s1; b0 += B) {
        if (b0 != s0) load(b0);
        float x[GR][G];
#pragma unroll
        for (int j = 0; j < GR; j++) {
            const int i = place(b0, j);
            if (i + G <= s1) {
                In::unpack(raw[j], x[j]);
            } else {
#pragma unroll
                for (int c = 0; c < G; c++) x[j][c] = i + c < s1 ? In::one(lg + i + c) : -INFINITY;
            }
        }
        if (mw) {
            uint32_t bits[GR];
#pragma unroll
            for (int j = 0; j < GR; j++) bits[j] = mw[min(place(b0, j), s1 - 1) >> 5];
#pragma unroll
            for (int j = 0; j < GR; j++) {
                bits[j] >>= place(b0, j) & 31;     /* (a group lies in one word) */
#pragma unroll
                for (int c = 0; c < G; c++) x[j][c] = allowed_or_ninf(x[j][c], bits[j], c);
            }
        }
        float most_of[GR], best;
#pragma unroll
        for (int j = 0; j < GR; j++) {
            most_of[j] = maximum3(x[j][0], x[j][1], x[j][2]);
#pragma unroll
            for (int c = 3; c < G; c += 2) most_of[j] = maximum3(most_of[j], x[j][c], x[j][min(c + 1, G - 1)]);
        }
        best = maximum3(maximum3(most_of[0], most_of[1], most_of[2]), most_of[3], most_of[3]);
        bad |= !(best < INFINITY);
        if (TOP) {
            if (b0 == s0) {
                const uint32_t k = score_bound(sh, best > -INFINITY && best < INFINITY ? ~desc_key(best) : 0u, p.n);
                if (k != 0) least = key_value(~k);           /* (0: every id is an entry) */
                bound = (uint64_t)k << 32;
            }
            const int had = listed;
            if (ballot(best >= least) != 0) {
#pragma unroll
                for (int j = 0; j < GR; j++) {
                    if (ballot(most_of[j] >= least) == 0) continue;
                    uint32_t at_least = 0;
#pragma unroll
                    for (int c = 0; c < G; c++) at_least |= x[j][c] >= least && x[j][c] > -INFINITY ? 1u << c : 0u;
                    while (ballot(at_least != 0) != 0) {
                        const int k = at_least != 0 ? __builtin_ctz(at_least) : 0;
                        float v = x[j][0];
#pragma unroll
                        for (int c = 1; c < G; c++) v = k == c ? x[j][c] : v;
                        const uint64_t e = entry_of(v, place(b0, j) + k);
                        put(at_least != 0 && e >= bound, e);
                        at_least &= at_least - 1;
                    }
                }
            }
            if (DLK_COLD(listed > kScoreWaveList)) {
                /* more than the list takes: of this batch only the wave's n largest (there is room for
                 * them, below), found bit by bit: the n-th largest value, then the last place of it */
                auto count = [&](auto holds) {
                    int c = 0;
#pragma unroll
                    for (int j = 0; j < GR; j++)
#pragma unroll
                        for (int q = 0; q < G; q++) {
                            float v = x[j][q];
                            asm volatile("" : "+v"(v));      /* (made anew each time: kept, the keys are registers) */
                            c += (int)__popcll(ballot(v > -INFINITY && holds(~desc_key(v), place(0, j) + q)));
                        }
                    return c;
                };
                uint32_t value = 0;
#pragma unroll 1
                for (uint32_t bit = 1u << 31; bit; bit >>= 1)
                    if (count([&](uint32_t k, int) { return k >= (value | bit); }) >= p.n) value |= bit;
                const int need = p.n - count([&](uint32_t k, int) { return k > value; });
                int at = 0;                                  /* the places below it hold fewer than `need` of that value */
#pragma unroll 1
                for (int bit = B >> 1; bit; bit >>= 1)
                    if (count([&](uint32_t k, int i) { return k == value && i < at + bit; }) < need) at += bit;
                uint64_t nth = (uint64_t)value << 32 | (uint32_t)~(b0 + at);
                nth = max(nth, bound);
                listed = had;
#pragma unroll
                for (int j = 0; j < GR; j++)
#pragma unroll
                    for (int c = 0; c < G; c++) {
                        const uint64_t e = entry_of(x[j][c], place(b0, j) + c);
                        put(x[j][c] > -INFINITY && e >= nth, e);                   /* n at most */
                    }
            }
            if (DLK_COLD(listed > kScoreWaveList - DLK_MAX_ALTERNATIVES) && b0 + B < s1) {
                /* the list's n largest, in order, and the last of them as the bound from here on */
                uint64_t e[kScoreWaveList / 64];
                int rank[kScoreWaveList / 64];
                wave_order();
#pragma unroll
                for (int k = 0; k < kScoreWaveList / 64; k++) {
                    const int i = lane + 64 * k;
                    int equal;
                    e[k] = list[min(i, listed - 1)];
                    rank[k] = i < listed ? rank_in(list, listed, e[k], equal) : p.n;
                }
                wave_order();
#pragma unroll
                for (int k = 0; k < kScoreWaveList / 64; k++)
                    if (rank[k] < p.n) list[rank[k]] = e[k];
                wave_order();
                listed = p.n;
                bound = max(bound, list[p.n - 1]);
                least = entry_logit(bound);
            }
        }
        /* (-inf counts as 2^-126 of the maximum's term: nothing) */
        const float to = fmaxf(fmaxf(most, best), -3.40282347e38f);
        float s[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < GR; j++)
#pragma unroll
            for (int c = 0; c < G; c++) {
                const float d = fmaxf((x[j][c] - to) * p.scale, -126.0f), e = __builtin_amdgcn_exp2f(d);
                s[c & 3] += e;
                u[c & 3] = fmaf(e, d, u[c & 3]);
            }
        lower(most, to, p.scale, sum, dot);
        sum += (double)((s[0] + s[1]) + (s[2] + s[3]));
        dot += (double)((u[0] + u[1]) + (u[2] + u[3]));
        most = fmaxf(most, best);
    }
    const float wtop = wave_max_dpp(most);
    if (lane == 0) sh.top[wave] = wtop;
    bad = ballot(bad) != 0;
    if (lane == 0) {
        sh.bad[wave] = bad;
        sh.listed[wave] = listed;
    }
    __syncthreads();
    float top = sh.top[0];
    bad = sh.bad[0] != 0;
#pragma unroll
    for (int w = 1; w < T / 64; w++) {
        top = fmaxf(top, sh.top[w]);
        bad |= sh.bad[w] != 0;
    }
    lower(most, fmaxf(top, -3.40282347e38f), p.scale, sum, dot);
    sum = wave_incl_scan_d(sum);
    dot = wave_incl_scan_d(dot);
    if (lane == 63) { sh.sum[wave] = sum; sh.dot[wave] = dot; }
    int all = 0;
    if (TOP) {
        /* the waves' lists in one */
        int first = 0;
#pragma unroll
        for (int w = 0; w < T / 64; w++) {
            const int c = sh.listed[w];
            first += w < wave ? c : 0;
            all += c;
        }
        wave_order();
        for (int a = lane; a < listed; a += 64) sh.joint[first + a] = list[a];
    }
    __syncthreads();
    sum = (sh.sum[0] + sh.sum[1]) + (sh.sum[2] + sh.sum[3]);
    dot = (sh.dot[0] + sh.dot[1]) + (sh.dot[2] + sh.dot[3]);
    static_assert(T / 64 == 4, "waves");
    if (p.slices == 1) {
        finish_row<TOP>(p, sh, row, top, sum, dot, bad, token, logit, sh.joint, all);
        return;
    }
    if (TOP) {
        uint64_t *out = p.cands + ((int64_t)rl * p.slices + slice) * p.n;
        for (int a = t; a < all; a += T) {
            const uint64_t e = sh.joint[a];
            int equal;
            const int rank = rank_in(sh.joint, all, e, equal);
            if (rank < p.n) bpub64(&out[rank], e);
        }
    }
    LogprobSlot *slot = p.slots + (int64_t)rl * p.slices + slice;
    if (t == 0) {
        bpub64(&slot->sum, d2u(sum));
        bpub64(&slot->dot, d2u(dot));
        bpub64(&slot->max_kept, (uint64_t)f2u(top) << 32 | (bad ? 0xffffffffu : (uint32_t)min(all, p.n)));
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t == 0) {
        const uint32_t old = __hip_atomic_fetch_add(&p.counters[rl], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.last = old == (uint32_t)(p.slices - 1);
    }
    __syncthreads();
    if (!sh.last) return;
    if (t == 0) __hip_atomic_store(&p.counters[rl], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    join_row<TOP>(p, sh, rl, token, logit);
}

template <int DT>
int launch_logprobs(const LogprobParams &p, int rows, hipStream_t stream) {
    const unsigned blocks = (unsigned)((int64_t)rows * p.slices);
    if (p.n > 0)
        hipLaunchKernelGGL((token_logprobs_kernel<DT, true>), dim3(blocks), dim3(kLogprobThreads), 0, stream, p);
    else
        hipLaunchKernelGGL((token_logprobs_kernel<DT, false>), dim3(blocks), dim3(kLogprobThreads), 0, stream, p);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

}  // namespace dlk

extern "C" int dlk_launch_token_logprobs(const dlk::LogprobParams *p, int dtype, int rows, hipStream_t stream) {
    if (dtype == DLK_F32) return dlk::launch_logprobs<DLK_F32>(*p, rows, stream);
    if (dtype == DLK_BF16) return dlk::launch_logprobs<DLK_BF16>(*p, rows, stream);
    return dlk::launch_logprobs<DLK_F16>(*p, rows, stream);
}
