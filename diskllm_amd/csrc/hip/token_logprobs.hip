/*
 * token_logprobs.hip -- log-probabilities of given tokens, the entropy and the largest
 * alternatives of each row of logits (dlk_token_logprobs).
 *
 *   t_v = (l_v - max) * log2(e) / T,  z = sum 2^t_v,  u = sum 2^t_v * t_v  (over the allowed ids)
 *   log p_v = (l_v - max) / T - log z,  entropy = log z - ln2 * u / z   (both terms >= 0: nothing cancels)
 *
 * One workgroup reads a slice of a row (logprob_slices() to a row) once, a batch of four
 * 16-byte groups a thread at a time, the next one's loads on their way.  Each thread keeps its
 * own maximum and its sums below it: 16 or 32 terms of a batch are added in 32 bits, batches in
 * 64.  The alternatives are found from the threads' maxima of each batch (see the kernel).  The
 * row's last workgroup to finish (relaxed agent-scope atomics, as the beam selection's) joins
 * sums and lists; no order of arrival shows.
 *
 * Bounds.  Large calls: reads (2,048 x 151,936 bfloat16 with 5 alternatives 123 us, 5.1 TB/s, without 119; a large
 * copy: 4.9).  Few rows: a chain of some 10 us from a slice's first load to its row's outputs (1 x 32,000 with 20
 * alternatives 10.7, without 5.2; 64 x 151,937 masked 19.6): the bound's steps, the list, its publishing, the
 * join's round trip and bound, each a microsecond or two of few instructions that wait for one another.  1,024
 * threads to a row and no join were slower (14.3 and 52).
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
    static constexpr int W = kLogprobThreads / 64;
    union {
        uint64_t list[W][kScoreWaveList];          /* each wave's entries */
        uint64_t ranked[kScoreJoin];               /* those that a join ranks */
    };
    double sum[W], dot[W];
    float top[W];
    uint32_t wave_key[W];
    int listed[W], bad[W];
    int last, count;
};

/* A key that at least r of the lanes' keys reach, of its 16 leading bits, and close to the largest such one (0:
 * fewer than r lanes have one).  Two bits a step, from where the lanes' keys differ: the steps wait for one
 * another (20 single ones 2,000 cycles, these some 500). */
DLK_DEV uint32_t wave_reach(uint32_t key, int r) {
    const uint32_t most = wave_minmax_u32<false>(key);
    if (r == 1) return most;
    const uint32_t differ = most ^ wave_minmax_u32<true>(key);
    int bit = differ ? (31 - __builtin_clz(differ)) & ~1 : 0;            /* of the step's two the lower */
    uint32_t K = bit < 30 ? most >> (bit + 2) << (bit + 2) : 0;          /* (every lane reaches it) */
#pragma unroll 1
    for (bit = max(bit, 14); bit >= 16; bit -= 2) {
        const int c1 = (int)__popcll(ballot(key >= (K | 1u << bit))), c2 = (int)__popcll(ballot(key >= (K | 2u << bit))),
                  c3 = (int)__popcll(ballot(key >= (K | 3u << bit)));
        K |= (c3 >= r ? 3u : c2 >= r ? 2u : c1 >= r ? 1u : 0u) << bit;
    }
    return (int)__popcll(ballot(key != 0)) >= r ? K : 0;
}

/* A bound that n of the threads' keys reach: n / W of each wave's do, or, where a wave has too
 * few, n of one wave's.  0: none. */
DLK_DEV uint32_t score_bound(ScoreShared &sh, uint32_t key, int n) {
    constexpr int W = ScoreShared::W;
    uint32_t bound = 0;
#pragma unroll 1
    for (int one = 0; one < 2 && bound == 0; one++) {
        const uint32_t kw = wave_reach(key, one ? n : (n + W - 1) / W);
        if (one) __syncthreads();
        if (lane_id() == 0) sh.wave_key[wave_id()] = kw;
        __syncthreads();
        bound = sh.wave_key[0];
#pragma unroll
        for (int w = 1; w < W; w++) bound = one ? max(bound, sh.wave_key[w]) : min(bound, sh.wave_key[w]);
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

/* How many of list[0 .. n) are above v. */
DLK_DEV int above_in(const uint64_t *list, int n, uint64_t v) {
    int above = 0, c = 0;
#pragma unroll 1
    for (; c + 16 <= n; c += 16) {
        ulonglong2 a[8];
#pragma unroll
        for (int q = 0; q < 8; q++) a[q] = *(const ulonglong2 *)&list[c + 2 * q];
#pragma unroll
        for (int q = 0; q < 8; q++) above += (a[q].x > v ? 1 : 0) + (a[q].y > v ? 1 : 0);
    }
#pragma unroll 4
    for (; c < n; c++) above += list[c] > v ? 1 : 0;
    return above;
}

/* The row's outputs: its maximum, sums and n largest entries (ranked among list[0 .. all)) are known. */
template <bool TOP>
DLK_DEV void finish_row(const LogprobParams &p, int64_t row, float top, double z, double u, bool bad,
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
            const int rank = above_in(list, all, e);
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
    const uint64_t *cands = p.cands + (int64_t)rl * p.slices * p.cap;
    const int E = p.slices * p.cap;
    uint64_t ent[PRE];
    /* entry i goes to thread (i % 4) * 64 + i / 4 % 64, so that the waves share few of them evenly */
    const int at0 = (t & 63) * 4 + (t >> 6);
    static_assert(T == 256, "waves");
    /* every wave joins the sums for itself; the entries are asked for at the same time */
    const bool mine = lane < p.slices;
    const LogprobSlot *slot = slots + min(lane, p.slices - 1);
    double z = u2d(bget64(&slot->sum)), u = u2d(bget64(&slot->dot));
    const uint64_t mk = bget64(&slot->max_kept);
    if (TOP) {
#pragma unroll
        for (int q = 0; q < PRE; q++)
            if (q * T < E) ent[q] = bget64(&cands[min(q * T + at0, E - 1)]);
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
        /* entry i of list s lies at s * cap + i; those that a list does not have are 0 */
        uint64_t best = 0;
        const float per_cap = 1.0f / (float)p.cap;
#pragma unroll
        for (int q = 0; q < PRE; q++) {
            if (q * T >= E) { ent[q] = 0; continue; }
            const int at = q * T + at0, s = (int)(((float)min(at, E - 1) + 0.5f) * per_cap);         /* exact: below 2^15 */
            const int kept = (int)(uint32_t)shfl((int)(uint32_t)mk, s);
            if (at >= E || at - s * p.cap >= kept) ent[q] = 0;
            best = max(best, ent[q]);
        }
        uint32_t bound = 0;
        /* few entries are all ranked, without a bound first (us without / with: 64 x 151,937 of 5 alternatives, 102
         * entries, 17.5 / 18.1; 1 x 32,000 of 20, 256, 11.3 / 10.3; 8 x 151,936 of 5, 425, 17.5 / 11.8) */
        if (E > 96) bound = score_bound(sh, (uint32_t)(best >> 32), p.n);
        else __syncthreads();
        auto gather = [&](uint64_t least) {
#pragma unroll
            for (int q = 0; q < PRE; q++)
                if (ent[q] != 0 && ent[q] >= least) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < kScoreJoin) sh.ranked[at] = ent[q];
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
    finish_row<TOP>(p, (int64_t)p.r0 + rl, top, z, u, bad, token, logit, sh.ranked, all);
}

/* A slice of a row: its share of the row's p.batches batches (shares differ by one at most).
 * Phase one reads it once: sums, and every thread's maximum of each batch (of `group` batches
 * where a slice has many) to LDS.  Then the bound: n entries reach the n-th largest thread's
 * maximum or so.  Phase two looks for entries only where a thread's maximum says that there are any: about n
 * threads load their groups of a batch again (a slice of one batch has them in registers).  (Entries listed
 * batch by batch under a bound that rises cost 100 us of 240 at 2,048 x 151,936 in bfloat16 with 5
 * alternatives.) */
template <int DT, bool TOP>
__global__ __launch_bounds__(kLogprobThreads, 4) void token_logprobs_kernel(LogprobParams p) {
    typedef LogitRow<DT> In;
    constexpr int T = kLogprobThreads, GR = 4, G = In::G, E = GR * G, B = T * E, W = T / 64;
    __shared__ ScoreShared sh;
    extern __shared__ __align__(16) unsigned char score_rest[];
    uint16_t *const best_of = (uint16_t *)score_rest + threadIdx.x;      /* leading halves of this thread's maxima's keys, T apart */
    uint64_t *const joint = (uint64_t *)score_rest;                      /* later: the waves' lists side by side */
    const int t = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int slice = blockIdx.x % p.slices, rl = blockIdx.x / p.slices;      /* rl: row of the launch */
    const int64_t row = (int64_t)p.r0 + rl;
    const typename In::T *lg = (const typename In::T *)p.logits + row * p.ld;
    const uint32_t *mw = p.mask ? p.mask + (int64_t)(p.mask_row ? p.mask_row[row] : row) * p.mask_ld : nullptr;
    const int first = (int)((int64_t)slice * p.batches / p.slices);
    const int count = (int)((int64_t)(slice + 1) * p.batches / p.slices) - first;
    const int s0 = first * B, s1 = (int)min((int64_t)p.V, (int64_t)(first + count) * B);
    const int group = (count + kLogprobRecords - 1) / kLogprobRecords;         /* batches of a record */
    /* the thread's group j of the batch at b0 */
    auto place = [&](int b0, int j) { return b0 + (j * T + t) * G; };
    float x[GR][G], best;
    typename In::Raw raw[GR];
    uint32_t bits[GR];
    /* asks for the batch at b0 (whole groups of it) and its mask's words */
    auto ask = [&](int b0) __attribute__((always_inline)) {
        if (b0 + B <= s1) {
#pragma unroll
            for (int j = 0; j < GR; j++) raw[j] = *(const typename In::Raw *)(lg + place(b0, j));
        } else {
#pragma unroll
            for (int j = 0; j < GR; j++)
                if (place(b0, j) + G <= s1) raw[j] = *(const typename In::Raw *)(lg + place(b0, j));
        }
        if (mw) {
#pragma unroll
            for (int j = 0; j < GR; j++) bits[j] = mw[min(place(b0, j), s1 - 1) >> 5];
        }
    };
    /* that batch in x (-inf where not allowed), and its maximum (NaN where one is) */
    auto take = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < GR; j++) In::unpack(raw[j], x[j]);
        if (b0 + B > s1) {
#pragma unroll
            for (int j = 0; j < GR; j++) {
                const int i = place(b0, j);
                if (i + G > s1) {
#pragma unroll
                    for (int c = 0; c < G; c++) x[j][c] = i + c < s1 ? In::one(lg + i + c) : -INFINITY;
                }
            }
        }
        if (mw) {
#pragma unroll
            for (int j = 0; j < GR; j++) {
                const uint32_t m = bits[j] >> (place(b0, j) & 31);       /* (a group lies in one word) */
#pragma unroll
                for (int c = 0; c < G; c++) x[j][c] = allowed_or_ninf(x[j][c], m, c);
            }
        }
        best = maximum3(x[0][0], x[0][1], x[0][2]);
#pragma unroll
        for (int q = 3; q < E; q += 2) best = maximum3(best, x[q / G][q % G], x[min(q + 1, E - 1) / G][min(q + 1, E - 1) % G]);
    };
    ask(s0);
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
    float best_here = -INFINITY;                   /* of this record */
    int record = 0, in_record = 0;
    for (int b = 0; b < count; b++) {
        take(s0 + b * B);
        if (b + 1 < count) ask(s0 + (b + 1) * B);            /* (on its way while this one is summed) */
        bad |= !(best < INFINITY);
        if (TOP) {
            best_here = fmaxf(in_record == 0 ? -INFINITY : best_here, best);
            best_of[record * T] = (uint16_t)(~desc_key(best_here) >> 16);
            if (++in_record == group) { in_record = 0; record++; }
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
    bad = ballot(bad) != 0;
    if (lane == 0) {
        sh.top[wave] = wtop;
        sh.bad[wave] = bad;
    }
    uint32_t bound_key = 0;
    if (TOP) bound_key = score_bound(sh, most > -INFINITY ? ~desc_key(most) : 0u, p.n);   /* (0: every id is an entry) */
    else __syncthreads();
    float top = sh.top[0];
    bad = sh.bad[0] != 0;
#pragma unroll
    for (int w = 1; w < W; w++) {
        top = fmaxf(top, sh.top[w]);
        bad |= sh.bad[w] != 0;
    }
    lower(most, fmaxf(top, -3.40282347e38f), p.scale, sum, dot);
    sum = wave_incl_scan_d(sum);
    dot = wave_incl_scan_d(dot);
    if (lane == 63) { sh.sum[wave] = sum; sh.dot[wave] = dot; }
    int all = 0;
    if (TOP) {
        uint64_t *list = sh.list[wave];
        int listed = 0;
        uint64_t bound = (uint64_t)bound_key << 32;
        float least = bound_key != 0 ? key_value(~bound_key) : -INFINITY;
        /* each thread's own records that hold entries, in order, so that of equal logits the lower ids are there first:
         * a round of loads for as many threads as have one left, one or two rounds in all.  (0x7f is -inf's, 0x80 the
         * lowest float's: where there is no bound, records without an allowed logit are still none) */
        const uint32_t reaches = max(bound_key >> 16, 0x80u);
        uint64_t records = 0;
#pragma unroll 4
        for (int r = 0; r * group < count; r++) records |= (uint64_t)(best_of[r * T] >= reaches) << r;
        if (bad) records = 0;
        int of_record = 0;
#pragma unroll 1
        while (ballot(records != 0) != 0) {
            const int b = records != 0 ? __builtin_ctzll(records) * group + of_record : count;
            const int b0 = s0 + b * B;
            if (++of_record == group) {
                of_record = 0;
                records &= records - 1;
            }
            if (count > 1) {
                if (b < count) {
                    ask(b0);
                    take(b0);
                }
            }
            if (b >= count) {
#pragma unroll
                for (int j = 0; j < GR; j++)
#pragma unroll
                    for (int c = 0; c < G; c++) x[j][c] = -INFINITY;
            }
            /* (equal to the bound's logit, of ids above the bound's: none of them; where all logits are equal that is all) */
            const bool equal_too = ((bound >> 32 << 32) | (uint32_t)~place(b0, 0)) >= bound;
            const float from_here = equal_too ? least : key_value(~((uint32_t)(bound >> 32) + 1));
            uint32_t at_least = 0;                           /* bit j * G + c */
#pragma unroll
            for (int q = 0; q < E; q++) at_least |= x[q / G][q % G] >= from_here && x[q / G][q % G] > -INFINITY ? 1u << q : 0u;
#pragma unroll 1
            while (ballot(at_least != 0) != 0) {
                const int k = at_least != 0 ? __builtin_ctz(at_least) : 0;
                float v = x[0][0];
#pragma unroll
                for (int q = 1; q < E; q++) v = k == q ? x[q / G][q % G] : v;
                const uint64_t e = entry_of(v, place(b0, k / G) + k % G);
                const bool wanted = at_least != 0 && e >= bound;
                const uint64_t who = ballot(wanted);
                if (wanted) list[place_in(who, listed)] = e;
                listed += (int)__popcll(who);
                at_least &= at_least - 1;
                if (DLK_COLD(listed > kScoreWaveList - 64)) {
                    /* the list's n largest, in order, and the last of them as the bound from here on */
                    uint64_t kept[kScoreWaveList / 64];
                    int rank[kScoreWaveList / 64];
                    wave_order();
#pragma unroll
                    for (int q = 0; q < kScoreWaveList / 64; q++) {
                        const int i = lane + 64 * q;
                        kept[q] = list[min(i, listed - 1)];
                        rank[q] = i < listed ? above_in(list, listed, kept[q]) : p.n;
                    }
                    wave_order();
#pragma unroll
                    for (int q = 0; q < kScoreWaveList / 64; q++)
                        if (rank[q] < p.n) list[rank[q]] = kept[q];
                    wave_order();
                    listed = p.n;
                    bound = max(bound, list[p.n - 1]);
                    least = entry_logit(bound);
                }
            }
        }
        if (lane == 0) sh.listed[wave] = listed;
        __syncthreads();                                     /* (the records are read) */
        /* the waves' lists in one */
        int from = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const int c = sh.listed[w];
            from += w < wave ? c : 0;
            all += c;
        }
        for (int a = lane; a < listed; a += 64) joint[from + a] = list[a];
    }
    __syncthreads();
    sum = 0.0;
    dot = 0.0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        sum += sh.sum[w];
        dot += sh.dot[w];
    }
    if (p.slices == 1) {
        finish_row<TOP>(p, row, top, sum, dot, bad, token, logit, joint, all);
        return;
    }
    if (TOP) {
        /* as they are where there is room for them, else the n largest */
        uint64_t *out = p.cands + ((int64_t)rl * p.slices + slice) * p.cap;
        for (int a = t; a < all; a += T) {
            const uint64_t e = joint[a];
            const int rank = all <= p.cap ? a : above_in(joint, all, e);
            if (rank < (all <= p.cap ? all : p.n)) bpub64(&out[rank], e);
        }
    }
    LogprobSlot *slot = p.slots + (int64_t)rl * p.slices + slice;
    if (t == 0) {
        bpub64(&slot->sum, d2u(sum));
        bpub64(&slot->dot, d2u(dot));
        bpub64(&slot->max_kept, (uint64_t)f2u(top) << 32 | (bad ? 0xffffffffu : (uint32_t)(all <= p.cap ? all : p.n)));
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
    if (p.n > 0) {
        const int most = (p.batches + p.slices - 1) / p.slices, records = most < kLogprobRecords ? most : kLogprobRecords;
        const size_t joint = (size_t)ScoreShared::W * kScoreWaveList * 8, best = (size_t)records * kLogprobThreads * 2;
        hipLaunchKernelGGL((token_logprobs_kernel<DT, true>), dim3(blocks), dim3(kLogprobThreads),
                           best > joint ? best : joint, stream, p);
    } else {
        hipLaunchKernelGGL((token_logprobs_kernel<DT, false>), dim3(blocks), dim3(kLogprobThreads), 0, stream, p);
    }
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

}  // namespace dlk

extern "C" int dlk_launch_token_logprobs(const dlk::LogprobParams *p, int dtype, int rows, hipStream_t stream) {
    if (dtype == DLK_F32) return dlk::launch_logprobs<DLK_F32>(*p, rows, stream);
    if (dtype == DLK_BF16) return dlk::launch_logprobs<DLK_BF16>(*p, rows, stream);
    return dlk::launch_logprobs<DLK_F16>(*p, rows, stream);
}
