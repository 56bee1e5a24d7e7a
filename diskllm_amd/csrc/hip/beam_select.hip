/*
 * beam_select.hip -- one step of a beam search: of the continuations (row, id) of a group
 * of rows the n with the largest score + log softmax(l)[id] (dlk_beam_select).
 *
 * One workgroup reads a slice of a row (beam_slices() to a row) once, 4,096 logits at a time
 * into registers; masks and penalises them; sums exp(l - its maximum so far) in 64 bits;
 * and lists the slice's n largest entries in order.  Log softmax is increasing in l, so a
 * row's n best continuations are its n largest logits and none of the others is needed
 * again.  Its four waves work alone from the first batch's bound (n entries of the
 * workgroup reach it) to the end: each has a list of its own, holds the history ids among its
 * logits, penalised once, and sums its own logits, where a mask leaves few of them (512 of
 * 1,024) packed side by side.
 * The group's last workgroup to finish (relaxed agent-scope atomics, as the top-k kernel's)
 * joins the slices' sums and merges the lists under the keys in 64 bits: one launch, and
 * no order of arrival shows in the result.
 *
 * A log-sum is off by 2^-43 at most: a term's exponential and its rescales, one for each of
 * 16 batches of a slice (where 64 beams leave four slices a row; else five or so) and five
 * as waves, slices and lanes are joined, 3.6e-15 each, and at most 280 additions in a
 * row of 1.1e-16.  Sums and keys are 64-bit because the order of continuations of different rows hangs on
 * differences of their log-sums, which a sum of 262,144 terms in 32 bits blurs by more than
 * neighbouring candidates differ; 64-bit FMAs run at the plain 32-bit ones' rate here.
 *
 * Bounds.  Large calls: reads, with what starts and ends a workgroup (512 x 262,144, 1 of 20
 * allowed: 129 us, 4.3 TB/s; with a list and barriers common to the waves and every logit
 * summed 145).  Calls that fit the chip once: the chain of a slice and the merge (64 x
 * 151,936 with penalties 32 us, of which 20 a slice's at the median, 28 at the last, 5 the
 * merge's; 128 x 50,257 in groups of 16 25.5, 16 and 8).  A history costs 13 us of 504 x
 * 64,960 with 64 ids and 31 with 1,000 of no order (53, 65, 84; with every wave looking through
 * all of it and ids put into place one by one 154); 107 where they are Zipf's and the common ones
 * the lowest, so that they are some few waves' (64 x 151,936: none 27, 256 ids 32 and 37,
 * 1,000 35 and 59), as a wave holds 128 occurrences and looks through the history in
 * every batch past that.  Small ones: a dozen round trips one after another (4 x 32,000: 11.5 us).  The next batch's loads ahead of this one's work
 * changed nothing: other workgroups' waves fill that time.
 */
#include "dlk_device.h"
#include "beam_select.h"
#include "top_list.h"
#include "../../../include/diskllm_amd.h"

namespace dlk {

constexpr int kBeamList = 512;         /* entries that a merge orders at once */
constexpr int kBeamWaveList = 256;     /* and that a wave lists of a slice */
constexpr int kBeamSaid = 128;         /* occurrences of a history's ids that a wave holds */
constexpr int kBeamPacked = 512;       /* of a wave's 1,024 logits: so many allowed ones or fewer are packed */

/* a * b + c with c in scalar registers and its own destination (the compiler's choice adds
 * a move of c for each). */
DLK_DEV double fma3(double a, double b, double c) {
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
    return d;
}

/* exp(x) for x <= 0 to 4e-15 of it (below -700: of exp(-700)): 2^k times the fourth power of a
 * polynomial of e^(r / 4) on |r| <= ln2 / 2, exactly 1 at 0 (sums are rescaled by it many
 * times), with the coefficients that bring its largest error to 2.9e-15 (least squares
 * re-weighted to equal peaks); evaluated in doubles 3.6e-15.  k by the addition that leaves
 * it in the sum's low bits.  Two squarings take the place of two degrees and cost what two
 * do, without their constants (64 x 151,936 with histories: 31.7 us with a polynomial of e^r
 * to 4.7e-11, of which the order of rows showed; 31.9 this; degree 9, 1.5e-14, 32.7; degree 10,
 * 2.2e-16, 32.8.  512 x 262,144: 132, 139, 140, 144). */
DLK_DEV double exp_neg(double x) {
    const double round = 6755399441055744.0;             /* 1.5 * 2^52 */
    x = fmax(x, -700.0);
    const double t = fma(x, 1.4426950408889634, round);
    const double r = fma(t - round, -0.6931471805599453, x);
    double y = 1.2107325684402232e-08;
    y = fma3(y, r, 3.391714957943183e-07);
    y = fma3(y, r, 8.138021736707668e-06);
    y = fma3(y, r, 0.00016276041059136318);
    y = fma3(y, r, 0.0026041666666089458);
    y = fma3(y, r, 0.03125000000012017);
    y = fma3(y, r, 0.2500000000000008);
    y = fma(y, r, 1.0);
    y = y * y;
    y = y * y;
    return __hiloint2double(__double2hiint(y) + (__double2loint(t) << 20), __double2loint(y));
}

/* The larger of three (NaN: of the others): one instruction, where fmaxf makes one for each
 * value to quiet it. */
DLK_DEV float max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

/* Ascending key of a double (no NaN); zero below every one. */
DLK_DEV uint64_t double_key(double d) {
    uint64_t u = d2u(d);
    if (u == 0x8000000000000000ull) u = 0;
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

/* The penalties of an id that occurs cnt times in the row's history, as penalties.hip. */
DLK_DEV float beam_penalised(const BeamParams &p, float x, int cnt) {
    for (int s = 0; s < 8; s++) {
        const uint32_t op = (p.order >> (4 * s)) & 0xFu;
        if (op == 0) break;
        if (op == DLK_OP_REPETITION) {
            if (p.rep > 1.0f)
                for (int k = 0; k < cnt; k++) x = x < 0.0f ? x * p.rep : x / p.rep;
        } else if (op == DLK_OP_FREQUENCY) {
            if (p.freq != 0.0f) { const float d = p.freq * (float)cnt; x = x - d; }
        } else if (op == DLK_OP_PRESENCE) {
            if (p.pres != 0.0f) x = x - p.pres;
        }
    }
    return x;
}

/* A key that at least r of the lanes' keys reach (0: fewer than r lanes have one): the largest
 * for r = 1, else the largest of 20 leading bits (0.5 us where few waves run). */
DLK_DEV uint32_t wave_rth(uint32_t a, int r) {
    uint32_t K = 0;
    if (r == 1) return wave_minmax_u32<false>(a);
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1)
        if ((int)__popcll(ballot(a >= (K | bit))) >= r) K |= bit;
    return K;
}

/* Maximum over each row of 16 lanes (every lane gets its row's). */
DLK_DEV float row_max(float v) {
    v = fmaxf(v, shfl_xor(v, 1));
    v = fmaxf(v, shfl_xor(v, 2));
    v = fmaxf(v, shfl_xor(v, 4));
    return fmaxf(v, shfl_xor(v, 8));
}

struct BeamShared {
    union {
        __align__(16) uint64_t list[kBeamThreads / 64][kBeamWaveList];      /* slice: each wave's entries */
        struct {
            uint64_t key[kBeamList];            /* merge: keys and entries */
            uint64_t ent[kBeamList];
        };
    };
    double base[DLK_MAX_BEAMS];         /* per row of the group: log-sum, norm, score, maximum */
    double norm[DLK_MAX_BEAMS];
    double part[kBeamThreads / 64];
    float cum[DLK_MAX_BEAMS];
    float top[DLK_MAX_BEAMS];
    float above;                        /* no key of the group is above it */
    uint32_t wave_key[kBeamThreads / 64];
    int wave_n[kBeamThreads / 64], wave_listed[kBeamThreads / 64];
    int place[kBeamList];               /* row of each entry */
    int kind[DLK_MAX_BEAMS];            /* 0: none, 1: by its lists, 2: finished */
    uint8_t kept[kBeamThreads];         /* entries of each list */
    int count, last;
    uint64_t best_key[kBeamThreads / 64], best_ent[kBeamThreads / 64];
    int best_row[kBeamThreads / 64];
};

/* A bound that n of the threads' keys reach: n / 4 of each wave's do, or, where a wave has too
 * few (the end of a vocabulary, lists of one or two entries), n of one wave's.  0: none. */
DLK_DEV uint32_t bound_of(BeamShared &sh, uint32_t key, int n) {
    uint32_t bound = 0;
#pragma unroll 1
    for (int one = 0; one < 2 && bound == 0; one++) {
        const uint32_t kw = wave_rth(key, one ? n : (n + 3) / 4);
        if (one) __syncthreads();
        if (lane_id() == 0) sh.wave_key[wave_id()] = kw;
        __syncthreads();
        bound = sh.wave_key[0];
#pragma unroll
        for (int w = 1; w < kBeamThreads / 64; w++) bound = one ? max(bound, sh.wave_key[w]) : min(bound, sh.wave_key[w]);
    }
    return __builtin_amdgcn_readfirstlane(bound);
}

/* a before b: larger key, lower row, larger entry. */
DLK_DEV bool before(uint64_t ka, int ra, uint64_t ea, uint64_t kb, int rb, uint64_t eb) {
    if (ka != kb) return ka > kb;
    if (ra != rb) return ra < rb;
    return ea > eb;
}

/* How many of list[0 .. n) are above v, and how many equal to it. */
DLK_DEV int rank_in(const uint64_t *list, int n, uint64_t v, int &equal) {
    int above = 0;
    equal = 0;
    int c = 0;
    for (; c + 4 <= n; c += 4) {
        const ulonglong2 a = *(const ulonglong2 *)&list[c], b = *(const ulonglong2 *)&list[c + 2];
        above += (a.x > v ? 1 : 0) + (a.y > v ? 1 : 0) + (b.x > v ? 1 : 0) + (b.y > v ? 1 : 0);
        equal += (a.x == v ? 1 : 0) + (a.y == v ? 1 : 0) + (b.x == v ? 1 : 0) + (b.y == v ? 1 : 0);
    }
    for (; c < n; c++) {
        const uint64_t a = list[c];
        above += a > v ? 1 : 0;
        equal += a == v ? 1 : 0;
    }
    return above;
}

/* What a row adds to its continuations, out of LDS once for many of them. */
struct BeamRow {
    double base, norm, top, cum;
    bool over;
    DLK_DEV BeamRow(const BeamShared &sh, int b)
        : base(sh.base[b]), norm(sh.norm[b]), top((double)sh.top[b]), cum((double)sh.cum[b]), over(sh.kind[b] == 2) {}
    /* the score of entry e in 64 bits, and its key */
    DLK_DEV double score(uint64_t e) const { return over ? cum : cum + (((double)entry_logit(e) - top) - base); }
    DLK_DEV uint64_t key(uint64_t e) const { return double_key(score(e) * norm); }
    /* that as a word, by its distance from a float that no key of the group is above (to 2^-11 of it, whatever the scores'
     * size is); never 0 */
    DLK_DEV uint32_t word(uint64_t e, double above) const { return ~f2u((float)(above - score(e) * norm)); }
};

DLK_DEV void write_continuation(const BeamParams &p, const BeamShared &sh, int g, int j, int b, uint64_t e) {
    const int64_t o = (int64_t)g * p.n + j, row = (int64_t)g * p.beams + b;
    const bool over = sh.kind[b] == 2;
    const int id = over ? p.eos : entry_id(e);
    const int len = p.lengths ? p.lengths[row] : 0;
    p.out_tokens[o] = id;
    p.out_parents[o] = (int32_t)row;
    p.out_scores[o] = (float)BeamRow(sh, b).score(e);
    if (p.out_lengths) p.out_lengths[o] = len + (over ? 0 : 1);
    if (p.out_finished) p.out_finished[o] = over || id == p.eos ? 1 : 0;
}

DLK_DEV void write_none(const BeamParams &p, int g, int j) {
    const int64_t o = (int64_t)g * p.n + j;
    p.out_tokens[o] = -1;
    p.out_parents[o] = -1;
    p.out_scores[o] = -INFINITY;
    if (p.out_lengths) p.out_lengths[o] = 0;
    if (p.out_finished) p.out_finished[o] = 0;
}

/* The group's lists (256 at most, one per thread) merged, by its last workgroup.  The slots are
 * asked for at once, and 16 entries per thread (4,096) with them: a round trip to the other
 * workgroups' words is most of what a merge takes. */
DLK_DEV void merge_group(const BeamParams &p, int gl, BeamShared &sh) {
    constexpr int T = kBeamThreads, PRE = kBeamEntries / T;
    const int t = threadIdx.x, lane = lane_id(), wave = wave_id(), g = p.g0 + gl;
    const int L = p.beams * p.slices, E = L * p.n;
    const BeamSlot *slots = p.slots + (int64_t)gl * L;
    const uint64_t *cands = p.cands + (int64_t)gl * L * p.n;
    /* list i is that of (row i / slices, slice i % slices).  List or entry i goes to thread
     * (i % 4) * 64 + i / 4 % 64, so that the waves share few of them evenly */
    const int mine = (t & 63) * 4 + (t >> 6);
    uint64_t pre[PRE];
    /* which of the T entries from e on: dealt anew for each T, or a thread would hold the same places
     * of many lists (n a power of two), the best of the threads be those of a few places, and
     * more reach their bound than are ranked at once (16 x 2 x 151,936 of 64, beams near one another:
     * 36 us, 102 that way; 16 x 4 52, 142) */
    auto place_of = [&](int m, int e0, int q) { return e0 + q * T + (m ^ (q * 37 & (T - 1))); };
    auto this_thread = [&]() {
        int m = mine;
        asm volatile("" : "+v"(m));                          /* (places kept from loop to loop are 16 registers) */
        return m;
    };
    auto load = [&](int e0) {
        const int m = this_thread();
#pragma unroll
        for (int q = 0; q < PRE; q++)
            if (e0 + q * T < E) pre[q] = bget64(&cands[min(place_of(m, e0, q), E - 1)]);
    };
    if (t < L) {
        const uint64_t mk = bget64(&slots[t].max_kept);
        sh.key[t] = bget64(&slots[t].sum);
        sh.ent[t] = mk;
        sh.kept[t] = (uint8_t)mk;
    }
    load(0);
    if (t == 0) sh.count = 0;
    __syncthreads();
    /* the rows' sums: 16 lanes each where they have 16 slices at most, else a wave each */
    const int width = p.slices <= 16 ? 16 : 64, sub = t & (width - 1);
    for (int b0 = 0; b0 < p.beams; b0 += T / width) {
        const int b = b0 + t / width;
        float top = -INFINITY;
        double sum = 0.0;
        bool bad = false;
        for (int s = sub; b < p.beams && s < p.slices; s += width) {
            const int i = b * p.slices + s;
            const uint64_t sm = sh.key[i], mk = sh.ent[i];
            const float m = u2f((uint32_t)(mk >> 32));
            bad |= (uint32_t)mk == 0xffffffffu;
            if (m > -INFINITY) {
                const float to = fmaxf(top, m);
                sum = (top > -INFINITY ? sum * exp_neg((double)top - (double)to) : 0.0) +
                      u2d(sm) * exp_neg((double)m - (double)to);
                top = to;
            }
        }
        float all = row_max(top);
        if (width == 64) all = wave_max_dpp(all);
        sum = top > -INFINITY ? sum * exp_neg((double)top - (double)all) : 0.0;
        sum = width == 64 ? wave_incl_scan_d(sum) : row_scan_d(sum);
        const uint64_t bads = width == 64 ? ballot(bad) : ballot(bad) >> (lane & 48) & 0xffff;
        if (sub == width - 1 && b < p.beams) {
            sh.top[b] = all;
            sh.base[b] = sum;
            sh.kind[b] = bads ? -1 : all > -INFINITY ? 1 : 0;
        }
    }
    __syncthreads();
    /* what each row adds to its continuations, a lane each; and the float after the group's best key (a row's best entry
     * is its maximum) */
    float most = -INFINITY;
    if (t < p.beams) {
        const int64_t row = (int64_t)g * p.beams + t;
        const float cum = p.scores ? p.scores[row] : 0.0f;
        const bool over = p.finished && p.finished[row];
        const int kind = sh.kind[t];
        const bool alive = cum > -INFINITY && cum < INFINITY;
        const double length = fmax((double)(p.lengths ? p.lengths[row] : 0) + (over ? 0.0 : 1.0), 1.0);
        const double base = kind == 1 ? log(sh.base[t]) : 0.0;
        const double norm = p.alpha == 0.0f ? 1.0 : 1.0 / pow(length, (double)p.alpha);
        const int by = !alive ? 0 : over ? 2 : kind == 1 ? 1 : 0;
        sh.cum[t] = cum;
        sh.base[t] = base;
        sh.norm[t] = norm;
        sh.kind[t] = by;
        if (by != 0) most = (float)(((double)cum - base) * norm);
        if (p.status && (!(cum < INFINITY) || (alive && !over && kind < 0))) atomicOr(p.status, DLK_STATUS_NOT_FINITE);
    }
    if (wave == 0) {
        most = wave_max_dpp(most);
        const uint32_t u = f2u(most);
        if (t == 0) sh.above = u2f(most > 0.0f ? (most < INFINITY ? u + 1 : u) : most < 0.0f ? u - 1 : 1u);
    }
    __syncthreads();
    const double above = (double)sh.above;
    /* list i of row b: its entries (a finished row's first list holds its one continuation) */
    auto listed = [&](int i, int b) {
        const int kind = sh.kind[b];
        return kind == 1 ? (int)sh.kept[i] : kind == 2 && i == b * p.slices ? 1 : 0;
    };
    auto add = [&](uint64_t k, uint64_t e, int b) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kBeamList) {
            sh.key[at] = k;
            sh.ent[at] = e;
            sh.place[at] = b;
        }
    };
    /* every entry's word for the bound, then those that reach it: PRE * T at a time, which are
     * kept from one to the other where they are all.  The bound has a word's 20 leading bits: of the
     * distance from the best, so that it is as close where scores are large (16 x 16 x 128,256
     * of 32: 71 us at scores of -20, 72 at -2,500; bits of the scores themselves were 8 apart there,
     * more reached it than are ranked at once, and it took 125). */
    uint32_t word[PRE], best = 0, bound = 0;                 /* 0: none */
    const float per_n = 1.0f / (float)p.n, per_slices = 1.0f / (float)p.slices;
    auto list_of = [&](int at) { return (int)(((float)at + 0.5f) * per_n); };              /* exact: below 2^15 */
    auto row_of = [&](int i) { return (int)(((float)i + 0.5f) * per_slices); };
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
#pragma unroll 1
        for (int e0 = 0; e0 < E; e0 += PRE * T) {
            if (pass == 0 || E > PRE * T) {
                if (pass > 0 || e0 > 0) load(e0);
                const int m = this_thread();
#pragma unroll
                for (int q = 0; q < PRE; q++) {              /* (few entries: few instructions, fetched for the first time) */
                    word[q] = 0;
                    if (e0 + q * T >= E) continue;
                    const int place = place_of(m, e0, q), at = min(place, E - 1), i = list_of(at), b = row_of(i);
                    if (sh.kind[b] == 2) pre[q] = ~(uint64_t)0;
                    if (place < E && at - i * p.n < listed(i, b)) word[q] = BeamRow(sh, b).word(pre[q], above);
                    best = max(best, word[q]);
                }
            }
            if (pass == 0) continue;
            const int m = this_thread();
#pragma unroll
            for (int q = 0; q < PRE; q++) {
                if (word[q] == 0 || word[q] < bound) continue;
                const int b = row_of(list_of(place_of(m, e0, q)));
                add(BeamRow(sh, b).key(pre[q]), pre[q], b);
            }
        }
        if (pass == 0) bound = bound_of(sh, best, p.n);
    }
    __syncthreads();
    const int C = sh.count;
    if (DLK_HOT(C <= kBeamList)) {
        for (int a = t; a < C; a += T) {
            const uint64_t k = sh.key[a], e = sh.ent[a];
            const int b = sh.place[a];
            int equal, rank = rank_in(sh.key, C, k, equal);
            if (equal > 1)
                for (int c = 0; c < C; c++)
                    rank += sh.key[c] == k && before(k, sh.place[c], sh.ent[c], k, b, e) ? 1 : 0;
            if (rank < p.n) write_continuation(p, sh, g, rank, b, e);
        }
        for (int j = C + t; j < p.n; j += T) write_none(p, g, j);
    } else {
        /* too many at or above the bound (few lists for n, or runs of equal keys): the best of the
         * lists' next entries, n times */
        const int i = min(mine, L - 1), b = i / p.slices, n = mine < L ? listed(i, b) : 0;
        const BeamRow row(sh, b);
        auto entry = [&](int q) -> uint64_t {
            return sh.kind[b] == 2 ? ~(uint64_t)0 : bget64(&cands[(int64_t)i * p.n + q]);
        };
        int q = 0;
        uint64_t be = n > 0 ? entry(0) : 0, bk = row.key(be);
        for (int j = 0; j < p.n; j++) {
            uint64_t k = bk, e = be;
            int r = q < n ? b : -1;
            for (int m = 1; m < 64; m <<= 1) {
                const uint64_t ok = shfl_xor(k, m), oe = shfl_xor(e, m);
                const int oi = shfl_xor(r, m);
                if (oi >= 0 && (r < 0 || before(ok, oi, oe, k, r, e))) { k = ok; e = oe; r = oi; }
            }
            if (lane == 0) { sh.best_key[wave] = k; sh.best_ent[wave] = e; sh.best_row[wave] = r; }
            __syncthreads();
            r = -1;
            for (int w = 0; w < T / 64; w++) {
                const int oi = sh.best_row[w];
                if (oi >= 0 && (r < 0 || before(sh.best_key[w], oi, sh.best_ent[w], k, r, e))) {
                    k = sh.best_key[w]; e = sh.best_ent[w]; r = oi;
                }
            }
            __syncthreads();
            if (t == 0) {
                if (r >= 0) write_continuation(p, sh, g, j, r, e);
                else write_none(p, g, j);
            }
            if (q < n && b == r && be == e) {                /* (an id of a row is in one list) */
                q++;
                be = q < n ? entry(q) : 0;
                bk = row.key(be);
            }
        }
    }
}

/* A slice of a row: its share of the row's p.batches batches of four groups of four logits per
 * thread (shares differ by one batch at most). */
template <bool HIST>
__global__ __launch_bounds__(kBeamThreads, 5) void beam_select_kernel(BeamParams p) {
    constexpr int T = kBeamThreads, GR = 4, B = kBeamBatch;
    __shared__ BeamShared sh;
    __shared__ __align__(16) float packed[T / 64][kBeamPacked];
    static_assert(sizeof(packed) >= sizeof(sh.list), "room for the lists side by side");
    __shared__ __align__(16) uint32_t times[HIST ? B / 2 : 4];               /* occurrences, 16 bits an id */
    const int t = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int slice = blockIdx.x % p.slices, rl = blockIdx.x / p.slices;      /* rl: row of the launch */
    const int64_t row = (int64_t)p.g0 * p.beams + rl;
    const float *lg = p.logits + row * p.ld;
    const uint32_t *mw = p.mask ? p.mask + (int64_t)(p.mask_row ? p.mask_row[row] : row) * p.mask_ld : nullptr;
    const int s0 = slice * p.batches / p.slices * B;
    const int s1 = (int)min((int64_t)p.V, (int64_t)((slice + 1) * p.batches / p.slices) * B);
    float x[GR][4];
    auto load = [&](int b0) {
        int t4 = t * 4;
        asm volatile("" : "+v"(t4));                         /* (places kept from batch to batch are 50 registers) */
        if (b0 + B <= s1) {
#pragma unroll
            for (int j = 0; j < GR; j++) {
                const float4 v = load4(lg + b0 + j * T * 4 + t4);
                x[j][0] = v.x; x[j][1] = v.y; x[j][2] = v.z; x[j][3] = v.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < GR; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int i = b0 + j * T * 4 + t4 + c;
                    const float v = lg[min(i, s1 - 1)];
                    x[j][c] = i < s1 ? v : -INFINITY;
                }
        }
    };
    load(s0);                                                /* (asked for before it is known whether the row is used) */
    const float cum = p.scores ? p.scores[row] : 0.0f;
    int hn = 0;
    const int32_t *hist = nullptr;
    if (HIST) {
        const int h0 = p.hist_off[row];
        hn = p.hist_off[row + 1] - h0;
        hist = p.hist_ids + h0;
    }
    /* a row without continuations, or a finished one: what its logits hold does not matter */
    bool idle = !(cum > -INFINITY && cum < INFINITY) || (p.finished && p.finished[row]);
    const bool too_long = HIST && !idle && hn > p.max_hist;
    idle |= too_long;
    if (too_long && t == 0 && slice == 0 && p.status) atomicOr(p.status, DLK_STATUS_HISTORY_TOO_LONG);
    float top = -INFINITY;
    double sum = 0.0;
    uint32_t kept = 0;
    if (!idle) {
        uint64_t *list = sh.list[wave];
        int listed = 0;
        /* The history's ids among this wave's logits, two a lane (each as often as it occurs), penalised once
         * and put into their places batch by batch; more than 128 are counted in LDS in each batch. */
        auto wave_of = [&](int32_t id) { return ((id - s0) >> 8) & 3; };
        int said = 0;
        int32_t mine[2] = {-1, -1};
        float becomes[2] = {0.0f, 0.0f};           /* those ids' logits with their penalties */
        if (HIST && hn > 0) {
            for (int i = t; i < B / 8; i += T) ((uint4 *)times)[i] = make_uint4(0, 0, 0, 0);
            if (t < T / 64) sh.wave_n[t] = 0;
            __syncthreads();
#pragma unroll 1
            for (int i0 = 0; i0 < hn; i0 += 4 * T) {
                int32_t id[4];
#pragma unroll
                for (int k = 0; k < 4; k++) id[k] = hist[min(i0 + k * T + t, hn - 1)];
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (i0 + k * T + t < hn && id[k] >= s0 && id[k] < s1) {
                        const int w = wave_of(id[k]), at = atomicAdd(&sh.wave_n[w], 1);
                        if (at < kBeamSaid) ((int32_t *)packed[w])[at] = id[k];
                    }
            }
            __syncthreads();
            said = __builtin_amdgcn_readfirstlane(sh.wave_n[wave]);
            if (said <= kBeamSaid) {
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (lane + 64 * h < said) {
                        mine[h] = ((int32_t *)packed[wave])[lane + 64 * h];
                        becomes[h] = lg[mine[h]];
                    }
                wave_order();
                int times_of[2] = {0, 0};
#pragma unroll 1
                for (int k = 0; k < said; k++) {
                    const int32_t id = __builtin_amdgcn_readlane(k < 64 ? mine[0] : mine[1], k & 63);
                    times_of[0] += id == mine[0] ? 1 : 0;
                    times_of[1] += id == mine[1] ? 1 : 0;
                }
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (mine[h] >= 0) becomes[h] = beam_penalised(p, becomes[h], times_of[h]);
            }
        }
        float most = -INFINITY;                    /* this thread's maximum, and its sum of exp(l - that) */
        double part = 0.0;
        bool bad = false;
        float least = -INFINITY;                   /* bound: n entries of the slice reach it (as a logit, and exactly) */
        uint64_t bound = 0;
        /* lists the lanes' entries side by side (past the list's end they are counted) */
        auto put = [&](bool take, uint64_t e) {
            const uint64_t who = ballot(take);
            const int at = place_in(who, listed);
            if (take && at < kBeamWaveList) list[at] = e;
            listed += (int)__popcll(who);
        };
        for (int b0 = s0; b0 < s1; b0 += B) {
            int t4 = t * 4;
            asm volatile("" : "+v"(t4));
            if (b0 != s0) load(b0);
            if (mw) {
                uint32_t bits[GR];
#pragma unroll
                for (int j = 0; j < GR; j++) bits[j] = mw[min(b0 + j * T * 4 + t4, s1 - 1) >> 5];
#pragma unroll
                for (int j = 0; j < GR; j++) {
                    bits[j] >>= (b0 + j * T * 4 + t4) & 31;
#pragma unroll
                    for (int c = 0; c < 4; c++) x[j][c] = allowed_or_ninf(x[j][c], bits[j], c);
                }
            }
            auto in_batch = [&](int32_t id) { return id >= b0 && id < s1 && id - b0 < B; };
            if (HIST && said > 0 && said <= kBeamSaid) {
                const bool now0 = in_batch(mine[0]), now1 = in_batch(mine[1]);
                if (ballot(now0 || now1) != 0) {
                    /* each id's holder + 1 at its place, where the logit's lane finds whose value it takes */
                    uint16_t *whose = (uint16_t *)times;
                    if (now0) whose[mine[0] - b0] = (uint16_t)(lane + 1);
                    if (now1) whose[mine[1] - b0] = (uint16_t)(lane + 65);
                    wave_order();
#pragma unroll
                    for (int j = 0; j < GR; j++) {
                        const uint2 w = ((const uint2 *)times)[j * T + t];
                        if (ballot((w.x | w.y) != 0) == 0) continue;
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const int from = (int)(((c < 2 ? w.x : w.y) >> (16 * (c & 1))) & 0xffff);
                            float y = shfl(becomes[0], (from - 1) & 63);
                            if (said > 64) {
                                const float y1 = shfl(becomes[1], (from - 1) & 63);
                                y = from > 64 ? y1 : y;
                            }
                            x[j][c] = from != 0 && x[j][c] != -INFINITY ? y : x[j][c];
                        }
                    }
                    wave_order();
                    if (now0) whose[mine[0] - b0] = 0;
                    if (now1) whose[mine[1] - b0] = 0;
                    wave_order();
                }
            } else if (HIST && said > kBeamSaid) {
                for (int i = lane; i < hn; i += 64) {
                    const int32_t id = hist[i];
                    if (in_batch(id) && wave_of(id) == wave) atomicAdd(&times[(id - b0) >> 1], 1u << (16 * (id & 1)));
                }
                wave_order();
#pragma unroll
                for (int j = 0; j < GR; j++) {
                    const uint2 w = ((const uint2 *)times)[j * T + t];
                    if ((w.x | w.y) != 0) {
                        ((uint2 *)times)[j * T + t] = make_uint2(0, 0);          /* for the next batch */
#pragma unroll 1
                        for (int c = 0; c < 4; c++) {
                            const int nc = (int)(((c < 2 ? w.x : w.y) >> (16 * (c & 1))) & 0xffff);
                            const float v = c == 0 ? x[j][0] : c == 1 ? x[j][1] : c == 2 ? x[j][2] : x[j][3];
                            if (nc == 0 || v == -INFINITY) continue;
                            const float y = beam_penalised(p, v, nc);
                            x[j][0] = c == 0 ? y : x[j][0];
                            x[j][1] = c == 1 ? y : x[j][1];
                            x[j][2] = c == 2 ? y : x[j][2];
                            x[j][3] = c == 3 ? y : x[j][3];
                        }
                    }
                }
            }
            float best = -INFINITY;
#pragma unroll
            for (int j = 0; j < GR; j++) {
#pragma unroll
                for (int c = 0; c < 4; c++) bad |= !(x[j][c] < INFINITY);
                best = max3(max3(best, x[j][0], x[j][1]), x[j][2], x[j][3]);
            }
            if (b0 == s0) {
                const uint32_t k = bound_of(sh, best > -INFINITY ? ~desc_key(best) : 0u, p.n);
                if (k != 0) least = key_value(~k);           /* (0: every continuation is an entry) */
                bound = (uint64_t)k << 32;
            }
            const int had = listed;
            if (ballot(best >= least) != 0) {
                uint32_t at_least = 0;                       /* bit 4 j + c */
#pragma unroll
                for (int j = 0; j < GR; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) at_least |= x[j][c] >= least && x[j][c] > -INFINITY ? 1u << (4 * j + c) : 0u;
                while (ballot(at_least != 0) != 0) {
                    const int k = at_least != 0 ? __builtin_ctz(at_least) : 0;
                    float v = x[0][0];
#pragma unroll
                    for (int q = 1; q < 4 * GR; q++) v = k == q ? x[q >> 2][q & 3] : v;
                    const uint64_t e = entry_of(v, b0 + (k >> 2) * T * 4 + t4 + (k & 3));
                    put(at_least != 0 && e >= bound, e);
                    at_least &= at_least - 1;
                }
            }
            /* (-inf counts as exp(-700) of the maximum: nothing) */
            const float up_to = mw ? wave_max_dpp(best) : best;
            const float to = fmaxf(fmaxf(most, up_to), -3.40282347e38f);
            double s = 0.0;
            int live = 64 * 4 * GR;
            uint64_t who[4 * GR];
            if (mw) {
                live = 0;
#pragma unroll
                for (int q = 0; q < 4 * GR; q++) {
                    who[q] = ballot(x[q >> 2][q & 3] > -INFINITY);
                    live += (int)__popcll(who[q]);
                }
            }
            if (live <= kBeamPacked) {
                /* few allowed: those of the wave, side by side */
                float *side = packed[wave];
                int at = 0;
#pragma unroll
                for (int q = 0; q < 4 * GR; q++) {
                    const int to_place = place_in(who[q], at);
                    if (x[q >> 2][q & 3] > -INFINITY) side[to_place] = x[q >> 2][q & 3];
                    at += (int)__popcll(who[q]);
                }
                wave_order();
#pragma unroll 1
                for (int i = lane; i - lane < live; i += 64) s += exp_neg((double)(i < live ? side[i] : -INFINITY) - (double)to);
                wave_order();
            } else {
#pragma unroll
                for (int j = 0; j < GR; j++) {
#pragma unroll
                    for (int c = 0; c < 4; c++) s += exp_neg((double)x[j][c] - (double)to);
                    asm volatile("" : "+v"(s));              /* (here and in order: all at once they spill) */
                }
            }
            part = part * exp_neg((double)most - (double)to) + s;
            most = fmaxf(most, up_to);
            if (DLK_COLD(listed > kBeamWaveList)) {
                /* more than the list takes: of this batch only the wave's n largest (there is room for
                 * them, below), found bit by bit: the n-th largest value, then the last place of it */
                auto count = [&](auto holds) {
                    int c = 0;
#pragma unroll
                    for (int j = 0; j < GR; j++)
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            float v = x[j][q];
                            asm volatile("" : "+v"(v));      /* (made anew each time: kept, the keys are registers) */
                            c += (int)__popcll(ballot(v > -INFINITY && holds(~desc_key(v), j * T * 4 + t4 + q)));
                        }
                    return c;
                };
                uint32_t value = 0;
#pragma unroll 1
                for (uint32_t bit = 1u << 31; bit; bit >>= 1)
                    if (count([&](uint32_t k, int) { return k >= (value | bit); }) >= p.n) value |= bit;
                const int need = p.n - count([&](uint32_t k, int) { return k > value; });
                int place = 0;                               /* the places below it hold fewer than `need` of that value */
#pragma unroll 1
                for (int bit = B >> 1; bit; bit >>= 1)
                    if (count([&](uint32_t k, int i) { return k == value && i < place + bit; }) < need) place += bit;
                uint64_t nth = (uint64_t)value << 32 | (uint32_t)~(b0 + place);
                nth = max(nth, bound);
                listed = had;
#pragma unroll
                for (int j = 0; j < GR; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const uint64_t e = entry_of(x[j][c], b0 + j * T * 4 + t4 + c);
                        put(x[j][c] > -INFINITY && e >= nth, e);                   /* n at most */
                    }
            }
            if (DLK_COLD(listed > kBeamWaveList - DLK_MAX_BEAMS) && b0 + B < s1) {
                /* the list's n largest, in order, and the last of them as the bound from here on */
                uint64_t e[kBeamWaveList / 64];
                int rank[kBeamWaveList / 64];
                wave_order();
#pragma unroll
                for (int k = 0; k < kBeamWaveList / 64; k++) {
                    const int i = lane + 64 * k;
                    int equal;
                    e[k] = list[min(i, listed - 1)];
                    rank[k] = i < listed ? rank_in(list, listed, e[k], equal) : p.n;
                }
                wave_order();
#pragma unroll
                for (int k = 0; k < kBeamWaveList / 64; k++)
                    if (rank[k] < p.n) list[rank[k]] = e[k];
                wave_order();
                listed = p.n;
                bound = max(bound, list[p.n - 1]);
                least = entry_logit(bound);
            }
        }
        const float wtop = wave_max_dpp(most);
        bad = ballot(bad) != 0;
        if (lane == 0) {
            sh.top[wave] = wtop;
            sh.wave_n[wave] = bad;
            sh.wave_listed[wave] = listed;
        }
        __syncthreads();
        top = sh.top[0];
        bad = sh.wave_n[0] != 0;
#pragma unroll
        for (int w = 1; w < T / 64; w++) {
            top = fmaxf(top, sh.top[w]);
            bad |= sh.wave_n[w] != 0;
        }
        if (bad) {
            top = -INFINITY;
            kept = 0xffffffffu;
        } else if (top > -INFINITY) {
            const double s = wave_incl_scan_d(part * exp_neg((double)fmaxf(most, -3.40282347e38f) - (double)top));
            if (lane == 63) sh.part[wave] = s;
            /* the waves' lists in one */
            uint64_t *joint = (uint64_t *)packed;
            int first = 0, all = 0;
#pragma unroll
            for (int w = 0; w < T / 64; w++) {
                const int c = sh.wave_listed[w];
                first += w < wave ? c : 0;
                all += c;
            }
            for (int a = lane; a < listed; a += 64) joint[first + a] = list[a];
            __syncthreads();
            sum = sh.part[0];
#pragma unroll
            for (int w = 1; w < T / 64; w++) sum += sh.part[w];
            kept = (uint32_t)min(all, p.n);
            uint64_t *out = p.cands + ((int64_t)rl * p.slices + slice) * p.n;
            for (int a = t; a < all; a += T) {
                const uint64_t e = joint[a];
                int equal;
                const int rank = rank_in(joint, all, e, equal);
                if (rank < p.n) bpub64(&out[rank], e);
            }
        }
    }
    BeamSlot *slot = p.slots + (int64_t)rl * p.slices + slice;
    if (t == 0) {
        bpub64(&slot->sum, d2u(sum));
        bpub64(&slot->max_kept, (uint64_t)f2u(top) << 32 | kept);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const int gl = rl / p.beams;
    if (t == 0) {
        const uint32_t old = __hip_atomic_fetch_add(&p.counters[gl], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.last = old == (uint32_t)(p.beams * p.slices - 1);
    }
    __syncthreads();
    if (!sh.last) return;
    if (t == 0) __hip_atomic_store(&p.counters[gl], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    merge_group(p, gl, sh);
}

}  // namespace dlk

extern "C" int dlk_launch_beam_select(const dlk::BeamParams *p, int groups, hipStream_t stream) {
    const unsigned blocks = (unsigned)((int64_t)groups * p->beams * p->slices);
    if (p->hist_off)
        hipLaunchKernelGGL((dlk::beam_select_kernel<true>), dim3(blocks), dim3(dlk::kBeamThreads), 0, stream, *p);
    else
        hipLaunchKernelGGL((dlk::beam_select_kernel<false>), dim3(blocks), dim3(dlk::kBeamThreads), 0, stream, *p);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}
