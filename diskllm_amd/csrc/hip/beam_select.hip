/*
 * beam_select.hip -- one step of a beam search: of the continuations (row, id) of a group
 * of rows the n with the largest score + log softmax(l)[id] (dlk_beam_select).
 *
 * One workgroup reads a slice of 8,192 logits of a row once, into registers; masks and
 * penalises them; sums exp(l - slice maximum) in 64 bits; and lists the slice's n
 * largest entries in order.  Log softmax is increasing in l, so a row's n best
 * continuations are its n largest logits and none of the others is needed again.  The
 * group's last workgroup to finish (relaxed agent-scope atomics, as the top-k kernel's)
 * joins the slices' sums and merges the lists under the keys in 64 bits.
 *
 * Sums and keys are 64-bit because the order of continuations of different rows hangs on
 * differences of their log-sums; 64-bit FMAs run at the plain 32-bit ones' rate here.
 */
#include "dlk_device.h"
#include "beam_select.h"
#include "../../../include/diskllm_amd.h"

namespace dlk {

constexpr int kBeamList = 512;         /* entries that a workgroup orders at once */

DLK_DEV void bpub64(uint64_t *a, uint64_t v) { __hip_atomic_store(a, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DLK_DEV uint64_t bget64(const uint64_t *a) {
    return __hip_atomic_load((uint64_t *)a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

/* exp(x) for x <= 0 to some 1e-11: 2^k times the series of e^r, |r| <= ln2 / 2. */
DLK_DEV double exp_neg(double x) {
    x = fmax(x, -700.0);
    const double k = rint(x * 1.4426950408889634);
    const double r = fma(-k, 1.9082149292705877e-10, fma(-k, 0.693147180369123816490, x));
    double y = 1.0 / 3628800.0;
    y = fma(y, r, 1.0 / 362880.0);
    y = fma(y, r, 1.0 / 40320.0);
    y = fma(y, r, 1.0 / 5040.0);
    y = fma(y, r, 1.0 / 720.0);
    y = fma(y, r, 1.0 / 120.0);
    y = fma(y, r, 1.0 / 24.0);
    y = fma(y, r, 1.0 / 6.0);
    y = fma(y, r, 0.5);
    y = fma(y, r, 1.0);
    y = fma(y, r, 1.0);
    return ldexp(y, (int)k);
}

/* An entry of a list: larger is better (the logit's ascending key, then the lower id). */
DLK_DEV uint64_t entry_of(float l, int id) { return (uint64_t)~desc_key(l) << 32 | (uint32_t)~id; }
DLK_DEV float entry_logit(uint64_t e) { return key_value(~(uint32_t)(e >> 32)); }
DLK_DEV int entry_id(uint64_t e) { return (int)~(uint32_t)e; }

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

/* The largest key of 20 leading bits that at least r of the lanes' keys reach (0: fewer
 * than r lanes have one). */
DLK_DEV uint32_t wave_rth(uint32_t a, int r) {
    uint32_t K = 0;
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1)
        if ((int)__popcll(ballot(a >= (K | bit))) >= r) K |= bit;
    return K;
}

template <class T>
DLK_DEV T block_sum(T v, T *part) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += shfl_xor(v, m);
    if (lane_id() == 0) part[wave_id()] = v;
    __syncthreads();
    T s = part[0];
#pragma unroll
    for (int w = 1; w < kBeamThreads / 64; w++) s += part[w];
    __syncthreads();
    return s;
}

struct BeamShared {
    uint64_t key[kBeamList];            /* merge: keys; slice: entries */
    uint64_t ent[kBeamList];
    double base[DLK_MAX_BEAMS];         /* per row of the group: log-sum, norm, score, maximum */
    double norm[DLK_MAX_BEAMS];
    double part[kBeamThreads / 64];
    float cum[DLK_MAX_BEAMS];
    float top[DLK_MAX_BEAMS];
    uint32_t wave_key[kBeamThreads / 64];
    int wave_n[kBeamThreads / 64];
    int place[kBeamList];               /* list of each entry */
    int kind[DLK_MAX_BEAMS];            /* 0: none, 1: by its lists, 2: finished */
    int count, last;
    uint64_t best_key[kBeamThreads / 64], best_ent[kBeamThreads / 64];
    int best_list[kBeamThreads / 64];
};

/* a before b: larger key, lower row, larger entry. */
DLK_DEV bool before(uint64_t ka, int ra, uint64_t ea, uint64_t kb, int rb, uint64_t eb) {
    if (ka != kb) return ka > kb;
    if (ra != rb) return ra < rb;
    return ea > eb;
}

/* The continuation (row b, entry e) in 64 bits. */
DLK_DEV double beam_score(const BeamShared &sh, int b, uint64_t e) {
    if (sh.kind[b] == 2) return (double)sh.cum[b];
    return (double)sh.cum[b] + (((double)entry_logit(e) - (double)sh.top[b]) - sh.base[b]);
}

DLK_DEV void write_continuation(const BeamParams &p, const BeamShared &sh, int g, int j, int b, uint64_t e) {
    const int64_t o = (int64_t)g * p.n + j, row = (int64_t)g * p.beams + b;
    const bool over = sh.kind[b] == 2;
    const int id = over ? p.eos : entry_id(e);
    const int len = p.lengths ? p.lengths[row] : 0;
    p.out_tokens[o] = id;
    p.out_parents[o] = (int32_t)row;
    p.out_scores[o] = (float)beam_score(sh, b, e);
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

/* The group's lists merged, by its last workgroup. */
DLK_DEV void merge_group(const BeamParams &p, int gl, BeamShared &sh) {
    const int t = threadIdx.x, lane = lane_id(), wave = wave_id(), g = p.g0 + gl;
    const int L = p.beams * p.slices;
    const BeamSlot *slots = p.slots + (int64_t)gl * L;
    const uint64_t *cands = p.cands + (int64_t)gl * L * p.n;
    /* the rows' sums, a wave each */
    for (int b = wave; b < p.beams; b += kBeamThreads / 64) {
        const int64_t row = (int64_t)g * p.beams + b;
        const float cum = p.scores ? p.scores[row] : 0.0f;
        const bool over = p.finished && p.finished[row];
        float top = -INFINITY;
        double sum = 0.0;
        bool bad = false;
        for (int s = lane; s < p.slices; s += 64) {
            const uint64_t sm = bget64(&slots[b * p.slices + s].sum), mk = bget64(&slots[b * p.slices + s].max_kept);
            const float m = u2f((uint32_t)(mk >> 32));
            bad |= (uint32_t)mk == 0xffffffffu;
            if (m > -INFINITY) {
                const float to = fmaxf(top, m);
                sum = sum * (top > -INFINITY ? exp_neg((double)top - (double)to) : 0.0) +
                      u2d(sm) * exp_neg((double)m - (double)to);
                top = to;
            }
        }
        const float all = wave_max_dpp(top);
        sum = all > -INFINITY && top > -INFINITY ? sum * exp_neg((double)top - (double)all) : 0.0;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) sum += shfl_xor(sum, m);
        bad = ballot(bad) != 0;
        if (lane == 0) {
            const int len = p.lengths ? p.lengths[row] : 0;
            const double length = fmax((double)len + (over ? 0.0 : 1.0), 1.0);
            const bool alive = cum > -INFINITY && cum < INFINITY;
            sh.cum[b] = cum;
            sh.top[b] = all;
            sh.base[b] = all > -INFINITY ? log(sum) : 0.0;
            sh.norm[b] = p.alpha == 0.0f ? 1.0 : pow(length, (double)p.alpha);
            sh.kind[b] = !alive ? 0 : over ? 2 : bad || !(all > -INFINITY) ? 0 : 1;
            if (p.status && (!(cum < INFINITY) || (alive && !over && bad))) atomicOr(p.status, DLK_STATUS_NOT_FINITE);
        }
    }
    if (t == 0) sh.count = 0;
    __syncthreads();
    /* a list per (row, slice); a finished row's first list holds its one continuation.  List i
     * goes to thread (i % 4) * 64 + i / 4 % 64, so that the waves share few lists evenly */
    const int mine = (t & 63) * 4 + (t >> 6);
    auto listed = [&](int i) {
        const int b = i / p.slices;
        if (sh.kind[b] == 0) return 0;
        if (sh.kind[b] == 2) return i % p.slices == 0 ? 1 : 0;
        return (int)(uint32_t)bget64(&slots[i].max_kept);
    };
    auto entry = [&](int i, int j) { return sh.kind[i / p.slices] == 2 ? ~0ull : bget64(&cands[(int64_t)i * p.n + j]); };
    auto key = [&](int i, uint64_t e) {
        const int b = i / p.slices;
        return double_key(beam_score(sh, b, e) / sh.norm[b]);
    };
    uint64_t head = 0;
    for (int i = mine; i < L; i += kBeamThreads)
        if (listed(i) > 0) head = max(head, key(i, entry(i, 0)));
    /* a bound that n heads, thus n continuations, reach */
    const uint32_t kw = wave_rth((uint32_t)(head >> 32), (p.n + 3) / 4);
    if (lane == 0) sh.wave_key[wave] = kw;
    __syncthreads();
    uint32_t bound = sh.wave_key[0];
#pragma unroll
    for (int w = 1; w < kBeamThreads / 64; w++) bound = min(bound, sh.wave_key[w]);
    for (int i = mine; i < L; i += kBeamThreads) {
        const int n = listed(i);
        for (int j = 0; j < n; j++) {
            const uint64_t e = entry(i, j), k = key(i, e);
            if ((uint32_t)(k >> 32) < bound) break;
            const int at = atomicAdd(&sh.count, 1);
            if (at < kBeamList) {
                sh.key[at] = k;
                sh.ent[at] = e;
                sh.place[at] = i;
            }
        }
    }
    __syncthreads();
    const int C = sh.count;
    if (DLK_HOT(C <= kBeamList)) {
        for (int a = t; a < C; a += kBeamThreads) {
            const uint64_t k = sh.key[a], e = sh.ent[a];
            const int i = sh.place[a], b = i / p.slices;
            int rank = 0;
            for (int c = 0; c < C; c++) rank += before(sh.key[c], sh.place[c] / p.slices, sh.ent[c], k, b, e) ? 1 : 0;
            if (rank < p.n) write_continuation(p, sh, g, rank, b, e);
        }
        for (int j = C + t; j < p.n; j += kBeamThreads) write_none(p, g, j);
    } else {
        /* too many at or above the bound (few lists for n, or runs of equal keys): the best one
         * still left, n times, the written ones known by the last one's place in the order */
        uint64_t lk = ~0ull, le = ~0ull;
        int lb = -1;
        for (int j = 0; j < p.n; j++) {
            uint64_t bk = 0, be = 0;
            int bi = -1;
            for (int i = mine; i < L; i += kBeamThreads) {
                const int n = listed(i), b = i / p.slices;
                for (int q = 0; q < n; q++) {
                    const uint64_t e = entry(i, q), k = key(i, e);
                    if (!before(lk, lb, le, k, b, e)) continue;               /* written */
                    if (bi < 0 || before(k, b, e, bk, bi / p.slices, be)) { bk = k; be = e; bi = i; }
                    break;                                                    /* (the list is in order) */
                }
            }
            for (int m = 1; m < 64; m <<= 1) {
                const uint64_t ok = shfl_xor(bk, m), oe = shfl_xor(be, m);
                const int oi = shfl_xor(bi, m);
                if (oi >= 0 && (bi < 0 || before(ok, oi / p.slices, oe, bk, bi / p.slices, be))) { bk = ok; be = oe; bi = oi; }
            }
            if (lane == 0) { sh.best_key[wave] = bk; sh.best_ent[wave] = be; sh.best_list[wave] = bi; }
            __syncthreads();
            bi = -1;
            for (int w = 0; w < kBeamThreads / 64; w++) {
                const int oi = sh.best_list[w];
                if (oi >= 0 && (bi < 0 || before(sh.best_key[w], oi / p.slices, sh.best_ent[w], bk, bi / p.slices, be))) {
                    bk = sh.best_key[w]; be = sh.best_ent[w]; bi = oi;
                }
            }
            __syncthreads();
            if (t == 0) {
                if (bi >= 0) write_continuation(p, sh, g, j, bi / p.slices, be);
                else write_none(p, g, j);
            }
            if (bi >= 0) { lk = bk; le = be; lb = bi / p.slices; }
        }
    }
}

template <bool HIST>
__global__ __launch_bounds__(kBeamThreads) void beam_select_kernel(BeamParams p) {
    __shared__ BeamShared sh;
    __shared__ __align__(16) uint32_t times[HIST ? kBeamSlice / 2 : 4];      /* occurrences, 16 bits an id */
    const int t = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int slice = blockIdx.x % p.slices, rl = blockIdx.x / p.slices;      /* rl: row of the launch */
    const int64_t row = (int64_t)p.g0 * p.beams + rl;
    const int s0 = slice * kBeamSlice;
    const float cum = p.scores ? p.scores[row] : 0.0f;
    int hn = 0;
    const int32_t *hist = nullptr;
    if (HIST) {
        const int h0 = p.hist_off[row];
        hn = p.hist_off[row + 1] - h0;
        hist = p.hist_ids + h0;
    }
    /* a row without continuations, or a finished one: its logits are not read */
    bool idle = !(cum > -INFINITY && cum < INFINITY) || (p.finished && p.finished[row]);
    const bool too_long = HIST && !idle && hn > p.max_hist;
    idle |= too_long;
    if (too_long && t == 0 && slice == 0 && p.status) atomicOr(p.status, DLK_STATUS_HISTORY_TOO_LONG);
    float top = -INFINITY;
    double sum = 0.0;
    uint32_t kept = 0;
    if (!idle) {
        const float *lg = p.logits + row * p.ld;
        float x[kBeamGroups][4];
#pragma unroll
        for (int j = 0; j < kBeamGroups; j++) {
            const int i = s0 + (j * kBeamThreads + t) * 4;
            if (i + 3 < p.V) {
                const float4 v = load4(lg + i);
                x[j][0] = v.x; x[j][1] = v.y; x[j][2] = v.z; x[j][3] = v.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++) x[j][c] = i + c < p.V ? lg[i + c] : -INFINITY;
            }
        }
        if (p.mask) {
            const uint32_t *mw = p.mask + (int64_t)(p.mask_row ? p.mask_row[row] : row) * p.mask_ld;
#pragma unroll
            for (int j = 0; j < kBeamGroups; j++) {
                const int i = s0 + (j * kBeamThreads + t) * 4;
                const uint32_t bits = i < p.V ? mw[i >> 5] >> (i & 31) : 0u;
#pragma unroll
                for (int c = 0; c < 4; c++) x[j][c] = (bits >> c) & 1u ? x[j][c] : -INFINITY;
            }
        }
        if (HIST && hn > 0) {
            for (int i = t; i < kBeamSlice / 8; i += kBeamThreads) ((uint4 *)times)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            for (int i = t; i < hn; i += kBeamThreads) {
                const int32_t id = hist[i];
                if (id >= 0 && id < p.V && id >= s0 && id - s0 < kBeamSlice)
                    atomicAdd(&times[(id - s0) >> 1], 1u << (16 * (id & 1)));
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kBeamGroups; j++) {
                const uint2 w = ((const uint2 *)times)[j * kBeamThreads + t];
                if ((w.x | w.y) != 0) {
                    const int n[4] = {(int)(w.x & 0xffff), (int)(w.x >> 16), (int)(w.y & 0xffff), (int)(w.y >> 16)};
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        const int nc = c == 0 ? n[0] : c == 1 ? n[1] : c == 2 ? n[2] : n[3];
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
        float mine = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < kBeamGroups; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                bad |= !(x[j][c] < INFINITY);
                mine = fmaxf(mine, x[j][c]);
            }
        const float wtop = wave_max_dpp(mine);
        const uint32_t akey = mine > -INFINITY ? ~desc_key(mine) : 0u;
        const uint32_t kw = wave_rth(akey, (p.n + 3) / 4);
        bad = ballot(bad) != 0;
        if (lane == 0) {
            sh.part[wave] = (double)wtop;
            sh.wave_key[wave] = kw;
            sh.wave_n[wave] = bad;
        }
        if (t == 0) sh.count = 0;
        __syncthreads();
        uint32_t bound = sh.wave_key[0];
        top = (float)sh.part[0];
        bad = sh.wave_n[0] != 0;
#pragma unroll
        for (int w = 1; w < kBeamThreads / 64; w++) {
            bound = min(bound, sh.wave_key[w]);
            top = fmaxf(top, (float)sh.part[w]);
            bad |= sh.wave_n[w] != 0;
        }
        __syncthreads();
        if (bad) {
            top = -INFINITY;
            kept = 0xffffffffu;
        } else if (top > -INFINITY) {
            double s = 0.0;
#pragma unroll
            for (int j = 0; j < kBeamGroups; j++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (x[j][c] > -INFINITY) s += exp_neg((double)x[j][c] - (double)top);
            sum = block_sum(s, sh.part);
            /* the entries at or above the bound */
            auto collect = [&](uint64_t least) {
                if (mine > -INFINITY && entry_of(mine, 0) >= least) {
#pragma unroll
                    for (int j = 0; j < kBeamGroups; j++)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const uint64_t e = entry_of(x[j][c], s0 + (j * kBeamThreads + t) * 4 + c);
                            if (x[j][c] > -INFINITY && e >= least) {
                                const int at = atomicAdd(&sh.count, 1);
                                if (at < kBeamList) sh.key[at] = e;
                            }
                        }
                }
                __syncthreads();
                return sh.count;
            };
            int C = collect((uint64_t)bound << 32);
            if (DLK_COLD(C > kBeamList)) {
                /* too many: the n-th largest entry exactly, bit by bit (entries are all unlike) */
                uint64_t least = 0;
                for (uint64_t bit = 1ull << 63; bit; bit >>= 1) {
                    int c = 0;
#pragma unroll
                    for (int j = 0; j < kBeamGroups; j++)
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            c += x[j][q] > -INFINITY &&
                                 entry_of(x[j][q], s0 + (j * kBeamThreads + t) * 4 + q) >= (least | bit) ? 1 : 0;
                    c = wave_sum_i32(c);
                    if (lane == 0) sh.wave_n[wave] = c;
                    __syncthreads();
                    c = sh.wave_n[0];
#pragma unroll
                    for (int w = 1; w < kBeamThreads / 64; w++) c += sh.wave_n[w];
                    __syncthreads();
                    if (c >= p.n) least |= bit;
                }
                if (t == 0) sh.count = 0;
                __syncthreads();
                C = collect(least);
            }
            kept = (uint32_t)min(C, p.n);
            uint64_t *out = p.cands + ((int64_t)rl * p.slices + slice) * p.n;
            for (int a = t; a < C; a += kBeamThreads) {
                const uint64_t e = sh.key[a];
                int rank = 0;
                for (int c = 0; c < C; c++) rank += sh.key[c] > e ? 1 : 0;
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
