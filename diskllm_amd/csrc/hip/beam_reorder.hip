/*
 * beam_reorder.hip -- the states of a beam search's rows follow their parents
 * (dlk_beam_reorder): rows of caches and small states, in place or into another buffer,
 * and the CSR histories with the new tokens appended.
 *
 * A copy, bound by memory.  One workgroup takes 4 KB of one group's rows at one (outer,
 * inner) place: each thread loads its 16 bytes of every row that moves, then stores them.
 * Reading all of a column before writing any of it makes the move in place safe for any
 * parents (a row may be parent to several and change its own place) with no second
 * buffer and no order among workgroups, since no two share a column.  Rows that are their
 * own parents are skipped in place: neither read nor written.  16-byte accesses of any
 * alignment.  A thread has as many rows' bytes in registers as a group has rows (rounded
 * up to 4, 8, .. 64): the loads of a column are in flight together.
 *
 * 16 requests of 4 beams with two caches of 1.07 GB, two thirds of the rows moving, 2.7 GB read and
 * written: 476-565 us by the parents and the box (531-561 under the profiler), 4.8 to 5.6 TB/s, a large
 * copy's rate (5.1).  A request's few small states: 4-5 us (13.5 with the
 * host's checks of the tensors), all of them and the histories in one launch.
 *
 * A history's place in the CSR is the sum of the lengths before it, which the workgroups of
 * few rows sum anew each rather than wait for another's.
 */
#include <hip/hip_runtime.h>

#include <utility>

#include "dlk_device.h"
#include "../../../include/diskllm_amd.h"

namespace dlk {

constexpr int kMoveThreads = 256;
constexpr int kMoveStates = 8;                   /* states of one launch */
/* Up to so many rows each history's workgroup sums the lengths before it, past that a launch
 * of one workgroup does (us, summed and launched: 1,024 rows 5.4, 7.2; 2,048 9.4, 8.3; 4,096
 * 20.8, 12.5; 65,536 2,782, 158). */
constexpr int64_t kMoveSummed = 1536;
constexpr int64_t kMoveBlocks = 0xffffff;        /* workgroups of one launch: 2^32 threads and over are refused */

typedef uint32_t u4_any __attribute__((ext_vector_type(4), aligned(1)));

struct MoveState {
    const unsigned char *src;
    unsigned char *dst;
    int64_t bytes, src_row, src_outer, src_inner, dst_row, dst_outer, dst_inner;
    int n_outer, n_inner;
    int tiles;                                   /* of kMoveThreads * 16 bytes */
    int in_place;
    int64_t first;                               /* first workgroup */
};

struct MoveParams {
    const int32_t *parents;
    int groups, beams, n_out, n_states;
    MoveState s[kMoveStates];
    int64_t hist_first;                          /* first workgroup of the histories, one per new row */
    const int32_t *off, *ids, *tokens;
    int32_t *out_off, *out_ids;
    int keep;
    int offsets;                                 /* out_off is there already (history_offsets_kernel) */
};

/* The row that new row r takes, -1 where its parent is none of its group's. */
DLK_DEV int parent_of(const MoveParams &p, int g, int r) {
    const int q = p.parents[(int64_t)g * p.n_out + r];
    return q >= g * p.beams && q < (g + 1) * p.beams ? q : -1;
}

/* Length of the history that new row r (of all) will have; the parent in q. */
DLK_DEV int new_length(const MoveParams &p, int64_t r, int &q) {
    q = parent_of(p, (int)(r / p.n_out), (int)(r % p.n_out));
    if (q < 0) return 0;
    const int64_t n = max(p.off[q + 1] - p.off[q], 0);
    return (int)min(n + (p.tokens && p.tokens[r] >= 0 ? 1 : 0), (int64_t)p.keep);
}

DLK_DEV void move_history(const MoveParams &p, int64_t r) {
    __shared__ int64_t part[kMoveThreads / 64];
    const int t = threadIdx.x;
    int64_t before = 0;
    int q;
    const int n = new_length(p, r, q);
    if (p.offsets) {
        before = p.out_off[r];
    } else {
        int other;
        for (int64_t i = t; i < r; i += kMoveThreads) before += new_length(p, i, other);
        for (int m = 1; m < 64; m <<= 1) before += shfl_xor(before, m);
        if (lane_id() == 0) part[wave_id()] = before;
        __syncthreads();
        before = part[0] + part[1] + part[2] + part[3];
        if (t == 0) {
            p.out_off[r] = (int32_t)before;
            if (r == (int64_t)p.groups * p.n_out - 1) p.out_off[r + 1] = (int32_t)(before + n);
        }
    }
    if (n == 0) return;
    const int add = p.tokens && p.tokens[r] >= 0 ? 1 : 0;
    const int32_t *from = p.ids + p.off[q + 1] - (n - add);
    int32_t *to = p.out_ids + before;
    for (int i = t; i < n; i += kMoveThreads) to[i] = i < n - add ? from[i] : p.tokens[r];
}

/* The new histories' offsets, by one workgroup (their sum fits 31 bits). */
__global__ __launch_bounds__(1024) void history_offsets_kernel(MoveParams p) {
    __shared__ int part[16];
    const int t = threadIdx.x, lane = lane_id(), wave = wave_id();
    const int64_t rows = (int64_t)p.groups * p.n_out;
    int before = 0;
    for (int64_t r0 = 0; r0 < rows; r0 += 1024) {
        int q;
        const int n = r0 + t < rows ? new_length(p, r0 + t, q) : 0;
        int upto = n;
        for (int m = 1; m < 64; m <<= 1) {
            const int o = __shfl_up(upto, m);
            upto += lane >= m ? o : 0;
        }
        if (lane == 63) part[wave] = upto;
        __syncthreads();
        int waves = 0;
        for (int w = 0; w < 16; w++) {
            upto += w < wave ? part[w] : 0;
            waves += part[w];
        }
        if (r0 + t < rows) p.out_off[r0 + t] = before + upto - n;
        before += waves;
        __syncthreads();
    }
    if (t == 0) p.out_off[rows] = before;
}

/* NB: the rows whose bytes a thread holds at once, at least n_out. */
template <int NB>
__global__ __launch_bounds__(kMoveThreads) void move_kernel(MoveParams p) {
    const int64_t blk = blockIdx.x;
    if (blk >= p.hist_first) {
        move_history(p, blk - p.hist_first);
        return;
    }
    int si = 0;
#pragma unroll
    for (int k = 1; k < kMoveStates; k++)
        if (k < p.n_states && blk >= p.s[k].first) si = k;
    const MoveState &s = p.s[si];
    int64_t k = blk - s.first;
    const int tile = (int)(k % s.tiles);
    k /= s.tiles;
    const int inner = (int)(k % s.n_inner);
    k /= s.n_inner;
    const int g = (int)(k % p.groups), outer = (int)(k / p.groups);
    const int64_t at = ((int64_t)tile * kMoveThreads + threadIdx.x) * 16;
    if (at >= s.bytes) return;
    const unsigned char *src = s.src + outer * s.src_outer + inner * s.src_inner;
    unsigned char *dst = s.dst + outer * s.dst_outer + inner * s.dst_inner + (int64_t)g * p.n_out * s.dst_row;
    int from[NB];                                /* uniform: scalar registers */
#pragma unroll
    for (int r = 0; r < NB; r++) {
        from[r] = r < p.n_out ? parent_of(p, g, r) : -1;
        if (s.in_place && from[r] == g * p.n_out + r) from[r] = -1;
    }
    if (at + 16 <= s.bytes) {
        u4_any v[NB];
#pragma unroll
        for (int r = 0; r < NB; r++)
            if (from[r] >= 0) v[r] = *(const u4_any *)(src + from[r] * s.src_row + at);
#pragma unroll
        for (int r = 0; r < NB; r++)
            if (from[r] >= 0) *(u4_any *)(dst + r * s.dst_row + at) = v[r];
    } else {
        /* the last bytes, one column at a time */
        for (int64_t b = at; b < s.bytes; b++) {
            unsigned char v[NB];
#pragma unroll
            for (int r = 0; r < NB; r++) v[r] = from[r] >= 0 ? src[from[r] * s.src_row + b] : 0;
#pragma unroll
            for (int r = 0; r < NB; r++)
                if (from[r] >= 0) dst[r * s.dst_row + b] = v[r];
        }
    }
}

template <int NB>
int launch_move(const MoveParams &p, int64_t blocks, hipStream_t stream) {
    hipLaunchKernelGGL((move_kernel<NB>), dim3((unsigned)blocks), dim3(kMoveThreads), 0, stream, p);
    return hipGetLastError() == hipSuccess ? DLK_OK : DLK_ERR_HIP;
}

int launch_moves(const MoveParams &p, int64_t blocks, hipStream_t stream) {
    if (p.n_out <= 4) return launch_move<4>(p, blocks, stream);
    if (p.n_out <= 8) return launch_move<8>(p, blocks, stream);
    if (p.n_out <= 16) return launch_move<16>(p, blocks, stream);
    if (p.n_out <= 32) return launch_move<32>(p, blocks, stream);
    return launch_move<64>(p, blocks, stream);
}

/* Whether the strides of a destination keep its bytes apart: sorted, each at least the
 * extent of what lies below it. */
bool apart(int64_t bytes, int64_t rows, int64_t row, int64_t no, int64_t outer, int64_t ni, int64_t inner) {
    struct Dim { int64_t stride, n; } c[3] = {{row, rows}, {outer, no}, {inner, ni}};
    if (c[0].stride > c[1].stride) std::swap(c[0], c[1]);
    if (c[1].stride > c[2].stride) std::swap(c[1], c[2]);
    if (c[0].stride > c[1].stride) std::swap(c[0], c[1]);
    int64_t extent = bytes;
    for (const Dim &d : c) {
        if (d.n <= 1) continue;
        if (d.stride < extent) return false;
        extent += (d.n - 1) * d.stride;
    }
    return true;
}

int64_t tiles_of(int64_t bytes) { return (bytes + kMoveThreads * 16 - 1) / (kMoveThreads * 16); }

}  // namespace dlk

extern "C" int dlk_beam_reorder(const int32_t *parents, int groups, int beams, int n_out, const dlk_beam_state *states,
                                int n_states, const dlk_beam_history *history, hipStream_t stream) {
    using namespace dlk;
    if (!parents || groups < 0 || beams <= 0 || n_out <= 0 || n_states < 0 || (n_states && !states)) return DLK_ERR_INVALID;
    if (beams > DLK_MAX_BEAMS || n_out > DLK_MAX_BEAMS) return DLK_ERR_UNSUPPORTED;
    const int64_t rows = (int64_t)groups * n_out, rows_in = (int64_t)groups * beams;
    if (rows > 0x3fffffff || rows_in > 0x3fffffff || (history && rows > kMoveBlocks)) return DLK_ERR_UNSUPPORTED;
    for (int i = 0; i < n_states; i++) {
        const dlk_beam_state &s = states[i];
        if (s.bytes < 0 || s.n_outer < 0 || s.n_inner < 0) return DLK_ERR_INVALID;
        if (s.src_row < 0 || s.src_outer < 0 || s.src_inner < 0 || s.dst_row < 0 || s.dst_outer < 0 || s.dst_inner < 0)
            return DLK_ERR_INVALID;
        if (s.bytes == 0 || s.n_outer == 0 || s.n_inner == 0 || groups == 0) continue;
        if (!s.src || !s.dst) return DLK_ERR_INVALID;          /* (empty ones may be nowhere) */
        if (!apart(s.bytes, rows, s.dst_row, s.n_outer, s.dst_outer, s.n_inner, s.dst_inner)) return DLK_ERR_INVALID;
        const unsigned char *a = (const unsigned char *)s.src, *d = (const unsigned char *)s.dst;
        if (a == d) {
            if (beams != n_out || s.src_row != s.dst_row || s.src_outer != s.dst_outer || s.src_inner != s.dst_inner)
                return DLK_ERR_INVALID;
        } else {
            const int64_t ea = (rows_in - 1) * s.src_row + (s.n_outer - 1) * s.src_outer + (s.n_inner - 1) * s.src_inner + s.bytes;
            const int64_t ed = (rows - 1) * s.dst_row + (s.n_outer - 1) * s.dst_outer + (s.n_inner - 1) * s.dst_inner + s.bytes;
            if (a < d + ed && d < a + ea) return DLK_ERR_INVALID;
        }
        /* one buffer twice, or two that change places (what else overlaps is the caller's to know:
         * the strides of two states may interleave) */
        for (int j = 0; j < i; j++)
            if (states[j].bytes > 0 && states[j].n_outer > 0 && states[j].n_inner > 0 &&
                (d == states[j].dst || d == states[j].src || a == states[j].dst))
                return DLK_ERR_INVALID;
        if ((double)tiles_of(s.bytes) * s.n_outer * s.n_inner * groups > (double)kMoveBlocks) return DLK_ERR_UNSUPPORTED;
    }
    const dlk_beam_history *h = history;
    if (h) {
        if (!h->off || !h->ids || !h->out_off || !h->out_ids || h->max_history <= 0) return DLK_ERR_INVALID;
        if (h->out_off == h->off || h->out_ids == h->ids) return DLK_ERR_INVALID;
        if (rows * h->max_history > 0x7fffffff) return DLK_ERR_UNSUPPORTED;       /* 32-bit offsets */
    }
    if (groups == 0) return DLK_OK;
    int at = 0;
    do {
        MoveParams p;
        p.parents = parents;
        p.groups = groups; p.beams = beams; p.n_out = n_out;
        p.n_states = 0;
        int64_t blocks = 0;
        for (; at < n_states && p.n_states < kMoveStates; at++) {
            const dlk_beam_state &s = states[at];
            if (s.bytes == 0 || s.n_outer == 0 || s.n_inner == 0) continue;
            MoveState &m = p.s[p.n_states];
            m.src = (const unsigned char *)s.src;
            m.dst = (unsigned char *)s.dst;
            m.bytes = s.bytes;
            m.src_row = s.src_row; m.src_outer = s.src_outer; m.src_inner = s.src_inner;
            m.dst_row = s.dst_row; m.dst_outer = s.dst_outer; m.dst_inner = s.dst_inner;
            m.n_outer = s.n_outer; m.n_inner = s.n_inner;
            m.in_place = s.src == s.dst;
            m.tiles = (int)tiles_of(s.bytes);
            m.first = blocks;
            const int64_t all = (int64_t)m.tiles * s.n_outer * s.n_inner * groups;
            if (blocks + all > kMoveBlocks) break;
            blocks += all;
            p.n_states++;
        }
        p.hist_first = blocks;
        if (h && at == n_states && blocks + rows <= kMoveBlocks) {
            p.off = h->off; p.ids = h->ids; p.tokens = h->tokens;
            p.out_off = h->out_off; p.out_ids = h->out_ids;
            p.keep = h->max_history;
            p.offsets = rows > kMoveSummed;
            if (p.offsets) {
                hipLaunchKernelGGL(history_offsets_kernel, dim3(1), dim3(1024), 0, stream, p);
                if (hipGetLastError() != hipSuccess) return DLK_ERR_HIP;
            }
            blocks += rows;
            h = nullptr;
        }
        if (blocks == 0) continue;
        const int rc = launch_moves(p, blocks, stream);
        if (rc != DLK_OK) return rc;
    } while (at < n_states || h);
    return DLK_OK;
}
