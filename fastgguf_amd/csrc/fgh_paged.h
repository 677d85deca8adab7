// fgh_paged.h - the paged KV cache's addressing and batch description, shared by its append
// (fgh_paged.hip) and its attention (fgh_pattn.hip). Internal.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace fgh {

// fgh_paged_cache and fgh_paged_batch as the kernels take them
struct Paged {
    uint8_t *k, *v;
    const int32_t *table, *tok, *len;
    int64_t page_stride;  // values between pages
    int type, n_pages, shift, table_stride, n_head_kv, hd;  // 1 << shift positions a page
    int n_seq, n_tok, max_tok, max_len;  // max_len: at most the table's positions
};

// offset in values of a head's block within k or v, for a page that is known to be in range
__host__ __device__ inline int64_t paged_head(const Paged &a, int page, int kvh) {
    return page * a.page_stride + ((int64_t)kvh * a.hd << a.shift);
}
__host__ __device__ inline bool paged_ok(const Paged &a, int page) { return (uint32_t)page < (uint32_t)a.n_pages; }

// A sequence's rows t0 .. t0 + n - 1 and its positions. ok: within the batch's bounds; otherwise its
// rows (clamped to the buffers) are NaN and nothing is appended.
struct PagedSeq {
    int t0, n, len;
    bool ok;
};
__device__ __forceinline__ PagedSeq paged_seq(const Paged &a, int s) {
    const int b = a.tok[s], e = a.tok[s + 1], len = a.len[s];
    PagedSeq q;
    q.t0 = min(max(b, 0), a.n_tok);
    q.n = max(min(max(e, 0), a.n_tok) - q.t0, 0);  // e may be anything: a difference with it as it is could wrap to many rows
    q.len = len;
    q.ok = b >= 0 && e <= a.n_tok && q.n <= a.max_tok && len >= q.n && len <= a.max_len;
    return q;
}
// the same of a uniform s, in scalar registers (the loads' results would stay in vector registers)
__device__ __forceinline__ PagedSeq paged_useq(const Paged &a, int s) {
    PagedSeq q = paged_seq(a, s);
    q.t0 = __builtin_amdgcn_readfirstlane(q.t0);
    q.n = __builtin_amdgcn_readfirstlane(q.n);
    q.len = __builtin_amdgcn_readfirstlane(q.len);
    q.ok = __builtin_amdgcn_readfirstlane(q.ok);
    return q;
}
// The rows that lane i's sequence, of 64 in order, has for itself: not those below the start of an earlier one (`top`: of the
// sequences before the 64, 0 at first). Only where starts decrease there are such: rows that are in two sequences, or in none. What is left of
// the sequences is then disjoint, so that launches sized by n_tok hold all of it; positions do not change, since the first rows go.
__device__ __forceinline__ void paged_own_rows(const Paged &a, int s, PagedSeq &q, int &top) {
    const bool falls = s < a.n_seq && a.tok[s + 1] < a.tok[s];
    int m = q.t0;  // 0 behind the last sequence
    if (__builtin_amdgcn_ballot_w64(falls) || __builtin_amdgcn_readfirstlane(m) < top) {
        const int lane = threadIdx.x & 63;
        for (int o = 1; o < 64; o <<= 1) m = max(m, __shfl_up(m, o, 64));  // lanes below o get their own
        const int before = __shfl_up(m, 1, 64), from = max(q.t0, max(lane > 0 ? before : 0, top));
        q.n = max(q.t0 + q.n - from, 0);
        q.t0 = from;
    }
    top = max(top, __builtin_amdgcn_readlane(m, 63));
}
// the same for one sequence s, uniform
__device__ __forceinline__ void paged_own_rows(const Paged &a, int s, PagedSeq &q) {
    int m = q.t0;
    for (int i = threadIdx.x & 63; i < s; i += 64) m = max(m, min(a.tok[i], a.n_tok));
    for (int o = 1; o < 64; o <<= 1) m = max(m, __shfl_xor(m, o, 64));
    const int from = __builtin_amdgcn_readfirstlane(m);
    q.n = max(q.t0 + q.n - from, 0);
    q.t0 = from;
}
// the sequence of row t, or -1: the last s with tok[s] <= t, if t < tok[s + 1]. Every wavefront finds
// it for itself, 64 starts a load.
__device__ __forceinline__ int paged_find(const Paged &a, int t) {
    const int lane = threadIdx.x & 63;
    int s = -1;
    for (int b = 0; b <= a.n_seq; b += 64) {  // starts tok[0] .. tok[n_seq]: the last one ends the batch
        const int i = b + lane;
        const uint64_t m = __builtin_amdgcn_ballot_w64(i <= a.n_seq && a.tok[min(i, a.n_seq)] <= t);
        s += __builtin_popcountll(m);
        if (m != ~0ull) break;
    }
    return s >= a.n_seq ? -1 : s;
}

// a launch's workgroups of 256: HIP takes up to 2^32 - 1 threads
constexpr int64_t PAGED_GRID = (1 << 24) - 1;
// at most as many tiles as sequences' new tokens can have: of n, n / 64 whole ones and two ends
inline int64_t paged_vtiles(int64_t n_tok, int64_t n_seq) { return n_tok / 64 + 2 * std::min(n_seq, n_tok); }
// A sequence's part of the batch in 64 positions from `base`, a multiple of 64: tile `index` of the sequences' tiles in
// order. s = -1: there are fewer.
struct PagedVTile {
    int s, base;
    PagedSeq q;
};
__device__ __forceinline__ PagedVTile paged_vtile(const Paged &a, int index) {
    const int lane = threadIdx.x & 63;
    int before = 0, top = 0;
    PagedVTile t;
    t.s = -1, t.base = 0, t.q = PagedSeq{};
    for (int b = 0; b < a.n_seq; b += 64) {
        const int s = b + lane;
        int own = 0, first = 0;
        PagedSeq q{};
        if (s < a.n_seq) q = paged_seq(a, s);
        paged_own_rows(a, s, q, top);
        if (s < a.n_seq) {
            first = (q.len - q.n) / 64;
            own = q.n > 0 && q.ok ? (q.len - 1) / 64 - first + 1 : 0;
        }
        int upto = own;
        for (int o = 1; o < 64; o <<= 1) {
            const int z = __shfl_up(upto, o, 64);
            if (lane >= o) upto += z;
        }
        const uint64_t m = __builtin_amdgcn_ballot_w64(before + upto > index);
        if (m) {
            const int at = __builtin_ctzll(m);
            t.s = __builtin_amdgcn_readfirstlane(b + at);
            t.base = __builtin_amdgcn_readfirstlane((__shfl(first, at, 64) + index - before - (__shfl(upto, at, 64) - __shfl(own, at, 64))) * 64);
            t.q.t0 = __builtin_amdgcn_readlane(q.t0, at), t.q.n = __builtin_amdgcn_readlane(q.n, at);
            t.q.len = __builtin_amdgcn_readlane(q.len, at), t.q.ok = true;
            return t;
        }
        before += __shfl(upto, 63, 64);
    }
    return t;
}

struct PagedRopeArgs {
    const float *qw, *kw, *factors;
    float eps;
    double log2_base, scale_turns;  // log2(freq_base), freq_scale / (2 pi)
    int n_rot, halves;
};
struct PagedStoreArgs {
    Paged p;
    PagedRopeArgs r;
    const float *q, *k, *v;
    float *qo;
    int64_t ldq, ldkv, ldo;
    int n_head;
    // set by the launch: a token's heads over `parts` workgroups of heads_part, at most v_tiles tiles of V
    int parts, heads_part, v_tiles;
};
hipError_t launch_paged_store(PagedStoreArgs &a, int num_cu, hipStream_t s);

// a slot: how many splits of its range were used (0, 1: nothing to join), its rows and where they are in the batch
struct PagedSlot {
    int32_t used, rows, t0, r0;
};
struct PagedSums {
    float *part, *stat;
    PagedSlot *info;
};
struct PagedAttnArgs {
    Paged p;
    const float *q, *slopes;
    float *o;
    const int32_t *prefix;
    int64_t ldq, ldo;
    int n_head, window;
    float scale, softcap;
    // Sequences of few rows per K / V head (new tokens x query heads of the head, at most drows) go to the decode kernel, the
    // others to the prompt kernel, prows rows a workgroup; each kernel's ranges of positions are split over up to ds / ps
    // workgroups (0: not launched). Split ranges leave their sums in part and stat, by slot (a workgroup's rows) and split, and
    // what the join has to know of a slot in info. alone: one workgroup of the prompt launch to a compute unit.
    int ds, ps, drows, prows;
    bool alone;
    PagedSums dsum, psum;
};
constexpr int PRO_ROWS = 128;  // rows of a workgroup of the prompt kernel, at most
// at most as many tiles of that many rows as a batch's sequences can have, per K / V head (G rows a token)
inline int64_t paged_tiles(int64_t n_tok, int64_t n_seq, int G, int rows) { return (n_tok * G + (rows - 1) * n_seq) / rows; }
struct PagedScratch {
    size_t dpart, ppart, drow, prow, dslot, pslot;  // floats of part, rows of stat, slots of info
    size_t bytes() const { return (dslot + pslot) * sizeof(PagedSlot) + (drow + prow) * 8 + (dpart + ppart) * 4; }
};
// the plan for a device of num_cu compute units, and the scratch it needs
PagedScratch paged_attention_plan(PagedAttnArgs &a, int num_cu);
hipError_t launch_paged_attention(const PagedAttnArgs &a, hipStream_t s);

}  // namespace fgh
