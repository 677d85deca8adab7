// fgh_reserve.hip - the pages and rows of a batch on gfx950: what each sequence's table gains or gives back, and where each row is.
//
// With P positions a page, a sequence that keeps k positions and adds n holds ceil((k + n) / P) pages after the call. Pages given
// back go to the end of the ring of free pages in the sequences' order, pages taken come from its front, where the
// given ones stand last. Who gets pages is a matter of sums over the sequences before: an exclusive scan of pages taken,
// pages given and rows asked for, a second one of the rows granted.
//
// A step's bytes are few (32 sequences: 1 KB; 4100 of them with 96000 pages and 60000 rows: 2 MB): what it takes is launches and loads that wait for
// each other: 4 to 6 us in one launch; in two, 2 to 3 us more for up to 1024 sequences (the kernels alone 4.7 and 3.3 to
// 3.9), and 14 for the 4100.
#include "fgh_serve.h"

#include <algorithm>

namespace fgh {

namespace {

// what the rows and pages are found by: [n_seq + 1] sums of pages taken, pages given and rows granted before a sequence, and
// of each sequence its pages before, its pages after and the positions it keeps
struct Sums {
    int32_t *take, *give, *row, *held, *want, *keep;
};
constexpr int SUMS = 6;
__device__ __forceinline__ Sums sums_at(int32_t *p, int n) {
    return Sums{p, p + (n + 1), p + 2 * (n + 1), p + 3 * (n + 1), p + 4 * (n + 1), p + 5 * (n + 1)};
}

// the ring's first entry and its number of entries; broken ones are an empty ring
__device__ __forceinline__ int2 ring_of(const ReserveArgs &a) {
    const int f = a.free[0], c = a.free[1];
    const bool ok = (uint32_t)f < (uint32_t)a.n_pages && c >= 0 && c <= a.n_pages;
    return ok ? int2{f, c} : int2{0, 0};
}
__device__ __forceinline__ int ring_at(const ReserveArgs &a, int first, int64_t k) {  // k < 2 n_pages
    int64_t i = first + k;
    if (i >= a.n_pages) i -= a.n_pages;
    return (int)(i >= a.n_pages ? i - a.n_pages : i);
}

struct Ask {
    int keep, add, held, want;
    bool fine, asks;
};
__device__ __forceinline__ Ask ask_of(const ReserveArgs &a, int s) {
    Ask q;
    q.keep = a.keep[s], q.add = a.add[s], q.held = a.held[s];
    const int P = 1 << a.shift;
    q.fine = q.keep >= 0 && q.held >= 0 && q.held <= a.table_stride && q.keep <= (int64_t)q.held * P;
    q.asks = q.fine && q.add >= 0 && q.add <= a.max_tok && (int64_t)q.keep + q.add <= a.max_len;
    q.want = q.asks ? (int)(((int64_t)q.keep + q.add + P - 1) >> a.shift) : q.fine ? (int)(((int64_t)q.keep + P - 1) >> a.shift) : q.held;
    return q;
}

// Sums of numbers that are not negative, kept at 2^32 - 1 where they would pass it: one instruction, in any order the same. What is
// compared with them is below that.
__device__ __forceinline__ uint32_t add(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }
// over each row of 16 lanes: the sum with the lanes before
__device__ __forceinline__ uint32_t scan_row(uint32_t v) {
    v = add(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true));  // row_shr 1, 2, 4, 8; 0 from before the row
    v = add(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true));
    v = add(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true));
    return add(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true));
}
// the same over a wavefront
__device__ __forceinline__ uint32_t scan_wave(uint32_t v) {
    const int lane = threadIdx.x & 63;
    v = scan_row(v);
    const uint32_t a = __builtin_amdgcn_readlane(v, 15), b = __builtin_amdgcn_readlane(v, 31), c = __builtin_amdgcn_readlane(v, 47);
    const uint32_t ab = add(a, b), abc = add(ab, c);
    return add(v, lane < 16 ? 0u : lane < 32 ? a : lane < 48 ? ab : abc);
}
// N sums over the workgroup's wavefronts before this one (v: a wavefront's, the same in its lanes), and of all in `all`: a row of lanes to each
template <int THREADS, int N>
__device__ __forceinline__ void scan_waves(uint32_t (&v)[N], uint32_t (&all)[N], uint32_t (*lds)[16]) {
    constexpr int W = THREADS / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane == 0) lds[i][wave] = v[i];
    __syncthreads();
    static_assert(N <= 4 && W <= 16);
    const uint32_t w = scan_row(lane >> 4 < N && (lane & 15) < W ? lds[lane >> 4][lane & 15] : 0u);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        all[i] = __builtin_amdgcn_readlane(w, 16 * i + W - 1);
        v[i] = wave ? (uint32_t)__builtin_amdgcn_readlane(w, 16 * i + wave - 1) : 0u;
    }
    __syncthreads();
}

// The scans, by one workgroup: a wavefront has C times 64 sequences in a row, 64 at a time, and goes over them in turns of C times 64 a
// wavefront where there are more. Writes tok, len, held_out, free_out and the sums. A sequence's inputs are read before an output that
// may be the same memory is written; with several turns, what is given in all, which every grant depends on, is summed first.
template <int THREADS, int C>
__device__ __forceinline__ void reserve_scan(const ReserveArgs &a, Sums z) {
    __shared__ uint32_t lds[3][16], lds2[2][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int2 ring = ring_of(a);
    auto more = [](const Ask &q) { return (uint32_t)max(q.want - q.held, 0); };
    auto less = [](const Ask &q) { return q.fine ? (uint32_t)max(q.held - q.want, 0) : 0u; };
    // the sum with the lanes before and with `carry`, which becomes the sum with all lanes
    auto scan = [](uint32_t v, uint32_t &carry) {
        const uint32_t r = add(scan_wave(v), carry);
        carry = __builtin_amdgcn_readlane(r, 63);
        return r;
    };
    uint32_t gives = 0;
    const bool once = a.n_seq <= THREADS * C;
    if (!once) {
        for (int s = threadIdx.x; s < a.n_seq; s += THREADS) gives = add(gives, less(ask_of(a, s)));
        uint32_t v[1] = {0}, all[1];
        (void)scan(gives, v[0]);
        scan_waves<THREADS, 1>(v, all, lds);
        gives = all[0];
    }
    uint32_t take0 = 0, give0 = 0, wish0 = 0, row0 = 0, got0 = 0;  // of the turns before
    for (int first = 0; first < a.n_seq; first += THREADS * C) {
        const int s0 = first + wave * 64 * C + lane;
        Ask q[C];
        uint32_t take[C], give[C], wish[C], row[C], got[C];  // with the lane's own, from the wavefront's first on; give without
#pragma unroll
        for (int i = 0; i < C; ++i) q[i] = ask_of(a, min(s0 + 64 * i, a.n_seq - 1));
        uint32_t before[3] = {0, 0, 0}, all[3];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if (s0 + 64 * i >= a.n_seq) q[i].fine = q[i].asks = false, q[i].want = q[i].held = q[i].add = 0;
            take[i] = scan(more(q[i]), before[0]);
            const uint32_t carry = before[1], g = scan(less(q[i]), before[1]), up = (uint32_t)__shfl_up((int)g, 1, 64);
            give[i] = lane ? up : carry;  // what is kept at 2^32 - 1, less the own part, would be too small
            wish[i] = scan(q[i].asks ? (uint32_t)q[i].add : 0u, before[2]);
        }
        scan_waves<THREADS, 3>(before, all, lds);  // its barriers stand between ring_of and the write of free_out
        if (once) gives = all[1];
        const uint32_t avail = min(add(ring.y, gives), (uint32_t)INT32_MAX);
        bool ok[C];
        uint32_t mine[2] = {0, 0}, sum[2];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const uint32_t t = add(add(take[i], before[0]), take0), w = add(add(wish[i], before[2]), wish0);
            ok[i] = q[i].asks && (more(q[i]) == 0 || t <= avail) && (q[i].add == 0 || w <= (uint32_t)a.n_tok);
            row[i] = scan(ok[i] ? (uint32_t)q[i].add : 0u, mine[0]);  // at most n_tok and avail in all
            got[i] = scan(ok[i] ? more(q[i]) : 0u, mine[1]);
        }
        scan_waves<THREADS, 2>(mine, sum, lds2);
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int s = s0 + 64 * i, rows = ok[i] ? q[i].add : 0, plus = ok[i] ? (int)more(q[i]) : 0;
            if (s >= a.n_seq) break;
            const int r = (int)(row0 + mine[0] + row[i]) - rows;
            z.take[s] = (int)(got0 + mine[1] + got[i]) - plus, z.give[s] = (int)min(add(add(give[i], before[1]), give0), (uint32_t)INT32_MAX);
            z.row[s] = r, z.held[s] = q[i].held, z.want[s] = q[i].want, z.keep[s] = q[i].keep;
            if (blockIdx.x) continue;
            a.tok[s] = r;
            a.len[s] = q[i].fine ? q[i].keep + rows : 0;
            a.held_out[s] = q[i].held + plus - (int)less(q[i]);
        }
        take0 = add(take0, all[0]), give0 = add(give0, all[1]), wish0 = add(wish0, all[2]), row0 += sum[0], got0 += sum[1];
    }
    if (threadIdx.x == 0) {
        const int n = a.n_seq;
        z.take[n] = (int)got0, z.give[n] = (int)min(gives, (uint32_t)INT32_MAX), z.row[n] = (int)row0, z.held[n] = ring.x, z.want[n] = ring.y;  // the ring as it was
        if (blockIdx.x) return;
        a.tok[n] = (int)row0;
        a.free_out[0] = ring_at(a, ring.x, got0 % (uint32_t)a.n_pages);
        a.free_out[1] = (int)min((int64_t)a.n_pages, (int64_t)ring.y + gives - got0);
    }
}

// the last s with sum[s] <= k: for k < sum[n] the one whose own part holds k
__device__ __forceinline__ int find(const int32_t *sum, int n, int k) {
    int lo = 0, hi = n;  // sum[lo] <= k < sum[hi]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (sum[m] <= k) lo = m;
        else hi = m;
    }
    return lo;
}

struct Pages {
    const ReserveArgs &a;
    const Sums &z;
    int first, count;  // the ring as it was
    __device__ __forceinline__ Pages(const ReserveArgs &a, const Sums &z) : a(a), z(z), first(z.held[a.n_seq]), count(z.want[a.n_seq]) {}
    __device__ __forceinline__ int given(int k) const {  // the k-th page that is given back
        const int s = find(z.give, a.n_seq, k);
        return a.table[(int64_t)s * a.table_stride + z.want[s] + (k - z.give[s])];
    }
    __device__ __forceinline__ int taken(int k) const { return k < count ? a.queue[ring_at(a, first, k)] : given(k - count); }
    // a ring that would hold more pages than there are (pages given twice) takes no more of them: what is read from it is not written
    __device__ __forceinline__ void give(int k, int page) const {
        if (k < a.n_pages - count) a.queue[ring_at(a, first, (int64_t)count + k)] = page;
    }
};
// the maps of row r, of sequence s (-1: none)
__device__ __forceinline__ void map_row(const ReserveArgs &a, const Sums &z, const Pages &p, int r, int s) {
    int pos = -1;
    int64_t slot = -1;
    if (s >= 0) {
        pos = z.keep[s] + (r - z.row[s]);
        const int i = pos >> a.shift, page = !a.slot ? -1 : i < z.held[s] ? a.table[(int64_t)s * a.table_stride + i] : p.taken(z.take[s] + i - z.held[s]);
        if ((uint32_t)page < (uint32_t)a.n_pages) slot = ((int64_t)page << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    if (a.seq) a.seq[r] = s;
    if (a.pos) a.pos[r] = pos;
    if (a.slot) a.slot[r] = slot;
}
// The pages that change hands, and the rows' maps, with the sums in LDS: each finds its sequence by halves. Where they are few each of the three has
// wavefronts of its own.
__device__ __forceinline__ void reserve_fill(const ReserveArgs &a, const Sums &z, int thread, int threads) {
    const int n = a.n_seq, gives = min(z.give[n], a.n_pages), takes = z.take[n], total = z.row[n];
    const Pages p(a, z);
    for (int k = thread; k < gives; k += threads) p.give(k, p.given(k));
    for (int k = (thread + 64) % threads; k < takes; k += threads) {
        const int s = find(z.take, n, k);
        a.table[(int64_t)s * a.table_stride + z.held[s] + (k - z.take[s])] = p.taken(k);
    }
    if (a.seq || a.pos || a.slot)
        for (int r = (thread + 128) % threads; r < a.n_tok; r += threads) map_row(a, z, p, r, r < total ? find(z.row, n, r) : -1);
}

// All of it in one launch, the sums in LDS: each workgroup makes them for itself, the first one writes what is not pages or rows (kernel alone: 3.8 us
// for 32 sequences, 6.0 for 250 with 11000 rows in 11 workgroups, 5.1 for prompts of 20000 rows in 20)
template <int THREADS>
__global__ __launch_bounds__(THREADS) void reserve_kernel(ReserveArgs a) {
    extern __shared__ int32_t sums[];
    const Sums z = sums_at(sums, a.n_seq);
    reserve_scan<THREADS, 1>(a, z);
    __syncthreads();
    reserve_fill(a, z, blockIdx.x * THREADS + threadIdx.x, gridDim.x * THREADS);
}

template <int C>
__global__ __launch_bounds__(1024) void reserve_scan_kernel(ReserveArgs a) { reserve_scan<1024, C>(a, sums_at(a.pre, a.n_seq)); }

// The same by many, the sums in memory: a wavefront to each sequence for its pages, and to 64 rows, of which the first is looked for and the
// others counted on from there. (By halves, a row's 12 steps in 4096 sequences wait for each other: 11 us instead of 5 for 96000 pages and 60000 rows.)
__global__ __launch_bounds__(256) void reserve_fill_kernel(ReserveArgs a, int row_groups) {
    __shared__ int marks[256];
    const Sums z = sums_at(a.pre, a.n_seq);
    const Pages p(a, z);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x >= row_groups) {
        const int s = ((int)blockIdx.x - row_groups) * 4 + wave;
        if (s >= a.n_seq) return;
        const int g0 = z.give[s], gives = min(z.give[s + 1] - g0, a.n_pages), t0 = z.take[s], takes = z.take[s + 1] - t0;
        const int64_t row = (int64_t)s * a.table_stride;
        if (gives > 0) {
            const int32_t *from = a.table + row + z.want[s];
            for (int k = lane; k < gives; k += 64) p.give(g0 + k, from[k]);
        }
        if (takes > 0) {
            int32_t *to = a.table + row + z.held[s];
            for (int k = lane; k < takes; k += 64) to[k] = p.taken(t0 + k);
        }
        return;
    }
    int *mark = marks + 64 * wave;
    const int base = (int)(blockIdx.x * 256) + 64 * wave, r = base + lane, total = z.row[a.n_seq];
    int own = -1;
    if (base < total) {
        mark[lane] = 0;
        __builtin_amdgcn_wave_barrier();  // LDS serves a wavefront in order: only the compiler must keep it
        const int top = min(base + 64, total);
        for (int b = max(seq_of_row(z.row, a.n_seq, base), 0); b < a.n_seq; b += 64) {
            const int s = min(b + lane, a.n_seq - 1), from = max(z.row[s], base), to = min(z.row[s + 1], top);
            if (b + lane < a.n_seq && from < to) mark[from - base] = s + 1;
            if (__builtin_amdgcn_ballot_w64(b + lane >= a.n_seq || to >= top)) break;
        }
        __builtin_amdgcn_wave_barrier();
        const int m = mark[lane];
        const uint64_t starts = __builtin_amdgcn_ballot_w64(m != 0), mine = starts & (~0ull >> (63 - lane));
        const int first = __shfl(m, 63 - __builtin_clzll(mine | 1), 64);
        own = r < total ? first - 1 : -1;
    }
    if (r < a.n_tok) map_row(a, z, p, r, own);
}

// The workgroups of the one launch, 0 for two. Up to 1024 sequences: one workgroup for few rows and pages, more only where no output is an
// input's memory, which others might still read (20000 rows: 5.2 us, in two launches 7.6).
int at_once(const ReserveArgs &a) {
    if (a.n_seq > 1024) return 0;
    const int64_t pages = std::min<int64_t>(a.n_pages, (int64_t)a.n_seq * a.table_stride);  // that could change hands: few do
    if (a.n_tok <= 4096 && pages <= 1 << 17) return 1;
    if (a.held == a.held_out || a.free == a.free_out || a.keep == a.len) return 0;
    return (int)std::min<int64_t>(128, std::max<int64_t>((a.n_tok + 1023) / 1024, pages / 8192));
}

}  // namespace

size_t reserve_scratch(const ReserveArgs &a) { return at_once(a) ? 0 : (size_t)(a.n_seq + 1) * SUMS * 4; }

hipError_t launch_reserve(const ReserveArgs &a, hipStream_t s) {
    if (const int groups = at_once(a)) {
        const size_t lds = (size_t)(a.n_seq + 1) * SUMS * 4;
        if (a.n_seq <= 256 && a.n_tok <= 512) reserve_kernel<256><<<groups, 256, lds, s>>>(a);
        else reserve_kernel<1024><<<groups, 1024, lds, s>>>(a);
        return hipGetLastError();
    }
    if (a.n_seq <= 1024) reserve_scan_kernel<1><<<1, 1024, 0, s>>>(a);
    else if (a.n_seq <= 2048) reserve_scan_kernel<2><<<1, 1024, 0, s>>>(a);
    else reserve_scan_kernel<5><<<1, 1024, 0, s>>>(a);
    const int row_groups = a.seq || a.pos || a.slot ? (a.n_tok + 255) / 256 : 0;
    reserve_fill_kernel<<<(unsigned)(row_groups + (a.n_seq + 3) / 4), 256, 0, s>>>(a, row_groups);
    return hipGetLastError();
}

}  // namespace fgh
