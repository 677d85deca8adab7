// fgh_reserve.hip - the pages and rows of a batch on gfx950: what each sequence's table gains or gives back, and where each row is.
//
// With P positions a page, a sequence that keeps k positions and adds n holds ceil((k + n) / P) pages after the call. Pages given
// back go to the end of the ring of free pages in the sequences' order, pages taken come from its front, where the
// given ones stand last. Who gets pages is a matter of sums over the sequences before: an exclusive scan of pages taken,
// pages given and rows asked for, a second one of the rows granted.
#include "fgh_serve.h"

#include <algorithm>

namespace fgh {

namespace {

constexpr int THREADS = 1024;

// what the rows and pages are found by: [n_seq + 1] sums of pages taken, pages given and rows granted before a sequence, and
// of each sequence its pages before, its pages after and the positions it keeps
struct Sums {
    int32_t *take, *give, *row, *held, *want, *keep;
};
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

// sums over the workgroup's threads before this one, and of all in `all`
template <int N>
__device__ __forceinline__ void scan_block(int64_t (&v)[N], int64_t (&all)[N], int64_t (*lds)[N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t upto[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        upto[i] = v[i];
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t z = __shfl_up(upto[i], o, 64);
            if (lane >= o) upto[i] += z;
        }
        if (lane == 63) lds[wave][i] = upto[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        int64_t before = 0, total = 0;
        for (int w = 0; w < THREADS / 64; ++w) {
            if (w < wave) before += lds[w][i];
            total += lds[w][i];
        }
        v[i] = before + upto[i] - v[i];
        all[i] = total;
    }
    __syncthreads();
}

__device__ __forceinline__ int32_t clip(int64_t v) { return (int32_t)min(v, (int64_t)INT32_MAX); }

// The scans, by one workgroup: a thread has `per` sequences in a row. Writes tok, len, held_out, free_out and the sums. Every
// input of a thread's sequences is read before an output that may be the same memory is written.
__device__ __forceinline__ void reserve_scan(const ReserveArgs &a, Sums z) {
    __shared__ int64_t lds[THREADS / 64][3];
    const int per = (a.n_seq + THREADS - 1) / THREADS, s0 = min(a.n_seq, (int)threadIdx.x * per), s1 = min(a.n_seq, s0 + per);
    const int2 ring = ring_of(a);
    int64_t before[3] = {0, 0, 0}, all[3];
    for (int s = s0; s < s1; ++s) {
        const Ask q = ask_of(a, s);
        before[0] += max(q.want - q.held, 0);
        before[1] += max(q.held - q.want, 0);
        before[2] += q.asks ? q.add : 0;
    }
    scan_block<3>(before, all, lds);  // its barriers stand between ring_of and the write of free_out
    const int64_t avail = ring.y + all[1];
    auto grant = [&](const Ask &q, int64_t take, int64_t rows) {  // sums with this sequence
        return q.asks && (q.want <= q.held || take <= avail) && (q.add == 0 || rows <= a.n_tok);
    };
    int64_t sub[2] = {0, 0}, got[2], take = before[0], rows = before[2];
    for (int s = s0; s < s1; ++s) {
        const Ask q = ask_of(a, s);
        take += max(q.want - q.held, 0);
        rows += q.asks ? q.add : 0;
        if (!grant(q, take, rows)) continue;
        sub[0] += q.add;
        sub[1] += max(q.want - q.held, 0);
    }
    int64_t pair[2] = {sub[0], sub[1]};
    {
        __shared__ int64_t lds2[THREADS / 64][2];
        scan_block<2>(pair, got, lds2);
    }
    int64_t row = pair[0], taken = pair[1], given = before[1];
    take = before[0], rows = before[2];
    for (int s = s0; s < s1; ++s) {
        const Ask q = ask_of(a, s);
        take += max(q.want - q.held, 0);
        rows += q.asks ? q.add : 0;
        const bool ok = grant(q, take, rows);
        const int more = ok ? max(q.want - q.held, 0) : 0, less = max(q.held - q.want, 0);
        z.take[s] = (int)taken, z.give[s] = clip(given), z.row[s] = (int)row, z.held[s] = q.held, z.want[s] = q.want, z.keep[s] = q.keep;
        a.tok[s] = (int)row;
        a.len[s] = q.fine ? q.keep + (ok ? q.add : 0) : 0;
        a.held_out[s] = q.held + more - less;
        taken += more, given += less, row += ok ? q.add : 0;
    }
    if (threadIdx.x == 0) {
        z.take[a.n_seq] = (int)got[1], z.give[a.n_seq] = clip(all[1]), z.row[a.n_seq] = (int)got[0];
        z.held[a.n_seq] = ring.x, z.want[a.n_seq] = ring.y;  // the ring as it was
        a.tok[a.n_seq] = (int)got[0];
        a.free_out[0] = ring_at(a, ring.x, got[1] % a.n_pages);
        a.free_out[1] = (int)min((int64_t)a.n_pages, ring.y + all[1] - got[1]);
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

// The pages that change hands, and the rows' maps, by `threads` threads.
__device__ __forceinline__ void reserve_fill(const ReserveArgs &a, Sums z, int thread, int threads) {
    const int n = a.n_seq, first = z.held[n], count = z.want[n];
    const int gives = min(z.give[n], a.n_pages), takes = z.take[n];
    auto given = [&](int k) {  // the k-th page that is given back
        const int s = find(z.give, n, k);
        return a.table[(int64_t)s * a.table_stride + z.want[s] + (k - z.give[s])];
    };
    auto taken = [&](int k) { return k < count ? a.queue[ring_at(a, first, k)] : given(k - count); };
    // a ring that would hold more pages than there are (pages given twice) takes no more of them: what is read from it is not written
    for (int k = thread; k < gives && k < a.n_pages - count; k += threads) a.queue[ring_at(a, first, (int64_t)count + k)] = given(k);
    for (int k = thread; k < takes; k += threads) {
        const int s = find(z.take, n, k);
        a.table[(int64_t)s * a.table_stride + z.held[s] + (k - z.take[s])] = taken(k);
    }
    if (!a.seq && !a.pos && !a.slot) return;
    const int total = z.row[n], P = 1 << a.shift;
    for (int r = thread; r < a.n_tok; r += threads) {
        int s = -1, pos = -1;
        int64_t slot = -1;
        if (r < total) {
            s = find(z.row, n, r);
            pos = z.keep[s] + (r - z.row[s]);
            const int i = pos >> a.shift, page = !a.slot ? 0 : i < z.held[s] ? a.table[(int64_t)s * a.table_stride + i] : taken(z.take[s] + i - z.held[s]);
            if ((uint32_t)page < (uint32_t)a.n_pages) slot = ((int64_t)page << a.shift) + (pos & (P - 1));
        }
        if (a.seq) a.seq[r] = s;
        if (a.pos) a.pos[r] = pos;
        if (a.slot) a.slot[r] = slot;
    }
}

__global__ __launch_bounds__(THREADS) void reserve_scan_kernel(ReserveArgs a) { reserve_scan(a, sums_at(a.pre, a.n_seq)); }

__global__ __launch_bounds__(256) void reserve_fill_kernel(ReserveArgs a) {
    reserve_fill(a, sums_at(a.pre, a.n_seq), blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

}  // namespace

size_t reserve_scratch(const ReserveArgs &a) { return (size_t)(a.n_seq + 1) * 6 * 4; }

hipError_t launch_reserve(const ReserveArgs &a, int num_cu, hipStream_t s) {
    reserve_scan_kernel<<<1, THREADS, 0, s>>>(a);
    const int64_t items = std::max<int64_t>(a.n_tok, std::min<int64_t>(a.n_pages, (int64_t)a.n_seq * a.table_stride));
    reserve_fill_kernel<<<(unsigned)std::min<int64_t>((items + 255) / 256, 4 * num_cu), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace fgh
