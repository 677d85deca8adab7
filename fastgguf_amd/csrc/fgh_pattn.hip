// fgh_pattn.hip - attention over the paged KV cache on gfx950: which kernel takes which sequences, and over how many
// workgroups a range of positions is split.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fgh_pattn.h"

namespace fgh {

namespace {

// Sums of split ranges added to a running (o, lr) at reference cm, U splits' loads in flight at a time: k = first, first + step, .. < used.
template <int NV, int U>
__device__ __forceinline__ void join_splits(const pf4 *part, int64_t part_step, int64_t value_step, const pf2 *stat, int64_t stat_step, int first,
                                            int step, int used, pf4 (&o)[NV], float &cm, float &lr) {
    for (int b = first; b < used; b += U * step) {
        pf4 z[U][NV];
        pf2 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = min(b + u * step, used - 1);
            w[u] = stat[k * stat_step];
#pragma unroll
            for (int i = 0; i < NV; ++i) z[u][i] = part[k * part_step + i * value_step];
        }
        float cn = cm;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (b + u * step >= used) w[u] = pf2{__FLT_MAX__, 0.0f};
            cn = fminf(cn, w[u].x);
        }
        float f = __builtin_amdgcn_exp2f(cn - cm);
        cm = cn;
        lr *= f;
#pragma unroll
        for (int i = 0; i < NV; ++i) o[i] *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            f = __builtin_amdgcn_exp2f(cm - w[u].x);
            lr += f * w[u].y;
            if (b + u * step < used)
#pragma unroll
                for (int i = 0; i < NV; ++i) o[i] += f * z[u][i];
        }
    }
}

// Decode slots, a workgroup for four rows of one: 4 values a thread, groups of threads take splits in turn. Always the
// same order of sums.
__device__ __forceinline__ void join_decode(const PagedAttnArgs &a, int slot, int part4) {
    __shared__ pf4 sum_l[256];
    __shared__ pf2 stat_l[256];
    const int nkv = a.p.n_head_kv, G = a.n_head / nkv, kvh = slot % nkv, hd = a.p.hd, tid = threadIdx.x;
    const PagedSlot in = a.dsum.info[slot];
    const int r0 = 4 * part4, rows = min(4, in.rows - r0);
    if (in.used < 2 || rows < 1) return;
    const int items = rows * (hd / 4), groups = 256 / items, g = tid / items, y = tid - g * items, r = r0 + y / (hd / 4);
    const pf4 *part = (const pf4 *)(a.dsum.part + (int64_t)slot * a.ds * a.drows * hd) + r0 * (hd / 4);
    const pf2 *stat = (const pf2 *)a.dsum.stat + (int64_t)slot * a.ds * a.drows;
    if (g < groups) {
        pf4 o[1] = {pf4{0.0f, 0.0f, 0.0f, 0.0f}};
        float cm = __FLT_MAX__, lr = 0.0f;
        join_splits<1, 16>(part + y, (int64_t)a.drows * (hd / 4), 0, stat + r, a.drows, g, groups, in.used, o, cm, lr);
        sum_l[tid] = o[0];
        stat_l[tid] = pf2{cm, lr};
    }
    __syncthreads();
    if (tid >= items) return;
    float cm = __FLT_MAX__, lr = 0.0f;
    pf4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < groups; ++i) cm = fminf(cm, stat_l[i * items + tid].x);
    for (int i = 0; i < groups; ++i) {
        const pf2 w = stat_l[i * items + tid];
        const float f = __builtin_amdgcn_exp2f(cm - w.x);
        lr += f * w.y;
        o += f * sum_l[i * items + tid];
    }
    *(pf4 *)(a.o + (in.t0 + r / G) * a.ldo + (int64_t)(kvh * G + r % G) * hd + 4 * (y - y / (hd / 4) * (hd / 4))) = o * (1.0f / lr);
}
// Prompt slots, a workgroup for 32 values of the head: the sums as the prompt kernel's lanes held them
__device__ __forceinline__ void join_prompt(const PagedAttnArgs &a, int slot, int b, int vb) {
    const int nkv = a.p.n_head_kv, G = a.n_head / nkv, kvh = slot % nkv, hd = a.p.hd;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = wave * 32 + (lane & 31);
    const PagedSlot in = a.psum.info[slot];
    if (in.used < 2 || r >= in.rows) return;
    pf4 o[4];
    for (int i = 0; i < 4; ++i) o[i] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
    float cm = __FLT_MAX__, lr = 0.0f;
    join_splits<4, 4>((const pf4 *)a.psum.part + ((int64_t)slot * a.ps * (a.prows / 32) + wave) * (vb * 4 * 64) + b * 4 * 64 + lane, (int64_t)vb * 4 * 64 * (a.prows / 32), 64,
                      (const pf2 *)a.psum.stat + (int64_t)slot * a.ps * a.prows + r, a.prows, 0, 1, in.used, o, cm, lr);
    const int row = in.r0 + r;
    float *out = a.o + (in.t0 + row / G) * a.ldo + (int64_t)(kvh * G + row % G) * hd;
    const float inv = 1.0f / lr;
    for (int i = 0; i < 4; ++i) {
        const int d = 32 * b + 8 * i + 4 * (lane >> 5);
        if (d < hd) *(pf4 *)(out + d) = o[i] * inv;
    }
}
// np workgroups of prompt slots, then those of decode slots
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, int np, int vb, int quads) {
    const int x = (int)blockIdx.x;
    if (x < np) join_prompt(a, x / vb, x % vb, vb);
    else join_decode(a, (x - np) / quads, (x - np) % quads);
}

}  // namespace

// Times here are of calls one after the other, the join with them.
// Prompt: workgroups of 128 rows, since a tile of K and V is read out of LDS once for all of them. Where they would not give
// every compute unit one in as many splits as there may be, of 64: 64 tokens behind 2000 positions, 8 heads over 4, take 34.9 us
// in 128 rows and 28.3 in 64 (bf16, hd 256), 42.0 and 29.8 (f32, hd 128); with more workgroups than that 64 rows gain nothing (32 tokens
// of each of 4 sequences behind 1000, f16: 25.4 and 25.7).
// Splits: as many as fit at once, two workgroups for every compute unit. More save nothing, and the join has its price (2032 tokens
// behind 7168, 512 tiles: 510 us whole, 513 in two splits; seven documents of up to 900 tokens, 252 tiles: 46.2 us whole, 36.8 in
// three). At least 4 units of 64 positions each, at most 8 splits: 64 tokens over 4096 positions take 27.7 us in 8, 31.3 in 16. These
// 8 are measured where they fill the device. Where a K / V head has only one or two tiles over a long range they leave compute units
// idle, and no rule for more is there yet: 3 tokens of 32 heads over 4 at 16384 positions take 54 us, 2 tokens, which are the
// decode kernel's, 18; one token of 48 heads over one 53, of 16 heads 16. Nor do the splits know how many of the tiles that a
// batch could have it has: the 64 tokens over 4096 with one token each of 63 short sequences take 105 us.
// One workgroup to a compute unit where all fit so: the dispatcher may put two on one and leave others idle (2 sequences of 64 tokens
// behind 4000, f16, 256 workgroups: 41.0 us, 34.7 so; most batches that fit take the same either way). A few too many lose a whole turn (150
// tokens behind 2000, 320 workgroups: 35 us, 43 so; 40 tokens of each of 4 behind 1000, bf16, hd 64: 16.1 and 21.4). Not where the
// sequences beside the longest have few rows, whose decode workgroups fit several (40 tokens of one sequence and one each of 63: 125
// us so, 105).
// Decode: as many as fit at once too, of 4 steps and more, a step for every wavefront (4 sequences of 3000 positions at hd 256, of
// which one workgroup fits a compute unit: 26.1 us in 256 workgroups, 33.9 in 512); up to eight for every compute
// unit where that leaves 16 steps each, since sequences' lengths differ: 32 sequences of 65 to 8192 positions take
// 141 us in 2 splits, 115 in 8, and 32 of 1024 31.5 in 2, 40.6 in 8. All sequences get as many splits, short ones leave theirs unused. At most 64: the join reads that many one after the other.
// The bounds may be far above the lengths: the kernels split what is there.
// The join is a launch of its own: a workgroup that arrives last and joins the others' sums within the same launch needs
// stores that pass the L2 caches of the XCDs, and took longer (one sequence of 4096 positions 14 to 16 us against 12.3).
PagedScratch paged_attention_plan(PagedAttnArgs &a, int num_cu) {
    const int G = a.n_head / a.p.n_head_kv;
    const int64_t most = (int64_t)a.p.max_tok * G;  // rows of a sequence and K / V head
    const int64_t heads = (int64_t)a.p.n_seq * a.p.n_head_kv;
    // positions that a sequence's rows see
    const int64_t seen = a.window > 0 && !a.prefix ? std::min<int64_t>(a.p.max_len, (int64_t)a.window + a.p.max_tok - 1) : a.p.max_len;
    PagedScratch n{0, 0, 0, 0, 0, 0};
    a.ps = a.ds = 0, a.alone = false;
    a.prows = PRO_ROWS;
    a.drows = (int)std::min<int64_t>(most, DEC_ROWS);
    if (most > DEC_ROWS) {
        const int64_t units = (seen + PRO_UNIT - 1) / PRO_UNIT + 1, splits = std::min<int64_t>(8, (units + PRO_LEAST - 1) / PRO_LEAST);
        int64_t wgs = paged_tiles(a) * a.p.n_head_kv;
        if (wgs * splits <= num_cu && pro_half(a.p.type, a.p.hd)) a.prows = PRO_ROWS / 2, wgs = paged_tiles(a) * a.p.n_head_kv;
        a.ps = (int)std::min<int64_t>(splits, std::max<int64_t>(1, (2 * (int64_t)num_cu + wgs / 2) / wgs));
        const bool mixed = (int64_t)(a.p.n_tok - a.p.max_tok) * G <= (int64_t)(a.p.n_seq - 1) * DEC_ROWS && a.p.n_seq > 1;
        // workgroups with rows, for tokens spread evenly over the sequences
        const int64_t seqs = pro_seqs(a), each = ((a.p.n_tok + seqs - 1) / seqs * G + a.prows - 1) / a.prows;
        a.alone = !mixed && std::min(paged_tiles(a), seqs * each) * a.p.n_head_kv * a.ps <= num_cu;
        if (a.ps > 1) n.pslot = (size_t)wgs, n.prow = n.pslot * a.ps * a.prows, n.ppart = n.prow * ((a.p.hd + 31) / 32 * 32);
    }
    if (a.ps == 0 || a.p.n_seq > 1) {
        const int64_t steps = seen / DEC_STEP + 1, at_once = dec_resident(a.p.type, a.p.hd) * (int64_t)num_cu;
        const int64_t even = std::min<int64_t>(at_once / heads, (steps + 3) / 4);
        const int64_t more = std::min<int64_t>(8 * (int64_t)num_cu / heads, steps / 16);
        a.ds = (int)std::min<int64_t>(64, std::max<int64_t>({1, even, more}));
        if (a.ds > 1) n.dslot = (size_t)heads, n.drow = n.dslot * a.ds * a.drows, n.dpart = n.drow * a.p.hd;
    }
    return n;
}

hipError_t launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
    const hipError_t e = a.ps > 0 ? launch_paged_prompt(a, s) : launch_paged_decode(a, s);
    if (e != hipSuccess || std::max(a.ds, a.ps) < 2) return e;
    const int vb = (a.p.hd + 31) / 32, quads = (a.drows + 3) / 4;
    const int np = a.ps > 1 ? (int)paged_tiles(a) * a.p.n_head_kv * vb : 0, nd = a.ds > 1 ? a.p.n_seq * a.p.n_head_kv * quads : 0;
    paged_join_kernel<<<np + nd, 256, 0, s>>>(a, np, vb, quads);
    return hipGetLastError();
}

}  // namespace fgh
