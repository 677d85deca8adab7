// fgh_pattn.hip - attention over the paged KV cache on gfx950.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fgh_pattn.h"

namespace fgh {

namespace {

// Sums of split ranges joined: a wavefront per row. Lane groups of hd / 4 lanes take splits in turn, 16 bytes a lane; always the
// same order. Slot `slot` of `slots`, used of its splits written; row to o.
__device__ __forceinline__ void join_row(const PagedAttnArgs &a, int64_t slot, int64_t slots, int used, float *out) {
    const int lane = threadIdx.x & 63, hd = a.p.hd;
    // at most 64 splits: lane i has split i's
    float c = __FLT_MAX__, l = 0.0f;
    if (lane < used) {
        c = a.stat[2 * (lane * slots + slot)];
        l = a.stat[2 * (lane * slots + slot) + 1];
    }
    float cm = c;
    for (int o = 1; o < 64; o <<= 1) cm = fminf(cm, __shfl_xor(cm, o, 64));
    const float f = __builtin_amdgcn_exp2f(cm - c);
    l *= f;
    for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o, 64);
    const int per = hd / 4, groups = 64 / per, g = lane / per, d = 4 * (lane - g * per);
    pf4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b = 0; b < used; b += groups) {  // uniform
        const int i = b + g;
        const float w = __shfl(f, min(i, 63), 64);
        if (g < groups && i < used) o += w * *(const pf4 *)(a.part + (i * slots + slot) * hd + d);
    }
    for (int k = 1; k < groups; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float z = __shfl(o[e], (lane + k * per) & 63, 64);
            if (g == 0) o[e] += z;
        }
    if (g == 0) *(pf4 *)(out + d) = o / l;
}

// grid (sequence x K / V head, fours of rows)
__global__ __launch_bounds__(256) void paged_join_decode_kernel(PagedAttnArgs a) {
    const int nkv = a.p.n_head_kv, G = a.n_head / nkv, s = blockIdx.x / nkv, kvh = blockIdx.x - s * nkv;
    const int r = __builtin_amdgcn_readfirstlane((int)blockIdx.y * 4 + (threadIdx.x >> 6));
    const PagedSeq q = paged_seq(a.p, s);
    if (!q.ok || (int64_t)q.n * G > DEC_ROWS || r >= q.n * G) return;
    const int used = paged_chunk(dec_steps(paged_span(a, q, paged_prefix(a, s, q), 0, q.n - 1)), a.ds, DEC_LEAST).used;
    if (used == 1) return;
    join_row(a, (int64_t)blockIdx.x * a.drows + r, (int64_t)gridDim.x * a.drows, used,
             a.o + (q.t0 + r / G) * a.ldo + (int64_t)(kvh * G + r % G) * a.p.hd);
}
// grid (tile x K / V head, eights of rows): each wavefront two rows
__global__ __launch_bounds__(256) void paged_join_prompt_kernel(PagedAttnArgs a) {
    const int nkv = a.p.n_head_kv, G = a.n_head / nkv, kvh = blockIdx.x % nkv;
    const PagedTile t = paged_tile(a, blockIdx.x / nkv);
    if (t.s < 0 || !t.q.ok) return;
    const int R = min(PRO_ROWS, t.q.n * G - t.r0);
    const int used = paged_chunk(pro_units(paged_span(a, t.q, paged_prefix(a, t.s, t.q), t.r0 / G, (t.r0 + R - 1) / G)), a.ps, PRO_LEAST).used;
    if (used == 1) return;
    for (int k = 0; k < 2; ++k) {
        const int r = __builtin_amdgcn_readfirstlane((int)blockIdx.y * 8 + k * 4 + (threadIdx.x >> 6));
        if (r >= R) return;
        const int row = t.r0 + r;
        join_row(a, (int64_t)blockIdx.x * PRO_ROWS + r, (int64_t)gridDim.x * PRO_ROWS, used,
                 a.o + (t.q.t0 + row / G) * a.ldo + (int64_t)(kvh * G + row % G) * a.p.hd);
    }
}

}  // namespace

// Splits: workgroups for every compute unit eight times over (sequences' lengths differ, and the bounds may be far above
// them: the kernels split what is there), at most 64 (a lane each in the join), at least 128 positions each.
size_t paged_attention_plan(PagedAttnArgs &a, int num_cu) {
    const int G = a.n_head / a.p.n_head_kv;
    const int64_t most = (int64_t)a.p.max_tok * G;  // rows of a sequence and K / V head
    const int64_t heads = (int64_t)a.p.n_seq * a.p.n_head_kv;
    a.ps = 0;
    a.ds = 0;
    a.drows = (int)std::min<int64_t>(most, DEC_ROWS);
    const int units = (a.p.max_len + PRO_UNIT - 1) / PRO_UNIT;
    size_t slots = 0;
    if (most > DEC_ROWS) {
        const int64_t wgs = paged_tiles(a) * a.p.n_head_kv;
        a.ps = (int)std::min<int64_t>({64, std::max<int64_t>(1, 2 * (int64_t)num_cu / wgs), units});
        if (a.ps > 1) slots = (size_t)a.ps * wgs * PRO_ROWS;
    }
    if (a.ps == 0 || a.p.n_seq > 1) {
        const int64_t want = std::max<int64_t>(1, 8 * (int64_t)num_cu / heads);
        a.ds = (int)std::min<int64_t>({64, want, (a.p.max_len + DEC_STEP * DEC_LEAST - 1) / (DEC_STEP * DEC_LEAST)});
        if (a.ds > 1) slots = std::max(slots, (size_t)a.ds * heads * a.drows);
    }
    return slots;
}

// the decode kernel's sums are joined before the prompt kernel's take their place
hipError_t launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (a.ds > 0 && (e = launch_paged_decode(a, s)) != hipSuccess) return e;
    if (a.ds > 1) {
        paged_join_decode_kernel<<<dim3((unsigned)a.p.n_seq * (unsigned)a.p.n_head_kv, (unsigned)(a.drows + 3) / 4), 256, 0, s>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (a.ps > 0 && (e = launch_paged_prompt(a, s)) != hipSuccess) return e;
    if (a.ps > 1) {
        paged_join_prompt_kernel<<<dim3((unsigned)(paged_tiles(a) * a.p.n_head_kv), PRO_ROWS / 8), 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace fgh
