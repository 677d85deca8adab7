// fgh_pattn.hip - attention over the paged KV cache on gfx950: which kernel takes which sequences, and over how many
// workgroups a range of positions is split.
#include <hip/hip_runtime.h>

#include <stdlib.h>

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

// Decode slots, a workgroup each: 4 values a thread; where rows are few, groups of threads take splits in turn. Always the same
// order of sums.
__global__ __launch_bounds__(256) void paged_join_decode_kernel(PagedAttnArgs a) {
    __shared__ pf4 sum_l[256];
    __shared__ pf2 stat_l[256];
    const int slot = blockIdx.x, nkv = a.p.n_head_kv, G = a.n_head / nkv, kvh = slot % nkv, hd = a.p.hd, tid = threadIdx.x;
    const PagedSlot in = a.info[slot];
    if (in.used < 2) return;
    const int items = in.rows * (hd / 4), groups = max(1, 256 / items);
    const pf4 *part = (const pf4 *)(a.part + (int64_t)slot * a.ds * a.drows * hd);
    const pf2 *stat = (const pf2 *)a.stat + (int64_t)slot * a.ds * a.drows;
    auto out = [&](int r, int d) { return (pf4 *)(a.o + (in.t0 + r / G) * a.ldo + (int64_t)(kvh * G + r % G) * hd + d); };
    for (int x = tid; x < items * groups; x += 256) {
        const int g = x / items, y = x - g * items, r = y / (hd / 4);
        pf4 o[1] = {pf4{0.0f, 0.0f, 0.0f, 0.0f}};
        float cm = __FLT_MAX__, lr = 0.0f;
        join_splits<1, 16>(part + y, (int64_t)a.drows * (hd / 4), 0, stat + r, a.drows, g, groups, in.used, o, cm, lr);
        if (groups == 1) *out(r, 4 * (y - r * (hd / 4))) = o[0] * (1.0f / lr);
        else {
            sum_l[x] = o[0];
            stat_l[x] = pf2{cm, lr};
        }
    }
    if (groups == 1) return;
    __syncthreads();
    if (tid < items) {
        const int r = tid / (hd / 4);
        float cm = __FLT_MAX__, lr = 0.0f;
        pf4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int g = 0; g < groups; ++g) cm = fminf(cm, stat_l[g * items + tid].x);
        for (int g = 0; g < groups; ++g) {
            const pf2 w = stat_l[g * items + tid];
            const float f = __builtin_amdgcn_exp2f(cm - w.x);
            lr += f * w.y;
            o += f * sum_l[g * items + tid];
        }
        *out(r, 4 * (tid - r * (hd / 4))) = o * (1.0f / lr);
    }
}
// Prompt slots, grid (slots, 32 values of the head): the sums as the prompt kernel's lanes held them
__global__ __launch_bounds__(256) void paged_join_prompt_kernel(PagedAttnArgs a) {
    const int slot = blockIdx.x, b = blockIdx.y, nkv = a.p.n_head_kv, G = a.n_head / nkv, kvh = slot % nkv, hd = a.p.hd;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = wave * 32 + (lane & 31), vb = gridDim.y;
    const PagedSlot in = a.info[slot];
    if (in.used < 2 || r >= in.rows) return;
    pf4 o[4];
    for (int i = 0; i < 4; ++i) o[i] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
    float cm = __FLT_MAX__, lr = 0.0f;
    join_splits<4, 4>((const pf4 *)a.part + ((int64_t)slot * a.ps * 4 + wave) * (vb * 4 * 64) + b * 4 * 64 + lane, (int64_t)vb * 4 * 64 * 4, 64,
                      (const pf2 *)a.stat + (int64_t)slot * a.ps * PRO_ROWS + r, PRO_ROWS, 0, 1, in.used, o, cm, lr);
    const int row = in.r0 + r;
    float *out = a.o + (in.t0 + row / G) * a.ldo + (int64_t)(kvh * G + row % G) * hd;
    const float inv = 1.0f / lr;
    for (int i = 0; i < 4; ++i) {
        const int d = 32 * b + 8 * i + 4 * (lane >> 5);
        if (d < hd) *(pf4 *)(out + d) = o[i] * inv;
    }
}

}  // namespace

// Decode: workgroups for every compute unit twice over (what fits at once), of 4 steps and more each, a step for every
// wavefront; up to eight times over where that leaves 16 steps each, since sequences' lengths differ. The kernels
// split what is there of a range: bounds may be far above it. At most 64 splits, which is what the join's factors hold.
// Prompt:
PagedScratch paged_attention_plan(PagedAttnArgs &a, int num_cu) {
    static const int PX = getenv("PG_PX") ? atoi(getenv("PG_PX")) : 2, PL = getenv("PG_PL") ? atoi(getenv("PG_PL")) : 4, PM = getenv("PG_PM") ? atoi(getenv("PG_PM")) : 8;  // TEMPORARY
    const int G = a.n_head / a.p.n_head_kv;
    const int64_t most = (int64_t)a.p.max_tok * G;  // rows of a sequence and K / V head
    const int64_t heads = (int64_t)a.p.n_seq * a.p.n_head_kv;
    // positions that a sequence's rows see
    const int64_t seen = a.window > 0 && !a.prefix ? std::min<int64_t>(a.p.max_len, (int64_t)a.window + a.p.max_tok - 1) : a.p.max_len;
    PagedScratch n{0, 0, 0};
    a.ps = a.ds = 0;
    a.dleast = 4, a.pleast = PL;
    a.drows = (int)std::min<int64_t>(most, DEC_ROWS);
    if (most > DEC_ROWS) {
        const int64_t wgs = paged_tiles(a) * a.p.n_head_kv, units = (seen + PRO_ROWS + PRO_UNIT - 1) / PRO_UNIT;
        a.ps = (int)std::min<int64_t>({PM, std::max<int64_t>(1, PX * (int64_t)num_cu / wgs), (units + a.pleast - 1) / a.pleast});
        if (a.ps > 1) n = PagedScratch{(size_t)(a.ps * wgs) * PRO_ROWS * ((a.p.hd + 31) / 32 * 32), (size_t)(a.ps * wgs) * PRO_ROWS * 2, (size_t)wgs};
    }
    if (a.ps == 0 || a.p.n_seq > 1) {
        const int64_t steps = seen / DEC_STEP + 1;
        const int64_t even = std::min<int64_t>(2 * (int64_t)num_cu / heads, (steps + 3) / 4), more = std::min<int64_t>(8 * (int64_t)num_cu / heads, steps / 16);
        a.ds = (int)std::min<int64_t>(64, std::max<int64_t>({1, even, more}));
        if (a.ds > 1) {
            const size_t rows = (size_t)a.ds * heads * a.drows;
            n = PagedScratch{std::max(n.part, rows * a.p.hd), std::max(n.stat, rows * 2), std::max(n.info, (size_t)heads)};
        }
    }
    return n;
}

// both kernels use the same scratch, one after the other
hipError_t launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (a.ds > 0 && (e = launch_paged_decode(a, s)) != hipSuccess) return e;
    if (a.ds > 1) {
        paged_join_decode_kernel<<<(unsigned)a.p.n_seq * (unsigned)a.p.n_head_kv, 256, 0, s>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (a.ps > 0 && (e = launch_paged_prompt(a, s)) != hipSuccess) return e;
    if (a.ps > 1) {
        paged_join_prompt_kernel<<<dim3((unsigned)(paged_tiles(a) * a.p.n_head_kv), (unsigned)(a.p.hd + 31) / 32), 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace fgh
