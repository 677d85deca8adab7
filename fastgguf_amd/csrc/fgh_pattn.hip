// fgh_pattn.hip - attention over the paged KV cache on gfx950.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fgh_pattn.h"

namespace fgh {

namespace {

__device__ __forceinline__ float paged_get(const uint8_t *base, int64_t i, int type) {
    if (type == T_F32) return ((const float *)base)[i];
    if (type == T_F16) return (float)((const _Float16 *)base)[i];
    return (float)((const __bf16 *)base)[i];
}

// one wavefront per (token, head): 64 positions at a time, a lane each for the scores, a lane per value of the head for
// the sums, with the softmax's running maximum and sum
__global__ __launch_bounds__(64) void paged_attn_kernel(PagedAttnArgs a) {
    __shared__ float q[256];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, hd = a.p.hd, kvh = h / (a.n_head / a.p.n_head_kv);
    const int s = paged_find(a.p, t);
    if (s < 0) return;
    float *o = a.o + t * a.ldo + (int64_t)h * hd;
    const PagedSeq sq = paged_seq(a.p, s);
    if (a.ds > 0 && (int64_t)sq.n * (a.n_head / a.p.n_head_kv) <= DEC_ROWS) return;
    if (!sq.ok) {
        for (int i = lane; i < hd; i += 64) o[i] = __builtin_nanf("");
        return;
    }
    const int pos = sq.len - sq.n + (t - sq.t0);
    const int hi = max(pos, a.prefix ? min(a.prefix[s], sq.len) - 1 : 0);
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    for (int i = lane; i < hd; i += 64) q[i] = a.q[t * a.ldq + (int64_t)h * hd + i];
    __syncthreads();
    const float slope = a.slopes ? a.slopes[h] : 0.0f;
    float m = -__builtin_inff(), l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t j0 = lo; j0 <= hi; j0 += 64) {
        const int j = (int)min(j0 + lane, (int64_t)hi);
        const int page = a.p.table[(int64_t)s * a.p.table_stride + (j >> a.p.shift)], in = j & ((1 << a.p.shift) - 1);
        const bool ok = paged_ok(a.p, page);
        const int64_t at = paged_head(a.p, ok ? page : 0, kvh);
        float x = 0.0f;
        for (int i = 0; i < hd; ++i) x = __builtin_fmaf(q[i], paged_get(a.p.k, at + (int64_t)in * hd + i, a.p.type), x);
        x *= a.scale;
        if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
        if (a.slopes) x -= slope * fabsf((float)(pos - j));
        if (!ok) x = __builtin_nanf("");
        if (j0 + lane > hi) x = -__builtin_inff();
        float mx = x;
        bool bad = x != x;
        for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
        const float mn = fmaxf(m, mx), scale = expf(m - mn), p = j0 + lane > hi ? 0.0f : bad ? x : expf(x - mn);
        float sum = p;
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
        l = l * scale + sum;
        m = mn;
        for (int e = 0; e < 4; ++e) acc[e] *= scale;
        for (int u = 0; u < 64 && j0 + u <= hi; ++u) {
            const float pu = __shfl(p, u, 64);
            const int64_t au = __shfl(at, u, 64) + __shfl(in, u, 64);
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < hd)
                    acc[e] = __builtin_fmaf(pu, paged_get(a.p.v, au + ((int64_t)(lane + 64 * e) << a.p.shift), a.p.type), acc[e]);
        }
    }
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < hd) o[lane + 64 * e] = acc[e] / l;
}

// Sums of split ranges joined: grid (sequence x K / V head, fours of rows), a wavefront per row. Lane groups of hd / 4 lanes take
// splits in turn, 16 bytes a lane; always the same order.
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    const int nkv = a.p.n_head_kv, G = a.n_head / nkv, s = blockIdx.x / nkv, kvh = blockIdx.x - s * nkv;
    const int r = __builtin_amdgcn_readfirstlane((int)blockIdx.y * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63, hd = a.p.hd;
    const PagedSeq q = paged_seq(a.p, s);
    if (!q.ok || (int64_t)q.n * G > DEC_ROWS || r >= q.n * G) return;
    const int used = paged_chunk(dec_steps(paged_span(a, q, paged_prefix(a, s, q), 0, q.n - 1)), a.ds, DEC_LEAST).used;
    if (used == 1) return;
    const int64_t t = q.t0 + r / G, row = (int64_t)blockIdx.x * a.drows + r, all = (int64_t)gridDim.x * a.drows;
    const int h = kvh * G + r % G;
    // at most 64 splits: lane i has split i's
    float c = __FLT_MAX__, l = 0.0f;
    if (lane < used) {
        c = a.stat[2 * (lane * all + row)];
        l = a.stat[2 * (lane * all + row) + 1];
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
        if (g < groups && i < used) o += w * *(const pf4 *)(a.part + (i * all + row) * hd + d);
    }
    for (int k = 1; k < groups; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float z = __shfl(o[e], (lane + k * per) & 63, 64);
            if (g == 0) o[e] += z;
        }
    if (g == 0) *(pf4 *)(a.o + t * a.ldo + (int64_t)h * hd + d) = o / l;
}

}  // namespace

// Splits: workgroups for every compute unit eight times over (sequences' lengths differ, and the bounds may be far above
// them: the kernels split what is there), at most 64 (a lane each in the join), at least 128 positions each.
size_t paged_attention_plan(PagedAttnArgs &a, int num_cu) {
    const int G = a.n_head / a.p.n_head_kv;
    const int64_t most = (int64_t)a.p.max_tok * G;  // rows of a sequence and K / V head
    const int64_t heads = (int64_t)a.p.n_seq * a.p.n_head_kv;
    a.ps = most > DEC_ROWS ? 1 : 0;
    a.ds = 0;
    a.drows = (int)std::min<int64_t>(most, DEC_ROWS);
    if (a.ps == 0 || a.p.n_seq > 1) {
        const int64_t want = std::max<int64_t>(1, 8 * (int64_t)num_cu / heads);
        a.ds = (int)std::min<int64_t>({64, want, (a.p.max_len + DEC_STEP * DEC_LEAST - 1) / (DEC_STEP * DEC_LEAST)});
    }
    return a.ds > 1 ? (size_t)a.ds * heads * a.drows : 0;
}

hipError_t launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (a.ds > 0 && (e = launch_paged_decode(a, s)) != hipSuccess) return e;
    if (a.ds > 1) {
        paged_join_kernel<<<dim3((unsigned)a.p.n_seq * (unsigned)a.p.n_head_kv, (unsigned)(a.drows + 3) / 4), 256, 0, s>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (a.ps > 0) {
        paged_attn_kernel<<<dim3((unsigned)a.p.n_tok, (unsigned)a.n_head), 64, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace fgh
