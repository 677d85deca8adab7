// fgh_pattn.hip - attention over the paged KV cache on gfx950.
#include "fgh_paged.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "fgh_internal.h"

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

}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
    paged_attn_kernel<<<dim3((unsigned)a.p.n_tok, (unsigned)a.n_head), 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace fgh
