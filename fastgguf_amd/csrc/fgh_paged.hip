// fgh_paged.hip - the paged KV cache's append on gfx950: the head norms and the position rotation of a
// batch's q and k rows, and k and v into their pages, in one launch.
#include "fgh_paged.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "fgh_internal.h"

namespace fgh {

namespace {

// fp32 to the cache's type, to nearest even
__device__ __forceinline__ void paged_put(uint8_t *base, int64_t i, int type, float x) {
    if (type == T_F32) ((float *)base)[i] = x;
    else if (type == T_F16) ((_Float16 *)base)[i] = (_Float16)x;
    else ((__bf16 *)base)[i] = (__bf16)x;
}

// one wavefront per (token, head of q, k or v)
__global__ __launch_bounds__(64) void paged_store_kernel(PagedStoreArgs a) {
    __shared__ float x[256];
    const int t = blockIdx.x, lane = threadIdx.x, hd = a.p.hd;
    int h = blockIdx.y;
    const int what = h < a.n_head ? 0 : h < a.n_head + a.p.n_head_kv ? 1 : 2;
    h -= what == 0 ? 0 : what == 1 ? a.n_head : a.n_head + a.p.n_head_kv;
    const int s = paged_find(a.p, t);
    if (s < 0) return;
    const PagedSeq q = paged_seq(a.p, s);
    if (!q.ok) {
        if (what == 0)
            for (int i = lane; i < hd; i += 64) a.qo[t * a.ldo + (int64_t)h * hd + i] = __builtin_nanf("");
        return;
    }
    const int pos = q.len - q.n + (t - q.t0);
    const float *src = (what == 0 ? a.q + t * a.ldq : (what == 1 ? a.k : a.v) + t * a.ldkv) + (int64_t)h * hd;
    float ss = 0.0f;
    for (int i = lane; i < hd; i += 64) {
        x[i] = src[i];
        ss += x[i] * x[i];
    }
    const float *w = what == 0 ? a.r.qw : what == 1 ? a.r.kw : nullptr;
    if (w) {
        for (int o = 1; o < 64; o <<= 1) ss += __shfl_xor(ss, o, 64);
        const float r = 1.0f / sqrtf(ss / (float)hd + a.r.eps);
        for (int i = lane; i < hd; i += 64) x[i] = x[i] * r * w[i];
    }
    __syncthreads();
    if (what < 2) {
        const int half = a.r.n_rot / 2;
        for (int i = lane; i < half; i += 64) {
            double f = exp2(-2.0 * i / a.r.n_rot * a.r.log2_base);
            if (a.r.factors) f /= (double)a.r.factors[i];
            double turn = pos * (f * a.r.scale_turns);
            turn -= rint(turn);
            const double ang = turn * 6.283185307179586476925;
            const float c = (float)cos(ang), sn = (float)sin(ang);
            const int ia = a.r.halves ? i : 2 * i, ib = a.r.halves ? i + half : 2 * i + 1;
            const float u = x[ia], v = x[ib];
            x[ia] = u * c - v * sn;
            x[ib] = u * sn + v * c;
        }
        __syncthreads();
    }
    if (what == 0) {
        for (int i = lane; i < hd; i += 64) a.qo[t * a.ldo + (int64_t)h * hd + i] = x[i];
        return;
    }
    const int page = a.p.table[(int64_t)s * a.p.table_stride + (pos >> a.p.shift)], in = pos & ((1 << a.p.shift) - 1);
    if (!paged_ok(a.p, page)) return;
    const int64_t at = paged_head(a.p, page, h);
    for (int i = lane; i < hd; i += 64)
        paged_put(what == 1 ? a.p.k : a.p.v, what == 1 ? at + (int64_t)in * hd + i : at + ((int64_t)i << a.p.shift) + in, a.p.type, x[i]);
}

}  // namespace

hipError_t launch_paged_store(const PagedStoreArgs &a, hipStream_t s) {
    paged_store_kernel<<<dim3((unsigned)a.p.n_tok, (unsigned)(a.n_head + 2 * a.p.n_head_kv)), 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace fgh
