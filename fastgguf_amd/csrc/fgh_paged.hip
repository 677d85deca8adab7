// fgh_paged.hip - the paged KV cache's append on gfx950: the head norms and the position rotation of a
// batch's q and k rows, and k and v into their pages, in one launch.
//
// Rows x of a head: x' = x w / sqrt(mean(x^2) + eps), then pairs (a, b) of it turned by angle_i = p f_i (store_heads);
// V goes in as it is, but transposed: V pages hold the positions of a value side by side (store_v). Bound by its bytes:
// every input value is read once and every output written once, 16 bytes a lane. Measured, 4.76 TB/s for a large copy: 16384 tokens, f32, 32
// heads over 4, hd 64: 335 MB in 73.7 us, 4.55 TB/s; five prompts of 37 to 1100 tokens, f16, 32 over 8, hd 128, with norms: 107 MB in
// 29 us, 3.7 TB/s; one token, or 48 of one each: 4.4 to 4.9 us, a launch.
#include "fgh_paged.h"

#include "fgh_internal.h"

namespace fgh {

namespace {

typedef float sf4 __attribute__((ext_vector_type(4)));
typedef _Float16 sh4 __attribute__((ext_vector_type(4)));
typedef __bf16 sb4 __attribute__((ext_vector_type(4)));

// 4 fp32 values as 4 of the cache's type, to nearest even
template <int TYPE>
__device__ __forceinline__ void put4(uint8_t *base, int64_t i, sf4 x) {
    if constexpr (TYPE == T_F32) *(sf4 *)(base + 4 * i) = x;
    else if constexpr (TYPE == T_F16) *(sh4 *)(base + 2 * i) = __builtin_convertvector(x, sh4);
    else *(sb4 *)(base + 2 * i) = __builtin_convertvector(x, sb4);
}

// cos and sin of p f turns, t = p f formed in 64 bits: its nearest quarter turn taken off exactly, what is left, at most 1/8
// turn, to fp32
__device__ __forceinline__ float2 turned(double t) {
    const double q = rint(4.0 * t);
    const float r = (float)(4.0 * t - q) * 0.5f;  // half turns, -1/4 .. 1/4
    float s, c;
    sincospif(r, &s, &c);
    const int k = (int)(int64_t)q & 3;
    const float x = k & 1 ? s : c, y = k & 1 ? c : s;
    return float2{k == 1 || k == 2 ? -x : x, k >= 2 ? -y : y};
}

constexpr int STORE_V_POS = 64;  // positions of a V tile

// q and k heads of one token: groups of hd / 4 lanes take a head at a time, 4 values a lane. The token's cosines and sines
// are formed once per workgroup.
template <int TYPE>
__device__ __forceinline__ void store_heads(const PagedStoreArgs &a, int t, int part, uint8_t *lds) {
    const int tid = threadIdx.x, hd = a.p.hd, lanes = hd / 4;
    const int all = a.n_head + a.p.n_head_kv;
    const int wave = tid >> 6, lane = tid & 63, per = 64 / lanes, mine = lane / lanes, x = 4 * (lane - mine * lanes);
    const bool in = mine < per;
    const int step = 4 * per;  // heads at a time
    int h = part * a.heads_part + wave * per + mine;
    const int end = min(all, (part + 1) * a.heads_part);
    auto src = [&](int h) { return (const sf4 *)(h < a.n_head ? a.q + t * a.ldq + (int64_t)h * hd + x : a.k + t * a.ldkv + (int64_t)(h - a.n_head) * hd + x); };
    sf4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in && h < end) v = *src(h);  // on its way while the token's sequence is found
    const int s = paged_find(a.p, t);
    if (s < 0) return;
    const PagedSeq sq = paged_useq(a.p, s);
    if ((uint32_t)(t - sq.t0) >= (uint32_t)sq.n) return;  // starts that decrease
    const int pos = sq.len - sq.n + (t - sq.t0);
    if (!sq.ok) {
        for (; in && h < min(end, a.n_head); h += step)
            *(sf4 *)(a.qo + t * a.ldo + (int64_t)h * hd + x) = sf4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        return;
    }
    const int page = a.p.table[(int64_t)s * a.p.table_stride + (pos >> a.p.shift)];

    float2 *cs = (float2 *)lds;                            // [128]
    sf4 *rows = (sf4 *)(lds + 1024) + wave * 64;           // a wavefront's values, for partners in other lanes
    const int half = a.r.n_rot / 2;
    if (tid < half) {
        double f = exp2(-2.0 * tid / a.r.n_rot * a.r.log2_base);
        if (a.r.factors) f /= (double)a.r.factors[tid];
        cs[tid] = turned(pos * (f * a.r.scale_turns));
    }
    __syncthreads();
    sf4 wq = {1.0f, 1.0f, 1.0f, 1.0f}, wk = wq;
    if (in && a.r.qw) wq = sf4{a.r.qw[x], a.r.qw[x + 1], a.r.qw[x + 2], a.r.qw[x + 3]};
    if (in && a.r.kw) wk = sf4{a.r.kw[x], a.r.kw[x + 1], a.r.kw[x + 2], a.r.kw[x + 3]};
    // h of a wavefront's groups differ by one: all take as many turns
    for (int hw = part * a.heads_part + wave * per; hw < end; hw += step, h += step) {
        const sf4 now = v;
        if (in && h + step < end) v = *src(h + step);
        sf4 y = now;
        const bool isq = h < a.n_head, norm = isq ? a.r.qw != nullptr : a.r.kw != nullptr;
        if (a.r.qw || a.r.kw) {
            float ss = y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
            // over the group's lanes: 16 and 64 lanes by exchanges, others through LDS
            if (lanes == 16 || lanes == 32 || lanes == 64) {
                for (int o = 1; o < lanes; o <<= 1) ss += __shfl_xor(ss, o, 64);
            } else {
                float *sum = (float *)rows;
                sum[lane] = ss;
                __builtin_amdgcn_wave_barrier();  // LDS serves a wavefront in order: only the compiler must keep it
                ss = 0.0f;
                for (int i = 0; i < lanes; ++i) ss += sum[in ? mine * lanes + i : 0];
                __builtin_amdgcn_wave_barrier();
            }
            const float r = 1.0f / sqrtf(ss / (float)hd + a.r.eps);
            if (norm) y = y * r * (isq ? wq : wk);
        }
        if (half) {
            sf4 o = {0.0f, 0.0f, 0.0f, 0.0f};
            if (a.r.halves) {
                rows[lane] = y;
                __builtin_amdgcn_wave_barrier();
                const float *row = (const float *)(rows + mine * lanes);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (in && x + e < a.r.n_rot) o[e] = row[x + e < half ? x + e + half : x + e - half];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (x + e < a.r.n_rot) {
                        const float2 c = cs[x + e < half ? x + e : x + e - half];
                        y[e] = x + e < half ? y[e] * c.x - o[e] * c.y : o[e] * c.y + y[e] * c.x;
                    }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e += 2)
                    if (x + e < a.r.n_rot) {
                        const float2 c = cs[(x + e) / 2];
                        const float u = y[e], w = y[e + 1];
                        y[e] = u * c.x - w * c.y;
                        y[e + 1] = u * c.y + w * c.x;
                    }
            }
        }
        if (!in || h >= end) continue;
        if (isq) *(sf4 *)(a.qo + t * a.ldo + (int64_t)h * hd + x) = y;
        else if (paged_ok(a.p, page))
            put4<TYPE>(a.p.k, paged_head(a.p, page, h - a.n_head) + (int64_t)(pos & ((1 << a.p.shift) - 1)) * hd + x, y);
    }
}

// V of a K / V head: the new tokens of a sequence in 64 positions that start at a multiple of 64, through LDS. A thread
// then writes 8 positions of a value as one word where all 8 are new, else one by one.
template <int TYPE>
__device__ __forceinline__ void store_v(const PagedStoreArgs &a, int tile, int kvh, uint8_t *lds) {
    constexpr int ES = TYPE == T_F32 ? 4 : 2, LD = STORE_V_POS * ES + 16;  // bytes of a value's positions, and of a row
    const int tid = threadIdx.x, hd = a.p.hd;
    const PagedVTile v = paged_vtile(a.p, tile);
    if (v.s < 0 || !v.q.ok) return;
    const int p0 = v.q.len - v.q.n, base = v.base, from = max(p0, base), to = min(v.q.len, base + STORE_V_POS);  // positions from .. to - 1
    const int lanes = hd / 4;
    for (int i = tid; i < (to - from) * lanes; i += 256) {
        const int p = i / lanes, x = 4 * (i - p * lanes), at = from + p - base;
        const int64_t t = v.q.t0 + (from + p - p0);
        const sf4 z = *(const sf4 *)(a.v + t * a.ldkv + (int64_t)kvh * hd + x);
        if constexpr (TYPE == T_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *(float *)(lds + (x + e) * LD + at * 4) = z[e];
        } else if constexpr (TYPE == T_F16) {
            const sh4 c = __builtin_convertvector(z, sh4);
#pragma unroll
            for (int e = 0; e < 4; ++e) *(_Float16 *)(lds + (x + e) * LD + at * 2) = c[e];
        } else {
            const sb4 c = __builtin_convertvector(z, sb4);
#pragma unroll
            for (int e = 0; e < 4; ++e) *(__bf16 *)(lds + (x + e) * LD + at * 2) = c[e];
        }
    }
    __syncthreads();
    const int32_t *table = a.p.table + (int64_t)v.s * a.p.table_stride;
    const int g0 = (from - base) / 8, ng = (to - base + 7) / 8 - g0;  // runs of 8 positions: in one page, at a multiple of 8
    for (int i = tid; i < hd * ng; i += 256) {
        const int d = i / ng, g = g0 + i - d * ng, p = base + 8 * g;
        const int page = table[p >> a.p.shift];
        if (!paged_ok(a.p, page)) continue;
        const int64_t at = paged_head(a.p, page, kvh) + ((int64_t)d << a.p.shift) + (p & ((1 << a.p.shift) - 1));
        const uint8_t *row = lds + d * LD + 8 * g * ES;
        if (p >= from && p + 8 <= to) {
#pragma unroll
            for (int w = 0; w < ES / 2; ++w) *(uint4 *)(a.p.v + at * ES + 16 * w) = *(const uint4 *)(row + 16 * w);
        } else
            for (int e = max(from - p, 0); e < min(to - p, 8); ++e) {
                if constexpr (ES == 4) *(uint32_t *)(a.p.v + (at + e) * 4) = *(const uint32_t *)(row + 4 * e);
                else *(uint16_t *)(a.p.v + (at + e) * 2) = *(const uint16_t *)(row + 2 * e);
            }
    }
}

template <int TYPE>
__global__ __launch_bounds__(256) void paged_store_kernel(PagedStoreArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int nv = a.v_tiles * a.p.n_head_kv;
    if ((int)blockIdx.x < nv) store_v<TYPE>(a, blockIdx.x / a.p.n_head_kv, blockIdx.x % a.p.n_head_kv, lds);
    else store_heads<TYPE>(a, (blockIdx.x - nv) / a.parts, (blockIdx.x - nv) % a.parts, lds);
}

template <int TYPE>
hipError_t launch_type(const PagedStoreArgs &a, unsigned grid, hipStream_t s) {
    const size_t v = (size_t)a.p.hd * (STORE_V_POS * (TYPE == T_F32 ? 4 : 2) + 16), heads = 1024 + 4 * 64 * 16;
    paged_store_kernel<TYPE><<<grid, 256, v > heads ? v : heads, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_store(PagedStoreArgs &a, int num_cu, hipStream_t s) {
    const int heads = a.n_head + a.p.n_head_kv, at_once = 4 * (64 / (a.p.hd / 4));
    // a token's heads over several workgroups where tokens are few: two for every compute unit, one turn each at the least
    const int most = (heads + at_once - 1) / at_once;
    a.parts = (int)std::min<int64_t>(most, std::max<int64_t>(1, 2 * (int64_t)num_cu / a.p.n_tok));
    a.heads_part = ((heads + a.parts - 1) / a.parts + at_once - 1) / at_once * at_once;
    a.parts = (heads + a.heads_part - 1) / a.heads_part;
    a.v_tiles = (int)paged_vtiles(a.p.n_tok, a.p.n_seq);
    const int64_t grid = (int64_t)a.v_tiles * a.p.n_head_kv + (int64_t)a.p.n_tok * a.parts;
    switch (a.p.type) {
    case T_F32: return launch_type<T_F32>(a, (unsigned)grid, s);
    case T_F16: return launch_type<T_F16>(a, (unsigned)grid, s);
    case T_BF16: return launch_type<T_BF16>(a, (unsigned)grid, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace fgh
