// fgh_pattn.h - what the paged attention's kernels share (fgh_pdecode.h, fgh_pprompt.h, fgh_pattn.hip). Internal.
//
// fp32 results from 16-bit matrix instructions: every operand is a sum of 16-bit parts, and the products of parts are
// summed in the fp32 accumulators.
//   F16 cache   q and the weights as 2 halves; K and V as they are: 2 products
//   BF16 cache  q and the weights as 3 bf16, cut so that they hold all 24 bits; 3 products
//   F32 cache   K and V too as 3 bf16; 6 products. The 3 left out are at most 2^-21 of the whole product, and 2^-24.6 on average:
//               the parts are cut, not rounded, so that each is up to 2^-7 of the one before
// Halves have 5 bits of exponent. So a q row's largest value is brought to [2^14, 2^15) by a power of two (the scores take it
// back with the scale): values down to 2^-17 of the largest keep 22 bits, smaller ones count to 2^-40 of it. The weights' second halves,
// which would leave the halves' range 12 bits before the first ones, are carried times 2^LOW and summed by themselves. With
// the largest weight at 2^12 to 2^15.9 a weight keeps 22 bits down to 2^-26 of the largest, 17 (the 1e-5 of a result) down
// to 2^-31, and is off by at most 2^-48 of it below: what decides where the largest weights stand at V near 0. (Both halves
// on one scale, the largest at 2^10, held 17 bits down to 2^-18 only, for 6 % less time of a long prompt.)
// q's small products are summed apart where registers allow: an error of 1.0 instead of 1.5 to 2 times a plain fp32 form's where few
// large scores decide.
#pragma once

#include "fgh_internal.h"
#include "fgh_paged.h"

namespace fgh {

typedef uint32_t pu4 __attribute__((ext_vector_type(4)));
typedef float pf2 __attribute__((ext_vector_type(2)));
typedef float pf4 __attribute__((ext_vector_type(4)));
typedef float pf16 __attribute__((ext_vector_type(16)));
typedef _Float16 ph2 __attribute__((ext_vector_type(2)));
typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef __bf16 pb8 __attribute__((ext_vector_type(8)));

template <int TYPE>
struct PagedType {
    static constexpr int ES = TYPE == T_F32 ? 4 : 2;  // bytes a cached value
    static constexpr int NQ = TYPE == T_F16 ? 2 : 3;  // parts of q and of the weights
    static constexpr int NK = TYPE == T_F32 ? 3 : 1;  // parts of K and V
    // Weights are 2^(PBIAS + s - m), s in powers of two, m a running reference of the row that follows a larger s where the exponent
    // would pass PTOP. Halves: up to what their range allows (2^16, and 2^15 for second ones times 2^LOW), and 2^3 below it after the
    // reference has moved: in 2^2 it moves more often (8192 tokens 1013 us, 997 so), in 2^6 weights lose 3 bits for 6 us. Elsewhere near
    // 1, where the exponent of the largest is rounded least.
    static constexpr float PBIAS = TYPE == T_F16 ? 13.0f : 0.0f, PTOP = TYPE == T_F16 ? 15.9f : 5.0f;
    static constexpr int LOW = TYPE == T_F16 ? 11 : 0;
    static constexpr float LOW_UP = 1 << LOW, LOW_DOWN = 1.0f / LOW_UP;
    static constexpr int NPROD = TYPE == T_F16 ? 2 : TYPE == T_F32 ? 6 : 3;  // products of parts
};

// D += A B, 16 x 16 with 32 products a sum, or 32 x 32 with 16. A: lane l holds row l % 16 (32), values 8 (l / 16 (32)) .. + 7; B: column
// l % 16 (32), the same values. D: column l % 16 (32); register r is row 4 (l / 16) + r, or 8 (r / 4) + 4 (l / 32) + r % 4.
template <int TYPE>
__device__ __forceinline__ void mma16(pf4 &d, pu4 x, pu4 y) {
    if constexpr (TYPE == T_F16) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, x), __builtin_bit_cast(ph8, y), d, 0, 0, 0);
    else d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pb8, x), __builtin_bit_cast(pb8, y), d, 0, 0, 0);
}
template <int TYPE>
__device__ __forceinline__ void mma32(pf16 &d, pu4 x, pu4 y) {
    if constexpr (TYPE == T_F16) d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ph8, x), __builtin_bit_cast(ph8, y), d, 0, 0, 0);
    else d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pb8, x), __builtin_bit_cast(pb8, y), d, 0, 0, 0);
}

// values 2 i and 2 i + 1 of 8 as NP vectors of 16-bit parts, a second half times `up`, a power of two
template <int TYPE, int NP>
__device__ __forceinline__ void parts2(float a, float b, int i, pu4 (&out)[NP], float up = 1.0f) {
    if constexpr (TYPE == T_F16) {  // to nearest, then what is left to nearest
        const pf2 v = {a, b};
        const ph2 h = __builtin_convertvector(v, ph2);
        out[0][i] = __builtin_bit_cast(uint32_t, h);
        const pf2 rest = {__builtin_fmaf((float)h.x, -up, a * up), __builtin_fmaf((float)h.y, -up, b * up)};  // exact
        out[1][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, ph2));
    } else {  // the upper halves of the words, cut: what is left is exact, and 8 + 8 + 8 bits hold it all
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const uint32_t u = __float_as_uint(a), v = __float_as_uint(b);
            out[k][i] = __builtin_amdgcn_perm(v, u, 0x07060302);
            a -= __uint_as_float(u & 0xffff0000u);
            b -= __uint_as_float(v & 0xffff0000u);
        }
    }
}
// 8 fp32 values as NP vectors of 8 16-bit parts
template <int TYPE, int NP>
__device__ __forceinline__ void parts8(const float *x, pu4 (&out)[NP], float up = 1.0f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) parts2<TYPE, NP>(x[2 * i], x[2 * i + 1], i, out, up);
}
// 8 weights, as parts, times a power of two of at most 1. Halves are put together and taken apart again: each by itself would
// lose what falls below 2^-24.
template <int TYPE, int NP>
__device__ __forceinline__ void scale8(pu4 (&x)[NP], float f) {
    if constexpr (TYPE == T_F16) {
        using T = PagedType<TYPE>;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const ph2 h = __builtin_bit_cast(ph2, (uint32_t)x[0][i]), r = __builtin_bit_cast(ph2, (uint32_t)x[1][i]);
            parts2<TYPE, NP>(__builtin_fmaf((float)r.x, T::LOW_DOWN, (float)h.x) * f, __builtin_fmaf((float)r.y, T::LOW_DOWN, (float)h.y) * f, i, x, T::LOW_UP);
        }
    } else
#pragma unroll
        for (int k = 0; k < NP; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[k][i] = __builtin_amdgcn_perm(__float_as_uint(__uint_as_float(x[k][i] & 0xffff0000u) * f), __float_as_uint(__uint_as_float(x[k][i] << 16) * f), 0x07060302);
}
// 8 cached values (16 or 32 bytes) as parts
template <int TYPE>
__device__ __forceinline__ void cache8(const pu4 *raw, pu4 (&out)[PagedType<TYPE>::NK]) {
    if constexpr (TYPE == T_F32) {
        const float x[8] = {__uint_as_float(raw[0].x), __uint_as_float(raw[0].y), __uint_as_float(raw[0].z), __uint_as_float(raw[0].w),
                            __uint_as_float(raw[1].x), __uint_as_float(raw[1].y), __uint_as_float(raw[1].z), __uint_as_float(raw[1].w)};
        parts8<TYPE, 3>(x, out);
    } else
        out[0] = raw[0];
}

// cached value e of 8 in raw: whether it is not finite
template <int TYPE>
__device__ __forceinline__ bool raw_bad(const pu4 *raw, int e) {
    if constexpr (TYPE == T_F32) return (raw[e / 4][e % 4] & 0x7f800000u) == 0x7f800000u;
    const uint32_t h = raw[0][e / 2] >> (16 * (e & 1));
    return TYPE == T_F16 ? (h & 0x7c00u) == 0x7c00u : (h & 0x7f80u) == 0x7f80u;
}
// a word of cached values: not 0 where one is not finite
template <int TYPE>
__device__ __forceinline__ uint32_t infinite(uint32_t w) {
    if constexpr (TYPE == T_F32) return ((w & 0x7f800000u) + 0x00800000u) & 0x80000000u;
    else if constexpr (TYPE == T_F16) return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    else return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
// the word with zeros in the place of what is not finite
template <int TYPE>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
    const uint32_t f = infinite<TYPE>(w);
    if constexpr (TYPE == T_F32) return f ? 0u : w;
    const uint32_t ones = f >> 15;  // 1 in each half that is not finite
    return w & ~((ones << 16) - ones);
}
template <int TYPE>
__device__ __forceinline__ void raw_zero(pu4 *raw, int e) {
    if constexpr (TYPE == T_F32) raw[e / 4][e % 4] = 0;
    else raw[0][e / 2] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
}
template <int TYPE>
__device__ __forceinline__ float cached(const uint8_t *base, int64_t i) {
    if constexpr (TYPE == T_F32) return ((const float *)base)[i];
    else if constexpr (TYPE == T_F16) return (float)((const _Float16 *)base)[i];
    else return __uint_as_float((uint32_t)((const uint16_t *)base)[i] << 16);
}
__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

constexpr float LOG2E = 1.44269504088896340736f;

// tanh within 3 roundings: y + y^3 g(y^2) below 0.65 (g fitted at Chebyshev nodes), 1 - 2 e / (1 + e), e = e^(-2 y), above
__device__ __forceinline__ float tanh_below(float y) {
    const float z = y * y;
    float g = -0.005932980682700872f;
    g = __builtin_fmaf(g, z, 0.020881319418549538f);
    g = __builtin_fmaf(g, z, -0.053825847804546356f);
    g = __builtin_fmaf(g, z, 0.13332600891590118f);
    g = __builtin_fmaf(g, z, -0.333333283662796f);
    return __builtin_fmaf(y * z, g, y);
}
__device__ __forceinline__ float tanh_above(float y) {
    const float e = __builtin_amdgcn_exp2f(fabsf(y) * (-2.0f * LOG2E)), d = 1.0f + e, r = __builtin_amdgcn_rcpf(d);
    return copysignf(__builtin_fmaf(-2.0f * e, __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.0f), r), 1.0f), y);
}
constexpr float TANH_SPLIT = 0.65f;

// Scores above 2^20 leave fewer than 4 bits behind the point: a score rounded for the maximum and the same score unrounded in its
// weight's sum would differ by powers of two, enough to pass a half's range, or from 2^30 on an fp32's. Once a reference of a wavefront's
// rows is that far from 0, scores are rounded before they are used, and such a reference is the maximum itself.
// (Not for an infinite one, which leaves its own row undefined and the others as they are.)
constexpr float SCORE_BIG = 0x1p20f;
__device__ __forceinline__ bool score_big(float mx) { return fabsf(mx) > SCORE_BIG && fabsf(mx) <= __FLT_MAX__; }
template <int TYPE>
__device__ __forceinline__ float score_bias(float mx) { return fabsf(mx) > SCORE_BIG ? 0.0f : PagedType<TYPE>::PBIAS; }

// What turns a row's products into scores in powers of two, s = v mul: v the products or, capped, their tanh, mul apply's result. The
// product with mul is rounded once, in the sum that follows it.
struct PagedScore {
    float mul;             // |scale| log2(e), times the power of two that q was divided by; above 0 and finite, so that -inf v
                           // are -inf scores and 0 is 0 (q takes the scale's sign, and is 0 for a scale of 0)
    float cap_in, cap_out; // |scale| / softcap (with that power), softcap log2(e); cap_out 0: none
    float slope, down;     // |slopes[h]| log2(e), and -1 or 1 with the slope's sign turned around
    bool bias;
    // NE products of positions j0 .. j0 + NE - 1 of a row at position p
    template <int NE>
    __device__ __forceinline__ float apply(float (&v)[NE], int j0, int p) const {
        if (cap_out > 0.0f) {
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                v[e] *= cap_in;
                top = fmaxf(top, fabsf(v[e]));
            }
            if (__builtin_amdgcn_ballot_w64(!(top < TANH_SPLIT))) {
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    v[e] = fabsf(v[e]) < TANH_SPLIT ? tanh_below(v[e]) : tanh_above(v[e]);
                    if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four at a time: all at once would cost registers
                }
            } else {
#pragma unroll
                for (int e = 0; e < NE; ++e) v[e] = tanh_below(v[e]);
            }
        }
        const float m = cap_out > 0.0f ? cap_out : mul;
        if (!bias) return m;
        const float base = slope * (float)(p - j0);  // slope |p - j0 - e| = |slope (p - j0) - slope e|
#pragma unroll
        for (int e = 0; e < NE; ++e) v[e] = __builtin_fmaf(v[e], m, down * fabsf(__builtin_fmaf((float)-e, slope, base)));
        return 1.0f;
    }
};
__device__ __forceinline__ PagedScore paged_score(const PagedAttnArgs &a, int head, float q_size) {
    PagedScore c;
    const float scale = fabsf(a.scale) * q_size;
    c.mul = fminf(fmaxf(scale * LOG2E, __FLT_MIN__), __FLT_MAX__);
    c.cap_in = a.softcap > 0.0f ? fminf(scale / a.softcap, __FLT_MAX__) : 0.0f;
    c.cap_out = a.softcap * LOG2E;
    c.bias = a.slopes != nullptr;
    const float slope = c.bias ? a.slopes[head] : 0.0f;
    c.slope = fabsf(slope) * LOG2E;
    c.down = slope < 0.0f ? 1.0f : -1.0f;
    return c;
}

// the power of two that brings a row's largest magnitude to [2^14, 2^15), or as near as 2^126 does, as the factor that undoes
// it (amax not finite: 1)
__device__ __forceinline__ float row_size(float amax) {
    const uint32_t e = __float_as_uint(amax) >> 23;
    return e == 255 ? 1.0f : __uint_as_float((e > 15 ? e - 14 : 1u) << 23);
}

// that power of two where q keeps its size (not F16): with scales below 2^-64 q and the scale meet halfway, since products
// of up to 2^128 would otherwise meet a factor below an fp32's normal ones
__device__ __forceinline__ float scale_size(float scale) { return fabsf(scale) < 0x1p-64f ? 0x1p64f : 1.0f; }
// and what q is multiplied by
__device__ __forceinline__ float q_factor(float scale, float size) { return (scale < 0.0f ? -1.0f : scale > 0.0f ? 1.0f : 0.0f) / size; }

// positions lo .. hi that the new tokens i0 .. i1 of a sequence see, and those that all of them see
struct PagedSpan {
    int lo, hi, in_lo, in_hi;
};
__device__ __forceinline__ int row_lo(const PagedAttnArgs &a, int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; }
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnArgs &a, const PagedSeq &q, int prefix, int i0, int i1) {
    const int p0 = q.len - q.n + i0, p1 = q.len - q.n + i1;
    return PagedSpan{row_lo(a, p0), max(p1, prefix - 1), row_lo(a, p1), max(p0, prefix - 1)};
}
__device__ __forceinline__ int paged_prefix(const PagedAttnArgs &a, int s, const PagedSeq &q) {
    return a.prefix ? min(max(__builtin_amdgcn_readfirstlane(a.prefix[s]), 0), q.len) : 0;  // s: uniform
}
// a range of n units over at most `splits` workgroups, `least` units or more each: the units of one, and how many
// workgroups have any
struct PagedChunk {
    int per, used;
};
__device__ __forceinline__ PagedChunk paged_chunk(int n, int splits, int least, int whole) {
    const int per = max(((n + splits - 1) / splits + whole - 1) / whole * whole, least);
    return PagedChunk{per, (n + per - 1) / per};
}

constexpr int DEC_ROWS = 16;                // rows of the decode kernel
constexpr int DEC_STEP = 32;                // positions a step of a wavefront
// workgroups of the decode kernel that a compute unit holds, by its registers
constexpr int dec_resident(int type, int hd) { return hd > 128 || (type == T_F32 && hd > 96) ? 1 : 2; }
// the decode kernel's steps of a range
__device__ __forceinline__ int dec_steps(const PagedSpan &r) { return (r.hi - (r.lo & ~(DEC_STEP - 1))) / DEC_STEP + 1; }

constexpr int PRO_UNIT = 64;                // positions are split in units of 64,
constexpr int PRO_LEAST = 4;                // that many and more each
__device__ __forceinline__ int pro_units(const PagedSpan &r) { return (r.hi - (r.lo & ~(PRO_UNIT - 1))) / PRO_UNIT + 1; }
// at most as many sequences of a batch with several are the prompt kernel's, and the tiles they can have
inline int64_t pro_seqs(const PagedAttnArgs &a) {
    return std::min<int64_t>(a.p.n_seq, (int64_t)a.p.n_tok * (a.n_head / a.p.n_head_kv) / (DEC_ROWS + 1));
}
inline int64_t paged_tiles(const PagedAttnArgs &a) { return paged_tiles(a.p.n_tok, pro_seqs(a), a.n_head / a.p.n_head_kv, a.prows); }
// whether there is a form of the prompt kernel with half the rows (not where its tiles are of 32 positions)
constexpr bool pro_half(int type, int hd) { return !(type == T_F32 && hd > 128); }
// Tile `index` of the batch: the sequences' tiles in order (of those that are the prompt kernel's). s = -1: there are fewer.
struct PagedTile {
    int s, r0, index;
    PagedSeq q;
};
__device__ __forceinline__ PagedTile paged_tile(const PagedAttnArgs &a, int tile_rows, int index) {
    const int lane = threadIdx.x & 63, G = a.n_head / a.p.n_head_kv;
    int before = 0, top = 0;  // tiles of the sequences before the 64 looked at
    PagedTile t;
    t.s = -1, t.r0 = 0, t.index = index, t.q = PagedSeq{};
    for (int b = 0; b < a.p.n_seq; b += 64) {
        const int s = b + lane;
        int own = 0;
        PagedSeq q{};
        if (s < a.p.n_seq) q = paged_seq(a.p, s);
        paged_own_rows(a.p, s, q, top);
        if (s < a.p.n_seq) {
            const int64_t rows = (int64_t)q.n * G;
            own = a.ds > 0 && rows <= DEC_ROWS ? 0 : (int)((rows + tile_rows - 1) / tile_rows);
        }
        int upto = own;  // with this lane's
        for (int o = 1; o < 64; o <<= 1) {
            const int z = __shfl_up(upto, o, 64);
            if (lane >= o) upto += z;
        }
        const uint64_t m = __builtin_amdgcn_ballot_w64(before + upto > index);
        if (m) {
            const int at = __builtin_ctzll(m);
            t.s = b + at;
            t.r0 = (index - before - (__shfl(upto, at, 64) - __shfl(own, at, 64))) * tile_rows;
            t.s = __builtin_amdgcn_readfirstlane(t.s);
            t.r0 = __builtin_amdgcn_readfirstlane(t.r0);
            t.q.t0 = __builtin_amdgcn_readlane(q.t0, at), t.q.n = __builtin_amdgcn_readlane(q.n, at);
            t.q.len = __builtin_amdgcn_readlane(q.len, at), t.q.ok = __builtin_amdgcn_readlane(q.ok, at);
            return t;
        }
        before += __shfl(upto, 63, 64);
    }
    return t;
}

hipError_t launch_paged_decode(const PagedAttnArgs &a, hipStream_t s);
hipError_t launch_paged_prompt(const PagedAttnArgs &a, hipStream_t s);

}  // namespace fgh
