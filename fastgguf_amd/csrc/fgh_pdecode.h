// fgh_pdecode.h - paged attention of few rows per K / V head: generation, a few drafted tokens.
//
// A sequence's up to 16 rows of a K / V head (its new tokens x the head's query heads) are the columns of
// 16 x 16 matrix products, so a head's pages are read once for all of them. Per 32 positions a wavefront forms
//   S^T = K q^T: A = K rows, B = q. The rows of the two 16-row products are the 32 positions in such an order that a
//         lane's 8 scores (4 of each product) are of 8 positions in a row.
//   O^T += V^T P^T: those 8 weights are what the lane has to give as B, and 8 positions of one value row of V^T are 16
//         bytes of a V page. So neither K, V nor the weights go through LDS or another lane.
// Softmax: weights 2^(PBIAS + s - m) with a reference m of the row, which follows the maximum only where a weight would pass 2^PTOP;
// the rows' sums stay in their lanes to the end. Each wavefront takes every fourth step of the workgroup's positions; the next step's K
// is asked for when the scores are done, its V when the sums are; the four wavefronts are joined in LDS.
//
// Bound by the rate of the cache's reads, as long as there are many: a step's 16 to 64 KB of K and V are in flight for each wavefront while
// the one before is used, and no byte is asked of memory twice. 16 rows, since that is the narrowest matrix product: fewer rows cost
// nothing less, more are the prompt kernel's. Measured with the join: 32 sequences of 65 to 8192 positions, f16, 32 heads over 8, hd 128: 535 MB
// in 115.5 us, 4.6 TB/s (a large copy here: 4.8, a plain read of 1 GB: 6.7); 8 of up to 4096 in a window, capped, bf16, hd 256: 239 MB in 56
// us; 4 tokens of 6 sequences over an f32 cache: 79 MB in 28 us; one sequence of 4096 positions: 17 MB in 11.9 us, of which two launches that
// wait for each other are 8.
#pragma once

#include "fgh_pattn.h"

namespace fgh {

template <int TYPE, int HD>
struct Dec {
    static constexpr int ES = PagedType<TYPE>::ES, NQ = PagedType<TYPE>::NQ, NK = PagedType<TYPE>::NK;
    static constexpr int W = ES / 2;             // 16-byte words of 8 values
    static constexpr int KS = (HD + 31) / 32;    // steps of 32 along the head
    static constexpr int VB = HD / 16;           // blocks of 16 of V's values
    static constexpr bool LOW = PagedType<TYPE>::LOW > 0;  // the weights' second parts are summed by themselves
    static constexpr int OCC = dec_resident(TYPE, HD);
};

constexpr int dec_lds(int hd) { return (4 * DEC_ROWS * (hd + 4) + 8 * DEC_ROWS) * 4; }

template <int TYPE, int HD>
__device__ __forceinline__ void paged_decode_block(const PagedAttnArgs &a, int block, uint8_t *lds) {
    using D = Dec<TYPE, HD>;
    constexpr int LD = HD + 4;
    float(*acc_l)[DEC_ROWS][LD] = (float(*)[DEC_ROWS][LD])lds;
    float(*c_l)[DEC_ROWS] = (float(*)[DEC_ROWS])(lds + 4 * DEC_ROWS * LD * 4), (*l_l)[DEC_ROWS] = c_l + 4;
    const int nkv = a.p.n_head_kv, G = a.n_head / nkv;
    const int kvh = block % nkv, split = block / nkv % a.ds, s = block / nkv / a.ds;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    PagedSeq q = paged_useq(a.p, s);
    // the prompt kernel's, unless starts decrease and only few of the rows are the sequence's own
    if (a.ps > 0 && (int64_t)q.n * G > DEC_ROWS) paged_own_rows(a.p, s, q);
    const int64_t rows = (int64_t)q.n * G;
    const bool none = q.n == 0 || (a.ps > 0 && rows > DEC_ROWS);
    if (a.ds > 1 && split == 0 && tid == 0 && (none || !q.ok)) a.dsum.info[s * nkv + kvh].used = 0;
    if (none) return;
    if (!q.ok) {
        if (split == 0)
            for (int64_t i = tid; i < rows * HD; i += 256) {
                const int r = (int)(i / HD), x = (int)(i - (int64_t)r * HD);
                a.o[(q.t0 + r / G) * a.ldo + (int64_t)(kvh * G + r % G) * HD + x] = __builtin_nanf("");
            }
        return;
    }
    const int prefix = paged_prefix(a, s, q);
    const PagedSpan sp = paged_span(a, q, prefix, 0, q.n - 1);
    const int base = sp.lo & ~(DEC_STEP - 1), steps = dec_steps(sp);
    const PagedChunk ch = paged_chunk(steps, a.ds, 4, 4);
    if (split >= ch.used) return;
    if (a.ds > 1 && split == 0 && tid == 0) a.dsum.info[s * nkv + kvh] = PagedSlot{ch.used, (int)rows, q.t0, 0};
    const int end = min(steps, (split + 1) * ch.per);

    // this lane's row: column m of the products
    const int m = lane & 15, quad = lane >> 4, R = (int)rows;
    const bool mine = m < R;
    const int i = mine ? m / G : 0, head = kvh * G + (mine ? m - i * G : 0);
    const int pos = q.len - q.n + i;
    const int lo = mine ? row_lo(a, pos) : 0x7fffffff, hi = mine ? max(pos, prefix - 1) : -1;

    const int mask = (1 << a.p.shift) - 1, kc = (lane >> 2) & 3;
    const int32_t *table = a.p.table + (int64_t)s * a.p.table_stride;
    auto entry = [&](int j) { return table[min(j, sp.hi) >> a.p.shift]; };
    int next_k = 0, next_v = 0;  // the pages of the step that is loaded next
    pu4 kr[2][D::KS][D::W], vr[D::VB][D::W];
    bool bad = false;            // the page of this lane's 8 V positions does not exist
    auto pages = [&](int st) {
        next_k = entry(base + st * DEC_STEP + kc * 8);
        next_v = entry(base + st * DEC_STEP + quad * 8);
    };
    auto load_k = [&](int st) {
        const int kb = base + st * DEC_STEP;
        const int64_t hk = paged_head(a.p, paged_ok(a.p, next_k) ? next_k : 0, kvh);
        const uint8_t *kp = a.p.k + (hk + (int64_t)((kb + kc * 8 + (lane & 3)) & mask) * HD + quad * 8) * D::ES;
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int ks = 0; ks < D::KS; ++ks) {
                // past the head (hd 80): its first values, times q's zeros
                const int x = HD % 32 != 0 && ks == D::KS - 1 && quad >= HD % 32 / 8 ? -quad * 8 : ks * 32;
#pragma unroll
                for (int w = 0; w < D::W; ++w) kr[g][ks][w] = *(const pu4 *)(kp + (g * 4 * HD + x) * D::ES + 16 * w);
            }
    };
    auto load_v = [&](int st) {
        const int kb = base + st * DEC_STEP;
        bad = !paged_ok(a.p, next_v);
        const int64_t hv = paged_head(a.p, bad ? 0 : next_v, kvh);
        const uint8_t *vp = a.p.v + (hv + ((int64_t)m << a.p.shift) + ((kb + quad * 8) & mask)) * D::ES;
#pragma unroll
        for (int b = 0; b < D::VB; ++b)
#pragma unroll
            for (int w = 0; w < D::W; ++w) vr[b][w] = *(const pu4 *)(vp + ((int64_t)(16 * b) << a.p.shift) * D::ES + 16 * w);
    };
    int st = split * ch.per + wave;
    if (st < end) pages(st);
    float x[D::KS][8];  // q, asked for ahead of K and V: loads return in order
#pragma unroll
    for (int ks = 0; ks < D::KS; ++ks) {
        const bool in = mine && ks * 32 + quad * 8 < HD;
        const pf4 *src = (const pf4 *)(a.q + (q.t0 + i) * a.ldq + (int64_t)head * HD + (in ? ks * 32 + quad * 8 : 0));
        const pf4 u = src[0], v = src[1];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[ks][e] = in ? (e < 4 ? u[e & 3] : v[e & 3]) : 0.0f;
    }
    if (st < end) {
        load_k(st);
        load_v(st);
        if (st + 4 < end) pages(st + 4);
    }

    pu4 qp[D::KS][D::NQ];
    PagedScore score;
    {
        float amax = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D::KS; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[ks][e]));
        float size = scale_size(a.scale);
        if constexpr (TYPE == T_F16) {
            amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
            amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
            size = row_size(amax);
        }
        const float inv = q_factor(a.scale, size);
#pragma unroll
        for (int ks = 0; ks < D::KS; ++ks) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[ks][e] *= inv;
            parts8<TYPE, D::NQ>(x[ks], qp[ks]);
        }
        score = paged_score(a, head, size);
    }

    pf4 acc[D::VB], low[D::VB];
#pragma unroll
    for (int b = 0; b < D::VB; ++b) acc[b] = low[b] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
    float c = __FLT_MAX__, l = 0.0f;  // c = PBIAS - m
    bool big = false;                 // a reference beyond SCORE_BIG

    for (; st < end; st += 4) {
        const int kb = base + st * DEC_STEP, j0 = kb + quad * 8;
        const bool more = st + 4 < end;
        // the first parts' products apart from the others', which are small: fewer roundings at the scores' size
        pf4 sc[2], rest[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) sc[g] = rest[g] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int ks = 0; ks < D::KS; ++ks) {
                pu4 kp[D::NK];
                cache8<TYPE>(kr[g][ks], kp);
#pragma unroll
                for (int x = D::NQ - 1; x >= 0; --x)
#pragma unroll
                    for (int y = D::NK - 1; y >= 0; --y)
                        if (x + y < 3) mma16<TYPE>(x + y == 0 ? sc[g] : rest[g], kp[y], qp[ks][x]);
            }
        if (more) load_k(st + 4);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sc[e / 4][e % 4] + rest[e / 4][e % 4];
        float mul = score.apply(v, j0, pos);
        // positions that some row does not see: at the ends of the ranges
        const bool whole = kb >= sp.in_lo && kb + DEC_STEP - 1 <= sp.in_hi && !__builtin_amdgcn_ballot_w64(bad);
        bool odd = false;  // a V value that only some rows see is not finite
        if (!whole) {
            pu4 keep[D::W];
#pragma unroll
            for (int w = 0; w < D::W; ++w) keep[w] = ~pu4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = j0 + e;
                if (bad) v[e] = __builtin_nanf("");
                if (j < lo || j > hi) v[e] = -__builtin_inff();
                if (bad || j < sp.lo || j > sp.hi) raw_zero<TYPE>(keep, e);  // seen by no row
            }
#pragma unroll
            for (int b = 0; b < D::VB; ++b)
#pragma unroll
                for (int w = 0; w < D::W; ++w) vr[b][w] &= keep[w];
            if (q.n > 1) {
#pragma unroll
                for (int b = 0; b < D::VB; ++b)
#pragma unroll
                    for (int w = 0; w < D::W; ++w)
#pragma unroll
                        for (int i = 0; i < 4; ++i) odd |= infinite<TYPE>(vr[b][w][i]) != 0;
                odd = __builtin_amdgcn_ballot_w64(odd) != 0;
                if (odd) {
#pragma unroll
                    for (int b = 0; b < D::VB; ++b)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (raw_bad<TYPE>(vr[b], e)) raw_zero<TYPE>(vr[b], e);
                }
            }
        }
        float top = v[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, v[e]);
        top *= mul;
        if (__builtin_amdgcn_ballot_w64(top + c > PagedType<TYPE>::PTOP)) {
            float mx = fmaxf(top, __shfl_xor(top, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            big = big || __builtin_amdgcn_ballot_w64(mx + c > PagedType<TYPE>::PTOP && score_big(mx)) != 0;
            if (mx + c > PagedType<TYPE>::PTOP) {  // of the whole row: its four lanes agree
                const float cn = score_bias<TYPE>(mx) - mx, f = __builtin_amdgcn_exp2f(cn - c);
                c = cn;
                l *= f;
#pragma unroll
                for (int b = 0; b < D::VB; ++b) {
                    acc[b] *= f;
                    if (D::LOW) low[b] *= f;
                }
            }
        }
        if (big) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= mul;
            mul = 1.0f;
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(v[e], mul, c));
            l += p[e];
        }
        pu4 pp[D::NQ];
        parts8<TYPE, D::NQ>(p, pp, PagedType<TYPE>::LOW_UP);
#pragma unroll
        for (int b = 0; b < D::VB; ++b) {
            pu4 vp[D::NK];
            cache8<TYPE>(vr[b], vp);
#pragma unroll
            for (int x = D::NQ - 1; x >= 0; --x)
#pragma unroll
                for (int y = D::NK - 1; y >= 0; --y)
                    if (x + y < 3) mma16<TYPE>(D::LOW && x > 0 ? low[b] : acc[b], vp[y], pp[x]);
        }
        if (more) {
            load_v(st + 4);
            if (st + 8 < end) pages(st + 8);
        }
        if (odd) {
            // values that are not finite, left out above: added to the rows that see them
            for (int u = 0; u < DEC_STEP; ++u) {
                const int j = kb + u;
                if (j < sp.lo || j > sp.hi) continue;
                const int page = entry(j);
                if (!paged_ok(a.p, page)) continue;
                int shift = a.p.shift;
                asm volatile("" : "+s"(shift));  // this rare path must not cost registers: no addresses formed ahead,
                const int64_t at = paged_head(a.p, page, kvh) + (j & mask) + ((int64_t)(quad * 4) << shift);
#pragma unroll
                for (int b = 0; b < D::VB; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float z = cached<TYPE>(a.p.v, at + ((int64_t)(16 * b + r) << shift));
                        if (not_finite(z) && j >= lo && j <= hi) acc[b][r] += z;
                        asm volatile("" : "+s"(shift)::"memory");  // and one value at a time
                    }
            }
        }
    }

    if (D::LOW)
#pragma unroll
        for (int b = 0; b < D::VB; ++b) acc[b] += low[b] * PagedType<TYPE>::LOW_DOWN;
    // the row's sum over its four lanes, then the four wavefronts' sums
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (quad == 0) {
        c_l[wave][m] = c;
        l_l[wave][m] = l;
    }
#pragma unroll
    for (int b = 0; b < D::VB; ++b) *(pf4 *)&acc_l[wave][m][16 * b + quad * 4] = acc[b];
    __syncthreads();
    const int64_t at = ((int64_t)s * nkv + kvh) * a.ds + split;
    float *part = a.dsum.part + at * a.drows * HD, *stat = a.dsum.stat + at * a.drows * 2;
    for (int x = tid; x < R * (HD / 4); x += 256) {
        const int r = x / (HD / 4), d = 4 * (x - r * (HD / 4));
        const float cm = fminf(fminf(c_l[0][r], c_l[1][r]), fminf(c_l[2][r], c_l[3][r]));
        pf4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        float lr = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(cm - c_l[w][r]);
            lr += f * l_l[w][r];
            o += f * *(const pf4 *)&acc_l[w][r][d];
        }
        const int64_t t = q.t0 + r / G;
        const int h = kvh * G + r % G;
        if (ch.used == 1) *(pf4 *)(a.o + t * a.ldo + (int64_t)h * HD + d) = o * (1.0f / lr);
        else {
            *(pf4 *)(part + r * HD + d) = o;
            if (d == 0) *(pf2 *)(stat + 2 * r) = pf2{cm, lr};
        }
    }
}

}  // namespace fgh
