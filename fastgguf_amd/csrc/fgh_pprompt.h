// fgh_pprompt.h - paged attention of many rows per K / V head: prompts.
//
// A workgroup takes 128 rows of a sequence and K / V head (row = new token x the head's query heads + query head, so the
// heads that share K and V share its tiles), 32 a wavefront, and goes over their positions in tiles of KT; or 64 rows, with two
// wavefronts to 32 of them that take half of every tile each and add their sums up at the end, where workgroups are few. K and V^T
// tiles come into LDS by direct loads (16 bytes a lane), two tiles deep: the next one is on its way while this one is used.
//   S^T = K q^T: 32 x 32 x 16 products, A = 32 K rows out of LDS, B = q in registers. LDS row m of a 16-position block holds position
//         (m & 3) | (m & 8) >> 1 | (m & 4) << 1, so that a lane's 16 scores of 32 positions are two runs of 8 positions,
//   O^T += V^T P^T: which are what it has to give as B. Neither scores nor weights leave their lane; a row's maximum takes
//         one exchange with the lane 32 away, and only where the row's reference has to follow it.
// 16-byte words of a row are kept in LDS at (word ^ row), so that lanes that read the same word of neighbouring rows
// meet in no bank.
//
// F16's sums over the weights' second halves are formed apart (fgh_pattn.h), by blocks of 32 values, each over the whole tile and added to the
// others while the next one's products run: registers for all of them at once there are none, and added per 32 positions they would take
// twice the vector instructions.
//
// Bound by the matrix pipe, for the 2 (F16) to 6 (F32) products that an fp32 result takes: 8192 tokens, f16, 32 heads over 8, hd 128 take
// 975 to 1000 us by the card, 1.10 to 1.13 PFLOP/s of products, 1.15 for a large f16 matrix product here, with the clock held
// down by power. Small batches are bound by what a tile costs a wavefront that is alone on its SIMD (64 tokens behind
// 4032: 27.5 us with the join; asking for the next tile took 1500 of a tile's 5500 cycles there before its loads' places were formed from
// one lane's by other bits). Three tiles deep gained nothing there: the tiles are in time.
#pragma once

#include "fgh_pattn.h"

namespace fgh {

// RW: wavefronts along the rows, 4, or 2 with the four in pairs that take half a tile's positions each
template <int TYPE, int HD, int RW>
struct Pro {
    static constexpr int ES = PagedType<TYPE>::ES, NQ = PagedType<TYPE>::NQ, NK = PagedType<TYPE>::NK;
    static constexpr int W = ES / 2;           // 16-byte words of 8 values
    static constexpr int ROWS = 32 * RW, PW = 4 / RW;
    static constexpr int KT = HD * ES > 512 ? 32 : 64;
    static constexpr int KS = HD / 16;         // steps of 16 along the head
    static constexpr int VB = (HD + 31) / 32;  // blocks of 32 of V's values
    static constexpr int KD = HD * ES / 16;    // words of a K row
    static constexpr int KW = KD <= 8 ? 8 : KD <= 16 ? 16 : KD <= 32 ? 32 : 64;  // and their places in LDS
    static constexpr int VW = KT * ES / 16;    // words of a V^T row
    static constexpr int KBYTES = KT * KW * 16;
    static constexpr int VROWS = VB * 32;      // with the rows behind hd 80, never loaded, their sums never stored
    static constexpr int VBYTES = VROWS * KT * ES;
    static constexpr int BYTES = KBYTES + VBYTES;
    static constexpr int LDS = 2 * BYTES + 16 + (PW > 1 ? RW * 512 : 0);
    static_assert(PW == 1 || (KT == 64 && RW * VB * 4096 <= 2 * BYTES - 16384), "a block for every wavefront, its sums beside the rows' staging");
    static constexpr int OCC = HD > 128 || (TYPE == T_F32 && HD > 64) ? 1 : 2;
    // The loads' places kept in registers, where there are any left: 64 tokens behind 4032, f16, hd 128 take 27.7 us so and 28.7
    // otherwise, 8192 975 and 985; 1008 tokens behind 7168, bf16, 327 with spills and 309.
    static constexpr bool KEEP = !(NQ > 2 && HD == 128 && RW == 4);
    static constexpr int KL = KT / 4 * KW / 64;           // direct loads of a wavefront for its KT / 4 K rows
    static constexpr int VL = HD * VW / 64;               // and of all four for V
};

// what a row's words are kept at: word w of row r at w ^ turn(r)
template <int NW>
__device__ __forceinline__ int turn(int r) {
    return NW == 4 ? r >> 1 & 3 : r & (NW < 16 ? NW - 1 : 15);
}
// LDS row of a 16-position block <-> position
__device__ __forceinline__ int swap_rows(int m) { return (m & ~12) | (m & 8) >> 1 | (m & 4) << 1; }

__device__ __forceinline__ void lds_load16(const uint8_t *src, uint8_t *dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
}

template <int TYPE, int HD, int RW>
__device__ __forceinline__ void paged_prompt_block(const PagedAttnArgs &a, int block, int blocks, int split, uint8_t *lds) {
    using P = Pro<TYPE, HD, RW>;
    constexpr int KT = P::KT, ES = P::ES, W = P::W;
    uint32_t *odd_l = (uint32_t *)(lds + 2 * P::BYTES);  // positions of the tile with a V value that is not finite
    const int nkv = a.p.n_head_kv, G = a.n_head / nkv;
    const int kvh = block % nkv;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // tiles in reverse: those late in a sequence have the most positions and start first
    const PagedTile tl = paged_tile(a, P::ROWS, (blocks - 1 - block) / nkv);
    const int64_t slot = (int64_t)tl.index * nkv + kvh;
    const PagedSeq q = tl.q;
    if (a.ps > 1 && split == 0 && tid == 0 && (tl.s < 0 || !q.ok)) a.psum.info[slot].used = 0;
    if (tl.s < 0) return;
    const int s = tl.s, r0 = tl.r0, R = min(P::ROWS, q.n * G - r0);
    if (!q.ok) {
        if (split == 0)
            for (int64_t i = tid; i < (int64_t)R * HD; i += 256) {
                const int r = r0 + (int)(i / HD), x = (int)(i % HD);
                a.o[(q.t0 + r / G) * a.ldo + (int64_t)(kvh * G + r % G) * HD + x] = __builtin_nanf("");
            }
        return;
    }
    const int prefix = paged_prefix(a, s, q);
    const PagedSpan sp = paged_span(a, q, prefix, r0 / G, (r0 + R - 1) / G);
    const PagedChunk ch = paged_chunk(pro_units(sp), a.ps, PRO_LEAST, 1);
    if (split >= ch.used) return;
    if (a.ps > 1 && split == 0 && tid == 0) a.psum.info[slot] = PagedSlot{ch.used, R, q.t0, r0};
    const int ubase = sp.lo & ~(PRO_UNIT - 1);  // the split's positions k0 .. k1, whole units but for the range's ends
    const int k0 = max(sp.lo & ~(KT - 1), ubase + split * ch.per * PRO_UNIT), k1 = min(sp.hi, ubase + (split + 1) * ch.per * PRO_UNIT - 1);

    // this lane's row: column lane % 32 of the wavefront's products
    const int half = lane >> 5, rg = wave % RW, pg = wave / RW, wr = rg * 32 + (lane & 31);
    const bool mine = wr < R;
    const int row = r0 + (mine ? wr : 0), tok = row / G, head = kvh * G + row - tok * G;
    const int pos = q.len - q.n + tok;
    const int lo = mine ? row_lo(a, pos) : 0x7fffffff, hi = mine ? max(pos, prefix - 1) : -1;

    const int mask = (1 << a.p.shift) - 1;
    const int32_t *table = a.p.table + (int64_t)s * a.p.table_stride;
    // Direct loads: V^T's are loads wave, wave + 4, .. of VR rows, a lane's word at the same positions (v_pos) in all of them; K's are of
    // this wavefront's KT / 4 LDS rows, positions of one 16-block. A lane asks for the page of its V positions one tile ahead; the
    // K rows' page is that of lane k_from.
    constexpr int NE = KT / 16, VR = 64 / P::VW, KR = 64 / P::KW;
    const int kr0 = wave * (KT / 4), kblk = kr0 & ~15;
    const int k_from = (kblk * ES / 16) ^ turn<P::VW>(wave * VR);
    auto lane_now = [&]() {  // what follows from it is kept, or formed for every tile
        int ln = lane;
        if (!P::KEEP) asm volatile("" : "+v"(ln));
        return ln;
    };
    auto v_row = [&](int ln) { return wave * VR + ln / P::VW; };
    auto v_pos = [&](int ln) { return (ln % P::VW ^ turn<P::VW>(v_row(ln))) * (16 / ES); };
    int ent = 0;
    auto pages = [&](int kb) { ent = table[min(kb + v_pos(lane_now()), sp.hi) >> a.p.shift]; };
    const int64_t hsize = (int64_t)kvh * HD << a.p.shift;
    uint32_t gone_next = 0;  // 16-position blocks of the next tile whose page does not exist
    auto load = [&](int kb, uint8_t *buf) {
        const int ln = lane_now(), vj = v_pos(ln);
        const int kq = (kr0 & 15) | ln / P::KW, kw = (ln % P::KW) ^ turn<P::KW>(kq), krow = swap_rows(kq) * HD * ES;
        const bool ok = paged_ok(a.p, ent);
        const int page = ok ? ent : 0;
        gone_next = 0;
        if (__builtin_amdgcn_ballot_w64(!ok) != 0)
#pragma unroll
            for (int e = 0; e < NE; ++e) gone_next |= __builtin_amdgcn_ballot_w64(!ok && vj / 16 == e) ? 1u << e : 0u;
        const uint8_t *kp = a.p.k + (__builtin_amdgcn_readlane(page, k_from) * a.p.page_stride + hsize + (int64_t)((kb + kblk) & mask) * HD) * ES;
#pragma unroll
        for (int i = 0; i < P::KL; ++i) {  // KR rows on: other bits of the row, so of its turn and its place
            const int w = kw ^ turn<P::KW>(i * KR);
            if (P::KD == P::KW || w < P::KD)
                lds_load16(kp + (uint32_t)(krow + w * 16) + swap_rows(i * KR) * HD * ES, buf + kr0 * P::KW * 16 + i * 1024);
        }
        const uint8_t *vp = a.p.v + (page * a.p.page_stride + hsize + ((int64_t)v_row(ln) << a.p.shift) + ((kb + vj) & mask)) * ES;
#pragma unroll
        for (int i = 0; i < (P::VL + 3) / 4; ++i)  // 4 VR rows on: the same turn
            if (P::VL % 4 == 0 || wave + 4 * i < P::VL)
                lds_load16(vp + (((uint32_t)(4 * VR * i) << a.p.shift) * ES), buf + P::KBYTES + (wave + 4 * i) * 1024);
    };
    int kb = k0;
    pages(kb);
    // q rows come in pieces of 32 values, 8 lanes a row, and change places in this wavefront's 4 KB of the second
    // buffer; so do the outputs. (A lane's own row straight from memory, 16 bytes of 32 rows a load, took 64 cycles a load.)
    uint8_t *own = lds + wave * 4096 + (2 * P::BYTES - 16384);
    struct Place {
        int64_t tok;
        uint32_t head;
    };
    auto place = [&](int r) {  // row r of this wavefront in q and o (past the last: the last)
        const int z = r0 + min(rg * 32 + r, R - 1), t = z / G;
        return Place{q.t0 + t, (uint32_t)((kvh * G + z - t * G) * HD)};
    };
    constexpr int QP = (HD + 31) / 32;
    pf4 qv[QP][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int rr = lane >> 3, rw = lane & 7;
        const Place at = place(8 * u + rr);
        const float *src = a.q + at.tok * a.ldq + at.head + 4 * rw;
#pragma unroll
        for (int g = 0; g < QP; ++g) qv[g][u] = *(const pf4 *)(src + (HD % 32 != 0 && g == QP - 1 && rw >= HD % 32 / 4 ? 0 : 32 * g));
    }
    load(kb, lds);
    uint32_t gone = gone_next;
    if (kb + KT <= k1) pages(kb + KT);

    pu4 qp[P::KS][P::NQ];
    PagedScore score;
    {
        float size = scale_size(a.scale);
        if constexpr (TYPE == T_F16) {  // the rows' largest magnitudes
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float m = 0.0f;
#pragma unroll
                for (int g = 0; g < QP; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(qv[g][u][e]));
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
                ((float *)own)[8 * u + (lane >> 3)] = m;
            }
            size = row_size(((const float *)own)[lane & 31]);
        }
        const float inv = q_factor(a.scale, size);
#pragma unroll
        for (int g = 0; g < QP; ++g) {
#pragma unroll
            for (int u = 0; u < 4; ++u) *(pf4 *)(own + (8 * u + (lane >> 3)) * 128 + ((lane ^ lane >> 3) & 7) * 16) = qv[g][u];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (2 * g + k < P::KS) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const pf4 z = *(const pf4 *)(own + (lane & 31) * 128 + ((4 * k + 2 * half + e) ^ (lane & 7)) * 16);
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[4 * e + i] = mine ? z[i] * inv : 0.0f;
                    }
                    parts8<TYPE, P::NQ>(x, qp[2 * g + k]);
                }
        }
        score = paged_score(a, head, size);
    }

    pf16 acc[P::VB];
#pragma unroll
    for (int b = 0; b < P::VB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][r] = 0.0f;
    float c = __FLT_MAX__, l = 0.0f;

    // where this lane's words are: the K row it gives, and the V^T row; word w of either at (place ^ 16 w)
    // (of the second block, where the wavefront takes that)
    const uint32_t k_at = (pg * 32 + (lane & 31)) * P::KW * 16 + ((half * W) ^ turn<P::KW>(lane & 31)) * 16;
    const uint32_t v_at = P::KBYTES + (lane & 31) * P::VW * 16 + ((half * W) ^ turn<P::VW>(lane & 31) ^ (pg * 4 * W)) * 16;
    const int first = max(sp.lo, k0), last = min(sp.hi, k1);  // the positions that count here

    // A tile in blocks of 32 positions, h: scores S(h), weights W(h), sums. The products of S(1) are issued among the
    // vector instructions of W(0), and those of the sums over block 0 among W(1)'s: a product takes the matrix pipe for 32 cycles, in which
    // the wavefront can issue 8 vector instructions.
    constexpr int NH = KT / 32 / P::PW, AHEAD = P::NQ > 2 ? 2 : 3, SLOTS = AHEAD + 1;  // LDS words read ahead of the products that take them
    struct Weights {
        float v[2][8];  // scores, then weights, of this lane's positions 16 kk + 8 half + e of the block
        float mul;
        pu4 pp[2][P::NQ];
    };
    // weight e, and the parts of two
    auto weigh = [&](Weights &w, int e) {
        float &v = w.v[e / 8][e % 8];
        v = __builtin_amdgcn_exp2f(__builtin_fmaf(v, w.mul, c));
        l += v;
        asm volatile("" : "+v"(v), "+v"(l));  // here, not where they are used
        if (e % 2 == 1) {
            parts2<TYPE, P::NQ>(w.v[e / 8][e % 8 - 1], v, e % 8 / 2, w.pp[e / 8], PagedType<TYPE>::LOW_UP);
#pragma unroll
            for (int i = 0; i < P::NQ; ++i) {
                uint32_t z = w.pp[e / 8][i][e % 8 / 2];
                asm volatile("" : "+v"(z));
                w.pp[e / 8][i][e % 8 / 2] = z;
            }
        }
    };
    // the scores' forms, and what of them is not seen; the row's reference follows them. False: it does not have to.
    const bool plain = !(score.cap_out > 0.0f) && !score.bias;
    auto forms = [&](Weights &w, int j, bool whole) {
        w.mul = score.mul;
        if (!(plain && whole)) {
            if (!plain)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) w.mul = score.apply(w.v[kk], j + kk * 16 + half * 8, pos);
            if (!whole)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const int j0 = j + kk * 16 + half * 8, l0 = max(lo, first) - j0, h0 = min(hi, last) - j0;
                    const bool no = gone >> ((j0 - kb) >> 4) & 1;
#pragma unroll
                    for (int e = 0; e < 8; ++e) w.v[kk][e] = e < l0 || e > h0 ? -__builtin_inff() : no ? __builtin_nanf("") : w.v[kk][e];
                }
        }
        float top = w.v[0][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, w.v[e / 8][e % 8]);
        return top * w.mul;
    };
    bool big = false;  // a reference beyond SCORE_BIG
    // the row's reference follows a larger score, in whole powers of two; the factor of what was formed before
    auto follow = [&](float top) {
        const float mx = fmaxf(top, __shfl_xor(top, 32, 64));
        float f = 1.0f;
        big = big || __builtin_amdgcn_ballot_w64(mx + c > PagedType<TYPE>::PTOP && score_big(mx)) != 0;
        if (mx + c > PagedType<TYPE>::PTOP) {
            const float cn = score_bias<TYPE>(mx) - ceilf(mx);
            f = __builtin_amdgcn_exp2f(cn - c);
            c = cn;
            l *= f;
#pragma unroll
            for (int b = 0; b < P::VB; ++b) acc[b] *= f;
        }
        return f;
    };
    auto round_big = [&](Weights &w) {
        if (big) {
#pragma unroll
            for (int e = 0; e < 16; ++e) w.v[e / 8][e % 8] *= w.mul;
            w.mul = 1.0f;
        }
    };
    auto tile = [&](const uint8_t *buf, bool whole) {
        uint32_t k_lane = k_at, v_lane = v_at;
        asm volatile("" : "+v"(k_lane), "+v"(v_lane));  // the words' places are formed where they are read, not kept
        pu4 raw[SLOTS][W];
        auto read_k = [&](int h, int ks) {
#pragma unroll
            for (int w = 0; w < W; ++w) raw[ks % SLOTS][w] = *(const pu4 *)(buf + (k_lane ^ (2 * ks * W + w) * 16) + h * 32 * P::KW * 16);
        };
        // V's words of the tile, in the order in which they are used: a block of positions' runs of 16, the blocks of values of each;
        // where the weights' second parts are summed by themselves (LOW) the first block so, then both by blocks of values
        constexpr bool LOW = PagedType<TYPE>::LOW > 0;
        constexpr int NX = 2 * P::VB, NA = LOW && NH == 1 ? 0 : LOW ? NX : NH * NX, NV = NA + (LOW ? NH * NX : 0);
        auto read_v = [&](int y) {
            const int k = y < NA ? y / P::VB : (y - NA) % (2 * NH), b = y < NA ? y % P::VB : (y - NA) / (2 * NH);
#pragma unroll
            for (int w = 0; w < W; ++w) raw[y % SLOTS][w] = *(const pu4 *)(buf + (v_lane ^ (2 * k * W + w) * 16) + b * 32 * P::VW * 16);
        };
        constexpr int NPROD = PagedType<TYPE>::NPROD;
        auto beside = [&](int m, int of, auto side) {  // product m of `of`: its share of the 16 weights beside it
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e >= m * 16 / of && e < (m + 1) * 16 / of) side(e);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto scores = [&](int h, Weights &out, auto side) {
            int m = 0;
            // the first parts' products apart from the others', which are small: fewer roundings at the scores' size, where
            // there are registers for it
            pf16 sc, rest;
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = rest[r] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < AHEAD; ++ks) read_k(h, ks);
#pragma unroll
            for (int ks = 0; ks < P::KS; ++ks) {
                if (ks + AHEAD < P::KS) read_k(h, ks + AHEAD);
                pu4 kp[P::NK];
                cache8<TYPE>(raw[ks % SLOTS], kp);
#pragma unroll
                for (int x = P::NQ - 1; x >= 0; --x)
#pragma unroll
                    for (int y = P::NK - 1; y >= 0; --y)
                        if (x + y < 3) {
                            mma32<TYPE>(x + y == 0 || P::PW == 1 ? sc : rest, kp[y], qp[ks][x]);
                            beside(m++, P::KS * NPROD, side);
                        }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) out.v[e / 8][e % 8] = P::PW == 1 ? sc[e] : sc[e] + rest[e];
        };
        auto sums = [&](int h, const Weights &w, auto side) {
            constexpr int NS = LOW ? 1 : NPROD;  // products of a word
            int m = 0;
#pragma unroll
            for (int x = 0; x < NX; ++x) {
                const int at = h * NX + x;
                if (at + AHEAD < NV) read_v(at + AHEAD);
                pu4 vp[P::NK];
                cache8<TYPE>(raw[at % SLOTS], vp);
#pragma unroll
                for (int i = P::NQ - 1; i >= 0; --i)
#pragma unroll
                    for (int y = P::NK - 1; y >= 0; --y)
                        if (i + y < 3 && !(LOW && i > 0)) {
                            mma32<TYPE>(acc[x % P::VB], vp[y], w.pp[x / P::VB][i]);
                            beside(m++, NX * NS, side);
                        }
            }
        };
        // what is left of the tile's sums, by blocks of values: those of the second parts, added while the next block's are formed, and
        // those of the first parts that `sums` has not taken
        auto sums_low = [&](const Weights &w0, const Weights &w1) {
            pf16 low[2];
            auto add = [&](int b, int r) { acc[b][r] = __builtin_fmaf(low[b % 2][r], PagedType<TYPE>::LOW_DOWN, acc[b][r]); };
#pragma unroll
            for (int b = 0; b < P::VB; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) low[b % 2][r] = 0.0f;
                int m = 0;
#pragma unroll
                for (int k = 0; k < 2 * NH; ++k) {
                    const int at = NA + b * 2 * NH + k;
                    if (at + AHEAD < NV) read_v(at + AHEAD);
                    const Weights &w = k < 2 ? w0 : w1;
#pragma unroll
                    for (int i = 1; i >= 0; --i)
                        if (i == 1 || k >= 2 * NH - 2) {
                            mma32<TYPE>(i == 1 ? low[b % 2] : acc[b], raw[at % SLOTS][0], w.pp[k % 2][i]);
                            beside(m++, 2 * NH + 2, [&](int e) {
                                if (b > 0) add(b - 1, e);
                            });
                        }
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) add(P::VB - 1, r);
        };
        auto first_v = [&]() {
#pragma unroll
            for (int x = 0; x < AHEAD; ++x) read_v(x);
        };
        Weights w0;
        auto alone = [](int) {};
        scores(0, w0, alone);
        if constexpr (NH == 1) first_v();
        const float top0 = forms(w0, kb + pg * 32, whole);
        if (__builtin_amdgcn_ballot_w64(top0 + c > PagedType<TYPE>::PTOP)) follow(top0);
        round_big(w0);
        if constexpr (NH == 1) {
#pragma unroll
            for (int e = 0; e < 16; ++e) weigh(w0, e);
            if constexpr (LOW) sums_low(w0, w0);
            else sums(0, w0, alone);
        } else {
            Weights w1;
            scores(1, w1, [&](int e) { weigh(w0, e); });
            first_v();
            const float top1 = forms(w1, kb + 32, whole);
            if (__builtin_amdgcn_ballot_w64(top1 + c > PagedType<TYPE>::PTOP)) {  // block 0's weights wait for their sums
                const float f = follow(top1);
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) scale8<TYPE, P::NQ>(w0.pp[kk], f);
            }
            round_big(w1);
            sums(0, w0, [&](int e) { weigh(w1, e); });
            if constexpr (LOW) sums_low(w0, w1);
            else sums(1, w1, alone);
        }
    };

    for (int n = 0; kb <= k1; kb += KT, n ^= 1) {
        uint8_t *buf = lds + n * P::BYTES;
        __builtin_amdgcn_s_waitcnt(0xF70);  // vmcnt 0: this wavefront's part of the tile is in LDS
        __syncthreads();                    // everyone's is, and the other buffer has been read
        if (kb + KT <= k1) {
            load(kb + KT, lds + (n ^ 1) * P::BYTES);
            if (kb + 2 * KT <= k1) pages(kb + 2 * KT);
        }
        const bool whole = kb >= max(sp.in_lo, k0) && kb + KT - 1 <= min(sp.in_hi, k1) && gone == 0;  // seen by every row
        uint64_t odd = 0;
        if (!whole) {
            // V values at positions that no row sees become zeros, and so do those that are not finite: what only some of
            // the rows see must not reach the others by way of 0 x NaN. The rows that see them get them below.
            if (tid < 2) odd_l[tid] = 0;
            __syncthreads();
            for (int x = tid; x < HD * P::VW; x += 256) {
                const int r = x / P::VW, at = x % P::VW, j = (at ^ turn<P::VW>(r)) * (16 / ES);
                pu4 *word = (pu4 *)(buf + P::KBYTES + (r * P::VW + at) * 16);
                // of the word's values (all in one page): from .. to - 1 are seen by some row
                constexpr int N = 16 / ES;
                const bool none = gone >> (j / 16) & 1;
                const int from = none ? N : min(max(first - kb - j, 0), N), to = min(max(last + 1 - kb - j, 0), N);
                pu4 v = *word;
                uint32_t inf = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (ES == 4) v[i] = i >= from && i < to ? v[i] : 0u;
                    else v[i] &= (2 * i >= from && 2 * i < to ? 0x0000ffffu : 0u) | (2 * i + 1 >= from && 2 * i + 1 < to ? 0xffff0000u : 0u);
                    inf |= infinite<TYPE>(v[i]);
                }
                if (inf) {  // rare
                    uint32_t bad = 0;
#pragma unroll
                    for (int e = 0; e < N; ++e) bad |= raw_bad<TYPE>(&v, e) ? 1u << e : 0u;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = finite_only<TYPE>(v[i]);
                    atomicOr(&odd_l[j / 32], bad << (j & 31));
                }
                if (inf || from > 0 || to < N) *word = v;
            }
            __syncthreads();
            odd = (uint32_t)__builtin_amdgcn_readfirstlane((int)odd_l[0]) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)odd_l[1]) << 32;
        }
        tile(buf, whole);
        while (odd) {
            const int j = kb + __builtin_ctzll(odd);
            odd &= odd - 1;
            if (P::PW > 1 && (j - kb) / 32 != pg) continue;
            int shift = a.p.shift;
            asm volatile("" : "+s"(shift));  // this rare path must not cost registers: no addresses formed ahead,
            const int64_t at = paged_head(a.p, table[j >> shift], kvh) + (j & mask) + ((int64_t)(4 * half) << shift);
#pragma unroll
            for (int b = 0; b < P::VB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = 32 * b + 8 * (r / 4) + r % 4;
                    if (HD % 32 == 0 || d + 4 * half < HD) {
                        const float z = cached<TYPE>(a.p.v, at + ((int64_t)d << shift));
                        if (not_finite(z) && j >= lo && j <= hi) acc[b][r] += z;
                        asm volatile("" : "+s"(shift)::"memory");  // and one value at a time
                    }
                }
        }
        gone = gone_next;
    }
    l += __shfl_xor(l, 32, 64);
    if constexpr (P::PW > 1) {  // the pair's sums come together in the first of the two
        pf4 *sum_l = (pf4 *)lds + rg * P::VB * 4 * 64 + lane;
        pf2 *stat_l = (pf2 *)(lds + 2 * P::BYTES + 16) + rg * 64 + lane;
        __syncthreads();
        if (pg == 1) {
            *stat_l = pf2{c, l};
#pragma unroll
            for (int b = 0; b < P::VB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum_l[(4 * b + i) * 64] = pf4{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]};
        }
        __syncthreads();
        if (pg == 1) return;
        const pf2 other = *stat_l;
        const float cn = fminf(c, other.x), f = __builtin_amdgcn_exp2f(cn - c), g = __builtin_amdgcn_exp2f(cn - other.x);
        c = cn;
        l = l * f + other.y * g;
#pragma unroll
        for (int b = 0; b < P::VB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const pf4 z = sum_l[(4 * b + i) * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[b][4 * i + e] = acc[b][4 * i + e] * f + z[e] * g;
            }
    }
    if (ch.used > 1) {  // sums as the lanes hold them
        if (rg * 32 >= R) return;
        pf4 *part = (pf4 *)a.psum.part + ((slot * a.ps + split) * RW + rg) * (P::VB * 4 * 64) + lane;
#pragma unroll
        for (int b = 0; b < P::VB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                part[(4 * b + i) * 64] = pf4{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]};
        if (half == 0) *(pf2 *)(a.psum.stat + ((slot * a.ps + split) * P::ROWS + wr) * 2) = pf2{c, l};
        return;
    }
    if constexpr (P::PW == 1) __syncthreads();  // the buffers have been read
    const float inv = 1.0f / l;
    int ln = lane;
    asm volatile("" : "+v"(ln));  // the rows' places are formed again rather than kept
    const int rr = ln >> 3, rw = ln & 7;
    Place at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) at[u] = place(8 * u + rr);
#pragma unroll
    for (int b = 0; b < P::VB; ++b) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *(pf4 *)(own + (lane & 31) * 128 + ((2 * i + half) ^ (lane & 7)) * 16) =
                pf4{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]} * inv;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const pf4 z = *(const pf4 *)(own + (8 * u + rr) * 128 + (rw ^ rr) * 16);
            if (rg * 32 + 8 * u + rr < R && (HD % 32 == 0 || 32 * b + 4 * rw < HD))
                *(pf4 *)(a.o + at[u].tok * a.ldo + at[u].head + 32 * b + 4 * rw) = z;
        }
    }
}

}  // namespace fgh
