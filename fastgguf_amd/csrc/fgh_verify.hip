// fgh_verify.hip - drafted tokens against the target's logits, and the token that follows the accepted ones, on gfx950.
//
// Row i of a sequence has p = softmax(logits / T); the draft d behind it stays while u q(d) < p(d). At the first that does not, the
// token is the first one whose running sum of max(p - q, 0) passes v times the whole; behind the last row, of p. The sums
// run over a vocabulary of 10^5 words, and which word v falls on is a matter of their last bits: exponentials, sums and
// comparisons are in 64 bits. A row is read once: each workgroup leaves the largest value of its words, its
// place and the sum of exp((x - largest) / T); whole rows, and the sums that a number has to be compared with, are joined
// from those.
//
// 64 sequences of 1 to 6 rows of 128256 words with the drafter's probabilities take 45 to 49 us: the rows 26 (each with the kernel's start: 20 for reading
// alone, 25 for the exponentials alone, in one kernel they overlap), the rejected rows' sums 15, the choice 7. Few rows are a matter of launches that wait for each
// other and, in the choice, of five loads that do: 8.1 us for one token of one row.
#include "fgh_serve.h"

#include <limits.h>

#include <algorithm>

namespace fgh {

namespace {

// rows are 4-byte aligned: 16 bytes a lane all the same
typedef float vf4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.69314718055994530942;

// 2^(d c) for -1000 <= d c <= 1000, off by 9e-13 of it: the product's nearest whole number by a sum that leaves it in the low bits, which go
// into the exponent, and a polynomial of what is left, at most 1/2 (its coefficients: the least largest error, 1 exactly at 0).
// 11 instructions of 64 bits; with rint, a conversion and an exponent function instead it took twice the time.
__device__ __forceinline__ double exp2_near(double d, double c) {
    const double whole = __builtin_fma(d, c, 0x1.8p52), f = __builtin_fma(d, c, 0x1.8p52 - whole);
    double r = 1.3178933573679677e-06;
    r = __builtin_fma(r, f, 1.5309156297959352e-05);
    r = __builtin_fma(r, f, 1.5403825462941963e-04);
    r = __builtin_fma(r, f, 1.3333454860108985e-03);
    r = __builtin_fma(r, f, 9.6181286161221811e-03);
    r = __builtin_fma(r, f, 5.5504109352666739e-02);
    r = __builtin_fma(r, f, 2.4022650698110606e-01);
    r = __builtin_fma(r, f, 6.9314718054821234e-01);
    r = __builtin_fma(r, f, 1.0);
    const uint64_t u = __builtin_bit_cast(uint64_t, r), n = __builtin_bit_cast(uint64_t, whole);
    return __builtin_bit_cast(double, u + (n << 52));
}
// 2^t: 0 below 2^-1000 and where t is NaN, 2^1000 at most
__device__ __forceinline__ double exp2_of(double t) {
    const double r = exp2_near(fmin(fmax(t, -1000.0), 1000.0), 1.0);
    return t >= -1000.0 ? r : 0.0;
}

// log2(e) / T of a sequence; T = 0, the largest value, has 1's; an infinite one a number that makes every word as likely. A T below 0 or NaN
// makes NaN.
__device__ __forceinline__ double heat_of(const VerifyArgs &a, int s, bool &greedy) {
    const float t = a.temp ? a.temp[s] : 1.0f;
    greedy = t == 0.0f;
    return greedy ? LOG2E : t > 0.0f ? fmax(LOG2E / (double)t, 1e-290) : (double)__builtin_nanf("");
}

// a row, or a part of one: its largest value (NaN where it has a NaN), the first place of it where the largest is asked for, sum of
// 2^((x - top) c)
struct Part {
    double sum;
    float top;
    int at;
};
// the largest value to take others relative to: 0 where there is none
__device__ __forceinline__ double level(float top) { return fabsf(top) <= 3.4028235e38f ? (double)top : 0.0; }
__device__ __forceinline__ float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }  // NaN if either is
// over a wavefront, every lane gets it: 8 steps without LDS
template <class F>
__device__ __forceinline__ int over_lanes(int v, F &&f) {
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));  // row_half_mirror
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));  // row_mirror
    return f(f(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)), f(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ float largest(float x) {
    return __int_as_float(over_lanes(__float_as_int(x), [](int a, int b) { return __float_as_int(larger(__int_as_float(a), __int_as_float(b))); }));
}
__device__ __forceinline__ int least(int x) {
    return over_lanes(x, [](int a, int b) { return min(a, b); });
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)u, (int)u, CTRL, 0xF, 0xF, false),
                   hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(u >> 32), (int)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_of(double x, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double total(double x) {
    x += dpp<0xB1>(x);
    x += dpp<0x4E>(x);
    x += dpp<0x141>(x);
    x += dpp<0x140>(x);
    return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}
template <int CTRL>
__device__ __forceinline__ double dpp0(double x) {  // 0 where no lane is
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, true), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// the sum with the lanes before: in rows of 16 lanes (row_shr 1, 2, 4, 8), then over the rows
__device__ __forceinline__ double upto_lane(double x) {
    const int lane = threadIdx.x & 63;
    x += dpp0<0x111>(x);
    x += dpp0<0x112>(x);
    x += dpp0<0x114>(x);
    x += dpp0<0x118>(x);
    const double a = lane_of(x, 15), b = a + lane_of(x, 31), c = b + lane_of(x, 47);
    return x + (lane < 16 ? 0.0 : lane < 32 ? a : lane < 48 ? b : c);
}
// the parts of a wavefront's lanes, as one; places only where the largest is asked for
__device__ __forceinline__ Part join_lanes(Part p, double c, bool greedy) {
    const float own = p.top;
    p.top = largest(own);
    if (greedy) p.at = least(own == p.top ? p.at : INT_MAX);
    p.sum = total(p.sum * exp2_of(((double)own - level(p.top)) * c));  // 0 for a part without words
    return p;
}

// Each row's largest value and sum, a workgroup to a part of its words, 4 NV words a thread at a time, all of whose loads are under way at
// once. Bound by vector instructions, 76 % of the compute units' busy cycles: 17 a word, of which 13 are of 64 bits, and a third as many again around
// them (64 sequences: 26 us, of which 21 busy and 16 of instructions at 4 cycles each; the rest is the start and the end). (The next
// block's loads a block ahead, at 86 registers instead of 63, gained nothing.)
template <int NV>
__global__ __launch_bounds__(256) void verify_rows_kernel(VerifyArgs a) {
    __shared__ Part lds[4];
    const int groups = (a.splits + a.group - 1) / a.group, row = blockIdx.x / groups, split0 = (blockIdx.x - row * groups) * a.group, tid = threadIdx.x;
    const float *x = a.logits + row * a.ld;
    vf4 v[NV] = {};
    auto load = [&](int base) {  // behind the last four words those again
        if (a.vocab >= 4)
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = *(const vf4 *)((const uint8_t *)x + 4 * (uint32_t)min(base + i * 1024 + 4 * tid, a.vocab - 4));
        else
            for (int e = 0; e < a.vocab; ++e) v[0][e] = x[e];
    };
    auto cut = [&](int base) {  // a row's last block: a lane's words from its first one on, then none
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = base + i * 1024 + 4 * tid, over = a.vocab >= 4 ? max(0, j - (a.vocab - 4)) : 0;
            if (over & 1) v[i] = vf4{v[i].y, v[i].z, v[i].w, v[i].w};
            if (over & 2) v[i] = vf4{v[i].z, v[i].w, v[i].w, v[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e >= a.vocab) v[i][e] = -__builtin_inff();
        }
    };
    const int s = seq_of_row(a.tok, a.n_seq, row);
    if (s < 0) return;
    load(split0 * a.per);  // rows of no sequence, of which a recorded call may have many, are not read (asked for before the search: 0.3 to 1.4 us more)
    bool greedy;
    const double c = heat_of(a, s, greedy), least_d = -1000.0 / c;
    for (int split = split0; split < min(a.splits, split0 + a.group); ++split) {
        const int from = split * a.per, to = min(a.vocab, from + a.per);
        Part p{0.0, -__builtin_inff(), INT_MAX};  // a wavefront's: the sum still a lane's
        for (int base = from; base < to; base += 1024 * NV) {
            if (base != split0 * a.per) load(base);
            if (base + 1024 * NV > a.vocab) cut(base);
            const float was = p.top;
            float own = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < NV; ++i) own = larger(larger(own, larger(v[i].x, v[i].y)), larger(v[i].z, v[i].w));
            p.top = larger(was, largest(own));
            if (greedy && p.top > was) {  // a lane's words rise: its first one that is as large
                p.at = INT_MAX;
#pragma unroll
                for (int i = NV - 1; i >= 0; --i)
#pragma unroll
                    for (int e = 3; e >= 0; --e)
                        if (v[i][e] == p.top) p.at = base + i * 1024 + 4 * tid + e;
            }
            const double m = level(p.top);
            if (base != from) p.sum *= exp2_of(((double)was - m) * c);
            // a word that is none, and a NaN, add 2^-1000
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) p.sum += exp2_near(fmax((double)v[i][e] - m, least_d), c);
        }
        p.sum = total(p.sum);
        if (greedy) p.at = least(p.at);
        if (split != split0) __syncthreads();
        if ((tid & 63) == 0) lds[tid >> 6] = p;
        __syncthreads();
        if (tid < 64) {
            p = join_lanes(tid < 4 ? lds[tid] : Part{0.0, -__builtin_inff(), INT_MAX}, c, greedy);
            if (tid == 0) {
                const int64_t i = (int64_t)row * a.splits + split;
                a.sum[i] = p.sum, a.top[i] = p.top, a.at[i] = p.at;
            }
        }
    }
}

constexpr int MOST_SPLITS = 64;  // parts of a row: a wavefront joins them
constexpr int WG = 512;  // threads that decide: 8 rows at a time

// the sequence's rows: none for what a batch cannot mean
__device__ __forceinline__ int2 rows_of(const VerifyArgs &a, int s) {
    const int b = a.tok[s], e = a.tok[s + 1];
    if (b < 0 || e > a.n_tok || e <= b || e - b > a.max_tok) return int2{0, 0};
    return int2{b, e - b};
}
// by a workgroup, a wavefront to a row, 8 rows at a time until one is rejected (all of them where `lse` is written)
__device__ VerifyChoice decide(const VerifyArgs &a, int s, double c, bool greedy, bool lse) {
    __shared__ Part rows[WG / 64];
    __shared__ int ok[WG / 64], word[WG / 64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int2 r = rows_of(a, s);
    VerifyChoice ch{0.0, 0.0f, 0, -1, -1, r.y, 0};
    bool open = true;
    for (int i0 = 0; i0 < r.y && (open || lse); i0 += WG / 64) {
        const int i = i0 + wave, t = r.x + i;
        if (i < r.y) {
            Part p{0.0, -__builtin_inff(), INT_MAX};
            if (lane < a.splits) {
                const int64_t k = (int64_t)t * a.splits + lane;
                p = Part{a.sum[k], a.top[k], a.at[k]};
            }
            const int d = i < r.y - 1 ? a.tokens[t + 1] : -1;
            const bool is_word = (uint32_t)d < (uint32_t)a.vocab;
            float x = 0.0f, u = 0.0f, q = 0.0f, q_lse = 0.0f;
            if (is_word) {
                x = a.logits[t * a.ld + d], u = a.u[t];
                if (a.q) q = a.q[t * a.ldq + d], q_lse = a.q_lse[t];
            }
            p = join_lanes(p, c, greedy);
            bool good = false;
            if (is_word && fabsf(p.top) <= 3.4028235e38f) {
                if (greedy) good = d == p.at;
                else {
                    const double under = (double)q * c - (double)q_lse * LOG2E;  // NaN passes no test
                    const double chance = !a.q ? 1.0 : under == under ? exp2_of(under) : under;
                    good = (double)u * chance < exp2_of(((double)x - p.top) * c) / p.sum && c == c;
                }
            }
            if (lane == 0) {
                rows[wave] = p, ok[wave] = good, word[wave] = is_word ? d : -1;  // no word: the token is drawn from p
                if (lse) a.lse[t] = p.top != p.top || c != c ? __builtin_nanf("") : fabsf(p.top) <= 3.4028235e38f ? (float)((double)p.top * c * LN2 + log(p.sum)) : p.top;
            }
        }
        __syncthreads();
        for (int w = 0; w < WG / 64 && open && i0 + w < r.y; ++w) {
            const bool last = i0 + w == r.y - 1;
            if (!last && ok[w]) {
                ++ch.good;
                continue;
            }
            open = false;
            ch.sum = rows[w].sum, ch.top = rows[w].top, ch.at = rows[w].at, ch.t = r.x + i0 + w, ch.d = last ? -1 : word[w];
        }
        __syncthreads();
    }
    return ch;
}

// a word's weight in the choice of the next token
enum { FROM_P, WITHOUT_DRAFT, FROM_REST };
struct Weigh {
    const float *x, *q;
    double m, c, z, lse, least_d;  // the row's largest, log2(e) / T, 1 / the sum, the draft row's lse in powers of two, -1000 / c
    int d;
};
template <int MODE>
__device__ __forceinline__ double weight(const Weigh &w, int j, float x, float q) {
    if (MODE == FROM_REST)  // a word that cannot be has 2^-1000 in p, and 2^-990 or more in q
        return fmax(__builtin_fma(exp2_near(fmax((double)x - w.m, w.least_d), w.c), w.z, -exp2_near(fmin(fmax(__builtin_fma((double)q, w.c, -w.lse), -990.0), 1000.0), 1.0)), 0.0);
    const double p = exp2_of(((double)x - w.m) * w.c);
    return MODE == WITHOUT_DRAFT && j == w.d ? 0.0 : p;
}
__device__ __forceinline__ Weigh weigh_of(const VerifyArgs &a, const VerifyChoice &ch, double c) {
    Weigh w;
    w.x = a.logits + ch.t * a.ld, w.q = a.q ? a.q + ch.t * a.ldq : nullptr;
    w.m = level(ch.top), w.c = c, w.z = 1.0 / ch.sum, w.lse = a.q ? (double)a.q_lse[ch.t] * LOG2E : 0.0, w.d = ch.d, w.least_d = -1000.0 / c;
    return w;
}
// f(first word, weights of 4) of a thread's words b .. e - 1
template <int MODE, class F>
__device__ __forceinline__ void each4(const Weigh &w, int b, int e, F &&f) {
    for (int j = b; j < e; j += 4) {
        double x[4];
        if (j + 4 <= e) {
            const vf4 p = *(const vf4 *)(w.x + j);
            vf4 q = p;
            if (MODE == FROM_REST) q = *(const vf4 *)(w.q + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = weight<MODE>(w, j + i, p[i], q[i]);
        } else
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = j + i < e ? weight<MODE>(w, j + i, w.x[j + i], MODE == FROM_REST ? w.q[j + i] : 0.0f) : 0.0;
        f(j, x);
    }
}
// over the workgroup: the sum of the wavefronts before, and the whole (v: a wavefront's, the same in its lanes)
__device__ __forceinline__ double2 scan_waves(double v) {
    __shared__ double lds[WG / 64];
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[wave] = v;
    __syncthreads();
    double before = 0.0, all = 0.0;
    for (int i = 0; i < WG / 64; ++i) {
        if (i < wave) before += lds[i];
        all += lds[i];
    }
    return double2{before, all};
}
constexpr int SUB = 4 * WG;                                // words that the workgroup takes at a time
constexpr int MOST_SUBS = (1 << 24) / (MOST_SPLITS * SUB);  // of a part
template <int MODE>
__device__ __forceinline__ double sum_words(const Weigh &w, int from, int to) {
    double v = 0.0;
    for (int b = from + 4 * (int)threadIdx.x; b < to; b += SUB) each4<MODE>(w, b, min(to, b + 4), [&](int, const double (&x)[4]) { v += (x[0] + x[1]) + (x[2] + x[3]); });
    return scan_waves(total(v)).y;
}

// the decision where the drafts have probabilities, and the sums of max(p - q, 0) of a rejected row, by parts of SUB words. Each of a sequence's
// workgroups decides for itself; the first one keeps it for the draw. (A launch for the decisions alone took as long.)
__global__ __launch_bounds__(WG) void verify_rest_kernel(VerifyArgs a) {
    const int s = blockIdx.x / a.splits, split = blockIdx.x - s * a.splits, subs = (a.per + SUB - 1) / SUB;
    bool greedy;
    const double c = heat_of(a, s, greedy);
    if (split > 0 && (greedy || !(c == c))) return;
    const VerifyChoice ch = decide(a, s, c, greedy, a.lse && split == 0);
    if (split == 0 && threadIdx.x == 0) a.choice[s] = ch;
    if (greedy || !(c == c) || ch.d < 0) return;
    const Weigh w = weigh_of(a, ch, c);
    __shared__ double sums[MOST_SUBS][WG / 64];
    const int first = split * a.per, to = min(a.vocab, first + a.per), wave = threadIdx.x >> 6;
    auto load = [&](int i, vf4 &x, vf4 &q) {  // words behind the last: the last again, no weight
        const int j = first + i * SUB + 4 * (int)threadIdx.x;
        if (a.vocab >= 4) {
            const uint32_t o = 4 * (uint32_t)min(j, a.vocab - 4);
            x = *(const vf4 *)((const uint8_t *)w.x + o), q = *(const vf4 *)((const uint8_t *)w.q + o);
        } else
            for (int e = 0; e < a.vocab; ++e) x[e] = w.x[e], q[e] = w.q[e];
    };
    vf4 x{}, q{}, xn{}, qn{};
    load(0, x, q);
    for (int i = 0; i < subs; ++i) {  // the next words on their way, no wavefront waits for another
        if (i + 1 < subs) load(i + 1, xn, qn);
        const int j = first + i * SUB + 4 * (int)threadIdx.x, over = a.vocab >= 4 ? max(0, j - (a.vocab - 4)) : 0;
        double v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = weight<FROM_REST>(w, j, x[e], q[e]);
        if (first + (i + 1) * SUB > to) {  // a row's last words: of four, those from j on
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < over || j - over + e >= to) v[e] = 0.0;
        }
        const double sum = total((v[0] + v[1]) + (v[2] + v[3]));
        if ((threadIdx.x & 63) == 0) sums[i][wave] = sum;
        x = xn, q = qn;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < subs; i += WG) {
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < WG / 64; ++k) v += sums[i][k];
        a.rest[((int64_t)s * a.splits + split) * subs + i] = v;
    }
}

// the first of words from .. to - 1 whose running sum passes `aim`, or the last of any weight (-1: none has)
template <int MODE>
__device__ int pick(const Weigh &w, int from, int to, double aim) {
    __shared__ int firsts[WG / 64], lasts[WG / 64];
    __shared__ double sum;
    const int per = ((to - from + WG - 1) / WG + 3) & ~3, b = min(to, from + (int)threadIdx.x * per), e = min(to, b + per), lane = threadIdx.x & 63;
    double own = 0.0;
    each4<MODE>(w, b, e, [&](int, const double (&x)[4]) { own += (x[0] + x[1]) + (x[2] + x[3]); });
    double run = upto_lane(own);
    run += scan_waves(lane_of(run, 63)).x;
    // the first thread that passes, or the last of any weight (by atomics in LDS, one lane after the other, this took 5 us)
    const uint64_t any = __builtin_amdgcn_ballot_w64(own > 0.0), over = __builtin_amdgcn_ballot_w64(own > 0.0 && run > aim);
    if (lane == 0) {
        const int t = (int)threadIdx.x;
        firsts[t >> 6] = over ? t + __builtin_ctzll(over) : WG;
        lasts[t >> 6] = any ? t + 63 - __builtin_clzll(any) : -1;
    }
    __syncthreads();
    int first = WG, last = -1;
#pragma unroll
    for (int i = 0; i < WG / 64; ++i) first = min(first, firsts[i]), last = max(last, lasts[i]);
    const int mine = first < WG ? first : last;
    if (mine < 0) return -1;
    if ((int)threadIdx.x == mine) sum = run - own;
    __syncthreads();
    // that thread's words, one to a lane
    const int b1 = min(to, from + mine * per), e1 = min(to, b1 + per);
    run = sum;
    int at = -1;
    for (int j0 = b1; j0 < e1; j0 += 64) {
        const int j = j0 + lane;
        const double x = j < e1 ? weight<MODE>(w, j, w.x[j], MODE == FROM_REST ? w.q[j] : 0.0f) : 0.0, upto = run + upto_lane(x);
        const uint64_t some = __builtin_amdgcn_ballot_w64(x > 0.0), past = __builtin_amdgcn_ballot_w64(x > 0.0 && upto > aim);
        if (past) return j0 + __builtin_ctzll(past);
        if (some) at = j0 + 63 - __builtin_clzll(some);
        run = lane_of(upto, 63);
    }
    return at;
}

// The part, then the word. part(i): the sum of part i; there are `subs` of up to `words` words to each split. Each wavefront goes through them for
// itself.
template <int MODE, class F>
__device__ int draw(const VerifyArgs &a, const Weigh &w, int subs, int words, double v, F &&part) {
    const int n = a.splits * subs;
    const int lane = threadIdx.x & 63;
    double whole = 0.0;
    for (int i = 0; i < n; i += 64) whole += total(i + lane < n ? part(i + lane) : 0.0);
    const double aim = v * whole;
    int at = -1;
    double run = 0.0, before = 0.0;
    for (int i = 0; i < n; i += 64) {
        const double x = i + lane < n ? part(i + lane) : 0.0, upto = run + upto_lane(x);
        const uint64_t some = __builtin_amdgcn_ballot_w64(x > 0.0), past = __builtin_amdgcn_ballot_w64(x > 0.0 && upto > aim);
        if (some) {  // none passes by a rounding, or v is 1 or more: the last
            const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
            at = i + l, before = l ? lane_of(upto, l - 1) : run;
        }
        if (past) break;
        run = lane_of(upto, 63);
    }
    if (at < 0) return -1;
    const int split = at / subs, from = split * a.per + (at - split * subs) * words;
    return pick<MODE>(w, from, min(from + words, min((split + 1) * a.per, a.vocab)), aim - before);
}

// The decision where drafts have no probabilities, and the draw: the part of the words that v falls on by the parts' sums, a thread's words
// in it by a scan over the workgroup, the word by one over a wavefront. One workgroup a sequence: 5 to 9 us up to 262144 words, waits for loads
// that depend on each other; 8 for a row of 2^20 and 70 for one of 2^24, whose parts are 16384 and 262144 words, all gone through by that
// workgroup. (Keeping the parts' sums from step to step saved nothing that could be measured.)
__global__ __launch_bounds__(WG) void verify_next_kernel(VerifyArgs a) {
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    bool greedy;
    const double c = heat_of(a, s, greedy);
    const double v = a.v[s];
    const int len = a.keep ? a.len[s] : 0;
    const VerifyChoice ch = a.q ? a.choice[s] : decide(a, s, c, greedy, a.lse != nullptr);
    int word = -1;
    if (ch.n > 0 && fabsf(ch.top) <= 3.4028235e38f && c == c) {
        if (greedy) word = ch.at;
        else {
            const Weigh w = weigh_of(a, ch, c);
            double part = 0.0;  // of p: what the rows' pass left, on the row's level
            if (lane < a.splits) {
                const int64_t i = (int64_t)ch.t * a.splits + lane;
                part = a.sum[i] * exp2_of(((double)a.top[i] - w.m) * c);
            }
            if (ch.d >= 0 && a.q) {
                const int subs = (a.per + SUB - 1) / SUB;
                const double *rest = a.rest + (int64_t)s * a.splits * subs;
                word = draw<FROM_REST>(a, w, subs, SUB, v, [&](int i) { return rest[i]; });
            } else if (ch.d >= 0) {
                // the draft's part without it: by a difference where that loses a bit at most, else anew
                const int mine = ch.d / a.per;
                const double with = lane_of(part, mine), x = weight<FROM_P>(w, ch.d, w.x[ch.d], 0.0f);
                const double left = x <= 0.5 * with ? with - x : sum_words<WITHOUT_DRAFT>(w, mine * a.per, min(a.vocab, (mine + 1) * a.per));
                word = draw<WITHOUT_DRAFT>(a, w, 1, a.per, v, [&](int) { return lane == mine ? left : part; });
            }
            if (word < 0) word = draw<FROM_P>(a, w, 1, a.per, v, [&](int) { return part; });  // behind the last row, or nothing is left of p
        }
    }
    if (tid == 0) {
        a.n_ok[s] = ch.good;
        a.next[s] = word;
        if (a.keep) a.keep[s] = ch.n > 0 ? max(0, len - (ch.n - 1 - ch.good)) : len;
    }
}

size_t subs_of(const VerifyArgs &a) { return (a.per + SUB - 1) / SUB; }
}  // namespace

// Blocks of 4096 words, smaller while the device would not be filled (64 rows of 32768 words: 4096 5.5 us, 2048 4.8, 1024 7.0); parts of two
// blocks where rows are many, which leaves fewer sums to write and join (189 rows of 128256: 31.1 us with one, 27.8 with two, and the rejected rows'
// sums 17.8 and 16.3; 106 of 50021, below the limit: 11.0 and 9.5, but 13.0 and 15.2 for the choice, which goes through a part word by word); two
// parts a workgroup where those are still many (27.8 and 27.1; with 800 workgroups left: 11.4 and 12.2).
size_t verify_plan(VerifyArgs &a, int num_cu) {
    auto parts = [&](int nv) { return (a.vocab + 1024 * nv - 1) / (1024 * nv); };
    a.nv = 4;
    while (a.nv > 1 && (int64_t)a.n_tok * parts(a.nv) < 4 * num_cu) a.nv /= 2;
    const int blocks = parts(a.nv), two = (int64_t)a.n_tok * blocks >= 8 * num_cu ? 2 : 1;
    a.splits = std::min(MOST_SPLITS, (blocks + two - 1) / two);
    a.per = (blocks + a.splits - 1) / a.splits * 1024 * a.nv;
    a.splits = (a.vocab + a.per - 1) / a.per;
    a.group = (int64_t)a.n_tok * a.splits >= 8 * num_cu ? 2 : 1;
    const size_t n = (size_t)a.n_tok * a.splits;
    return n * 16 + (a.q ? (size_t)a.n_seq * ((size_t)a.splits * subs_of(a) * 8 + sizeof(VerifyChoice)) : 0);
}
void verify_scratch(VerifyArgs &a, void *p) {
    const size_t n = (size_t)a.n_tok * a.splits, m = a.q ? a.n_seq : 0;
    a.sum = (double *)p;
    a.rest = a.sum + n;
    a.choice = (VerifyChoice *)(a.rest + m * a.splits * subs_of(a));
    a.top = (float *)(a.choice + m);
    a.at = (int32_t *)(a.top + n);
}

hipError_t launch_verify(const VerifyArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)((int64_t)a.n_tok * ((a.splits + a.group - 1) / a.group));
    switch (a.nv) {
    case 1: verify_rows_kernel<1><<<grid, 256, 0, s>>>(a); break;
    case 2: verify_rows_kernel<2><<<grid, 256, 0, s>>>(a); break;
    default: verify_rows_kernel<4><<<grid, 256, 0, s>>>(a); break;
    }
    if (a.q) verify_rest_kernel<<<(unsigned)((int64_t)a.n_seq * a.splits), WG, 0, s>>>(a);
    verify_next_kernel<<<(unsigned)a.n_seq, WG, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace fgh
