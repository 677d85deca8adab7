// fgh_verify.hip - drafted tokens against the target's logits, and the token that follows the accepted ones, on gfx950.
//
// Row i of a sequence has p = softmax(logits / T); the draft d behind it stays while u q(d) < p(d). At the first that does not, the
// token is the first one whose running sum of max(p - q, 0) passes v times the whole; behind the last row, of p. The sums
// run over a vocabulary of 10^5 words, and which word v falls on is a matter of their last bits: exponentials, sums and
// comparisons are in 64 bits. A row is read once: each workgroup leaves the largest value of its words, its
// place and the sum of exp((x - largest) / T); whole rows, and the sums that a number has to be compared with, are joined
// from those.
#include "fgh_serve.h"

#include <algorithm>

namespace fgh {

namespace {

// rows are 4-byte aligned: 16 bytes a lane all the same
typedef float vf4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.69314718055994530942;

// 2^t, off by at most 1e-14 of it: t - rint(t) in the exponential's series to the 11th power. -infinity and NaN give 0.
__device__ __forceinline__ double exp2_of(double t) {
    t = fmin(fmax(t, -1100.0), 1100.0);
    const double n = rint(t), f = (t - n) * LN2;
    double r = 1.0 / 39916800;
    r = __builtin_fma(r, f, 1.0 / 3628800);
    r = __builtin_fma(r, f, 1.0 / 362880);
    r = __builtin_fma(r, f, 1.0 / 40320);
    r = __builtin_fma(r, f, 1.0 / 5040);
    r = __builtin_fma(r, f, 1.0 / 720);
    r = __builtin_fma(r, f, 1.0 / 120);
    r = __builtin_fma(r, f, 1.0 / 24);
    r = __builtin_fma(r, f, 1.0 / 6);
    r = __builtin_fma(r, f, 0.5);
    r = __builtin_fma(r, f, 1.0);
    r = __builtin_fma(r, f, 1.0);
    return __builtin_amdgcn_ldexp(r, (int)n);
}

// log2(e) / T of a sequence; T = 0, the largest value, has 1's. A T below 0 or NaN makes NaN.
__device__ __forceinline__ double heat_of(const VerifyArgs &a, int s, bool &greedy) {
    const float t = a.temp ? a.temp[s] : 1.0f;
    greedy = t == 0.0f;
    return greedy ? LOG2E : t > 0.0f ? LOG2E / (double)t : (double)__builtin_nanf("");
}

// a row, or a part of one: its largest value (NaN where it has a NaN), the first place of it, sum of 2^((x - top) c)
struct Part {
    double sum;
    float top;
    int at;
};
// the largest value to take others relative to: 0 where there is none
__device__ __forceinline__ double level(float top) { return fabsf(top) <= 3.4028235e38f ? (double)top : 0.0; }
__device__ __forceinline__ Part join(const Part &x, const Part &y, double c) {  // x's words stand before y's
    Part r;
    const bool nan = x.top != x.top || y.top != y.top, second = y.top > x.top;
    r.top = nan ? __builtin_nanf("") : second ? y.top : x.top;
    r.at = second ? y.at : x.at;
    const double m = level(r.top);
    r.sum = x.sum * exp2_of(((double)x.top - m) * c) + y.sum * exp2_of(((double)y.top - m) * c);  // 0 for a part without words
    return r;
}
__device__ __forceinline__ Part shfl_part(const Part &p, int mask) {
    return Part{__shfl_xor(p.sum, mask, 64), __shfl_xor(p.top, mask, 64), __shfl_xor(p.at, mask, 64)};
}
// over a wavefront's lanes, in the lanes' order; every lane gets it
__device__ __forceinline__ Part join_wave(Part p, double c) {
    const int lane = threadIdx.x & 63;
    for (int o = 1; o < 64; o <<= 1) {
        const Part z = shfl_part(p, o);
        p = lane & o ? join(z, p, c) : join(p, z, c);
    }
    return p;
}

template <int NV>
__global__ __launch_bounds__(256) void verify_rows_kernel(VerifyArgs a) {
    __shared__ Part lds[4];
    const int row = blockIdx.x / a.splits, split = blockIdx.x - row * a.splits, tid = threadIdx.x;
    const int from = split * a.per, to = min(a.vocab, from + a.per);
    const float *x = a.logits + row * a.ld;
    vf4 v[NV];
    auto load = [&](int base) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = base + i * 1024 + 4 * tid;
            if (j + 4 <= to) v[i] = *(const vf4 *)(x + j);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i][e] = j + e < to ? x[j + e] : -__builtin_inff();
        }
    };
    load(from);  // on its way while the row's sequence is found
    const int s = seq_of_row(a.tok, a.n_seq, row);
    if (s < 0) return;
    bool greedy;
    const double c = heat_of(a, s, greedy);
    Part p{0.0, -__builtin_inff(), from};
    for (int base = from; base < to; base += 1024 * NV) {
        if (base != from) load(base);
        Part b{0.0, -__builtin_inff(), base};
        bool nan = false;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = v[i][e];
                nan |= y != y;
                if (y > b.top) b.top = y, b.at = base + i * 1024 + 4 * tid + e;
            }
        const double m = level(b.top);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) b.sum += exp2_of(((double)v[i][e] - m) * c);
        if (nan) b.top = __builtin_nanf("");
        // lanes' words are not in order: the smaller place of two equal ones
        Part r = join(p, b, c);
        p = r;
    }
    // a lane's words lie between other lanes': equal largest values go to the lower place
    for (int o = 1; o < 64; o <<= 1) {
        const Part z = shfl_part(p, o);
        const int at = p.top == z.top ? min(p.at, z.at) : z.top > p.top ? z.at : p.at;
        p = (tid & o) ? join(z, p, c) : join(p, z, c);
        p.at = at;
    }
    if ((tid & 63) == 0) lds[tid >> 6] = p;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 4; ++w) {
            const Part z = lds[w];
            const int at = p.top == z.top ? min(p.at, z.at) : z.top > p.top ? z.at : p.at;
            p = join(p, z, c);
            p.at = at;
        }
        const int64_t i = (int64_t)row * a.splits + split;
        a.sum[i] = p.sum, a.top[i] = p.top, a.at[i] = p.at;
    }
}

// what a sequence's rows come to
struct Choice {
    Part row;       // of the row that the next token is drawn from
    int t, d;       // that row; the draft that it rejects, or -1
    int n, good;    // rows, accepted drafts; n = 0: no token
};
// the sequence's rows, their ends in the buffers: none for what a batch cannot mean
__device__ __forceinline__ int2 rows_of(const VerifyArgs &a, int s) {
    const int b = a.tok[s], e = a.tok[s + 1];
    if (b < 0 || e > a.n_tok || e <= b || e - b > a.max_tok) return int2{0, 0};
    return int2{b, e - b};
}
__device__ __forceinline__ Part row_part(const VerifyArgs &a, int t, double c) {
    const int lane = threadIdx.x & 63;
    Part p{0.0, -__builtin_inff(), 0};
    if (lane < a.splits) {
        const int64_t i = (int64_t)t * a.splits + lane;
        p = Part{a.sum[i], a.top[i], a.at[i]};
    }
    return join_wave(p, c);
}
// the draft's probability under q; NaN, which passes no test, where q has one
__device__ __forceinline__ double q_at(const VerifyArgs &a, int t, int d, double c) {
    const double x = (double)a.q[t * a.ldq + d] * c - (double)a.q_lse[t] * LOG2E;
    return x == x ? exp2_of(x) : x;
}
// by a workgroup of 256, a wavefront to a row, four rows at a time until one is rejected (all of them where `lse` is written)
__device__ Choice decide(const VerifyArgs &a, int s, double c, bool greedy, bool lse) {
    __shared__ Part rows[4];
    __shared__ int ok[4];
    const int wave = threadIdx.x >> 6;
    const int2 r = rows_of(a, s);
    Choice ch;
    ch.n = r.y, ch.good = 0, ch.t = -1, ch.d = -1, ch.row = Part{0.0, 0.0f, 0};
    bool open = true;
    for (int i0 = 0; i0 < r.y && (open || lse); i0 += 4) {
        const int i = i0 + wave, t = r.x + i;
        if (i < r.y) {
            const Part p = row_part(a, t, c);
            bool good = false;
            if (i < r.y - 1) {
                const int d = a.tokens[t + 1];
                if ((uint32_t)d < (uint32_t)a.vocab && fabsf(p.top) <= 3.4028235e38f) {
                    if (greedy) good = d == p.at;
                    else {
                        const double w = exp2_of(((double)a.logits[t * a.ld + d] - p.top) * c) / p.sum;
                        good = (double)a.u[t] * (a.q ? q_at(a, t, d, c) : 1.0) < w && c == c;
                    }
                }
            }
            if ((threadIdx.x & 63) == 0) {
                rows[wave] = p, ok[wave] = good;
                if (lse) a.lse[t] = p.top != p.top || c != c ? __builtin_nanf("") : fabsf(p.top) <= 3.4028235e38f ? (float)(level(p.top) * c * LN2 + log(p.sum)) : p.top;
            }
        }
        __syncthreads();
        for (int w = 0; w < 4 && open && i0 + w < r.y; ++w) {
            ch.row = rows[w], ch.t = r.x + i0 + w;
            if (i0 + w == r.y - 1 || !ok[w]) {
                open = false;
                ch.d = i0 + w == r.y - 1 ? -1 : a.tokens[ch.t + 1];
                if ((uint32_t)ch.d >= (uint32_t)a.vocab) ch.d = -1;  // no word: the token is drawn from p
            } else ++ch.good;
        }
        __syncthreads();
    }
    return ch;
}

// a word's weight in the choice of the next token
enum { FROM_P, WITHOUT_DRAFT, FROM_REST };
struct Weigh {
    const float *x, *q;
    double m, c, z, lse;  // the row's largest, log2(e) / T, 1 / the sum, the draft row's lse in powers of two
    int d;
};
template <int MODE>
__device__ __forceinline__ double weight(const Weigh &w, int j) {
    if (MODE == WITHOUT_DRAFT && j == w.d) return 0.0;
    const double p = exp2_of(((double)w.x[j] - w.m) * w.c);
    if (MODE != FROM_REST) return p;
    const double q = exp2_of((double)w.q[j] * w.c - w.lse);
    return fmax(p * w.z - q, 0.0);
}
__device__ __forceinline__ Weigh weigh_of(const VerifyArgs &a, const Choice &ch, double c) {
    Weigh w;
    w.x = a.logits + ch.t * a.ld, w.q = a.q ? a.q + ch.t * a.ldq : nullptr;
    w.m = level(ch.row.top), w.c = c, w.z = 1.0 / ch.row.sum, w.lse = a.q ? (double)a.q_lse[ch.t] * LOG2E : 0.0, w.d = ch.d;
    return w;
}
__device__ __forceinline__ double sum_block(double v) {
    __shared__ double lds[4];
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}
template <int MODE>
__device__ __forceinline__ double sum_words(const Weigh &w, int from, int to) {
    double v = 0.0;
    for (int j = from + threadIdx.x; j < to; j += 256) v += weight<MODE>(w, j);
    return sum_block(v);
}

// sums of max(p - q, 0) of a rejected row, by parts
__global__ __launch_bounds__(256) void verify_rest_kernel(VerifyArgs a) {
    const int s = blockIdx.x / a.splits, split = blockIdx.x - s * a.splits;
    bool greedy;
    const double c = heat_of(a, s, greedy);
    if (greedy || !(c == c)) return;
    const Choice ch = decide(a, s, c, greedy, false);
    if (ch.d < 0) return;
    const double v = sum_words<FROM_REST>(weigh_of(a, ch, c), split * a.per, min(a.vocab, (split + 1) * a.per));
    if (threadIdx.x == 0) a.rest[(int64_t)s * a.splits + split] = v;
}

// the first of words from .. to - 1 whose running sum passes `aim`, or the last of any weight (-1: none has)
template <int MODE>
__device__ int pick(const Weigh &w, int from, int to, double aim) {
    __shared__ double sums[4];
    __shared__ int word, last;
    const int per = (to - from + 255) / 256, b = min(to, from + (int)threadIdx.x * per), e = min(to, b + per), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double own = 0.0;
    for (int j = b; j < e; ++j) own += weight<MODE>(w, j);
    double upto = own;
    for (int o = 1; o < 64; o <<= 1) {
        const double z = __shfl_up(upto, o, 64);
        if (lane >= o) upto += z;
    }
    if (lane == 63) sums[wave] = upto;
    if (threadIdx.x == 0) word = to, last = -1;
    __syncthreads();
    for (int i = 0; i < wave; ++i) upto += sums[i];
    double run = upto - own;
    if (own > 0.0) {
        int at = to, end = -1;
        for (int j = b; j < e; ++j) {
            const double x = weight<MODE>(w, j);
            run += x;
            if (x > 0.0) {
                end = j;
                if (run > aim && at == to) at = j;
            }
        }
        if (at < to) atomicMin(&word, at);
        if (end >= 0) atomicMax(&last, end);
    }
    __syncthreads();
    return word < to ? word : last;
}

// chooses the part, then the word; sums[] holds the parts' sums
template <int MODE>
__device__ int draw(const VerifyArgs &a, const Weigh &w, const double *sums, double aim) {
    double run = 0.0;
    int part = -1;
    double before = 0.0;
    for (int i = 0; i < a.splits; ++i) {  // the first part that passes the aim, or the last of any weight
        const double x = sums[i];
        if (x > 0.0) {
            part = i, before = run;
            run += x;
            if (run > aim) break;
        }
    }
    if (part < 0) return -1;
    return pick<MODE>(w, part * a.per, min(a.vocab, (part + 1) * a.per), aim - before);
}

__global__ __launch_bounds__(256) void verify_next_kernel(VerifyArgs a) {
    __shared__ double sums[64];
    const int s = blockIdx.x, tid = threadIdx.x;
    bool greedy;
    const double c = heat_of(a, s, greedy);
    const Choice ch = decide(a, s, c, greedy, a.lse != nullptr);
    int word = -1;
    if (ch.n > 0 && fabsf(ch.row.top) <= 3.4028235e38f && c == c) {
        if (greedy) word = ch.row.at;
        else {
            const Weigh w = weigh_of(a, ch, c);
            const double v = a.v[s];
            auto parts = [&] {  // of p: what the rows' pass left, on the row's level
                if (tid < a.splits) {
                    const int64_t i = (int64_t)ch.t * a.splits + tid;
                    sums[tid] = a.sum[i] * exp2_of(((double)a.top[i] - w.m) * c);
                }
                __syncthreads();
            };
            auto whole = [&] {
                double r = 0.0;
                for (int i = 0; i < a.splits; ++i) r += sums[i];
                return r;
            };
            if (ch.d >= 0 && a.q) {
                if (tid < a.splits) sums[tid] = a.rest[(int64_t)s * a.splits + tid];
                __syncthreads();
                word = draw<FROM_REST>(a, w, sums, v * whole());
            } else if (ch.d >= 0) {
                parts();
                const int mine = ch.d / a.per;  // the draft's part without it
                const double left = sum_words<WITHOUT_DRAFT>(w, mine * a.per, min(a.vocab, (mine + 1) * a.per));
                if (tid == 0) sums[mine] = left;
                __syncthreads();
                word = draw<WITHOUT_DRAFT>(a, w, sums, v * whole());
            }
            if (word < 0) {  // behind the last row, or nothing is left of p
                __syncthreads();
                parts();
                word = draw<FROM_P>(a, w, sums, v * whole());
            }
        }
    }
    if (tid == 0) {
        a.n_ok[s] = ch.good;
        a.next[s] = word;
        if (a.keep) a.keep[s] = ch.n > 0 ? max(0, a.len[s] - (ch.n - 1 - ch.good)) : a.len[s];
    }
}

}  // namespace

size_t verify_plan(VerifyArgs &a, int num_cu) {
    auto parts = [&](int nv) { return (a.vocab + 1024 * nv - 1) / (1024 * nv); };
    a.nv = 8;
    while (a.nv > 1 && (int64_t)a.n_tok * parts(a.nv) < 2 * num_cu) a.nv /= 2;
    const int blocks = parts(a.nv);
    a.splits = std::min(64, blocks);  // a wavefront joins them
    a.per = (blocks + a.splits - 1) / a.splits * 1024 * a.nv;
    a.splits = (a.vocab + a.per - 1) / a.per;
    const size_t n = (size_t)a.n_tok * a.splits;
    return n * 16 + (a.q ? (size_t)a.n_seq * a.splits * 8 : 0);
}
void verify_scratch(VerifyArgs &a, void *p) {
    const size_t n = (size_t)a.n_tok * a.splits;
    a.sum = (double *)p;
    a.rest = a.sum + n;
    a.top = (float *)(a.rest + (a.q ? (size_t)a.n_seq * a.splits : 0));
    a.at = (int32_t *)(a.top + n);
}

hipError_t launch_verify(const VerifyArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)((int64_t)a.n_tok * a.splits);
    switch (a.nv) {
    case 1: verify_rows_kernel<1><<<grid, 256, 0, s>>>(a); break;
    case 2: verify_rows_kernel<2><<<grid, 256, 0, s>>>(a); break;
    case 4: verify_rows_kernel<4><<<grid, 256, 0, s>>>(a); break;
    default: verify_rows_kernel<8><<<grid, 256, 0, s>>>(a); break;
    }
    if (a.q) verify_rest_kernel<<<(unsigned)((int64_t)a.n_seq * a.splits), 256, 0, s>>>(a);
    verify_next_kernel<<<(unsigned)a.n_seq, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace fgh
