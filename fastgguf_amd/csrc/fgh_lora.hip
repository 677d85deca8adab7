// fgh_lora.hip - low-rank adapters of many requests beside a shared projection on gfx950: y = y_in + scale B (A x), each row with
// its sequence's adapter.
//
// Two launches: h = A x, split over columns where rows are few, then y from the sums of h. A workgroup has the rows of one adapter
// that stand together in a tile of the batch. Both products run on 16 x 16 x 32 bf16 matrix instructions whose fp32 operands are
// taken apart into bf16 parts that hold all their bits (x and h: 3; adapters F32 3, F16 2, BF16 1), so that results are
// those of fp32 products and sums; F32 adapters leave 3 of 9 products out, up to 2^-21 of one, 2^-24 of the whole on average.
// A part below 2^-126 is a bf16 subnormal: its bits end at 2^-133.
//
// Bound by memory where rows are many: 8192 tokens, 4096 -> 14336, rank 64, F16: 238 us for 1.08 GB, 4.5 TB/s; y alone at 5.0. By loads that wait for
// each other where they are few: 64 tokens with 24 adapters 21 us (38 MB), one token 9.
#include <algorithm>
#include <type_traits>

#include "fgh_pattn.h"
#include "fgh_serve.h"

namespace fgh {

namespace {

typedef float lf4 __attribute__((ext_vector_type(4), aligned(4)));  // x and y: rows of any stride

constexpr int NONE = 1, BAD = 2, FIRST = 3;  // an adapter as a mark that is not 0
// The adapters of the rows base .. base + tile - 1, tile <= 64, a lane each: as marks, 0 for a row of no sequence. Every wavefront finds them
// for itself: mark[64] is its own LDS.
__device__ __forceinline__ int adapters_of(const LoraArgs &a, int base, int *mark) {
    const int lane = threadIdx.x & 63, top = min(base + a.tile, a.n_tok), end = min(a.tok[a.n_seq], top);
    mark[lane] = 0;
    __builtin_amdgcn_wave_barrier();  // LDS serves a wavefront in order: only the compiler must keep it
    // few sequences are looked through from the first one: a load less that others wait for
    for (int b = a.n_seq > 256 ? max(seq_of_row(a.tok, a.n_seq, base), 0) : 0; b < a.n_seq; b += 64) {
        const int s = min(b + lane, a.n_seq - 1), id = a.id[s];
        const int from = max(a.tok[s], base), to = min(a.tok[s + 1], top);
        if (b + lane < a.n_seq && from < to) mark[from - base] = id == -1 ? NONE : (uint32_t)id < (uint32_t)a.n_adapter ? FIRST + id : BAD;
        if (__builtin_amdgcn_ballot_w64(b + lane >= a.n_seq || to >= end || base >= end)) break;
    }
    __builtin_amdgcn_wave_barrier();
    const int m = mark[lane];
    const uint64_t starts = __builtin_amdgcn_ballot_w64(m != 0), mine = starts & (~0ull >> (63 - lane));
    const int first = __shfl(m, 63 - __builtin_clzll(mine | 1), 64);
    return mine && base + lane < end ? first : 0;
}
// what the rows `rows` of a tile, whose mark is `m`, have in common
__device__ __forceinline__ LoraRun run_of(const LoraArgs &a, uint64_t rows, int m) {
    if (m == NONE) return LoraRun{rows, -1, 0, 0.0f};
    LoraRun r{rows, -2, 0, __builtin_nanf("")};
    if (m == BAD) return r;
    const int rank = __builtin_amdgcn_readfirstlane(a.rank ? a.rank[m - FIRST] : a.max_rank);
    if ((uint32_t)rank > (uint32_t)a.max_rank) return r;
    return LoraRun{rows, m - FIRST, rank, a.scale ? a.scale[m - FIRST] : 1.0f};
}
// the rows of a tile that a run has, in order, into a wavefront's own LDS; how many
__device__ __forceinline__ int list_rows(uint64_t rows, int *list) {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_wave_barrier();
    if (rows >> lane & 1) list[__builtin_popcountll(rows & ((1ull << lane) - 1))] = lane;
    __builtin_amdgcn_wave_barrier();
    return __builtin_popcountll(rows);
}

template <int TYPE>
struct Weights {
    static constexpr int NW = TYPE == T_F32 ? 3 : TYPE == T_F16 ? 2 : 1, ES = TYPE == T_F32 ? 4 : 2;
};
// 8 values of an adapter as they are in memory, and as bf16 parts
template <int TYPE>
struct Raw {
    pu4 v[TYPE == T_F32 ? 2 : 1];
};
template <int TYPE>
__device__ __forceinline__ Raw<TYPE> raw8(const uint8_t *p) {
    Raw<TYPE> r;
    r.v[0] = *(const pu4 *)p;
    if constexpr (TYPE == T_F32) r.v[1] = *(const pu4 *)(p + 16);
    return r;
}
// the first n of them, then 0: masks, and what they leave
template <int TYPE>
__device__ __forceinline__ Raw<TYPE> first8(int n) {
    Raw<TYPE> m;
    if constexpr (TYPE == T_F32)
#pragma unroll
        for (int e = 0; e < 8; ++e) m.v[e / 4][e % 4] = e < n ? ~0u : 0u;
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) m.v[0][e] = n >= 2 * e + 2 ? ~0u : n > 2 * e ? 0xffffu : 0u;
    return m;
}
template <int TYPE>
__device__ __forceinline__ void mask8(Raw<TYPE> &raw, const Raw<TYPE> &m) {
    raw.v[0] &= m.v[0];
    if constexpr (TYPE == T_F32) raw.v[1] &= m.v[1];
}
template <int TYPE>
__device__ __forceinline__ void weights8(const Raw<TYPE> &raw, pu4 (&w)[Weights<TYPE>::NW]) {
    if constexpr (TYPE == T_F32) {
        const float x[8] = {__uint_as_float(raw.v[0].x), __uint_as_float(raw.v[0].y), __uint_as_float(raw.v[0].z), __uint_as_float(raw.v[0].w),
                            __uint_as_float(raw.v[1].x), __uint_as_float(raw.v[1].y), __uint_as_float(raw.v[1].z), __uint_as_float(raw.v[1].w)};
        parts8<T_BF16, 3>(x, w);
    } else if constexpr (TYPE == T_BF16) w[0] = raw.v[0];
    else {
        const ph8 h = __builtin_bit_cast(ph8, raw.v[0]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
        parts8<T_BF16, 2>(x, w);  // 11 bits: nothing is left
    }
}
// D_j += W_j X, the smallest products first; those of different j between two of one
template <int TYPE, int J>
__device__ __forceinline__ void multiply(pf4 *d, const pu4 (&w)[J][Weights<TYPE>::NW], const pu4 (&x)[3]) {
    constexpr int NW = Weights<TYPE>::NW;
#pragma unroll
    for (int sum = NW == 3 ? 2 : NW + 1; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i < NW; ++i)
            if (sum - i >= 0 && sum - i < 3)
#pragma unroll
                for (int j = 0; j < J; ++j) mma16<T_BF16>(d[j], w[j][i], x[sum - i]);
}

// Adapter values of 64 rows (of A: ranks, of B: outputs) and 32 or 64 (SB 1, 2) values along them, shared by a workgroup: a thread takes 8 values of a
// row, its neighbours the row's next ones, so that an access finds whole lines, and leaves their parts in LDS as the products take them:
// [4 tiles][SB steps][parts][64 lanes]. (Loaded as the products take them, neighbouring lanes in 16 different rows, every lane was an access of its own to
// the first cache: 1.0 a cycle, the bound of such a kernel.) Lanes are exchanged so that neighbours write to different banks.
template <int TYPE, int SB>
struct Stage {
    static constexpr int NW = Weights<TYPE>::NW, ES = Weights<TYPE>::ES, VALUES = 4 * SB * NW * 64;  // 16-byte values in LDS
    static __device__ __forceinline__ int slot(int c, int g, int k) { return 16 * g + (c ^ (4 * g + k)); }
    static __device__ __forceinline__ void put(pu4 *lds, int row, int chunk, const Raw<TYPE> &raw) {
        const int j = row >> 4, k = chunk >> 2;
        pu4 w[NW];
        weights8<TYPE>(raw, w);
#pragma unroll
        for (int e = 0; e < NW; ++e) lds[((SB * j + k) * NW + e) * 64 + slot(row & 15, chunk & 3, k)] = w[e];
    }
    static __device__ __forceinline__ void get(const pu4 *lds, int j, int k, int lane, pu4 (&w)[NW]) {
#pragma unroll
        for (int e = 0; e < NW; ++e) w[e] = lds[((SB * j + k) * NW + e) * 64 + slot(lane & 15, lane >> 4, k)];
    }
};
constexpr int MOST_PARTS = 8;  // of h
constexpr int LD = 68;  // floats between rows of 64 in LDS: 16 rows start in 16 different groups of banks

// h of few rows that have an adapter in common (64 tokens of 24 adapters, BF16, rank 64: 8.7 us, of which 5 are the way to the first load; one token:
// 5.0), 16 NR ranks, over a part of the columns: the wavefronts take steps of 64 columns in turn, the next one's values on their way during the
// products of one. A's values and x's go through a wavefront's own LDS, so that neighbouring lanes read neighbouring values: as the products take
// them, 16 rows an access, the first cache gave one lane a cycle.
template <int TYPE, int NR>
__global__ __launch_bounds__(256) void lora_down_split_kernel(LoraArgs a) {
    constexpr int ES = Weights<TYPE>::ES, NW = Weights<TYPE>::NW;
    constexpr int CH = 4 * ES, PER = 64 / CH, LOADS = 16 * NR / PER, ROW = 64 * ES + 16;  // 16-byte values of a row, rows of an access; bytes of a row in LDS
    __shared__ __attribute__((aligned(16))) uint8_t wl[4][16 * NR * ROW];
    __shared__ __attribute__((aligned(16))) float xl[4][16 * LD];
    __shared__ int marks[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int blocks = (a.max_rank + 16 * NR - 1) / (16 * NR);
    int b = blockIdx.x;
    const int part = b % a.ks;
    b /= a.ks;
    const int block = b % blocks;
    b /= blocks;
    const int all = (a.n_tok + a.tile - 1) / a.tile, tile = b % all, slot = b / all, base = tile * a.tile;  // first the first runs, which every tile has
    const int from = part * a.kper, to = min(a.cols, from + a.kper), r0 = block * 16 * NR;
    const int padded = (a.max_rank + 15) & ~15;
    int *list = marks + 64 * wave;
    uint8_t *wo = wl[wave];
    float *xo = xl[wave];
    const int mark = adapters_of(a, base, list);
    uint64_t left = __builtin_amdgcn_ballot_w64(mark != 0);
    for (int which = 0, mine = slot;; ++which) {  // the tile's runs; every `slots`-th one is this workgroup's
        const int m = left ? __builtin_amdgcn_readlane(mark, __builtin_ctzll(left)) : 0;
        const uint64_t rows_of = __builtin_amdgcn_ballot_w64(mark == m) & left;
        left &= ~rows_of;
        if (m && which != mine) continue;
        const LoraRun run = m ? run_of(a, rows_of, m) : LoraRun{};
        if (part == 0 && block == 0 && tid == 0 && mine < a.most) a.runs[(int64_t)tile * a.most + mine] = run;  // behind the last: no rows
        if (!m) break;
        mine += a.slots;
        if (run.adapter < 0 || r0 >= run.rank) continue;
        const int n = list_rows(rows_of, list), tiles = min(NR, (run.rank - r0 + 15) / 16);
        const uint8_t *A = a.a + ((int64_t)run.adapter * a.max_rank + r0) * a.cols * ES;
        const uint8_t *X = (const uint8_t *)(a.x + base * a.ldx);
        for (int t0 = 0; t0 < n; t0 += 16) {
            pf4 acc[NR];
#pragma unroll
            for (int j = 0; j < NR; ++j) acc[j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
            uint32_t xr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) xr[i] = 4 * ((uint32_t)list[min(t0 + 4 * i + g, n - 1)] * (uint32_t)a.ldx);
            pu4 wn[LOADS];
            lf4 xn[4];
            auto load = [&](int k0) {  // behind the last column and the last rank those again
                const uint32_t k = ES * (uint32_t)min(k0 + 16 / ES * (lane % CH), a.cols - 16 / ES), kx = 4 * (uint32_t)min(k0 + 4 * c, a.cols - 4);
#pragma unroll
                for (int i = 0; i < LOADS; ++i)
                    if (i * PER < 16 * tiles) wn[i] = *(const pu4 *)(A + (uint32_t)(ES * ((uint32_t)min(i * PER + lane / CH, run.rank - r0 - 1) * (uint32_t)a.cols) + k));
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t0 + 4 * i < n) xn[i] = *(const lf4 *)(X + (uint32_t)(xr[i] + kx));
            };
            int k0 = from + 64 * wave;
            if (k0 < to) load(k0);
            for (; k0 < to; k0 += 256) {
                // LDS serves a wavefront in order: only the compiler must keep it
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < LOADS; ++i) *(pu4 *)(wo + (i * PER + lane / CH) * ROW + 16 * (lane % CH)) = wn[i];
#pragma unroll
                for (int i = 0; i < 4; ++i) *(pf4 *)(xo + (4 * i + g) * LD + 4 * c) = xn[i];
                __builtin_amdgcn_wave_barrier();
                if (k0 + 256 < to) load(k0 + 256);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float v[8];
                    *(pf4 *)v = *(const pf4 *)(xo + c * LD + 32 * k + 8 * g), *(pf4 *)(v + 4) = *(const pf4 *)(xo + c * LD + 32 * k + 8 * g + 4);
                    pu4 p[3];
                    parts8<T_BF16, 3>(v, p);
#pragma unroll
                    for (int j = 0; j < NR; ++j) {
                        if (j >= tiles) break;
                        Raw<TYPE> raw = raw8<TYPE>(wo + (16 * j + c) * ROW + ES * (32 * k + 8 * g));
                        if (k0 + 32 * k + 8 * g >= to) raw = Raw<TYPE>{};  // times 0 behind the last column
                        pu4 w[1][NW];
                        weights8<TYPE>(raw, w[0]);
                        multiply<TYPE, 1>(acc + j, w, p);
                    }
                }
            }
            // the wavefronts' sums, in the order of the wavefronts
            __syncthreads();
            pf4 *sums = (pf4 *)wl;  // [4][NR][64]
#pragma unroll
            for (int j = 0; j < NR; ++j) sums[(wave * NR + j) * 64 + lane] = acc[j];
            __syncthreads();
            for (int j = wave; j < NR; j += 4) {
                const int row = t0 + c, r = r0 + 16 * j + 4 * g;
                const pf4 v = (sums[j * 64 + lane] + sums[(NR + j) * 64 + lane]) + (sums[(2 * NR + j) * 64 + lane] + sums[(3 * NR + j) * 64 + lane]);
                if (row < n && r < padded) *(pf4 *)(a.part + ((int64_t)part * a.n_tok + base + list[row]) * padded + r) = v;
            }
            __syncthreads();
        }
    }
}

// h of a prompt's rows (8192 tokens of 4096 columns, F16, rank 64: 52 us, 2.6 TB/s of x), 16 NR ranks, over a part of the columns: 64 rows to a
// workgroup, 16 to a wavefront, 64 columns at a time, the next ones' values on their way during the products of some. x too goes through LDS, each
// wavefront's by itself: 16 lanes read 256 bytes of a row.
template <int TYPE, int NR>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    using S = Stage<TYPE, 2>;
    constexpr int ES = S::ES, UNITS = (128 * NR + 255) / 256;
    __shared__ __attribute__((aligned(16))) pu4 wl[2][S::VALUES * NR / 4];
    __shared__ __attribute__((aligned(16))) float xl[4][16 * LD];
    __shared__ int lists[4 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int blocks = (a.max_rank + 16 * NR - 1) / (16 * NR);
    int b = blockIdx.x;
    const int part = b % a.ks;
    b /= a.ks;
    const int block = b % blocks;
    b /= blocks;
    const int all = (a.n_tok + a.tile - 1) / a.tile, tile = b % all, slot = b / all, base = tile * a.tile;  // first the first runs, which every tile has
    const int from = part * a.kper, to = min(a.cols, from + a.kper), r0 = block * 16 * NR;
    const int padded = (a.max_rank + 15) & ~15;
    int *list = lists + 64 * wave;
    const int mark = adapters_of(a, base, list);
    uint64_t left = __builtin_amdgcn_ballot_w64(mark != 0);
    for (int which = 0, mine = slot;; ++which) {  // the tile's runs; every `slots`-th one is this workgroup's
        const int m = left ? __builtin_amdgcn_readlane(mark, __builtin_ctzll(left)) : 0;
        const uint64_t rows_of = __builtin_amdgcn_ballot_w64(mark == m) & left;
        left &= ~rows_of;
        if (m && which != mine) continue;
        const LoraRun run = m ? run_of(a, rows_of, m) : LoraRun{};
        if (part == 0 && block == 0 && tid == 0 && mine < a.most) a.runs[(int64_t)tile * a.most + mine] = run;  // behind the last: no rows
        if (!m) break;
        mine += a.slots;
        if (run.adapter < 0 || r0 >= run.rank) continue;
        const int n = list_rows(rows_of, list);
        const uint8_t *A = a.a + (int64_t)run.adapter * a.max_rank * a.cols * ES;
        const uint8_t *X = (const uint8_t *)(a.x + base * a.ldx);
        // what a thread loads: rows 4 i + g of its wavefront's, columns 4 c .. + 3; ranks tid / 8 (+ 32), columns 8 (tid % 8) .. + 7
        uint32_t xo[4], wo[UNITS];
#pragma unroll
        for (int i = 0; i < 4; ++i) xo[i] = 4 * ((uint32_t)list[min(16 * wave + 4 * i + g, n - 1)] * (uint32_t)a.ldx);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) wo[u] = ES * ((uint32_t)min(r0 + (tid >> 3) + 32 * u, run.rank - 1) * (uint32_t)a.cols);
        lf4 xn[2][4];  // of the next two steps
        Raw<TYPE> wn[2][UNITS];
        // behind the last column the last ones again
        auto load_w = [&](Raw<TYPE> (&v)[UNITS], int k0) {
            const uint32_t k = min(k0 + 8 * (tid & 7), a.cols - 8);
#pragma unroll
            for (int u = 0; u < UNITS; ++u) v[u] = raw8<TYPE>(A + (uint32_t)(wo[u] + ES * k));
        };
        auto load_x = [&](lf4 (&v)[4], int k0) {
            const uint32_t k = min(k0 + 4 * c, a.cols - 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *(const lf4 *)(X + (uint32_t)(xo[i] + 4 * k));
        };
        auto put_w = [&](pu4 *lds, Raw<TYPE> (&v)[UNITS], int k0) {  // times 0 behind the last column
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                if (k0 + 8 * (tid & 7) >= to) v[u] = Raw<TYPE>{};
                if (NR > 1 || tid < 128) S::put(lds, (tid >> 3) + 32 * u, tid & 7, v[u]);
            }
        };
        pf4 acc[NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) acc[j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
        float *own = xl[wave];
        // The steps start at another column in each tile and go round: rows lie a power of two apart, and workgroups that read the same columns
        // of their rows at a time would ask few of the memory's channels.
        const int steps = (to - from + 63) / 64, turn = (int)((unsigned)(tile * 5) % (unsigned)steps);
        // Every step asks for the next ones' values, the last two for the last ones' again: loads in branches would be waited for at once.
        auto column = [&](int i) {
            const int j = min(i, steps - 1) + turn;
            return from + 64 * (j < steps ? j : j - steps);
        };
        load_w(wn[0], column(0));
        load_x(xn[0], column(0));
        load_w(wn[1], column(1));
        load_x(xn[1], column(1));
        put_w(wl[0], wn[0], column(0));
        auto step = [&](int i, int at) {
            // LDS serves a wavefront in order: only the compiler must keep it
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < 4; ++j) *(pf4 *)(own + (4 * j + g) * LD + 4 * c) = xn[at][j];
            __builtin_amdgcn_wave_barrier();
            load_w(wn[at], column(i + 2));
            load_x(xn[at], column(i + 2));
            lds_barrier();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                pu4 p[3];
                float v[8];
                *(pf4 *)v = *(const pf4 *)(own + c * LD + 32 * k + 8 * g), *(pf4 *)(v + 4) = *(const pf4 *)(own + c * LD + 32 * k + 8 * g + 4);
                parts8<T_BF16, 3>(v, p);
                constexpr int J = NR > 1 ? 2 : 1;
#pragma unroll
                for (int j0 = 0; j0 < NR; j0 += J) {
                    pu4 w[J][S::NW];
#pragma unroll
                    for (int j = 0; j < J; ++j) S::get(wl[at], j0 + j, k, lane, w[j]);
                    multiply<TYPE, J>(acc + j0, w, p);
                }
            }
            put_w(wl[at ^ 1], wn[at ^ 1], column(i + 1));
        };
#pragma clang loop unroll(disable)
        for (int i = 0; i + 1 < steps; i += 2) {
            step(i, 0);
            step(i + 1, 1);
        }
        if (steps & 1) step(steps - 1, 0);
        lds_barrier();
        const int row = 16 * wave + c;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const int r = r0 + 16 * j + 4 * g;
            if (row < n && r < padded) *(pf4 *)(a.part + ((int64_t)part * a.n_tok + base + list[row]) * padded + r) = acc[j];
        }
    }
}

// y of rows that have an adapter in common (8192 tokens of 14336 outputs: 187 us, 5.0 TB/s; 64 tokens of 24 adapters: 12.5), ucols of the outputs, 64
// at a time and 32 SB ranks of them, the next ones' values on their way during the products of some. ROWS (prompts): each wavefront has 16 rows and
// all 64 outputs; else (few rows) 16 of the outputs and the same rows. Products: lane l has output l % 16 of a tile and row l % 16, ranks 8 (l / 16)
// .. + 7, and gets outputs 4 (l / 16) .. + 3 of its row; through LDS they come to lie as y does, 16 lanes with 256 bytes of a row. KB: such blocks of
// ranks, whose h stays in registers; 0: any number (max_rank above 128), whose h is summed and taken apart for every turn (64 tokens, 24
// adapters, BF16: rank 128 40 us, 136 87, 512 158; 8192 tokens, F16: 307, 513, 1309). ROWS: three workgroups a compute unit, since at
// four registers spill (2500 tokens, F32: 46.8 us, without 35.7).
template <int TYPE, int SB, int KB, bool ROWS>
__global__ __launch_bounds__(256, KB != 1 ? 2 : ROWS ? 3 : 4) void lora_up_kernel(LoraArgs a) {
    using S = Stage<TYPE, SB>;
    constexpr int ES = S::ES, NW = S::NW, J = ROWS ? 4 : 1, P = ROWS ? 2 : 1, KH = KB ? SB * KB : 1, CH = 4 * SB;  // CH: threads to a row's values
    __shared__ __attribute__((aligned(16))) pu4 wl[S::VALUES];
    __shared__ __attribute__((aligned(16))) float tiles[ROWS ? 4 : 1][16 * LD];
    __shared__ int lists[4 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int blocks = (a.rows + a.ucols - 1) / a.ucols;
    int b = blockIdx.x;
    const int b_chunk = b % blocks, first = b_chunk * a.ucols, end = min(a.rows, first + a.ucols);
    b /= blocks;
    const int all = (a.n_tok + a.tile - 1) / a.tile, tile = b % all, slot = b / all, base = tile * a.tile;  // first the first runs, which every tile has
    const int padded = (a.max_rank + 15) & ~15;
    float *out = tiles[ROWS ? wave : 0], *y = a.y + base * a.ldy;
    const float *yin = a.yin + base * a.ldyi;
    int *list = lists + 64 * wave;
    // The turns start at another one in each tile and go round: rows lie a power of two or a few apart, and workgroups that read and write the same
    // columns of their rows at a time would ask few of the memory's channels.
    const int turns = (end - first + 63) / 64, rot = (int)((unsigned)(tile + b_chunk) % (unsigned)turns);
    auto column = [&](int i) {  // behind the last turn the last one again
        const int j = min(i, turns - 1) + rot;
        return first + 64 * (j < turns ? j : j - turns);
    };
    for (int which = slot; which < a.most; which += a.slots) {
        const LoraRun run = a.runs[(int64_t)tile * a.most + which];
        if (run.rows == 0) break;
        if (run.adapter == -1 && a.y == a.yin) continue;
        const int n = list_rows(run.rows, list), steps = (run.rank + 31) / 32, kbs = max(1, (run.rank + 32 * SB - 1) / (32 * SB));
        const uint8_t *B = a.b + (int64_t)max(run.adapter, 0) * a.rows * a.max_rank * ES;
        for (int t0 = 0; t0 < n; t0 += ROWS ? 64 : 16) {
            const int mine = t0 + (ROWS ? 16 * wave : 0);  // the wavefront's first row
            // what a thread reads and writes of y: row 4 i + g of the wavefront's, or row tid / 16 of all, values 4 c .. + 3
            constexpr int I = ROWS ? 4 : 1;
            uint32_t yo[I], yio[I];
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const uint32_t row = list[min(ROWS ? mine + 4 * i + g : t0 + (tid >> 4), n - 1)];
                yo[i] = 4 * (row * (uint32_t)a.ldy), yio[i] = 4 * (row * (uint32_t)a.ldyi);
            }
            lf4 yn[2][I] = {};  // of the next two turns
            Raw<TYPE> wn[SB];
            auto load_w = [&](int n0, int kb) {  // outputs and ranks behind the last: others, which are not used, or cut
                const int r = min(32 * SB * kb + 8 * (tid % CH), max(run.rank - 1, 0) & ~7);
#pragma unroll
                for (int u = 0; u < SB; ++u) wn[u] = raw8<TYPE>(B + ES * ((int64_t)min(n0 + tid / CH + 256 / CH * u, a.rows - 1) * a.max_rank + r));
            };
            auto put_w = [&](int kb) {
                const int have = run.rank - 32 * SB * kb - 8 * (tid % CH);
#pragma unroll
                for (int u = 0; u < SB; ++u) {
                    if (have < 8) mask8<TYPE>(wn[u], first8<TYPE>(have));
                    S::put(wl, tid / CH + 256 / CH * u, tid % CH, wn[u]);
                }
            };
            // a row's last 4 values for lanes behind them: what is not four whole values is read again where it is written
            const bool ahead = a.yin && a.rows >= 4;
            auto load_y = [&](lf4 (&v)[I], int n0) {
                const uint32_t o = 4 * (uint32_t)min(n0 + 4 * c, a.rows - 4);
#pragma unroll
                for (int i = 0; i < I; ++i) v[i] = *(const lf4 *)((const uint8_t *)yin + (uint32_t)(yio[i] + o));
            };
            const float *part = a.part + (int64_t)(base + list[min(mine + c, n - 1)]) * padded + 8 * g;
            auto sums = [&](int k, pu4 (&x)[3]) {  // h of a row, 8 ranks, as parts
                float h[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                if (32 * k + 8 * g < run.rank)
#pragma unroll 4
                    for (int s = 0; s < a.ks; ++s) {
                        const float *p = part + (int64_t)s * a.n_tok * padded + 32 * k;
                        const pf4 u = *(const pf4 *)p, v = *(const pf4 *)(p + 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] += u[e], h[4 + e] += v[e];
                    }
                parts8<T_BF16, 3>(h, x);
            };
            load_w(column(0), 0);
            if (ahead) {
                load_y(yn[0], column(0));
                load_y(yn[1], column(1));
            }
            // h, summed over the parts by neighbouring threads for the workgroup, through the LDS of the results
            pu4 x[KH][3];
            if constexpr (KB > 0) {
                constexpr int Q = 8 * SB, ALL = (ROWS ? 64 : 16) * Q;  // threads to a row, and to all
                auto sum = [&](int kb, auto parts) {  // every load is under way before the first is waited for
                    constexpr int N = decltype(parts)::value;
#pragma unroll
                    for (int i0 = 0; i0 < ALL; i0 += 256) {
                        const int i = i0 + tid, row = min(i / Q, (ROWS ? 64 : 16) - 1), r = 32 * SB * kb + 4 * (i % Q);
                        // eights of ranks: what is behind the last one is finite if that is; behind them, and behind the rows, others, which are not used
                        const float *p = a.part + (int64_t)(base + list[min(t0 + row, n - 1)]) * padded + ((r & ~7) < run.rank ? r : 0);
                        pf4 v[N];
#pragma unroll
                        for (int s = 0; s < N; ++s) v[s] = *(const pf4 *)(p + (int64_t)min(s, a.ks - 1) * a.n_tok * padded);
#pragma unroll
                        for (int s = 1; s < N; ++s)
                            if (s < a.ks) v[0] += v[s];
                        if (ALL >= 256 || i < ALL) *(pf4 *)(&tiles[0][0] + row * LD + 4 * (i % Q)) = v[0];
                    }
                };
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    if (kb) lds_barrier();
                    if (a.ks > 4) sum(kb, std::integral_constant<int, MOST_PARTS>{});
                    else sum(kb, std::integral_constant<int, 4>{});
                    lds_barrier();
#pragma unroll
                    for (int k = 0; k < SB; ++k) {
                        const float *p = out + c * LD + 32 * k + 8 * g;
                        float h[8];
                        *(pf4 *)h = *(const pf4 *)p, *(pf4 *)(h + 4) = *(const pf4 *)(p + 4);
#pragma unroll
                        for (int e = 0; e < 8; ++e) h[e] = 32 * (SB * kb + k) + 8 * g < run.rank ? h[e] : 0.0f;
                        parts8<T_BF16, 3>(h, x[SB * kb + k]);
                    }
                }
            }
            auto turn = [&](lf4 (&v)[I], int i) {
                const int n0 = column(i), next = column(i + 1);
                pf4 acc[J];
#pragma unroll
                for (int j = 0; j < J; ++j) acc[j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
                auto block = [&](int kb, const pu4 (*h)[3]) {
                    const bool last = kb + 1 == kbs;
                    lds_barrier();  // the products before are done
                    put_w(kb);
                    load_w(last ? next : n0, last ? 0 : kb + 1);  // behind the last the last again: in a branch it would be waited for at once
                    lds_barrier();
#pragma unroll
                    for (int k = 0; k < SB; ++k)
                        if (SB * kb + k < steps)
#pragma unroll
                            for (int j0 = 0; j0 < J; j0 += P) {
                                pu4 w[P][NW];
#pragma unroll
                                for (int j = 0; j < P; ++j) S::get(wl, ROWS ? j0 + j : wave, k, lane, w[j]);
                                multiply<TYPE, P>(acc + j0, w, h[k]);
                            }
                };
                if constexpr (KB > 0) {
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
                        if (kb < kbs) block(kb, x + SB * kb);
                } else
                    for (int kb = 0; kb < kbs; ++kb) {
                        pu4 h[SB][3];
#pragma unroll
                        for (int k = 0; k < SB; ++k) sums(SB * kb + k, h[k]);
                        block(kb, h);
                    }
                // LDS serves a wavefront in order: only the compiler must keep it, and the workgroup where the rows are shared
                if (ROWS) __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int j = 0; j < J; ++j) *(pf4 *)(out + c * LD + 16 * (ROWS ? j : wave) + 4 * g) = acc[j];
                if (ROWS) __builtin_amdgcn_wave_barrier();
                else lds_barrier();
                const uint32_t o = 4 * (n0 + 4 * c);
                if (n0 + 64 <= a.rows) {
                    pf4 d[I];
#pragma unroll
                    for (int i = 0; i < I; ++i) d[i] = *(const pf4 *)(out + (ROWS ? 4 * i + g : tid >> 4) * LD + 4 * c);
                    if (run.adapter != -1)
#pragma unroll
                        for (int i = 0; i < I; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[i][e] += run.scale * d[i][e];
#pragma unroll
                    for (int i = 0; i < I; ++i)
                        if ((ROWS ? mine + 4 * i + g : t0 + (tid >> 4)) < n) *(lf4 *)((uint8_t *)y + (uint32_t)(yo[i] + o)) = v[i];
                } else {  // a row's last outputs, fewer than 64: one by one
#pragma clang loop unroll(disable)
                    for (int i = ROWS ? lane : tid; i < 1024; i += ROWS ? 64 : 256) {
                        const int row = i >> 6, col = i & 63;
                        if (mine + row >= n || n0 + col >= a.rows) continue;
                        const int64_t at = list[mine + row];
                        const float u = a.yin ? yin[at * a.ldyi + n0 + col] : 0.0f;
                        y[at * a.ldy + n0 + col] = run.adapter != -1 ? u + run.scale * out[row * LD + col] : u;
                    }
                }
                if (ahead) load_y(v, column(i + 2));
                else
#pragma unroll
                    for (int i = 0; i < I; ++i) v[i] = lf4{0.0f, 0.0f, 0.0f, 0.0f};
            };
#pragma clang loop unroll(disable)
            for (int i = 0; i < turns; i += 2) {
                turn(yn[0], i);
                if (i + 1 >= turns) break;
                turn(yn[1], i + 1);
            }
            lds_barrier();  // the next rows' values go where these were
        }
    }
}

int rank_blocks(const LoraArgs &a) { return (a.max_rank + 16 * a.nr - 1) / (16 * a.nr); }
int64_t tiles_of(const LoraArgs &a) { return ((int64_t)a.n_tok + a.tile - 1) / a.tile; }

template <int TYPE, bool ROWS>
void launch_up(const LoraArgs &a, unsigned grid, hipStream_t s) {
    if (a.max_rank <= 32) lora_up_kernel<TYPE, 1, 1, ROWS><<<grid, 256, 0, s>>>(a);
    else if (a.max_rank <= 64) lora_up_kernel<TYPE, 2, 1, ROWS><<<grid, 256, 0, s>>>(a);
    else if (a.max_rank <= 128) lora_up_kernel<TYPE, 2, 2, ROWS><<<grid, 256, 0, s>>>(a);
    else lora_up_kernel<TYPE, 2, 0, ROWS><<<grid, 256, 0, s>>>(a);
}
template <int TYPE>
hipError_t launch_type(const LoraArgs &a, hipStream_t s) {
    const int64_t tiles = tiles_of(a) * a.slots;
    const unsigned down = (unsigned)(tiles * a.ks * rank_blocks(a)), up = (unsigned)(tiles * ((a.rows + a.ucols - 1) / a.ucols));
    if (a.whole) {
        if (a.nr == 1) lora_down_kernel<TYPE, 1><<<down, 256, 0, s>>>(a);
        else if (a.nr == 2) lora_down_kernel<TYPE, 2><<<down, 256, 0, s>>>(a);
        else lora_down_kernel<TYPE, 4><<<down, 256, 0, s>>>(a);
        launch_up<TYPE, true>(a, up, s);
    } else {
        if (a.nr == 1) lora_down_split_kernel<TYPE, 1><<<down, 256, 0, s>>>(a);
        else if (a.nr == 2) lora_down_split_kernel<TYPE, 2><<<down, 256, 0, s>>>(a);
        else lora_down_split_kernel<TYPE, 4><<<down, 256, 0, s>>>(a);
        launch_up<TYPE, false>(a, up, s);
    }
    return hipGetLastError();
}

}  // namespace

size_t lora_plan(LoraArgs &a, int num_cu) {
    // Tiles of 64 rows, whose rows of one adapter share its reads. In prompts most of a tile is one sequence's, and each wavefront has rows of its own,
    // if there are tiles for the device; few rows, and many short prompts, are better in tiles of 16 (4096 -> 14336, F16, rank 64; one prompt of 512: 27 us,
    // 34 with 64; of 1024: 48 and 49; of 2048: 82 and 76; 64 of 63: 220 and 200. 4096 -> 6144, F32, rank 32; 128 of 16: 46 and 74; 256 of 4, which are
    // tiles of 64 again: 40, of 16: 69).
    // One plan for all rows: prompts beside single tokens of many adapters are better in calls of their own (24 adapters, BF16, rank 64; 8192 + 63 single:
    // 1009 us, in two calls 269; 2048 + 63: 286 and 94; 512 + 255: 356 and 79).
    const bool prompts = a.n_tok >= 16 * (int64_t)a.n_seq;
    a.whole = a.n_tok >= 32 * (int64_t)a.n_seq && a.n_tok >= 4 * num_cu;
    a.tile = a.whole || !prompts ? 64 : 16;
    const int64_t tiles = tiles_of(a);
    a.most = (int)std::min<int64_t>(std::min(a.n_seq, a.tile), (int64_t)a.n_adapter + 2);
    a.nr = a.max_rank <= 16 ? 1 : a.max_rank <= 32 ? 2 : 4;
    // A workgroup for every run that a tile could have, while that fills the device twice at most: one after the other they add up (64 tokens of 24
    // adapters: 139 us by one workgroup a tile, 31 by 8, 21 by 26). In prompts 3, more are mostly idle.
    a.slots = (int)std::max<int64_t>(1, std::min<int64_t>(prompts ? std::min(a.most, 3) : a.most, 2 * num_cu / tiles));
    // Columns over as many workgroups as that leaves room for, a step of each wavefront, or of the workgroup, at the least; 8 parts at most, since the
    // second launch sums them (64 tokens: 4 parts 22.5 us, 8 21.1, 16 21.1).
    const int64_t unit = a.whole ? 64 : 256, units = (a.cols + unit - 1) / unit;
    const int64_t ks = std::max<int64_t>(1, std::min<int64_t>({units, MOST_PARTS, 2 * num_cu / (tiles * (prompts ? 1 : a.slots) * rank_blocks(a))}));
    a.kper = (int)((units + ks - 1) / ks * unit);
    a.ks = (a.cols + a.kper - 1) / a.kper;
    // Outputs over so many workgroups that the device is filled, a turn of 64 at the least: 4 a compute unit (64 tokens: 12.7 us; 2 14.0, 3 13.8, 6 15.1,
    // 8 15.8), 2 where a prompt's rows fill it (8192 tokens: 189 us; 1 290, 3 196, 4 215).
    const int64_t steps = (a.rows + 63) / 64, chunks = std::max<int64_t>(1, std::min<int64_t>(steps, (a.whole ? 2 : 4) * num_cu / (tiles * (prompts ? 1 : a.slots))));
    a.ucols = (int)((steps + chunks - 1) / chunks * 64);
    return (size_t)tiles * a.most * sizeof(LoraRun) + (size_t)a.ks * a.n_tok * ((a.max_rank + 15) & ~15) * 4;
}
void lora_scratch(LoraArgs &a, void *p) {
    a.part = (float *)p;  // an even number of floats
    a.runs = (LoraRun *)(a.part + (size_t)a.ks * a.n_tok * ((a.max_rank + 15) & ~15));
}
int64_t lora_grid(const LoraArgs &a) {
    const int64_t tiles = tiles_of(a) * a.slots;
    return std::max(2 * tiles * a.ks * rank_blocks(a), tiles * ((a.rows + 63) / 64));  // at the most
}

hipError_t launch_lora(const LoraArgs &a, hipStream_t s) {
    switch (a.type) {
    case T_F32: return launch_type<T_F32>(a, s);
    case T_F16: return launch_type<T_F16>(a, s);
    case T_BF16: return launch_type<T_BF16>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace fgh
