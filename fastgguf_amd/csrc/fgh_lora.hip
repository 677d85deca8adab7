// fgh_lora.hip - low-rank adapters of many requests beside a shared projection on gfx950: y = y_in + scale B (A x), each row with
// its sequence's adapter.
//
// Two launches: h = A x, split over columns where rows are few, then y from the sums of h. A workgroup has the rows of one adapter
// that stand together in a tile of the batch. Both products run on 16 x 16 x 32 bf16 matrix instructions whose fp32 operands are
// taken apart into bf16 parts that hold all their bits (x and h: 3; adapters F32 3, F16 2, BF16 1), so that results are
// those of fp32 products and sums; F32 adapters leave 3 of 9 products out, 2^-24 of the whole on average.
#include <algorithm>

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
        if (__builtin_amdgcn_ballot_w64(b + lane >= a.n_seq || to >= end)) break;
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

// Adapter values of 64 rows (of A: ranks, of B: outputs) and 64 values along them, shared by a workgroup: a thread takes 8 values of a row,
// 8 threads a row's 64, so that an access finds whole lines, and leaves their parts in LDS as the products take them: [4 tiles][2 steps]
// [parts][64 lanes]. (Loaded as the products take them, neighbouring lanes in 16 different rows, every lane was an access of its own to
// the first cache: 1.0 a cycle, the bound of such a kernel.) Lanes are exchanged so that 8 threads write to different banks.
template <int TYPE>
struct Stage {
    static constexpr int NW = Weights<TYPE>::NW, ES = Weights<TYPE>::ES, VALUES = 8 * NW * 64;  // 16-byte values in LDS
    static __device__ __forceinline__ int slot(int c, int g, int k) { return 16 * g + (c ^ (4 * g + k)); }
    static __device__ __forceinline__ void put(pu4 *lds, int row, int chunk, const Raw<TYPE> &raw) {
        const int j = row >> 4, k = chunk >> 2;
        pu4 w[NW];
        weights8<TYPE>(raw, w);
#pragma unroll
        for (int e = 0; e < NW; ++e) lds[((2 * j + k) * NW + e) * 64 + slot(row & 15, chunk & 3, k)] = w[e];
    }
    static __device__ __forceinline__ void get(const pu4 *lds, int j, int k, int lane, pu4 (&w)[NW]) {
#pragma unroll
        for (int e = 0; e < NW; ++e) w[e] = lds[((2 * j + k) * NW + e) * 64 + slot(lane & 15, lane >> 4, k)];
    }
};
constexpr int LD = 68;  // floats between rows of 64 in LDS: 16 rows start in 16 different groups of banks

constexpr int DOWN_WAVES = 8;

// h of few rows that have an adapter in common, 16 NR ranks, over a part of the columns: the wavefronts take steps of 32 columns in turn, the next one's values on their
// way during the products of one. Lane l: rank l % 16 of a tile and row l % 16, columns 8 (l / 16) .. + 7.
template <int TYPE, int NR>
__global__ __launch_bounds__(64 * DOWN_WAVES, 4) void lora_down_split_kernel(LoraArgs a) {
    constexpr int ES = Weights<TYPE>::ES, NW = Weights<TYPE>::NW, HALF = DOWN_WAVES / 2;
    __shared__ __attribute__((aligned(16))) pf4 lds[HALF * NR * 64];
    __shared__ int marks[DOWN_WAVES * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int blocks = (a.max_rank + 16 * NR - 1) / (16 * NR);
    int b = blockIdx.x;
    const int part = b % a.ks;
    b /= a.ks;
    const int block = b % blocks;
    b /= blocks;
    const int slot = b % a.slots, tile = b / a.slots, base = tile * a.tile;
    const int from = part * a.kper, to = min(a.cols, from + a.kper), r0 = block * 16 * NR;
    const int padded = (a.max_rank + 15) & ~15;
    int *list = marks + 64 * wave;
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
        for (int t0 = 0; t0 < n; t0 += 16) {
            pf4 acc[NR];
#pragma unroll
            for (int j = 0; j < NR; ++j) acc[j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
            // a lane's place in its rows of x and of A, from addresses that move along the columns: offsets of 32 bits
            const uint32_t xo = 4 * ((uint32_t)list[min(t0 + c, n - 1)] * (uint32_t)a.ldx + 8 * g);
            uint32_t wo[NR];
            // behind the last rank that one again: what it gives is not used
#pragma unroll
            for (int j = 0; j < NR; ++j) wo[j] = ES * ((uint32_t)min(r0 + 16 * j + c, run.rank - 1) * (uint32_t)a.cols + 8 * g);
            const uint8_t *X = (const uint8_t *)(a.x + base * a.ldx);
            const int tiles = min(NR, (run.rank - r0 + 15) / 16);
            lf4 xn[2];
            Raw<TYPE> wn[NR];
            // columns end at a multiple of 8: lanes behind them look back to the last ones
            auto back = [&](int k0) { return (uint32_t)max(0, k0 + 8 * g + 8 - a.cols); };
            auto load_x = [&](int k0) {
                const uint8_t *p = X + 4 * (int64_t)k0;
                const uint32_t z = k0 + 32 <= a.cols ? 0 : 4 * back(k0);
                xn[0] = *(const lf4 *)(p + xo - z), xn[1] = *(const lf4 *)(p + xo - z + 16);
            };
            auto load_w = [&](int j, int k0) {
                const uint32_t z = k0 + 32 <= a.cols ? 0 : ES * back(k0);
                if (j < tiles) wn[j] = raw8<TYPE>(A + (int64_t)ES * k0 + wo[j] - z);
            };
            int k0 = from + 32 * wave;
            if (k0 < to) {
#pragma unroll
                for (int j = 0; j < NR; ++j) load_w(j, k0);
                load_x(k0);
            }
            for (; k0 < to; k0 += 32 * DOWN_WAVES) {
                const bool more = k0 + 32 * DOWN_WAVES < to, whole = k0 + 32 <= to;
                const float v[8] = {xn[0].x, xn[0].y, xn[0].z, xn[0].w, xn[1].x, xn[1].y, xn[1].z, xn[1].w};
                pu4 p[3];
                parts8<T_BF16, 3>(v, p);
                if (more) load_x(k0 + 32 * DOWN_WAVES);
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    if (j >= tiles) break;
                    pu4 q[1][NW];
                    if (!whole && k0 + 8 * g >= to) wn[j] = Raw<TYPE>{};
                    weights8<TYPE>(wn[j], q[0]);
                    if (more) load_w(j, k0 + 32 * DOWN_WAVES);
                    multiply<TYPE, 1>(acc + j, q, p);
                }
            }
            // the wavefronts' sums: the second half to the first, then all to the first ones
            auto at = [&](int w, int i) -> pf4 & { return lds[(w * NR + i) * 64 + lane]; };
            if (wave >= HALF)
#pragma unroll
                for (int i = 0; i < NR; ++i) at(wave - HALF, i) = acc[i];
            __syncthreads();
            if (wave < HALF)
#pragma unroll
                for (int i = 0; i < NR; ++i) at(wave, i) += acc[i];
            __syncthreads();
            for (int i = wave; i < NR; i += DOWN_WAVES) {
                const int row = t0 + c, r = r0 + 16 * i + 4 * g;
                pf4 v = at(0, i);
#pragma unroll
                for (int w = 1; w < HALF; ++w) v += at(w, i);
                if (row < n && r < padded) *(pf4 *)(a.part + ((int64_t)part * a.n_tok + base + list[row]) * padded + r) = v;
            }
            __syncthreads();
        }
    }
}

// h of a prompt's rows, 16 NR ranks, over a part of the columns: 64 rows to a workgroup, 16 to a wavefront, 64 columns at a time, the next ones'
// values on their way during the products of some. x too goes through LDS, each wavefront's by itself: 16 lanes read 256 bytes of a row.
template <int TYPE, int NR>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    using S = Stage<TYPE>;
    constexpr int ES = S::ES, UNITS = (128 * NR + 255) / 256;
    __shared__ __attribute__((aligned(16))) pu4 wl[2][S::VALUES * NR / 4];
    __shared__ __attribute__((aligned(16))) float xl[4][16 * LD];
    __shared__ int lists[4 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int blocks = (a.max_rank + 16 * NR - 1) / (16 * NR);
    int b = blockIdx.x;
    const int part = b % a.ks;
    b /= a.ks;
    const int block = b % blocks, tile = b / blocks, base = tile * a.tile;
    const int from = part * a.kper, to = min(a.cols, from + a.kper), r0 = block * 16 * NR;
    const int padded = (a.max_rank + 15) & ~15;
    int *list = lists + 64 * wave;
    const int mark = adapters_of(a, base, list);
    uint64_t left = __builtin_amdgcn_ballot_w64(mark != 0);
    for (int which = 0;; ++which) {
        const int m = left ? __builtin_amdgcn_readlane(mark, __builtin_ctzll(left)) : 0;
        const uint64_t rows_of = __builtin_amdgcn_ballot_w64(mark == m) & left;
        left &= ~rows_of;
        const LoraRun run = m ? run_of(a, rows_of, m) : LoraRun{};
        if (part == 0 && block == 0 && tid == 0 && which < a.most) a.runs[(int64_t)tile * a.most + which] = run;  // behind the last: no rows
        if (!m) break;
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
        lf4 xn[4];
        Raw<TYPE> wn[UNITS];
        auto load = [&](int k0) {  // behind the last column the last ones again
            const uint32_t kx = min(k0 + 4 * c, a.cols - 4), kw = min(k0 + 8 * (tid & 7), a.cols - 8);
#pragma unroll
            for (int u = 0; u < UNITS; ++u) wn[u] = raw8<TYPE>(A + wo[u] + ES * kw);
#pragma unroll
            for (int i = 0; i < 4; ++i) xn[i] = *(const lf4 *)(X + xo[i] + 4 * kx);
        };
        auto put_w = [&](pu4 *lds, int k0) {  // times 0 behind the last column
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                if (k0 + 8 * (tid & 7) >= to) wn[u] = Raw<TYPE>{};
                if (NR > 1 || tid < 128) S::put(lds, (tid >> 3) + 32 * u, tid & 7, wn[u]);
            }
        };
        pf4 acc[NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) acc[j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
        float *own = xl[wave];
        load(from);
        put_w(wl[0], from);
        int at = 0;
#pragma clang loop unroll(disable)
        for (int k0 = from; k0 < to; k0 += 64, at ^= 1) {
            // LDS serves a wavefront in order: only the compiler must keep it
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 4; ++i) *(pf4 *)(own + (4 * i + g) * LD + 4 * c) = xn[i];
            __builtin_amdgcn_wave_barrier();
            if (k0 + 64 < to) load(k0 + 64);
            lds_barrier();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                pu4 p[3];
                float v[8];
                *(pf4 *)v = *(const pf4 *)(own + c * LD + 32 * k + 8 * g), *(pf4 *)(v + 4) = *(const pf4 *)(own + c * LD + 32 * k + 8 * g + 4);
                parts8<T_BF16, 3>(v, p);
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    pu4 w[1][S::NW];
                    S::get(wl[at], j, k, lane, w[0]);
                    multiply<TYPE, 1>(acc + j, w, p);
                }
            }
            if (k0 + 64 < to) put_w(wl[at ^ 1], k0 + 64);
        }
        lds_barrier();
        const int row = 16 * wave + c;
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const int r = r0 + 16 * j + 4 * g;
            if (row < n && r < padded) *(pf4 *)(a.part + ((int64_t)part * a.n_tok + base + list[row]) * padded + r) = acc[j];
        }
    }
}

// y of rows that have an adapter in common, ucols of the outputs, 64 at a time and 64 ranks of them, the next ones' values on their way
// during the products of some. ROWS (prompts): each wavefront has 16 rows and all 64 outputs; else (few rows) 16 of the outputs and the
// same rows. Products: lane l has output l % 16 of a tile and row l % 16, ranks 8 (l / 16) .. + 7, and gets outputs 4 (l / 16) .. + 3 of its row;
// through LDS they come to lie as y does, 16 lanes with 256 bytes of a row. KB: blocks of 64 ranks, whose h stays in registers; 0: any number,
// which does not.
template <int TYPE, int KB, bool ROWS>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a) {
    using S = Stage<TYPE>;
    constexpr int ES = S::ES, NW = S::NW, J = ROWS ? 4 : 1, KH = KB ? 2 * KB : 1;
    __shared__ __attribute__((aligned(16))) pu4 wl[2][S::VALUES];
    __shared__ __attribute__((aligned(16))) float tiles[ROWS ? 4 : 1][16 * LD];
    __shared__ int lists[4 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int blocks = (a.rows + a.ucols - 1) / a.ucols;
    int b = blockIdx.x;
    const int first = b % blocks * a.ucols, end = min(a.rows, first + a.ucols);
    b /= blocks;
    const int slot = b % a.slots, tile = b / a.slots, base = tile * a.tile;
    const int padded = (a.max_rank + 15) & ~15;
    float *out = tiles[ROWS ? wave : 0];
    int *list = lists + 64 * wave;
    for (int which = slot; which < a.most; which += a.slots) {
        const LoraRun run = a.runs[(int64_t)tile * a.most + which];
        if (run.rows == 0) break;
        if (run.adapter == -1 && a.y == a.yin) continue;
        const int n = list_rows(run.rows, list), steps = (run.rank + 31) / 32, kbs = max(1, (run.rank + 63) / 64);
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
            lf4 yn[I] = {};
            Raw<TYPE> wn[2];
            auto load_w = [&](int n0, int kb) {  // outputs and ranks behind the last: others, which are not used, or cut
                const int r = min(64 * kb + 8 * (tid & 7), a.max_rank - 8);
#pragma unroll
                for (int u = 0; u < 2; ++u) wn[u] = raw8<TYPE>(B + ES * ((int64_t)min(n0 + (tid >> 3) + 32 * u, a.rows - 1) * a.max_rank + r));
            };
            auto put_w = [&](pu4 *lds, int kb) {
                const int have = run.rank - 64 * kb - 8 * (tid & 7);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (have < 8) mask8<TYPE>(wn[u], first8<TYPE>(have));
                    S::put(lds, (tid >> 3) + 32 * u, tid & 7, wn[u]);
                }
            };
            auto load_y = [&](int n0) {  // a row's last values one by one
                const uint8_t *p = (const uint8_t *)(a.yin + base * a.ldyi + n0 + 4 * c);
                if (n0 + 64 <= a.rows)
#pragma unroll
                    for (int i = 0; i < I; ++i) yn[i] = *(const lf4 *)(p + yio[i]);
                else
#pragma unroll
                    for (int i = 0; i < I; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (n0 + 4 * c + e < a.rows) yn[i][e] = *(const float *)(p + yio[i] + 4 * e);
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
            load_w(first, 0);
            if (a.yin) load_y(first);
            pu4 x[KH][3];
            if (KB)
#pragma unroll
                for (int k = 0; k < KH; ++k)
                    if (k < steps) sums(k, x[k]);
            put_w(wl[0], 0);
            int at = 0;
#pragma clang loop unroll(disable)
            for (int n0 = first; n0 < end; n0 += 64) {
                pf4 acc[J];
#pragma unroll
                for (int j = 0; j < J; ++j) acc[j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
                auto block = [&](int kb, const pu4 (&h0)[3], const pu4 (&h1)[3]) {
                    const bool last = kb + 1 == kbs, more = !last || n0 + 64 < end;
                    if (more) load_w(last ? n0 + 64 : n0, last ? 0 : kb + 1);
                    lds_barrier();
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (2 * kb + k < steps)
#pragma unroll
                            for (int j = 0; j < J; ++j) {
                                pu4 w[1][NW];
                                S::get(wl[at], ROWS ? j : wave, k, lane, w[0]);
                                multiply<TYPE, 1>(acc + j, w, k ? h1 : h0);
                            }
                    at ^= 1;
                    if (more) put_w(wl[at], last ? 0 : kb + 1);
                };
                if constexpr (KB > 0) {
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb)
                        if (kb < kbs) block(kb, x[2 * kb], x[2 * kb + 1]);
                } else
                    for (int kb = 0; kb < kbs; ++kb) {
                        pu4 h[2][3];
                        sums(2 * kb, h[0]);
                        sums(2 * kb + 1, h[1]);
                        block(kb, h[0], h[1]);
                    }
                // LDS serves a wavefront in order: only the compiler must keep it, and the workgroup where the rows are shared
                if (ROWS) __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int j = 0; j < J; ++j) *(pf4 *)(out + c * LD + 16 * (ROWS ? j : wave) + 4 * g) = acc[j];
                if (ROWS) __builtin_amdgcn_wave_barrier();
                else lds_barrier();
                uint8_t *y = (uint8_t *)(a.y + base * a.ldy + n0 + 4 * c);
#pragma unroll
                for (int i = 0; i < I; ++i) {
                    const pf4 d = *(const pf4 *)(out + (ROWS ? 4 * i + g : tid >> 4) * LD + 4 * c);
                    lf4 v = yn[i];
                    if (run.adapter != -1)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += run.scale * d[e];
                    if ((ROWS ? mine + 4 * i + g : t0 + (tid >> 4)) >= n) continue;
                    if (n0 + 64 <= a.rows) *(lf4 *)(y + yo[i]) = v;
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (n0 + 4 * c + e < a.rows) *(float *)(y + yo[i] + 4 * e) = v[e];
                }
                if (a.yin && n0 + 64 < end) load_y(n0 + 64);
            }
            lds_barrier();  // the next rows' values go where these were
        }
    }
}

int rank_blocks(const LoraArgs &a) { return (a.max_rank + 16 * a.nr - 1) / (16 * a.nr); }
int64_t tiles_of(const LoraArgs &a) { return ((int64_t)a.n_tok + a.tile - 1) / a.tile; }

template <int TYPE, bool ROWS>
void launch_up(const LoraArgs &a, unsigned grid, hipStream_t s) {
    if (a.max_rank <= 64) lora_up_kernel<TYPE, 1, ROWS><<<grid, 256, 0, s>>>(a);
    else if (a.max_rank <= 128) lora_up_kernel<TYPE, 2, ROWS><<<grid, 256, 0, s>>>(a);
    else lora_up_kernel<TYPE, 0, ROWS><<<grid, 256, 0, s>>>(a);
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
        if (a.nr == 1) lora_down_split_kernel<TYPE, 1><<<down, 64 * DOWN_WAVES, 0, s>>>(a);
        else if (a.nr == 2) lora_down_split_kernel<TYPE, 2><<<down, 64 * DOWN_WAVES, 0, s>>>(a);
        else lora_down_split_kernel<TYPE, 4><<<down, 64 * DOWN_WAVES, 0, s>>>(a);
        launch_up<TYPE, false>(a, up, s);
    }
    return hipGetLastError();
}

}  // namespace

size_t lora_plan(LoraArgs &a, int num_cu) {
    // tiles of 64 rows, whose rows of one adapter share its reads; prompts with few rows take tiles of 16
    const bool prompts = a.n_tok >= 16 * (int64_t)a.n_seq;
    a.whole = prompts && a.n_tok >= 4 * num_cu;
    a.tile = a.whole || !prompts ? 64 : 16;
    const int64_t tiles = tiles_of(a);
    a.most = (int)std::min<int64_t>(std::min(a.n_seq, a.tile), (int64_t)a.n_adapter + 2);
    a.nr = a.max_rank <= 16 ? 1 : a.max_rank <= 32 ? 2 : 4;
    // a workgroup for every run that a tile of short sequences could have, while that fills the device twice at most
    a.slots = prompts ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(a.most, 2 * num_cu / tiles));
    // columns over as many workgroups as that leaves room for, a step of each wavefront, or of the workgroup, at the least
    const int64_t unit = a.whole ? 64 : 32 * DOWN_WAVES, units = (a.cols + unit - 1) / unit;
    const int64_t ks = std::max<int64_t>(1, std::min<int64_t>({units, 8, 2 * num_cu / (tiles * a.slots * rank_blocks(a))}));
    a.kper = (int)((units + ks - 1) / ks * unit);
    a.ks = (a.cols + a.kper - 1) / a.kper;
    // outputs over so many workgroups that the device is filled, 256 at the least
    const int64_t steps = (a.rows + 255) / 256, chunks = std::max<int64_t>(1, std::min<int64_t>(steps, 4 * num_cu / (tiles * a.slots)));
    a.ucols = (int)((steps + chunks - 1) / chunks * 256);
    return (size_t)tiles * a.most * sizeof(LoraRun) + (size_t)a.ks * a.n_tok * ((a.max_rank + 15) & ~15) * 4;
}
void lora_scratch(LoraArgs &a, void *p) {
    a.part = (float *)p;  // an even number of floats
    a.runs = (LoraRun *)(a.part + (size_t)a.ks * a.n_tok * ((a.max_rank + 15) & ~15));
}
int64_t lora_grid(const LoraArgs &a) {
    const int64_t tiles = tiles_of(a) * a.slots;
    return std::max(2 * tiles * a.ks * rank_blocks(a), tiles * ((a.rows + a.ucols - 1) / a.ucols));
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
