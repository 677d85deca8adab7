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
// The `which`-th run of rows of one adapter in the tile of rows base .. base + tile - 1, tile <= 64; n = 0: there are fewer. Every
// wavefront finds it for itself: mark[64] is its own LDS.
__device__ __forceinline__ LoraRun run_of(const LoraArgs &a, int base, int which, int *mark) {
    const int lane = threadIdx.x & 63, top = min(base + a.tile, a.n_tok), end = min(a.tok[a.n_seq], top);
    LoraRun r{0, 0, -1, 0, 0.0f};
    mark[lane] = 0;
    __builtin_amdgcn_wave_barrier();  // LDS serves a wavefront in order: only the compiler must keep it
    // few sequences are looked through from the first one: a load less that others wait for
    for (int b = a.n_seq > 256 ? max(seq_of_row(a.tok, a.n_seq, base), 0) : 0; b < a.n_seq; b += 64) {
        const int s = min(b + lane, a.n_seq - 1), id = a.id[s];
        const int from = max(a.tok[s], base), to = min(a.tok[s + 1], top);
        if (b + lane < a.n_seq && from < to)
            mark[from - base] = id == -1 ? NONE : (uint32_t)id < (uint32_t)a.n_adapter ? FIRST + id : BAD;
        if (__builtin_amdgcn_ballot_w64(b + lane >= a.n_seq || to >= end)) break;
    }
    __builtin_amdgcn_wave_barrier();
    const int m = mark[lane];
    const uint64_t starts = __builtin_amdgcn_ballot_w64(m != 0), mine = starts & (~0ull >> (63 - lane));
    const int first = __shfl(m, 63 - __builtin_clzll(mine | 1), 64), own = mine && base + lane < end ? first : 0;
    const int before = __shfl_up(own, 1, 64);
    uint64_t runs = __builtin_amdgcn_ballot_w64(own != 0 && (lane == 0 || before != own));
    const uint64_t none = __builtin_amdgcn_ballot_w64(own == 0);
    for (int i = 0; i < which && runs; ++i) runs &= runs - 1;
    if (!runs) return r;
    const int at = __builtin_ctzll(runs);
    const uint64_t stop = (runs & (runs - 1)) | (none & ~((2ull << at) - 1));
    r.row = base + at;
    r.n = (stop ? __builtin_ctzll(stop) : 64) - at;
    const int o = __builtin_amdgcn_readlane(own, at);
    if (o == NONE) return r;
    r.adapter = -2, r.scale = __builtin_nanf("");
    if (o == BAD) return r;
    const int rank = __builtin_amdgcn_readfirstlane(a.rank ? a.rank[o - FIRST] : a.max_rank);
    if ((uint32_t)rank > (uint32_t)a.max_rank) return r;
    r.adapter = o - FIRST, r.rank = rank;
    r.scale = a.scale ? a.scale[o - FIRST] : 1.0f;
    return r;
}

template <int TYPE>
struct Weights {
    static constexpr int NW = TYPE == T_F32 ? 3 : TYPE == T_F16 ? 2 : 1, ES = TYPE == T_F32 ? 4 : 2;
};
// 8 values of an adapter as they are in memory, and, those from `n` on 0, as bf16 parts
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
template <int TYPE>
__device__ __forceinline__ void weights8(const Raw<TYPE> &raw, int n, pu4 (&w)[Weights<TYPE>::NW]) {
    if constexpr (TYPE == T_F32) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e < n ? __uint_as_float(raw.v[e / 4][e % 4]) : 0.0f;
        parts8<T_BF16, 3>(x, w);
    } else {
        pu4 u = raw.v[0];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = n >= 2 * e + 2 ? u[e] : n > 2 * e ? u[e] & 0xffffu : 0u;
        if constexpr (TYPE == T_BF16) w[0] = u;
        else {
            const ph8 h = __builtin_bit_cast(ph8, u);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
            parts8<T_BF16, 2>(x, w);  // 11 bits: nothing is left
        }
    }
}
// D += W X, the smallest products first
template <int TYPE>
__device__ __forceinline__ void multiply(pf4 &d, const pu4 (&w)[Weights<TYPE>::NW], const pu4 (&x)[3]) {
    constexpr int NW = Weights<TYPE>::NW;
#pragma unroll
    for (int sum = NW == 3 ? 2 : NW + 1; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i < NW; ++i)
            if (sum - i >= 0 && sum - i < 3) mma16<T_BF16>(d, w[i], x[sum - i]);
}

constexpr int DOWN_WAVES = 8;

// h of a run's rows, 16 NR ranks, over a part of the columns: the wavefronts take steps of 32 columns in turn, the next one's values on their
// way during the products of one. Lane l: rank l % 16 of a tile and row l % 16, columns 8 (l / 16) .. + 7.
template <int TYPE, int RT, int NR>
__global__ __launch_bounds__(64 * DOWN_WAVES) void lora_down_kernel(LoraArgs a) {
    constexpr int ES = Weights<TYPE>::ES, NW = Weights<TYPE>::NW, HALF = DOWN_WAVES / 2, TILES = RT * NR;
    __shared__ __attribute__((aligned(16))) pf4 lds[HALF * TILES * 64];
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
    for (int which = slot; which < a.most; which += a.slots) {
        const LoraRun run = run_of(a, base, which, marks + 64 * wave);
        if (part == 0 && block == 0 && tid == 0) a.runs[(int64_t)tile * a.most + which] = run;
        if (run.n == 0) break;
        if (run.adapter < 0 || r0 >= run.rank) continue;
        const uint8_t *A = a.a + (int64_t)run.adapter * a.max_rank * a.cols * ES;
        for (int t0 = 0; t0 < run.n; t0 += 16 * RT) {
            pf4 acc[RT][NR];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int j = 0; j < NR; ++j) acc[t][j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
            const float *x[RT];
            const uint8_t *w[NR];
#pragma unroll
            for (int t = 0; t < RT; ++t) x[t] = a.x + (run.row + min(t0 + 16 * t + c, run.n - 1)) * a.ldx;
#pragma unroll
            for (int j = 0; j < NR; ++j) w[j] = A + (int64_t)min(r0 + 16 * j + c, run.rank - 1) * a.cols * ES;
            const int tiles = min(NR, (run.rank - r0 + 15) / 16), rows = min(RT, (run.n - t0 + 15) / 16);
            lf4 xn[RT][2];
            Raw<TYPE> wn[NR];
            auto load = [&](int k0) {  // columns end at a multiple of 8; behind them any column's, times 0
                const int k = min(k0 + 8 * g, a.cols - 8);
#pragma unroll
                for (int j = 0; j < NR; ++j)
                    if (j < tiles) wn[j] = raw8<TYPE>(w[j] + (int64_t)k * ES);
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    if (t < rows) xn[t][0] = *(const lf4 *)(x[t] + k), xn[t][1] = *(const lf4 *)(x[t] + k + 4);
            };
            int k0 = from + 32 * wave;
            if (k0 < to) load(k0);
            for (; k0 < to; k0 += 32 * DOWN_WAVES) {
                const bool in = k0 + 8 * g < to;
                pu4 p[RT][3];
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = in ? xn[t][e / 4][e % 4] : 0.0f;
                    parts8<T_BF16, 3>(v, p[t]);
                }
                Raw<TYPE> wc[NR];
#pragma unroll
                for (int j = 0; j < NR; ++j) wc[j] = wn[j];
                if (k0 + 32 * DOWN_WAVES < to) load(k0 + 32 * DOWN_WAVES);
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    if (j >= tiles) break;
                    pu4 q[NW];
                    weights8<TYPE>(wc[j], in && r0 + 16 * j + c < run.rank ? 8 : 0, q);
#pragma unroll
                    for (int t = 0; t < RT; ++t)
                        if (t < rows) multiply<TYPE>(acc[t][j], q, p[t]);
                }
            }
            // the wavefronts' sums: the second half to the first, then all to the first ones
            auto at = [&](int w, int i) -> pf4 & { return lds[(w * TILES + i) * 64 + lane]; };
            if (wave >= HALF)
#pragma unroll
                for (int i = 0; i < TILES; ++i) at(wave - HALF, i) = acc[i / NR][i % NR];
            __syncthreads();
            if (wave < HALF)
#pragma unroll
                for (int i = 0; i < TILES; ++i) at(wave, i) += acc[i / NR][i % NR];
            __syncthreads();
            for (int i = wave; i < TILES; i += DOWN_WAVES) {
                const int row = t0 + 16 * (i / NR) + c, r = r0 + 16 * (i % NR) + 4 * g;
                pf4 v = at(0, i);
#pragma unroll
                for (int w = 1; w < HALF; ++w) v += at(w, i);
                if (row < run.n && r < padded) *(pf4 *)(a.part + ((int64_t)part * a.n_tok + run.row + row) * padded + r) = v;
            }
            __syncthreads();
        }
    }
}

// y of a run's rows, ucols of the outputs: the sums of h go to LDS once, as parts, and each wavefront takes 32 outputs at a time, the
// next ones' values on their way during the products of some. Lane l: output l % 16 of a tile and row l % 16, ranks 8 (l / 16) .. + 7; it gets
// outputs 4 (l / 16) .. + 3 of its row. KR: steps of 32 ranks whose adapter values wait in registers, 0: any number, none wait.
template <int TYPE, int RT, int KR>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a) {
    constexpr int ES = Weights<TYPE>::ES, NW = Weights<TYPE>::NW;
    extern __shared__ __attribute__((aligned(16))) pu4 hs[];  // [steps][RT][3][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int blocks = (a.rows + a.ucols - 1) / a.ucols;
    int b = blockIdx.x;
    const int first = b % blocks * a.ucols, end = min(a.rows, first + a.ucols);
    b /= blocks;
    const int slot = b % a.slots, tile = b / a.slots;
    const int padded = (a.max_rank + 15) & ~15;
    for (int which = slot; which < a.most; which += a.slots) {
        const LoraRun run = a.runs[(int64_t)tile * a.most + which];
        if (run.n == 0) break;
        if (run.adapter == -1 && a.y == a.yin) continue;
        const int steps = (run.rank + 31) / 32;
        const uint8_t *B = a.b + (int64_t)max(run.adapter, 0) * a.rows * a.max_rank * ES;
        for (int t0 = 0; t0 < run.n; t0 += 16 * RT) {
            const int rows = min(RT, (run.n - t0 + 15) / 16);
            lf4 yn[2][RT];
            Raw<TYPE> wn[2][KR ? KR : 1];
            auto raw = [&](int n0, int j, int k0) {  // ranks behind the adapter's are cut later: any that there are
                return raw8<TYPE>(B + ((int64_t)min(n0 + 16 * j + c, a.rows - 1) * a.max_rank + min(k0 + 8 * g, a.max_rank - 8)) * ES);
            };
            auto load = [&](int n0) {
                if (KR)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int k = 0; k < KR; ++k)
                            if (k < steps) wn[j][k] = raw(n0, j, 32 * k);
                if (a.yin)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int t = 0; t < RT; ++t) {
                            const int n = n0 + 16 * j + 4 * g;
                            if (t < rows && n + 4 <= a.rows) yn[j][t] = *(const lf4 *)(a.yin + (run.row + min(t0 + 16 * t + c, run.n - 1)) * a.ldyi + n);
                        }
            };
            int n0 = first + 32 * wave;
            if (n0 < end) load(n0);
            for (int i = tid; i < steps * rows * 64; i += 256) {
                const int l = i & 63, t = (i >> 6) % rows, k = (i >> 6) / rows, r = 32 * k + 8 * (l >> 4);
                float h[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                if (r < run.rank) {
                    const float *p = a.part + (int64_t)(run.row + min(t0 + 16 * t + (l & 15), run.n - 1)) * padded + r;
#pragma unroll 8
                    for (int s = 0; s < a.ks; ++s) {
                        const pf4 u = *(const pf4 *)(p + (int64_t)s * a.n_tok * padded), v = *(const pf4 *)(p + (int64_t)s * a.n_tok * padded + 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] += u[e], h[4 + e] += v[e];
                    }
                }
                pu4 x[3];
                parts8<T_BF16, 3>(h, x);
#pragma unroll
                for (int e = 0; e < 3; ++e) hs[((k * RT + t) * 3 + e) * 64 + l] = x[e];
            }
            __syncthreads();
            for (; n0 < end; n0 += 128) {
                lf4 y[2][RT];
                Raw<TYPE> wc[2][KR ? KR : 1];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int t = 0; t < RT; ++t) y[j][t] = a.yin ? yn[j][t] : lf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < (KR ? KR : 1); ++k) wc[j][k] = wn[j][k];
                }
                if (n0 + 128 < end) load(n0 + 128);
                pf4 acc[2][RT];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int t = 0; t < RT; ++t) acc[j][t] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
                auto step = [&](int k, const Raw<TYPE> &w0, const Raw<TYPE> &w1) {
                    pu4 w[2][NW];
                    weights8<TYPE>(w0, run.rank - 32 * k - 8 * g, w[0]);
                    weights8<TYPE>(w1, run.rank - 32 * k - 8 * g, w[1]);
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        if (t >= rows) break;
                        pu4 x[3];
#pragma unroll
                        for (int e = 0; e < 3; ++e) x[e] = hs[((k * RT + t) * 3 + e) * 64 + lane];
                        multiply<TYPE>(acc[0][t], w[0], x);
                        multiply<TYPE>(acc[1][t], w[1], x);
                    }
                };
                if constexpr (KR > 0) {
#pragma unroll
                    for (int k = 0; k < KR; ++k)
                        if (k < steps) step(k, wc[0][k], wc[1][k]);
                } else
                    for (int k = 0; k < steps; ++k) step(k, raw(n0, 0, 32 * k), raw(n0, 1, 32 * k));
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const int row = t0 + 16 * t + c;
                    if (row >= run.n) continue;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int n = n0 + 16 * j + 4 * g;
                        float *out = a.y + (run.row + row) * a.ldy + n;
                        if (n + 4 <= a.rows) {
                            lf4 v = y[j][t];
                            if (run.adapter != -1)
#pragma unroll
                                for (int e = 0; e < 4; ++e) v[e] += run.scale * acc[j][t][e];
                            *(lf4 *)out = v;
                        } else
                            for (int e = 0; e < 4 && n + e < a.rows; ++e) {
                                const float v = a.yin ? a.yin[(run.row + row) * a.ldyi + n + e] : 0.0f;
                                out[e] = run.adapter != -1 ? v + run.scale * acc[j][t][e] : v;
                            }
                    }
                }
            }
            __syncthreads();
        }
    }
}

int rank_blocks(const LoraArgs &a) { return (a.max_rank + 16 * a.nr - 1) / (16 * a.nr); }
int64_t tiles_of(const LoraArgs &a) { return ((int64_t)a.n_tok + a.tile - 1) / a.tile; }

template <int TYPE, int RT>
hipError_t launch_type(const LoraArgs &a, hipStream_t s) {
    const int64_t tiles = tiles_of(a) * a.slots;
    const unsigned down = (unsigned)(tiles * a.ks * rank_blocks(a)), up = (unsigned)(tiles * ((a.rows + a.ucols - 1) / a.ucols));
    switch (a.nr) {
    case 1: lora_down_kernel<TYPE, RT, 1><<<down, 64 * DOWN_WAVES, 0, s>>>(a); break;
    case 2: lora_down_kernel<TYPE, RT, 2><<<down, 64 * DOWN_WAVES, 0, s>>>(a); break;
    default: lora_down_kernel<TYPE, RT, 4><<<down, 64 * DOWN_WAVES, 0, s>>>(a); break;
    }
    const int steps = (a.max_rank + 31) / 32, lds = steps * RT * 3 * 1024;
    if (steps == 1) lora_up_kernel<TYPE, RT, 1><<<up, 256, lds, s>>>(a);
    else if (steps == 2) lora_up_kernel<TYPE, RT, 2><<<up, 256, lds, s>>>(a);
    else lora_up_kernel<TYPE, RT, 0><<<up, 256, lds, s>>>(a);
    return hipGetLastError();
}

}  // namespace

size_t lora_plan(LoraArgs &a, int num_cu) {
    // tiles of 64 rows where there are enough of them and h fits the 64 KB of LDS, else of 16
    a.tile = a.n_tok >= 32 * (int64_t)a.n_seq && a.n_tok >= 4 * num_cu && a.max_rank <= 160 ? 64 : 16;
    const int64_t tiles = tiles_of(a);
    a.most = std::min(a.n_seq, a.tile);
    a.nr = a.max_rank <= 16 ? 1 : a.max_rank <= 32 ? 2 : 4;
    // a workgroup for every run that a tile could have where sequences are short, while that fills the device twice at most
    a.slots = a.tile == 64 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(a.most, (int64_t)a.n_seq * a.tile / a.n_tok + 2), 2 * num_cu / tiles));
    // columns over as many workgroups as that leaves room for, a step of each wavefront at the least
    const int64_t unit = 32 * DOWN_WAVES, units = (a.cols + unit - 1) / unit;
    const int64_t ks = std::max<int64_t>(1, std::min<int64_t>({units, 8, 2 * num_cu / (tiles * a.slots * rank_blocks(a))}));
    a.kper = (int)((units + ks - 1) / ks * unit);
    a.ks = (a.cols + a.kper - 1) / a.kper;
    // outputs over so many workgroups that the device is filled, 128 (a step of each wavefront) at the least
    const int64_t steps = (a.rows + 127) / 128, chunks = std::max<int64_t>(1, std::min<int64_t>(steps, 4 * num_cu / (tiles * a.slots)));
    a.ucols = (int)((steps + chunks - 1) / chunks * 128);
    return (size_t)tiles * a.most * sizeof(LoraRun) + (size_t)a.ks * a.n_tok * ((a.max_rank + 15) & ~15) * 4;
}
void lora_scratch(LoraArgs &a, void *p) {
    a.part = (float *)p;
    a.runs = (LoraRun *)(a.part + (size_t)a.ks * a.n_tok * ((a.max_rank + 15) & ~15));
}
int64_t lora_grid(const LoraArgs &a) {
    const int64_t tiles = tiles_of(a) * a.slots;
    return std::max(2 * tiles * a.ks * rank_blocks(a), tiles * ((a.rows + a.ucols - 1) / a.ucols));
}

hipError_t launch_lora(const LoraArgs &a, hipStream_t s) {
    switch (a.type) {
    case T_F32: return a.tile == 64 ? launch_type<T_F32, 4>(a, s) : launch_type<T_F32, 1>(a, s);
    case T_F16: return a.tile == 64 ? launch_type<T_F16, 4>(a, s) : launch_type<T_F16, 1>(a, s);
    case T_BF16: return a.tile == 64 ? launch_type<T_BF16, 4>(a, s) : launch_type<T_BF16, 1>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace fgh
