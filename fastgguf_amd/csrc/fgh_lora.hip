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

// rows of a batch in one tile that have one adapter and stand together
struct Run {
    int row, n, adapter;  // adapter -1: none, -2: what is no adapter
};
constexpr int NONE = 1, BAD = 2, FIRST = 3;  // an adapter as a mark that is not 0
// The `which`-th run of the tile of rows base .. base + tile - 1, tile <= 64; n = 0: there are fewer. Every wavefront finds
// it for itself: mark[64] is its own LDS.
__device__ __forceinline__ Run run_of(const LoraArgs &a, int base, int which, int *mark) {
    const int lane = threadIdx.x & 63, top = min(base + a.tile, a.n_tok);
    Run r{0, 0, -1};
    const int end = min(a.tok[a.n_seq], top);
    if (end <= base) return r;
    mark[lane] = 0;
    __builtin_amdgcn_wave_barrier();  // LDS serves a wavefront in order: only the compiler must keep it
    for (int b = max(seq_of_row(a.tok, a.n_seq, base), 0); b < a.n_seq; b += 64) {
        const int s = b + lane;
        const int from = s < a.n_seq ? max(a.tok[s], base) : top, to = s < a.n_seq ? min(a.tok[s + 1], top) : top;
        if (from < to) {
            const int id = a.id[s];
            mark[from - base] = id == -1 ? NONE : (uint32_t)id < (uint32_t)a.n_adapter && (!a.rank || (uint32_t)a.rank[id] <= (uint32_t)a.max_rank) ? FIRST + id : BAD;
        }
        if (__builtin_amdgcn_ballot_w64(s >= a.n_seq || to >= end)) break;
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
    r.adapter = o == NONE ? -1 : o == BAD ? -2 : o - FIRST;
    return r;
}

template <int TYPE>
struct Weights {
    static constexpr int NW = TYPE == T_F32 ? 3 : TYPE == T_F16 ? 2 : 1, ES = TYPE == T_F32 ? 4 : 2;
};
// 8 values of an adapter, those from `n` on 0, as bf16 parts
template <int TYPE>
__device__ __forceinline__ void weights8(const uint8_t *p, int n, pu4 (&w)[Weights<TYPE>::NW]) {
    pu4 raw[2] = {pu4{0, 0, 0, 0}, pu4{0, 0, 0, 0}};
    if (n > 0) {
        raw[0] = *(const pu4 *)p;
        if constexpr (TYPE == T_F32) raw[1] = *(const pu4 *)(p + 16);
    }
    if constexpr (TYPE == T_F32) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e < n ? __uint_as_float(raw[e / 4][e % 4]) : 0.0f;
        parts8<T_BF16, 3>(x, w);
    } else {
        if (n < 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[0][e] &= 2 * e + 1 < n ? ~0u : 2 * e < n ? 0xffffu : 0u;
        if constexpr (TYPE == T_BF16) w[0] = raw[0];
        else {
            const ph8 h = __builtin_bit_cast(ph8, raw[0]);
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

// h of a run's rows, 16 NR ranks, over a part of the columns: the wavefronts take steps of 32 columns in turn. Lane l: rank l % 16 of a
// tile and row l % 16, columns 8 (l / 16) .. + 7.
template <int TYPE, int RT, int NR>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    constexpr int ES = Weights<TYPE>::ES, NW = Weights<TYPE>::NW;
    __shared__ __attribute__((aligned(16))) pf4 lds[4 * RT * NR * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int blocks = (a.max_rank + 16 * NR - 1) / (16 * NR);
    int b = blockIdx.x;
    const int part = b % a.ks;
    b /= a.ks;
    const int block = b % blocks;
    b /= blocks;
    const int slot = b % a.slots, base = b / a.slots * a.tile;
    const int from = part * a.kper, to = min(a.cols, from + a.kper), r0 = block * 16 * NR;
    const int padded = (a.max_rank + 15) & ~15;
    for (int which = slot;; which += a.slots) {
        const Run run = run_of(a, base, which, (int *)lds + 64 * wave);
        if (run.n == 0) break;
        const int rank = run.adapter < 0 ? 0 : a.rank ? a.rank[run.adapter] : a.max_rank;
        __syncthreads();  // the marks are LDS of the sums, too
        if (r0 >= rank) continue;
        const uint8_t *A = a.a + (int64_t)run.adapter * a.max_rank * a.cols * ES;
        for (int t0 = 0; t0 < run.n; t0 += 16 * RT) {
            pf4 acc[RT][NR];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int j = 0; j < NR; ++j) acc[t][j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
            const float *x[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) x[t] = a.x + (run.row + min(t0 + 16 * t + c, run.n - 1)) * a.ldx;
            for (int k0 = from + 32 * wave; k0 < to; k0 += 128) {
                const int k = k0 + 8 * g;
                const bool in = k < to;  // columns end at a multiple of 8
                pu4 w[NR][NW];
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    const int r = r0 + 16 * j + c;
                    weights8<TYPE>(A + ((int64_t)min(r, rank - 1) * a.cols + (in ? k : 0)) * ES, in && r < rank ? 8 : 0, w[j]);
                }
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    if (t0 + 16 * t >= run.n) break;
                    float v[8];
                    const lf4 u0 = *(const lf4 *)(x[t] + (in ? k : 0)), u1 = *(const lf4 *)(x[t] + (in ? k : 0) + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = in ? u0[e] : 0.0f, v[4 + e] = in ? u1[e] : 0.0f;
                    pu4 p[3];
                    parts8<T_BF16, 3>(v, p);
#pragma unroll
                    for (int j = 0; j < NR; ++j) multiply<TYPE>(acc[t][j], w[j], p);
                }
            }
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int j = 0; j < NR; ++j) lds[((wave * RT + t) * NR + j) * 64 + lane] = acc[t][j];
            __syncthreads();
            for (int i = wave; i < RT * NR; i += 4) {
                const int t = i / NR, j = i - t * NR, row = t0 + 16 * t + c, r = r0 + 16 * j + 4 * g;
                const pf4 v = (lds[i * 64 + lane] + lds[(RT * NR + i) * 64 + lane]) + (lds[(2 * RT * NR + i) * 64 + lane] + lds[(3 * RT * NR + i) * 64 + lane]);
                if (row < run.n && r < padded) *(pf4 *)(a.part + ((int64_t)part * a.n_tok + run.row + row) * padded + r) = v;
            }
            __syncthreads();
        }
    }
}

constexpr int UP_COLS = 256;  // outputs of a workgroup, 64 a wavefront

// y of a run's rows, 256 of the outputs. Lane l: output l % 16 of a tile and row l % 16, ranks 8 (l / 16) .. + 7; it gets outputs
// 4 (l / 16) .. + 3 of its row.
template <int TYPE, int RT>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a) {
    constexpr int ES = Weights<TYPE>::ES, NW = Weights<TYPE>::NW;
    __shared__ int marks[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int blocks = (a.rows + UP_COLS - 1) / UP_COLS;
    int b = blockIdx.x;
    const int n0 = b % blocks * UP_COLS + 64 * wave;
    b /= blocks;
    const int slot = b % a.slots, base = b / a.slots * a.tile;
    const int padded = (a.max_rank + 15) & ~15;
    for (int which = slot;; which += a.slots) {
        const Run run = run_of(a, base, which, marks + 64 * wave);
        if (run.n == 0) break;
        if (run.adapter == -1 && a.y == a.yin) continue;
        const int rank = run.adapter < 0 ? 0 : a.rank ? a.rank[run.adapter] : a.max_rank;
        const float scale = run.adapter == -2 ? __builtin_nanf("") : run.adapter < 0 ? 0.0f : a.scale ? a.scale[run.adapter] : 1.0f;
        const uint8_t *B = a.b + (int64_t)max(run.adapter, 0) * a.rows * a.max_rank * ES;
        for (int t0 = 0; t0 < run.n; t0 += 16 * RT) {
            pf4 acc[RT][4];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][j] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
            for (int k0 = 0; k0 < rank; k0 += 32) {
                const int k = k0 + 8 * g, have = rank - k;
                pu4 w[4][NW];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    weights8<TYPE>(B + ((int64_t)min(n0 + 16 * j + c, a.rows - 1) * a.max_rank + (have > 0 ? k : 0)) * ES, have, w[j]);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    if (t0 + 16 * t >= run.n) break;
                    float h[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                    if (have > 0)
                        for (int s = 0; s < a.ks; ++s) {
                            const float *p = a.part + ((int64_t)s * a.n_tok + run.row + min(t0 + 16 * t + c, run.n - 1)) * padded + k;
                            const pf4 u = *(const pf4 *)p, v = *(const pf4 *)(p + 4);
#pragma unroll
                            for (int e = 0; e < 4; ++e) h[e] += u[e], h[4 + e] += v[e];
                        }
                    pu4 x[3];
                    parts8<T_BF16, 3>(h, x);
#pragma unroll
                    for (int j = 0; j < 4; ++j) multiply<TYPE>(acc[t][j], w[j], x);
                }
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const int row = t0 + 16 * t + c;
                if (row >= run.n) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = n0 + 16 * j + 4 * g;
                    const float *in = a.yin + (run.row + row) * a.ldyi + n;
                    float *out = a.y + (run.row + row) * a.ldy + n;
                    if (n + 4 <= a.rows) {
                        lf4 y = lf4{0.0f, 0.0f, 0.0f, 0.0f};
                        if (a.yin) y = *(const lf4 *)in;
                        if (run.adapter != -1)
#pragma unroll
                            for (int e = 0; e < 4; ++e) y[e] += scale * acc[t][j][e];
                        *(lf4 *)out = y;
                    } else
                        for (int e = 0; e < 4 && n + e < a.rows; ++e) {
                            const float y = a.yin ? in[e] : 0.0f;
                            out[e] = run.adapter != -1 ? y + scale * acc[t][j][e] : y;
                        }
                }
            }
        }
    }
}

template <int TYPE, int RT>
hipError_t launch_type(const LoraArgs &a, hipStream_t s) {
    const int64_t tiles = ((int64_t)a.n_tok + a.tile - 1) / a.tile * a.slots;
    const unsigned down = (unsigned)(tiles * a.ks * ((a.max_rank + 16 * a.nr - 1) / (16 * a.nr)));
    switch (a.nr) {
    case 1: lora_down_kernel<TYPE, RT, 1><<<down, 256, 0, s>>>(a); break;
    case 2: lora_down_kernel<TYPE, RT, 2><<<down, 256, 0, s>>>(a); break;
    default: lora_down_kernel<TYPE, RT, 4><<<down, 256, 0, s>>>(a); break;
    }
    lora_up_kernel<TYPE, RT><<<(unsigned)(tiles * ((a.rows + UP_COLS - 1) / UP_COLS)), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

size_t lora_plan(LoraArgs &a, int num_cu) {
    // tiles of 16 rows, or of 64 where sequences have that many
    a.tile = a.n_tok >= 32 * (int64_t)a.n_seq ? 64 : 16;
    const int64_t tiles = ((int64_t)a.n_tok + a.tile - 1) / a.tile;
    a.nr = a.max_rank <= 16 ? 1 : a.max_rank <= 32 ? 2 : 4;
    const int blocks = (a.max_rank + 16 * a.nr - 1) / (16 * a.nr);
    // a workgroup for every run that a tile could have, while that fills the device twice at most
    const int most = std::min(a.n_seq, a.tile);
    a.slots = (int)std::max<int64_t>(1, std::min<int64_t>(most, 2 * num_cu / std::max<int64_t>(1, tiles)));
    // columns over as many workgroups as that leaves room for, 128 columns each at the least
    const int64_t steps = (a.cols + 127) / 128;
    const int64_t ks = std::max<int64_t>(1, std::min<int64_t>({steps, 32, 2 * num_cu / (tiles * a.slots * blocks)}));
    a.kper = (int)((steps + ks - 1) / ks * 128);
    a.ks = (a.cols + a.kper - 1) / a.kper;
    return (size_t)a.ks * a.n_tok * ((a.max_rank + 15) & ~15) * 4;
}
int64_t lora_grid(const LoraArgs &a) {
    const int64_t tiles = ((int64_t)a.n_tok + a.tile - 1) / a.tile * a.slots;
    return std::max(tiles * a.ks * ((a.max_rank + 16 * a.nr - 1) / (16 * a.nr)), tiles * ((a.rows + UP_COLS - 1) / UP_COLS));
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
