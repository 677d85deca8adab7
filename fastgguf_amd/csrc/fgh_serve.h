// fgh_serve.h - what a server of many sequences does around the paged cache: pages and rows of a batch (fgh_reserve.hip), drafted
// tokens checked and tokens drawn (fgh_verify.hip), adapters of many requests (fgh_lora.hip). Internal.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fgh {

// The sequence of row t, or -1: the last s with tok[s] <= t, if t < tok[s + 1]; tok[0 .. n_seq] does not decrease. A wavefront's 64
// lanes look at 256 starts at a time, evenly apart: 65535 sequences take two loads that wait for each other.
__device__ __forceinline__ int seq_of_row(const int32_t *tok, int n_seq, int t) {
    const int lane = threadIdx.x & 63;
    int base = 0, len = n_seq + 1;
    while (true) {
        const int step = (len + 255) / 256;
        int c = 0;
        int32_t at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) at[i] = tok[base + min((lane + 64 * i) * step, len - 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64((lane + 64 * i) * step < len && at[i] <= t));
        if (c == 0) return base - 1;
        base += (c - 1) * step;
        len = min(step, len - (c - 1) * step);
        if (len == 1) return base >= n_seq ? -1 : base;
    }
}

struct ReserveArgs {
    const int32_t *keep, *add, *held, *free;
    int32_t *held_out, *free_out, *queue, *table, *tok, *len, *seq, *pos;
    int64_t *slot;
    int n_seq, n_tok, max_tok, max_len, n_pages, shift, table_stride;  // max_len: at most the table's positions
    int32_t *pre;  // reserve_scratch bytes
};
size_t reserve_scratch(const ReserveArgs &a);
hipError_t launch_reserve(const ReserveArgs &a, hipStream_t s);

// what a sequence's rows come to: the row t that the next token is drawn from, its sum, largest value and the place of that; the draft d that
// it rejects, or -1; the rows n (0: no token) and the accepted drafts
struct VerifyChoice {
    double sum;
    float top;
    int at, t, d, n, good;
};
struct VerifyArgs {
    const float *logits, *q, *q_lse, *temp, *u, *v;
    const int32_t *tok, *tokens, *len;
    int32_t *n_ok, *next, *keep;
    float *lse;
    int64_t ld, ldq;
    int n_seq, n_tok, max_tok, vocab;
    // set by verify_plan: a row's words over `splits` workgroups, `per` words each, in blocks of 1024 nv; `group` such parts to a workgroup
    int splits, per, nv, group;
    double *sum, *rest;  // [n_tok][splits], [n_seq][splits][(per + 2047) / 2048]
    float *top;          // [n_tok][splits]
    int32_t *at;         // [n_tok][splits]
    VerifyChoice *choice;  // [n_seq]
};
size_t verify_plan(VerifyArgs &a, int num_cu);  // the scratch it takes
void verify_scratch(VerifyArgs &a, void *p);
hipError_t launch_verify(const VerifyArgs &a, hipStream_t s);

// rows of a tile of a batch that have one adapter, a bit each. adapter -1: none, -2: what is no adapter
struct LoraRun {
    uint64_t rows;
    int adapter, rank;
    float scale;
};
struct LoraArgs {
    const uint8_t *a, *b;
    const int32_t *rank, *tok, *id;
    const float *scale, *x, *yin;
    float *y, *part;
    int64_t ldx, ldyi, ldy;
    int type, n_adapter, max_rank, cols, rows, n_seq, n_tok;
    LoraRun *runs;  // [tiles][most]: the second launch takes them from the first
    // set by lora_plan: tiles of `tile` rows, with up to `most` runs each over `slots` workgroups, A x over ks workgroups of kper
    // columns, ranks in blocks of 16 nr; ucols outputs to a workgroup of the second launch
    // `whole`: tiles mostly of one sequence's rows
    int tile, most, slots, ks, kper, nr, ucols;
    bool whole;
};
size_t lora_plan(LoraArgs &a, int num_cu);  // the scratch it takes
void lora_scratch(LoraArgs &a, void *p);
int64_t lora_grid(const LoraArgs &a);  // workgroups of the larger launch, of 256 threads
hipError_t launch_lora(const LoraArgs &a, hipStream_t s);

}  // namespace fgh
