// fgh_pdecode.hip - paged attention where every sequence has few rows per K / V head: the decode kernel alone.
#include <hip/hip_runtime.h>

#include "fgh_pdecode.h"

namespace fgh {

namespace {

template <int TYPE, int HD>
__global__ __launch_bounds__(256, (Dec<TYPE, HD>::OCC)) void paged_decode_kernel(PagedAttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    a.ps = 0;  // as the plan says: without what only batches with prompts need
    paged_decode_block<TYPE, HD>(a, blockIdx.x, lds);
}

template <int TYPE>
hipError_t launch_type(const PagedAttnArgs &a, unsigned grid, hipStream_t s) {
    switch (a.p.hd) {
    case 64: paged_decode_kernel<TYPE, 64><<<grid, 256, dec_lds(64), s>>>(a); break;
    case 80: paged_decode_kernel<TYPE, 80><<<grid, 256, dec_lds(80), s>>>(a); break;
    case 96: paged_decode_kernel<TYPE, 96><<<grid, 256, dec_lds(96), s>>>(a); break;
    case 128: paged_decode_kernel<TYPE, 128><<<grid, 256, dec_lds(128), s>>>(a); break;
    case 256: paged_decode_kernel<TYPE, 256><<<grid, 256, dec_lds(256), s>>>(a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_decode(const PagedAttnArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)a.p.n_seq * (unsigned)a.ds * (unsigned)a.p.n_head_kv;
    switch (a.p.type) {
    case T_F32: return launch_type<T_F32>(a, grid, s);
    case T_F16: return launch_type<T_F16>(a, grid, s);
    case T_BF16: return launch_type<T_BF16>(a, grid, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace fgh
