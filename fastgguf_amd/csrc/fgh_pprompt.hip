// fgh_pprompt.hip - paged attention of batches with prompts: the prompt kernel's workgroups, then those of the decode kernel for the
// sequences with few rows, in one launch.
#include <hip/hip_runtime.h>

#include "fgh_pdecode.h"
#include "fgh_pprompt.h"

namespace fgh {

namespace {

template <int TYPE, int HD, int RW>
__global__ __launch_bounds__(256, (Pro<TYPE, HD, RW>::OCC)) void paged_prompt_kernel(PagedAttnArgs a, int nd) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    // grid (tiles x K / V heads, prompt splits and what the decode workgroups need)
    const int block = blockIdx.x, y = blockIdx.y, d = (y - a.ps) * (int)gridDim.x + block;
    if (y < a.ps) paged_prompt_block<TYPE, HD, RW>(a, block, gridDim.x, y, lds);
    else if (d < nd) paged_decode_block<TYPE, HD>(a, d, lds);
}

constexpr int ALONE = 82 * 1024;  // more than half a compute unit's LDS
template <int TYPE, int HD, int RW>
hipError_t launch_rows(const PagedAttnArgs &a, hipStream_t s) {
    constexpr int pro = Pro<TYPE, HD, RW>::LDS, bytes = pro > dec_lds(HD) ? pro : dec_lds(HD);
    const int x = (int)paged_tiles(a) * a.p.n_head_kv, nd = a.p.n_seq * a.ds * a.p.n_head_kv;
    const dim3 grid((unsigned)x, (unsigned)(a.ps + (nd + x - 1) / x));
    paged_prompt_kernel<TYPE, HD, RW><<<grid, 256, a.alone ? std::max(bytes, ALONE) : bytes, s>>>(a, nd);
    return hipGetLastError();
}
template <int TYPE, int HD>
hipError_t launch_one(const PagedAttnArgs &a, hipStream_t s) {
    if constexpr (pro_half(TYPE, HD))
        if (a.prows == PRO_ROWS / 2) return launch_rows<TYPE, HD, 2>(a, s);
    return launch_rows<TYPE, HD, 4>(a, s);
}
template <int TYPE>
hipError_t launch_type(const PagedAttnArgs &a, hipStream_t s) {
    switch (a.p.hd) {
    case 64: return launch_one<TYPE, 64>(a, s);
    case 80: return launch_one<TYPE, 80>(a, s);
    case 96: return launch_one<TYPE, 96>(a, s);
    case 128: return launch_one<TYPE, 128>(a, s);
    case 256: return launch_one<TYPE, 256>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_paged_prompt(const PagedAttnArgs &a, hipStream_t s) {
    switch (a.p.type) {
    case T_F32: return launch_type<T_F32>(a, s);
    case T_F16: return launch_type<T_F16>(a, s);
    case T_BF16: return launch_type<T_BF16>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace fgh
