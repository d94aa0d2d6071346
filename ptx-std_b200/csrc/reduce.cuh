// Launch attributes of programmatic dependent launch, and the second step of column sums: adding
// the partial rows that a first kernel's blocks wrote.
#pragma once

#include "common.cuh"
#include "mx_block.cuh"

namespace ptxstd {

// One-dimensional launch with programmatic stream serialisation; `attr` has room for one.
inline void set_pdl(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, uint32_t grid,
                    uint32_t block, cudaStream_t stream) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
}

// Sums over the P rows of partial [P][sums * cols]: o0 takes the first `cols` columns' sums; the
// second `cols` columns' sums, times scale and a bf16 factor per column (null: 1), go to o1 and o2
// (either may be null). A block covers 32 columns with GROUPS warps, each adding every GROUPS-th row;
// the warps' sums are added in order.
struct Reduce {
    const float* partial;
    float *o0, *o1, *o2;
    const uint16_t *f1, *f2;
    float scale;
    uint32_t P, sums, cols;
};
template <uint32_t GROUPS>
static __global__ void __launch_bounds__(32 * GROUPS)
    reduce_kernel(const __grid_constant__ Reduce p) {
    __shared__ float part[GROUPS][32];
    const uint32_t lane = lane_id(), g = threadIdx.x >> 5;
    const uint32_t c = blockIdx.x * 32 + lane, width = p.sums * p.cols;
    pdl_launch_dependents();
    pdl_wait();
    float s = 0.0f;
    if (c < width) {
#pragma unroll 8
        for (uint32_t r = g; r < p.P; r += GROUPS)
            s += p.partial[static_cast<size_t>(r) * width + c];
    }
    part[g][lane] = s;
    __syncthreads();
    if (g || c >= width) return;
#pragma unroll
    for (uint32_t k = 1; k < GROUPS; ++k) s += part[k][lane];
    if (c < p.cols) {
        p.o0[c] = s;
        return;
    }
    const uint32_t i = c - p.cols;
    s *= p.scale;
    if (p.o1) p.o1[i] = p.f1 ? s * data_types::bf16_lo(p.f1[i]) : s;
    if (p.o2) p.o2[i] = p.f2 ? s * data_types::bf16_lo(p.f2[i]) : s;
}

inline int launch_reduce(const Reduce& r, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    const uint32_t blocks = (r.sums * r.cols + 31) / 32;
    // Many rows and few columns (the norms: 296 rows, 8192 columns) want more warps per column;
    // fewer rows and more columns (an activation's: 64 rows, 16384 columns) do not: 70.9 -> 67.8 us
    // for rmsnorm_residual_backward of 8192 x 4096 with 32 groups, but 83.1 -> 85.7 us for
    // act_backward_mx of 4096 x 16384.
    const bool tall = r.P >= 128;
    set_pdl(cfg, attr, blocks, 32 * (tall ? 32 : 8), stream);
    const cudaError_t e = tall ? cudaLaunchKernelEx(&cfg, reduce_kernel<32>, r)
                               : cudaLaunchKernelEx(&cfg, reduce_kernel<8>, r);
    return e == cudaSuccess ? launch_status() : PTXSTD_ECUDA;
}

}  // namespace ptxstd
