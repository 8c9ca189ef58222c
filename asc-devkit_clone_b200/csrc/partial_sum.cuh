// The second half of a reproducible sum over rows: blocks have left one row of fp32 partial sums each.
#pragma once
#include "common.cuh"

namespace ascb200 {
namespace {

template <typename G>
__device__ __forceinline__ G rounded(float v);
template <>
__device__ __forceinline__ float rounded<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half rounded<__half>(float v) { return f32_to_f16_sat(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return f32_to_bf16(v); }

// out[col] = sum over `rows` of partial[row][col]: each of a block's 32 warps adds every 32nd row of 32 columns in order, then the warps'
// sums are added in order.  Reads come from L2, where the first kernel has just put them; with 296 rows a thread has all its ten
// loads in flight at once.
constexpr int kSumWarps = 32;
template <typename G>
__global__ void __launch_bounds__(kSumWarps * 32)
sum_partials_kernel(const float* __restrict__ partial, G* __restrict__ out, int rows, int cols)
{
    __shared__ float part[kSumWarps][32];
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (col < cols) {
#pragma unroll 10
        for (int r = w; r < rows; r += kSumWarps) v += partial[static_cast<size_t>(r) * cols + col];
    }
    part[w][lane] = v;
    __syncthreads();
    if (w == 0 && col < cols) {
#pragma unroll
        for (int i = 1; i < kSumWarps; ++i) v += part[i][lane];
        out[col] = rounded<G>(v);
    }
}

inline int sum_partials(const float* partial, void* out, int dtype, int rows, int cols, cudaStream_t st)
{
    const unsigned grid = static_cast<unsigned>((cols + 31) / 32);
    if (dtype == ASCB200_F32) ASCB200_CUDA(launch_pdl(sum_partials_kernel<float>, grid, kSumWarps * 32, 0, st, partial, static_cast<float*>(out), rows, cols));
    else if (dtype == ASCB200_F16) ASCB200_CUDA(launch_pdl(sum_partials_kernel<__half>, grid, kSumWarps * 32, 0, st, partial, static_cast<__half*>(out), rows, cols));
    else ASCB200_CUDA(launch_pdl(sum_partials_kernel<__nv_bfloat16>, grid, kSumWarps * 32, 0, st, partial, static_cast<__nv_bfloat16*>(out), rows, cols));
    return ASCB200_OK;
}

}  // namespace
}  // namespace ascb200
