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

// out[col] = sum over `rows` of partial[row][col].  A block owns COLS columns; its 1024 threads form 1024 / COLS rows of readers, each of which adds
// every so-manieth row in order (with 296 rows all ten or fewer loads of a thread are in flight at once); the readers' sums are then
// added in a fixed tree.  Reads come from L2, where the first kernel has just put them.  Few columns with many rows take blocks
// of eight columns, so that there are enough blocks (rows of 1000 x 1024 bf16, all of the gradient: 11.4 us with 32, 8.3 with eight).
constexpr int kSumThreads = 1024;
template <typename G, int COLS>
__global__ void __launch_bounds__(kSumThreads)
sum_partials_kernel(const float* __restrict__ partial, G* __restrict__ out, int rows, int cols)
{
    constexpr int READERS = kSumThreads / COLS;
    __shared__ float part[32][COLS];
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c = threadIdx.x % COLS, col = blockIdx.x * COLS + c;
    float v = 0.0f;
    if (col < cols) {
#pragma unroll 10
        for (int r = threadIdx.x / COLS; r < rows; r += READERS) v += partial[static_cast<size_t>(r) * cols + col];
    }
#pragma unroll
    for (int o = COLS; o < 32; o <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);  // the readers of a warp
    if (lane < COLS) part[w][lane] = v;
    __syncthreads();
    if (w == 0 && lane < COLS && col < cols) {
#pragma unroll
        for (int i = 1; i < 32; ++i) v += part[i][lane];
        out[col] = rounded<G>(v);
    }
}

template <int COLS>
int sum_partials_as(const float* partial, void* out, int dtype, int rows, int cols, cudaStream_t st)
{
    const unsigned grid = static_cast<unsigned>((cols + COLS - 1) / COLS);
    if (dtype == ASCB200_F32) ASCB200_CUDA(launch_pdl(sum_partials_kernel<float, COLS>, grid, kSumThreads, 0, st, partial, static_cast<float*>(out), rows, cols));
    else if (dtype == ASCB200_F16) ASCB200_CUDA(launch_pdl(sum_partials_kernel<__half, COLS>, grid, kSumThreads, 0, st, partial, static_cast<__half*>(out), rows, cols));
    else ASCB200_CUDA(launch_pdl(sum_partials_kernel<__nv_bfloat16, COLS>, grid, kSumThreads, 0, st, partial, static_cast<__nv_bfloat16*>(out), rows, cols));
    return ASCB200_OK;
}
inline int sum_partials(const float* partial, void* out, int dtype, int rows, int cols, cudaStream_t st)
{
    return cols < 4096 && rows > 64 ? sum_partials_as<8>(partial, out, dtype, rows, cols, st) : sum_partials_as<32>(partial, out, dtype, rows, cols, st);
}

}  // namespace
}  // namespace ascb200
