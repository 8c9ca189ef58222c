// The host entry of the tensor-core GEMM, for the operators that are built on it.
#pragma once
#include "common.cuh"

namespace ascb200 {
namespace gemm {

// Device resources of one call when they do not come from the per-device state of ascb200_init.
struct FixedResources {
    uint32_t* status_dev;
    uint8_t* scale_scratch_dev;
    size_t scale_scratch_bytes;
    int sm_count;
    long long l2_bytes;  // 0: unknown, tiles keep the plain order
};

constexpr int kFirstOfTwo = 1, kSecondOfTwo = 2;

// What a linear layer adds to the product's output stage: y = act(z) + residual, z = product (scaled, for int8) + bias.
// Its z, when wanted, is the descriptor's second output.
struct LinearArgs {
    const void* bias;      // [n] or nullptr
    int bias_f32;          // fp32, else the type of y
    int act;               // ASCB200_ACT_*
    const void* residual;  // [m][ld_residual] of y's type, or nullptr
    long long ld_residual;
    int order = 0;  // kFirstOfTwo, kSecondOfTwo: this product and the next / the one before do not depend on each other and may overlap
};

int run_gemm(const ascb200_gemm_desc* d, const int64_t* group_counts, int groups, cudaStream_t stream, const FixedResources* fixed = nullptr,
             const LinearArgs* linear = nullptr);

}  // namespace gemm
}  // namespace ascb200
