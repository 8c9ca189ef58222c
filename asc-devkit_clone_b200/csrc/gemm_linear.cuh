// Launch of the linear build of the GEMM kernels (instances: gemm_linear.cu).
#pragma once
#include "gemm_kernels.cuh"

namespace ascb200 {
namespace gemm {
// kind: KIND_F16 (fp16 and bf16) or KIND_I8; `count`: CTA pairs, or CTAs.
int launch_linear_gemm(int kind, bool pair, int block_n, const CUtensorMap& ta, const CUtensorMap& tb, const OutMaps& outs, const GemmParams& p, int count,
                       cudaStream_t stream);
}  // namespace gemm
}  // namespace ascb200
