// The GEMM kernels with the output stage of a linear layer (kBuildLinear of gemm_kernels.cuh), in a translation unit of their own.
#include "gemm_linear.cuh"

namespace ascb200 {
namespace gemm {

template <int KIND>
static int launch_kind(bool pair, int block_n, const CUtensorMap& ta, const CUtensorMap& tb, const OutMaps& outs, const GemmParams& p, int count, cudaStream_t stream)
{
    if (pair) {
        if (!p.a_mn && !p.b_mn) return launch_gemm_pair_as<KIND, 256, kBuildLinear, true>(ta, tb, ta, tb, outs, p, count, stream);
        return launch_gemm_pair_as<KIND, 256, kBuildLinear, false>(ta, tb, ta, tb, outs, p, count, stream);
    }
    if (block_n == 256) return launch_gemm_as<KIND, 256, kBuildLinear>(ta, tb, outs, p, count, stream);
    if (block_n == 128) return launch_gemm_as<KIND, 128, kBuildLinear>(ta, tb, outs, p, count, stream);
    return launch_gemm_as<KIND, 64, kBuildLinear>(ta, tb, outs, p, count, stream);
}

int launch_linear_gemm(int kind, bool pair, int block_n, const CUtensorMap& ta, const CUtensorMap& tb, const OutMaps& outs, const GemmParams& p, int count,
                       cudaStream_t stream)
{
    return kind == KIND_I8 ? launch_kind<KIND_I8>(pair, block_n, ta, tb, outs, p, count, stream) : launch_kind<KIND_F16>(pair, block_n, ta, tb, outs, p, count, stream);
}

}  // namespace gemm
}  // namespace ascb200
