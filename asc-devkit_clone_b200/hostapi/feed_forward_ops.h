// The feed-forward operators (norm, linear layer, routing) over the C ABI, in the manner of adv_api_ops.h: tensors are device memory
// holding whole operands, calls go to the thread's stream, the first failing code is latched (GetLastError).  The typed forms cover
// packed tensors; everything else is reached through a descriptor of ascb200.h.
// Included by kernel_operator.h.
#pragma once

namespace AscendC {

inline void RmsNorm(const ascb200_rms_norm_desc& desc) { detail::Latch(ascb200_rms_norm(&desc, detail::CurrentStream()), "RmsNorm"); }
inline void RmsNormGrad(const ascb200_rms_norm_grad_desc& desc) { detail::Latch(ascb200_rms_norm_grad(&desc, detail::CurrentStream()), "RmsNormGrad"); }
inline void Linear(const ascb200_linear_desc& desc) { detail::Latch(ascb200_linear(&desc, detail::CurrentStream()), "Linear"); }
inline void LinearGrad(const ascb200_linear_grad_desc& desc) { detail::Latch(ascb200_linear_grad(&desc, detail::CurrentStream()), "LinearGrad"); }
inline void Route(const ascb200_route_desc& desc) { detail::Latch(ascb200_route(&desc, detail::CurrentStream()), "Route"); }
inline void RouteGrad(const ascb200_route_grad_desc& desc) { detail::Latch(ascb200_route_grad(&desc, detail::CurrentStream()), "RouteGrad"); }

// dst[m, k] = src / sqrt(mean(src^2) + epsilon) * gamma over rows of k = gamma.GetSize().
template <typename T>
inline void RmsNorm(const LocalTensor<T>& dst, const LocalTensor<T>& src, const LocalTensor<T>& gamma, const float epsilon)
{
    ascb200_rms_norm_desc d = {};
    d.k = static_cast<int32_t>(gamma.GetSize());
    d.m = d.k ? static_cast<int32_t>(src.GetSize() / gamma.GetSize()) : 0;
    d.dtype = d.gamma_dtype = detail::DTypeOf<T>::value;
    d.x_dev = src.GetPhyAddr(), d.gamma_dev = gamma.GetPhyAddr(), d.y_dev = dst.GetPhyAddr();
    d.eps = epsilon;
    RmsNorm(d);
}
// The same of src + residual, in 8 bits with one scale per row (dstT int8_t or fp8_e4m3fn_t); sum receives src + residual.
template <typename T, typename dstT>
inline void RmsNormQuant(const LocalTensor<dstT>& dst, const LocalTensor<float>& scale, const LocalTensor<T>& sum, const LocalTensor<T>& src,
                         const LocalTensor<T>& residual, const LocalTensor<T>& gamma, const float epsilon)
{
    static_assert(detail::DTypeOf<dstT>::value == ASCB200_S8 || detail::DTypeOf<dstT>::value == ASCB200_FP8_E4M3, "int8 or e4m3 destinations");
    ascb200_rms_norm_desc d = {};
    d.k = static_cast<int32_t>(gamma.GetSize());
    d.m = d.k ? static_cast<int32_t>(src.GetSize() / gamma.GetSize()) : 0;
    d.dtype = d.gamma_dtype = detail::DTypeOf<T>::value;
    d.x_dev = src.GetPhyAddr(), d.residual_dev = residual.GetPhyAddr(), d.gamma_dev = gamma.GetPhyAddr(), d.sum_dev = sum.GetPhyAddr();
    d.q_dev = dst.GetPhyAddr(), d.scale_dev = scale.GetPhyAddr(), d.q_dtype = detail::DTypeOf<dstT>::value, d.scale_mode = ASCB200_SCALE_PER_TOKEN;
    d.eps = epsilon;
    RmsNorm(d);
}
// dst[m, n] = act((src[m, k] * weight[n, k]^T) * channelScale[n] * tokenScale[m] + bias[n]) + residual[m, n], int8 operands; bias and residual may be
// empty tensors; n = channelScale.GetSize(), m = tokenScale.GetSize().
template <typename dstT>
inline void LinearA8W8(const LocalTensor<dstT>& dst, const LocalTensor<int8_t>& src, const LocalTensor<int8_t>& weight, const LocalTensor<float>& tokenScale,
                       const LocalTensor<float>& channelScale, const LocalTensor<float>& bias, const LocalTensor<dstT>& residual, const int32_t act)
{
    ascb200_linear_desc d = {};
    d.kind = ASCB200_KIND_S8;
    d.m = static_cast<int32_t>(tokenScale.GetSize()), d.n = static_cast<int32_t>(channelScale.GetSize());
    d.k = d.n ? static_cast<int32_t>(weight.GetSize() / channelScale.GetSize()) : 0;
    d.x_dev = src.GetPhyAddr(), d.w_dev = weight.GetPhyAddr(), d.trans_w = 1, d.act = act;
    d.tok_scale_dev = tokenScale.GetPhyAddr(), d.ch_scale_dev = channelScale.GetPhyAddr(), d.bias_dev = bias.GetPhyAddr(), d.bias_dtype = ASCB200_F32;
    d.residual_dev = residual.GetPhyAddr(), d.y_dev = dst.GetPhyAddr(), d.y_dtype = detail::DTypeOf<dstT>::value;
    Linear(d);
}

}  // namespace AscendC
