// gemm_gate_instances.hip -- instantiates gemm_f32_sp for a gated block's projections, in one
// tile (-DMT_CFG=<n>: GateCfg), x and the weight contiguous along k or across it.
#include "gemm_configs.hpp"
#include "gemm_sp_kernel.hpp"

#ifndef MT_CFG
#error "build with -DMT_CFG=<configuration index>"
#endif

namespace mtk {
namespace {

template <int LA, int LB>
hipError_t launch_gate(const GemmParams& p, unsigned nblocks, hipStream_t s) {
    using C = GateCfg<MT_CFG>;
    hipLaunchKernelGGL((gemm_f32_sp<C::BM, C::BN, C::BN, C::WM, C::WN, LA, LB, C::WPE>),
                       dim3(nblocks), dim3((C::BM / C::WM) * (C::BN / C::WN) * 64), 0, s, p);
    return hipGetLastError();
}

}  // namespace

#define MT_CAT(a, b) a##b
#define MT_NAME(n) MT_CAT(gate_launcher_cfg, n)
GemmLaunchFn MT_NAME(MT_CFG)(int la, int lb) {
    if (lb == L_GKV) return la == L_KV ? launch_gate<L_KV, L_GKV> : launch_gate<L_MV, L_GKV>;
    return la == L_KV ? launch_gate<L_KV, L_GMV> : launch_gate<L_MV, L_GMV>;
}

}  // namespace mtk
