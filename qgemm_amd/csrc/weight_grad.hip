// Launches of the weight gradient kernels.
#include <algorithm>

#include "weight_grad.cuh"

namespace qgemm {

namespace {
template <class C>
hipError_t launch(const WeightGradArgs &a, hipStream_t stream) {
    static const hipError_t raised = hipFuncSetAttribute((const void *)weight_grad_kernel<C>, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
    if (raised != hipSuccess) return raised;
    const uint32_t tiles_n = (a.n + C::BN - 1) / C::BN, tiles_k = (a.cols + C::BK - 1) / C::BK;
    return launch_kernel(weight_grad_kernel<C>, dim3(tiles_n * tiles_k), dim3(C::THREADS), C::LDS, stream, a, make_tile_map(tiles_n, tiles_k, 8));
}
}  // namespace

size_t weight_grad_room(const WeightGradArgs &, int) { return 0; }

hipError_t launch_weight_grad(const WeightGradArgs &a, int, hipStream_t stream) {
    auto typed = [&](auto dy) {
        return a.q_dt == QGEMM_DT_I8 ? launch<GradCfg<dy.value, QGEMM_DT_I8, 128, 128, 2, 2>>(a, stream)
                                     : launch<GradCfg<dy.value, QGEMM_DT_F8E4M3, 128, 128, 2, 2>>(a, stream);
    };
    return a.dy_dt == QGEMM_DT_BF16 ? typed(std::integral_constant<int, QGEMM_DT_BF16>{}) : typed(std::integral_constant<int, QGEMM_DT_F16>{});
}

}  // namespace qgemm
