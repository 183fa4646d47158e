// Launches of the kernels that take activations into 8 bits and back.
#include <algorithm>

#include "keep_kernels.cuh"

namespace qgemm {

namespace {
dim3 keep_grid(const KeepArgs &a) {
    const uint32_t across = (uint32_t)(((uint64_t)a.cols + 2047) / 2048);
    return dim3(std::min<uint32_t>(a.rows, 1 << 16), across);
}
}  // namespace

hipError_t launch_checkpoint(const KeepArgs &a, hipStream_t stream) {
    auto launch = [&](auto in, auto q) { return launch_kernel(checkpoint_kernel<in.value, q.value>, keep_grid(a), dim3(256), 0, stream, a); };
    auto typed = [&](auto in) {
        return a.out_dt == QGEMM_DT_I8 ? launch(in, std::integral_constant<int, QGEMM_DT_I8>{}) : launch(in, std::integral_constant<int, QGEMM_DT_F8E4M3>{});
    };
    if (a.in_dt == QGEMM_DT_F32) return typed(std::integral_constant<int, QGEMM_DT_F32>{});
    if (a.in_dt == QGEMM_DT_BF16) return typed(std::integral_constant<int, QGEMM_DT_BF16>{});
    return typed(std::integral_constant<int, QGEMM_DT_F16>{});
}

hipError_t launch_restore(const KeepArgs &a, hipStream_t stream) {
    return a.in_dt == QGEMM_DT_I8 ? launch_kernel(restore_kernel<QGEMM_DT_I8>, keep_grid(a), dim3(256), 0, stream, a)
                                  : launch_kernel(restore_kernel<QGEMM_DT_F8E4M3>, keep_grid(a), dim3(256), 0, stream, a);
}

}  // namespace qgemm
