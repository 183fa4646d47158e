// Launches of the layer norm kernels.
#include <algorithm>

#include "norm_kernels.cuh"

namespace qgemm {

namespace {
constexpr uint32_t kMostRowGroups = 1 << 16;          // workgroups that share out the rows of a launch

template <class F>
auto with_type(int dt, F f) {
    if (dt == QGEMM_DT_F32) return f(std::integral_constant<int, QGEMM_DT_F32>{});
    if (dt == QGEMM_DT_BF16) return f(std::integral_constant<int, QGEMM_DT_BF16>{});
    return f(std::integral_constant<int, QGEMM_DT_F16>{});
}
template <class F>
auto with_any_type(int dt, F f) {
    if (dt == QGEMM_DT_I8) return f(std::integral_constant<int, QGEMM_DT_I8>{});
    if (dt == QGEMM_DT_F8E4M3) return f(std::integral_constant<int, QGEMM_DT_F8E4M3>{});
    return with_type(dt, f);
}
}  // namespace

hipError_t launch_layer_norm(const NormArgs &a, int, hipStream_t stream) {
    return with_type(a.x_dt, [&](auto dt) {
        return launch_kernel(norm_any_kernel<dt.value>, dim3(std::min(a.rows, kMostRowGroups)), dim3(256), 0, stream, a);
    });
}

uint32_t norm_backward_groups(const NormBackwardArgs &a, int) {
    if (a.rows == 0 || (!a.dweight && !a.dbias)) return 0;
    return std::min<uint32_t>((a.rows + 15) / 16, 64);
}

hipError_t launch_layer_norm_backward(const NormBackwardArgs &a, int, hipStream_t stream) {
    hipError_t e = hipSuccess;
    if (a.rows) {
        e = with_type(a.dy_dt, [&](auto dy) {
            return with_any_type(a.x_dt, [&](auto x) {
                hipError_t f = launch_kernel(norm_backward_any_kernel<dy.value, x.value>, dim3(std::min(a.rows, kMostRowGroups)), dim3(256), 0, stream, a);
                if (f == hipSuccess && a.groups)
                    f = launch_kernel(norm_column_sums_kernel<dy.value, x.value>, dim3((a.cols + 127) / 128, a.groups), dim3(256), 0, stream, a);
                return f;
            });
        });
    }
    if (e == hipSuccess && (a.dweight || a.dbias))
        e = launch_kernel(norm_parameter_sums_kernel, dim3((a.cols + 63) / 64, 2), dim3(256), 0, stream, a);
    return e;
}

}  // namespace qgemm
