// Launches of the root-mean-square norm's kernels.
#include <algorithm>

#include "rms_kernels.cuh"

namespace qgemm {

namespace {
constexpr uint32_t kMostRowGroups = 1 << 16;          // workgroups that share out the rows of a launch
constexpr size_t kMostPartials = (size_t)128 << 20;   // partial sums that a stream's own workspace block holds
constexpr uint32_t kMostColumnGroups = 1 << 16;       // workgroups across of the weight's sums: a launch has fewer than 2^32 threads across
}  // namespace

hipError_t launch_rms_norm(const RmsArgs &a, int, hipStream_t stream) {
    return launch_kernel(rms_any_kernel, dim3(std::min(a.rows, kMostRowGroups)), dim3(256), 0, stream, a);
}

size_t rms_partial_bytes(uint32_t groups, uint32_t cols) { return (size_t)groups * norm_partial_cols(cols) * sizeof(float); }

uint32_t rms_backward_groups(const RmsBackwardArgs &a, int) {
    if (a.rows == 0 || !a.dweight) return 0;
    const size_t room = std::max<size_t>(kMostPartials / rms_partial_bytes(1, a.cols), 1);
    return (uint32_t)std::min<size_t>({(a.rows + 15) / 16, 64, room});
}

hipError_t launch_rms_norm_backward(const RmsBackwardArgs &a, int, hipStream_t stream) {
    hipError_t e = hipSuccess;
    if (a.rows) {
        e = launch_kernel(rms_backward_any_kernel, dim3(std::min(a.rows, kMostRowGroups)), dim3(256), 0, stream, a);
        if (e == hipSuccess && a.groups) e = launch_kernel(rms_column_sums_kernel, dim3((a.cols + 127) / 128, a.groups), dim3(256), 0, stream, a);
    }
    if (e == hipSuccess && a.dweight) {
        const uint32_t groups = (a.cols + 31) / 32, across = std::min(groups, kMostColumnGroups);
        e = launch_kernel(rms_parameter_sums_kernel, dim3(across, (groups + across - 1) / across), dim3(512), 0, stream, a);
    }
    return e;
}

}  // namespace qgemm
