// Launches of the log probabilities' kernels.
#include <algorithm>

#include "log_prob_kernels.cuh"

namespace qgemm {

namespace {
constexpr uint32_t kMostRowGroups = 65535;            // workgroups down that share out the rows of a launch
constexpr uint32_t kMostSplits = 64;                  // lanes of the joining wave
template <class F>
auto with_type(int dt, F f) {
    if (dt == QGEMM_DT_F32) return f(std::integral_constant<int, QGEMM_DT_F32>{});
    if (dt == QGEMM_DT_BF16) return f(std::integral_constant<int, QGEMM_DT_BF16>{});
    return f(std::integral_constant<int, QGEMM_DT_F16>{});
}
}  // namespace

size_t plan_log_prob(LogProbArgs &a, int cus) {
    // (a part has one trip to memory's worth of columns for a workgroup: less gains nothing and leaves more to join)
    const uint32_t trip = kLogProbAhead * kLogProbTurn, want = (uint32_t)cus * 4 / std::max<uint32_t>(a.rows, 1), most = (a.cols + trip - 1) / trip;
    a.splits = std::max<uint32_t>(1, std::min({want, most, kMostSplits}));
    a.part = ((a.cols + a.splits - 1) / a.splits + kOctet - 1) / kOctet * kOctet;
    a.splits = (a.cols + a.part - 1) / a.part;
    return a.splits > 1 ? (size_t)a.rows * a.splits * log_prob_part(a.top) * sizeof(float) : 0;
}

hipError_t launch_log_prob(const LogProbArgs &a, hipStream_t stream) {
    const hipError_t e = with_type(a.dt, [&](auto dt) {
        return launch_kernel(a.top ? log_prob_kernel<dt.value, true> : log_prob_kernel<dt.value, false>, dim3(a.splits, std::min(a.rows, kMostRowGroups)),
                             dim3(kLogProbThreads), 0, stream, a);
    });
    if (e != hipSuccess || a.splits == 1) return e;
    return launch_kernel(log_prob_join_kernel, dim3(a.rows), dim3(256), 0, stream, a);
}

hipError_t launch_log_prob_backward(const LogProbBackwardArgs &a, hipStream_t stream) {
    // (two octets of a thread: us, 2048 x 65536 bf16 with one / two / four 115 / 92 / 93)
    const uint32_t across = std::min<uint32_t>((a.cols + 2 * kLogProbTurn - 1) / (2 * kLogProbTurn), 64);
    return with_type(a.dt, [&](auto dt) {
        return launch_kernel(log_prob_backward_kernel<dt.value>, dim3(across, std::min(a.rows, kMostRowGroups)), dim3(kLogProbThreads), 0, stream, a);
    });
}

}  // namespace qgemm
