// Launches of the adapters' kernels.
#include <algorithm>

#include "adapter_kernels.cuh"

namespace qgemm {

namespace {
constexpr size_t kMostRoom = (size_t)128 << 20;       // partial sums that a stream's own workspace block holds

template <class F>
auto with_dt(int dt, F f) {
    return dt == QGEMM_DT_BF16 ? f(std::integral_constant<int, QGEMM_DT_BF16>{}) : f(std::integral_constant<int, QGEMM_DT_F16>{});
}
template <class F>
auto with_ranks(uint32_t rank, F f) {
    if (rank <= 16) return f(std::integral_constant<int, 1>{});
    if (rank <= 32) return f(std::integral_constant<int, 2>{});
    if (rank <= 64) return f(std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, 8>{});
}
uint32_t column_tiles(uint32_t cols) { return (cols + 255) / 256; }
}  // namespace

hipError_t launch_group_rows(const void *ids, int id_bytes, const RowGroups &g, hipStream_t stream) {
    return launch_kernel(group_rows_kernel, dim3(g.adapters + 1), dim3(1024), 0, stream, ids, id_bytes, g);
}

uint32_t plan_shrink(const ShrinkArgs &a, int cus) {
    const uint32_t want = std::max<uint32_t>(1, (uint32_t)cus * 2 / std::max<uint32_t>(a.g.slot_count, 1)), most = std::max<uint32_t>(1, a.cols / 512);
    return std::min({want, most, 16u});
}

hipError_t launch_shrink(const ShrinkArgs &a, hipStream_t stream) {
    return with_dt(a.dt, [&](auto dt) {
        return with_ranks(a.rank, [&](auto rt) {
            return launch_kernel(adapter_shrink_kernel<dt.value, rt.value>, dim3(a.g.slot_count, a.u.planes), dim3(256), 0, stream, a);
        });
    });
}

hipError_t launch_expand(const ExpandArgs &a, hipStream_t stream) {
    const dim3 grid(a.g.slot_count, column_tiles(a.cols));
    return with_dt(a.dt, [&](auto dt) {
        auto typed = [&](auto y) {
            return launch_kernel(a.rank <= 16 ? adapter_expand_kernel<dt.value, y.value, true> : adapter_expand_kernel<dt.value, y.value, false>, grid, dim3(256),
                                 0, stream, a);
        };
        if (a.y_dt == QGEMM_DT_F32) return typed(std::integral_constant<int, QGEMM_DT_F32>{});
        if (a.y_dt == QGEMM_DT_BF16) return typed(std::integral_constant<int, QGEMM_DT_BF16>{});
        return typed(std::integral_constant<int, QGEMM_DT_F16>{});
    });
}

size_t plan_adapter_grad(AdapterGradArgs &a, int cus) {
    const size_t plane = (size_t)a.rank * adapter_plane_cols(a.cols) * sizeof(float);
    auto room = [&] { return (size_t)a.chunk * kSlotRows >= a.g.rows ? 0 : 2 * ((size_t)a.g.slot_count / a.chunk + 1) * plane; };
    a.chunk = 4;
    while (room() && (room() > kMostRoom || (uint64_t)a.g.rows / kSlotRows / a.chunk * column_tiles(a.cols) > (uint64_t)cus * 4)) a.chunk *= 2;
    return room();
}

hipError_t launch_adapter_grad(const AdapterGradArgs &a, hipStream_t stream) {
    hipError_t e = hipSuccess;
    if (a.g.rows)
        e = with_dt(a.dt, [&](auto dt) {
            return with_ranks(a.rank, [&](auto rt) {
                return launch_kernel(a.dw_dt == QGEMM_DT_F32 ? adapter_grad_kernel<dt.value, rt.value, 3> : adapter_grad_kernel<dt.value, rt.value, 2>,
                                     dim3(a.g.slot_count, column_tiles(a.cols)), dim3(256), 0, stream, a);
            });
        });
    if (e != hipSuccess) return e;
    return launch_kernel(adapter_grad_join_kernel, dim3(a.g.adapters * a.rank, std::min<uint32_t>((a.cols + 2047) / 2048, 64)), dim3(256), 0, stream, a);
}

}  // namespace qgemm
