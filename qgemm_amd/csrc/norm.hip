// Launches of the layer norm kernels.
#include <algorithm>

#include "norm_kernels.cuh"

namespace qgemm {

namespace {
constexpr uint32_t kMostRowGroups = 1 << 16;          // workgroups that share out the rows of a launch
constexpr size_t kMostPartials = (size_t)128 << 20;   // partial sums that a stream's own workspace block holds (registers' forms need 32 MiB at the most)
constexpr uint32_t kMostColumnGroups = 1 << 16;       // workgroups across of the parameters' sums: a launch has fewer than 2^32 threads across

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

// GROUP threads of P octets for a row
struct NormShape {
    int group, p;
};
template <class F>
hipError_t with_shape(NormShape s, F f) {
#define SHAPE(G, P) if (s.group == G && s.p == P) return f(std::integral_constant<int, G>{}, std::integral_constant<int, P>{})
    SHAPE(16, 1);
    SHAPE(32, 1);
    SHAPE(64, 1);
    SHAPE(64, 2);
    SHAPE(64, 4);
    SHAPE(256, 1);
    SHAPE(256, 2);
    SHAPE(256, 4);
    SHAPE(512, 2);
    SHAPE(512, 4);
#undef SHAPE
    return hipErrorInvalidValue;
}
// Up to kFewRows rows, which one round of workgroups holds, more threads for a row end it sooner; beyond it fewer threads of more octets leave
// room for more rows (us, 6144 x 7168 bf16 kept: 256 threads of four 42.5, 512 of two 50.0, on other buffers each time 54.5 and 58.0, not kept 35.0
// and 43.8; 128 x 8192 5.4 and 4.9; 16384 x 2048: 64 of four 30.6, 256 of one 39.4, 1 x 2048 4.1 and 3.1).
constexpr uint32_t kFewRows = 1024, kMostCols = 16384;
bool in_registers(uint32_t cols) { return cols >= kOctet && cols <= kMostCols; }
NormShape norm_shape(uint32_t rows, uint32_t cols) {
    const uint32_t octets = (cols + 7) / 8;
    if (octets <= 16) return {16, 1};
    if (octets <= 32) return {32, 1};
    if (octets <= 64) return {64, 1};
    if (octets <= 128) return {64, 2};
    if (octets <= 256) return rows <= kFewRows ? NormShape{256, 1} : NormShape{64, 4};
    if (octets <= 512) return {256, 2};
    if (octets <= 1024) return rows <= kFewRows ? NormShape{512, 2} : NormShape{256, 4};
    return {512, 4};
}

hipError_t launch_layer_norm(const NormArgs &a, int, hipStream_t stream) {
    const bool same = !a.weight || a.param_dt == a.x_dt;
    if (in_registers(a.cols) && (same || a.param_dt == QGEMM_DT_F32)) {
        return with_shape(norm_shape(a.rows, a.cols), [&](auto group, auto p) {
            return with_type(a.x_dt, [&](auto dt) {
                constexpr int threads = group.value < 256 ? 256 : group.value;
                constexpr uint32_t rows = threads / group.value, most = (1u << 31) / threads;
                const dim3 grid(std::min((a.rows + rows - 1) / rows, most));
                auto go = [&](auto same_type) {
                    // (one octet a lane: there is nothing to save; two: by the number of rows; four: many rows)
                    auto kernel = [&](auto ahead) {
                        return a.cols % kOctet ? norm_rows_kernel<dt.value, group.value, p.value, same_type.value, ahead.value, ROW_RAGGED>
                                               : norm_rows_kernel<dt.value, group.value, p.value, same_type.value, ahead.value, ROW_WHOLE>;
                    };
                    if constexpr (p.value == 1) return launch_kernel(kernel(std::true_type{}), grid, dim3(threads), 0, stream, a);
                    else if constexpr (p.value == 2 && group.value > 64)
                        return launch_kernel(a.rows <= kFewRows ? kernel(std::true_type{}) : kernel(std::false_type{}), grid, dim3(threads), 0, stream, a);
                    else return launch_kernel(kernel(std::false_type{}), grid, dim3(threads), 0, stream, a);
                };
                if constexpr (dt.value != QGEMM_DT_F32)
                    if (!same) return go(std::false_type{});
                return go(std::true_type{});
            });
        });
    }
    return with_type(a.x_dt, [&](auto dt) {
        return launch_kernel(norm_any_kernel<dt.value>, dim3(std::min(a.rows, kMostRowGroups)), dim3(256), 0, stream, a);
    });
}

namespace {
template <class F>
hipError_t with_backward_shape(NormShape s, F f) {
#define SHAPE(G, P) if (s.group == G && s.p == P) return f(std::integral_constant<int, G>{}, std::integral_constant<int, P>{})
    SHAPE(16, 1);
    SHAPE(32, 1);
    SHAPE(64, 1);
    SHAPE(64, 2);
    SHAPE(256, 1);
    SHAPE(512, 1);
    SHAPE(512, 2);
    SHAPE(512, 4);
#undef SHAPE
    return hipErrorInvalidValue;
}
NormShape backward_shape(uint32_t cols) {
    const uint32_t octets = (cols + 7) / 8;
    if (octets <= 16) return {16, 1};
    if (octets <= 32) return {32, 1};
    if (octets <= 64) return {64, 1};
    if (octets <= 128) return {64, 2};
    if (octets <= 256) return {256, 1};
    if (octets <= 512) return {512, 1};
    if (octets <= 1024) return {512, 2};
    return {512, 4};
}
// Workgroups: g of them write g rows of column sums, and each goes over units / g rows: the sum of both is least at g ~ sqrt(units).  Twenty
// shapes of 64 - 131072 rows and 128 - 14336 columns with every power of two are fastest at 8 sqrt(units), or a power of two beside it within 8 % (us,
// 4096 columns bf16: 64 rows in 16 / 64 / 128 workgroups 9.1 / 7.2 / 7.1, 1024 in 128 / 256 / 512 16.8 / 15.5 / 18.6, 8192 in 256 / 512 / 1024
// 47.7 / 43.4 / 49.3), up to what the CUs hold at a time.
uint32_t row_workgroups(const NormBackwardArgs &a, int cus) {
    const NormShape s = backward_shape(a.cols);
    const uint32_t rows = s.group < 256 ? 256 / s.group : 1, units = (a.rows + rows - 1) / rows;
    const uint32_t most = (uint32_t)cus * (s.group < 512 ? 4 : s.p == 1 ? 2 : 1);
    uint32_t g = 1;
    while (g < most && (uint64_t)g * g * 4 <= (uint64_t)units * 64) g *= 2;            // the power of two below 8 sqrt(units)
    return std::min({g, most, units});
}
}  // namespace

uint32_t norm_backward_groups(const NormBackwardArgs &a, int cus) {
    if (a.rows == 0 || (!a.dweight && !a.dbias)) return 0;
    if (in_registers(a.cols)) return row_workgroups(a, cus);
    const size_t room = std::max<size_t>(kMostPartials / norm_partial_bytes(1, a.cols), 1);
    return (uint32_t)std::min<size_t>({(a.rows + 15) / 16, 64, room});
}

hipError_t launch_layer_norm_backward(const NormBackwardArgs &a, int cus, hipStream_t stream) {
    hipError_t e = hipSuccess;
    if (a.rows) {
        e = with_type(a.dy_dt, [&](auto dy) {
            return with_any_type(a.x_dt, [&](auto x) {
                if (in_registers(a.cols))
                    return with_backward_shape(backward_shape(a.cols), [&](auto group, auto p) {
                        auto kernel = a.cols % kOctet ? norm_backward_rows_kernel<dy.value, x.value, group.value, p.value, ROW_RAGGED>
                                                      : norm_backward_rows_kernel<dy.value, x.value, group.value, p.value, ROW_WHOLE>;
                        if constexpr ((x.value == QGEMM_DT_I8 || x.value == QGEMM_DT_F8E4M3) && group.value > 16)      // (two blocks or more)
                            if (a.cols % kScaleBlock - 1 < kOctet - 1)
                                kernel = norm_backward_rows_kernel<dy.value, x.value, group.value, p.value, ROW_RAGGED, true>;
                        return launch_kernel(kernel, dim3(row_workgroups(a, cus)), dim3(group.value < 256 ? 256 : group.value), 0, stream, a);
                    });
                hipError_t f = launch_kernel(norm_backward_any_kernel<dy.value, x.value>, dim3(std::min(a.rows, kMostRowGroups)), dim3(256), 0, stream, a);
                if (f == hipSuccess && a.groups)
                    f = launch_kernel(norm_column_sums_kernel<dy.value, x.value>, dim3((a.cols + 127) / 128, a.groups), dim3(256), 0, stream, a);
                return f;
            });
        });
    }
    if (e == hipSuccess && (a.dweight || a.dbias)) {
        const uint32_t groups = (a.cols + 31) / 32, across = std::min(groups, kMostColumnGroups);
        e = launch_kernel(norm_parameter_sums_kernel, dim3(across, (groups + across - 1) / across * 2), dim3(512), 0, stream, a);
    }
    return e;
}

}  // namespace qgemm
