// Launches of the root-mean-square norm's kernels.
#include <algorithm>

#include "rms_kernels.cuh"

namespace qgemm {

namespace {
constexpr uint32_t kMostRowGroups = 1 << 16;          // workgroups that share out the rows of a launch
constexpr size_t kMostPartials = (size_t)128 << 20;   // partial sums that a stream's own workspace block holds
constexpr uint32_t kMostColumnGroups = 1 << 16;       // workgroups across of the weight's sums: a launch has fewer than 2^32 threads across
constexpr uint32_t kMostCols = 16384;

// rows that the registers of a workgroup hold
bool in_registers(uint32_t cols) { return cols >= kOctet && cols <= kMostCols; }
// GROUP threads of P octets for a row
struct Shape {
    int group, p;
};
// The same for few rows and many, so that a row's numbers do not depend on how many others there are.  (us, 512 threads of two octets / 256 of four: bf16 with
// residual and int8 codes 6144 x 7168 82 / 82, 2048 x 7168 29 / 32, 512 x 7168 9.9 / 11.7, 16384 x 4608 143 / 146; without either 6144 x 7168 39 / 38,
// 16384 x 4608 80 / 75, 512 x 7168 6.0 / 7.1.)
Shape forward_shape(uint32_t cols) {
    const uint32_t octets = (cols + 7) / 8;
    if (octets <= 16) return {16, 1};
    if (octets <= 32) return {32, 1};
    if (octets <= 64) return {64, 1};
    if (octets <= 128) return {64, 2};
    if (octets <= 256) return {256, 1};
    if (octets <= 512) return {256, 2};
    if (octets <= 1024) return {512, 2};
    return {512, 4};
}
Shape backward_shape(uint32_t cols) {
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
template <class F>
hipError_t with_shape(Shape s, F f) {
#define SHAPE(G, P) if (s.group == G && s.p == P) return f(std::integral_constant<int, G>{}, std::integral_constant<int, P>{})
    SHAPE(16, 1);
    SHAPE(32, 1);
    SHAPE(64, 1);
    SHAPE(64, 2);
    SHAPE(256, 1);
    SHAPE(256, 2);
    SHAPE(512, 2);
    SHAPE(512, 4);
#undef SHAPE
    return hipErrorInvalidValue;
}
template <class F>
hipError_t with_backward_shape(Shape s, F f) {
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
template <class F>
auto with_type(int dt, F f) {
    if (dt == QGEMM_DT_F32) return f(std::integral_constant<int, QGEMM_DT_F32>{});
    if (dt == QGEMM_DT_BF16) return f(std::integral_constant<int, QGEMM_DT_BF16>{});
    return f(std::integral_constant<int, QGEMM_DT_F16>{});
}
}  // namespace

hipError_t launch_rms_norm(const RmsArgs &a, hipStream_t stream) {
    if (in_registers(a.cols) && (!a.residual || a.r_dt == a.x_dt || a.r_dt == QGEMM_DT_F32))
        return with_shape(forward_shape(a.cols), [&](auto group, auto p) {
            return with_type(a.x_dt, [&](auto dt) {
                constexpr int threads = group.value < 256 ? 256 : group.value;
                constexpr uint32_t rows = threads / group.value, most = (1u << 31) / threads;
                const dim3 grid(std::min((a.rows + rows - 1) / rows, most));
                auto go = [&](auto res) {
                    return launch_kernel(a.cols % kOctet ? rms_rows_kernel<dt.value, res.value, group.value, p.value, ROW_RAGGED>
                                                         : rms_rows_kernel<dt.value, res.value, group.value, p.value, ROW_WHOLE>, grid, dim3(threads), 0, stream, a);
                };
                if (!a.residual) return go(std::integral_constant<int, -1>{});
                if constexpr (dt.value != QGEMM_DT_F32)
                    if (a.r_dt == QGEMM_DT_F32) return go(std::integral_constant<int, QGEMM_DT_F32>{});
                return go(dt);
            });
        });
    return launch_kernel(rms_any_kernel, dim3(std::min(a.rows, kMostRowGroups)), dim3(256), 0, stream, a);
}

size_t rms_partial_bytes(uint32_t groups, uint32_t cols) { return (size_t)groups * norm_partial_cols(cols) * sizeof(float); }

namespace {
// h and dh of one type, dy's or fp32
bool backward_in_registers(const RmsBackwardArgs &a) {
    return in_registers(a.cols) && (a.h_dt == a.dy_dt || a.h_dt == QGEMM_DT_F32) && (!a.dh || a.dh_dt == a.h_dt);
}
// g workgroups go over units / g rows each, one of them in flight, and leave g rows of sums for the second launch: the power of two from 8 sqrt(units) on, as far as
// the CUs hold them at a time (us, 3001 columns fp16 in 128 / 256 / 512 / 1024 workgroups: 500 rows 9.8 / 8.6 / 9.7 / 9.7, 1999 22 / 14.9 / 13.7 / 15.1; 2000 x 2056
// bf16 19 / 12.9 / 11.7 / 13.5, 8192 x 4096 65 / 40.6 / 38.5 / 39.6; 64 rows in 64 7.1, in 128 7.6.  256 threads of two octets are 1 - 2 us behind throughout.)
uint32_t row_workgroups(const RmsBackwardArgs &a, int cus) {
    const Shape s = backward_shape(a.cols);
    const uint32_t rows = s.group < 256 ? 256 / s.group : 1, units = (a.rows + rows - 1) / rows;
    const uint32_t most = (uint32_t)cus * (s.group < 512 ? 4 : s.p == 1 ? 2 : 1);
    uint32_t g = 1;
    while (g < most && (uint64_t)g * g < (uint64_t)units * 64) g *= 2;
    return std::min({g, most, units});
}
}  // namespace

uint32_t rms_backward_groups(const RmsBackwardArgs &a, int cus) {
    if (a.rows == 0 || !a.dweight) return 0;
    if (backward_in_registers(a)) return row_workgroups(a, cus);
    const size_t room = std::max<size_t>(kMostPartials / rms_partial_bytes(1, a.cols), 1);
    return (uint32_t)std::min<size_t>({(a.rows + 15) / 16, 64, room});
}

hipError_t launch_rms_norm_backward(const RmsBackwardArgs &a, int cus, hipStream_t stream) {
    hipError_t e = hipSuccess;
    if (a.rows && backward_in_registers(a)) {
        e = with_backward_shape(backward_shape(a.cols), [&](auto group, auto p) {
            return with_type(a.dy_dt, [&](auto dy) {
                auto go = [&](auto stream_type) {
                    auto kernel = [&](auto dh) {
                        return launch_kernel(a.cols % kOctet ? rms_backward_rows_kernel<dy.value, stream_type.value, dh.value, group.value, p.value, ROW_RAGGED>
                                                             : rms_backward_rows_kernel<dy.value, stream_type.value, dh.value, group.value, p.value, ROW_WHOLE>,
                                             dim3(row_workgroups(a, cus)), dim3(group.value < 256 ? 256 : group.value), 0, stream, a);
                    };
                    return a.dh ? kernel(std::true_type{}) : kernel(std::false_type{});
                };
                if constexpr (dy.value != QGEMM_DT_F32)
                    if (a.h_dt == QGEMM_DT_F32) return go(std::integral_constant<int, QGEMM_DT_F32>{});
                return go(dy);
            });
        });
    } else if (a.rows) {
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
