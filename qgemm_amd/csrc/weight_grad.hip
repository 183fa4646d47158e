// Launches of the weight gradient kernels.
#include <algorithm>

#include "weight_grad.cuh"

namespace qgemm {

namespace {
constexpr size_t kGradMostRoom = (size_t)128 << 20;       // partial sums that a stream's own workspace block holds

template <class C>
hipError_t launch(const WeightGradArgs &a, hipStream_t stream) {
    static const hipError_t raised = hipFuncSetAttribute((const void *)weight_grad_kernel<C>, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
    if (raised != hipSuccess) return raised;
    const uint32_t tiles_n = (a.n + C::BN - 1) / C::BN, tiles_k = (a.cols + C::BK - 1) / C::BK;
    return launch_kernel(weight_grad_kernel<C>, dim3(tiles_n * tiles_k, a.slices), dim3(C::THREADS), C::LDS, stream, a, make_tile_map(tiles_n, tiles_k, 8));
}
template <int DY, int Q>
hipError_t launch_tile(const WeightGradArgs &a, hipStream_t stream) {
    switch (a.tile) {
        case TILE_256x256: return launch<GradCfg<DY, Q, 256, 256, 2, 4>>(a, stream);
        case TILE_256x128: return launch<GradCfg<DY, Q, 256, 128, 4, 2>>(a, stream);
        default: return launch<GradCfg<DY, Q, 128, 128, 2, 2>>(a, stream);
    }
}
}  // namespace

// Rounds of workgroups times steps of 32 rows, and for slices of the rows the joining of their sums.  The times are measured (every tile with every
// number of slices on 16 shapes of 64 - 32768 rows: the choice is the fastest or within 4 % of it on 13, within 11 % on all).
size_t plan_weight_grad(WeightGradArgs &a, int cus) {
    // a workgroup's rows and columns, workgroups of a CU, and us for a step where half of the CUs or fewer are at work and where all are
    struct Tile {
        uint32_t bn, bk, per_cu;
        double alone, full;
    };
    static constexpr Tile tiles[GRAD_TILES] = {{128, 128, 2, 0.39, 0.63}, {256, 128, 1, 0.51, 0.58}, {256, 256, 1, 0.82, 0.95}};
    // (a step's rows within 32 bits of its first, and eight elements in a row)
    a.plain = a.n >= 8 && a.cols >= 8 && a.lddy < ((uint64_t)1 << 24) && a.ldq < ((uint64_t)1 << 24);
    const uint32_t steps = (a.rows + kGradStep - 1) / kGradStep;
    const size_t plane = grad_plane(a.n, a.cols) * sizeof(float);
    double least = 1e300;
    for (int t = 0; t < GRAD_TILES; ++t) {
        const uint64_t n = (uint64_t)((a.n + tiles[t].bn - 1) / tiles[t].bn) * ((a.cols + tiles[t].bk - 1) / tiles[t].bk);
        static constexpr uint32_t parts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
        for (uint32_t want : parts) {
            const uint32_t slice = std::max<uint32_t>(1, (steps + want - 1) / want), slices = std::max<uint32_t>(1, (steps + slice - 1) / slice);
            if (want > 1 && (slice < 4 || slices * plane > kGradMostRoom)) break;
            const uint64_t wgs = n * slices, at_once = (uint64_t)cus * tiles[t].per_cu, rounds = (wgs + at_once - 1) / at_once;
            const double step = wgs * 2 <= (uint64_t)cus ? tiles[t].alone : wgs <= (uint64_t)cus ? std::min(tiles[t].full, tiles[t].alone * 1.1) : tiles[t].full;
            // (a workgroup's beginning and end; the joining launch, and the slices' sums at the rate at which they are written and read)
            const double us = rounds * (slice * step + 4) + (slices > 1 ? 2.5 + slices * (double)a.n * a.cols * 8 / 4.2e6 : 0);
            if (us < least) {
                least = us;
                a.tile = t;
                a.slices = slices;
                a.slice = slice * kGradStep;
            }
        }
    }
    return a.slices > 1 ? a.slices * plane : 0;
}

hipError_t launch_weight_grad(const WeightGradArgs &a, hipStream_t stream) {
    auto typed = [&](auto dy) {
        return a.q_dt == QGEMM_DT_I8 ? launch_tile<dy.value, QGEMM_DT_I8>(a, stream) : launch_tile<dy.value, QGEMM_DT_F8E4M3>(a, stream);
    };
    const hipError_t e = a.dy_dt == QGEMM_DT_BF16 ? typed(std::integral_constant<int, QGEMM_DT_BF16>{}) : typed(std::integral_constant<int, QGEMM_DT_F16>{});
    if (e != hipSuccess || a.slices == 1) return e;
    return launch_kernel(a.dw_dt == QGEMM_DT_F32 ? weight_grad_join_kernel<QGEMM_DT_F32>
                         : a.dw_dt == QGEMM_DT_BF16 ? weight_grad_join_kernel<QGEMM_DT_BF16> : weight_grad_join_kernel<QGEMM_DT_F16>,
                         dim3((a.cols + 1023) / 1024, std::min<uint32_t>(a.n, 32768)), dim3(256), 0, stream, a, a.slices);
}

}  // namespace qgemm
