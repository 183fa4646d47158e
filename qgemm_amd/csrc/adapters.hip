// Launches of the adapters' kernels.
#include <algorithm>

#include "adapter_kernels.cuh"

namespace qgemm {

namespace {
constexpr size_t kMostRoom = (size_t)128 << 20;       // the gradients' partial sums (sums over the rank lie in front of them: together they may pass a stream's own workspace block)

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
// Slots that there are likely to be, by which work is shared out.  Up to 1024 rows may be a decoding step whose requests all have adapters of their own; more are prompts, and of
// the adapters that there is room for most then have no row.  (Rank 16, bf16, us of shrink + expand by the slots that there could be / by those of prompts: 512 rows of 500
// adapters, 4096 x 4096 14 + 20 / 20 + 30; 1024 of 1000, 2048 x 8192 16 + 85 / 25 + 95; but 8192 rows of 32 prompts among 1000 adapters, 4096 x 4096 45 + 138 / 27 + 75.)
uint32_t likely_slots(const RowGroups &g) {
    const uint32_t whole = g.rows / kSlotRows, groups = g.rows <= 1024 ? g.rows : std::max<uint32_t>(64, whole);
    return std::max<uint32_t>(1, std::min(g.slot_count, whole + std::min(g.adapters + 1, groups)));
}
uint32_t column_tiles(uint32_t cols) { return (cols + 255) / 256; }
}  // namespace

hipError_t launch_group_rows(const void *ids, int id_bytes, const RowGroups &g, hipStream_t stream) {
    auto launch = [&](auto waves, auto turns) {
        return launch_kernel(id_bytes == 8 ? group_rows_kernel<8, waves.value, turns.value> : group_rows_kernel<4, waves.value, turns.value>, dim3(g.adapters + 1),
                             dim3(64 * waves.value), 0, stream, ids, g);
    };
    if (g.rows <= 256) return launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
    if (g.rows <= 2048) return launch(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
    return launch(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
}

// Splits of the columns until the CUs' two workgroups each are all there, each wave on 64 columns or more (us, 8192 rows x 8192 in 137 slots, rank 16, 1 / 2 / 3 / 4 / 6 / 8 /
// 16 splits: 39 / 41 / 33 / 27 / 30 / 28 / 30 on the same buffers again, 71 / 73 / 59 / 45 / 57 / 52 / 54 out of HBM)
void plan_shrink(ShrinkArgs &a, int cus) {
    const uint32_t least = kShrinkWaves * 64, most = (a.cols + least - 1) / least, slots = likely_slots(a.g);
    const uint32_t splits = std::min({((uint32_t)cus * 2 + slots - 1) / slots, most, 16u});
    a.part = ((a.cols + splits - 1) / splits + least - 1) / least * least;
    a.u.planes = (a.cols + a.part - 1) / a.part;
}

hipError_t launch_shrink(const ShrinkArgs &a, hipStream_t stream) {
    return with_dt(a.dt, [&](auto dt) {
        return with_ranks(a.rank, [&](auto rt) {
            constexpr auto kernel = adapter_shrink_kernel<dt.value, rt.value>;
            constexpr int room = ShrinkShape<rt.value>::BYTES;
            static const hipError_t raised = room > 65536 ? hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, room) : hipSuccess;
            if (raised != hipSuccess) return raised;
            return launch_kernel(kernel, dim3(a.g.slot_count, a.u.planes), dim3(64 * kShrinkWaves), room, stream, a);
        });
    });
}

// Column tiles of a workgroup: as few as leave all workgroups room at the same time
hipError_t launch_expand(ExpandArgs a, int cus, hipStream_t stream) {
    const uint32_t tiles = (a.cols + kExpandCols - 1) / kExpandCols, room = (uint32_t)cus * (a.rank <= 64 ? 4 : 3);
    const uint32_t across = std::min<uint32_t>(std::max<uint32_t>(1, room / likely_slots(a.g)), 65535);
    const uint32_t each = (tiles + across - 1) / across;
    a.wide = each * kExpandCols;
    const dim3 grid(a.g.slot_count, (tiles + each - 1) / each);
    return with_dt(a.dt, [&](auto dt) {
        return with_ranks(a.rank, [&](auto rt) {
            auto typed = [&](auto y) {
                return launch_kernel(a.cols % kOctet ? adapter_expand_kernel<dt.value, y.value, rt.value * 16, ROW_ANY>
                                                     : adapter_expand_kernel<dt.value, y.value, rt.value * 16, ROW_WHOLE>, grid, dim3(256), 0, stream, a);
            };
            if (a.y_dt == QGEMM_DT_F32) return typed(std::integral_constant<int, QGEMM_DT_F32>{});
            if (a.y_dt == QGEMM_DT_BF16) return typed(std::integral_constant<int, QGEMM_DT_BF16>{});
            return typed(std::integral_constant<int, QGEMM_DT_F16>{});
        });
    });
}

namespace {
size_t grad_room(const AdapterGradArgs &a, int which) {
    if (!a.of[which].dw || (size_t)a.chunk * kSlotRows >= a.g.rows) return 0;
    return 2 * ((size_t)a.g.slot_count / a.chunk + 1) * a.rank * adapter_plane_cols(a.of[which].cols) * sizeof(float);
}
}  // namespace

size_t plan_adapter_grad(AdapterGradArgs &a, int cus) {
    a.tiles = column_tiles(a.of[0].cols);
    const uint64_t tiles = (a.of[0].dw ? a.tiles : 0) + (a.of[1].dw ? column_tiles(a.of[1].cols) : 0);
    a.chunk = 2;
    auto room = [&] { return grad_room(a, 0) + grad_room(a, 1); };
    while (room() && (room() > kMostRoom || (uint64_t)a.g.rows / kSlotRows / a.chunk * tiles > (uint64_t)cus * 4)) a.chunk *= 2;
    return room();
}
void place_adapter_grad(AdapterGradArgs &a, float *room) {
    a.of[0].room = room;
    a.of[1].room = (float *)((char *)room + grad_room(a, 0));
}

hipError_t launch_adapter_grad(AdapterGradArgs a, hipStream_t stream) {
    const dim3 grid(a.g.slot_count + a.g.adapters, a.tiles + column_tiles(a.of[1].cols));
    const hipError_t e = with_dt(a.dt, [&](auto dt) {
        return with_ranks(a.rank, [&](auto rt) {
            auto launch = [&](auto parts, auto row) {
                constexpr auto kernel = adapter_grad_kernel<dt.value, rt.value, parts.value, row.value>;
                constexpr int room = GradRoom<dt.value, rt.value, parts.value>::BYTES;
                static const hipError_t raised = room > 65536 ? hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, room) : hipSuccess;
                if (raised != hipSuccess) return raised;
                return launch_kernel(kernel, grid, dim3(rt.value == 8 ? 512 : 256), room, stream, a);
            };
            auto typed = [&](auto row) {
                return a.dw_dt == QGEMM_DT_F32 ? launch(std::integral_constant<int, 3>{}, row) : launch(std::integral_constant<int, 2>{}, row);
            };
            return a.of[0].cols % kOctet || a.of[1].cols % kOctet ? typed(std::integral_constant<int, ROW_ANY>{}) : typed(std::integral_constant<int, ROW_WHOLE>{});
        });
    });
    if (e != hipSuccess || grad_room(a, 0) + grad_room(a, 1) == 0) return e;
    // a workgroup for every rank while that makes some thousands; of many adapters most have no parts
    const uint32_t across = std::min<uint32_t>((std::max(a.of[0].cols, a.of[1].cols) + 2047) / 2048, 64);
    a.join = std::min(a.rank, std::max<uint32_t>(1, 4096 / a.g.adapters / across));
    return launch_kernel(adapter_grad_join_kernel, dim3(a.g.adapters * a.join, across, 2), dim3(256), 0, stream, a);
}

}  // namespace qgemm
