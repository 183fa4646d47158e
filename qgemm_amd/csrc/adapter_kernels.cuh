// Low-rank adapters of many requests at once: row t has adapter i = ids[t] (or none), and
//   u[t] = A_i x[t],   out[t] = y[t] + s_i B_i^T u[t];   backward   v[t] = B_i dy[t],   dx[t] += s_i A_i^T v[t],
//   dA_i = s_i sum over its rows of v[t] x[t]^T,   dB_i = s_i sum over its rows of u[t] dy[t]^T,   A_i [rank x k], B_i [rank x n].
// Three products serve all of it, because both factors lie with the rank as rows: "shrink" (a row times the factor's rows), "expand" (rank times the
// factor) and "gradient" (sums over the rows).
//
// Rows are grouped by adapter once for all of a step's products, and a workgroup takes a slot, up to 64 rows of one group, wherever
// they lie: rows are gathered and scattered as whole lines.
//
// u and v are fp32.  Where they are an operand of the matrix cores they are split into bf16 numbers that add up to them, two of them (16 bits) where
// the result has 16 bits, three (24) where it has 32; fp16 operands beside them are split into two, exactly, which keeps bf16's exponents:
// gradients are often below what fp16 holds.  An infinite operand meets all parts of the other, of which some are 0 or have the other sign: what depends on it is
// infinite or NaN, not always the formula's infinity.  (The sums of a result are its own: nothing else changes.)
//
// What bounds them, times of the kernels in a trace: memory, and for few rows the chain of trips to it (slot, order, operands) behind a launch.  64 rows of 48 adapters of
// rank 16, 4096 x 4096: group 2.8 us, shrink 4.4, expand 6.4; 8192 rows of 8 adapters of rank 32: 6.2, 16.6 and 31.2 (4.0 TB/s of x; 4.3 of y in and out).  Backward of 4096 rows of
// 16 adapters of rank 16, 2048 x 8192: 5.7, 19.2, 12.5, both gradients 23.6 and their parts' sums 6.5.  High ranks read the factors out of the L2 once
// a slot: shrink of 8192 rows of 8192 at rank 16 26.7 and at rank 64 50, 2048 rows at rank 128 46.
#pragma once
#include "model.h"
#include "octet.cuh"

namespace qgemm {

typedef short tr_v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) tr_v4s tr_quad;

// ---- groups.  One workgroup for each group: how many rows come in front of it, in how many groups, then its rows in their order.  Slots: with o rows and
// d groups in front, a group starts at slot o / 64 + d, and has room up to the next group's start, (o + n) / 64 + d + 1: at
// least its n / 64 rounded up.  So every group finds its slots without knowing the others' sizes.  Where there are more rows than adapters its number stands for d,
// which is no smaller and needs no counting (8192 rows 7.8 us with it, 6.2 without).
//
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
    auto dpp = [&](auto ctrl) { v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, true); };
    dpp(std::integral_constant<int, 0xB1>{});
    dpp(std::integral_constant<int, 0x4E>{});
    dpp(std::integral_constant<int, 0x141>{});
    dpp(std::integral_constant<int, 0x140>{});
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    v = a0 + a1;
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return b0 + b1;
}
// A thread has 4 neighbouring ids of each turn, of which TURNS stay in registers: of more rows all are read again for the second half.
template <int ID_BYTES, int WAVES, int TURNS>
__global__ void __launch_bounds__(64 * WAVES) group_rows_kernel(const void *ids, RowGroups g) {
    constexpr uint32_t THREADS = 64 * WAVES, TURN = THREADS * 4;
    __shared__ uint32_t seen[(kMostAdapters + 32) / 32], sums[WAVES][3], before[64];
    const uint32_t a = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, none = g.adapters;
    // groups of rows t .. t + 3, one beyond all groups for rows that there are none of
    auto fetch = [&](uint32_t t, uint32_t (&of)[4]) __attribute__((always_inline)) {
        int64_t id[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) id[e] = -1;
        if (t + 4 <= g.rows) {
            if constexpr (ID_BYTES == 4) {
                const v4i v = *(const v4i_any *)((const int32_t *)ids + t);
#pragma unroll
                for (int e = 0; e < 4; ++e) id[e] = v[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) id[e] = ((const int64_t *)ids)[t + e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (t + e < g.rows) id[e] = ID_BYTES == 4 ? (int64_t)((const int32_t *)ids)[t + e] : ((const int64_t *)ids)[t + e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) of[e] = t + e >= g.rows ? 0xFFFFFFFFu : id[e] >= 0 && id[e] < (int64_t)none ? (uint32_t)id[e] : none;
    };
    static_assert(WAVES * TURNS <= 64, "a lane for each part of a turn");
    const bool marks = g.rows <= none;                      // groups in front of this one have to be counted
    if (marks)
        for (uint32_t i = tid; i <= none / 32; i += THREADS) seen[i] = 0;
    if (tid < 64) before[tid] = 0;
    uint32_t of[TURNS][4], less = 0, equal = 0;
#pragma unroll
    for (uint32_t k = 0; k < TURNS; ++k) fetch(k * TURN + tid * 4, of[k]);
    if (marks) __syncthreads();
    auto count = [&](const uint32_t (&o)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            equal += o[e] == a ? 1 : 0;
            less += o[e] < a ? 1 : 0;
            if (marks && o[e] < a) atomicOr(&seen[o[e] / 32], 1u << (o[e] % 32));
        }
    };
#pragma unroll
    for (uint32_t k = 0; k < TURNS; ++k) count(of[k]);
    for (uint32_t t = TURNS * TURN + tid * 4; t < g.rows; t += TURN) {
        uint32_t o[4];
        fetch(t, o);
        count(o);
    }
    uint32_t distinct = 0;
    if (marks) {
        __syncthreads();
        for (uint32_t i = tid; i <= none / 32; i += THREADS) distinct += __builtin_popcount(seen[i]);
    }
    less = wave_total(less), equal = wave_total(equal), distinct = wave_total(distinct);
    if (lane == 0) sums[wave][0] = less, sums[wave][1] = equal, sums[wave][2] = distinct;
    __syncthreads();
    less = equal = distinct = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) less += sums[i][0], equal += sums[i][1], distinct += sums[i][2];
    if (!marks) distinct = a;

    const uint32_t slot = less / kSlotRows + distinct, filled = (equal + kSlotRows - 1) / kSlotRows;
    const uint32_t behind = a == none ? g.slot_count : !marks || equal ? (less + equal) / kSlotRows + distinct + 1 : slot;
    int32_t *order = const_cast<int32_t *>(g.order), *offsets = const_cast<int32_t *>(g.offsets), *first = const_cast<int32_t *>(g.first);
    v4i *slots = const_cast<v4i *>(g.slots);
    if (tid == 0) {
        offsets[a] = (int32_t)less;
        first[a] = (int32_t)slot;
        if (a == none) offsets[a + 1] = (int32_t)g.rows;
    }
    for (uint32_t i = tid; i < behind - slot; i += THREADS) {
        const uint32_t left = equal - (i < filled ? i : 0) * kSlotRows;
        slots[slot + i] = i < filled ? v4i{(int)a, (int)(less + i * kSlotRows), (int)(left < kSlotRows ? left : kSlotRows), (int)i} : v4i{-1, 0, 0, 0};
    }
    if (equal == 0) return;
    uint32_t at = less;
    for (uint32_t t0 = 0; t0 < g.rows; t0 += TURNS * TURN) {
        if (t0)
#pragma unroll
            for (uint32_t k = 0; k < TURNS; ++k) fetch(t0 + k * TURN + tid * 4, of[k]);
        uint32_t rank[TURNS];                              // of a thread's first row among the wave's
#pragma unroll
        for (uint32_t k = 0; k < TURNS; ++k) {
            uint32_t own = 0, all = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t mask = __ballot(of[k][e] == a);
                own += __builtin_popcountll(mask & (((uint64_t)1 << lane) - 1));
                all += __builtin_popcountll(mask);
            }
            rank[k] = own;
            if (lane == 0) before[k * WAVES + wave] = all;
        }
        __syncthreads();
        // what lies in front of the wave's part of a turn: an exclusive sum over the 64 parts
        uint32_t sum = before[lane];
        const uint32_t n = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t up = __shfl_up(sum, d);
            sum += lane >= (uint32_t)d ? up : 0;
        }
#pragma unroll
        for (uint32_t k = 0; k < TURNS; ++k) {
            uint32_t place = at + rank[k] + __shfl(sum - n, (int)(k * WAVES + wave));
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (of[k][e] == a) order[place++] = (int32_t)(t0 + k * TURN + tid * 4 + e);
        }
        at += __shfl(sum, 63);
        __syncthreads();
    }
}

// ---- what the three kernels share
struct Slot {
    uint32_t adapter, begin, count, nth;
    bool any;
};
__device__ __forceinline__ Slot slot_of(const RowGroups &g, uint32_t i) {
    const v4i s = g.slots[i];
    return Slot{(uint32_t)s[0], (uint32_t)s[1], (uint32_t)s[2], (uint32_t)s[3], s[0] >= 0};
}
template <int DT>
__device__ __forceinline__ v4f multiply16(v4i a, v4i b, v4f c) {
    if constexpr (DT == QGEMM_DT_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
// the bf16 nearest to v, and v without it (0 where that would be no number)
__device__ __forceinline__ uint16_t split_off(float &v) {
    const uint16_t h = f32_to_bf16_bits(v);
    const float rest = v - __builtin_bit_cast(float, (uint32_t)h << 16);
    v = __builtin_fabsf(rest) < __builtin_inff() ? rest : 0.0f;
    return h;
}
// the row of u that belongs to place `at` of the order
__device__ __forceinline__ uint32_t sums_row(const RankSums &u, const RowGroups &g, uint32_t at) { return u.grouped ? at : (uint32_t)g.order[at]; }
// four sums of a row from rank q on, those behind the last are 0; four or eight parts of them in flight
__device__ __forceinline__ v4f rank_sums(const RankSums &u, size_t row, uint32_t q, uint32_t rank) {
    v4f sum = {};
    const float *at = u.at + row * u.pitch + q;
    if (u.planes == 1 && q + 4 <= rank) return *(const v4f_any *)at;
    auto add = [&](auto flight, uint32_t i) __attribute__((always_inline)) {
        constexpr uint32_t N = decltype(flight)::value;
        v4f part[N];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            const float *p = at + (i + k < u.planes ? i + k : i) * u.stride;
            if (q + 4 <= rank) {
                part[k] = *(const v4f_any *)p;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) part[k][e] = q + e < rank ? p[e] : 0.0f;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < N; ++k)
            if (i + k < u.planes) sum += part[k];
    };
    if (u.planes <= 4) add(std::integral_constant<uint32_t, 4>{}, 0);
    else
        for (uint32_t i = 0; i < u.planes; i += 8) add(std::integral_constant<uint32_t, 8>{}, i);
    return sum;
}
// A panel is up to 32 rows of 16 FC columns of 16 bits, a wave's own.  `columns` gives the matrix cores' operand along the rows: lane j of a group of 16 supplies
// the address of 8 bytes of row j >> 2 and receives column j of the four.  The columns are taken so that a lane's results of FC fragments f are 4 FC
// neighbours: result i of fragment f in lane group g is column 4 FC g + 4 f + i.
template <int FC>
struct Panel {
    static constexpr int PITCH = 32 * FC + 16, BYTES = 32 * PITCH;
};
template <int FC>
__device__ __forceinline__ v4i columns(const char *panel, int f, int fr, int row) {
    const char *at = panel + (row + (fr >> 2)) * Panel<FC>::PITCH + 8 * FC * (fr & 3) + 8 * f;
    const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_quad *)at));
    const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_quad *)(at + 4 * Panel<FC>::PITCH)));
    return v4i{lo[0], lo[1], hi[0], hi[1]};
}
// an octet of 16-bit numbers as bf16 in PARTS panels
template <int DT, int PARTS>
__device__ __forceinline__ void stage_octet(const Octet<DT> &o, char *at, int part_stride) {
    if constexpr (DT == QGEMM_DT_BF16) {
        *(v4i *)at = v4i{(int)o.w[0], (int)o.w[1], (int)o.w[2], (int)o.w[3]};
    } else {
        float v[8];
        o.floats(v);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a = split_off(v[2 * i]), b = split_off(v[2 * i + 1]);
                w[i] = a | b << 16;
            }
            *(v4i *)(at + part * part_stride) = v4i{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
        }
    }
}
template <int DT>
constexpr int factor_parts() { return DT == QGEMM_DT_BF16 ? 1 : 2; }
template <int Y_DT>
constexpr int sum_parts() { return Y_DT == QGEMM_DT_F32 ? 3 : 2; }

// ---- shrink: both operands straight from memory to the matrix cores' registers; a lane takes 16 neighbouring columns of a row for two products, and four lanes a
// whole line.  The waves of a workgroup share its split's columns out between them, and ranks beyond 32 between two or four of them, which read the same rows.  Their sums meet in
// LDS, in BUFFERS places one after the other.  (8192 x 4096 at rank 32: four waves of 256 columns by three splits 23.5 us, half lines a request with a step ahead in flight
// 23.2, whole lines 21.2, and 16.6 with a fourth split, so that every CU has its two workgroups.  Sixteen waves a workgroup, one a CU: 27.)
constexpr int kShrinkWaves = 8;
template <int RT>
struct ShrinkShape {
    static constexpr int RW = RT < 2 ? RT : 2, RANK_WAVES = RT / RW, COLUMN_WAVES = kShrinkWaves / RANK_WAVES;
    static constexpr int BUFFERS = COLUMN_WAVES < 4 ? COLUMN_WAVES : 4, PITCH = RT * 16 + 4, BYTES = BUFFERS * kSlotRows * PITCH * 4;
};
template <int DT, int RT>
__global__ void __launch_bounds__(64 * kShrinkWaves, 4) adapter_shrink_kernel(const ShrinkArgs p) {
    typedef ShrinkShape<RT> Shape;
    constexpr int RANKS = RT * 16, THREADS = 64 * kShrinkWaves, RW = Shape::RW, BUFFERS = Shape::BUFFERS, PITCH = Shape::PITCH;
    extern __shared__ __align__(16) float red[];                // [BUFFERS][kSlotRows][PITCH]
    const Slot s = slot_of(p.g, blockIdx.x);
    if (!s.any) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
    float *u = p.u.at + blockIdx.y * p.u.stride;
    auto write = [&](auto value) __attribute__((always_inline)) {
        const uint32_t wide = p.u.pitch < RANKS ? p.u.pitch : RANKS;
        for (uint32_t i = tid; i < s.count * RANKS; i += THREADS) {
            const uint32_t row = i / RANKS, k = i % RANKS;
            if (k < wide) u[(size_t)sums_row(p.u, p.g, s.begin + row) * p.u.pitch + k] = k < p.rank ? value(row, k) : 0.0f;
        }
    };
    if (s.adapter == p.g.adapters) {
        if (p.zero) write([](uint32_t, uint32_t) { return 0.0f; });
        return;
    }
    const uint32_t ranks0 = wave % Shape::RANK_WAVES * RW, part = wave / Shape::RANK_WAVES, step = 64 * Shape::COLUMN_WAVES;
    const uint32_t from = blockIdx.y * p.part, k1 = p.cols - from < p.part ? p.cols : from + p.part;
    const char *w[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        const uint32_t k = (ranks0 + i) * 16 + fr < p.rank ? (ranks0 + i) * 16 + fr : p.rank - 1;      // (what comes of others is not written)
        w[i] = (const char *)p.w + ((size_t)s.adapter * p.rank + k) * p.cols * 2;
    }
    auto body = [&](auto frags) __attribute__((always_inline)) {
        constexpr int F = decltype(frags)::value;
        const char *x[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const uint32_t at = f * 16 + fr;
            x[f] = (const char *)p.x + (size_t)(uint32_t)p.g.order[s.begin + (at < s.count ? at : s.count - 1)] * p.ldx * 2;
        }
        v4f acc[F][RW] = {};
        struct Step {
            v4i a[RW][2], b[F][2];
        };
        auto products = [&](const Step &r) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int f = 0; f < F; ++f)
#pragma unroll
                    for (int i = 0; i < RW; ++i) acc[f][i] = multiply16<DT>(r.a[i][j], r.b[f][j], acc[f][i]);
        };
        // (side by side: all waves together read 512 columns of a row at a time)
        uint32_t k = from + part * 64;
#pragma unroll 1
        for (; k + 64 <= k1; k += step) {
            Step r;
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int j = 0; j < 2; ++j) r.b[f][j] = *(const v4i_any *)(x[f] + (k + fg * 16 + j * 8) * 2);
#pragma unroll
            for (int i = 0; i < RW; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) r.a[i][j] = *(const v4i_any *)(w[i] + (k + fg * 16 + j * 8) * 2);
            products(r);
        }
        if (k < k1) {                                       // the last columns of a row
            auto fetch = [&](const char *row, uint32_t c) __attribute__((always_inline)) {
                Octet<DT> o;
                o.request(row, c, p.cols);
                o.settle(c, p.cols);
                return v4i{(int)o.w[0], (int)o.w[1], (int)o.w[2], (int)o.w[3]};
            };
            Step r;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t c = k + fg * 16 + j * 8;
#pragma unroll
                for (int f = 0; f < F; ++f) r.b[f][j] = fetch(x[f], c);
#pragma unroll
                for (int i = 0; i < RW; ++i) r.a[i][j] = fetch(w[i], c);
            }
            products(r);
        }
        // a lane has ranks 16 i + 4 fg .. + 3 of row 16 f + fr
#pragma unroll 1
        for (uint32_t turn = 0; turn < Shape::COLUMN_WAVES / BUFFERS; ++turn) {
            if (part / BUFFERS == turn)
#pragma unroll
                for (int f = 0; f < F; ++f)
#pragma unroll
                    for (int i = 0; i < RW; ++i) {
                        v4f *at = (v4f *)(red + ((part % BUFFERS) * kSlotRows + f * 16 + fr) * PITCH + (ranks0 + i) * 16 + fg * 4);
                        *at = turn ? *at + acc[f][i] : acc[f][i];
                    }
            __syncthreads();
        }
    };
    if (s.count <= 16) body(std::integral_constant<int, 1>{});
    else if (s.count <= 32) body(std::integral_constant<int, 2>{});
    else body(std::integral_constant<int, 4>{});
    write([&](uint32_t row, uint32_t k) {
        float v = red[row * PITCH + k];
#pragma unroll
        for (int i = 1; i < BUFFERS; ++i) v += red[(i * kSlotRows + row) * PITCH + k];
        return v;
    });
}

// ---- expand: 32 columns a wave, all rows of the slot; y is what the accumulators start with.  A workgroup goes over `wide` columns, 128 at a time, the next tile's y
// and factor in flight behind a tile's products.  RANKS: the rank rounded up to 16, 32, 64 or 128;
// ROW: see RowKind
// (8192 x 4096 at rank 32: one tile of 256 columns a workgroup, everything loaded where it is wanted, 45 us; loads in front 37; 128 columns, several tiles a workgroup, 33;
// the factor of a whole tile a tile ahead, no more workgroups than run at a time 31.  Eight waves a workgroup: 32.  Rank 128, 2048 x 8192: 91, 49 and 35.)
constexpr int kExpandCols = 128;
template <int DT, int Y_DT, int RANKS, int ROW>
constexpr int expand_waves() {                                  // of a SIMD: what LDS and registers have room for
    const int lds = sum_parts<Y_DT>() * (int)kSlotRows * (RANKS * 2 + 16) + factor_parts<DT>() * 4 * Panel<2>::BYTES, fit = 160 * 1024 / lds;
    constexpr bool more = Y_DT == QGEMM_DT_F16 || ROW == ROW_ANY;
    const int most = RANKS < 64 ? (more ? 3 : 4) : more ? 2 : Y_DT == QGEMM_DT_F32 ? 3 : 4;
    return fit < most ? fit : most;
}
template <int DT, int Y_DT, int RANKS, int ROW>
__global__ void __launch_bounds__(256, (expand_waves<DT, Y_DT, RANKS, ROW>())) adapter_expand_kernel(const ExpandArgs p) {
    // PACKED (rank up to 16): two parts of u, 16 ranks each, make one product's 32
    constexpr bool PACKED = RANKS == 16;
    constexpr int PARTS = sum_parts<Y_DT>(), FACTORS = factor_parts<DT>(), STEP = PACKED ? 16 : 32, QUADS = RANKS / 4, PITCH = RANKS * 2 + 16;
    typedef Panel<2> P;
    __shared__ __align__(16) char sums[PARTS][kSlotRows * PITCH], panels[FACTORS][4 * P::BYTES];
    const Slot s = slot_of(p.g, blockIdx.x);
    if (!s.any) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fg = lane >> 4;
    const bool plain = s.adapter == p.g.adapters;
    if (plain && (const void *)p.out == p.y && !p.keep) return;
    const uint32_t ranks = plain ? 0 : p.rank, from = blockIdx.y * p.wide, to = p.cols - from < p.wide ? p.cols : from + p.wide;
    // (needs nothing but the slot)
    const uint32_t at_rank = lane >> 2, at_col = wave * 32 + (lane & 3) * 8;
    Octet<DT> w[RANKS / 16];                                     // of a whole tile: a wave has 16 ranks of 32 columns in one octet a lane
    auto request_w = [&](uint32_t tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < RANKS / 16; ++i) {
            const uint32_t r = i * 16 + at_rank;
            w[i].template request<ROW>((const char *)p.w + ((size_t)s.adapter * p.rank + (r < p.rank ? r : p.rank - 1)) * p.cols * 2, tile + at_col, p.cols);
        }
    };
    if (!plain) request_w(from);
    Octet<Y_DT> y[4];
    uint32_t row[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const uint32_t at = f * 16 + fr;
        row[f] = (uint32_t)p.g.order[s.begin + (at < s.count ? at : s.count - 1)];
    }
    const uint32_t own = wave * 32 + fg * 8;                     // a lane's columns of a tile
    auto request_y = [&](uint32_t tile) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            if (p.y) y[f].template request<ROW>((const char *)p.y + (size_t)row[f] * p.ldy * Octet<Y_DT>::ES, tile + own, p.cols);
            else y[f] = Octet<Y_DT>{};
        }
    };
    request_y(from);
    const float by = plain || !p.scaling ? 1.0f : p.scaling[s.adapter];
    // the rank's sums of the slot's rows, in parts: a lane has EACH quads of them (what lies behind the rows goes into products that nobody stores)
    constexpr int EACH = (int)kSlotRows * QUADS / 256;
    uint32_t sum_row[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const uint32_t at = (tid + 256 * i) / QUADS;
        sum_row[i] = sums_row(p.u, p.g, s.begin + (at < s.count ? at : s.count - 1));
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (256 * i / QUADS >= (int)s.count) break;
        const uint32_t n = tid + 256 * i, at = n / QUADS, q = n % QUADS * 4;
        v4f v = q < ranks ? rank_sums(p.u, sum_row[i], q, ranks) : v4f{};
        if (at >= s.count) break;
        if (p.keep && blockIdx.y == 0) {
            const size_t to_row = p.keep_grouped ? s.begin + at : (uint32_t)p.g.order[s.begin + at];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (q + e < p.rank) p.keep[to_row * p.rank + q + e] = v[e];
        }
        v *= by;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = v[e];
                h[e] = split_off(x);
                v[e] = x;
            }
            *(v2i *)(sums[part] + at * PITCH + q * 2) = v2i{(int)(h[0] | h[1] << 16), (int)(h[2] | h[3] << 16)};
        }
    }
    if (plain && (const void *)p.out == p.y) return;
    __syncthreads();
    char *panel = panels[0] + wave * P::BYTES;
    const uint32_t frags = (s.count + 15) / 16;
#pragma unroll 1
    for (uint32_t tile = from; tile < to; tile += kExpandCols) {
        const uint32_t n = tile + own, then = tile + kExpandCols;
        v4f acc[4][2];
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            float v[8];
            y[f].template settle<ROW>(n, p.cols);
            y[f].hold();
            y[f].floats(v);
            acc[f][0] = v4f{v[0], v[1], v[2], v[3]};
            acc[f][1] = v4f{v[4], v[5], v[6], v[7]};
        }
        if (then < to) request_y(then);
#pragma unroll
        for (int k = 0; k < RANKS; k += STEP) {
            if ((uint32_t)k >= ranks) break;
            // (a wave's panel is its own: what it writes and reads there comes in its own order)
#pragma unroll
            for (int i = 0; i < STEP / 16; ++i) {
                const uint32_t r = i * 16 + at_rank;
                Octet<DT> &o = w[k / 16 + i];
                o.template settle<ROW>(k + r < p.rank ? tile + at_col : p.cols, p.cols);
                stage_octet<DT, FACTORS>(o, panel + r * P::PITCH + (lane & 3) * 16, 4 * P::BYTES);
            }
            if ((uint32_t)k + STEP >= ranks && then < to) request_w(then);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            v4i z[FACTORS][2];
#pragma unroll
            for (int part = 0; part < FACTORS; ++part)
#pragma unroll
                for (int g = 0; g < 2; ++g) z[part][g] = columns<2>(panel + part * 4 * P::BYTES, g, fr, PACKED ? 8 * (fg & 1) : 8 * fg);
            constexpr int TURNS = PACKED ? (PARTS + 1) / 2 : PARTS;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                if ((uint32_t)f >= frags) break;
#pragma unroll
                for (int turn = 0; turn < TURNS; ++turn) {
                    v4i u;
                    if constexpr (PACKED) {
                        const int part = 2 * turn + (fg >> 1);
                        u = *(const v4i *)(sums[part < PARTS ? part : 0] + (f * 16 + fr) * PITCH + 16 * (fg & 1));
                        if (part >= PARTS) u = v4i{};
                    } else {
                        u = *(const v4i *)(sums[turn] + (f * 16 + fr) * PITCH + (k + 8 * fg) * 2);
                    }
#pragma unroll
                    for (int part = 0; part < FACTORS; ++part)
#pragma unroll
                        for (int g = 0; g < 2; ++g) acc[f][g] = multiply16<QGEMM_DT_BF16>(z[part][g], u, acc[f][g]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            if (f * 16 + fr >= s.count || n >= p.cols) continue;
            const v4f a = acc[f][0], b = acc[f][1];
            const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            store_octet<ROW>((char *)p.out + (size_t)row[f] * p.ldo * Octet<Y_DT>::ES, Y_DT, n, p.cols, v);
        }
    }
}

// ---- gradient: 64 columns a wave, all ranks, the rows of `chunk` slots of a group 32 at a time.  A group of more than that leaves its parts in the
// workspace: part j of a group whose slots start at f lies at slot f + j chunk, and between two multiples of `chunk` there is at most one
// such start with j > 0 and one with j = 0.
__device__ __forceinline__ size_t grad_plane_of(uint32_t slot, uint32_t chunk, bool later) { return (size_t)(slot / chunk) * 2 + (later ? 1 : 0); }
__host__ __device__ inline uint32_t adapter_plane_cols(uint32_t cols) { return (cols + 15) / 16 * 16; }

//
// Both factors' gradients are one launch: x counts slots, and behind them adapters, for those that have no rows; y the column tiles of the first and then of the
// second.  A step's loads are requested a step ahead, the numbers of its rows two.  (Both factors of 4096 rows, 2048 x 8192 at rank 16: two launches without loads ahead 65 us
// and 10 for their parts; 23.6 and 6.5.  u and v lie in LDS as rows, as they come, and are turned by the transposing reads: written turned, by elements, 2048 rows
// of 8192 at rank 128 took 150, 76 so.)
template <int DT, int RT, int PARTS>
struct GradRoom {
    static constexpr int BYTES = 2 * (PARTS * 32 * (RT * 32 + 16) + factor_parts<DT>() * 4 * Panel<4>::BYTES);
};
template <int DT, int RT, int PARTS, int ROW>
__global__ void __launch_bounds__(RT == 8 ? 512 : 256) adapter_grad_kernel(const AdapterGradArgs p) {
    // 128 ranks are shared out between two groups of waves
    constexpr int RG = RT == 8 ? 2 : 1, THREADS = 256 * RG, RI = RT / RG;
    constexpr int RANKS = RT * 16, FACTORS = factor_parts<DT>(), PITCH = RANKS * 2 + 16, QUADS = 32 * RANKS / 4, LOADS = (QUADS + THREADS - 1) / THREADS, OCTETS = 4 / RG;
    constexpr int SUMS = PARTS * 32 * PITCH, BUFFER = SUMS + FACTORS * 4 * Panel<4>::BYTES;
    extern __shared__ __align__(16) char lds[];                  // [2][BUFFER]
    const bool second = blockIdx.y >= p.tiles;
    const AdapterGrad &of = p.of[second];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fg = lane >> 4, cols = of.cols;
    const uint32_t panel = wave & 3, ranks0 = (wave >> 2) * RI, c0 = (blockIdx.y - (second ? p.tiles : 0)) * 256 + panel * 64;
    if (!of.dw) return;
    if (blockIdx.x >= p.g.slot_count) {
        const uint32_t a = blockIdx.x - p.g.slot_count;
        if (p.g.offsets[a + 1] != p.g.offsets[a]) return;
        const float zero[8] = {};
        for (uint32_t k = (wave >> 2) * 8 + (lane >> 3); k < p.rank; k += 8 * RG)
            if (c0 + (lane & 7) * 8 < cols) store_octet((char *)of.dw + ((size_t)a * p.rank + k) * cols * dtype_bytes(p.dw_dt), p.dw_dt, c0 + (lane & 7) * 8, cols, zero);
        return;
    }
    const Slot s = slot_of(p.g, blockIdx.x);
    const uint32_t a = s.adapter;
    if (!s.any || a == p.g.adapters || s.nth % p.chunk) return;
    const uint32_t start = (uint32_t)p.g.offsets[a], end = (uint32_t)p.g.offsets[a + 1], from = s.begin;
    const uint32_t to = end - from < p.chunk * kSlotRows ? end : from + p.chunk * kSlotRows;
    const float by = p.scaling ? p.scaling[a] : 1.0f;
    // rows of a lane's octets, and of its sums; none behind the last
    struct Rows {
        uint32_t z[OCTETS], u[LOADS];
    };
    struct Step {
        Octet<DT> z[OCTETS];
        v4f u[LOADS];
    };
    const uint32_t c = c0 + (lane & 7) * 8, octet0 = (wave >> 2) * OCTETS;      // a lane's octets: rows 8 (octet0 + i) + lane / 8 of the step
    auto rows_of = [&](Rows &r, uint32_t t) __attribute__((always_inline)) {
        auto at = [&](uint32_t i) { return i < to ? i : to - 1; };
#pragma unroll
        for (int i = 0; i < OCTETS; ++i) r.z[i] = (uint32_t)p.g.order[at(t + (octet0 + i) * 8 + (lane >> 3))];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) r.u[i] = sums_row(of.u, p.g, at(t + (tid + THREADS * i) / (RANKS / 4) % 32));
    };
    auto request = [&](Step &b, const Rows &r) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < OCTETS; ++i) b.z[i].template request<ROW>((const char *)of.z + (size_t)r.z[i] * of.ldz * 2, c, cols);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t q = (tid + THREADS * i) % (RANKS / 4) * 4;
            b.u[i] = q < p.rank ? rank_sums(of.u, r.u[i], q, p.rank) : v4f{};
        }
    };
    v4f acc[RI][4] = {};
    Rows rows;
    Step step;
    rows_of(rows, from);
    request(step, rows);
    rows_of(rows, from + 32);
    char *buffer = lds;
#pragma unroll 1
    for (uint32_t t = from; t < to; t += 32, buffer = buffer == lds ? lds + BUFFER : lds) {
#pragma unroll
        for (int i = 0; i < OCTETS; ++i) {
            const uint32_t at = (octet0 + i) * 8 + (lane >> 3);
            step.z[i].template settle<ROW>(t + at < to ? c : cols, cols);
            stage_octet<DT, FACTORS>(step.z[i], buffer + SUMS + panel * Panel<4>::BYTES + at * Panel<4>::PITCH + (lane & 7) * 16, 4 * Panel<4>::BYTES);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t n = tid + THREADS * i, at = n / (RANKS / 4), q = n % (RANKS / 4) * 4;
            if (QUADS % THREADS != 0 && n >= QUADS) continue;
            v4f v = t + at < to ? step.u[i] * by : v4f{};
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = v[e];
                    h[e] = split_off(x);
                    v[e] = x;
                }
                *(v2i *)(buffer + (part * 32 + at) * PITCH + q * 2) = v2i{(int)(h[0] | h[1] << 16), (int)(h[2] | h[3] << 16)};
            }
        }
        if (t + 32 < to) {
            request(step, rows);
            rows_of(rows, t + 64);
        }
        // (one barrier a step: who writes the buffer again has passed the next one, and that everyone passes behind these products)
        __syncthreads();
        v4i z[FACTORS][4];
#pragma unroll
        for (int part = 0; part < FACTORS; ++part)
#pragma unroll
            for (int f = 0; f < 4; ++f) z[part][f] = columns<4>(buffer + SUMS + (part * 4 + panel) * Panel<4>::BYTES, f, fr, 8 * fg);
#pragma unroll
        for (int i = 0; i < RI; ++i)
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const char *at = buffer + (part * 32 + 8 * fg + (fr >> 2)) * PITCH + 32 * (ranks0 + i) + 8 * (fr & 3);
                const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_quad *)at));
                const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_quad *)(at + 4 * PITCH)));
                const v4i u = v4i{lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                for (int k = 0; k < FACTORS; ++k)
#pragma unroll
                    for (int f = 0; f < 4; ++f) acc[i][f] = multiply16<QGEMM_DT_BF16>(z[k][f], u, acc[i][f]);
            }
    }
    // a lane has columns n .. n + 15 of rank 16 i + fr
    const uint32_t n = c0 + fg * 16, wide = adapter_plane_cols(cols);
    const bool parts = end - start > p.chunk * kSlotRows;
    float *plane = of.room + grad_plane_of(blockIdx.x, p.chunk, s.nth > 0) * p.rank * wide;
#pragma unroll
    for (int i = 0; i < RI; ++i) {
        const uint32_t k = (ranks0 + i) * 16 + fr;
        if (k >= p.rank || n >= cols) continue;
        if (parts) {
#pragma unroll
            for (int f = 0; f < 4; ++f) *(v4f *)(plane + (size_t)k * wide + n + 4 * f) = acc[i][f];
            continue;
        }
        char *out = (char *)of.dw + ((size_t)a * p.rank + k) * cols * dtype_bytes(p.dw_dt);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const v4f x = acc[i][2 * h], y = acc[i][2 * h + 1];
            const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            if (n + 8 * h < cols) store_octet(out, p.dw_dt, n + 8 * h, cols, v);
        }
    }
}

// groups of several parts, added up in their order: a workgroup has 2048 columns at a time of every p.join-th rank of one adapter
__global__ void __launch_bounds__(256) adapter_grad_join_kernel(const AdapterGradArgs p) {
    const AdapterGrad &of = p.of[blockIdx.z];
    const uint32_t a = blockIdx.x / p.join, rows = (uint32_t)p.g.offsets[a + 1] - (uint32_t)p.g.offsets[a], slots = (rows + kSlotRows - 1) / kSlotRows;
    const uint32_t wide = adapter_plane_cols(of.cols), first = (uint32_t)p.g.first[a];
    if (slots <= p.chunk || !of.dw) return;
#pragma unroll 1
    for (uint32_t k = blockIdx.x % p.join; k < p.rank; k += p.join) {
        char *out = (char *)of.dw + ((size_t)a * p.rank + k) * of.cols * dtype_bytes(p.dw_dt);
        for (uint32_t c = (blockIdx.y * 256 + threadIdx.x) * kOctet; c < of.cols; c += gridDim.y * 2048) {
            v4f lo = {}, hi = {};
            for (uint32_t at = 0; at < slots; at += p.chunk * 4) {
                v4f part[4][2];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t j = at + i * p.chunk < slots ? at + i * p.chunk : at;
                    const float *plane = of.room + (grad_plane_of(first + j, p.chunk, j > 0) * p.rank + k) * wide + c;
                    part[i][0] = *(const v4f *)plane;
                    part[i][1] = *(const v4f *)(plane + 4);
                }
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    if (at + i * p.chunk < slots) lo += part[i][0], hi += part[i][1];
            }
            const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            store_octet(out, p.dw_dt, c, of.cols, v);
        }
    }
}

}  // namespace qgemm
