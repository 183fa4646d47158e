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
// gradients are often below what fp16 holds.
#pragma once
#include "model.h"
#include "octet.cuh"

namespace qgemm {

typedef short tr_v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) tr_v4s tr_quad;

// ---- groups.  One workgroup for each group: how many rows come in front of it, in how many groups, then its rows in their order.  Slots: with o rows and
// d groups in front, a group starts at slot o / 64 + d, and has room up to the next group's start, (o + n) / 64 + d + 1: at
// least its n / 64 rounded up.  So every group finds its slots without knowing the others' sizes.
__global__ void __launch_bounds__(1024) group_rows_kernel(const void *ids, int id_bytes, RowGroups g) {
    __shared__ uint32_t seen[(kMostAdapters + 32) / 32], sums[16][3], before[2][16];
    const uint32_t a = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, none = g.adapters;
    auto group_of = [&](uint32_t t) {
        const int64_t id = id_bytes == 8 ? ((const int64_t *)ids)[t] : (int64_t)((const int32_t *)ids)[t];
        return id >= 0 && id < (int64_t)none ? (uint32_t)id : none;
    };
    for (uint32_t i = tid; i <= none / 32; i += 1024) seen[i] = 0;
    __syncthreads();
    uint32_t less = 0, equal = 0;
#pragma unroll 4
    for (uint32_t t = tid; t < g.rows; t += 1024) {
        const uint32_t of = group_of(t);
        if (of < a) {
            ++less;
            if (!(seen[of / 32] >> (of % 32) & 1)) atomicOr(&seen[of / 32], 1u << (of % 32));
        } else if (of == a) {
            ++equal;
        }
    }
    __syncthreads();
    uint32_t distinct = 0;
    for (uint32_t i = tid; i <= none / 32; i += 1024) distinct += __builtin_popcount(seen[i]);
    auto total = [&](uint32_t v) {
#pragma unroll
        for (int d = 32; d; d /= 2) v += __shfl_xor(v, d);
        return v;
    };
    less = total(less), equal = total(equal), distinct = total(distinct);
    if (lane == 0) sums[wave][0] = less, sums[wave][1] = equal, sums[wave][2] = distinct;
    __syncthreads();
    less = equal = distinct = 0;
    for (int i = 0; i < 16; ++i) less += sums[i][0], equal += sums[i][1], distinct += sums[i][2];

    const uint32_t slot = less / kSlotRows + distinct, filled = (equal + kSlotRows - 1) / kSlotRows;
    const uint32_t behind = a == none ? g.slot_count : equal ? (less + equal) / kSlotRows + distinct + 1 : slot;
    int32_t *order = const_cast<int32_t *>(g.order), *offsets = const_cast<int32_t *>(g.offsets), *first = const_cast<int32_t *>(g.first);
    v2i *slots = const_cast<v2i *>(g.slots);
    if (tid == 0) {
        offsets[a] = (int32_t)less;
        first[a] = (int32_t)slot;
        if (a == none) offsets[a + 1] = (int32_t)g.rows;
    }
    for (uint32_t i = slot + tid; i < behind; i += 1024)
        slots[i] = i - slot < filled ? v2i{(int)a, (int)(less + (i - slot) * kSlotRows)} : v2i{-1, 0};
    if (equal == 0) return;
    uint32_t at = less;
    int turn = 0;
    for (uint32_t t0 = 0; t0 < g.rows; t0 += 1024, turn ^= 1) {
        const bool own = t0 + tid < g.rows && group_of(t0 + tid) == a;
        const uint64_t mask = __ballot(own);
        if (lane == 0) before[turn][wave] = __builtin_popcountll(mask);
        __syncthreads();
        uint32_t place = at + __builtin_popcountll(mask & (((uint64_t)1 << lane) - 1));
        for (uint32_t i = 0; i < 16; ++i) {
            const uint32_t n = before[turn][i];
            if (i < wave) place += n;
            at += n;
        }
        if (own) order[place] = (int32_t)(t0 + tid);
    }
}

// ---- what the three kernels share
struct Slot {
    uint32_t adapter, begin, count;
    bool any;
};
__device__ __forceinline__ Slot slot_of(const RowGroups &g, uint32_t i) {
    const v2i s = g.slots[i];
    Slot r{(uint32_t)s[0], (uint32_t)s[1], 0, s[0] >= 0};
    if (r.any) {
        const uint32_t left = (uint32_t)g.offsets[r.adapter + 1] - r.begin;
        r.count = left < kSlotRows ? left : kSlotRows;
    }
    return r;
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
// four sums of a row from rank q on, those behind the last are 0
__device__ __forceinline__ v4f rank_sums(const RankSums &u, size_t row, uint32_t q, uint32_t rank, float by) {
    v4f sum = {};
    const float *at = u.at + row * u.pitch + q;
    for (uint32_t i = 0; i < u.planes; ++i, at += u.stride) {
        if (q + 4 <= rank) {
            sum += *(const v4f_any *)at;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (q + e < rank) sum[e] += at[e];
        }
    }
    return sum * by;
}
// A panel is up to 32 rows of 64 columns of 16 bits, a wave's own.  `columns` gives the matrix cores' operand along the rows: lane j of a group of 16 supplies
// the address of 8 bytes of row j >> 2 and receives column j of the four.  The columns are taken so that a lane's results of four fragments f
// are 16 neighbours: result i of fragment f in lane group g is column 16 g + 4 f + i.
constexpr int kPanelPitch = 144, kPanel = 32 * kPanelPitch;
__device__ __forceinline__ v4i columns(const char *panel, int f, int fr, int row) {
    const char *at = panel + (row + (fr >> 2)) * kPanelPitch + 32 * (fr & 3) + 8 * f;
    const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_quad *)at));
    const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_quad *)(at + 4 * kPanelPitch)));
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

// ---- shrink: the four waves of a workgroup share the columns of its split out between them, both operands straight from memory to the
// matrix cores' registers; a lane takes 16 neighbouring columns of a row for two products
template <int DT, int RT>
__global__ void __launch_bounds__(256) adapter_shrink_kernel(const ShrinkArgs p) {
    constexpr int RANKS = RT * 16;
    __shared__ float red[kSlotRows][RANKS + 4];
    const Slot s = slot_of(p.g, blockIdx.x);
    if (!s.any) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fg = lane >> 4;
    float *u = p.u.at + blockIdx.y * p.u.stride;
    auto write = [&](auto value) {
        const uint32_t wide = p.u.pitch < RANKS ? p.u.pitch : RANKS;
        for (uint32_t i = tid; i < s.count * RANKS; i += 256) {
            const uint32_t row = i / RANKS, k = i % RANKS;
            if (k < wide) u[(size_t)p.g.order[s.begin + row] * p.u.pitch + k] = k < p.rank ? value(row, k) : 0.0f;
        }
    };
    if (s.adapter == p.g.adapters) {
        if (p.zero) write([](uint32_t, uint32_t) { return 0.0f; });
        return;
    }
    const uint32_t quarter = p.part / 4, k0 = blockIdx.y * p.part + wave * quarter, k1 = p.cols < k0 + quarter ? p.cols : k0 + quarter;
    const char *w[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const uint32_t k = i * 16 + fr < p.rank ? i * 16 + fr : p.rank - 1;      // (what comes of others is not written)
        w[i] = (const char *)p.w + ((size_t)s.adapter * p.rank + k) * p.cols * 2;
    }
    auto body = [&](auto frags) {
        constexpr int F = decltype(frags)::value;
        const char *x[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const uint32_t at = f * 16 + fr;
            x[f] = (const char *)p.x + (size_t)p.g.order[s.begin + (at < s.count ? at : s.count - 1)] * p.ldx * 2;
        }
        v4f acc[F][RT] = {};
        for (uint32_t k = k0; k < k1; k += 64) {
            v4i a[RT][2], b[F][2];
            auto fetch = [&](const char *row, v4i &v, uint32_t c) {
                if (k + 64 <= p.cols) {
                    v = *(const v4i_any *)(row + (size_t)c * 2);
                } else {
                    Octet<DT> o;
                    o.request(row, c, p.cols);
                    o.settle(c, p.cols);
                    v = v4i{(int)o.w[0], (int)o.w[1], (int)o.w[2], (int)o.w[3]};
                }
            };
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t c = k + fg * 16 + j * 8;
#pragma unroll
                for (int f = 0; f < F; ++f) fetch(x[f], b[f][j], c);
#pragma unroll
                for (int i = 0; i < RT; ++i) fetch(w[i], a[i][j], c);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int f = 0; f < F; ++f)
#pragma unroll
                    for (int i = 0; i < RT; ++i) acc[f][i] = multiply16<DT>(a[i][j], b[f][j], acc[f][i]);
        }
        // a lane has ranks 16 i + 4 fg .. + 3 of row 16 f + fr; the waves one after the other
        for (uint32_t turn = 0; turn < 4; ++turn) {
            if (wave == turn)
#pragma unroll
                for (int f = 0; f < F; ++f)
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        v4f *at = (v4f *)&red[f * 16 + fr][i * 16 + fg * 4];
                        *at = turn ? *at + acc[f][i] : acc[f][i];
                    }
            __syncthreads();
        }
    };
    if (s.count <= 16) body(std::integral_constant<int, 1>{});
    else body(std::integral_constant<int, 4>{});
    write([&](uint32_t row, uint32_t k) { return red[row][k]; });
}

// ---- expand: 64 columns a wave, all rows of the slot; y is what the accumulators start with
template <int DT, int Y_DT, bool PACKED>
__global__ void __launch_bounds__(256) adapter_expand_kernel(const ExpandArgs p) {
    // PACKED (rank up to 16): two parts of u, 16 ranks each, make one product's 32
    constexpr int PARTS = sum_parts<Y_DT>(), FACTORS = factor_parts<DT>(), STEP = PACKED ? 16 : 32;
    constexpr int PITCH = PACKED ? 48 : kMostRank * 2 + 16;
    __shared__ __align__(16) char sums[PARTS][kSlotRows * PITCH], panels[FACTORS][4 * kPanel];
    const Slot s = slot_of(p.g, blockIdx.x);
    if (!s.any) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fg = lane >> 4;
    const uint32_t n0 = blockIdx.y * 256 + wave * 64, n = n0 + fg * 16;
    const bool plain = s.adapter == p.g.adapters;
    if (plain && (const void *)p.out == p.y && !p.keep) return;
    Octet<Y_DT> y[4][2];
    uint32_t row[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const uint32_t at = f * 16 + fr;
        row[f] = (uint32_t)p.g.order[s.begin + (at < s.count ? at : s.count - 1)];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (p.y) y[f][h].request((const char *)p.y + (size_t)row[f] * p.ldy * Octet<Y_DT>::ES, n + 8 * h, p.cols);
            else y[f][h] = Octet<Y_DT>{};
        }
    }
    const uint32_t ranks = plain ? 0 : p.rank, padded = (p.rank + STEP - 1) / STEP * STEP, quads = padded / 4;
    const float by = plain || !p.scaling ? 1.0f : p.scaling[s.adapter];
    for (uint32_t i = tid; i < kSlotRows * quads; i += 256) {
        const uint32_t at = i / quads, q = i % quads * 4;
        v4f v = {};
        if (at < s.count) {
            const size_t r = (uint32_t)p.g.order[s.begin + at];
            v = rank_sums(p.u, r, q, ranks, 1.0f);
            if (p.keep && blockIdx.y == 0)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (q + e < p.rank) p.keep[r * p.rank + q + e] = v[e];
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
    v4f acc[4][4];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[8];
            y[f][h].settle(n + 8 * h, p.cols);
            y[f][h].floats(v);
            acc[f][2 * h] = v4f{v[0], v[1], v[2], v[3]};
            acc[f][2 * h + 1] = v4f{v[4], v[5], v[6], v[7]};
        }
    for (uint32_t k = 0; k < ranks; k += STEP) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < STEP / 8; ++i) {
            const uint32_t at = i * 8 + (lane >> 3), r = k + at, c = n0 + (lane & 7) * 8;
            Octet<DT> o;
            o.request((const char *)p.w + ((size_t)s.adapter * p.rank + (r < p.rank ? r : p.rank - 1)) * p.cols * 2, c, p.cols);
            o.settle(r < p.rank ? c : p.cols, p.cols);
            stage_octet<DT, FACTORS>(o, panels[0] + wave * kPanel + at * kPanelPitch + (lane & 7) * 16, 4 * kPanel);
        }
        __syncthreads();
        v4i w[FACTORS][4];
#pragma unroll
        for (int part = 0; part < FACTORS; ++part)
#pragma unroll
            for (int f = 0; f < 4; ++f) w[part][f] = columns(panels[part] + wave * kPanel, f, fr, PACKED ? 8 * (fg & 1) : 8 * fg);
        constexpr int TURNS = PACKED ? (PARTS + 1) / 2 : PARTS;
#pragma unroll
        for (int turn = 0; turn < TURNS; ++turn)
#pragma unroll
            for (int f = 0; f < 4; ++f) {
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
                    for (int g = 0; g < 4; ++g) acc[f][g] = multiply16<QGEMM_DT_BF16>(w[part][g], u, acc[f][g]);
            }
    }
    if (plain && (const void *)p.out == p.y) return;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        if (f * 16 + fr >= s.count) continue;
        char *out = (char *)p.out + (size_t)row[f] * p.ldo * Octet<Y_DT>::ES;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const v4f a = acc[f][2 * h], b = acc[f][2 * h + 1];
            const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            if (n + 8 * h < p.cols) store_octet(out, Y_DT, n + 8 * h, p.cols, v);
        }
    }
}

// ---- gradient: 64 columns a wave, all ranks, the rows of `chunk` slots of a group 32 at a time.  A group of more than that leaves its parts in the
// workspace: part j of a group whose slots start at f lies at slot f + j chunk, and between two multiples of `chunk` there is at most one
// such start with j > 0 and one with j = 0.
__device__ __forceinline__ size_t grad_plane_of(uint32_t slot, uint32_t chunk, bool later) { return (size_t)(slot / chunk) * 2 + (later ? 1 : 0); }
__host__ __device__ inline uint32_t adapter_plane_cols(uint32_t cols) { return (cols + 15) / 16 * 16; }

template <int DT, int RT, int PARTS>
__global__ void __launch_bounds__(256) adapter_grad_kernel(const AdapterGradArgs p) {
    constexpr int RANKS = RT * 16, FACTORS = factor_parts<DT>(), PITCH = 80;
    __shared__ __align__(16) char sums[PARTS][RANKS * PITCH], panels[FACTORS][4 * kPanel];
    const v2i slot = p.g.slots[blockIdx.x];
    const uint32_t a = (uint32_t)slot[0];
    if (slot[0] < 0 || a == p.g.adapters) return;
    const uint32_t nth = blockIdx.x - (uint32_t)p.g.first[a];
    if (nth % p.chunk) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fg = lane >> 4;
    const uint32_t c0 = blockIdx.y * 256 + wave * 64, start = (uint32_t)p.g.offsets[a], end = (uint32_t)p.g.offsets[a + 1], from = (uint32_t)slot[1];
    const uint32_t to = end - from < p.chunk * kSlotRows ? end : from + p.chunk * kSlotRows;
    const float by = p.scaling ? p.scaling[a] : 1.0f;
    v4f acc[RT][4] = {};
    for (uint32_t t = from; t < to; t += 32) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t at = i * 8 + (lane >> 3), c = c0 + (lane & 7) * 8;
            Octet<DT> o;
            o.request((const char *)p.z + (size_t)(uint32_t)p.g.order[t + at < to ? t + at : to - 1] * p.ldz * 2, c, p.cols);
            o.settle(t + at < to ? c : p.cols, p.cols);
            stage_octet<DT, FACTORS>(o, panels[0] + wave * kPanel + at * kPanelPitch + (lane & 7) * 16, 4 * kPanel);
        }
        for (uint32_t i = tid; i < 32 * RANKS / 4; i += 256) {
            const uint32_t at = i / (RANKS / 4), q = i % (RANKS / 4) * 4;
            v4f v = {};
            if (t + at < to && q < p.rank) v = rank_sums(p.u, (uint32_t)p.g.order[t + at], q, p.rank, by);
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = v[e];
                    *(uint16_t *)(sums[part] + (q + e) * PITCH + at * 2) = split_off(x);
                    v[e] = x;
                }
        }
        __syncthreads();
        v4i z[FACTORS][4];
#pragma unroll
        for (int part = 0; part < FACTORS; ++part)
#pragma unroll
            for (int f = 0; f < 4; ++f) z[part][f] = columns(panels[part] + wave * kPanel, f, fr, 8 * fg);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const v4i u = *(const v4i *)(sums[part] + (i * 16 + fr) * PITCH + 16 * fg);
#pragma unroll
                for (int k = 0; k < FACTORS; ++k)
#pragma unroll
                    for (int f = 0; f < 4; ++f) acc[i][f] = multiply16<QGEMM_DT_BF16>(z[k][f], u, acc[i][f]);
            }
    }
    // a lane has columns n .. n + 15 of rank 16 i + fr
    const uint32_t n = c0 + fg * 16, wide = adapter_plane_cols(p.cols);
    const bool parts = end - start > p.chunk * kSlotRows;
    float *plane = p.room + grad_plane_of(blockIdx.x, p.chunk, nth > 0) * p.rank * wide;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const uint32_t k = i * 16 + fr;
        if (k >= p.rank || n >= p.cols) continue;
        if (parts) {
#pragma unroll
            for (int f = 0; f < 4; ++f) *(v4f *)(plane + (size_t)k * wide + n + 4 * f) = acc[i][f];
            continue;
        }
        char *out = (char *)p.dw + ((size_t)a * p.rank + k) * p.cols * dtype_bytes(p.dw_dt);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const v4f x = acc[i][2 * h], y = acc[i][2 * h + 1];
            const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            if (n + 8 * h < p.cols) store_octet(out, p.dw_dt, n + 8 * h, p.cols, v);
        }
    }
}

// groups of several parts added up in their order, groups of no rows to zeros: a workgroup has up to 2048 columns of one rank of one adapter
__global__ void __launch_bounds__(256) adapter_grad_join_kernel(const AdapterGradArgs p) {
    const uint32_t a = blockIdx.x / p.rank, k = blockIdx.x % p.rank, rows = (uint32_t)p.g.offsets[a + 1] - (uint32_t)p.g.offsets[a];
    const uint32_t slots = (rows + kSlotRows - 1) / kSlotRows;
    if (rows && slots <= p.chunk) return;
    const uint32_t wide = adapter_plane_cols(p.cols), first = (uint32_t)p.g.first[a];
    char *out = (char *)p.dw + ((size_t)a * p.rank + k) * p.cols * dtype_bytes(p.dw_dt);
    for (uint32_t c = (blockIdx.y * 256 + threadIdx.x) * kOctet; c < p.cols; c += gridDim.y * 2048) {
        v4f lo = {}, hi = {};
        for (uint32_t at = 0; at < slots; at += p.chunk) {
            const float *plane = p.room + (grad_plane_of(first + at, p.chunk, at > 0) * p.rank + k) * wide + c;
            lo += *(const v4f *)plane;
            hi += *(const v4f *)(plane + 4);
        }
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        store_octet(out, p.dw_dt, c, p.cols, v);
    }
}

}  // namespace qgemm
