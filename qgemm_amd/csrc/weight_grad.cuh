// Weight gradient of a linear layer out of an activation in 8 bits: dW[n, k] = sum over rows m of dy[m, n] v[m, k] with
// v = q s, s one scale for a row's 128 columns, and db[n] = sum over m of dy[m, n].  Where q holds a norm's xhat, and the layer's input
// was xhat w + b, the two vectors leave the sum: dW[n, k] = w[k] sum dy xhat + b[k] db[n], and the product reads codes alone.
//
// Both operands lie with their rows along the contraction, as they were written.  A step is 32 rows: dy goes from memory through registers
// into LDS as it is, codes are widened to dy's type on the way (exact for powers of two as scales, see power_of_two; other scales' products are
// rounded to fp32 and then to dy's type), and the matrix cores' operands, which run along the rows, are taken out of both with transposing reads.
// fp32 accumulators, fp32 planes.
//
// What bounds it: at 8192 x 8192 x 4096 (bf16, int8 codes) 480 - 510 us, 1.08 - 1.14 PFLOP/s of the 1.54 that the product of two bf16 matrices
// reaches at 8192^3 on the same card.  Steps to there, us: waves that load, convert and multiply in turn, 128 x 128 tiles 1118, 256 x 256 610;
// conversions between the products and buffers of four steps 570; waves of their own for copies and conversions 522; those in two pairs that work on
// alternate steps 507; both operands in both of a pair's turns 485.  Without any copying the computing waves take 405, without LDS reads as well
// 313; one computing wave a SIMD with 128 x 128 of its own took 832 (nothing hides what it waits for).  Converting costs the copying waves 2.5
// vector instructions an element, which go between products that hold the same port: without them 470.  The 256 x 256 form keeps 20 bytes a
// lane in scratch.  Few rows are bound by dW's own bytes: 64 rows of 8192 x 4096 33.7 us into fp32 (27 at the rate of a copy) and 26.6 into
// bf16 (13), 512 rows 54 (28) and 49 (22).
#pragma once
#include "octet.cuh"
#include "training.h"

namespace qgemm {

typedef short grad_v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) grad_v4s lds_quad;

constexpr int kGradStep = 32;          // rows of a step: the contraction of one matrix instruction

// The tile of a workgroup: BN x BK of dW by WN x WK computing waves, and four that copy
template <int DY_DT, int Q_DT, int BN_, int BK_, int WN_, int WK_>
struct GradCfg {
    static constexpr int DY = DY_DT, Q = Q_DT, BN = BN_, BK = BK_, WN = WN_, WK = WK_;
    static constexpr int COMPUTE = 64 * WN * WK, COPY = 128, THREADS = COMPUTE + 2 * COPY;       // COPY: a pair of copying waves
    static constexpr int FN = BN / WN / 16, FK = BK / WK / 16;                     // fragments of a computing wave
    static constexpr int FS = BN / 64;                                             // fragments of dy that a copying wave sums up
    static constexpr int LOAD_N = kGradStep * BN / 8 / COPY, LOAD_K = kGradStep * BK / 8 / COPY;      // octets of a copying lane
    static constexpr int PANEL = kGradStep * 128;                                  // 64 columns of 16 bits
    static constexpr int STAGE = (BN + BK) / 64 * PANEL;
    static constexpr int STAGES = 4, RING = STAGES * STAGE, LDS = RING + BN * 4;   // and a float for each row of the tile
    static constexpr int PASSES = (BN * BK * 4 + RING - 1) / RING, PASS_ROWS = BN / PASSES;      // the tile leaves through the ring
    static constexpr int AHEAD = 2;                                                // fragments of dy that are read in front of their products
    static constexpr bool EVEN = BN * BK > 256 * 128;                              // both of a step's turns bring some of both operands
    static_assert(BN % 64 == 0 && BK % 64 == 0 && LOAD_N % 2 == 0 && LOAD_K % 2 == 0, "whole panels, two halves");
    static_assert(BN % PASSES == 0 && PASS_ROWS % (BN / WN) == 0 && THREADS % (BK / 4) == 0, "whole waves in a pass, whole rows in a turn");
    static_assert(COPY % (BN / 8) == 0 && COPY % (BK / 8) == 0, "a lane's octets lie under one another");
};

// 16-byte chunk c of row k of a panel lies in slot c ^ grad_swizzle(k): the rows that a transposing read takes together, k0 .. k0 + 3 of
// two groups of lanes eight rows apart, lie in different banks
__device__ __forceinline__ constexpr int grad_swizzle(int k) { return (((k >> 1) & 1) << 1) | (((k >> 3) & 1) << 2); }

__device__ __forceinline__ float grad_parameter(const void *v, int dt, uint32_t k) {
    if (dt == QGEMM_DT_F32) return ((const float *)v)[k];
    const uint16_t h = ((const uint16_t *)v)[k];
    return dt == QGEMM_DT_BF16 ? __builtin_bit_cast(float, (uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}
// The norm's parameters of four neighbouring columns, some of which may lie behind the last
struct GradColumns {
    float w[4], b[4];
    __device__ __forceinline__ GradColumns(const WeightGradArgs &p, uint32_t k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t at = k + e < p.cols ? k + e : p.cols - 1;
            w[e] = p.weight ? grad_parameter(p.weight, p.param_dt, at) : 1.0f;
            b[e] = p.bias ? grad_parameter(p.bias, p.param_dt, at) : 0.0f;
        }
    }
};
// four neighbouring sums of row n, from column k on, as dW; db is 0 where there is no bias
template <int DT>
__device__ __forceinline__ void grad_store(const WeightGradArgs &p, const GradColumns &c, uint32_t n, uint32_t k, v4f sum, float db) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = p.weight ? sum[e] * c.w[e] : sum[e];
        v[e] = p.bias ? v[e] + c.b[e] * db : v[e];
    }
    store_out4(p.dw, (size_t)n * p.lddw + k, v, DT, (int)(p.cols - k < 4 ? p.cols - k : 4));
}

#define ALWAYS_INLINE __attribute__((always_inline))
template <class C>
__global__ void __launch_bounds__(C::THREADS) weight_grad_kernel(const WeightGradArgs p, const TileMap map) {
    extern __shared__ __align__(16) char lds[];
    typedef Octet<C::DY> OctetN;
    typedef Octet<C::Q> OctetK;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t tn, tk;
    tile_map(blockIdx.x, map, tn, tk);
    const uint32_t n0 = tn * C::BN, k0 = tk * C::BK;
    const uint32_t from = blockIdx.y * p.slice, to = p.rows - from < p.slice ? p.rows : from + p.slice;      // rows of this workgroup

    // ---- memory to registers: octet i of a lane is row row_n + i ROWS_N of the step, columns cn .. cn + 7
    constexpr uint32_t ROWS_N = C::COPY / (C::BN / 8), ROWS_K = C::COPY / (C::BK / 8);
    const uint32_t copier = tid % C::COPY;             // (COMPUTE is a multiple of COPY: a pair is two neighbouring waves)
    const uint32_t row_n = copier / (C::BN / 8), cn = n0 + copier % (C::BN / 8) * 8, row_k = copier / (C::BK / 8), ck = k0 + copier % (C::BK / 8) * 8;
    const uint32_t kb = ck < p.cols ? ck / kScaleBlock : 0;
    struct Set {
        OctetN on[C::LOAD_N];
        OctetK ok[C::LOAD_K];
        float scale[C::LOAD_K];
    };
    // Steps of which every octet may be fetched as it lies: what a row's last octet has behind the row is the next row's, and counts in
    // columns only that nobody stores.  In the last row there is no next one.
    const uint32_t behind = p.rows - (p.n % 8 != 0 || p.cols % 8 != 0 ? 1 : 0), plain_to = p.plain ? (to < behind ? to : behind) : 0;
    const uint32_t at_n = (uint32_t)((row_n * p.lddy + (cn < p.n ? cn : 0)) * 2), at_k = (uint32_t)(row_k * p.ldq + (ck < p.cols ? ck : 0));
    const uint32_t at_s = (row_k * p.kb + kb) * 4;
    // buffer loads: the step's base and the octet's rows in scalar registers, the lane's place in one that never changes
    auto base = [&](const void *at, uint64_t bytes) ALWAYS_INLINE {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>((const char *)at + bytes), 0, 0x7FFFFFFF, 0x00020000);
    };
    const uint32_t next_n = (uint32_t)(ROWS_N * p.lddy * 2), next_k = (uint32_t)(ROWS_K * p.ldq), next_s = ROWS_K * p.kb * 4;
    auto plain_n = [&](Set &r, int i0, int i1, uint32_t m0) ALWAYS_INLINE {
        const auto from = base(p.dy, (uint64_t)m0 * p.lddy * 2);
#pragma unroll
        for (int i = i0; i < i1; ++i) {
            const v4i v = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(from, at_n, i * next_n, 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) r.on[i].w[e] = (uint32_t)v[e];
        }
    };
    auto plain_k = [&](Set &r, int i0, int i1, uint32_t m0) ALWAYS_INLINE {
        const auto q = base(p.q, (uint64_t)m0 * p.ldq), s = base(p.scales, (uint64_t)m0 * p.kb * 4);
#pragma unroll
        for (int i = i0; i < i1; ++i) {
            const v2i v = __builtin_bit_cast(v2i, __builtin_amdgcn_raw_buffer_load_b64(q, at_k, i * next_k, 0));
            r.ok[i].w[0] = (uint32_t)v[0], r.ok[i].w[1] = (uint32_t)v[1];
            r.scale[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(s, at_s, i * next_s, 0));
        }
    };
    auto request_n = [&](Set &r, int i0, int i1, uint32_t m0) ALWAYS_INLINE {
        if (m0 + kGradStep <= plain_to) return plain_n(r, i0, i1, m0);
#pragma unroll
        for (int i = i0; i < i1; ++i) {
            const uint32_t m = m0 + row_n + i * ROWS_N;
            r.on[i].request((const char *)p.dy + (size_t)(m < to ? m : p.rows - 1) * p.lddy * 2, cn, p.n);
            r.on[i].settle(m < to ? cn : p.n, p.n);
        }
    };
    auto request_k = [&](Set &r, int i0, int i1, uint32_t m0) ALWAYS_INLINE {
        if (m0 + kGradStep <= plain_to) return plain_k(r, i0, i1, m0);
#pragma unroll
        for (int i = i0; i < i1; ++i) {
            const uint32_t m = m0 + row_k + i * ROWS_K;
            const size_t row = m < to ? m : p.rows - 1;
            r.ok[i].request((const char *)p.q + row * p.ldq, ck, p.cols);
            r.ok[i].settle(m < to ? ck : p.cols, p.cols);
            r.scale[i] = m < to ? p.scales[row * p.kb + kb] : 0.0f;
        }
    };
    // ---- registers to LDS
    auto slot = [&](uint32_t k, uint32_t chunk) ALWAYS_INLINE { return (chunk >> 3) * C::PANEL + k * 128 + (((chunk & 7) ^ grad_swizzle(k)) << 4); };
    auto stage_n = [&](Set &r, int i, char *to) ALWAYS_INLINE {
        *(v4i *)(to + slot(row_n + i * ROWS_N, copier % (C::BN / 8))) = v4i{(int)r.on[i].w[0], (int)r.on[i].w[1], (int)r.on[i].w[2], (int)r.on[i].w[3]};
    };
    auto stage_k = [&](Set &r, int i, char *to) ALWAYS_INLINE {
        float v[8];
        r.ok[i].floats(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= r.scale[i];
        const v2i a = C::DY == QGEMM_DT_BF16 ? pack4_bf16(v[0], v[1], v[2], v[3]) : pack4_f16(v[0], v[1], v[2], v[3]);
        const v2i b = C::DY == QGEMM_DT_BF16 ? pack4_bf16(v[4], v[5], v[6], v[7]) : pack4_f16(v[4], v[5], v[6], v[7]);
        *(v4i *)(to + C::BN / 64 * C::PANEL + slot(row_k + i * ROWS_K, copier % (C::BK / 8))) = v4i{a[0], a[1], b[0], b[1]};
    };
    // ---- LDS to operands: columns 16 x .. 16 x + 15 along the rows.  Lane j of a group of 16 supplies the address of
    // 8 bytes of row j >> 2 and receives column j of the four rows
    const int fr = lane & 15, fg = lane >> 4;
    const int lane_at = (8 * fg + (fr >> 2)) * 128 + 16 * (((fr >> 1) & 1) | grad_swizzle(8 * fg + (fr >> 2))) + 8 * (fr & 1);
    auto fragment = [&](const char *panels, int x) ALWAYS_INLINE {
        const char *at = panels + (x >> 2) * C::PANEL + (lane_at ^ ((x & 3) * 32));
        const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad *)at));
        const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad *)(at + 4 * 128)));
        return v4i{lo[0], lo[1], hi[0], hi[1]};
    };
    auto multiply = [&](v4i x, v4i y, v4f c) ALWAYS_INLINE {
        if constexpr (C::DY == QGEMM_DT_BF16)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x), __builtin_bit_cast(v8bf, y), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0, 0);
    };

    auto buffer = [&](uint32_t t) ALWAYS_INLINE { return lds + (t & 3) * C::STAGE; };
    const uint32_t steps = from < to ? (to - from + kGradStep - 1) / kGradStep : 0;
    const bool split = gridDim.y > 1, sums = (tk == 0 && (p.db || (split && p.bias))) || (p.bias && !split);
    float *row_sums = (float *)(lds + C::RING);

    // ---- dW: the computing waves leave their accumulators in LDS, PASS_ROWS rows at a time, and all waves take whole rows out of it.  The 16
    // bytes of columns 4 c .. 4 c + 3 of row r lie in slot c ^ (r & 15): a lane has four columns of one row, sixteen rows side by side
    auto leave = [&](auto put) ALWAYS_INLINE {
        constexpr uint32_t CHUNKS = C::BK / 4, ROWS = C::THREADS / CHUNKS;
        const uint32_t chunk = tid % CHUNKS, k = k0 + chunk * 4;
        const GradColumns columns(p, k < p.cols ? k : 0);
        auto out = [&](uint32_t n1, auto to_row) ALWAYS_INLINE {
#pragma unroll 1
            for (uint32_t row = tid / CHUNKS; row < C::PASS_ROWS; row += ROWS)
                if (n1 + row < p.n && k < p.cols) to_row(n1 + row, *(const v4f *)(lds + row * (C::BK * 4) + ((chunk ^ (row & 15)) << 4)));
        };
#pragma unroll 1
        for (uint32_t pass = 0; pass < C::PASSES; ++pass) {
            __syncthreads();
            put(pass);
            __syncthreads();
            const uint32_t n1 = n0 + pass * C::PASS_ROWS;
            auto as = [&](auto dt) ALWAYS_INLINE {
                out(n1, [&](uint32_t n, v4f sum) ALWAYS_INLINE { grad_store<dt.value>(p, columns, n, k, sum, p.bias ? row_sums[n - n0] : 0.0f); });
            };
            if (split) {
                float *plane = (float *)p.room + (size_t)blockIdx.y * grad_plane(p.n, p.cols) + grad_round(p.n);
                const size_t ld = grad_round(p.cols);
                out(n1, [&](uint32_t n, v4f sum) ALWAYS_INLINE { *(v4f *)(plane + n * ld + k) = sum; });
            } else if (p.dw_dt == QGEMM_DT_F32) as(std::integral_constant<int, QGEMM_DT_F32>{});
            else if (p.dw_dt == QGEMM_DT_BF16) as(std::integral_constant<int, QGEMM_DT_BF16>{});
            else as(std::integral_constant<int, QGEMM_DT_F16>{});
        }
    };

    if (wave >= C::COMPUTE / 64) {
        // ---- The copying waves.  One pair brings the even steps from registers to LDS, the other the odd ones, each for two turns of the
        // computing waves, so that one converts while the other's loads are issued.  A step s is written in turns s - 3 and s - 2, and
        // what step s + 2 holds is requested in its place, two turns ahead (four ahead, in a second set of registers, gained nothing): of the four buffers, those of s - 3, s - 2 and s - 1 may be
        // read in those turns.  The sums of dy are one more product, with ones.
        const uint32_t w = wave - C::COMPUTE / 64, pair = w >> 1;
        const int one = C::DY == QGEMM_DT_BF16 ? 0x3F803F80 : 0x3C003C00;
        const v4i ones = v4i{one, one, one, one};
        v4f sum[C::FS] = {};
        // (they have few instructions beside the others' products, and the products wait for them: us, 256 x 256 tiles alone on their CUs, 256
        // steps, 230 -> 203)
        __builtin_amdgcn_s_setprio(1);
        Set r;
        auto add_up = [&](uint32_t t) ALWAYS_INLINE {
            if (sums && t < steps) {
#pragma unroll
                for (int i = 0; i < C::FS; ++i) sum[i] = multiply(ones, fragment(buffer(t), w * C::FS + i), sum[i]);
            }
        };
        // Half of a step's octets: half of dy's and half of the codes', or in the smaller tiles dy in the first turn and the codes in the second.  (us,
        // the second way and then the first: 256 x 256 tiles, 8192 x 8192 x 4096 516 and 492; 128 x 128 tiles, 1999 x 3001 x 1000 35.2 and 36.7.)
        auto half = [&](Set &r, auto which, uint32_t s, auto plain) ALWAYS_INLINE {
            constexpr int W = which.value, N0 = C::EVEN ? W * C::LOAD_N / 2 : W * C::LOAD_N, N1 = C::EVEN ? N0 + C::LOAD_N / 2 : C::LOAD_N;
            constexpr int K0 = C::EVEN ? W * C::LOAD_K / 2 : 0, K1 = C::EVEN ? K0 + C::LOAD_K / 2 : W * C::LOAD_K;
#pragma unroll
            for (int i = N0; i < N1; ++i) stage_n(r, i, buffer(s));
#pragma unroll
            for (int i = K0; i < K1; ++i) stage_k(r, i, buffer(s));
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (plain.value) {
                plain_n(r, N0, N1, from + (s + 2) * kGradStep);
                plain_k(r, K0, K1, from + (s + 2) * kGradStep);
            } else if (s + 2 < steps) {
                request_n(r, N0, N1, from + (s + 2) * kGradStep);
                request_k(r, K0, K1, from + (s + 2) * kGradStep);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        constexpr std::integral_constant<int, 0> first;
        constexpr std::integral_constant<int, 1> second;
        // Steps whose requests are plain have no branch around them, nor have those in front of them: behind one the compiler takes the
        // fewest loads that may be in flight on either way, and waits for more than it has to.
        const uint32_t plain_steps = plain_to > from ? (plain_to - from) / kGradStep : 0;
        uint32_t s = pair, turns = steps + 1;             // the step that is written next; barriers still to come
        auto both = [&](Set &r, auto plain) ALWAYS_INLINE {
            half(r, first, s, plain);
            add_up(s - 3);                                // (in front of the first turn, s = 2: none)
            __syncthreads();
            half(r, second, s, plain);
            add_up(s - 2);
            __syncthreads();
            s += 2;
            turns -= 2;
        };
        auto first_step = [&](auto plain) ALWAYS_INLINE {
            half(r, first, s, plain);
            half(r, second, s, plain);
            s += 2;
            if (pair == 1) {                              // (the even steps are a turn ahead)
                __syncthreads();
                --turns;
            }
        };
        if (plain_steps >= 4) {
            plain_n(r, 0, C::LOAD_N, from + s * kGradStep);
            plain_k(r, 0, C::LOAD_K, from + s * kGradStep);
            __builtin_amdgcn_sched_barrier(0);
            first_step(std::true_type{});
#pragma unroll 1
            while (s + 3 <= plain_steps) both(r, std::true_type{});
        } else {
            if (s < steps) {
                request_n(r, 0, C::LOAD_N, from + s * kGradStep);
                request_k(r, 0, C::LOAD_K, from + s * kGradStep);
            }
            first_step(std::false_type{});
        }
#pragma unroll 1
        while (turns >= 2) both(r, std::false_type{});
        if (turns) {
            add_up(s - 3);
            __syncthreads();
        }
        if (sums) {
#pragma unroll
            for (int i = 0; i < C::FS; ++i)
                if (fg == 0) row_sums[(w * C::FS + i) * 16 + fr] = sum[i][0];
        }
        leave([&](uint32_t pass) ALWAYS_INLINE {
            float *db = split ? (float *)p.room + (size_t)blockIdx.y * grad_plane(p.n, p.cols) : p.db;
            if (pass == 0 && sums && db && tk == 0)
                for (uint32_t i = tid - C::COMPUTE; i < (uint32_t)C::BN; i += 2 * C::COPY)
                    if (n0 + i < p.n) db[n0 + i] = row_sums[i];
        });
        return;
    }

    // ---- The computing waves: products of step t, while the first fragments of step t + 1, which is whole, are on their way: the codes' go where
    // the last products of step t let go of theirs.  (All fragments of a step read during the step in front, in tiles with registers for both, changed
    // no time by more than 2 %.)
    const uint32_t wn = wave / C::WK, wk = wave % C::WK;
    v4f acc[C::FN][C::FK] = {};
    auto fragment_x = [&](const char *of, int g) ALWAYS_INLINE { return fragment(of + C::BN / 64 * C::PANEL, wk * C::FK + g); };
    auto fragment_y = [&](const char *of, int f) ALWAYS_INLINE { return fragment(of, wn * C::FN + f); };
    __syncthreads();
    v4i x[C::FK], y[C::AHEAD + 1];
#pragma unroll
    for (int g = 0; g < C::FK; ++g) x[g] = fragment_x(lds, g);
#pragma unroll
    for (int i = 0; i < C::AHEAD; ++i) y[i] = fragment_y(lds, i);
#pragma unroll 1
    for (uint32_t t = 0; t < steps; ++t) {
        const char *now = buffer(t), *then = buffer(t + 1);
#pragma unroll
        for (int f = 0; f < C::FN; ++f) {
            if (f + C::AHEAD < C::FN) y[(f + C::AHEAD) % (C::AHEAD + 1)] = fragment_y(now, f + C::AHEAD);
#pragma unroll
            for (int g = 0; g < C::FK; ++g) {
                acc[f][g] = multiply(x[g], y[f % (C::AHEAD + 1)], acc[f][g]);
                if (f == C::FN - 1) x[g] = fragment_x(then, g);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < C::AHEAD; ++i) y[i] = fragment_y(then, i);
        __builtin_amdgcn_sched_barrier(0);
        // (nothing of this wave has to arrive anywhere in front of the barrier: the fragments of step t are in its products)
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
    leave([&](uint32_t pass) ALWAYS_INLINE {
        if (wn * (C::BN / C::WN) / C::PASS_ROWS != pass) return;
        const uint32_t row0 = wn * (C::BN / C::WN) % C::PASS_ROWS;
#pragma unroll
        for (int g = 0; g < C::FK; ++g)
#pragma unroll
            for (int f = 0; f < C::FN; ++f)
                *(v4f *)(lds + (row0 + f * 16 + fr) * (C::BK * 4) + ((((wk * C::FK + g) * 4 + fg) ^ fr) << 4)) = acc[f][g];
    });
}
#undef ALWAYS_INLINE

// The slices' sums, in order: a lane has four columns of a row.  Bound by
// memory, and by the trips to it where there are many slices: eight planes in flight instead of four, and dy's sums beside dW's instead of in
// front, took 32 slices of 256 x 256 from 34 us, product and all, to 25, and 16 of 512 x 1024 from 64 to 61
template <int DT>
__global__ void __launch_bounds__(256) weight_grad_join_kernel(const WeightGradArgs p, uint32_t slices) {
    const uint32_t k = (blockIdx.x * 256 + threadIdx.x) * 4;
    const size_t ld = grad_round(p.cols), stride = grad_plane(p.n, p.cols);
    const GradColumns columns(p, k < p.cols ? k : 0);
    for (uint32_t n = blockIdx.y; n < p.n; n += gridDim.y) {
        const bool wants = p.bias || (p.db && k == 0);
        const float *bt = (const float *)p.room + n, *at = (const float *)p.room + grad_round(p.n) + n * ld + (k < p.cols ? k : 0);
        float db = 0.0f;
        v4f sum = {};
        for (uint32_t i0 = 0; i0 < slices; i0 += 8) {
            v4f part[8];
            float of_db[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t s = i0 + i < slices ? i0 + i : 0;
                part[i] = *(const v4f *)(at + s * stride);
                of_db[i] = wants ? bt[s * stride] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i0 + i >= slices) break;
                sum += part[i];
                db += of_db[i];
            }
        }
        if (p.db && k == 0) p.db[n] = db;
        if (k >= p.cols) continue;
        grad_store<DT>(p, columns, n, k, sum, db);
    }
}

}  // namespace qgemm
