// Weight gradient of a linear layer out of an activation in 8 bits: dW[n, k] = sum over rows m of dy[m, n] v[m, k] with
// v = q s, s one scale for a row's 128 columns, and db[n] = sum over m of dy[m, n].  Where q holds a norm's xhat, and the layer's input
// was xhat w + b, the two vectors leave the sum: dW[n, k] = w[k] sum dy xhat + b[k] db[n], and the product reads codes alone.
//
// Both operands lie with their rows along the contraction, as they were written.  A step is 64 rows: dy goes from memory through
// registers into LDS as it is, codes are widened to 16 bits on the way (exact where scales are powers of two), and the matrix
// cores' operands, which run along the rows, are taken out of both with transposing reads.  fp32 accumulators.
#pragma once
#include "octet.cuh"
#include "training.h"

namespace qgemm {

typedef short wg_v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) wg_v4s lds_quad;

constexpr int kGradStep = 64;          // rows of a step

// The tile of a workgroup: BN x BK of dW, WN x WK waves
template <int DY_DT, int Q_DT, int BN_, int BK_, int WN_, int WK_>
struct GradCfg {
    static constexpr int DY = DY_DT, Q = Q_DT, BN = BN_, BK = BK_, WN = WN_, WK = WK_;
    static constexpr int THREADS = 64 * WN * WK;
    static constexpr int FN = BN / WN / 16, FK = BK / WK / 16;                     // fragments of a wave
    static constexpr int LOAD_N = kGradStep * BN / 8 / THREADS, LOAD_K = kGradStep * BK / 8 / THREADS;      // octets of a lane and step
    static constexpr int PANEL = kGradStep * 128;                                  // 64 columns of 16 bits
    static constexpr int STAGE = (BN + BK) / 64 * PANEL;
    static constexpr int LDS = 2 * STAGE;
    static_assert(BN % 64 == 0 && BK % 64 == 0 && LOAD_N >= 1 && LOAD_K >= 1, "whole panels");
};

// 16-byte chunk c of row k of a panel lies in slot c ^ grad_swizzle(k): the rows that a transposing read takes together, k0 .. k0 + 3 of
// two groups of lanes eight rows apart, lie in different banks
__device__ __forceinline__ constexpr int grad_swizzle(int k) { return (((k >> 1) & 1) << 1) | (((k >> 3) & 1) << 2); }

template <class C>
__global__ void __launch_bounds__(C::THREADS) weight_grad_kernel(const WeightGradArgs p, const TileMap map) {
    extern __shared__ __align__(16) char lds[];
    typedef Octet<C::DY> OctetN;
    typedef Octet<C::Q> OctetK;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wn = wave / C::WK, wk = wave % C::WK;
    uint32_t tn, tk;
    tile_map(blockIdx.x, map, tn, tk);
    const uint32_t n0 = tn * C::BN, k0 = tk * C::BK;

    // ---- memory to registers
    OctetN on[C::LOAD_N];
    OctetK ok[C::LOAD_K];
    float scale[C::LOAD_K];
    auto request = [&](uint32_t m0) {
#pragma unroll
        for (int i = 0; i < C::LOAD_N; ++i) {
            const uint32_t at = i * C::THREADS + tid, m = m0 + at / (C::BN / 8), c = n0 + at % (C::BN / 8) * 8;
            on[i].request((const char *)p.dy + (size_t)(m < p.rows ? m : p.rows - 1) * p.lddy * OctetN::ES, c, p.n);
        }
#pragma unroll
        for (int i = 0; i < C::LOAD_K; ++i) {
            const uint32_t at = i * C::THREADS + tid, m = m0 + at / (C::BK / 8), c = k0 + at % (C::BK / 8) * 8;
            const size_t row = m < p.rows ? m : p.rows - 1;
            ok[i].request((const char *)p.q + row * p.ldq, c, p.cols);
            scale[i] = p.scales[row * p.kb + (c < p.cols ? c / kScaleBlock : 0)];
        }
    };
    // ---- registers to LDS
    auto place = [&](char *panels, uint32_t k, uint32_t chunk, v4i v) {
        *(v4i *)(panels + (chunk >> 3) * C::PANEL + k * 128 + (((chunk & 7) ^ grad_swizzle(k)) << 4)) = v;
    };
    auto stage = [&](uint32_t m0, char *to) {
#pragma unroll
        for (int i = 0; i < C::LOAD_N; ++i) {
            const uint32_t at = i * C::THREADS + tid, k = at / (C::BN / 8), chunk = at % (C::BN / 8);
            on[i].settle(m0 + k < p.rows ? n0 + chunk * 8 : p.n, p.n);
            place(to, k, chunk, v4i{(int)on[i].w[0], (int)on[i].w[1], (int)on[i].w[2], (int)on[i].w[3]});
        }
#pragma unroll
        for (int i = 0; i < C::LOAD_K; ++i) {
            const uint32_t at = i * C::THREADS + tid, k = at / (C::BK / 8), chunk = at % (C::BK / 8);
            const bool in = m0 + k < p.rows;
            float v[8];
            ok[i].settle(in ? k0 + chunk * 8 : p.cols, p.cols);
            ok[i].floats(v);
            const float s = in ? scale[i] : 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= s;
            const v2i a = C::DY == QGEMM_DT_BF16 ? pack4_bf16(v[0], v[1], v[2], v[3]) : pack4_f16(v[0], v[1], v[2], v[3]);
            const v2i b = C::DY == QGEMM_DT_BF16 ? pack4_bf16(v[4], v[5], v[6], v[7]) : pack4_f16(v[4], v[5], v[6], v[7]);
            place(to + C::BN / 64 * C::PANEL, k, chunk, v4i{a[0], a[1], b[0], b[1]});
        }
    };
    // ---- LDS to operands: columns 16 x .. 16 x + 15 along rows 32 half .. 32 half + 31.  Lane j of a group of 16 supplies the address of
    // 8 bytes of row j >> 2 and receives column j of the four rows
    const int fr = lane & 15, fg = lane >> 4;
    const int lane_at = (8 * fg + (fr >> 2)) * 128 + 16 * (((fr >> 1) & 1) | grad_swizzle(8 * fg + (fr >> 2))) + 8 * (fr & 1);
    auto fragment = [&](const char *panels, int x, int half) {
        const char *at = panels + (x >> 2) * C::PANEL + half * 32 * 128 + (lane_at ^ ((x & 3) * 32));
        const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad *)at));
        const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad *)(at + 4 * 128)));
        return v4i{lo[0], lo[1], hi[0], hi[1]};
    };
    auto multiply = [&](v4i x, v4i y, v4f c) {
        if constexpr (C::DY == QGEMM_DT_BF16)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x), __builtin_bit_cast(v8bf, y), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0, 0);
    };

    // the sums of dy are one more product, with ones; the waves that share rows of the tile share its fragments out
    const bool sums = (p.db && tk == 0) || p.bias;
    constexpr int FS = (C::FN + C::WK - 1) / C::WK;
    const int one = C::DY == QGEMM_DT_BF16 ? 0x3F803F80 : 0x3C003C00;
    const v4i ones = v4i{one, one, one, one};
    v4f acc[C::FN][C::FK] = {}, row_sum[FS] = {};
    if (p.rows) {
        request(0);
        stage(0, lds);
    }
    int at = 0;
    for (uint32_t m0 = 0; m0 < p.rows; m0 += kGradStep, at ^= 1) {
        __syncthreads();
        const bool more = m0 + kGradStep < p.rows;
        if (more) request(m0 + kGradStep);
        const char *now = lds + at * C::STAGE;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            v4i x[C::FK], y[C::FN];
#pragma unroll
            for (int f = 0; f < C::FK; ++f) x[f] = fragment(now + C::BN / 64 * C::PANEL, wk * C::FK + f, half);
#pragma unroll
            for (int f = 0; f < C::FN; ++f) y[f] = fragment(now, wn * C::FN + f, half);
#pragma unroll
            for (int f = 0; f < C::FN; ++f)
#pragma unroll
                for (int g = 0; g < C::FK; ++g) acc[f][g] = multiply(x[g], y[f], acc[f][g]);
            if (sums) {
#pragma unroll
                for (int f = 0; f < C::FN; ++f)
                    if ((uint32_t)(f % C::WK) == wk) row_sum[f / C::WK] = multiply(ones, y[f], row_sum[f / C::WK]);
            }
        }
        if (more) stage(m0 + kGradStep, lds + (at ^ 1) * C::STAGE);
    }

    // ---- a lane has four neighbouring columns of dW of one row in every fragment
    float *row_sums = (float *)lds;
    if (sums) {
        __syncthreads();
#pragma unroll
        for (int f = 0; f < C::FN; ++f)
            if ((uint32_t)(f % C::WK) == wk && fg == 0) row_sums[(wn * C::FN + f) * 16 + fr] = row_sum[f / C::WK][0];
        __syncthreads();
        if (p.db && tk == 0)
            for (uint32_t i = tid; i < (uint32_t)C::BN; i += C::THREADS)
                if (n0 + i < p.n) p.db[n0 + i] = row_sums[i];
    }
    auto parameter = [&](const void *v, uint32_t k) {
        if (p.param_dt == QGEMM_DT_F32) return ((const float *)v)[k];
        const uint16_t h = ((const uint16_t *)v)[k];
        return p.param_dt == QGEMM_DT_BF16 ? __builtin_bit_cast(float, (uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
    };
#pragma unroll
    for (int g = 0; g < C::FK; ++g) {
        const uint32_t k = k0 + (wk * C::FK + g) * 16 + fg * 4;
        if (k >= p.cols) continue;
        float w[4], b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t at_k = k + e < p.cols ? k + e : p.cols - 1;
            w[e] = p.weight ? parameter(p.weight, at_k) : 1.0f;
            b[e] = p.bias ? parameter(p.bias, at_k) : 0.0f;
        }
#pragma unroll
        for (int f = 0; f < C::FN; ++f) {
            const uint32_t i = (wn * C::FN + f) * 16 + fr, n = n0 + i;
            if (n >= p.n) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = p.weight ? acc[f][g][e] * w[e] : acc[f][g][e];
            if (p.bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += b[e] * row_sums[i];
            }
            store_out4(p.dw, (size_t)n * p.lddw + k, v, p.dw_dt, (int)(p.cols - k < 4 ? p.cols - k : 4));
        }
    }
}

}  // namespace qgemm
