// Root-mean-square norm, row by row: h = x + residual as it is stored, rstd = 1 / sqrt(sum h^2 / n + eps), xhat = h rstd, y = xhat w, and y in
// 8 bits under s = max|y| / 127 (448) for a row's 128 columns; and backward, with g = dy w:
//   dx = rstd (g - xhat sum(g xhat) / n) + dh,   dw = sum over rows of dy xhat.
// All sums are fp32.
#pragma once
#include "model.h"
#include "octet.cuh"
#include "quant_kernels.cuh"
#include "training.h"

namespace qgemm {

// v as it reads when it has been stored as dt
__device__ __forceinline__ void as_stored(int dt, float (&v)[8]) {
    if (dt == QGEMM_DT_BF16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(float, (uint32_t)f32_to_bf16_bits(v[e]) << 16);
    } else if (dt == QGEMM_DT_F16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)(_Float16)v[e];
    }
}

// Codes of an octet under the scale of its block, of which m is the largest magnitude's bits: the quantisers' division and rounding.  A block
// with an infinity or a NaN has no scale that could say so but NaN: all of it reads as NaN.
template <int Q_DT>
__device__ __forceinline__ v2i quantized_octet(const float (&v)[8], uint32_t m, float &scale) {
    const bool finite = m < 0x7F800000u;
    const Divisor d = make_divisor(scale_of<Q_DT>(__builtin_bit_cast(float, finite ? m : 0u)), finite);
    scale = finite ? d.s : __builtin_bit_cast(float, 0x7FC00000u);
    v2i q;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const v4f f = finite ? v4f{v[4 * half], v[4 * half + 1], v[4 * half + 2], v[4 * half + 3]} : v4f{0, 0, 0, 0};
        q[half] = quant_piece<QGEMM_DT_F32, Q_DT>(__builtin_bit_cast(v4i, f), d)[0];
    }
    return q;
}
// y, zeros behind the row's end, as codes and scale; all 16 lanes of a block come here
template <int ROW = ROW_ANY>
__device__ __forceinline__ void quantize_octet(const RmsArgs &p, uint32_t row, uint32_t c, const float (&y)[8]) {
    float own[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) own[e] = y[e];
    if (any_repeated<ROW>(c, p.cols))
#pragma unroll
        for (int e = 0; e < 8; ++e) own[e] = e < (int)repeated<ROW>(c, p.cols) ? 0.0f : own[e];
    const uint32_t m = block_max_bits(own);
    if (c >= p.cols) return;
    float scale;
    const v2i q = p.q_dt == QGEMM_DT_I8 ? quantized_octet<QGEMM_DT_I8>(y, m, scale) : quantized_octet<QGEMM_DT_F8E4M3>(y, m, scale);
    store_codes<ROW>((uint8_t *)p.q + (size_t)row * p.ldq, c, p.cols, q);
    if (c % kScaleBlock == 0) p.scales[(size_t)row * p.kb + c / kScaleBlock] = scale;
}

// ---- rows of any length: a workgroup goes over its row twice, the second time out of the caches
__global__ void __launch_bounds__(256) rms_any_kernel(const RmsArgs p) {
    __shared__ float red[2][4][1];
    const uint32_t end = (p.cols + 127) / 128 * 128;               // (whole blocks: the 16 lanes of one stay together)
    int turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const char *x = (const char *)p.x + (size_t)row * p.ldx * dtype_bytes(p.x_dt);
        const char *r = (const char *)p.residual + (size_t)row * p.ldr * dtype_bytes(p.r_dt);
        auto octet = [&](uint32_t c, float (&v)[8]) {
            parameter_octet(x, p.x_dt, c, p.cols, v);
            if (!p.residual) return;
            float more[8];
            parameter_octet(r, p.r_dt, c, p.cols, more);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += more[e];
            as_stored(p.r_dt, v);
        };
        float v[8], sum[1] = {0.0f};
        for (uint32_t c = threadIdx.x * kOctet; c < p.cols; c += 256 * kOctet) {
            octet(c, v);
            if (p.residual) store_octet((char *)p.h + (size_t)row * p.ldh * dtype_bytes(p.r_dt), p.r_dt, c, p.cols, v);
            sum[0] += ((v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3])) + ((v[4] * v[4] + v[5] * v[5]) + (v[6] * v[6] + v[7] * v[7]));
        }
        workgroup_sums<4, 1>(sum, red[turn]);
        const float rstd = 1.0f / __builtin_sqrtf(sum[0] / (float)p.cols + p.eps);
        if (threadIdx.x == 0 && p.rstd) p.rstd[row] = rstd;
        for (uint32_t c = threadIdx.x * kOctet; c < end; c += 256 * kOctet) {
            octet(c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < p.cols ? v[e] * rstd : 0.0f;      // (rstd may be infinite)
            if (p.weight) {
                float w[8];
                parameter_octet(p.weight, p.param_dt, c, p.cols, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= w[e];
            }
            if (p.q) quantize_octet(p, row, c, v);
            if (p.y && c < p.cols) store_octet((char *)p.y + (size_t)row * p.ldy * dtype_bytes(p.y_dt), p.y_dt, c, p.cols, v);
        }
    }
}

// ---- backward
// rows of any length: sums of a row, then its dx, out of the caches
__global__ void __launch_bounds__(256) rms_backward_any_kernel(const RmsBackwardArgs p) {
    __shared__ float red[2][4][1];
    int turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const char *dy = (const char *)p.dy + (size_t)row * p.lddy * dtype_bytes(p.dy_dt), *h = (const char *)p.h + (size_t)row * p.ldh * dtype_bytes(p.h_dt);
        const float rstd = p.rstd[row];
        auto octet = [&](uint32_t c, float (&g)[8], float (&xhat)[8]) {
            parameter_octet(dy, p.dy_dt, c, p.cols, g);
            parameter_octet(h, p.h_dt, c, p.cols, xhat);
#pragma unroll
            for (int e = 0; e < 8; ++e) xhat[e] = c + e < p.cols ? xhat[e] * rstd : 0.0f;
            if (p.weight) {
                float w[8];
                parameter_octet(p.weight, p.param_dt, c, p.cols, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] *= w[e];
            }
        };
        float sum[1] = {0.0f}, g[8], xhat[8];
        for (uint32_t c = threadIdx.x * kOctet; c < p.cols; c += 256 * kOctet) {
            octet(c, g, xhat);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[0] += g[e] * xhat[e];
        }
        workgroup_sums<4, 1>(sum, red[turn]);
        const float b = sum[0] / (float)p.cols;
        for (uint32_t c = threadIdx.x * kOctet; c < p.cols; c += 256 * kOctet) {
            octet(c, g, xhat);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = rstd * (g[e] - xhat[e] * b);
            if (p.dh) {
                parameter_octet((const char *)p.dh + (size_t)row * p.lddh * dtype_bytes(p.dh_dt), p.dh_dt, c, p.cols, xhat);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] += xhat[e];
            }
            store_octet((char *)p.dx + (size_t)row * p.lddx * dtype_bytes(p.dx_dt), p.dx_dt, c, p.cols, g);
        }
    }
}

// column sums over the rows of a slice: 128 columns a workgroup, 16 rows at a time; for rows of any length
__global__ void __launch_bounds__(256) rms_column_sums_kernel(const RmsBackwardArgs p) {
    __shared__ float red[16][128];
    const uint32_t lane = threadIdx.x & 15, sub = threadIdx.x >> 4, c = blockIdx.x * 128 + lane * kOctet;
    float dw[8] = {};
    for (uint32_t row = blockIdx.y * 16 + sub; row < p.rows; row += p.groups * 16) {
        float dy[8], h[8];
        parameter_octet((const char *)p.dy + (size_t)row * p.lddy * dtype_bytes(p.dy_dt), p.dy_dt, c, p.cols, dy);
        parameter_octet((const char *)p.h + (size_t)row * p.ldh * dtype_bytes(p.h_dt), p.h_dt, c, p.cols, h);
        const float rstd = p.rstd[row];
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[e] += dy[e] * (h[e] * rstd);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[sub][lane * 8 + e] = dw[e];
    __syncthreads();
    if (threadIdx.x >= 128 || blockIdx.x * 128 + threadIdx.x >= p.cols) return;
    float s = red[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
    p.partial[(size_t)blockIdx.y * norm_partial_cols(p.cols) + blockIdx.x * 128 + threadIdx.x] = s;
}

// dweight out of the workgroups' sums: 32 columns a workgroup, 64 partial sums at a time, eight of which a lane has in flight, always in the same
// order; x has kMostColumnGroups workgroups at the most, y what that leaves over
__global__ void __launch_bounds__(512) rms_parameter_sums_kernel(const RmsBackwardArgs p) {
    constexpr uint32_t SLICES = 64, DEEP = 8;
    __shared__ v4f red[SLICES][8];
    const size_t stride = norm_partial_cols(p.cols);
    const uint32_t lane = threadIdx.x & 7, sub = threadIdx.x >> 3, c0 = (blockIdx.y * gridDim.x + blockIdx.x) * 32;
    if (c0 >= p.cols) return;
    const float *in = p.partial + c0 + lane * 4;
    v4f s = v4f{0, 0, 0, 0};
    for (uint32_t g = sub; g < p.groups; g += SLICES * DEEP) {
        v4f v[DEEP];
#pragma unroll
        for (uint32_t i = 0; i < DEEP; ++i) {
            const uint32_t at = g + i * SLICES;
            v[i] = *(const v4f *)(in + (size_t)(at < p.groups ? at : g) * stride);
        }
#pragma unroll
        for (uint32_t i = 0; i < DEEP; ++i)
            if (g + i * SLICES < p.groups) s += v[i];
    }
    red[sub][lane] = s;
    __syncthreads();
#pragma unroll
    for (uint32_t half = SLICES / 2; half >= 8; half /= 2) {
        if (sub < half) red[sub][lane] += red[sub + half][lane];
        __syncthreads();
    }
    const uint32_t c = c0 + threadIdx.x;
    if (threadIdx.x >= 32 || c >= p.cols) return;
    const float *at = (const float *)red + threadIdx.x;
    float v = at[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) v += at[i * 32];
    if (p.param_dt == QGEMM_DT_F32) ((float *)p.dweight)[c] = v;
    else ((uint16_t *)p.dweight)[c] = p.param_dt == QGEMM_DT_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}

}  // namespace qgemm
