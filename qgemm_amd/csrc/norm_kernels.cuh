// Layer norm, row by row: mean = sum x / n, var = sum (x - mean)^2 / n, rstd = 1 / sqrt(var + eps), xhat = (x - mean) rstd,
// y = xhat w + b; and backward, with g = dy w:
//   dx = rstd (g - sum g / n - xhat sum(g xhat) / n),   dw = sum over rows of dy xhat,   db = sum over rows of dy.
// xhat comes out of x, mean and rstd, or out of 8-bit codes under 128-column scales.  All sums are fp32.
#pragma once
#include "octet.cuh"
#include "training.h"

namespace qgemm {

// sums of N values over a workgroup of WAVES waves, in every lane; `red` is free again after the next barrier behind this
template <int WAVES, int N>
__device__ __forceinline__ void workgroup_sums(float (&v)[N], float (*red)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<64>(v[i]);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[threadIdx.x >> 6][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = red[0][i];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) v[i] += red[w][i];
        }
    }
}

// x - mean for the elements that the row has, zeros behind it
__device__ __forceinline__ void centre(float (&v)[8], float mean, uint32_t c, uint32_t cols) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? v[e] - mean : 0.0f;
}

// codes and scale of an octet of xhat, which holds zeros behind the row's end; all 16 lanes of a block come here
__device__ __forceinline__ void keep_octet(const NormArgs &p, uint32_t row, uint32_t c, const float (&xhat)[8]) {
    const uint32_t m = block_max_bits(xhat);
    const bool i8 = p.q_dt == QGEMM_DT_I8;
    const PowerOfTwo s = i8 ? power_of_two<QGEMM_DT_I8>(m) : power_of_two<QGEMM_DT_F8E4M3>(m);
    if (c >= p.cols) return;
    const v2i q = i8 ? octet_codes<QGEMM_DT_I8>(xhat, s.inv) : octet_codes<QGEMM_DT_F8E4M3>(xhat, s.inv);
    store_codes((uint8_t *)p.q + (size_t)row * p.ldq, c, p.cols, q);
    if (c % kScaleBlock == 0) p.scales[(size_t)row * p.kb + c / kScaleBlock] = s.s;
}

__device__ __forceinline__ void affine(const NormArgs &p, uint32_t c, const float (&xhat)[8], float (&y)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = xhat[e];
    if (!p.weight) return;
    float w[8];
    parameter_octet(p.weight, p.param_dt, c, p.cols, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= w[e];
    if (!p.bias) return;
    parameter_octet(p.bias, p.param_dt, c, p.cols, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] += w[e];
}

// ---- rows of any length: a workgroup goes over its row three times, the second and third time out of the caches
template <int DT>
__global__ void __launch_bounds__(256) norm_any_kernel(const NormArgs p) {
    __shared__ float red[2][4][1];
    const uint32_t end = (p.cols + 127) / 128 * 128;               // (whole blocks: the 16 lanes of one stay together)
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const char *x = (const char *)p.x + (size_t)row * p.ldx * Octet<DT>::ES;
        float sum[1] = {0.0f};
        for (uint32_t c = threadIdx.x * kOctet; c < p.cols; c += 256 * kOctet) {
            Octet<DT> o;
            float v[8];
            o.request(x, c, p.cols);
            o.settle(c, p.cols);
            o.floats(v);
            sum[0] += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        workgroup_sums<4, 1>(sum, red[0]);
        const float mean = sum[0] / (float)p.cols;
        sum[0] = 0.0f;
        for (uint32_t c = threadIdx.x * kOctet; c < p.cols; c += 256 * kOctet) {
            Octet<DT> o;
            float v[8];
            o.request(x, c, p.cols);
            o.settle(c, p.cols);
            o.floats(v);
            centre(v, mean, c, p.cols);
            sum[0] += ((v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3])) + ((v[4] * v[4] + v[5] * v[5]) + (v[6] * v[6] + v[7] * v[7]));
        }
        workgroup_sums<4, 1>(sum, red[1]);
        const float rstd = 1.0f / __builtin_sqrtf(sum[0] / (float)p.cols + p.eps);
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        for (uint32_t c = threadIdx.x * kOctet; c < end; c += 256 * kOctet) {
            Octet<DT> o;
            float v[8], y[8];
            o.request(x, c, p.cols);
            o.settle(c, p.cols);
            o.floats(v);
            centre(v, mean, c, p.cols);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= rstd;
            if (p.q) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = c + e < p.cols ? v[e] : 0.0f;       // (rstd may be infinite)
                keep_octet(p, row, c, v);
            }
            if (c < p.cols) {
                affine(p, c, v, y);
                store_octet((char *)p.y + (size_t)row * p.ldy * dtype_bytes(p.y_dt), p.y_dt, c, p.cols, y);
            }
        }
    }
}

// ---- backward
// xhat of an octet: out of x, or codes times their scale
template <int X_DT>
struct Normalised {
    static constexpr bool CODES = X_DT == QGEMM_DT_I8 || X_DT == QGEMM_DT_F8E4M3;
    Octet<X_DT> o;
    float scale;
    __device__ __forceinline__ void request(const NormBackwardArgs &p, uint32_t row, uint32_t c) {
        o.request((const char *)p.x + (size_t)row * p.ldx * Octet<X_DT>::ES, c, p.cols);
        if constexpr (CODES) scale = p.scales[(size_t)row * p.kb + (c < p.cols ? c / kScaleBlock : 0)];
    }
    __device__ __forceinline__ void values(const NormBackwardArgs &p, uint32_t c, float mean, float rstd, float (&v)[8]) {
        o.settle(c, p.cols);
        o.floats(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = CODES ? v[e] * scale : (v[e] - mean) * rstd;
    }
};

// rows of any length: sums of a row, then its dx
template <int DY_DT, int X_DT>
__global__ void __launch_bounds__(256) norm_backward_any_kernel(const NormBackwardArgs p) {
    __shared__ float red[2][4][2];
    int turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const char *dy = (const char *)p.dy + (size_t)row * p.lddy * Octet<DY_DT>::ES;
        const float rstd = p.rstd[row], mean = Normalised<X_DT>::CODES ? 0.0f : p.mean[row];
        auto octet = [&](uint32_t c, float (&g)[8], float (&xhat)[8]) {
            Octet<DY_DT> o;
            Normalised<X_DT> n;
            o.request(dy, c, p.cols);
            n.request(p, row, c);
            o.settle(c, p.cols);
            o.floats(g);
            n.values(p, c, mean, rstd, xhat);
            if (p.weight) {
                float w[8];
                parameter_octet(p.weight, p.param_dt, c, p.cols, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] *= w[e];
            }
        };
        float sum[2] = {0.0f, 0.0f}, g[8], xhat[8];
        for (uint32_t c = threadIdx.x * kOctet; c < p.cols; c += 256 * kOctet) {
            octet(c, g, xhat);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (c + e >= p.cols) break;
                sum[0] += g[e];
                sum[1] += g[e] * xhat[e];
            }
        }
        workgroup_sums<4, 2>(sum, red[turn]);
        const float a = sum[0] / (float)p.cols, b = sum[1] / (float)p.cols;
        for (uint32_t c = threadIdx.x * kOctet; c < p.cols; c += 256 * kOctet) {
            octet(c, g, xhat);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = rstd * (g[e] - a - xhat[e] * b);
            store_octet((char *)p.dx + (size_t)row * p.lddx * dtype_bytes(p.dx_dt), p.dx_dt, c, p.cols, g);
        }
    }
}

// column sums over the rows of a slice: 128 columns a workgroup, 16 rows at a time
template <int DY_DT, int X_DT>
__global__ void __launch_bounds__(256) norm_column_sums_kernel(const NormBackwardArgs p) {
    __shared__ float red[16][128];
    const uint32_t lane = threadIdx.x & 15, sub = threadIdx.x >> 4, c = blockIdx.x * 128 + lane * kOctet;
    float dw[8] = {}, db[8] = {};
    for (uint32_t row = blockIdx.y * 16 + sub; row < p.rows; row += p.groups * 16) {
        const float rstd = p.rstd[row], mean = Normalised<X_DT>::CODES ? 0.0f : p.mean[row];
        Octet<DY_DT> o;
        Normalised<X_DT> n;
        float dy[8], xhat[8];
        o.request((const char *)p.dy + (size_t)row * p.lddy * Octet<DY_DT>::ES, c, p.cols);
        n.request(p, row, c);
        o.settle(c, p.cols);
        o.floats(dy);
        n.values(p, c, mean, rstd, xhat);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dw[e] += dy[e] * xhat[e];
            db[e] += dy[e];
        }
    }
    const size_t stride = ((size_t)p.cols + 63) / 64 * 64;
    float *out = p.partial + (size_t)blockIdx.y * 2 * stride;
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) red[sub][lane * 8 + e] = which ? db[e] : dw[e];
        __syncthreads();
        if (threadIdx.x < 128 && blockIdx.x * 128 + threadIdx.x < p.cols) {
            float s = red[0][threadIdx.x];
#pragma unroll
            for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
            out[which * stride + blockIdx.x * 128 + threadIdx.x] = s;
        }
    }
}

// dweight / dbias out of the workgroups' sums: 64 columns a workgroup, always in the same order.  blockIdx.y: which of the two
__global__ void __launch_bounds__(256) norm_parameter_sums_kernel(const NormBackwardArgs p) {
    __shared__ float red[16][64];
    const size_t stride = ((size_t)p.cols + 63) / 64 * 64;
    const uint32_t lane = threadIdx.x & 15, sub = threadIdx.x >> 4, which = blockIdx.y;
    void *out = which ? p.dbias : p.dweight;
    if (!out) return;
    const float *in = p.partial + which * stride + (size_t)blockIdx.x * 64 + lane * 4;
    v4f s = v4f{0, 0, 0, 0};
    for (uint32_t g = sub; g < p.groups; g += 16) s += *(const v4f *)(in + (size_t)g * 2 * stride);
    *(v4f *)&red[sub][lane * 4] = s;
    __syncthreads();
    const uint32_t c = blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x >= 64 || c >= p.cols) return;
    float v = red[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 16; ++i) v += red[i][threadIdx.x];
    if (p.param_dt == QGEMM_DT_F32) ((float *)out)[c] = v;
    else ((uint16_t *)out)[c] = p.param_dt == QGEMM_DT_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}

}  // namespace qgemm
