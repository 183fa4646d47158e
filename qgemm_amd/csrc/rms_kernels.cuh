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

// A lane's octets of the weight, of any type, as they come from memory (ones where there is none), and as numbers.  (Registers for fp32, and one branch for all
// octets: the kernels would be twice as many with the weight's type among their own.)
template <int TYPE, int P, int ROW, class Args>
__device__ __forceinline__ void weight_octets(const Args &p, uint32_t first, uint32_t step, uint32_t (&w)[P][8]) {
    Octet<TYPE> all[P];
#pragma unroll
    for (int i = 0; i < P; ++i) all[i].template request<ROW>(p.weight, first + i * step, p.cols);
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) w[i][k] = k < Octet<TYPE>::DW ? all[i].w[k % Octet<TYPE>::DW] : 0;
}
// columns first + i step
template <int P, int ROW, class Args>
__device__ __forceinline__ void weight_request(const Args &p, uint32_t first, uint32_t step, uint32_t (&w)[P][8]) {
    if (!p.weight) {
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) w[i][k] = 0x3F800000u;
    } else if (p.param_dt == QGEMM_DT_F32) {
        weight_octets<QGEMM_DT_F32, P, ROW>(p, first, step, w);
    } else {
        weight_octets<QGEMM_DT_BF16, P, ROW>(p, first, step, w);          // (16 bits, whichever)
    }
}
template <class Args>
__device__ __forceinline__ void weight_floats(const Args &p, const uint32_t (&w)[8], float (&f)[8]) {
    const bool wide = !p.weight || p.param_dt == QGEMM_DT_F32, bf16 = p.param_dt == QGEMM_DT_BF16;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t half = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
        const float narrow = bf16 ? __builtin_bit_cast(float, half << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)half);
        f[e] = wide ? __builtin_bit_cast(float, w[e]) : narrow;
    }
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

// ---- rows in registers: GROUP threads hold a row, P octets each, and read x and the residual once.  RES: type of the residual, -1 where there is none.
// Bound by memory: 6144 x 7168 bf16 with residual, y and int8 codes 80 us in a trace, 4.95 TB/s, the rate of a copy; 107 in two passes out of the caches
// (rms_any_kernel).  1 x 7168: 5.5, a trip to memory, a barrier, the division by the scale and the stores.
template <int DT, int RES, int GROUP, int P, int ROW>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) rms_rows_kernel(const RmsArgs p) {
    constexpr int THREADS = GROUP < 256 ? 256 : GROUP, ROWS = THREADS / GROUP, WAVES = GROUP / 64, LANES = GROUP < 64 ? GROUP : 64;
    constexpr int H_DT = RES < 0 ? DT : RES;
    const uint32_t t = threadIdx.x % GROUP, cols = p.cols;
    auto column = [&](int i) { return (i * GROUP + t) * kOctet; };
    int turn = 0;
    for (uint32_t first = blockIdx.x * ROWS; first < p.rows; first += gridDim.x * ROWS, turn ^= 1) {
        const uint32_t row = ROWS == 1 ? first : first + threadIdx.x / GROUP;
        const bool in_rows = ROWS == 1 || row < p.rows;
        const size_t at = in_rows ? row : p.rows - 1;
        Octet<DT> x[P];
        Octet<H_DT> h[P];
        uint32_t w[P][8];
        const char *xr = (const char *)p.x + at * p.ldx * Octet<DT>::ES, *rr = (const char *)p.residual + at * p.ldr * Octet<H_DT>::ES;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            x[i].template request<ROW>(xr, column(i), cols);
            if constexpr (RES >= 0) h[i].template request<ROW>(rr, column(i), cols);
        }
        weight_request<P, ROW>(p, t * kOctet, GROUP * kOctet, w);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float v[8];
            x[i].template settle<ROW>(column(i), cols);
            x[i].floats(v);
            if constexpr (RES >= 0) {
                float r[8];
                h[i].template settle<ROW>(column(i), cols);
                h[i].floats(r);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += r[e];
                h[i].take(v);
                h[i].hold();
                h[i].floats(v);
                if (in_rows && column(i) < cols)
                    h[i].template put<ROW>((char *)p.h + at * p.ldh * Octet<H_DT>::ES, column(i), cols);
            } else {
                h[i] = x[i];
                h[i].hold();
            }
            if (any_repeated<ROW>(column(i), cols))
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = e < (int)repeated<ROW>(column(i), cols) ? 0.0f : v[e];
            sum += ((v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3])) + ((v[4] * v[4] + v[5] * v[5]) + (v[6] * v[6] + v[7] * v[7]));
            __builtin_amdgcn_sched_barrier(0);
        }
        sum = lanes_sum<LANES>(sum);
        if constexpr (WAVES > 1) {
            __shared__ float red[2][WAVES];
            if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = sum;
            __syncthreads();
            sum = red[turn][0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) sum += red[turn][i];
        }
        const float rstd = 1.0f / __builtin_sqrtf(sum / (float)cols + p.eps);
        if (t == 0 && in_rows && p.rstd) p.rstd[row] = rstd;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const uint32_t c = column(i);
            float v[8], f[8];
            h[i].hold();
            h[i].floats(v);
            weight_floats(p, w[i], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c < cols ? v[e] * rstd * f[e] : 0.0f;
            if (p.q && in_rows) quantize_octet<ROW>(p, row, c, v);
            if (p.y && in_rows && c < cols) store_octet<ROW>((char *)p.y + at * p.ldy * dtype_bytes(p.y_dt), p.y_dt, c, cols, v);
            __builtin_amdgcn_sched_barrier(0);
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

// Rows in registers: GROUP threads hold a row of dy and of h, P octets each; a workgroup goes over its rows with the next one's loads in flight, and
// keeps the sums of its columns in registers until the end.  S_DT: type of h and dh; DH: there is a dh, which is wanted at the end of a row's work
// and requested at its beginning.  Bound by memory: 8192 x 4096 bf16 with dh 42 us, 6.4 TB/s, part of it out of the last-level cache, and 4.5 for the workgroups'
// sums; 77 in two passes over the rows and one for the columns.  1999 x 3001 fp16 13.7 with both launches, 25 before: four rows a workgroup, one in flight.  With 512 threads of four octets
// and fp32 h a part of the registers is in scratch (60 - 204 bytes a lane): 2048 x 14336 fp32 83 us, with dh 135.
template <int DY_DT, int S_DT, bool DH, int GROUP, int P, int ROW>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) rms_backward_rows_kernel(const RmsBackwardArgs p) {
    constexpr int THREADS = GROUP < 256 ? 256 : GROUP, ROWS = THREADS / GROUP, WAVES = GROUP / 64, LANES = GROUP < 64 ? GROUP : 64;
    const uint32_t t = threadIdx.x % GROUP, sub = ROWS == 1 ? 0 : threadIdx.x / GROUP, cols = p.cols;
    auto column = [&](int i) { return (i * GROUP + t) * kOctet; };
    struct Row {
        Octet<DY_DT> dy[P];
        Octet<S_DT> h[P];
        float rstd;
    };
    auto row_of = [&](uint32_t first) {
        const uint32_t row = first + sub;
        return ROWS == 1 || row < p.rows ? row : p.rows - 1;
    };
    auto fetch = [&](Row &r, uint32_t first) {
        const size_t row = row_of(first);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            r.dy[i].template request<ROW>((const char *)p.dy + row * p.lddy * Octet<DY_DT>::ES, column(i), cols);
            r.h[i].template request<ROW>((const char *)p.h + row * p.ldh * Octet<S_DT>::ES, column(i), cols);
        }
        r.rstd = p.rstd[row];
    };
    float w[P][8], dw[P][8] = {};
    {
        uint32_t bits[P][8];
        weight_request<P, ROW>(p, t * kOctet, GROUP * kOctet, bits);
#pragma unroll
        for (int i = 0; i < P; ++i) weight_floats(p, bits[i], w[i]);
    }
    Row next;
    const uint32_t stride = gridDim.x * ROWS;
    fetch(next, blockIdx.x * ROWS);
    int turn = 0;
    for (uint32_t first = blockIdx.x * ROWS; first < p.rows; first += stride, turn ^= 1) {
        Row r = next;
        const bool in_rows = ROWS == 1 || first + sub < p.rows;
        Octet<S_DT> dh[DH ? P : 1];
        if constexpr (DH)
#pragma unroll
            for (int i = 0; i < P; ++i) dh[i].template request<ROW>((const char *)p.dh + (size_t)row_of(first) * p.lddh * Octet<S_DT>::ES, column(i), cols);
        if (p.rows - first > stride) fetch(next, first + stride);
        float b = 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float g[8], xhat[8];
            r.dy[i].template settle<ROW>(in_rows ? column(i) : cols, cols);
            r.h[i].template settle<ROW>(column(i), cols);
            r.dy[i].hold();
            r.h[i].hold();
            r.dy[i].floats(g);
            r.h[i].floats(xhat);
            const float by = column(i) < cols ? r.rstd : 0.0f;      // (0 times an infinite rstd is no 0)
            if (any_repeated<ROW>(column(i), cols))
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = e < (int)repeated<ROW>(column(i), cols) ? 0.0f : g[e];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float product = g[e] * (xhat[e] * by);
                dw[i][e] += product;
                b += product * w[i][e];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        b = lanes_sum<LANES>(b);
        if constexpr (WAVES > 1) {
            __shared__ float red[2][WAVES];
            if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = b;
            __syncthreads();
            b = red[turn][0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) b += red[turn][i];
        }
        b /= (float)cols;
        char *dx = (char *)p.dx + (size_t)(first + sub) * p.lddx * dtype_bytes(p.dx_dt);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float g[8], xhat[8];
            r.dy[i].hold();
            r.h[i].hold();
            r.dy[i].floats(g);
            r.h[i].floats(xhat);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = r.rstd * (g[e] * w[i][e] - xhat[e] * r.rstd * b);
            if constexpr (DH) {
                float more[8];
                dh[i].template settle<ROW>(column(i), cols);
                dh[i].floats(more);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] += more[e];
            }
            if (in_rows && column(i) < cols) store_octet<ROW>(dx, p.dx_dt, column(i), cols, g);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (!p.dweight) return;
    float *out = p.partial + (size_t)blockIdx.x * norm_partial_cols(cols);
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (column(i) >= cols) continue;
            if (const uint32_t before = repeated<ROW>(column(i), cols)) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e >= (int)before) out[column(i) - before + e] = dw[i][e];
                continue;
            }
            v4f *at = (v4f *)(out + column(i));
            at[0] = v4f{dw[i][0], dw[i][1], dw[i][2], dw[i][3]};
            at[1] = v4f{dw[i][4], dw[i][5], dw[i][6], dw[i][7]};
        }
    } else {
        __shared__ float fold[THREADS * 8];                     // [ROWS][GROUP * 8]
#pragma unroll
        for (int i = 0; i < P; ++i) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int before = (int)repeated<ROW>(column(i), cols);
                if (ROW != ROW_RAGGED || e >= before) fold[threadIdx.x * 8 + e - before] = dw[i][e];
            }
            __syncthreads();
#pragma unroll 1
            for (uint32_t c = threadIdx.x; c < GROUP * 8; c += THREADS) {
                float s = fold[c];
#pragma unroll
                for (int k = 1; k < ROWS; ++k) s += fold[k * GROUP * 8 + c];
                if (i * GROUP * 8 + c < cols) out[i * GROUP * 8 + c] = s;
            }
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
