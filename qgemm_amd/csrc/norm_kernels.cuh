// Layer norm, row by row: mean = sum x / n, var = sum (x - mean)^2 / n, rstd = 1 / sqrt(var + eps), xhat = (x - mean) rstd,
// y = xhat w + b; and backward, with g = dy w:
//   dx = rstd (g - sum g / n - xhat sum(g xhat) / n),   dw = sum over rows of dy xhat,   db = sum over rows of dy.
// xhat comes out of x, mean and rstd, or out of 8-bit codes under 128-column scales.  All sums are fp32.
#pragma once
#include "octet.cuh"
#include "training.h"

namespace qgemm {

// x - mean for the elements that the row has, zeros behind it
__device__ __forceinline__ void centre(float (&v)[8], float mean, uint32_t c, uint32_t cols) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? v[e] - mean : 0.0f;
}

// codes and scale of an octet of xhat, which holds zeros behind the row's end; all 16 lanes of a block come here
template <int ROW = ROW_ANY>
__device__ __forceinline__ void keep_octet(const NormArgs &p, uint32_t row, uint32_t c, const float (&xhat)[8]) {
    float own[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) own[e] = xhat[e];
    if (any_repeated<ROW>(c, p.cols))
#pragma unroll
        for (int e = 0; e < 8; ++e) own[e] = e < (int)repeated<ROW>(c, p.cols) ? 0.0f : own[e];
    const uint32_t m = block_max_bits(own);
    const bool i8 = p.q_dt == QGEMM_DT_I8;
    const PowerOfTwo s = i8 ? power_of_two<QGEMM_DT_I8>(m) : power_of_two<QGEMM_DT_F8E4M3>(m);
    if (c >= p.cols) return;
    const v2i q = i8 ? octet_codes<QGEMM_DT_I8>(xhat, s.inv) : octet_codes<QGEMM_DT_F8E4M3>(xhat, s.inv);
    store_codes<ROW>((uint8_t *)p.q + (size_t)row * p.ldq, c, p.cols, q);
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

// ---- rows of any length: a workgroup goes over its row three times, the second and third time out of the caches.  Rows that the registers of
// 512 threads do not hold, or of a few elements; 8192 x 20000 bf16 218 us, 3.0 TB/s, bound by the trips to the caches.  And parameters whose type is
// neither x's nor fp32, at any width (us, parameters of x's type or fp32 / of another: 4096 x 7168 fp32 with bf16 42 / 63, bf16 with fp16 26 / 36,
// 1 x 7168 4.1 / 7.2; on short rows most of the 256 threads have nothing to do: 131072 x 128 bf16 with fp16 14 / 184).
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

// ---- rows in registers: GROUP threads hold a row, P octets each, and read it once.
// Statistics of a wave's part are exact to two passes (sum, then squares about its own mean), both in registers; parts of a row meet
// once: with n_w elements, mean m_w and squares M_w of part w, sum (x - mean)^2 = sum M_w + n_w (m_w - mean)^2, which cancels nothing.
// SAME: the parameters have x's type, else they are fp32.  AHEAD: an octet of them is requested in front of the one that is being worked
// on, the first with the row: half a trip to memory less for a row by itself, and registers that many rows want for more waves
// (us, without / with: 1 x 7168 bf16 4.3 / 3.9, 6144 x 7168 kept 42.5 / 49.5 on the same buffers again and 54.5 / 62.5 on others each time, not kept
// 35.0 / 34.5; not all of them: 16384 x 2048 26.0 / 24.1).  ROW: see RowKind.
template <int DT, int GROUP, int P, bool SAME, bool AHEAD, int ROW>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) norm_rows_kernel(const NormArgs p) {
    constexpr int THREADS = GROUP < 256 ? 256 : GROUP, ROWS = THREADS / GROUP, WAVES = GROUP / 64, LANES = GROUP < 64 ? GROUP : 64;
    typedef Octet<SAME ? DT : QGEMM_DT_F32> Param;
    const uint32_t t = threadIdx.x % GROUP, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), cols = p.cols;
    const float n = (float)cols;
    auto column = [&](int i) { return (i * GROUP + t) * kOctet; };
    int turn = 0;
    for (uint32_t first = blockIdx.x * ROWS; first < p.rows; first += gridDim.x * ROWS, turn ^= 1) {
        const uint32_t row = ROWS == 1 ? first : first + threadIdx.x / GROUP;
        const bool in_rows = ROWS == 1 || row < p.rows;
        const char *x = (const char *)p.x + (size_t)(in_rows ? row : p.rows - 1) * p.ldx * Octet<DT>::ES;
        Octet<DT> o[P];
        Param w[P], b[P];
        auto parameters = [&](int i) {
            if (p.weight) w[i].template request<ROW>(p.weight, column(i), cols);
            if (p.bias) b[i].template request<ROW>(p.bias, column(i), cols);
        };
#pragma unroll
        for (int i = 0; i < P; ++i) o[i].template request<ROW>(x, column(i), cols);
        if (AHEAD) parameters(0);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float v[8];
            o[i].template settle<ROW>(column(i), cols);
            o[i].hold();
            o[i].floats(v);
            if (any_repeated<ROW>(column(i), cols))
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = e < (int)repeated<ROW>(column(i), cols) ? 0.0f : v[e];
            sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            __builtin_amdgcn_sched_barrier(0);
        }
        sum = lanes_sum<LANES>(sum);
        float part = n;                                      // elements of the row in this wave
        if constexpr (WAVES > 1) {
            uint32_t have = 0;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const uint32_t from = (i * GROUP + wave * 64) * kOctet;
                have += from < cols ? (cols - from < 512 ? cols - from : 512) : 0;
            }
            part = (float)have;
        }
        float mean = WAVES > 1 && part == 0.0f ? 0.0f : sum / part, squares = 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const uint32_t c = column(i);
            float v[8];
            o[i].hold();
            o[i].floats(v);
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] -= mean;
            if (any_repeated<ROW>(c, cols))
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = e < (int)repeated<ROW>(c, cols) ? 0.0f : v[e];
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[e] * v[e];
            squares += c < cols ? s : 0.0f;
            __builtin_amdgcn_sched_barrier(0);
        }
        squares = lanes_sum<LANES>(squares);
        if constexpr (WAVES > 1) {
            __shared__ float red[2][WAVES][3];
            if ((threadIdx.x & 63) == 0) {
                red[turn][wave][0] = sum;
                red[turn][wave][1] = squares;
                red[turn][wave][2] = part;
            }
            __syncthreads();
            float all = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) all += red[turn][i][0];
            mean = all / n;
            squares = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                const float k = red[turn][i][2], d = k == 0.0f ? 0.0f : red[turn][i][0] / k - mean;
                squares += red[turn][i][1] + k * (d * d);
            }
        }
        const float rstd = 1.0f / __builtin_sqrtf(squares / n + p.eps);
        if (t == 0 && in_rows) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        char *y = (char *)p.y + (size_t)row * p.ldy * dtype_bytes(p.y_dt);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const uint32_t c = column(i);
            float v[8];
            if (AHEAD && i + 1 < P) parameters(i + 1);
            o[i].hold();
            o[i].floats(v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (v[e] - mean) * rstd;
            if (p.q) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = c < cols ? v[e] : 0.0f;
                if (in_rows) keep_octet<ROW>(p, row, c, v);
            }
            if (in_rows && c < cols) {
                float f[8];
                if (p.weight) {
                    if (!AHEAD) w[i].template request<ROW>(p.weight, c, cols);
                    w[i].template settle<ROW>(c, cols);
                    w[i].floats(f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= f[e];
                }
                if (p.bias) {
                    if (!AHEAD) b[i].template request<ROW>(p.bias, c, cols);
                    b[i].template settle<ROW>(c, cols);
                    b[i].floats(f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += f[e];
                }
                store_octet<ROW>(y, p.y_dt, c, cols, v);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// ---- backward
// xhat of an octet: out of x, or codes times the scale of column c's block
template <int X_DT>
struct Normalised {
    static constexpr bool CODES = X_DT == QGEMM_DT_I8 || X_DT == QGEMM_DT_F8E4M3;
    Octet<X_DT> o;
    float scale;
    template <int ROW = ROW_ANY>
    __device__ __forceinline__ void request(const NormBackwardArgs &p, uint32_t row, uint32_t c) {
        o.template request<ROW>((const char *)p.x + (size_t)row * p.ldx * Octet<X_DT>::ES, c, p.cols);
        if constexpr (CODES) scale = p.scales[(size_t)row * p.kb + (c < p.cols ? c / kScaleBlock : 0)];
    }
    template <int ROW = ROW_ANY>
    __device__ __forceinline__ void settle(uint32_t c, uint32_t cols) {
        o.template settle<ROW>(c, cols);
    }
    __device__ __forceinline__ void values(float mean, float rstd, float (&v)[8]) const {
        o.floats(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = CODES ? v[e] * scale : (v[e] - mean) * rstd;
    }
};

// rows of any length: sums of a row, then its dx, out of the caches (8192 x 20000 bf16 283 us, 3.5 TB/s)
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
            n.settle(c, p.cols);
            n.values(mean, rstd, xhat);
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

// Rows in registers: GROUP threads hold a row of dy and of x, P octets each; a workgroup goes over its rows with the next one's
// loads in flight, and keeps the sums of its columns in registers until the end: dy and x are read once.  Bound by memory: 8192 x 4096 bf16 36 us,
// 5.7 TB/s, and 4.5 for the workgroups' sums; with a second reading for the columns it was 76.  1999 x 3001 fp16 out of e4m3 14.4, 2.1 TB/s: eight
// rows a workgroup, each at an odd address, and one in flight.  Four octets (8193 - 16384 columns) are more than the registers hold beside the next
// row: 12 - 320 bytes a lane in scratch; 4096 x 14336 bf16 79 us with the sums' launch, 69 at the rate of a copy.
// EDGE: out of codes, rows that end one to seven columns into a block of 128.  What their last octet repeats lies under the scale of the block in
// front, and dx is the same from both lanes that write it only where both take that one.  A form of its own, because the scale in flight costs
// other ragged rows 2 - 9 % (us, without / with: 1999 x 3001 fp16 out of e4m3 17.4 / 18.3, 4096 x 8237 bf16 out of int8 57.2 / 62.8; loaded where
// it is wanted 17.8 and 59.8), and storing the last octet's own elements one by one holds back the next row (8192 x 4100 73.6, this way 55).
template <int DY_DT, int X_DT, int GROUP, int P, int ROW, bool EDGE = false>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) norm_backward_rows_kernel(const NormBackwardArgs p) {
    constexpr int THREADS = GROUP < 256 ? 256 : GROUP, ROWS = THREADS / GROUP, WAVES = GROUP / 64, LANES = GROUP < 64 ? GROUP : 64;
    constexpr bool CODES = Normalised<X_DT>::CODES;
    const uint32_t t = threadIdx.x % GROUP, sub = ROWS == 1 ? 0 : threadIdx.x / GROUP, cols = p.cols;
    const float n = (float)cols;
    const bool sums = p.dweight || p.dbias;
    auto column = [&](int i) { return (i * GROUP + t) * kOctet; };
    struct Row {
        Octet<DY_DT> dy[P];
        Normalised<X_DT> x[P];
        float mean, rstd, front;                             // front (EDGE): scale of the row's last block but one
    };
    auto fetch = [&](Row &r, uint32_t first) {
        uint32_t row = first + sub;
        if (ROWS > 1) row = row < p.rows ? row : p.rows - 1;
        const char *dy = (const char *)p.dy + (size_t)row * p.lddy * Octet<DY_DT>::ES;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            r.dy[i].template request<ROW>(dy, column(i), cols);
            r.x[i].template request<ROW>(p, row, column(i));
        }
        r.rstd = p.rstd[row];
        r.mean = CODES ? 0.0f : p.mean[row];
        if constexpr (EDGE) r.front = p.scales[(size_t)row * p.kb + (cols - kOctet) / kScaleBlock];
    };
    float w[P][8], dw[P][8] = {}, db[P][8] = {};
#pragma unroll
    for (int i = 0; i < P; ++i) {
        if (p.weight) parameter_octet<ROW>(p.weight, p.param_dt, column(i), cols, w[i]);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) w[i][e] = 1.0f;
    }
    Row next;
    const uint32_t stride = gridDim.x * ROWS;
    fetch(next, blockIdx.x * ROWS);
    int turn = 0;
    for (uint32_t first = blockIdx.x * ROWS; first < p.rows; first += stride, turn ^= 1) {
        Row r = next;
        const bool in_rows = ROWS == 1 || first + sub < p.rows;
        if (p.rows - first > stride) fetch(next, first + stride);
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float g[8], xhat[8];
            r.dy[i].template settle<ROW>(in_rows ? column(i) : cols, cols);
            r.x[i].template settle<ROW>(column(i), cols);
            r.dy[i].hold();
            r.x[i].o.hold();
            r.dy[i].floats(g);
            // (behind the row's end x - mean is -mean, and its product with rstd may be infinite: 0 times it is no 0)
            r.x[i].values(r.mean, CODES || column(i) < cols ? r.rstd : 0.0f, xhat);
            if (any_repeated<ROW>(column(i), cols))
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = e < (int)repeated<ROW>(column(i), cols) ? 0.0f : g[e];
            if (sums) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    dw[i][e] += g[e] * xhat[e];
                    db[i][e] += g[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                g[e] *= w[i][e];
                a += g[e];
                b += g[e] * xhat[e];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        a = lanes_sum<LANES>(a);
        b = lanes_sum<LANES>(b);
        if constexpr (WAVES > 1) {
            __shared__ float red[2][2][WAVES];
            if ((threadIdx.x & 63) == 0) {
                red[turn][0][threadIdx.x >> 6] = a;
                red[turn][1][threadIdx.x >> 6] = b;
            }
            __syncthreads();
            a = red[turn][0][0];
            b = red[turn][1][0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) {
                a += red[turn][0][i];
                b += red[turn][1][i];
            }
        }
        a /= n;
        b /= n;
        char *dx = (char *)p.dx + (size_t)(first + sub) * p.lddx * dtype_bytes(p.dx_dt);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float g[8], xhat[8];
            r.dy[i].hold();
            r.x[i].o.hold();
            r.dy[i].floats(g);
            r.x[i].values(r.mean, r.rstd, xhat);
            if constexpr (EDGE)
                if (any_repeated<ROW>(column(i), cols)) {
                    float q[8];
                    r.x[i].o.floats(q);
#pragma unroll
                    for (int e = 0; e < 8; ++e) xhat[e] = e < (int)repeated<ROW>(column(i), cols) ? q[e] * r.front : xhat[e];
                }
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = r.rstd * (g[e] * w[i][e] - a - xhat[e] * b);
            if (in_rows && column(i) < cols) store_octet<ROW>(dx, p.dx_dt, column(i), cols, g);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (!sums) return;
    float *out = p.partial + (size_t)blockIdx.x * 2 * norm_partial_cols(cols);
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (column(i) >= cols) continue;
            if (const uint32_t before = repeated<ROW>(column(i), cols)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (e < (int)before) continue;
                    out[column(i) - before + e] = dw[i][e];
                    out[norm_partial_cols(cols) + column(i) - before + e] = db[i][e];
                }
                continue;
            }
            v4f *at = (v4f *)(out + column(i)), *bt = (v4f *)(out + norm_partial_cols(cols) + column(i));
            at[0] = v4f{dw[i][0], dw[i][1], dw[i][2], dw[i][3]};
            at[1] = v4f{dw[i][4], dw[i][5], dw[i][6], dw[i][7]};
            bt[0] = v4f{db[i][0], db[i][1], db[i][2], db[i][3]};
            bt[1] = v4f{db[i][4], db[i][5], db[i][6], db[i][7]};
        }
    } else {
        __shared__ float fold[THREADS * 8];                     // [ROWS][GROUP * 8]
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int before = (int)repeated<ROW>(column(i), cols);
                    if (ROW != ROW_RAGGED || e >= before) fold[threadIdx.x * 8 + e - before] = which ? db[i][e] : dw[i][e];
                }
                __syncthreads();
#pragma unroll 1
                for (uint32_t c = threadIdx.x; c < GROUP * 8; c += THREADS) {
                    float s = fold[c];
#pragma unroll
                    for (int k = 1; k < ROWS; ++k) s += fold[k * GROUP * 8 + c];
                    if (i * GROUP * 8 + c < cols) out[which * norm_partial_cols(cols) + i * GROUP * 8 + c] = s;
                }
            }
        }
    }
}

// column sums over the rows of a slice: 128 columns a workgroup, 16 rows at a time; for rows of any length (8192 x 20000 bf16 127 us, 5.2 TB/s)
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
        n.settle(c, p.cols);
        n.values(mean, rstd, xhat);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dw[e] += dy[e] * xhat[e];
            db[e] += dy[e];
        }
    }
    const size_t stride = norm_partial_cols(p.cols);
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

// dweight / dbias out of the workgroups' sums: 32 columns a workgroup, 64 partial sums at a time, eight of which a lane has in flight, always in
// the same order.  blockIdx.y: which of the two, and the columns that x, of kMostColumnGroups workgroups at the most, leaves over.  512 rows of
// 4096 columns 4.5 us, three trips to memory one behind the other.
__global__ void __launch_bounds__(512) norm_parameter_sums_kernel(const NormBackwardArgs p) {
    constexpr uint32_t SLICES = 64, DEEP = 8;
    __shared__ v4f red[SLICES][8];
    const size_t stride = norm_partial_cols(p.cols);
    const uint32_t lane = threadIdx.x & 7, sub = threadIdx.x >> 3, which = blockIdx.y & 1, c0 = ((blockIdx.y >> 1) * gridDim.x + blockIdx.x) * 32;
    void *out = which ? p.dbias : p.dweight;
    if (!out || c0 >= p.cols) return;
    const float *in = p.partial + which * stride + c0 + lane * 4;
    v4f s = v4f{0, 0, 0, 0};
    for (uint32_t g = sub; g < p.groups; g += SLICES * DEEP) {
        v4f v[DEEP];
#pragma unroll
        for (uint32_t i = 0; i < DEEP; ++i) {
            const uint32_t at = g + i * SLICES;
            v[i] = *(const v4f *)(in + (size_t)(at < p.groups ? at : g) * 2 * stride);
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
    if (p.param_dt == QGEMM_DT_F32) ((float *)out)[c] = v;
    else ((uint16_t *)out)[c] = p.param_dt == QGEMM_DT_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}

}  // namespace qgemm
