// Activations into 8 bits and back: codes of 1 x 128 blocks under scales that are powers of two (see power_of_two).
#pragma once
#include "octet.cuh"
#include "training.h"

namespace qgemm {

// A lane is an octet, sixteen lanes a block: the block's maximum takes four exchanges between neighbours and no LDS, and memory bounds it.
// blockIdx.y counts blocks of 128 columns in groups of 16, blockIdx.x rows.  6144 x 14336 bf16 to e4m3 48 - 56 us, 4.8 - 5.6 TB/s of the 5.1 at
// which a copy runs; 16 x 2048 2.5.
template <int IN_DT, int Q_DT>
__global__ void __launch_bounds__(256) checkpoint_kernel(const KeepArgs p) {
    // the scale from which a code above LIMIT would stand for more than the input's type holds: 64 or 256 of them are its first infinity
    constexpr int TOP = (IN_DT == QGEMM_DT_F16 ? 16 : 128) - (Q_DT == QGEMM_DT_I8 ? 6 : 8);
    constexpr float LIMIT = Q_DT == QGEMM_DT_I8 ? 63.0f : 240.0f;
    const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * kOctet;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        Octet<IN_DT> o;
        float v[8];
        o.request((const char *)p.in + (size_t)row * p.ld_in * Octet<IN_DT>::ES, c, p.cols);
        o.settle(c, p.cols);
        o.floats(v);
        const PowerOfTwo s = power_of_two<Q_DT>(block_max_bits(v));
        if (s.s >= __builtin_bit_cast(float, (uint32_t)(TOP + 127) << 23)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_fminf(__builtin_fmaxf(v[e], -LIMIT * s.s), LIMIT * s.s);
        }
        if (c < p.cols) {
            store_codes((uint8_t *)p.out + (size_t)row * p.ld_out, c, p.cols, octet_codes<Q_DT>(v, s.inv));
            if (c % kScaleBlock == 0) p.scales[(size_t)row * p.kb + c / kScaleBlock] = s.s;
        }
    }
}

// Bound by memory: 6144 x 14336 bf16 out of e4m3 41 us, 6144 x 7168 out of int8 21, 6.5 TB/s where the codes were written shortly before.
template <int Q_DT>
__global__ void __launch_bounds__(256) restore_kernel(const KeepArgs p) {
    const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * kOctet;
    if (c >= p.cols) return;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        Octet<Q_DT> o;
        float v[8];
        const float s = p.scales[(size_t)row * p.kb + c / kScaleBlock];
        o.request((const char *)p.in + (size_t)row * p.ld_in, c, p.cols);
        o.settle(c, p.cols);
        o.floats(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= s;
        store_octet((char *)p.out + (size_t)row * p.ld_out * dtype_bytes(p.out_dt), p.out_dt, c, p.cols, v);
    }
}

}  // namespace qgemm
