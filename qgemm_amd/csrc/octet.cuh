// Eight neighbouring elements of a row: what a lane of the layer norm, checkpoint and gradient kernels works on.  Sixteen lanes hold
// the 128 columns that share a scale, whatever the element type.
#pragma once
#include "common.h"

namespace qgemm {

constexpr uint32_t kOctet = 8;

// What is known of a row's length: anything; eight elements or more, of fewer than 2^32 bytes; the same, a multiple of eight
enum RowKind : int { ROW_ANY = 0, ROW_RAGGED = 1, ROW_WHOLE = 2 };
template <int ROW>
using row_offset = std::conditional_t<ROW == ROW_ANY, size_t, uint32_t>;

// A row that ends inside its last octet: no lane reads behind it, and nothing branches between loads, as the last eight elements are
// fetched from where they lie.
//   ROW_RAGGED  the lane works on those eight: the first `repeated` of them are the octet in front's as well, count in no sum and are
//               written twice, with the same values.  (They may lie in the block of 128 columns in front of the lane's own, which has another
//               scale: whatever comes out of codes there takes the scale of column cols - 8 for them.)  (Moving them down instead, and writing the end element by element, kept one wave of
//               every row a third longer than the others: norm of 4096 x 3001 bf16 19.1 us, 14.2 for 3000)
//   ROW_ANY     they are moved down, zeros behind them; rows of fewer than eight are fetched one by one
template <int ROW>
__device__ __forceinline__ uint32_t octet_begin(uint32_t c, uint32_t cols) {
    return ROW == ROW_RAGGED && c < cols && cols - c < kOctet ? cols - kOctet : c;
}
// how many elements in front of column c the octet of a lane starts, and whether any lane of the wave has such
template <int ROW>
__device__ __forceinline__ uint32_t repeated(uint32_t c, uint32_t cols) {
    return c - octet_begin<ROW>(c, cols);
}
template <int ROW>
__device__ __forceinline__ bool any_repeated(uint32_t c, uint32_t cols) {
    return ROW == ROW_RAGGED && __any(repeated<ROW>(c, cols) != 0);
}
template <int DT>
struct Octet {
    static constexpr int TYPE = DT;
    static constexpr int ES = DT == QGEMM_DT_F32 ? 4 : (DT == QGEMM_DT_BF16 || DT == QGEMM_DT_F16) ? 2 : 1, DW = 2 * ES;
    uint32_t w[DW];

    // elements c .. c + 7 of a row of `cols`, as they come from memory; `settle` brings them in order
    template <int ROW = ROW_ANY>
    __device__ __forceinline__ void request(const void *row, uint32_t c, uint32_t cols) {
        const char *p = (const char *)row;
        if (ROW != ROW_ANY || cols >= kOctet) {
            p += (row_offset<ROW>)(c < cols - kOctet ? c : cols - kOctet) * ES;
            if constexpr (DW == 2) {
                const v2i v = *(const v2i_any *)p;
                w[0] = v[0], w[1] = v[1];
            } else {
#pragma unroll
                for (int i = 0; i < DW / 4; ++i) {
                    const v4i v = *(const v4i_any *)(p + 16 * i);
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[4 * i + k] = (uint32_t)v[k];
                }
            }
        } else {
            few(p, c < cols ? cols - c : 0);
        }
    }
    // zeros where the row has nothing
    template <int ROW = ROW_ANY>
    __device__ __forceinline__ void settle(uint32_t c, uint32_t cols) {
        const bool in = c < cols;
        if (ROW == ROW_ANY && cols >= kOctet) {
            const uint32_t gone = in && c > cols - kOctet ? c - (cols - kOctet) : 0;
            if (__any(gone != 0)) move_down<DW, ES == 4>(w, gone * ES);
        }
#pragma unroll
        for (int i = 0; i < DW; ++i) w[i] = in ? w[i] : 0;
    }
    // (the compiler converts again what it would otherwise keep as floats, in up to four times the registers)
    __device__ __forceinline__ void hold() {
#pragma unroll
        for (int i = 0; i < DW; ++i) asm volatile("" : "+v"(w[i]));
    }
    __device__ __forceinline__ void floats(float (&v)[8]) const {
        if constexpr (DT == QGEMM_DT_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, w[i]);
        } else if constexpr (DT == QGEMM_DT_BF16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __builtin_bit_cast(float, w[i] << 16);
                v[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xFFFF0000u);
            }
        } else if constexpr (DT == QGEMM_DT_F16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f16x2_t h = __builtin_bit_cast(f16x2_t, w[i]);
                v[2 * i] = (float)h[0];
                v[2 * i + 1] = (float)h[1];
            }
        } else if constexpr (DT == QGEMM_DT_I8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3)));
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
                v[4 * i] = lo[0], v[4 * i + 1] = lo[1], v[4 * i + 2] = hi[0], v[4 * i + 3] = hi[1];
            }
        }
    }
    // eight numbers, rounded to nearest even where the type has fewer bits (fp32, bf16 and fp16)
    __device__ __forceinline__ void take(const float (&v)[8]) {
        if constexpr (DT == QGEMM_DT_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __builtin_bit_cast(uint32_t, v[i]);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v2i p = DT == QGEMM_DT_BF16 ? pack4_bf16(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3])
                                                  : pack4_f16(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
                w[2 * h] = (uint32_t)p[0], w[2 * h + 1] = (uint32_t)p[1];
            }
        }
    }
    // as elements of a row of eight or more (c < cols; rows that are no ROW_ANY)
    template <int ROW>
    __device__ __forceinline__ void put(void *row, uint32_t c, uint32_t cols) const {
        static_assert(ROW != ROW_ANY, "rows of eight elements and more");
        char *at = (char *)row + (row_offset<ROW>)octet_begin<ROW>(c, cols) * ES;
#pragma unroll
        for (int i = 0; i < DW / 4; ++i) *(v4i_any *)(at + 16 * i) = v4i{(int)w[4 * i], (int)w[4 * i + 1], (int)w[4 * i + 2], (int)w[4 * i + 3]};
    }

private:
    __device__ void few(const char *p, uint32_t n) {
#pragma unroll
        for (int i = 0; i < DW; ++i) w[i] = 0;
#pragma unroll 1
        for (uint32_t e = n; e-- > 0;) {                       // the last first: each moves up what is there
            constexpr int UP = 32 - 8 * ES;
#pragma unroll
            for (int i = DW - 1; i >= 0; --i) {
                if constexpr (ES == 4) w[i] = i ? w[i - 1] : ((const uint32_t *)p)[e];
                else w[i] = w[i] << (8 * ES) | (i ? w[i - 1] >> UP : (ES == 2 ? (uint32_t)((const u16_any *)p)[e] : (uint32_t)((const uint8_t *)p)[e]));
            }
        }
    }
};

// the same of a type that is known to the launch only (parameters: fp32, bf16 or fp16)
template <int ROW = ROW_ANY>
__device__ __forceinline__ void parameter_octet(const void *p, int dt, uint32_t c, uint32_t cols, float (&v)[8]) {
    auto take = [&](auto o) {
        o.template request<ROW>(p, c, cols);
        o.template settle<ROW>(c, cols);
        o.floats(v);
    };
    if (dt == QGEMM_DT_F32) take(Octet<QGEMM_DT_F32>());
    else if (dt == QGEMM_DT_BF16) take(Octet<QGEMM_DT_BF16>());
    else take(Octet<QGEMM_DT_F16>());
}

// v as elements c .. c + 7 of a row of `cols` (c < cols), one rounding to nearest even where the type has fewer bits
template <int ROW = ROW_ANY>
__device__ __forceinline__ void store_octet(void *row, int dt, uint32_t c, uint32_t cols, const float (&v)[8]) {
    if (ROW == ROW_RAGGED) c = octet_begin<ROW>(c, cols);
    if (ROW != ROW_ANY || cols - c >= kOctet) {
        if (dt == QGEMM_DT_F32) {
            v4f_any *p = (v4f_any *)((char *)row + (row_offset<ROW>)c * 4);
            p[0] = v4f{v[0], v[1], v[2], v[3]};
            p[1] = v4f{v[4], v[5], v[6], v[7]};
        } else {
            const v2i a = dt == QGEMM_DT_BF16 ? pack4_bf16(v[0], v[1], v[2], v[3]) : pack4_f16(v[0], v[1], v[2], v[3]);
            const v2i b = dt == QGEMM_DT_BF16 ? pack4_bf16(v[4], v[5], v[6], v[7]) : pack4_f16(v[4], v[5], v[6], v[7]);
            *(v4i_any *)((char *)row + (row_offset<ROW>)c * 2) = v4i{a[0], a[1], b[0], b[1]};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 7; ++e) {
        if (e >= (int)(cols - c)) break;
        if (dt == QGEMM_DT_F32) ((float *)row)[c + e] = v[e];
        else ((uint16_t *)row)[c + e] = dt == QGEMM_DT_BF16 ? f32_to_bf16_bits(v[e]) : f32_to_f16_bits(v[e]);
    }
}
template <int ROW = ROW_ANY>
__device__ __forceinline__ void store_codes(void *row, uint32_t c, uint32_t cols, v2i q) {
    uint8_t *p = (uint8_t *)row + c;
    if (ROW == ROW_WHOLE || cols - c >= kOctet) {
        *(v2i_any *)p = q;
        return;
    }
    const uint32_t before = repeated<ROW>(c, cols);
    if (ROW == ROW_RAGGED && c % kScaleBlock != 0) {          // (what is repeated lies under the same scale)
        *(v2i_any *)(p - before) = q;
        return;
    }
    const uint64_t all = ((uint64_t)(uint32_t)q[1] << 32 | (uint32_t)q[0]) >> (8 * before);
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (e < (int)(cols - c)) p[e] = (uint8_t)(all >> (8 * e));
}

// Sum over groups of 16, 32 or 64 neighbouring lanes, in every lane and in the same order whatever the lane (see lanes_max)
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    auto dpp = [&](auto ctrl) {
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    dpp(std::integral_constant<int, 0xB1>{});      // quad_perm [1,0,3,2]
    dpp(std::integral_constant<int, 0x4E>{});      // quad_perm [2,3,0,1]
    dpp(std::integral_constant<int, 0x141>{});     // row_half_mirror
    dpp(std::integral_constant<int, 0x140>{});     // row_mirror
    if constexpr (LANES >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto sw = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const uint32_t a = sw[0], b = sw[1];
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    if constexpr (LANES == 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const uint32_t a = sw[0], b = sw[1];
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    return v;
}
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
// largest |v| of the 128 columns that 16 neighbouring lanes hold, as bits: their order is that of the numbers, with infinity and NaNs on top
__device__ __forceinline__ uint32_t block_max_bits(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu;
        m = b > m ? b : m;
    }
    auto with = [&](auto ctrl) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, decltype(ctrl)::value, 0xF, 0xF, true);
        m = o > m ? o : m;
    };
    with(std::integral_constant<int, 0xB1>{});
    with(std::integral_constant<int, 0x4E>{});
    with(std::integral_constant<int, 0x141>{});
    with(std::integral_constant<int, 0x140>{});
    return m;
}

// ---- 8-bit codes under a scale that is a power of two
// s is the smallest power of two (2^-126 at the least) with max|v| <= 127 s (int8) or 448 s (e4m3), 1 for zeros; q = rne(v / s), and v / s is
// exact.  Powers of two cost up to one bit of the eight against s = max / 127, and buy that q s needs no more bits than q: it is
// exact in bf16, and in fp16 within its range, so that a product that reads q s on the 16-bit matrix cores rounds nothing.  (Where q s is no multiple of
// the type's smallest number it is rounded to one: bf16 from e4m3 under s < 2^-124, fp16 under s < 2^-24, from e4m3 under s < 2^-15.)
// A block with an infinity or a NaN gets s = NaN: all of it reads as NaN, and nothing is hidden from what is computed from it.
struct PowerOfTwo {
    float s, inv;       // the scale and 1 / s; inv is 0 where s is NaN
};
template <int Q_DT>
__device__ __forceinline__ PowerOfTwo power_of_two(uint32_t max_bits) {
    // 127 = 1.984375 x 2^6, 448 = 1.75 x 2^8
    constexpr uint32_t MANTISSA = Q_DT == QGEMM_DT_I8 ? 0x7E0000u : 0x600000u;
    constexpr int EXPONENT = Q_DT == QGEMM_DT_I8 ? 6 : 8;
    int e = (int)(max_bits >> 23) - EXPONENT + ((max_bits & 0x7FFFFFu) > MANTISSA ? 1 : 0);      // biased
    e = e < 1 ? 1 : e;
    e = max_bits == 0 ? 127 : e;
    const bool finite = max_bits < 0x7F800000u;
    PowerOfTwo r;
    r.s = __builtin_bit_cast(float, finite ? (uint32_t)e << 23 : 0x7FC00000u);
    r.inv = __builtin_bit_cast(float, finite ? (uint32_t)(254 - e) << 23 : 0u);
    return r;
}
// |v| inv is at most 127 / 448.  (A code that its type could not hold cannot come up; NaN under inv = 0 is masked by the caller's s = NaN.)
template <int Q_DT>
__device__ __forceinline__ v2i octet_codes(const float (&v)[8], float inv) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (Q_DT == QGEMM_DT_F8E4M3) {
            uint32_t p = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * inv, v[4 * h + 1] * inv, 0, false);
            w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * inv, v[4 * h + 3] * inv, (int)p, true);
        } else {
            // 1.5 x 2^23 rounds to the nearest integer, ties to even, and leaves it in the low byte
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = __builtin_bit_cast(uint32_t, __builtin_fmaf(v[4 * h + e], inv, 12582912.0f));
            const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400);
            w[h] = lo | (hi << 16);
        }
    }
    return v2i{(int)w[0], (int)w[1]};
}

}  // namespace qgemm
