// Log probabilities of given tokens out of logits, row by row: with m = max x, e = exp(x - m), S = sum e, T = sum e (x - m),
//   lse = m + log S,   log p of a token = (x[token] - m) - log S,   entropy = log S - T / S,   and the largest x with their log p;
// (lse has lost bits of log S where m is far from zero, all of them in a row that is masked throughout with the type's lowest value)
// and backward, with p = exp(log p), a = dlogp, b = dentropy:
//   dx_j = a ([j = token] - p_j) - b p_j (log p_j + entropy).
// One pass: every thread keeps the maximum of what it has seen, S and T under it, and puts them right when the maximum grows.  All fp32.
//
// Minus infinity is a token that cannot be: p = 0, and it adds nothing to S, T or the gradient.  A row that holds nothing else has lse = -inf,
// log p = -inf, entropy 0 and gradient 0.  Infinity and NaN make S NaN, and with it all that the row gives.
//
// The top k without sorting: L, the k-th largest of 64 groups' maxima, is no more than the k-th largest element, and only threads whose own maximum
// reaches L hold any element that does.  Their columns are read once more, what reaches L is gathered, and an element's place is the
// number of those above it.  Elements are compared as 64-bit keys, value above, then the lower index: no two are equal, and the order is that of
// the values with ties to the lowest index.
//
// What bounds it: memory, with the vector instructions (eleven slots an element, four of them the exponential) close behind: 2048 x 65536 bf16 with five tokens 61 us in a
// trace, 4.4 TB/s; a plain sum of as many bytes reads 4.0.  8 x 131072 fp32 with twenty tokens 7.3 and 5 for the join, trips to memory and to LDS one behind
// the other; backward 2048 x 65536 bf16 92, 5.8 TB/s read and written.
#pragma once
#include "model.h"
#include "octet.cuh"

namespace qgemm {

constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kNothing = -200.0f;                    // exp of it is 0 in fp32, and products with it are finite
constexpr float kMinusInf = -__builtin_inff();

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2E); }
// S and T from one maximum to a larger one (m = -inf: nothing has been added)
struct Sums {
    float m, s, t;
    __device__ __forceinline__ void raise(float to) {
        const float d = __builtin_fmaxf(m - to, kNothing), f = m == kMinusInf ? 0.0f : exp_of(d);
        t = m == kMinusInf ? 0.0f : f * (t + s * d);       // (s and t may be NaN where m is -inf: NaNs alone)
        s = m == kMinusInf && s == 0.0f ? 0.0f : s * f;
        m = to;
    }
    __device__ __forceinline__ void add(const float (&v)[8], float most) {
        if (__any(most > m)) raise(__builtin_fmaxf(m, most));
        const float r = m == kMinusInf ? 0.0f : m;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = v[e] - r, w = exp_of(d);
            s += w;
            t = __builtin_fmaf(w, __builtin_fmaxf(d, kNothing), t);
        }
    }
};
__device__ __forceinline__ float max8(const float (&v)[8]) {
    return __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(v[0], v[1]), __builtin_fmaxf(v[2], v[3])),
                           __builtin_fmaxf(__builtin_fmaxf(v[4], v[5]), __builtin_fmaxf(v[6], v[7])));
}
__device__ __forceinline__ float wave_max(float v) {
    auto dpp = [&](auto ctrl) {
        v = __builtin_fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, true)));
    };
    dpp(std::integral_constant<int, 0xB1>{});
    dpp(std::integral_constant<int, 0x4E>{});
    dpp(std::integral_constant<int, 0x141>{});
    dpp(std::integral_constant<int, 0x140>{});
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    v = __builtin_fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
    u = __builtin_bit_cast(uint32_t, v);
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return __builtin_fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// ---- keys: 0 is below every element's
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v != v ? kMinusInf : v + 0.0f);      // (NaN below all numbers; -0 is 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) { return (uint64_t)order_of(v) << 32 | (0xFFFFFFFFu - index); }
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }
template <int CTRL>
__device__ __forceinline__ uint64_t key_dpp(uint64_t k) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)k, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(k >> 32), CTRL, 0xF, 0xF, true);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t key_lane(uint64_t k, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(k >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ int64_t token_at(const void *tokens, int bytes, uint32_t row) {
    return bytes == 8 ? ((const int64_t *)tokens)[row] : (int64_t)((const int32_t *)tokens)[row];
}
__device__ __forceinline__ float logit_at(const void *row, int dt, size_t c) {
    if (dt == QGEMM_DT_F32) return ((const float *)row)[c];
    const uint16_t h = ((const uint16_t *)row)[c];
    return dt == QGEMM_DT_BF16 ? __builtin_bit_cast(float, (uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}
// the logit that a row's token asks for, fetched ahead of its use: two trips to memory one behind the other
struct Asked {
    bool any;
    float logit;
    __device__ __forceinline__ Asked(const LogProbArgs &p, uint32_t row) {
        const int64_t token = token_at(p.tokens, p.token_bytes, row);
        any = token >= 0 && token < (int64_t)p.cols;
        logit = logit_at((const char *)p.logits + (size_t)row * p.ld * dtype_bytes(p.dt), p.dt, any ? (size_t)token : 0);
    }
};
// a row's numbers out of its sums
__device__ __forceinline__ void log_prob_finish(const LogProbArgs &p, uint32_t row, const Asked &asked, float m, float s, float t, float l) {
    const bool none = s == 0.0f;
    p.logp[row] = !asked.any ? 0.0f : none ? kMinusInf : (asked.logit - m) - l;
    p.entropy[row] = none ? 0.0f : l - t / s;
    p.lse[row] = none ? kMinusInf : m + l;
}
__device__ __forceinline__ void store_top(const LogProbArgs &p, uint32_t row, uint32_t place, uint64_t key, float m, float l) {
    const float v = value_of(key);
    p.values[(size_t)row * p.top + place] = v == kMinusInf && l == l ? v : (v - m) - l;
    p.indices[(size_t)row * p.top + place] = index_of(key);
}

// how many of the first n keys of a list are above `mine`; the list has room for seven zeros behind them, and has them
__device__ __forceinline__ uint32_t keys_above(const uint64_t *list, uint32_t n, uint64_t mine) {
    uint32_t above = 0;
    for (uint32_t k = 0; k < n; k += 8) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) above += list[k + i] > mine ? 1 : 0;
    }
    return above;
}
// the k-th largest of a wave's keys, of which no two are equal but zeros; 0 where there are fewer
__device__ __forceinline__ uint64_t kth_largest(uint64_t mine, uint32_t k) {
    uint32_t above = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) above += key_lane(mine, i) > mine ? 1 : 0;
    const uint64_t at = __ballot(above == k - 1 && mine != 0);
    return at ? key_lane(mine, __builtin_ctzll(at)) : 0;
}

constexpr uint32_t kLogProbThreads = 256, kLogProbTurn = kLogProbThreads * kOctet, kLogProbAhead = 4, kCandidates = 2048;

// The `top` largest of columns begin .. end - 1, `own` the key of a thread's largest octet (its value, its first column; 0: it has none), to
// put(place, key) in place 0 .. top - 1, key 0 where there are fewer
template <int DT, class Put>
__device__ __forceinline__ void top_of(const void *row, uint32_t begin, uint32_t end, uint32_t top, uint64_t own, Put put) {
    __shared__ __align__(16) uint64_t group[64], list[kCandidates + 8];
    __shared__ uint32_t count, holders, holder[kLogProbThreads];
    const uint32_t tid = threadIdx.x;
    const uint64_t two = larger(own, key_dpp<0xB1>(own)), four = larger(two, key_dpp<0x4E>(two));
    if ((tid & 3) == 0) group[tid >> 2] = four;
    if (tid == 0) count = holders = 0;
    __syncthreads();
    // (one wave for all: done by each of the four it was half of the time of rows of a thousand columns, 4096 x 1000 bf16 20 us)
    if (tid < 64) {
        const uint64_t least = kth_largest(group[tid], top);
        if (tid == 0) list[0] = least;
    }
    __syncthreads();
    const uint64_t least = list[0];                        // L
    // an octet's key stands for any of its elements
    uint64_t bound = least == 0 ? 0 : (least & 0xFFFFFFFF00000000ull) | (0xFFFFFFFFu - (index_of(least) + kOctet - 1));
    if (own != 0 && own >= least) holder[atomicAdd(&holders, 1u)] = tid;
    __syncthreads();
    const uint32_t turns = (end - begin + kLogProbTurn - 1) / kLogProbTurn, items = holders * turns;
    for (;;) {
        for (uint32_t i = tid; i < items; i += kLogProbThreads) {
            const uint32_t which = i / turns, c = begin + holder[which] * kOctet + (i - which * turns) * kLogProbTurn;
            if (c >= end) continue;
            Octet<DT> o;
            float v[8];
            o.request(row, c, end);
            o.settle(c, end);
            o.floats(v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint64_t key = key_of(v[e], c + e);
                if (c + e >= end || key < bound) continue;
                const uint32_t at = atomicAdd(&count, 1u);
                if (at < kCandidates) list[at] = key;
            }
        }
        __syncthreads();
        const uint32_t found = count, n = found < kCandidates ? found : kCandidates;
        if (tid < 8) list[n + tid] = 0;
        __syncthreads();                                   // (and count is cleared below)
        if (found <= kCandidates) {
            for (uint32_t i = tid; i < n; i += kLogProbThreads) {
                const uint64_t mine = list[i];
                const uint32_t above = keys_above(list, n, mine);
                if (above < top) put(above, mine);
            }
            for (uint32_t i = n + tid; i < top; i += kLogProbThreads) put(i, 0ull);
            __syncthreads();
            return;
        }
        // more than there is room for: the k-th largest of those that were kept is a higher bound still
        for (uint32_t i = tid; i < n; i += kLogProbThreads) {
            const uint64_t mine = list[i];
            if (keys_above(list, n, mine) == top - 1) group[0] = mine;
        }
        if (tid == 0) count = 0;
        __syncthreads();
        bound = group[0];
        __syncthreads();
    }
}

// A workgroup's sums of columns begin .. end - 1 of a row, in every thread; `each` is told of each octet's largest element and first column
template <int DT, int AHEAD, class Each>
__device__ __forceinline__ Sums row_sums(const char *x, uint32_t begin, uint32_t end, Each each) {
    constexpr int WAVES = kLogProbThreads / 64;
    __shared__ float red[3][WAVES];
    const uint32_t tid = threadIdx.x;
    Sums sums{kMinusInf, 0.0f, 0.0f};
    for (uint32_t c0 = begin + tid * kOctet; c0 < end; c0 += AHEAD * kLogProbTurn) {
        Octet<DT> o[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) o[i].request(x, c0 + i * kLogProbTurn, end);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const uint32_t c = c0 + i * kLogProbTurn;
            if (c >= end) break;
            float v[8];
            o[i].settle(c, end);
            o[i].floats(v);
            if (end - c < kOctet)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = c + e < end ? v[e] : kMinusInf;
            const float most = max8(v);
            each(most, c);
            sums.add(v, most);
        }
    }
    const float wave = wave_max(sums.m);
    if ((tid & 63) == 0) red[0][tid >> 6] = wave;
    __syncthreads();
    float m = red[0][0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) m = __builtin_fmaxf(m, red[0][i]);
    sums.raise(m);
    const float s = lanes_sum<64>(sums.s), t = lanes_sum<64>(sums.t);
    if ((tid & 63) == 0) {
        red[1][tid >> 6] = s;
        red[2][tid >> 6] = t;
    }
    __syncthreads();                                       // (the next row's maxima go where nobody reads any more)
    Sums all{m, red[1][0], red[2][0]};
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        all.s += red[1][i];
        all.t += red[2][i];
    }
    return all;
}

// one workgroup for a split of a row
template <int DT, bool TOP>
__global__ void __launch_bounds__(kLogProbThreads) log_prob_kernel(const LogProbArgs p) {
    const uint32_t tid = threadIdx.x, begin = blockIdx.x * p.part, end = p.cols - begin < p.part ? p.cols : begin + p.part;
    for (uint32_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const char *x = (const char *)p.logits + (size_t)row * p.ld * Octet<DT>::ES;
        const Asked asked(p, row);
        float best = kMinusInf;
        uint32_t best_at = begin + tid * kOctet;
        const Sums sums = row_sums<DT, kLogProbAhead>(x, begin, end, [&](float most, uint32_t c) {
            if (TOP && most > best) {
                best = most;
                best_at = c;
            }
        });
        const float m = sums.m, l = logf(sums.s);
        float *part = p.splits > 1 ? p.partial + ((size_t)row * p.splits + blockIdx.x) * log_prob_part(p.top) : nullptr;
        if (tid == 0) {
            if (part) {
                part[0] = m;
                part[1] = sums.s;
                part[2] = sums.t;
            } else {
                log_prob_finish(p, row, asked, m, sums.s, sums.t, l);
            }
        }
        if constexpr (TOP) {
            const uint64_t own = begin + tid * kOctet < end ? key_of(best, best_at) : 0;
            top_of<DT>(x, begin, end, p.top, own, [&](uint32_t place, uint64_t key) {
                if (part) ((uint64_t *)(part + 4))[place] = key;
                else store_top(p, row, place, key, m, l);
            });
        }
        __syncthreads();
    }
}

// The splits of a row together.  Their lists are in order: where there are no fewer splits than places, the k-th largest of the heads is no more than the k-th
// largest of all, else the smallest of what is in place k / splits, rounded up, of each; what reaches that is gathered and placed as above.  (One wave that takes the largest
// head k times: 13 us for 64 splits with twenty tokens; 5.)
__global__ void __launch_bounds__(256) log_prob_join_kernel(const LogProbArgs p) {
    __shared__ __align__(16) uint64_t list[64 * kMostTop + 8];
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const bool in = lane < p.splits;
        const Asked asked(p, row);
        const float *parts = p.partial + (size_t)row * p.splits * log_prob_part(p.top), *part = parts + (in ? lane : 0) * log_prob_part(p.top);
        constexpr uint32_t MOST = 64 * kMostTop / 256;
        uint64_t own[MOST], bound = 0;
        const uint32_t n = p.splits * p.top, place = p.top ? (p.top + p.splits - 1) / p.splits - 1 : 0;
#pragma unroll
        for (uint32_t i = 0; i < MOST; ++i) {
            const uint32_t at = tid + i * 256;
            own[i] = at < n ? ((const uint64_t *)(parts + at / p.top * log_prob_part(p.top) + 4))[at % p.top] : 0;
        }
        if (p.top) bound = ((const uint64_t *)(part + 4))[place];
        Sums sums{in ? part[0] : kMinusInf, in ? part[1] : 0.0f, in ? part[2] : 0.0f};
        const float m = wave_max(sums.m);
        sums.raise(m);
        const float s = lanes_sum<64>(sums.s), t = lanes_sum<64>(sums.t), l = logf(s);
        if (tid == 0) log_prob_finish(p, row, asked, m, s, t, l);
        if (!p.top) continue;
        if (place == 0) {
            bound = kth_largest(in ? bound : 0, p.top);
        } else {
            bound = in ? bound : ~0ull;
#pragma unroll
            for (int d = 32; d; d /= 2) {
                const uint64_t other = __shfl_xor(bound, d);
                bound = other < bound ? other : bound;
            }
        }
        if (tid == 0) count = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < MOST; ++i)
            if (own[i] != 0 && own[i] >= bound) list[atomicAdd(&count, 1u)] = own[i];
        __syncthreads();
        const uint32_t found = count;
        if (tid < 8) list[found + tid] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < found; i += 256) {
            const uint64_t mine = list[i];
            const uint32_t above = keys_above(list, found, mine);
            if (above < p.top) store_top(p, row, above, mine, m, l);
        }
        __syncthreads();
    }
}

// ---- backward: a workgroup takes AHEAD times kLogProbTurn columns a turn.  log p = x - lse is off by the rounding of lse, half its last place: 2^-18 of p at kFar, as much as
// the exponential's own roundings leave of p = exp(-30).  Beyond it, up to where lse holds nothing of log S, one workgroup sums the row again and writes all of it with
// log p = (x - m) - log S.  (us, no row / every row beyond: 2048 x 65536 bf16 112 / 230, fp32 183 / 400, 8 x 131072 fp32 4 / 52.  The choice costs rows that are near
// 1.4 us of 2048 x 65536: 90.9 without it, 92.3 so, 94.5 with what the row asks for fetched one behind the other; 93.4 with rows that ask for nothing.)
constexpr float kFar = 128.0f;
template <int DT>
__global__ void __launch_bounds__(kLogProbThreads) log_prob_backward_kernel(const LogProbBackwardArgs p) {
    constexpr uint32_t AHEAD = 2;
    for (uint32_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const char *x = (const char *)p.logits + (size_t)row * p.ld * Octet<DT>::ES;
        char *dx = (char *)p.dlogits + (size_t)row * p.ldd * dtype_bytes(p.out_dt);
        const int64_t token = token_at(p.tokens, p.token_bytes, row);
        const bool asked = token >= 0 && token < (int64_t)p.cols;
        const float lse = p.lse[row], dlogp = p.dlogp[row], b = p.dentropy ? p.dentropy[row] : 0.0f, entropy = p.dentropy ? p.entropy[row] : 0.0f;
        const bool none = lse == kMinusInf, far = __builtin_fabsf(lse) > kFar && __builtin_fabsf(lse) < __builtin_inff();
        const float a = asked && !none ? dlogp : 0.0f, h = b != 0.0f ? entropy : 0.0f;      // (chosen when they are there: no trip to memory behind another)
        const bool nothing = !asked && b == 0.0f;      // (padding may hold anything: 0 times its NaNs is no 0)
        Octet<DT> o[AHEAD];
        auto request = [&](uint32_t c0) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) o[i].request(x, c0 + i * kLogProbTurn, p.cols);
        };
        constexpr uint32_t turn = AHEAD * kLogProbTurn;
        uint32_t c0 = blockIdx.x * turn + threadIdx.x * kOctet, step = gridDim.x * turn;
        float m = lse, log_s = 0.0f;
        request(c0);
        if (far) {
            if (blockIdx.x != row % gridDim.x) continue;       // (the first of each row would be on the same XCD where their number is a multiple of 8)
            const Sums sums = row_sums<DT, AHEAD>(x, 0, p.cols, [](float, uint32_t) {});
            c0 = threadIdx.x * kOctet, step = turn;
            m = sums.m, log_s = logf(sums.s);
            request(c0);
        }
        for (; c0 < p.cols; c0 += step) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const uint32_t c = c0 + i * kLogProbTurn;
                if (c >= p.cols) break;
                float v[8];
                o[i].settle(c, p.cols);
                o[i].floats(v);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float l = (v[e] - m) - log_s, q = none ? 0.0f : exp_of(l);
                    const float g = a + b * (__builtin_fmaxf(l, kNothing) + h);
                    v[e] = -(q * g);
                    if (asked && (int64_t)(c + e) == token) v[e] += a;
                }
                if (none || nothing)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
                store_octet(dx, p.out_dt, c, p.cols, v);
            }
            if (p.cols - c0 > step) request(c0 + step);
        }
    }
}

}  // namespace qgemm
