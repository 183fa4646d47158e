// Layer norm, activations in 8 bits and weight gradients: what the entries of qgemm_capi.hip hand to the launchers.
#pragma once
#include "common.h"

namespace qgemm {

struct NormArgs {
    const void *x, *weight, *bias;     // weight null: y = xhat; bias null: none
    void *y, *q;                       // q null: nothing is kept
    float *mean, *rstd, *scales;       // mean, rstd: null where nobody wants them
    uint64_t ldx, ldy, ldq;
    uint32_t rows, cols, kb;           // kb: scales of a row
    float eps;
    int x_dt, y_dt, param_dt, q_dt;
};
hipError_t launch_layer_norm(const NormArgs &a, int cus, hipStream_t stream);

struct NormBackwardArgs {
    const void *dy, *x, *weight;       // x: the norm's input, or the codes of xhat (scales not null)
    const float *scales, *mean, *rstd;
    void *dx, *dweight, *dbias;        // dweight, dbias: null where nobody wants them
    float *partial;                    // [groups][2][norm_partial_cols(cols)]
    uint64_t lddy, ldx, lddx;
    uint32_t rows, cols, kb, groups;
    int dy_dt, x_dt, dx_dt, param_dt;
};
// workgroups whose column sums a launch leaves in `partial`, 0 where nobody wants sums or there are no rows
uint32_t norm_backward_groups(const NormBackwardArgs &a, int cus);
__host__ __device__ inline size_t norm_partial_cols(uint32_t cols) { return ((size_t)cols + 63) / 64 * 64; }
inline size_t norm_partial_bytes(uint32_t groups, uint32_t cols) { return (size_t)groups * 2 * norm_partial_cols(cols) * sizeof(float); }
hipError_t launch_layer_norm_backward(const NormBackwardArgs &a, int cus, hipStream_t stream);

struct KeepArgs {
    const void *in;
    void *out;
    float *scales;
    uint64_t ld_in, ld_out;
    uint32_t rows, cols, kb;
    int in_dt, out_dt;
};
hipError_t launch_checkpoint(const KeepArgs &a, hipStream_t stream);
hipError_t launch_restore(const KeepArgs &a, hipStream_t stream);

struct WeightGradArgs {
    const void *dy, *q, *weight, *bias;     // dy rows x n, q rows x cols codes
    const float *scales;
    void *dw;                               // n x cols
    float *db;                              // n, or null
    void *room;                             // the slices' partial sums
    uint64_t lddy, ldq, lddw;
    uint32_t rows, n, cols, kb;
    int dy_dt, q_dt, param_dt, dw_dt;
    int tile;                               // GradTile
    uint32_t slices, slice;                 // slices of the rows, and rows of one, a multiple of kGradStep
    int plain;                              // octets of a step may be fetched by 32-bit offsets, as they lie
};
enum GradTile : int { TILE_128x128, TILE_256x128, TILE_256x256, GRAD_TILES };
// partial sums of a slice: n of dy, then n rows of dW
__host__ __device__ inline size_t grad_round(uint32_t v) { return ((size_t)v + 3) / 4 * 4; }
__host__ __device__ inline size_t grad_plane(uint32_t n, uint32_t cols) { return grad_round(n) + n * grad_round(cols); }
size_t plan_weight_grad(WeightGradArgs &a, int cus);          // chooses tile and slices; bytes of `room`
hipError_t launch_weight_grad(const WeightGradArgs &a, hipStream_t stream);

}  // namespace qgemm
