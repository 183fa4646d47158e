// Root-mean-square norm, adapters beside a product and log probabilities: what the entries of qgemm_capi.hip hand to the launchers.
#pragma once
#include "common.h"

namespace qgemm {

struct RmsArgs {
    const void *x, *residual, *weight;   // residual null: h is x; weight null: y = h rstd
    void *h, *y, *q;                     // h: with a residual only; y, q null: nobody wants them
    float *rstd, *scales;                // rstd: null where nobody wants it
    uint64_t ldx, ldr, ldh, ldy, ldq;
    uint32_t rows, cols, kb;             // kb: scales of a row
    float eps;
    int x_dt, r_dt, y_dt, param_dt, q_dt;
};
hipError_t launch_rms_norm(const RmsArgs &a, hipStream_t stream);

struct RmsBackwardArgs {
    const void *dy, *h, *dh, *weight;    // dh: what arrives along the residual stream, or null
    const float *rstd;
    void *dx, *dweight;                  // dweight: null where nobody wants it
    float *partial;                      // [groups][norm_partial_cols(cols)]
    uint64_t lddy, ldh, lddh, lddx;
    uint32_t rows, cols, groups;
    int dy_dt, h_dt, dh_dt, dx_dt, param_dt;
};
uint32_t rms_backward_groups(const RmsBackwardArgs &a, int cus);      // workgroups whose column sums a launch leaves in `partial`
size_t rms_partial_bytes(uint32_t groups, uint32_t cols);
hipError_t launch_rms_norm_backward(const RmsBackwardArgs &a, int cus, hipStream_t stream);

// ---- log probabilities
constexpr uint32_t kMostTop = 32;
struct LogProbArgs {
    const void *logits, *tokens;
    float *logp, *entropy, *lse, *values;
    int64_t *indices;
    float *partial;                      // [rows][splits][log_prob_part(top)]
    uint64_t ld;
    uint32_t rows, cols, top, splits, part;   // part: columns of a split, a multiple of 8
    int dt, token_bytes;
};
// a split's maximum and sums, then its top: values and indices
__host__ __device__ inline uint32_t log_prob_part(uint32_t top) { return 4 + 2 * top; }
size_t plan_log_prob(LogProbArgs &a, int cus);            // chooses splits; bytes of `partial`
hipError_t launch_log_prob(const LogProbArgs &a, hipStream_t stream);

struct LogProbBackwardArgs {
    const void *logits, *tokens;
    const float *lse, *entropy, *dlogp, *dentropy;       // dentropy null: no gradient of the entropies
    void *dlogits;
    uint64_t ld, ldd;
    uint32_t rows, cols;
    int dt, out_dt, token_bytes;
};
hipError_t launch_log_prob_backward(const LogProbBackwardArgs &a, hipStream_t stream);

// ---- adapters.  Rows are grouped by adapter, those of none last, and the groups cut into slots of kSlotRows rows; see group_rows_kernel
constexpr uint32_t kSlotRows = 64, kMostAdapters = 65535, kMostRank = 128;
struct RowGroups {
    const int32_t *order;                // rows, group by group, in their own order within a group
    const int32_t *offsets;              // where group i starts in `order`: adapters + 2, the last being the number of rows
    const int32_t *first;                // first slot of group i: adapters + 1
    const v4i *slots;                    // group of a slot (-1: none), where it starts in `order`, its rows, its number in the group
    uint32_t rows, adapters, slot_count;
};
inline size_t group_slots(size_t rows, size_t adapters) { return rows / kSlotRows + (rows < adapters + 1 ? rows : adapters + 1); }
inline size_t group_slots_at(size_t rows, size_t adapters) { return (rows + 2 * adapters + 3 + 3) / 4 * 4; }
inline size_t group_words(size_t rows, size_t adapters) { return group_slots_at(rows, adapters) + 4 * group_slots(rows, adapters); }
inline RowGroups row_groups(const void *words, size_t rows, size_t adapters) {
    const int32_t *w = (const int32_t *)words;
    return RowGroups{w, w + rows, w + rows + adapters + 2, (const v4i *)(w + group_slots_at(rows, adapters)), (uint32_t)rows, (uint32_t)adapters,
                     (uint32_t)group_slots(rows, adapters)};
}
hipError_t launch_group_rows(const void *ids, int id_bytes, const RowGroups &g, hipStream_t stream);

// sums over the rank of a row, in `planes` parts that have to be added up
struct RankSums {
    float *at;
    uint64_t stride;                     // from a part to the next
    uint32_t pitch, planes;              // pitch: from a row to the next
    int grouped;                         // the rows lie as they are grouped, so that nothing has to be looked up for them
};
inline uint32_t rank_pitch(uint32_t rank) { return (rank + 15) / 16 * 16; }

struct ShrinkArgs {                      // u[row] = W[its adapter] x[row]
    RowGroups g;
    const void *x, *w;                   // w [adapters][rank][cols]
    RankSums u;                          // a part for each split of the columns
    uint64_t ldx;
    uint32_t cols, rank, part;           // part: columns of a split
    int dt, zero;                        // zero: rows without an adapter get zeros
};
void plan_shrink(ShrinkArgs &a, int cus);                 // chooses u.planes and part
hipError_t launch_shrink(const ShrinkArgs &a, hipStream_t stream);

struct ExpandArgs {                      // out[row] = y[row] + scaling[its adapter] u[row] W[its adapter]; y null: zeros
    RowGroups g;
    const void *w, *y;
    const float *scaling;                // null: 1
    void *out;
    float *keep;                         // u's parts added up, [rows][rank], or null
    int keep_grouped;
    RankSums u;
    uint64_t ldy, ldo;
    uint32_t cols, rank, wide;           // wide: columns of a workgroup
    int dt, y_dt;
};
hipError_t launch_expand(ExpandArgs a, int cus, hipStream_t stream);

// dw[i] = scaling[i] sum over the rows of adapter i of u[row] z[row]^T, of up to two factors in one launch
struct AdapterGrad {
    const void *z;
    void *dw;                            // [adapters][rank][cols]; null: not wanted
    float *room;                         // parts of groups of more than `chunk` slots
    RankSums u;
    uint64_t ldz;
    uint32_t cols;
};
struct AdapterGradArgs {
    RowGroups g;
    AdapterGrad of[2];
    const float *scaling;
    uint32_t rank, chunk, tiles, join;   // tiles: column tiles of the first factor; join: workgroups that share an adapter's ranks out when parts are added up
    int dt, dw_dt;
};
size_t plan_adapter_grad(AdapterGradArgs &a, int cus);    // chooses chunk; bytes of both rooms, one behind the other
void place_adapter_grad(AdapterGradArgs &a, float *room);
hipError_t launch_adapter_grad(AdapterGradArgs a, hipStream_t stream);

}  // namespace qgemm
