// Host interface of the 32 x 32 MFMA projection kernel (iq3s_wide.hip).
#pragma once
#include "experts.h"

// Launch shape of gemm_wide_kernel for one call.
struct WidePlan {
    int mt;     // 32-token sub-tiles per workgroup
    int waves;  // per K group, 32 weight rows each
    int kg;     // K groups of waves per workgroup
    int splits; // K slices (more than one: f32 atomics into outputs zeroed beforehand)
    int bps;    // K blocks per slice
    double us;  // what the plan's cost model expects of it
};

// Whether the kernel takes the call (it can, and is the faster choice), and its plan. other: the
// configuration that takes the call otherwise.
bool mambo_wide_plan(int64_t m, const mambo_projection *proj, int count, int64_t blocks, int64_t ldxv,
                     const uint8_t *xs, int64_t ldxs, const mambo_gemm_config &other, WidePlan *plan);

// Queues the launch; the caller has checked the operands and zeroed the outputs of a plan with
// several slices.
int mambo_wide_launch(const WidePlan &plan, const uint8_t *xv, int64_t ldxv, const uint8_t *xs, int64_t ldxs, int64_t m,
                      const mambo_projection *proj, int count, int64_t blocks, hipStream_t stream);

// Rows grouped by expert: the plan for the tiles of 64 and of 128 rows that are expected (tiles_of), and its launch. The caller has checked the operands, that the offsets of all rows fit 32 bits where they are gathered, and that
// expert_row_tiles of 64 rows fit a grid's y.
void mambo_wide_experts_plan(const ExpertRows &er, int64_t n, int64_t blocks, double tiles_of[2], WidePlan *plan);
int mambo_wide_experts_launch(const WidePlan &plan, const uint8_t *xv, int64_t ldxv, const uint8_t *xs, int64_t ldxs,
                              const ExpertRows &er, const uint8_t *packed, int64_t expert_stride, int64_t n, int64_t blocks,
                              void *out, bool bf16, int64_t ldo, hipStream_t stream);
