// The block norms (residual_norm.cuh): what the kernels take, how a call is cut, and the launchers, one file per type.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"

namespace pcb {

struct RNParams {
    int comps, n, features, groups, per_group;     // groups: rows of the gate per component (0: no gate); per_group: samples of each
    uint32_t magic;                                // ceil(2^32 / features): e / features = umulhi(e, magic) for the widths below (0: features == 1)
    float scale, eps;
    const void *x, *branch, *gate;
    const float *post, *pre;
    void *y, *h;
    float* stats;                                  // [2][n]: r(branch), r(y)
    // backward
    const void *dy, *dh;
    void *dx, *dbranch, *dgate;
    float *dpost, *dpre;
    float *part_w;                                 // [CTAs][2][comps * features]: dpre, dpost
    float *part_gate;                              // [groups * parts][comps * features]
    int parts, items;                              // pieces per group
};

// Warps per row, values per thread and rows of a CTA (one per SM) for a width; warps 0: wider than the registers.
struct RNShape { int warps, values, rows; };
inline RNShape fwd_shape(long long width) {
    if (width <= 32 * 8) return {1, 8, 16};
    if (width <= 32 * 32) return {1, 32, 12};
    if (width <= 128 * 16) return {4, 16, 4};
    if (width <= 128 * 32) return {4, 32, 3};
    if (width <= 256 * 32) return {8, 32, 1};
    if (width <= 512 * 32) return {16, 32, 1};
    return {0, 0, 1};
}
inline RNShape bwd_shape(long long width) {
    if (width <= 32 * 8) return {1, 8, 16};
    if (width <= 32 * 16) return {1, 16, 12};
    if (width <= 128 * 16) return {4, 16, 3};
    if (width <= 256 * 16) return {8, 16, 2};
    if (width <= 512 * 16) return {16, 16, 1};
    return {0, 0, 1};
}

struct RNPlan { RNShape shape; int grid, slots, parts, items; size_t part_w, part_gate, total; };
inline RNPlan bwd_plan(int comps, int n, int features, int groups) {
    RNPlan q = {};
    const long long width = (long long)comps * features;
    q.shape = bwd_shape(width);
    const int rows_per_cta = q.shape.rows, most = tc::device_sms() * (q.shape.warps ? rows_per_cta : 4);      // (wide rows: four CTAs on an SM)
    const bool shared = groups > 0 && groups < n;
    const int g = shared || (groups == n && n > 0) ? groups : 1;
    if (groups == n && groups > 1 && !shared) { q.parts = 1; q.items = n; }          // a gate for each value: every sample is an item
    else {
        // pieces per group: as many as fill the machine for one to eight rounds, whichever has the fewest rounds x samples per piece
        const int per = n / g;
        long long best = -1;
        for (long long rounds = 1; rounds <= 8; ++rounds) {
            const long long fit = rounds * most / g, parts = fit < 1 ? 1 : (fit < per ? fit : per);
            const long long cost = (g * parts + most - 1) / most * ((per + parts - 1) / parts);
            if (best < 0 || cost < best) { best = cost; q.parts = (int)parts; }
        }
        q.items = g * q.parts;
    }
    const int want = q.items < most ? q.items : most;
    q.grid = (want + rows_per_cta - 1) / rows_per_cta;
    q.slots = q.grid;                                   // sums of the weights' gradients: one set per CTA
    q.part_w = (size_t)q.slots * 2 * width * 4;
    q.part_gate = shared && (q.parts > 1 || q.shape.warps == 0) ? (size_t)q.items * width * 4 : (groups == n && n > 0 && q.shape.warps == 0 ? (size_t)n * width * 4 : 0);
    q.total = q.part_w + q.part_gate;
    return q;
}

#define PCB_NORM_LAUNCHERS(name)                                                     \
    int norm_fwd_##name(const RNParams& p, cudaStream_t stream);                     \
    int norm_bwd_##name(const RNParams& p, const RNPlan& plan, cudaStream_t stream);
PCB_NORM_LAUNCHERS(f32)
PCB_NORM_LAUNCHERS(f16)
PCB_NORM_LAUNCHERS(bf16)

}  // namespace pcb
