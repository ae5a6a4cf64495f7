// The block norms (residual_norm.cuh): what the kernels take, how a call is cut, and the launchers, one file per type.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"

namespace pcb {

struct RNParams {
    int comps, n, features, groups, per_group;     // groups: rows of the gate per component (0: no gate); per_group: samples of each
    int period;                                    // rows that start at different places within 16 bytes
    float scale, eps;
    const void *x, *branch, *gate;
    const float *post, *pre;
    void *y, *h;
    float* stats;                                  // [2][n]: r(branch), r(y)
    // backward
    const void *dy, *dh;
    void *dx, *dbranch, *dgate;
    float *dpost, *dpre;
    uint8_t* workspace;                            // where the sums lie
    int* status;                                   // the call's status word, which the first CTA resets (the call has no waits to report)
    float *part_w;                                 // [CTAs][2][comps * features]: dpre, dpost
    float *part_gate;                              // [groups * parts][comps * features]
    int parts, pieces, items;                      // per group: sums that make its gate's gradient, pieces of each class's rows; pieces in all
};

// Warps per row, values per thread and rows of a CTA (one per SM) for a width; warps 0: wider than the registers. A thread's values are few enough that the backward pass keeps a row
// of four tensors in registers, and idle lanes cost rows in flight: backward, 3001 x (4 x 509) f16 30 us with five warps a row, 41 with eight; 16384 x 1024 bf16 40 with two, 57 with
// four; 16384 x 1536 bf16 55 with three, 61 with four; forward 3001 x (4 x 509) 20 with five of 16 values, 26 with four of 32.
struct RNShape { int warps, values, rows; };
inline RNShape fwd_shape(long long width) {
    if (width <= 32 * 8) return {1, 8, 16};
    if (width <= 32 * 32) return {1, 32, 12};
    if (width <= 128 * 16) return {4, 16, 4};
    if (width <= 160 * 16) return {5, 16, 3};
    if (width <= 128 * 32) return {4, 32, 3};
    if (width <= 256 * 32) return {8, 32, 1};
    if (width <= 512 * 32) return {16, 32, 1};
    return {0, 0, 1};
}
inline RNShape bwd_shape(long long width) {
    if (width <= 32 * 8) return {1, 8, 16};
    if (width <= 32 * 16) return {1, 16, 12};
    if (width <= 64 * 16) return {2, 16, 6};
    if (width <= 96 * 16) return {3, 16, 4};
    if (width <= 128 * 16) return {4, 16, 3};
    if (width <= 160 * 16) return {5, 16, 3};
    if (width <= 256 * 16) return {8, 16, 2};
    if (width <= 512 * 16) return {16, 16, 1};
    return {0, 0, 1};
}

// Rows after which a row starts at the same place within 16 bytes again, and values of a row with those that its vectors reach over.
inline int row_period(int features, int size) {
    const int bytes = features * size % 16;
    return bytes == 0 ? 1 : (bytes % 8 == 0 ? 2 : (bytes % 4 == 0 ? 4 : 8));
}
inline long long padded_width(int comps, int features, int size) {
    const int vec = 16 / size;
    return row_period(features, size) == 1 ? (long long)comps * features : (long long)comps * ((features + 2 * vec - 2) / vec) * vec;
}

// How a backward call is cut, and the bytes of its sums.
struct RNPlan { RNShape shape; int grid, parts, pieces, items; size_t part_w, part_gate, total; };
// Pieces of a group's `per` rows where `groups` of them share `most` workers: as many as fill those for one to eight rounds, whichever has the fewest rounds x rows
// per piece.
inline int pieces_of(int groups, int per, long long most) {
    long long best = -1;
    int pieces = 1;
    for (long long rounds = 1; rounds <= 8; ++rounds) {
        const long long fit = rounds * most / groups, n = fit < 1 ? 1 : (fit < per ? fit : per);
        const long long cost = (groups * n + most - 1) / most * ((per + n - 1) / n);
        if (best < 0 || cost < best) { best = cost; pieces = (int)n; }
    }
    return pieces;
}
// (A gate for each value has no sums over samples: its gradient is written where it is made.)
inline void sums_of(RNPlan& q, long long width, int gates, int n) {
    q.part_w = (size_t)q.grid * 2 * width * 4;
    q.part_gate = gates > 0 && gates < n && (q.shape.warps == 0 || q.parts > 1) ? (size_t)gates * q.parts * width * 4 : 0;
    q.total = q.part_w + q.part_gate;
}
// Rows wider than the registers, tensors that start anywhere, and groups of fewer rows than there are places for them to start at: four CTAs on an SM, a row each.
inline RNPlan wide_plan(int comps, int n, int features, int gates) {
    RNPlan q = {};
    const int groups = gates > 0 ? gates : 1;
    const long long most = 4LL * tc::device_sms();
    q.parts = q.pieces = pieces_of(groups, n / groups, most);
    q.items = groups * q.parts;
    q.grid = (int)(q.items < most ? q.items : most);
    sums_of(q, (long long)comps * features, gates, n);
    return q;
}
inline RNPlan bwd_plan(int comps, int n, int features, int gates, int size) {
    const int period = row_period(features, size);
    const bool shared = gates > 0 && gates < n;
    RNPlan q = {};
    q.shape = bwd_shape(padded_width(comps, features, size));
    if (q.shape.warps == 0 || (shared && n / gates < period)) return wide_plan(comps, n, features, gates);
    const int sms = tc::device_sms(), rows = q.shape.rows;
    q.pieces = shared ? pieces_of(gates, n / gates / period, (long long)(sms / period > 0 ? sms / period : 1) * rows) : 1;
    q.parts = shared ? q.pieces * period : 1;
    // a CTA for each place that rows start at, at least, and no more than have work
    const long long work = shared ? (long long)gates * q.pieces : (n + period - 1) / period;
    long long per_class = (work + rows - 1) / rows;
    if (per_class * period > sms) per_class = sms / period > 0 ? sms / period : 1;
    q.grid = (int)(per_class * period);
    if (!shared && q.grid > n) q.grid = n;
    sums_of(q, (long long)comps * features, gates, n);
    // (a call whose tensors do not start on 16 bytes takes the other plan: room for either)
    const RNPlan w = wide_plan(comps, n, features, gates);
    q.total = q.total > w.total ? q.total : w.total;
    return q;
}

#define PCB_NORM_LAUNCHERS(name)                                                     \
    int norm_fwd_##name(const RNParams& p, cudaStream_t stream);                     \
    int norm_bwd_##name(const RNParams& p, const RNPlan& plan, cudaStream_t stream);
PCB_NORM_LAUNCHERS(f32)
PCB_NORM_LAUNCHERS(f16)
PCB_NORM_LAUNCHERS(bf16)

}  // namespace pcb
