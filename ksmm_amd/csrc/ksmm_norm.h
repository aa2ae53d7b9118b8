// What the residual norm's kernels are given.
#pragma once
#include <stdint.h>

namespace ksmm {

struct NormArgs {
    const void *x, *residual;                          // x null: r' is the residual
    const void *gate, *post_weight, *weight, *bias;    // null: 1, no norm of x, 1, 0
    void *r_out = nullptr, *n_out = nullptr;           // null: not wanted
    float *stats = nullptr;                            // mean and factor of x's norm, then of r's: a value a row each
    float alpha, eps;
    int layer, features;
    int64_t batch, group_rows;
};

struct NormGrads {
    const void *dr_out, *dn_out;  // gradients of the results, null: zero
    void *dx, *dresidual;         // null: not wanted
    float *dweight, *dbias, *dpost_weight, *dgate;  // partial sums, null: not wanted
    float *means;                 // of dv and of dv v, a value a row each: for gates of groups batch-size-last, null: not wanted
};

// How the rows are dealt to workgroups where sums over them are taken (batch-size-first).
struct NormSplit {
    int64_t groups, groups_per, part_rows, ranges;
    int parts;
    bool one_gate;
};

}  // namespace ksmm
