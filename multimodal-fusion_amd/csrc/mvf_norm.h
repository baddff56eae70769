// Launches of the BatchNorm statistics shared with the kernels that fuse a Linear.
#pragma once

#include "mvf_common.h"

namespace mvf {

// Column sums of the workgroups: rows [2][C] of float64 (sum g, sum g * zhat), at most this many.
constexpr int BN_MAX_BLOCKS = 1024;

// Layout of the workspace of mvf_batch_norm_act8_workspace_bytes(C) bytes.
struct Bn8Workspace {
    double *partial;        // [BN_MAX_BLOCKS][2][C]
    float *terms;           // [2][C]: float32 mean (forward); column means of g and g * zhat (backward)
    double *terms64;        // [2][C]: mean and 1 / spread (forward)
};
Bn8Workspace bn8_workspace(void *workspace, int C);

// mean and invstd in float32 (terms, save_invstd) and float64 (terms64): of the batch, from col_sums if
// given, with the running statistics updated and the batch counted in num_batches (may be NULL); or of
// the running statistics.
void bn8_statistics(const float *z, i64 rows, int C, float *running_mean, float *running_var, int training, float momentum,
                    float eps, const double *col_sums, int n_col_sums, long long *num_batches, const Bn8Workspace &w,
                    float *save_invstd, hipStream_t st);

// gradients of weight and bias (may be NULL) and the column means, from nblk rows of w.partial
void bn8_grad_terms(const Bn8Workspace &w, int nblk, int C, i64 rows, float *grad_weight, float *grad_bias, hipStream_t st);

}  // namespace mvf
