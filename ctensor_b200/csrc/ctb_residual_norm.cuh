// Host-visible interface of the residual-norm kernels (ctb_residual_norm.cu).
#pragma once
#include "ctb_common.cuh"

namespace ctb {

// Rows of `cols` floats at a fixed distance, columns contiguous.
struct RowsIn {
    const float* p;
    int64_t stride;
};

// How the gate varies: kGateRow = one row of `cols` values for every `gate_rows` consecutive rows,
// kGateScalar = one value for every `gate_rows` consecutive rows.
enum { kGateNone = 0, kGateRow = 1, kGateScalar = 2 };

struct ResidualNormGeom {
    int64_t rows;                       // < 2^31
    int64_t cols;                       // <= kResidualNormMaxCols
    int32_t post_kind, pre_kind;        // CTB_NORM_*
    float post_eps, pre_eps, scale;
    const float *post_weight, *post_bias, *pre_weight, *pre_bias;      // [cols] or NULL
    int32_t gate_mode;
    int64_t gate_rows;                  // rows that share a gate row / value
    RowsIn gate;                        // stride: between one gate row / value and the next
    double inv_cols;                    // these two are set by the launchers
    FastDiv by_gate_rows;
};
constexpr int64_t kResidualNormMaxCols = 32768;

int launch_residual_norm(const ResidualNormGeom& g, RowsIn x, RowsIn f, float* y, float* h, float* stats, cudaStream_t stream);

struct ResidualNormGrads {
    float *x, *f, *gate, *post_weight, *post_bias, *pre_weight, *pre_bias;      // NULL: not wanted
};
// `gate_groups`: gate rows / values whose gradient is summed over rows or columns (0: none), each `gate_width` wide.
size_t residual_norm_workspace_bytes(int64_t rows, int64_t cols, int64_t gate_groups, int64_t gate_width);
int launch_residual_norm_backward(const ResidualNormGeom& g, RowsIn f, RowsIn y, const float* stats, RowsIn grad_y, RowsIn grad_h,
                                  const ResidualNormGrads& out, void* workspace, cudaStream_t stream);

}  // namespace ctb
