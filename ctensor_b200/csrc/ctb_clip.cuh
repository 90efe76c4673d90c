// Host-visible interface of the gradient-norm and clipping kernels (ctb_clip.cu).
#pragma once
#include "ctb_common.cuh"

namespace ctb {

enum { kNormP2 = 0, kNormP1 = 1, kNormInf = 2 };

// One gradient tensor as a run of `n` elements (its memory order does not matter) and where the
// scaled values go (`dst` == `src`: in place).
struct ClipTensor {
    const void* src;
    void* dst;
    int64_t n;
};

// Scratch for `n32` Float32 and `n64` Double64 tensors.
size_t clip_workspace_bytes(int64_t n32, int64_t n64);

// norm = (sum |g|^p)^(1/p) over all tensors of both lists; with `scale` != 0 every tensor is then
// multiplied by max_norm / norm if max_norm < norm < inf, and otherwise copied (nothing happens in place).
int launch_clip(int kind, const ClipTensor* t32, int64_t n32, const ClipTensor* t64, int64_t n64, int scale,
                double max_norm, void* norm, int norm_dtype, void* workspace, cudaStream_t stream);

}  // namespace ctb
