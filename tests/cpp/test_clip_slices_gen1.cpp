// Gradient clipping of parameters that are slices of one tensor, through the first-generation host layer's
// optimizers.  Needs a CUDA device; prints "ALL PASSED" and exits 0.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

struct GradFn { int unused; };      // autograd nodes belong to the caller
#include "ctb_gen1.h"
#include "train_utils.h"

#define CHECK(cond)                                                                                                    \
    do {                                                                                                               \
        if (!(cond)) { std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); std::exit(1); }          \
    } while (0)

int main() {
    Tensor flat({3, 4}, DType::Float32, true);
    float* g = (float*)flat.impl->storage->grad.get();
    for (int i = 0; i < 12; ++i) g[i] = 1.0f + i / 4;
    Tensor a = flat.select(0, 0), b = flat.select(0, 2);
    SGD opt({&a, &b, &a}, 0.1);
    const double total = std::sqrt(4 * 1.0 + 4 * 9.0);
    CHECK(std::fabs(opt.clip_grad_norm(100.0) - total) < 1e-12 * total);
    CHECK(std::fabs(opt.clip_grad_norm(total / 4) - total) < 1e-12 * total);
    const float want[3] = {0.25f, 2.0f, 0.75f};               // the slice that was not named stays as it was
    for (int i = 0; i < 12; ++i) CHECK(std::fabs(g[i] - want[i / 4]) < 2e-7);
    std::printf("ALL PASSED\n");
    return 0;
}
