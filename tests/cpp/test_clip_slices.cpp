// Gradient clipping of parameters whose gradients are slices of one buffer, through the second-generation host
// layer's optimizers.  Needs a CUDA device; prints "ALL PASSED" and exits 0.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <stdexcept>
#include <vector>

struct GradFn { int unused; };      // autograd nodes belong to the caller
#include "ctb_host.h"
#include "ops_dispatch.h"
#include "train_utils.h"

#define CHECK(cond)                                                                                                    \
    do {                                                                                                               \
        if (!(cond)) { std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); std::exit(1); }          \
    } while (0)

int main() {
    Tensor flat = Tensor::from_vector({1, 1, 1, 1, 2, 2, 2, 2, 3, 3, 3, 3}, {3, 4});
    Tensor a = Tensor::ones({4}), b = Tensor::ones({2, 2}), again = Tensor::ones({4});
    a.impl->grad = flat.select(0, 0).impl;
    b.impl->grad = flat.select(0, 2).impl;
    again.impl->grad = flat.select(0, 0).impl;               // the same slice twice counts once
    SGD opt({&a, &b, &again}, 0.1);
    const double total = std::sqrt(4 * 1.0 + 4 * 9.0);
    CHECK(std::fabs(opt.clip_grad_norm(100.0) - total) < 1e-12 * total);
    CHECK(std::fabs(opt.clip_grad_norm(total / 4) - total) < 1e-12 * total);
    const float* g = (const float*)flat.impl->data->data.get();
    const float want[3] = {0.25f, 2.0f, 0.75f};               // the slice that belongs to no parameter stays as it was
    for (int i = 0; i < 12; ++i) CHECK(std::fabs(g[i] - want[i / 4]) < 2e-7);
    b.impl->grad = flat.impl;                                // a slice and the whole: neither can be scaled by itself
    bool thrown = false;
    try { opt.clip_grad_norm(0.1); } catch (const std::exception&) { thrown = true; }
    CHECK(thrown);
    for (int i = 0; i < 12; ++i) CHECK(std::fabs(g[i] - want[i / 4]) < 2e-7);
    std::printf("ALL PASSED\n");
    return 0;
}
