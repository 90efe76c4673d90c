// Gradient clipping through the first-generation host layer's optimizers.  Needs a CUDA device; prints
// "ALL PASSED" and exits 0.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <stdexcept>
#include <string>
#include <vector>

struct GradFn { int unused; };      // autograd nodes belong to the caller
#include "ctb_gen1.h"
#include "train_utils.h"

#define CHECK(cond)                                                                                                    \
    do {                                                                                                               \
        if (!(cond)) { std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); std::exit(1); }          \
    } while (0)

namespace {
Tensor parameter(size_t n, float grad) {
    Tensor p({n}, DType::Float32, true);
    float *data = (float*)p.impl->storage->data.get(), *g = (float*)p.impl->storage->grad.get();
    for (size_t i = 0; i < n; ++i) { data[i] = 1.0f; g[i] = grad; }
    return p;
}
float grad_at(const Tensor& t, size_t i) { return ((float*)t.impl->storage->grad.get())[i]; }
}  // namespace

int main() {
    Tensor a = parameter(12, 1.0f), b = parameter(5, 2.0f), none({7}, DType::Float32, false);
    SGD opt({&a, nullptr, &none, &b, &a}, 0.1);
    const double total = std::sqrt(12.0 + 20.0);
    CHECK(std::fabs(opt.clip_grad_norm(100.0) - total) < 1e-12 * total);
    CHECK(grad_at(a, 0) == 1.0f && grad_at(b, 4) == 2.0f);
    CHECK(std::fabs(opt.clip_grad_norm(total / 4) - total) < 1e-12 * total);
    CHECK(std::fabs(grad_at(a, 11) - 0.25) < 1e-7 && std::fabs(grad_at(b, 0) - 0.5) < 2e-7);
    SGD step({&a, &b}, 0.1);
    step.step();
    CHECK(std::fabs(((float*)a.impl->storage->data.get())[3] - 0.975) < 2e-7);
    bool thrown = false;
    try { opt.clip_grad_norm(std::nan("")); } catch (const std::exception& e) { thrown = std::string(e.what()).find("max_norm") != std::string::npos; }
    CHECK(thrown);
    std::printf("ALL PASSED\n");
    return 0;
}
