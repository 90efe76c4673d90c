// Gradient clipping from many host threads, one after the other, through the first-generation host layer: managed memory
// is set aside once.  Needs a CUDA device; prints "ALL PASSED" and exits 0.
#include <dlfcn.h>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>

struct GradFn { int unused; };      // autograd nodes belong to the caller
#include "ctb_gen1.h"
#include "train_utils.h"

#define CHECK(cond)                                                                                                    \
    do {                                                                                                               \
        if (!(cond)) { std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); std::exit(1); }          \
    } while (0)

// Stands in front of the library's function for the host layer's calls, and counts them.
static int g_blocks = 0;
extern "C" int ctb_alloc_managed(void** ptr, size_t bytes, int zero) {
    ++g_blocks;
    static auto next = (int (*)(void**, size_t, int))dlsym(RTLD_NEXT, "ctb_alloc_managed");
    return next(ptr, bytes, zero);
}

int main() {
    Tensor a({9}, DType::Float32, true);
    for (int i = 0; i < 9; ++i) ((float*)a.impl->storage->grad.get())[i] = 2.0f;
    SGD opt({&a}, 0.1);
    int after_first = 0;
    for (int i = 0; i < 12; ++i) {
        std::thread([&] { CHECK(std::fabs(opt.clip_grad_norm(100.0) - 6.0) < 1e-12); }).join();
        if (i == 0) after_first = g_blocks;
    }
    CHECK(after_first > 0 && g_blocks == after_first);
    std::printf("ALL PASSED\n");
    return 0;
}
