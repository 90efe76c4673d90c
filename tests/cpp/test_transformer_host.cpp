// The transformer-step operators and gradient clipping through the second-generation host layer: known
// answers, gradients against differences, refusals.  Needs a CUDA device; prints "ALL PASSED" and exits 0.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

struct GradFn { int unused; };      // autograd nodes belong to the caller
#include "ctb_host.h"
#include "ops_dispatch.h"
#include "train_utils.h"

#define CHECK(cond)                                                                                                    \
    do {                                                                                                               \
        if (!(cond)) { std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); std::exit(1); }          \
    } while (0)
#define CHECK_NEAR(a, b, eps) CHECK(std::fabs(double(a) - double(b)) <= (eps))
#define CHECK_THROWS(expr, text)                                                                                       \
    do {                                                                                                               \
        bool ok = false;                                                                                               \
        try { (void)(expr); } catch (const std::exception& e) { ok = std::string(e.what()).find(text) != std::string::npos; } \
        CHECK(ok);                                                                                                     \
    } while (0)

namespace {

unsigned g_state = 12345;
double uniform() {                   // a small generator of the test's own: the same values everywhere
    g_state = g_state * 1664525u + 1013904223u;
    return (g_state >> 8) / 16777216.0 * 2.0 - 1.0;
}
Tensor random_tensor(const std::vector<size_t>& shape) {
    size_t n = 1;
    for (size_t d : shape) n *= d;
    std::vector<double> v(n);
    for (double& x : v) x = (double)(float)uniform();
    return Tensor::from_vector(v, shape);
}
Tensor int_tensor(const std::vector<double>& v, const std::vector<size_t>& shape) { return Tensor::from_vector(v, shape, DType::Int32); }
float* data(const Tensor& t) { return (float*)t.impl->data->data.get() + t.impl->offset; }
double dot(const Tensor& a, const Tensor& b) {
    double s = 0.0;
    for (size_t i = 0; i < a.numel(); ++i) s += (double)data(a)[i] * data(b)[i];
    return s;
}

void scores() {
    // one head, three queries, four keys, causal, cap 2, bias 0.5 per position
    const size_t Q = 3, K = 4;
    Tensor s = random_tensor({1, 1, Q, K});
    ctb_host::ScoreRules rules;
    rules.scale = 3.0;
    rules.cap = 2.0;
    rules.causal = true;
    rules.slopes = Tensor::full({1}, 0.5);
    auto plain = [&](const std::vector<double>& x, double slope, std::vector<double>* p) {
        for (size_t i = 0; i < Q; ++i) {
            const size_t pos = i + K - Q;
            double z = 0.0;
            for (size_t j = 0; j <= pos; ++j) z += std::exp(2.0 * std::tanh(3.0 * x[i * K + j] / 2.0) - slope * (double)(pos - j));
            for (size_t j = 0; j < K; ++j) (*p)[i * K + j] = j <= pos ? std::exp(2.0 * std::tanh(3.0 * x[i * K + j] / 2.0) - slope * (double)(pos - j)) / z : 0.0;
        }
    };
    std::vector<double> x(data(s), data(s) + Q * K), p(Q * K);
    plain(x, 0.5, &p);
    Tensor got = ctb_host::score_softmax(s, rules);
    for (size_t i = 0; i < Q * K; ++i) CHECK_NEAR(data(got)[i], p[i], 1e-6);
    // gradients against central differences (step^2 times a third derivative of a few units, and fp32)
    Tensor grad = random_tensor({1, 1, Q, K}), slope_grad;
    Tensor ds = ctb_host::score_softmax_backward(grad, got, rules, s, &slope_grad);
    auto loss = [&](const std::vector<double>& at, double slope) {
        std::vector<double> q(Q * K);
        plain(at, slope, &q);
        double l = 0.0;
        for (size_t i = 0; i < Q * K; ++i) l += q[i] * data(grad)[i];
        return l;
    };
    const double step = 1e-4;
    for (size_t i = 0; i < Q * K; ++i) {
        std::vector<double> a = x, b = x;
        a[i] += step;
        b[i] -= step;
        CHECK_NEAR(data(ds)[i], (loss(a, 0.5) - loss(b, 0.5)) / (2 * step), 2e-6);
    }
    CHECK_NEAR(data(slope_grad)[0], (loss(x, 0.5 + step) - loss(x, 0.5 - step)) / (2 * step), 2e-6);
    // documents and an empty row: the second query belongs to no document of the keys
    ctb_host::ScoreRules docs;
    docs.query_docs = int_tensor({0, 7, 1}, {1, 3});
    docs.key_docs = int_tensor({0, 0, 1, 1}, {1, 4});
    Tensor d = ctb_host::score_softmax(Tensor::zeros({1, 1, 3, 4}), docs);
    const double want[12] = {0.5, 0.5, 0, 0, 0, 0, 0, 0, 0, 0, 0.5, 0.5};
    for (size_t i = 0; i < 12; ++i) CHECK(data(d)[i] == (float)want[i]);
    docs.key_docs = Tensor();
    CHECK_THROWS(ctb_host::score_softmax(s, docs), "come together");
    CHECK_THROWS(ctb_host::score_softmax(Tensor::zeros({3, 4}), ctb_host::ScoreRules()), "4D");
    CHECK_THROWS(ctb_host::score_softmax_backward(grad, got, rules), "scores are needed");
    CHECK_THROWS(ctb_host::score_softmax(Tensor(), rules), "null input");
}

void norms() {
    const size_t T = 5, C = 12;
    Tensor x = random_tensor({T, C}), f = random_tensor({T, C}), gate = random_tensor({C}), dy = random_tensor({T, C}), dh = random_tensor({T, C});
    ctb_host::ResidualNorm params;
    params.post = ctb_host::NormKind::RMS;
    params.pre = ctb_host::NormKind::Layer;
    params.scale = 0.5;
    params.post_weight = random_tensor({C});
    params.pre_weight = random_tensor({C});
    params.pre_bias = random_tensor({C});
    std::vector<Tensor> ins = {x, f, gate, params.post_weight, params.pre_weight, params.pre_bias};
    // the sum of <y, dy> and <h, dh> with input `which` moved by t * way
    auto loss = [&](int which, const std::vector<double>& way, double t, std::vector<double>* ys, std::vector<double>* hs) {
        std::vector<std::vector<double>> v;
        for (size_t k = 0; k < ins.size(); ++k) {
            v.emplace_back(data(ins[k]), data(ins[k]) + ins[k].numel());
            if ((int)k == which)
                for (size_t i = 0; i < way.size(); ++i) v[k][i] += t * way[i];
        }
        double l = 0.0;
        for (size_t r = 0; r < T; ++r) {
            std::vector<double> y(C);
            double sq = 0.0, mean = 0.0, var = 0.0;
            for (size_t c = 0; c < C; ++c) sq += v[1][r * C + c] * v[1][r * C + c] / C;
            for (size_t c = 0; c < C; ++c) {
                y[c] = v[0][r * C + c] + 0.5 * v[2][c] * v[1][r * C + c] / std::sqrt(sq + 1e-5) * v[3][c];
                mean += y[c] / C;
            }
            for (size_t c = 0; c < C; ++c) var += (y[c] - mean) * (y[c] - mean) / C;
            for (size_t c = 0; c < C; ++c) {
                const double h = (y[c] - mean) / std::sqrt(var + 1e-5) * v[4][c] + v[5][c];
                l += y[c] * data(dy)[r * C + c] + h * data(dh)[r * C + c];
                if (ys) { (*ys)[r * C + c] = y[c]; (*hs)[r * C + c] = h; }
            }
        }
        return l;
    };
    std::vector<double> ys(T * C), hs(T * C);
    loss(-1, {}, 0.0, &ys, &hs);
    const ctb_host::ResidualNormResult r = ctb_host::residual_norm(x, f, params, gate);
    for (size_t i = 0; i < T * C; ++i) {
        CHECK_NEAR(data(r.y)[i], ys[i], 1e-6);
        CHECK_NEAR(data(r.h)[i], hs[i], 4e-6);
    }
    CHECK(r.stats.shape() == (std::vector<size_t>{T, 4}));
    const ctb_host::ResidualNormGrads g = ctb_host::residual_norm_backward(f, r, params, dy, dh, gate);
    const Tensor grads[6] = {g.x, g.f, g.gate, g.post_weight, g.pre_weight, g.pre_bias};
    CHECK(!g.post_bias.impl);
    for (int k = 0; k < 6; ++k) {
        CHECK(grads[k].shape() == ins[k].shape());
        std::vector<double> way(ins[k].numel());
        double got = 0.0, size = 0.0;
        for (size_t i = 0; i < way.size(); ++i) {
            way[i] = uniform();
            got += data(grads[k])[i] * way[i];
            size += std::fabs(data(grads[k])[i] * way[i]);
        }
        const double step = 1e-5;
        CHECK_NEAR(got, (loss(k, way, step, nullptr, nullptr) - loss(k, way, -step, nullptr, nullptr)) / (2 * step), 1e-5 * (1 + size));
    }
    // the first norm of a network: no block output yet
    ctb_host::ResidualNorm entry;
    const ctb_host::ResidualNormResult e = ctb_host::residual_norm(x, Tensor(), entry);
    CHECK(e.y.impl == x.impl);
    double mean = 0.0;
    for (size_t c = 0; c < C; ++c) mean += data(e.h)[c] / C;
    CHECK_NEAR(mean, 0.0, 1e-6);
    CHECK_THROWS(ctb_host::residual_norm(x, Tensor(), params), "without a block output");
    CHECK_THROWS(ctb_host::residual_norm(x, random_tensor({T, C + 1}), entry), "shapes differ");
    CHECK_THROWS(ctb_host::residual_norm(Tensor(), f, entry), "null input");
}

Tensor parameter(const std::vector<size_t>& shape, double grad, DType dt = DType::Float32) {
    Tensor p = Tensor::full(shape, 1.0, dt);
    Tensor g = Tensor::full(shape, grad, dt);
    p.impl->grad = g.impl;
    return p;
}

void clipping() {
    Tensor a = parameter({4, 3}, 1.0), b = parameter({5}, 2.0), none = Tensor::ones({7}), d = parameter({3}, 4.0, DType::Double64);
    SGD opt({&a, nullptr, &none, &b, &a, &d}, 0.1);          // a twice: its buffer counts once
    const double total = std::sqrt(12 * 1.0 + 5 * 4.0 + 3 * 16.0);
    CHECK_NEAR(opt.clip_grad_norm(100.0), total, 1e-12 * total);
    CHECK(a.grad()[0][0] == 1.0 && b.grad()[4] == 2.0);        // below the limit: as they were
    CHECK_NEAR(opt.clip_grad_norm(100.0, 1.0), 12 + 10 + 12, 1e-12);
    CHECK_NEAR(opt.clip_grad_norm(100.0, INFINITY), 4.0, 1e-12);
    CHECK_NEAR(opt.clip_grad_norm(total / 4), total, 1e-12 * total);
    CHECK_NEAR(a.grad()[3][2], 0.25, 1e-7);
    CHECK_NEAR(b.grad()[0], 0.5, 2e-7);
    CHECK_NEAR(d.grad()[1], 1.0, 1e-12);
    SGD step({&a, &b, &d}, 0.1);
    step.step();
    CHECK_NEAR(a[0][0], 1.0 - 0.025, 2e-7);
    CHECK_NEAR(d[2], 0.9, 1e-7);
    CHECK_THROWS(opt.clip_grad_norm(-1.0), "max_norm");
    CHECK_THROWS(opt.clip_grad_norm(1.0, 3.0), "p must be");
    SGD empty({}, 0.1);
    CHECK(empty.clip_grad_norm(1.0) == 0.0);
}

}  // namespace

int main() {
    scores();
    norms();
    clipping();
    std::printf("ALL PASSED\n");
    return 0;
}
