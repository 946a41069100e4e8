// GPU tests of the tracked head_token_log_probs of the C++ host mirror (noetic_tensor_b200/host/noetic_rl.hpp) under vocabulary
// masks (bytes or bits, a row each or one for all) and temperatures, with log-prob and entropy terms in one backward: the second
// node's gradients are added to the first one's. Against f64 on the host. Run by tests/test_gpu_head_cpp_tape.py.
#include <cmath>
#include <cstdio>
#include <random>

#include "../../noetic_tensor_b200/host/noetic_rl.hpp"

using namespace noetic;
namespace rl = noetic::nn::rl;
using rl::TokenReduction;

static int g_checks = 0;
static const Device dev = Device::Cuda(0);
#define CHECK(cond, ...)                                                    \
    do {                                                                    \
        g_checks++;                                                         \
        if (!(cond)) {                                                      \
            std::printf("FAILED %s:%d: %s\n  ", __FILE__, __LINE__, #cond); \
            std::printf(__VA_ARGS__);                                       \
            std::printf("\n");                                              \
            std::exit(1);                                                   \
        }                                                                   \
    } while (0)

static float through_bf16(float x) {
    uint32_t b = (uint32_t)bf16_from_f32(x) << 16;
    float y;
    std::memcpy(&y, &b, 4);
    return y;
}

constexpr size_t S = 2, B = 2, T = 19, d = 72, V = 264, N = S * B * T, WORDS = (V + 31) / 32;
static std::vector<float> x(N* d), w(d* V), adv(N), mask(N);
static std::vector<int64_t> tok(N);
static std::vector<uint8_t> allow(N* V);

static void make() {
    std::mt19937 gen(23);
    std::normal_distribution<float> nd(0.f, 1.f);
    for (auto& v : x) v = through_bf16(nd(gen));
    for (auto& v : w) v = through_bf16(nd(gen) * 0.35f);
    for (size_t i = 0; i < N; i++) {
        tok[i] = (int64_t)(gen() % V);
        adv[i] = nd(gen);
        mask[i] = gen() % 4 ? 1.f : 0.f;
    }
    for (auto& v : allow) v = gen() % 3 == 0;
    for (size_t r = 0; r < N; r++) allow[r * V + tok[r]] = 1;
    for (size_t r = 0; r < N; r++) allow[tok[r]] = 1;  // the first row serves all rows too
}

struct Truth {
    std::vector<double> lp, H, dx, dw, ex, ew;  // values; gradients and the majorants of their rounding
};
// loss = Σ_s Σ −lp·adv·mask / count_s + β Σ H, from hidden states xs normalised by the statistics of x
static Truth truth(const std::vector<double>& xs, double beta, double tau, bool masked, bool shared) {
    Truth t;
    t.lp.resize(N); t.H.resize(N); t.dx.assign(N * d, 0.0); t.dw.assign(d * V, 0.0); t.ex.assign(N * d, 0.0); t.ew.assign(d * V, 0.0);
    for (size_t r = 0; r < N; r++) {
        double count = 0.0;
        for (size_t i = 0; i < B * T; i++) count += mask[r / (B * T) * B * T + i];
        const double a = -(double)adv[r] * mask[r] / std::max(count, 1.0), b = beta;
        auto on = [&](size_t v) { return !masked || allow[(shared ? 0 : r) * V + v] != 0; };
        std::vector<double> z(V, 0.0), zs(V, 0.0);
        for (size_t k = 0; k < d; k++)
            for (size_t v = 0; v < V; v++) {
                z[v] += (double)x[r * d + k] * w[k * V + v] / tau;
                zs[v] += xs[r * d + k] * w[k * V + v] / tau;
            }
        double m = -1e300, Z = 0.0;
        for (size_t v = 0; v < V; v++)
            if (on(v)) m = std::max(m, z[v]);
        for (size_t v = 0; v < V; v++)
            if (on(v)) Z += std::exp(z[v] - m);
        const double lse = m + std::log(Z);
        double H = 0.0;
        for (size_t v = 0; v < V; v++)
            if (on(v)) H -= std::exp(z[v] - lse) * (z[v] - lse);
        t.lp[r] = z[tok[r]] - lse;
        t.H[r] = H;
        for (size_t v = 0; v < V; v++) {
            if (!on(v)) continue;
            const double l = zs[v] - lse, p = std::exp(l), hot = (int64_t)v == tok[r] ? 1.0 : 0.0;
            const double g = (a * (hot - p) - b * p * (l + H)) / tau, D = (std::fabs(a) * (hot + p) + std::fabs(b) * p * (std::fabs(l) + H + 1.0)) / tau;
            for (size_t k = 0; k < d; k++) {
                t.dx[r * d + k] += g * w[k * V + v];
                t.dw[k * V + v] += xs[r * d + k] * g;
                t.ex[r * d + k] += D * std::fabs(w[k * V + v]);
                t.ew[k * V + v] += std::fabs(xs[r * d + k]) * D;
            }
        }
    }
    return t;
}
// an entry of each node's ∂/∂z is rounded to bf16 once (2^-8 of itself), sums and exponentials are f32
static void held(const std::vector<float>& got, const std::vector<double>& want, const std::vector<double>& major, const char* what) {
    for (size_t i = 0; i < got.size(); i++) {
        const double tol = (std::ldexp(1.0, -8) + 1e-4) * major[i] + 1e-6 * std::fabs(want[i]);
        CHECK(std::fabs(got[i] - want[i]) <= tol, "%s[%zu]: got %.9g, want %.9g, tolerance %.3e", what, i, (double)got[i], want[i], tol);
    }
}

enum Form { kNone, kBytes, kByteRow, kBits, kBitRow };
static Tensor mask_tensor(Form f) {
    const size_t rows = f == kByteRow || f == kBitRow ? 1 : N;
    if (f == kBytes || f == kByteRow) return Tensor::from_u8(std::vector<uint8_t>(allow.begin(), allow.begin() + rows * V), {rows, V}, dev);
    std::vector<int32_t> bits(rows * WORDS, 0);
    for (size_t r = 0; r < rows; r++)
        for (size_t v = 0; v < V; v++)
            if (allow[r * V + v]) bits[r * WORDS + v / 32] |= (int32_t)(1u << (v % 32));
    Tensor t = Tensor::empty({rows, WORDS}, DType::I32, dev);
    cu(cudaMemcpy(t.ptr(), bits.data(), bits.size() * 4, cudaMemcpyHostToDevice), "upload bits");
    return t;
}

static void test(Form form, double tau, bool checkpoint) {
    const Tensor hx = Tensor::from_f32(x, {S, B, T, d}, dev, DType::BF16).require_grad(), hw = Tensor::from_f32(w, {d, V}, dev, DType::BF16).require_grad();
    const Tensor hm = Tensor::from_f32(mask, {S, B, T}, dev), ha = Tensor::from_f32(adv, {S, B, T}, dev);
    const bool masked = form != kNone, shared = form == kByteRow || form == kBitRow;
    Tensor vm;
    if (masked) vm = mask_tensor(form);
    Tensor ent;
    const Tensor lp = rl::head_token_log_probs(hx, hw, IntTensor::from_data(tok, {S, B, T}), &ent, false, masked ? &vm : nullptr, tau, checkpoint);
    std::vector<double> xs(x.begin(), x.end());
    if (checkpoint)
        for (size_t r = 0; r < N; r++) {
            float big = 0.f;
            for (size_t k = 0; k < d; k++) big = std::max(big, std::fabs(x[r * d + k]));
            for (size_t k = 0; k < d; k++) xs[r * d + k] = std::nearbyint(127.0 * x[r * d + k] / big) * (double)(float)((double)big / 127.0);
        }
    const double beta = 0.01;
    const Truth t = truth(xs, beta, tau, masked, shared);
    const std::vector<float> glp = lp.to_vec(), gH = ent.to_vec();
    for (size_t r = 0; r < N; r++) {
        CHECK(std::fabs(glp[r] - t.lp[r]) <= 2e-5 * (1 + std::fabs(t.lp[r])), "log-prob %zu: %.9g, %.9g", r, (double)glp[r], t.lp[r]);
        CHECK(std::fabs(gH[r] - t.H[r]) <= 2e-5 * (1 + std::fabs(t.H[r])), "entropy %zu: %.9g, %.9g", r, (double)gH[r], t.H[r]);
    }
    const Tensor pg = rl::policy_gradient_loss(lp, ha, &hm, TokenReduction::TokenMean);
    const Gradients g = backward({{pg, 1.0}, {ent, beta}});
    CHECK(g.grad(hx) && g.grad(hw), "gradients of both");
    held(g.grad(hx)->to_vec(), t.dx, t.ex, "d hidden");
    held(g.grad(hw)->to_vec(), t.dw, t.ew, "d weight");
    // the same states and weight through two calls: four nodes add up
    Tensor ent2;
    const Tensor lp2 = rl::head_token_log_probs(hx, hw, IntTensor::from_data(tok, {S, B, T}), &ent2, false, masked ? &vm : nullptr, tau, checkpoint);
    const Gradients twice = backward({{pg, 1.0}, {ent, beta}, {rl::policy_gradient_loss(lp2, ha, &hm, TokenReduction::TokenMean), 1.0}, {ent2, beta}});
    auto both = [](std::vector<double> v) {
        for (double& e : v) e *= 2.0;
        return v;
    };
    held(twice.grad(hx)->to_vec(), both(t.dx), both(t.ex), "d hidden, twice");
    held(twice.grad(hw)->to_vec(), both(t.dw), both(t.ew), "d weight, twice");
}

// a mask whose last axis is not the vocabulary is refused, not regrouped into rows of V
static void test_mask_shapes() {
    const Tensor hx = Tensor::from_f32(x, {S, B, T, d}, dev, DType::BF16), hw = Tensor::from_f32(w, {d, V}, dev, DType::BF16);
    for (const Shape& shape : {Shape{2, V / 2}, Shape{V, 1}, Shape{2 * N, V / 2}, Shape{V, N}}) {
        const Tensor vm = Tensor::from_u8(std::vector<uint8_t>(numel(shape), 1), shape, dev);
        bool refused = false;
        try {
            rl::head_token_log_probs(hx, hw, IntTensor::from_data(tok, {S, B, T}), nullptr, false, &vm);
        } catch (const std::exception& e) {
            refused = std::string(e.what()).find("mask shape") != std::string::npos;
        }
        CHECK(refused, "mask of %zu rows of %zu", shape[0], shape[1]);
    }
}

// a temperature that is 0 in 32 bits: no temperature to score with, and the first maximum when drawing
static void test_temperatures() {
    const Tensor hx = Tensor::from_f32(x, {S, B, T, d}, dev, DType::BF16), hw = Tensor::from_f32(w, {d, V}, dev, DType::BF16), u = Tensor::from_f32(std::vector<float>(N, 0.5f), {S, B, T}, dev);
    for (double tau : {0.0, 1e-50}) {
        bool refused = false;
        try {
            rl::head_token_log_probs(hx, hw, IntTensor::from_data(tok, {S, B, T}), nullptr, false, nullptr, tau);
        } catch (const std::exception& e) {
            refused = std::string(e.what()).find("temperature") != std::string::npos;
        }
        CHECK(refused, "temperature %g", tau);
        CHECK(rl::head_sample_categorical(hx, hw, u, nullptr, nullptr, nullptr, tau).data == rl::head_sample_categorical(hx, hw, u, nullptr, nullptr, nullptr, 1e-3).data, "temperature %g", tau);
    }
}

int main() {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        std::printf("no CUDA device: this program tests the GPU path and has nothing to fall back to\n");
        return 2;
    }
    make();
    try {
        test_mask_shapes();
        test_temperatures();
        for (Form f : {kNone, kBytes, kByteRow, kBits, kBitRow})
            for (double tau : {1.0, 0.7, 1.5})
                for (bool checkpoint : {false, true}) test(f, tau, checkpoint);
    } catch (const std::exception& e) {
        std::printf("FAILED: exception: %s\n", e.what());
        return 1;
    }
    std::printf("all passed: %d checks\n", g_checks);
    return 0;
}
