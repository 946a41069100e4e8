// GPU tests of the head in the C++ host mirror (noetic_tensor_b200/host/noetic_rl.hpp): the tracked
// head_token_log_probs (log-probs, entropies and the gradients of the hidden states and the weight, whole and from an
// 8-bit checkpoint) and the 8-bit head_logits, against f64 on the host. Run by tests/test_gpu_head_cpp.py.
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

template <class F>
static bool throws(F f, const char* needle) {
    try {
        f();
    } catch (const std::exception& e) {
        return std::string(e.what()).find(needle) != std::string::npos;
    }
    return false;
}
static float through_bf16(float x) {
    uint32_t b = (uint32_t)bf16_from_f32(x) << 16;
    float y;
    std::memcpy(&y, &b, 4);
    return y;
}

constexpr size_t S = 2, B = 3, T = 25, d = 72, V = 264, N = S * B * T;
static std::vector<float> x(N* d), w(d* V), adv(N), mask(N);
static std::vector<int64_t> tok(N);

static void make() {
    std::mt19937 gen(11);
    std::normal_distribution<float> nd(0.f, 1.f);
    for (auto& v : x) v = through_bf16(nd(gen));
    for (auto& v : w) v = through_bf16(nd(gen) * 0.35f);
    for (size_t i = 0; i < N; i++) {
        tok[i] = (int64_t)(gen() % V);
        adv[i] = nd(gen);
        mask[i] = gen() % 4 ? 1.f : 0.f;
    }
}

struct Truth {
    std::vector<double> lp, H, dx, dw, ex, ew;  // values; gradients and the majorants of their rounding
};
// loss = Σ_s Σ −lp·adv·mask / count_s + β Σ_s Σ H·mask / count_s, from hidden states xs normalised by the statistics of x
static Truth truth(const std::vector<double>& xs, double beta) {
    Truth t;
    t.lp.resize(N); t.H.resize(N); t.dx.assign(N * d, 0.0); t.dw.assign(d * V, 0.0); t.ex.assign(N * d, 0.0); t.ew.assign(d * V, 0.0);
    for (size_t r = 0; r < N; r++) {
        double count = 0.0;
        for (size_t i = 0; i < B * T; i++) count += mask[r / (B * T) * B * T + i];
        const double a = -(double)adv[r] * mask[r] / std::max(count, 1.0), b = beta * mask[r] / std::max(count, 1.0);
        std::vector<double> z(V, 0.0), zs(V, 0.0);
        for (size_t k = 0; k < d; k++)
            for (size_t v = 0; v < V; v++) {
                z[v] += (double)x[r * d + k] * w[k * V + v];
                zs[v] += xs[r * d + k] * w[k * V + v];
            }
        double m = z[0], Z = 0.0;
        for (double v : z) m = std::max(m, v);
        for (double v : z) Z += std::exp(v - m);
        const double lse = m + std::log(Z);
        double H = 0.0;
        for (double v : z) H -= std::exp(v - lse) * (v - lse);
        t.lp[r] = z[tok[r]] - lse;
        t.H[r] = H;
        for (size_t v = 0; v < V; v++) {
            const double l = zs[v] - lse, p = std::exp(l), hot = (int64_t)v == tok[r] ? 1.0 : 0.0;
            const double g = a * (hot - p) - b * p * (l + H), D = std::fabs(a) * (hot + p) + std::fabs(b) * p * (std::fabs(l) + H + 1.0);
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
// an entry of ∂/∂z is rounded to bf16 once (2^-8 of itself), sums and exponentials are f32
static void held(const std::vector<float>& got, const std::vector<double>& want, const std::vector<double>& major, const char* what) {
    for (size_t i = 0; i < got.size(); i++) {
        const double tol = (std::ldexp(1.0, -8) + 1e-4) * major[i] + 1e-6 * std::fabs(want[i]);
        CHECK(std::fabs(got[i] - want[i]) <= tol, "%s[%zu]: got %.9g, want %.9g, tolerance %.3e", what, i, (double)got[i], want[i], tol);
    }
}

static void test_gradients(bool checkpoint) {
    const Tensor hx = Tensor::from_f32(x, {S, B, T, d}, dev, DType::BF16).require_grad(), hw = Tensor::from_f32(w, {d, V}, dev, DType::BF16).require_grad();
    const Tensor hm = Tensor::from_f32(mask, {S, B, T}, dev), ha = Tensor::from_f32(adv, {S, B, T}, dev);
    Tensor ent;
    const Tensor lp = rl::head_token_log_probs(hx, hw, IntTensor::from_data(tok, {S, B, T}), &ent, false, nullptr, 1.0, checkpoint);
    std::vector<double> xs(x.begin(), x.end());
    if (checkpoint)
        for (size_t r = 0; r < N; r++) {
            float big = 0.f;
            for (size_t k = 0; k < d; k++) big = std::max(big, std::fabs(x[r * d + k]));
            for (size_t k = 0; k < d; k++) xs[r * d + k] = std::nearbyint(127.0 * x[r * d + k] / big) * (double)(float)((double)big / 127.0);
        }
    const Truth t = truth(xs, 0.1);
    const std::vector<float> glp = lp.to_vec(), gH = ent.to_vec();
    for (size_t r = 0; r < N; r++) {
        CHECK(std::fabs(glp[r] - t.lp[r]) <= 2e-5 * (1 + std::fabs(t.lp[r])), "log-prob %zu: %.9g, %.9g", r, (double)glp[r], t.lp[r]);
        CHECK(std::fabs(gH[r] - t.H[r]) <= 2e-5 * (1 + std::fabs(t.H[r])), "entropy %zu: %.9g, %.9g", r, (double)gH[r], t.H[r]);
    }
    // the log-probs and entropies feed a policy loss and an entropy term: the tape sums both nodes' gradients (per-token upstreams)
    std::vector<float> up(N), ue(N);
    for (size_t r = 0; r < N; r++) {
        double count = 0.0;
        for (size_t i = 0; i < B * T; i++) count += mask[r / (B * T) * B * T + i];
        ue[r] = (float)(0.1 * mask[r] / count);
    }
    const Tensor pg = rl::policy_gradient_loss(lp, ha, &hm, TokenReduction::TokenMean);
    const Gradients g = backward(pg);
    const Gradients ge = backward(ent, Tensor::from_f32(ue, {S, B, T}, dev));
    CHECK(g.grad(hx) && g.grad(hw) && ge.grad(hx) && ge.grad(hw), "gradients of both");
    auto sum = [](const std::vector<float>& p, const std::vector<float>& q) {
        std::vector<float> s(p.size());
        for (size_t i = 0; i < p.size(); i++) s[i] = p[i] + q[i];
        return s;
    };
    held(sum(g.grad(hx)->to_vec(), ge.grad(hx)->to_vec()), t.dx, t.ex, "d hidden");
    held(sum(g.grad(hw)->to_vec(), ge.grad(hw)->to_vec()), t.dw, t.ew, "d weight");
    // both terms in one backward: the second node adds to the first one's gradients
    const Tensor total = rl::policy_gradient_loss(lp, ha, &hm, TokenReduction::TokenMean);
    const Gradients both = backward({{total, 1.0}, {ent, 0.01}});
    CHECK(both.grad(hx) && both.grad(hw), "gradients of a sum of terms");
    for (float v : both.grad(hw)->to_vec()) CHECK(std::isfinite(v), "finite");
    // only the weight tracked
    const Tensor lw = rl::head_token_log_probs(hx.detach(), hw, IntTensor::from_data(tok, {S, B, T}));
    const Gradients gw = backward(rl::policy_gradient_loss(lw, ha, &hm, TokenReduction::TokenMean));
    CHECK(!gw.grad(hx) && gw.grad(hw), "the hidden states are not tracked");
    // tracking changes no value; of rounded logits the results are untracked
    CHECK(rl::head_token_log_probs(hx.detach(), hw.detach(), IntTensor::from_data(tok, {S, B, T})).to_vec() == glp, "the tracked values are the untracked ones");
    const Tensor lr = rl::head_token_log_probs(hx, hw, IntTensor::from_data(tok, {S, B, T}), nullptr, true);
    CHECK(!lr.tracked() && lr.to_vec() == rl::head_token_log_probs(hx.detach(), hw.detach(), IntTensor::from_data(tok, {S, B, T}), nullptr, true).to_vec(), "rounded logits are untracked");
}

static void test_int8() {
    const Tensor hx = Tensor::from_f32(x, {S, B, T, d}, dev), hw = Tensor::from_f32(w, {d, V}, dev, DType::BF16);
    const rl::Int8Weight w8 = rl::Int8Weight::of(hw);
    const std::vector<float> z = rl::head_logits(hx, w8).to_vec();
    std::vector<float> wbig(V, 0.f);
    for (size_t k = 0; k < d; k++)
        for (size_t v = 0; v < V; v++) wbig[v] = std::max(wbig[v], std::fabs(w[k * V + v]));
    for (size_t r = 0; r < N; r++) {
        float big = 0.f;
        for (size_t k = 0; k < d; k++) big = std::max(big, std::fabs(x[r * d + k]));
        for (size_t v = 0; v < V; v++) {
            double sum = 0.0;
            for (size_t k = 0; k < d; k++) sum += std::nearbyint(127.0 * x[r * d + k] / big) * std::nearbyint(127.0 * w[k * V + v] / wbig[v]);
            const double want = sum * (double)(float)((double)big / 127.0) * (double)(float)((double)wbig[v] / 127.0);
            CHECK(std::fabs(z[r * V + v] - want) <= 4 * std::ldexp(1.0, -24) * std::fabs(want), "logit %zu %zu: %.9g, %.9g", r, v, (double)z[r * V + v], want);
        }
    }
    CHECK(throws([&] { rl::head_logits(Tensor::from_f32(std::vector<float>(6), {2, 3}, dev), w8); }, "head_logits"), "another width");
    CHECK(throws([&] { rl::Int8Weight::of(hx); }, "Int8Weight"), "an F32 weight");
}

int main() {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        std::printf("no CUDA device: this program tests the GPU path and has nothing to fall back to\n");
        return 2;
    }
    make();
    try {
        test_gradients(false);
        test_gradients(true);
        test_int8();
    } catch (const std::exception& e) {
        std::printf("FAILED: exception: %s\n", e.what());
        return 1;
    }
    std::printf("all passed: %d checks\n", g_checks);
    return 0;
}
