// C++ test of the residual feed-forward operators on the nt:: surface: RMSNorm, Linear with activation and residual, Int8 rows,
// the distillation loss.
#include <nt/nt.h>

#include <cstdio>

static int g_failed = 0, g_run = 0;
template <class F>
void run_test(const char* name, F&& f) {
    ++g_run;
    try {
        f();
        std::printf("PASS %s\n", name);
    } catch (const std::exception& e) {
        ++g_failed;
        std::printf("FAIL %s: %s\n", name, e.what());
    }
    uint64_t in_use = 0;
    ntb200_pool_stats(&in_use, nullptr);
    if (in_use != 0) {
        ++g_failed;
        std::printf("FAIL %s: %llu bytes still allocated from the pool\n", name, (unsigned long long)in_use);
    }
}
#define REQUIRE(cond) nt::utils::throw_exception((cond), "requirement failed: " #cond " (line ", __LINE__, ")")
template <class F>
bool throws_invalid_argument(F&& f) {
    try { f(); } catch (const std::invalid_argument&) { return true; }
    return false;
}

using nt::DType;
using nt::Tensor;
namespace fn = nt::functional;

int main() {
    run_test("residual feed-forward block: norm, linear with activation and residual, distillation loss, gradients by differences", [&] {
        nt::layers::RMSNorm norm(24);
        nt::layers::Linear up(24, 40, true, DType::Float32, 61), down(40, 24, true, DType::Float32, 62), head(24, 50, false, DType::Float32, 63);
        Tensor x0 = nt::randn_seeded({6, 24}, DType::Float32, 64), stream = nt::randn_seeded({6, 24}, DType::Float32, 65);
        Tensor teacher = nt::randn_seeded({6, 3}, DType::Float32, 66);
        std::vector<int32_t> columns;
        for (int i = 0; i < 18; ++i) columns.push_back((7 * i) % 50);
        Tensor index = Tensor::from_host(columns.data(), {6, 3}, DType::int32);
        auto step = [&](const Tensor& x, nt::TensorGrad* leaf) {
            nt::TensorGrad in(x), s(stream);
            auto [y, h] = norm.forward(in, s);
            nt::TensorGrad out = down.forward(up.forward(y, fn::Activation::GELU), fn::Activation::None, h);
            nt::ScalarGrad loss = nt::loss::DistillTopK(fn::linear_act(out, head.Weight, head.Bias, fn::Activation::None), teacher, index, 1.5);
            if (leaf) {
                loss.backward();
                *leaf = in;
                REQUIRE(s.grad().to_vector<float>() == in.grad().to_vector<float>());   // x and the residual share one gradient
            }
            return loss.item();
        };
        nt::TensorGrad leaf;
        step(x0, &leaf);
        REQUIRE(norm.Weight.has_grad() && up.Weight.has_grad() && up.Bias.has_grad() && down.Weight.has_grad() && head.Weight.has_grad());
        std::vector<float> g = leaf.grad().to_vector<float>(), x = x0.to_vector<float>();
        const float e = 1.f / 64;
        for (int at : {0, 17, 60, 143}) {   // central differences: e^2 / 6 of a third derivative below 8, and Float32's rounding of the loss over e
            std::vector<float> a = x, b = x;
            a[size_t(at)] += e;
            b[size_t(at)] -= e;
            const double d = (step(Tensor::from_host(a.data(), {6, 24}, DType::Float32), nullptr) -
                              step(Tensor::from_host(b.data(), {6, 24}, DType::Float32), nullptr)) / (2.0 * e);
            REQUIRE(std::fabs(d - double(g[size_t(at)])) <= 8.0 * e * e / 6 + 64 * 1e-6);
        }
        // the same block on Int8 rows stays within a few steps of 1 / 127
        auto wq = fn::quantize_rows(up.Weight.detach().transpose(0, 1).contiguous());
        auto q = fn::rms_norm_int8(x0, norm.Weight.detach(), 1e-6, stream);
        Tensor full = fn::linear_act(fn::rms_norm(x0, norm.Weight.detach(), 1e-6, stream).y, up.Weight.detach(), up.Bias.detach(), fn::Activation::SiLU);
        Tensor small = fn::linear_int8(q.q, q.scale, wq.q, wq.scale, up.Bias.detach(), fn::Activation::SiLU, Tensor(), true, DType::Float32);
        std::vector<float> u = full.to_vector<float>(), v = small.to_vector<float>();
        double num = 0, den = 0;
        for (size_t i = 0; i < u.size(); ++i) { num += (u[i] - v[i]) * (u[i] - v[i]); den += u[i] * u[i]; }
        REQUIRE(std::sqrt(num / den) < 4.0 / 127);
        REQUIRE(throws_invalid_argument([&] { fn::rms_norm(x0, up.Bias.detach()); }));
        REQUIRE(throws_invalid_argument([&] { fn::linear_act(x0, down.Weight.detach()); }));
    });

    nt::utils::check(ntb200_check_device_status(nullptr));
    std::printf("%d of %d cases failed\n", g_failed, g_run);
    return g_failed ? 1 : 0;
}
