// C++ test of the residual feed-forward operators' edges: refusals (argument "refusals", no GPU needed), and the block in 16 bits
// ("block16").
#include <nt/nt.h>

#include <cstdio>
#include <cstring>

#define REQUIRE(cond) nt::utils::throw_exception((cond), "requirement failed: " #cond " (line ", __LINE__, ")")

using nt::DType;
using nt::Tensor;
namespace fn = nt::functional;

// Tensors over memory that nothing reads: a refused call must not get as far as a launch.
static Tensor device_tensor(nt::SizeRef shape, DType dt = DType::Float32) {
    return Tensor::adopt(reinterpret_cast<void*>(uintptr_t(1) << 20), std::move(shape), dt, nt::DeviceType::CUDA);
}
static float g_host[4096];
static Tensor host_tensor(nt::SizeRef shape, DType dt = DType::Float32) { return Tensor::adopt(g_host, std::move(shape), dt, nt::DeviceType::CPU); }
template <class F>
bool refuses_host(F&& f) {
    try { f(); } catch (const std::invalid_argument& e) { return std::strstr(e.what(), "DeviceType::CUDA") != nullptr; }
    return false;
}

static void host_operands_are_refused() {
    Tensor x = device_tensor({4, 8}), w = device_tensor({8}), W = device_tensor({8, 16}), b = device_tensor({16}), r = device_tensor({4, 16});
    REQUIRE(refuses_host([&] { fn::rms_norm(host_tensor({4, 8}), w); }));
    REQUIRE(refuses_host([&] { fn::rms_norm(x, host_tensor({8})); }));
    REQUIRE(refuses_host([&] { fn::rms_norm(x, w, 1e-6, host_tensor({4, 8})); }));
    REQUIRE(refuses_host([&] { fn::rms_norm_int8(x, host_tensor({8})); }));
    REQUIRE(refuses_host([&] { fn::rms_norm_int8(x, w, 1e-6, host_tensor({4, 8})); }));
    REQUIRE(refuses_host([&] { fn::quantize_rows(host_tensor({4, 8})); }));
    REQUIRE(refuses_host([&] { fn::linear_act(host_tensor({4, 8}), W); }));
    REQUIRE(refuses_host([&] { fn::linear_act(x, W, host_tensor({16})); }));
    REQUIRE(refuses_host([&] { fn::linear_act(x, W, b, fn::Activation::GELU, host_tensor({4, 16})); }));
    Tensor q = device_tensor({4, 8}, DType::int8), Q = device_tensor({8, 16}, DType::int8), s = device_tensor({4}), S = device_tensor({16});
    REQUIRE(refuses_host([&] { fn::linear_int8(q, host_tensor({4}), Q, S); }));
    REQUIRE(refuses_host([&] { fn::linear_int8(q, s, Q, host_tensor({16})); }));
    nt::TensorGrad logits(device_tensor({4, 16}));
    Tensor t = device_tensor({4, 2}), i = device_tensor({4, 2}, DType::int32);
    REQUIRE(refuses_host([&] { nt::loss::DistillTopK(logits, host_tensor({4, 2}), i); }));
    REQUIRE(refuses_host([&] { nt::loss::DistillTopK(logits, t, host_tensor({4, 2}, DType::int32)); }));
    REQUIRE(refuses_host([&] { nt::loss::DistillTopK(logits, t, i, 1.0, host_tensor({4})); }));
}

// The block's loss and gradients on Float32 parameters, or on the same values in 16 bits.
struct Block {
    nt::TensorGrad norm, up, up_bias, down, down_bias, head, x, stream;
    double loss;
};
static Block run_block(DType dt, DType values) {
    auto param = [&](nt::SizeRef shape, unsigned seed, double stddev) {
        Tensor t = nt::randn_seeded(std::move(shape), DType::Float32, seed, stddev).to(values);
        return nt::TensorGrad(values == dt ? t : t.to(dt));
    };
    Block b{param({64}, 1, 1.0), param({64, 136}, 2, 0.125), param({136}, 3, 0.2), param({136, 64}, 4, 0.086), param({64}, 5, 0.2),
            param({64, 200}, 6, 0.25), param({40, 64}, 7, 1.0), param({40, 64}, 8, 2.0), 0};
    Tensor teacher = nt::randn_seeded({40, 5}, DType::Float32, 9);
    std::vector<int64_t> columns;
    for (int i = 0; i < 200; ++i) columns.push_back((37 * i) % 200);
    auto [y, h] = fn::rms_norm(b.x, b.norm, 1e-6, b.stream);
    nt::TensorGrad a = fn::linear_act(y, b.up, b.up_bias, fn::Activation::SiLU);
    nt::TensorGrad out = fn::linear_act(a, b.down, b.down_bias, fn::Activation::None, h);
    nt::TensorGrad logits = fn::linear_act(fn::rms_norm(out, b.norm).y, b.head, nt::TensorGrad(), fn::Activation::None);
    Tensor weight = Tensor::from_host(std::vector<float>(40, 16.f).data(), {40}, DType::Float32);   // Float16's smallest gradients stay normal
    nt::ScalarGrad loss = nt::loss::DistillTopK(logits, teacher, Tensor::from_host(columns.data(), {40, 5}, DType::int64), 2.0, weight);
    loss.backward();
    b.loss = loss.item();
    return b;
}
// At most 10 roundings to the type on the way, each half a step at worst; twice that through norms and activations of slope near 1.
static void block_in_16_bits() {
    for (DType dt : {DType::Float16, DType::BFloat16}) {
        const double bound = 20 * (dt == DType::Float16 ? 1.0 / 2048 : 1.0 / 256);
        Block got = run_block(dt, dt), want = run_block(DType::Float32, dt);
        REQUIRE(std::fabs(got.loss - want.loss) <= bound * want.loss);
        using Pair = std::pair<const nt::TensorGrad*, const nt::TensorGrad*>;
        for (auto [g, w] : {Pair{&got.norm, &want.norm}, {&got.up, &want.up}, {&got.up_bias, &want.up_bias}, {&got.down, &want.down},
                            {&got.down_bias, &want.down_bias}, {&got.head, &want.head}, {&got.x, &want.x}, {&got.stream, &want.stream}}) {
            REQUIRE(g->grad().dtype() == dt && g->grad().shape() == w->grad().shape());
            const std::vector<float> u = g->grad().to(DType::Float32).to_vector<float>(), v = w->grad().to_vector<float>();
            double off = 0, size = 0;
            for (size_t i = 0; i < v.size(); ++i) { off += (u[i] - v[i]) * (u[i] - v[i]); size += v[i] * v[i]; }
            REQUIRE(size > 0 && std::sqrt(off / size) <= bound);
        }
    }
    nt::utils::check(ntb200_check_device_status(nullptr));
}

int main(int argc, char** argv) {
    const char* which = argc > 1 ? argv[1] : "";
    try {
        if (!std::strcmp(which, "refusals")) host_operands_are_refused();
        else if (!std::strcmp(which, "block16")) block_in_16_bits();
        else throw std::invalid_argument("no such case");
    } catch (const std::exception& e) {
        std::printf("FAIL %s: %s\n", which, e.what());
        return 1;
    }
    std::printf("PASS %s\n", which);
    return 0;
}
