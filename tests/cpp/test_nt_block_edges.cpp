// C++ test of the residual feed-forward operators' refusals (argument "refusals", no GPU needed).
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

int main(int argc, char** argv) {
    const char* which = argc > 1 ? argv[1] : "";
    try {
        if (!std::strcmp(which, "refusals")) host_operands_are_refused();
        else throw std::invalid_argument("no such case");
    } catch (const std::exception& e) {
        std::printf("FAIL %s: %s\n", which, e.what());
        return 1;
    }
    std::printf("PASS %s\n", which);
    return 0;
}
