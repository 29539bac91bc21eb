// ops/experts.h through Tensor and the dispatcher: arguments that do not belong together, by the name of the test on the command line. Needs a CUDA device.
#include <cstdio>
#include <cstring>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

#include "b200q.h"
#include "brotensor_b200/ops/experts.h"
#include "brotensor_b200/runtime.h"

namespace bt = brotensor_b200;
using bt::Device;
using bt::Dtype;
using bt::Tensor;

static int g_failures = 0;
#define CHECK(c) do { if (!(c)) { std::printf("  FAIL %s:%d %s\n", __FILE__, __LINE__, #c); ++g_failures; } } while (0)
static bool throws_with(const std::function<void()>& f, const char* needle) {
    try {
        f();
    } catch (const std::runtime_error& e) {
        if (std::strstr(e.what(), needle)) return true;
        std::printf("  message was: %s\n", e.what());
    }
    return false;
}
static const Device kGpu = Device::cuda(0);
static std::vector<uint8_t> make_blocks(size_t n, uint32_t seed) {
    std::vector<uint8_t> b(n * 17);
    for (size_t i = 0; i < b.size(); ++i) {
        seed = seed * 1664525u + 1013904223u;
        b[i] = i % 17 ? (uint8_t)(seed >> 24) : (uint8_t)(118 + (seed >> 30));
    }
    return b;
}

// A plan that was made for other tokens or experts is laid out otherwise: read as one of these, it would name experts and places that do not exist.
static void test_plan_of_other_sizes() {
    const int E = 6, k = 2, N = 96, K = 64;
    const std::vector<uint8_t> b = make_blocks((size_t)E * N * K / 32, 1);
    Tensor image, ids, weights, plan, Y;
    bt::mxfp4_pack(Tensor::from_raw_bytes_on(kGpu, b.data(), E * N, K, Dtype::MXFP4, b.size()), E, image);
    for (int T : {9, 40, 300}) {
        bt::moe_route_forward(Tensor::zeros_on(kGpu, T, E), k, true, 1.f, ids, weights, plan);
        const Tensor X = Tensor::zeros_on(kGpu, T, K), fewer = Tensor::zeros_on(kGpu, T - 1, K);
        CHECK(throws_with([&] { bt::moe_linear_forward(image, E, N, nullptr, fewer, plan, T - 1, k, Y); }, "plan must be of these"));
        CHECK(throws_with([&] { bt::moe_linear_forward(image, E - 1, N, nullptr, X, plan, T, k, Y); }, "plan must be of these"));
        CHECK(throws_with([&] { bt::moe_swiglu_forward(image, image, E, N, X, plan, T, k - 1, Y); }, "plan must be of these"));
        bt::moe_linear_forward(image, E, N, nullptr, X, plan, T, k, Y);
        CHECK(Y.rows == T * k && Y.cols == N);
    }
    bt::sync(kGpu);
}

// 31 experts of 16128 x 8192 are an image of 2.18 GB. The first and the last are filled; what they give is what they give on their own.
static void test_image_beyond_two_gigabytes() {
    const int E = 31, N = 16128, K = 8192, T = 6;
    const size_t each = (size_t)N * K / 32 * 17;
    Tensor W = Tensor::empty_on(kGpu, E * N, K, Dtype::MXFP4), image;
    CHECK(W.bytes() == E * each);
    W.zero();
    Tensor alone[2];
    for (int i = 0; i < 2; ++i) {
        const std::vector<uint8_t> b = make_blocks((size_t)N * K / 32, 7 + i);
        const Tensor part = Tensor::from_raw_bytes_on(kGpu, b.data(), N, K, Dtype::MXFP4, b.size());
        Tensor here = Tensor::view(kGpu, static_cast<uint8_t*>(W.data) + (i ? (E - 1) * each : 0), N, K, Dtype::MXFP4);
        here.copy_raw_from_host_async(b.data());
        bt::sync(kGpu);
        bt::mxfp4_pack(part, 1, alone[i]);
        CHECK(alone[i].dtype == Dtype::INT8);
    }
    bt::mxfp4_pack(W, E, image);
    CHECK(image.dtype == Dtype::INT32 && image.cols == 4352 && image.rows == E * 126 * 32 && image.bytes() == E * alone[0].bytes());
    std::vector<float> x((size_t)T * K), logits((size_t)T * E, 0.f);
    for (size_t i = 0; i < x.size(); ++i) x[i] = (float)((int)(i * 2654435761u >> 20) - 2048) / 700.f;
    for (int t = 0; t < T; ++t) logits[(size_t)t * E + (t % 2 ? E - 1 : 0)] = 1.f;
    const Tensor X = Tensor::from_host_on(kGpu, x.data(), T, K);
    Tensor ids, weights, plan, Y, A[2];
    bt::moe_route_forward(Tensor::from_host_on(kGpu, logits.data(), T, E), 1, true, 1.f, ids, weights, plan);
    bt::moe_linear_forward(image, E, N, nullptr, X, plan, T, 1, Y);
    for (int i = 0; i < 2; ++i) bt::mxfp4_linear_forward(alone[i], N, nullptr, X, A[i]);
    bt::sync(kGpu);
    const std::vector<float> y = Y.to_host_vector(), a[2] = {A[0].to_host_vector(), A[1].to_host_vector()};
    double off = 0, top = 0;
    for (int t = 0; t < T; ++t)
        for (int n = 0; n < N; ++n) {
            const double want = a[t % 2][(size_t)t * N + n], d = y[(size_t)t * N + n] - want;
            off += d * d;
            top += want * want;
        }
    CHECK(top > 0 && off < top * 1e-12);  // (sums of another order)
    // by its numbers alone: a view that claims more than there is
    const Tensor more = Tensor::view(kGpu, W.data, 1 << 20, 16384, Dtype::MXFP4);
    Tensor none;
    CHECK(throws_with([&] { bt::mxfp4_pack(more, 1, none); }, "larger than a Tensor holds"));
    CHECK(!none.data);
}

int main(int argc, char** argv) {
    const std::string which = argc > 1 ? argv[1] : "";
    bt::init();
    if (!bt::is_available(Device::CUDA)) {
        std::printf("no CUDA device available - skipping\n");
        return 0;
    }
    if (which == "plan") test_plan_of_other_sizes();
    else if (which == "image") test_image_beyond_two_gigabytes();
    else CHECK(!"the name of a test");
    int st = 0;
    CHECK(b200q_device_status(&st) == B200Q_OK && st == 0);
    std::printf("%s (%d failures)\n", g_failures ? "FAILED" : "OK", g_failures);
    return g_failures ? 1 : 0;
}
