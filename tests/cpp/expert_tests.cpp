// Tests of ops/experts.h through Tensor and the dispatcher:
//   expert_tests cpu   the MXFP4 dtype, a GGUF file with an MXFP4 tensor, ops on host tensors refused
//   expert_tests gpu   an expert layer from the file's blocks to the sum, against plain loops in double
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <fstream>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

#include "b200q.h"
#include "brotensor_b200/gguf.h"
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

static uint32_t g_lcg = 0x51ED27u;
static uint32_t lcg() { g_lcg = g_lcg * 1664525u + 1013904223u; return g_lcg >> 8; }
static float frand() { return float(lcg()) / float(1u << 23) - 1.f; }
static std::vector<uint8_t> make_blocks(size_t n) {
    std::vector<uint8_t> b(n * 17);
    for (size_t i = 0; i < n; ++i) {
        b[17 * i] = (uint8_t)(118 + lcg() % 4);
        for (int j = 1; j < 17; ++j) b[17 * i + j] = (uint8_t)lcg();
    }
    return b;
}
static const double kValues[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};
static double element(const std::vector<uint8_t>& b, size_t i) {  // element i of a row-major matrix of blocks
    const uint8_t* blk = &b[i / 32 * 17];
    const int j = (int)(i % 32), q = j < 16 ? blk[1 + j] & 15 : blk[1 + j - 16] >> 4;
    return std::ldexp(q & 8 ? -kValues[q & 7] : kValues[q & 7], blk[0] - 127);
}
static std::vector<double> quantised(const std::vector<float>& x) {
    std::vector<double> out(x.size());
    for (size_t b = 0; b < x.size(); b += 32) {
        float top = 0.f;
        for (int i = 0; i < 32; ++i) top = std::max(top, std::fabs(x[b + i]));
        const int e = top > 0 ? std::max(std::ilogb(top) - 2, -127) : -127;
        for (int i = 0; i < 32; ++i) {
            const double a = std::fabs(std::ldexp((double)x[b + i], -e));
            int best = 0;
            for (int c = 1; c < 8; ++c) {
                const double d = std::fabs(a - kValues[c]), o = std::fabs(a - kValues[best]);
                if (d < o || (d == o && !(c & 1))) best = c;  // the even code of two that are as near
            }
            out[b + i] = std::ldexp(x[b + i] < 0 ? -kValues[best] : kValues[best], e);
        }
    }
    return out;
}
static std::vector<float> random_rows(size_t n) {
    std::vector<float> v(n);
    for (auto& x : v) x = 2.f * frand();
    return v;
}
static double worst(const std::vector<float>& got, const std::vector<double>& want) {
    double top = 0, off = 0;
    for (size_t i = 0; i < want.size(); ++i) {
        top = std::max(top, std::fabs(want[i]));
        off = std::max(off, std::fabs(want[i] - got[i]));
    }
    return off / top;
}

static std::string write_gguf(const std::vector<uint8_t>& blocks, uint64_t K, uint64_t N, uint64_t E) {
    std::vector<uint8_t> f;
    const auto put = [&](auto v) { const auto* p = reinterpret_cast<const uint8_t*>(&v); f.insert(f.end(), p, p + sizeof v); };
    put(uint32_t(0x46554747u)); put(uint32_t(3)); put(uint64_t(1)); put(uint64_t(0));
    const std::string name = "blk.0.ffn_up_exps.weight";
    put(uint64_t(name.size())); f.insert(f.end(), name.begin(), name.end());
    put(uint32_t(3)); put(K); put(N); put(E); put(uint32_t(39)); put(uint64_t(0));
    while (f.size() % 32) f.push_back(0);
    f.insert(f.end(), blocks.begin(), blocks.end());
    const std::string path = "/tmp/b200_mxfp4.gguf";
    std::ofstream(path, std::ios::binary).write(reinterpret_cast<const char*>(f.data()), (std::streamsize)f.size());
    return path;
}

static void test_cpu() {
    std::printf("test_cpu\n");
    CHECK(bt::dtype_block_size(Dtype::MXFP4) == 32 && bt::dtype_block_bytes(Dtype::MXFP4) == 17 && bt::dtype_is_quant(Dtype::MXFP4));
    CHECK(bt::dtype_storage_bytes(Dtype::MXFP4, 64 * 96) == 64 * 3 * 17u);
    const std::vector<uint8_t> b = make_blocks(3 * 8 * 2);
    const auto file = bt::gguf::File::open(write_gguf(b, 64, 8, 3));
    const auto& t = file.get_tensor("blk.0.ffn_up_exps.weight");
    CHECK(t.dtype == Dtype::MXFP4 && t.dtype_supported && t.nbytes == b.size());
    const auto [rows, cols] = bt::gguf::shape_to_2d(t.shape);
    CHECK(rows == 24 && cols == 64);
    Tensor W;
    bt::gguf::upload_rows(t, rows, cols, 0, rows, Device::CPU, W);
    CHECK(W.bytes() == b.size() && !std::memcmp(W.data, b.data(), b.size()));
    Tensor image, ids, w, plan;
    CHECK(throws_with([&] { bt::mxfp4_pack(W, 3, image); }, "mxfp4_pack"));  // no CPU backend for any op
    CHECK(throws_with([&] { bt::moe_route_forward(Tensor::zeros_on(Device::CPU, 2, 4), 2, true, 1.f, ids, w, plan); }, "moe_route_forward"));
}

static Tensor on_gpu(const std::vector<float>& v, int r, int c) { return Tensor::from_host_on(Device::cuda(0), v.data(), r, c); }
static std::vector<int32_t> ints(const Tensor& t) {
    std::vector<int32_t> v((size_t)t.size());
    bt::sync(t.device);
    t.copy_raw_to_host(v.data());
    return v;
}
static std::vector<float> floats(const Tensor& t) {
    bt::sync(t.device);
    return t.to_host_vector();
}

static void test_gpu_linear() {
    std::printf("test_gpu_linear\n");
    const int N = 70, K = 160;
    const std::vector<uint8_t> b = make_blocks((size_t)N * K / 32);
    const Tensor W = Tensor::from_raw_bytes_on(Device::cuda(0), b.data(), N, K, Dtype::MXFP4, b.size());
    Tensor image;
    bt::mxfp4_pack(W, 1, image);
    CHECK(image.dtype == Dtype::INT8 && image.cols == 17408 && image.rows == 1);
    for (int M : {1, 9, 40, 200}) {
        const std::vector<float> x = random_rows((size_t)M * K), bias = random_rows(N);
        const std::vector<double> q = quantised(x);
        std::vector<double> want((size_t)M * N);
        for (int m = 0; m < M; ++m)
            for (int n = 0; n < N; ++n) {
                double s = bias[n];
                for (int k = 0; k < K; ++k) s += q[(size_t)m * K + k] * element(b, (size_t)n * K + k);
                want[(size_t)m * N + n] = s;
            }
        const Tensor X = on_gpu(x, M, K), B = on_gpu(bias, 1, N);
        Tensor Y;
        bt::mxfp4_linear_forward(image, N, &B, X, Y);
        CHECK(Y.rows == M && Y.cols == N && Y.dtype == Dtype::FP32 && worst(floats(Y), want) < 1e-6);
    }
    Tensor X = Tensor::zeros_on(Device::cuda(0), 2, K + 32), Y, bad = Tensor::zeros_on(Device::cuda(0), 2, K, Dtype::INT32);
    CHECK(throws_with([&] { bt::mxfp4_linear_forward(image, N + 128, nullptr, X, Y); }, "image"));
    CHECK(throws_with([&] { bt::mxfp4_linear_forward(image, N, nullptr, bad, Y); }, "X must be"));
    CHECK(throws_with([&] { bt::mxfp4_linear_forward(W, N, nullptr, X, Y); }, "image"));
    CHECK(throws_with([&] { bt::mxfp4_pack(W, 3, image); }, "multiple of the number of experts"));
    CHECK(throws_with([&] { bt::mxfp4_pack(X, 1, image); }, "Dtype::MXFP4"));
}

static void test_gpu_layer(int T) {
    std::printf("test_gpu_layer %d\n", T);
    const int E = 6, k = 2, N = 96, K = 64;
    const std::vector<uint8_t> g = make_blocks((size_t)E * N * K / 32), u = make_blocks((size_t)E * N * K / 32), d = make_blocks((size_t)E * K * N / 32);
    const auto up = [&](const std::vector<uint8_t>& b, int r, int c, Tensor& image) {
        bt::mxfp4_pack(Tensor::from_raw_bytes_on(Device::cuda(0), b.data(), r, c, Dtype::MXFP4, b.size()), E, image);
    };
    Tensor G, U, D;
    up(g, E * N, K, G);
    up(u, E * N, K, U);
    up(d, E * K, N, D);
    const std::vector<float> lg = random_rows((size_t)T * E), x = random_rows((size_t)T * K);
    const Tensor L = on_gpu(lg, T, E), X = on_gpu(x, T, K);
    Tensor ids, weights, plan, H, Y, out;
    bt::moe_route_forward(L, k, true, 1.f, ids, weights, plan);
    bt::moe_swiglu_forward(G, U, E, N, X, plan, T, k, H);
    bt::moe_linear_forward(D, E, K, nullptr, H, plan, T, k, Y);
    bt::moe_combine_forward(Y, ids, weights, E, out);
    const std::vector<int32_t> id = ints(ids);
    const std::vector<float> w = floats(weights), h = floats(H);
    const std::vector<double> xq = quantised(x), hq = quantised(h);  // (the second product is checked on the first one's results)
    std::vector<double> want_h, want(size_t(T) * K, 0.0);
    for (int t = 0; t < T; ++t) {
        std::vector<int> order(E);
        for (int e = 0; e < E; ++e) order[e] = e;
        std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return lg[(size_t)t * E + a] > lg[(size_t)t * E + b]; });
        double sum = 0;
        for (int j = 0; j < k; ++j) sum += std::exp((double)lg[(size_t)t * E + order[j]] - lg[(size_t)t * E + order[0]]);
        for (int j = 0; j < k; ++j) {
            const int e = order[j];
            const double p = std::exp((double)lg[(size_t)t * E + e] - lg[(size_t)t * E + order[0]]) / sum;
            CHECK(id[(size_t)t * k + j] == e && std::fabs(w[(size_t)t * k + j] - p) < 1e-6);
            for (int n = 0; n < N; ++n) {
                double a = 0, b = 0;
                for (int i = 0; i < K; ++i) {
                    a += xq[(size_t)t * K + i] * element(g, ((size_t)e * N + n) * K + i);
                    b += xq[(size_t)t * K + i] * element(u, ((size_t)e * N + n) * K + i);
                }
                want_h.push_back(a / (1 + std::exp(-a)) * b);
            }
            for (int i = 0; i < K; ++i) {
                double s = 0;
                for (int n = 0; n < N; ++n) s += hq[((size_t)t * k + j) * N + n] * element(d, ((size_t)e * K + i) * N + n);
                want[(size_t)t * K + i] += p * s;
            }
        }
    }
    CHECK(H.rows == T * k && H.cols == N && worst(h, want_h) < 4e-6);
    CHECK(out.rows == T && out.cols == K && worst(floats(out), want) < 4e-6);
    Tensor other = Tensor::zeros_on(Device::cuda(0), 8, 1, Dtype::INT32);
    CHECK(throws_with([&] { bt::moe_linear_forward(D, E, K, nullptr, H, other, T, k, Y); }, "plan"));
    CHECK(throws_with([&] { bt::moe_linear_forward(D, E, K, nullptr, Tensor::zeros_on(Device::cuda(0), T * k + 1, N), plan, T, k, Y); }, "a row for each token"));
    CHECK(throws_with([&] { bt::moe_combine_forward(X, ids, weights, E, out); }, "Y must have a row"));
    CHECK(throws_with([&] { bt::moe_route_forward(L, E + 1, true, 1.f, ids, weights, plan); }, "more than E"));
}

// Sizes whose products leave an int: refused by their numbers alone (views that claim more rows than there is memory behind them).
static void test_gpu_sizes() {
    std::printf("test_gpu_sizes\n");
    const Tensor some = Tensor::zeros_on(Device::cuda(0), 256, 1);
    const auto claim = [&](int rows, int cols, Dtype dt) { return Tensor::view(Device::cuda(0), some.data, rows, cols, dt); };
    Tensor ids, weights, plan, out;
    for (int T : {40000000, 67000000})  // the plan's size in 32-bit words is beyond 2^31 and beyond 2^32
        CHECK(throws_with([&] { bt::moe_route_forward(claim(T, 32, Dtype::FP16), 32, true, 1.f, ids, weights, plan); }, "larger than a Tensor holds"));
    CHECK(!ids.data && !plan.data);
    // 65536 x 65537 pairs are 2^32 + 65536
    CHECK(throws_with([&] { bt::moe_combine_forward(claim(65536, 1, Dtype::FP32), claim(65536, 65537, Dtype::INT32), claim(65536, 65537, Dtype::FP32), 4, out); },
                      "a row for each token"));
}

int main(int argc, char** argv) {
    const std::string mode = argc > 1 ? argv[1] : "cpu";
    bt::init();
    if (mode == "cpu") {
        test_cpu();
    } else if (!bt::is_available(Device::CUDA)) {
        std::printf("no CUDA device available - skipping\n");
        return 0;
    } else {
        test_gpu_linear();
        for (int T : {1, 7, 150}) test_gpu_layer(T);
        test_gpu_sizes();
        int st = 0;
        CHECK(b200q_device_status(&st) == B200Q_OK && st == 0);
    }
    std::printf("%s (%d failures)\n", g_failures ? "FAILED" : "OK", g_failures);
    return g_failures ? 1 : 0;
}
