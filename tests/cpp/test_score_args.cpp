// test_score_args.cpp -- what lm_head_argmax_i8 of include/loom_select.hpp refuses, and that it then leaves the residual alone.
//
// `test_score_args cpu` passes pointers that are never read: the arguments are refused before anything is allocated or
// enqueued. `test_score_args gpu` does the same with device memory and looks at the residual afterwards. Exit 0 = pass.
#include "loom_select.hpp"

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

static int g_failures = 0;

#define CHECK(cond)                                                                         \
    do {                                                                                    \
        if (!(cond)) {                                                                      \
            ++g_failures;                                                                   \
            std::fprintf(stderr, "CHECK FAILED at %s:%d: %s\n", __FILE__, __LINE__, #cond); \
        }                                                                                   \
    } while (0)

template <class F>
static bool throws(F&& f, const char* text) {
    try {
        f();
    } catch (const loom::Error& e) {
        return std::string(e.what()).find(text) != std::string::npos;
    }
    return false;
}

// x, residual: rows of 64 bf16; norm: 64 f32; w: 300 x 64 int8; scale: 300 f32.
static void refusals(const void* x, void* residual, const float* norm, const int8_t* w, const float* scale) {
    using loom::select::lm_head_argmax_i8;
    const float* odd = reinterpret_cast<const float*>(reinterpret_cast<uintptr_t>(scale) + 1);
    CHECK(throws([&] { lm_head_argmax_i8(x, residual, norm, 1e-6, nullptr, scale, 2, 64, 300); }, "invalid argument"));
    CHECK(throws([&] { lm_head_argmax_i8(x, residual, norm, 1e-6, w + 4, scale, 2, 64, 300); }, "invalid argument"));
    CHECK(throws([&] { lm_head_argmax_i8(x, residual, norm, 1e-6, w, nullptr, 2, 64, 300); }, "invalid argument"));
    CHECK(throws([&] { lm_head_argmax_i8(x, residual, norm, 1e-6, w, odd, 2, 64, 300); }, "invalid argument"));
    CHECK(throws([&] { lm_head_argmax_i8(x, residual, norm, 1e-6, w, scale, 2, 24, 300); }, "beyond what the kernels support"));
    CHECK(throws([&] { lm_head_argmax_i8(x, residual, norm, 1e-6, w, scale, 2, 64, int64_t(1) << 31); },
                 "beyond what the kernels support"));
    CHECK(throws([&] { lm_head_argmax_i8(x, residual, norm, 1e-6, w, scale, int64_t(1) << 28, 64, 300); },
                 "beyond what the kernels support"));
}

template <class T>
static T* upload(const std::vector<T>& h) {
    T* d = nullptr;
    if (cudaMalloc(&d, h.size() * sizeof(T)) != cudaSuccess) return nullptr;
    cudaMemcpy(d, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice);
    return d;
}

static void gpu_checks() {
    std::vector<uint16_t> x(2 * 64, 0x3F80), r(2 * 64, 0x4000);  // 1.0 and 2.0
    uint16_t* dx = upload(x);
    uint16_t* dr = upload(r);
    float* norm = upload(std::vector<float>(64, 1.0f));
    std::vector<int8_t> w(300 * 64, 1);
    for (int i = 0; i < 300; ++i) w[i * 64] = int8_t(i % 100);
    int8_t* dw = upload(w);
    float* scale = upload(std::vector<float>(300, 0.001f));
    refusals(dx, dr, norm, dw, scale);
    std::vector<uint16_t> after(r.size());
    cudaDeviceSynchronize();
    cudaMemcpy(after.data(), dr, after.size() * 2, cudaMemcpyDeviceToHost);
    CHECK(after == r);
    const loom::select::GreedyResult g = loom::select::lm_head_argmax_i8(dx, dr, norm, 1e-6, dw, scale, 2, 64, 300);
    cudaMemcpy(after.data(), dr, after.size() * 2, cudaMemcpyDeviceToHost);
    CHECK(after == std::vector<uint16_t>(r.size(), 0x4040));  // 3.0
    // rows of 127 with the scale 1 / 127 (of y = 1, off by the norm's 1e-6 / 9): id 99 has 127 (99 + 63) 0.001 / 127
    CHECK(g.ids == std::vector<int32_t>(2, 99));
    for (int i = 0; i < 2; ++i) CHECK(std::fabs(g.logit[i] - 0.162) < 1e-6);
    for (void* p : {static_cast<void*>(dx), static_cast<void*>(dr), static_cast<void*>(norm), static_cast<void*>(dw),
                    static_cast<void*>(scale)})
        cudaFree(p);
}

int main(int argc, char** argv) {
    void* never = reinterpret_cast<void*>(uintptr_t(1) << 20);
    refusals(never, never, static_cast<const float*>(never), static_cast<const int8_t*>(never), static_cast<const float*>(never));
    if (argc > 1 && std::strcmp(argv[1], "gpu") == 0) gpu_checks();
    std::fprintf(stderr, "%d failures\n", g_failures);
    return g_failures == 0 ? 0 : 1;
}
