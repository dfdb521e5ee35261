// test_score_api.cpp -- the scoring and 8-bit LM-head helpers of include/loom_select.hpp.
//
// `test_score_api cpu` checks the argument errors, which are raised before anything is enqueued; `test_score_api gpu`
// also known answers on device memory. A dependency-free harness; exit 0 = pass.
#include "loom_select.hpp"

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

static int g_checks = 0;
static int g_failures = 0;

#define CHECK(cond)                                                                         \
    do {                                                                                    \
        ++g_checks;                                                                         \
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

template <class T>
static T* upload(const std::vector<T>& h) {
    T* d = nullptr;
    if (cudaMalloc(&d, h.size() * sizeof(T)) != cudaSuccess) return nullptr;
    cudaMemcpy(d, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice);
    return d;
}

static void cpu_checks() {
    using namespace loom::select;
    CHECK(throws([] { lm_head_argmax_i8(nullptr, nullptr, nullptr, 1e-6, nullptr, nullptr, 0, 64, 10); }, "invalid argument"));
    CHECK(throws([] { lm_head_argmax_i8(nullptr, nullptr, nullptr, 1e-6, nullptr, nullptr, 1, 0, 10); }, "invalid argument"));
}

static void gpu_checks() {
    using namespace loom::select;
    // rows [0, ln 2, ln 4] and [3, 1, 3] with a padded third: probabilities 1/7, 2/7, 4/7
    const float l2 = std::log(2.0f), l4 = std::log(4.0f);
    float* dl = upload(std::vector<float>{0.0f, l2, l4, 3.0f, 1.0f, 3.0f, 5.0f, 5.0f, 5.0f});
    int32_t* di = upload(std::vector<int32_t>{1, 2, -1});
    const TokenScores s = token_logprobs(dl, 3, 3, 3, di, 1.0f, 2);
    CHECK(std::fabs(s.logprob[0] - std::log(2.0 / 7.0)) < 1e-5);
    const double z = 2.0 * std::exp(3.0) + std::exp(1.0);
    CHECK(std::fabs(s.logprob[1] - (3.0 - std::log(z))) < 1e-5);
    CHECK(s.logprob[2] == 0.0f);
    CHECK((s.rank == std::vector<int32_t>{1, 1, -1}));
    CHECK((s.top_ids == std::vector<int32_t>{2, 1, 0, 2, 0, 1}));
    CHECK(std::fabs(s.top_logprobs[0] - std::log(4.0 / 7.0)) < 1e-5);
    CHECK(std::fabs(s.entropy[2] - std::log(3.0)) < 1e-5);
    CHECK(throws([&] { token_logprobs(dl, 3, 3, 3, di, 0.0f); }, "parameter out of range"));
    CHECK(throws([&] { token_logprobs(dl, 3, 3, 2, di); }, "invalid argument"));

    // hidden rows e0 and e1 plus a residual of the same: the sum is 2 e, its norm sqrt(64) e, so 8 in one place and q = 127.
    // Weight rows: 100 at id 250 for e0, 50 at id 5, 127 at id 17 for e1; scales 1 / 127
    std::vector<uint16_t> x(2 * 64, 0);
    x[0] = x[64 + 1] = 0x3F80;  // 1.0
    uint16_t* dx = upload(x);
    uint16_t* dr = upload(x);
    float* dn = upload(std::vector<float>(64, 1.0f));
    std::vector<int8_t> w(300 * 64, 0);
    w[250 * 64] = 100, w[5 * 64] = 50, w[17 * 64 + 1] = 127;
    int8_t* dw = upload(w);
    float* dws = upload(std::vector<float>(300, 1.0f / 127.0f));
    const GreedyResult g = lm_head_argmax_i8(dx, dr, dn, 1e-12, dw, dws, 2, 64, 300);
    CHECK((g.ids == std::vector<int32_t>{250, 17}));
    const double a = 8.0 * 100.0 / 127.0, b = 8.0 * 50.0 / 127.0;
    CHECK(std::fabs(g.logit[0] - a) < 1e-4 && std::fabs(g.logit[1] - 8.0) < 1e-4);
    CHECK(std::fabs(g.logprob[0] - (a - std::log(std::exp(a) + std::exp(b) + 298.0))) < 1e-4);
    CHECK(std::fabs(g.logprob[1] - (8.0 - std::log(std::exp(8.0) + 299.0))) < 1e-4);
    std::vector<uint16_t> sum(2 * 64);
    cudaMemcpy(sum.data(), dr, sum.size() * 2, cudaMemcpyDeviceToHost);
    CHECK(sum[0] == 0x4000 && sum[64 + 1] == 0x4000 && sum[1] == 0);  // 2.0
    CHECK(throws([&] { lm_head_argmax_i8(dx, dr, dn, 1e-12, dw, dws, 2, 24, 300); }, "beyond what the kernels support"));
    for (void* p : {static_cast<void*>(dl), static_cast<void*>(di), static_cast<void*>(dx), static_cast<void*>(dr),
                    static_cast<void*>(dn), static_cast<void*>(dw), static_cast<void*>(dws)})
        cudaFree(p);
}

int main(int argc, char** argv) {
    cpu_checks();
    if (argc > 1 && std::strcmp(argv[1], "gpu") == 0) gpu_checks();
    std::fprintf(stderr, "%d checks, %d failures\n", g_checks, g_failures);
    return g_failures == 0 ? 0 : 1;
}
