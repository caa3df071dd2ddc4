// The operators on whole prompts through the C++ host-side mirror (izwi_amd/host/izwi_qmm.hpp).
//   prompt_mirror_test cpu   frequencies, and calls that are refused before any device work
//   prompt_mirror_test gpu   rotary positions, attention and routing of a few tokens against their formulas in 64 bits
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "izwi_qmm.hpp"

extern "C" {
int hipMalloc(void** ptr, size_t bytes);
int hipMemcpy(void* to, const void* from, size_t bytes, int kind); // 1 to the device, 2 from it
int hipDeviceSynchronize();
}

static int failures = 0;
#define EXPECT(cond)                                                    \
    do {                                                                \
        if (!(cond)) {                                                  \
            std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            failures++;                                                 \
        }                                                               \
    } while (0)

template <class F>
static bool refused(F&& f) {
    try {
        f();
    } catch (const izwi::Error& e) {
        return e.kind() == izwi::Error::Kind::InvalidInput;
    }
    return false;
}

template <typename T>
static T* on_device(const std::vector<T>& v) {
    void* p = nullptr;
    if (hipMalloc(&p, v.size() * sizeof(T)) || hipMemcpy(p, v.data(), v.size() * sizeof(T), 1)) std::printf("no device memory\n"), failures++;
    return static_cast<T*>(p);
}
template <typename T>
static std::vector<T> on_host(const T* p, size_t n) {
    std::vector<T> v(n);
    if (hipDeviceSynchronize() || hipMemcpy(v.data(), p, n * sizeof(T), 2)) std::printf("no copy\n"), failures++;
    return v;
}

static void cpu() {
    std::vector<double> f;
    EXPECT(izwi::kernels::rope_frequencies(IZWI_ROPE_PLAIN, 8, 1e4, 1, 0, 0, 0, f) == 1.0);
    EXPECT(f.size() == 4);
    for (int i = 0; i < 4; i++) EXPECT(std::fabs(f[i] - std::pow(1e4, -2.0 * i / 8)) <= 1e-15 * f[i]);
    EXPECT(std::fabs(izwi::kernels::rope_frequencies(IZWI_ROPE_YARN, 64, 1e4, 4, 4096, 1, 32, f) - (0.1 * std::log(4.0) + 1)) <= 1e-15);
    EXPECT(f.size() == 32 && f[0] == 1.0 && std::fabs(f[31] * 4 - std::pow(1e4, -62.0 / 64)) <= 1e-15);
    for (int64_t dim : {(int64_t)0, (int64_t)-2, (int64_t)7, (int64_t)2048, (int64_t)1 << 40})
        EXPECT(refused([&] { izwi::kernels::rope_frequencies(IZWI_ROPE_PLAIN, dim, 1e4, 1, 0, 0, 0, f); }));
    float* p = reinterpret_cast<float*>(4096); // (never followed)
    const int32_t* ids = reinterpret_cast<int32_t*>(4096);
    EXPECT(refused([&] { izwi::kernels::prompt_attention(p, 100, p, 64, p, 64, nullptr, nullptr, 1, 4, 4, 4, 2, 1, 64, true, 0.1f, p, 128); }));
    EXPECT(refused([&] { izwi::kernels::rope_positions(p, 128, nullptr, 0, ids, nullptr, 1.0, 4, 2, 0, 64, 64, false, nullptr, 0, p, 128, nullptr, 0); }));
    EXPECT(refused([&] { izwi::kernels::moe_route_scored(p, 8, nullptr, 4, 8, 9, IZWI_MOE_SOFTMAX, 1, 1, 1, true, 1.0f, reinterpret_cast<int32_t*>(p), p); }));
}

static void gpu() {
    const int tokens = 5, heads = 2, d = 64, experts = 8, top_k = 2;
    std::vector<float> x(tokens * heads * d);
    for (size_t i = 0; i < x.size(); i++) x[i] = std::sin(0.7f * (float)i);
    std::vector<double> f;
    const double factor = izwi::kernels::rope_frequencies(IZWI_ROPE_PLAIN, d, 1e4, 1, 0, 0, 0, f);
    float *q = on_device(x), *turned = on_device(x), *out = on_device(x);
    int32_t* positions = on_device(std::vector<int32_t>{0, 1, 7, 100, 1000});
    const double* frequencies = on_device(f);
    izwi::kernels::rope_positions(q, heads * d, nullptr, 0, positions, frequencies, factor, tokens, heads, 0, d, d, false, nullptr, 0.0f, turned, heads * d, nullptr, 0);
    const std::vector<float> y = on_host(turned, x.size());
    const int at[] = {0, 1, 7, 100, 1000};
    double off = 0;
    for (int t = 0; t < tokens; t++)
        for (int h = 0; h < heads; h++)
            for (int i = 0; i < d / 2; i++) {
                const double a = x[(t * heads + h) * d + i], b = x[(t * heads + h) * d + d / 2 + i], c = std::cos(at[t] * f[i]), s = std::sin(at[t] * f[i]);
                off = std::fmax(off, std::fabs(y[(t * heads + h) * d + i] - (a * c - b * s)));
                off = std::fmax(off, std::fabs(y[(t * heads + h) * d + d / 2 + i] - (a * s + b * c)));
            }
    EXPECT(off <= 4e-7); // two products and a sum of numbers up to 1, rounded, of factors rounded once: 5 times 2^-24
    // two prompts of 2 and 3 tokens on one kv head (the first head of every row)
    int32_t* starts = on_device(std::vector<int32_t>{0, 2, 5});
    izwi::kernels::prompt_attention(q, heads * d, turned, heads * d, q, heads * d, starts, starts, 2, tokens, tokens, 3, heads, 1, d, true, 0.125f, out, heads * d);
    const std::vector<float> o = on_host(out, x.size());
    off = 0;
    for (int t = 0; t < tokens; t++)
        for (int h = 0; h < heads; h++) {
            const int first = t < 2 ? 0 : 2;
            std::vector<double> w, sum(d, 0.0);
            double total = 0;
            for (int j = first; j <= t; j++) {
                double s = 0;
                for (int i = 0; i < d; i++) s += (double)x[(t * heads + h) * d + i] * y[j * heads * d + i];
                total += std::exp(0.125 * s);
                for (int i = 0; i < d; i++) sum[i] += std::exp(0.125 * s) * x[j * heads * d + i];
            }
            for (int i = 0; i < d; i++) off = std::fmax(off, std::fabs(o[(t * heads + h) * d + i] - sum[i] / total));
        }
    // scores of up to 8 (64 products below 1, an eighth): off by 8 (6 * 64 / 16 + 20) 2^-24 at most, a mean of values below 1 by that and 2^-21
    EXPECT(off <= 8 * 44 * std::ldexp(1.0, -24) + std::ldexp(1.0, -21));
    std::vector<float> logits(tokens * experts);
    for (size_t i = 0; i < logits.size(); i++) logits[i] = std::cos(1.3f * (float)i);
    float *l = on_device(logits), *weights = on_device(std::vector<float>(tokens * top_k));
    int32_t* chosen = on_device(std::vector<int32_t>(tokens * top_k));
    izwi::kernels::moe_route_scored(l, experts, nullptr, tokens, experts, top_k, IZWI_MOE_SOFTMAX, 1, 1, 1, true, 1.0f, chosen, weights);
    const std::vector<int32_t> ids = on_host(chosen, tokens * top_k);
    const std::vector<float> w = on_host(weights, tokens * top_k);
    for (int t = 0; t < tokens; t++) {
        const float* row = logits.data() + t * experts;
        int one = 0, two = -1;
        for (int e = 1; e < experts; e++)
            if (row[e] > row[one]) one = e;
        for (int e = 0; e < experts; e++)
            if (e != one && (two < 0 || row[e] > row[two])) two = e;
        const double share = 1 / (1 + std::exp((double)row[two] - row[one]));
        EXPECT(ids[t * top_k] == one && ids[t * top_k + 1] == two);
        EXPECT(std::fabs(w[t * top_k] - share) <= std::ldexp(1.0, -24) && std::fabs(w[t * top_k + 1] - (1 - share)) <= std::ldexp(1.0, -24));
    }
}

int main(int argc, char** argv) {
    try {
        if (argc > 1 && !std::strcmp(argv[1], "gpu")) gpu();
        else cpu();
    } catch (const izwi::Error& e) {
        std::printf("unexpected error: %s\n", e.what());
        failures++;
    }
    std::printf(failures ? "%d checks failed\n" : "all checks passed\n", failures);
    return failures != 0;
}
