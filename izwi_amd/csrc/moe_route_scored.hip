// Routing to experts by scores: softmax or sigmoid of the logits, a bias for the choice, groups of experts, the best top_k, weights
// renormalised and scaled.
//
// Scores and choices are worked out and compared in 64 bits: sums of a score and a bias lie closer together than 32 bits tell apart,
// and which experts a token goes to is a whole number that has no tolerance.  Without a bias the order of the scores is the
// order of the logits, which are compared instead.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/izwi_qmm.h"
#include "qmm_internal.h"
#include "qmm_lanes.h"

namespace {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

struct RouteParams {
    const void* logits;
    int64_t stride;
    const float* bias;
    int64_t t;
    int n, top_k, groups, top_groups, group_best, renormalize;
    float scale;
    int32_t* ids;
    float* weights;
};

// A key whose order is that of v: 0 is left for what cannot be chosen, a NaN is below every number.
__device__ __forceinline__ uint64_t key_of(double v) {
    if (v != v) v = -INFINITY;
    uint64_t u = (uint64_t)__double_as_longlong(v);
    if (u == 0x8000000000000000ull) u = 0; // -0
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double value_of(uint64_t key) { return __longlong_as_double((long long)(key >> 63 ? key & 0x7fffffffffffffffull : ~key)); }

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, o));
    return v;
}
__device__ __forceinline__ double wave_add(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// A wave per token, lane l having experts l, l + 64, ..
template <typename T, int PER, bool SIGMOID>
__global__ __launch_bounds__(256) void route_scored_kernel(RouteParams P) {
    extern __shared__ uint64_t smem[]; // per wave: keys of the experts (where there are groups)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t token = (int64_t)blockIdx.x * 4 + wave;
    if (token >= P.t) return; // whole waves
    const T* const row = static_cast<const T*>(P.logits) + token * P.stride;
    float l[PER];
    uint64_t key[PER];
    double top = -INFINITY, sum = 0.0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 64 * i;
        const float v = e < P.n ? (float)row[e] : -INFINITY;
        l[i] = v != v ? -INFINITY : fminf(v, 3.402823466e38f);
        key[i] = e < P.n ? key_of(v != v ? (double)-INFINITY : (double)l[i]) : 0;
        top = fmax(top, (double)l[i]);
    }
    if constexpr (!SIGMOID) {
#pragma unroll
        for (int o = 32; o; o >>= 1) top = fmax(top, __shfl_xor(top, o));
        if (P.bias || !P.renormalize || (P.groups > 1 && P.group_best > 1)) {
#pragma unroll
            for (int i = 0; i < PER; i++) sum += top == -INFINITY ? 0.0 : exp((double)l[i] - top);
            sum = wave_add(sum);
        }
    }
    const auto score = [&](double v) -> double {
        if constexpr (SIGMOID) return 1.0 / (1.0 + exp(-v));
        return sum == 0.0 ? 0.0 : exp(v - top) / sum;
    };
    const bool by_score = P.bias || (P.groups > 1 && P.group_best > 1); // (uniform)
    if (P.bias) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane + 64 * i;
            if (e >= P.n) continue;
            const float v = (float)row[e];
            key[i] = key_of(v != v ? (double)-INFINITY : score((double)l[i]) + (double)P.bias[e]);
        }
    }
    if (P.groups > 1) {
        uint64_t* const keys = smem + wave * P.n;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 64 * i < P.n) keys[lane + 64 * i] = key[i];
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        const int size = P.n / P.groups;
        uint64_t worth = 0; // of group `lane`
        if (lane < P.groups) {
            uint64_t a = 0, b = 0; // its two best
            for (int i = 0; i < size; i++) {
                const uint64_t v = keys[lane * size + i];
                if (v > a) b = a, a = v;
                else if (v > b) b = v;
            }
            worth = a;
            if (P.group_best > 1) {
                double w = P.bias ? value_of(a) : score(value_of(a));
                if (b) w += P.bias ? value_of(b) : score(value_of(b));
                worth = key_of(w);
            }
        }
        (void)by_score;
        int before = 0; // groups that are worth more, or as much and come first
        for (int g = 0; g < P.groups; g++) {
            const uint64_t other = __shfl((unsigned long long)worth, g);
            before += other > worth || (other == worth && g < lane);
        }
        const uint64_t kept = __ballot(lane < P.groups && before < P.top_groups);
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 64 * i < P.n && !(kept >> ((lane + 64 * i) / size) & 1)) key[i] = 0;
    }
    int my_id = 0;
    float my_logit = -INFINITY, best = -INFINITY; // lane s: slot s; the largest chosen logit
    for (int s = 0; s < P.top_k; s++) {
        uint64_t most = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) most = max(most, key[i]);
        most = wave_max(most);
        int win = -1;
        float logit = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const uint64_t holders = __ballot(key[i] == most);
            if (win < 0 && holders) {
                const int at = __ffsll((long long)holders) - 1;
                win = at + 64 * i;
                logit = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l[i]), at));
                if (lane == at) key[i] = 0;
            }
        }
        best = fmaxf(best, logit);
        if (lane == s) my_id = win, my_logit = logit;
    }
    // weights: renormalised ones relative to the largest chosen logit, so that none is lost however small the scores are
    double w = 0.0;
    if (lane < P.top_k && my_logit > -INFINITY) {
        const double v = (double)my_logit;
        if (!P.renormalize) {
            w = score(v);
        } else if constexpr (SIGMOID) {
            const double m = fmin((double)best, 0.0);
            w = v <= 0.0 ? exp(v - m) / (1.0 + exp(v)) : exp(-m) / (1.0 + exp(-v));
        } else {
            w = exp(v - (double)best);
        }
    }
    if (P.renormalize) {
        const double total = wave_add(w);
        w = total == 0.0 ? 0.0 : w / total;
    }
    if (lane < P.top_k) {
        P.ids[token * P.top_k + lane] = my_id;
        P.weights[token * P.top_k + lane] = (float)(w * (double)P.scale);
    }
}

template <typename T, int PER>
hipError_t launch_of(const RouteParams& P, int sigmoid, hipStream_t stream) {
    const unsigned grid = (unsigned)((P.t + 3) / 4);
    const size_t lds = P.groups > 1 ? (size_t)4 * P.n * sizeof(uint64_t) : 0;
    if (sigmoid) route_scored_kernel<T, PER, true><<<grid, 256, lds, stream>>>(P);
    else route_scored_kernel<T, PER, false><<<grid, 256, lds, stream>>>(P);
    return hipGetLastError();
}

template <typename T>
int route_scored_impl(const T* logits, int64_t stride, const float* bias, int64_t t, int32_t n, int32_t top_k, int32_t scoring, int32_t groups,
                      int32_t top_groups, int32_t group_best, int32_t renormalize, float scale, int32_t* ids, float* weights, void* stream_) {
    constexpr const char* what = "moe_route_scored";
    if (t < 0 || n < 1 || stride < n) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: bad shape (%lld tokens, %d experts, rows %lld apart)", what, (long long)t, n, (long long)stride);
    if (n > 1024) return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: %d experts (at most 1024)", what, n);
    if (groups < 1 || groups > 64 || n % groups || top_groups < 1 || top_groups > groups || group_best < 1 || group_best > 2)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: %d of %d groups of %d experts by their best %d (1 or 2)", what, top_groups, groups, n, group_best);
    if (top_k < 1 || top_k > 64 || top_k > n / groups * top_groups)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: top_k %d of %d experts in %d of %d groups (at most 64)", what, top_k, n, top_groups, groups);
    if (scoring != IZWI_MOE_SOFTMAX && scoring != IZWI_MOE_SIGMOID) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: scoring %d", what, scoring);
    if (!std::isfinite(scale)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: scale %g", what, (double)scale);
    if (t > 0x3fffffff / top_k || stride > 0x3fffffff) return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: %lld tokens, rows %lld apart", what, (long long)t, (long long)stride);
    if (t == 0) return IZWI_QMM_OK;
    if (!logits || !ids || !weights) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: NULL buffer", what);
    const auto overlap = [](const void* a, uintptr_t an, const void* b, uintptr_t bn) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
        return x < y + bn && y < x + an;
    };
    const uintptr_t in = ((uintptr_t)(t - 1) * stride + n) * sizeof(T), out = (uintptr_t)t * top_k * 4, b = bias ? (uintptr_t)n * 4 : 0;
    if (overlap(ids, out, weights, out) || overlap(ids, out, logits, in) || overlap(weights, out, logits, in) || (bias && (overlap(ids, out, bias, b) || overlap(weights, out, bias, b))))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: an output shares memory with another tensor", what);
    int device = 0, n_cus = 0;
    if (int rc = qmm_current_device(&device, &n_cus)) return rc;
    const RouteParams P{logits, stride, bias, t, n, top_k, groups, top_groups, group_best, renormalize != 0, scale, ids, weights};
    hipStream_t stream = (hipStream_t)stream_;
    const int per = (n + 63) / 64;
    const hipError_t e = per <= 1   ? launch_of<T, 1>(P, scoring, stream)
                         : per <= 2 ? launch_of<T, 2>(P, scoring, stream)
                         : per <= 4 ? launch_of<T, 4>(P, scoring, stream)
                         : per <= 8 ? launch_of<T, 8>(P, scoring, stream)
                                    : launch_of<T, 16>(P, scoring, stream);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        return qmm_fail(IZWI_QMM_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    }
    return IZWI_QMM_OK;
}

} // namespace

extern "C" {

#define ROUTE_SCORED(NAME, C, T)                                                                                                                          \
    int NAME(const C* logits, int64_t stride, const float* bias, int64_t t, int32_t n_experts, int32_t top_k, int32_t scoring, int32_t groups,            \
             int32_t top_groups, int32_t group_best, int32_t renormalize, float scale, int32_t* ids, float* weights, void* stream) {                      \
        return qmm_guarded(#NAME, [&]() -> int {                                                                                                          \
            return route_scored_impl<T>((const T*)logits, stride, bias, t, n_experts, top_k, scoring, groups, top_groups, group_best, renormalize, scale, \
                                        ids, weights, stream);                                                                                            \
        });                                                                                                                                               \
    }
ROUTE_SCORED(izwi_moe_route_scored_f32, float, float)
ROUTE_SCORED(izwi_moe_route_scored_f16, uint16_t, f16_t)
ROUTE_SCORED(izwi_moe_route_scored_bf16, uint16_t, bf16_t)

} // extern "C"
