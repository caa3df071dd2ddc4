// Routing to experts by scores: softmax or sigmoid of the logits, a bias for the choice, groups of experts, the best top_k, weights
// renormalised and scaled.
//
// Which experts a token goes to is a whole number that has no tolerance, and sums of a score and a bias lie closer together than 32 bits
// tell apart: what is compared is worked out in 64 bits (whose instructions take the vector ALU no longer than 32-bit ones).  Without
// a bias the order of the scores is that of the logits, which are compared as they are, in 32.
//
// LANES lanes have a token's experts, e = i LANES + lane: 64 where tokens are few, 16 where they are many, so that a round of the selection
// (a maximum over the lanes on the vector ALU, the lowest expert that has it, its removal) serves four tokens.
//
// Bound by vector instructions where tokens are many, most of them the rounds of the selection: 16384 tokens of 128 experts with a bias 10.2 us, 0.86 TB/s, 1350
// instructions a wave, of which the exponentials, nineteen for each of a lane's eight experts, are an eighth; by launch and the chain of rounds where
// they are few: one token 3.3 us, 509 of 256 experts in eight groups 7.1.
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
    int n, top_k, groups, top_groups, group_best, renormalize, sigmoid;
    float scale;
    int32_t* ids;
    float* weights;
    int lds, group_bits; // bytes of a token; 2^group_bits groups or fewer
    uint32_t by_size;    // 2^20 over the experts of a group, rounded up
};

// A key whose order is that of v (no NaN); 0 is left for what cannot be chosen.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f); // (-0 is 0)
    return u >> 31 ? ~u : u | 0x80000000u;
}
// The larger and the smaller of two f64 numbers, NaN being none.  (fmax first makes sure that neither is a signalling NaN, an instruction each.)
__device__ __forceinline__ double larger(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double smaller(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
// f over LANES (16 or 64) lanes, in all of them
template <int LANES, class F>
__device__ __forceinline__ uint32_t over(uint32_t v, F&& f) {
    v = f(v, dpp_u<0xB1>(v));  // quad_perm [1,0,3,2]
    v = f(v, dpp_u<0x4E>(v));  // quad_perm [2,3,0,1]
    v = f(v, dpp_u<0x141>(v)); // row_half_mirror
    v = f(v, dpp_u<0x140>(v)); // row_mirror
    if constexpr (LANES == 64) {
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f(a[0], a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f(b[0], b[1]);
    }
    return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t most_of(uint32_t v) {
    return over<LANES>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int LANES>
__device__ __forceinline__ uint32_t least_of(uint32_t v) {
    return over<LANES>(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
template <int LANES>
__device__ __forceinline__ float most_of(float v) {
    return __uint_as_float(over<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
// f(v, v of the lanes 16, then 32 away)
template <class F>
__device__ __forceinline__ double over_rows(double v, F&& f) {
    const auto of = [](uint32_t lo, uint32_t hi) { return __longlong_as_double((long long)((uint64_t)hi << 32 | lo)); };
    uint64_t u = (uint64_t)__double_as_longlong(v);
    const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false), b = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    u = (uint64_t)__double_as_longlong(f(of(a[0], b[0]), of(a[1], b[1])));
    const auto c = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false), d = __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    return f(of(c[0], d[0]), of(c[1], d[1]));
}
template <int LANES>
__device__ __forceinline__ double sum_of(double v) {
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    v += dpp_d<0x140>(v);
    if constexpr (LANES == 64) v = over_rows(v, [](double a, double b) { return a + b; });
    return v;
}
template <int LANES>
__device__ __forceinline__ double most_of(double v) {
    v = larger(v, dpp_d<0xB1>(v));
    v = larger(v, dpp_d<0x4E>(v));
    v = larger(v, dpp_d<0x141>(v));
    v = larger(v, dpp_d<0x140>(v));
    if constexpr (LANES == 64) v = over_rows(v, [](double a, double b) { return larger(a, b); });
    return v;
}

__device__ __forceinline__ double sigmoid_of(double l) { // (exponents at most 0)
    const double t = exp_of(-fabs(l));
    return (l >= 0.0 ? 1.0 : t) / (1.0 + t);
}

// What is compared: logits as keys, or (WIDE) f64 numbers, a NaN being none.
template <bool WIDE>
struct Compared {
    typedef uint32_t type;
    static constexpr uint32_t none = 0, least = 0;
    static __device__ __forceinline__ uint32_t more(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t less(uint32_t a, uint32_t b) { return min(a, b); }
    template <int LANES>
    static __device__ __forceinline__ uint32_t of_lane(uint32_t v, int at) { // (the same lane for the whole wave where a token has all 64)
        if constexpr (LANES == 64) return (uint32_t)__builtin_amdgcn_readlane((int)v, at);
        else return __shfl(v, at);
    }
};
template <>
struct Compared<true> {
    typedef double type;
    static constexpr double none = __builtin_nan(""), least = -__builtin_inf();
    static __device__ __forceinline__ double more(double a, double b) { return larger(a, b); }
    static __device__ __forceinline__ double less(double a, double b) { return smaller(a, b); }
    template <int LANES>
    static __device__ __forceinline__ double of_lane(double v, int at) {
        const uint64_t u = (uint64_t)__double_as_longlong(v);
        const uint32_t lo = Compared<false>::of_lane<LANES>((uint32_t)u, at), hi = Compared<false>::of_lane<LANES>((uint32_t)(u >> 32), at);
        return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
    }
};

template <typename T, int PER, int LANES, bool WIDE>
__global__ __launch_bounds__(256) void route_scored_kernel(RouteParams P) {
    using C = Compared<WIDE>;
    typedef typename C::type key_t;
    extern __shared__ __attribute__((aligned(8))) uint8_t smem[]; // per token: with groups what they are compared by, then the logits
    constexpr int kTokens = 64 / LANES;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LANES, here = lane / LANES;
    const int64_t token0 = ((int64_t)blockIdx.x * 4 + wave) * kTokens;
    if (token0 >= P.t) return; // whole waves
    const bool real = token0 + here < P.t;
    const int64_t token = real ? token0 + here : P.t - 1;
    const bool grouped = P.groups > 1 && P.top_groups < P.groups;
    uint8_t* const mine = smem + (wave * kTokens + here) * P.lds;
    key_t* const compared = reinterpret_cast<key_t*>(mine);
    float* const logits = reinterpret_cast<float*>(mine + (grouped ? P.n * (int)sizeof(key_t) : 0));
    const T* const row = static_cast<const T*>(P.logits) + token * P.stride;

    // a NaN counts as -infinity, +infinity as the largest finite number
    float l[PER];
    uint32_t nan = 0;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * LANES + sub;
        l[i] = e < P.n ? (float)row[e] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * LANES + sub;
        nan |= (l[i] != l[i] ? 1u : 0u) << i;
        l[i] = l[i] != l[i] ? -INFINITY : fminf(l[i], 3.402823466e38f);
        if (e < P.n) logits[e] = l[i];
        top = fmaxf(top, l[i]);
    }
    double sum = 0.0, s[WIDE ? PER : 1];
    if (!P.sigmoid) {
        top = most_of<LANES>(top);
        if (WIDE || !P.renormalize) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const double x = top == -INFINITY ? 0.0 : exp_of((double)l[i] - (double)top);
                sum += x;
                if constexpr (WIDE) s[i] = x;
            }
            sum = sum_of<LANES>(sum);
            const double by = sum == 0.0 ? 0.0 : 1.0 / sum;
            if constexpr (WIDE)
#pragma unroll
                for (int i = 0; i < PER; i++) s[i] *= by;
        }
    } else if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < PER; i++) s[i] = sigmoid_of((double)l[i]);
    }
    key_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * LANES + sub;
        if constexpr (WIDE) {
            double c = (double)l[i];
            if (P.bias) {
                c = s[i] + (e < P.n ? (double)P.bias[e] : 0.0);
                c = c != c || nan >> i & 1 ? -INFINITY : c;
            }
            key[i] = e < P.n ? c : C::none;
            if (grouped && e < P.n) compared[e] = P.bias ? c : s[i];
        } else {
            key[i] = e < P.n ? key_of(l[i]) : 0u;
            if (grouped && e < P.n) compared[e] = key[i];
        }
    }
    if (grouped) {
        asm volatile("" ::: "memory"); // (a wave's LDS instructions run in their order)
        __builtin_amdgcn_wave_barrier();
        // `share` lanes to a group look for its two best
        const int share = LANES >> P.group_bits, g = sub / share, size = P.n / P.groups;
        key_t a = C::least, b = C::least;
        if (g < P.groups)
            for (int i = sub % share; i < size; i += share) {
                const key_t v = compared[g * size + i];
                b = C::more(b, C::less(a, v)), a = C::more(a, v);
            }
        for (int o = 1; o < share; o <<= 1) {
            const key_t c = __shfl_xor(a, o), d = __shfl_xor(b, o);
            b = C::more(C::less(a, c), C::more(b, d)), a = C::more(a, c);
        }
        key_t worth = a;
        if constexpr (WIDE)
            if (P.group_best > 1 && size > 1) {
                worth = a + b;
                worth = worth != worth ? -INFINITY : worth;
            }
        int before = 0; // groups that are worth more, or as much and come first
        for (int o = 0; o < P.groups; o++) {
            const key_t other = C::template of_lane<LANES>(worth, here * LANES + o * share);
            before += other > worth || (other == worth && o < g);
        }
        const uint64_t kept = __ballot(g < P.groups && before < P.top_groups) >> (here * LANES); // (of this token: from bit 0 on)
#pragma unroll
        for (int i = 0; i < PER; i++) { // (e / size by its reciprocal: exact for all e < 1024)
            const int e = i * LANES + sub, at = (int)((uint32_t)e * P.by_size >> 20) * share;
            if (!(kept >> at & 1)) key[i] = C::none;
        }
    }
    int my_id = 0; // lane k: of slot k
    for (int k = 0; k < P.top_k; k++) {
        key_t most = key[0];
#pragma unroll
        for (int i = 1; i < PER; i++) most = C::more(most, key[i]);
        most = most_of<LANES>(most);
        uint32_t e = 0xffffu;
#pragma unroll
        for (int i = PER - 1; i >= 0; i--) e = key[i] == most ? i * LANES + sub : e;
        e = least_of<LANES>(e);
#pragma unroll
        for (int i = 0; i < PER; i++) key[i] = (uint32_t)(i * LANES + sub) == e ? C::none : key[i];
        my_id = sub == k ? (int)e : my_id;
    }

    // weights: renormalised ones relative to the largest chosen logit, so that none is lost however small the scores are
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    const float my_logit = sub < P.top_k ? logits[my_id] : -INFINITY;
    const double v = (double)my_logit;
    double w = 0.0;
    if (P.renormalize) {
        const double best = (double)most_of<LANES>(my_logit);
        if (my_logit > -INFINITY) {
            if (P.sigmoid) w = (v <= 0.0 ? exp_of(v - fmin(best, 0.0)) : 1.0) / (1.0 + exp_of(-fabs(v)));
            else w = exp_of(v - best);
        }
        const double total = sum_of<LANES>(w);
        w = total == 0.0 ? 0.0 : w / total;
    } else if (my_logit > -INFINITY) {
        w = P.sigmoid ? sigmoid_of(v) : exp_of(v - (double)top) / sum;
    }
    if (sub < P.top_k && real) {
        P.ids[token * P.top_k + sub] = my_id;
        P.weights[token * P.top_k + sub] = (float)(w * (double)P.scale);
    }
}

template <typename T, int PER, int LANES>
hipError_t launch(RouteParams P, hipStream_t stream) {
    constexpr int kTokens = 4 * 64 / LANES; // of a workgroup
    const bool grouped = P.groups > 1 && P.top_groups < P.groups, wide = P.bias || (grouped && P.group_best > 1);
    P.lds = (P.n * (4 + (grouped ? (wide ? 8 : 4) : 0)) + 7) / 8 * 8;
    while (1 << P.group_bits < P.groups) P.group_bits++;
    P.by_size = (1u << 20) / (uint32_t)(P.n / P.groups) + 1;
    const unsigned grid = (unsigned)((P.t + kTokens - 1) / kTokens);
    if (wide) route_scored_kernel<T, PER, LANES, true><<<grid, 256, (size_t)kTokens * P.lds, stream>>>(P);
    else route_scored_kernel<T, PER, LANES, false><<<grid, 256, (size_t)kTokens * P.lds, stream>>>(P);
    return hipGetLastError();
}
// Sixteen lanes a token where tokens are many: 128 experts 4096 tokens 4.3 us, 5.8 with 64 lanes, 2000 4.2 either way; 64 experts with a bias 2000
// tokens 4.6, 5.2; 256 in groups, sixteen of them a lane, 16384 tokens 26, 28.5, but 4096 12.0, 10.3.
template <typename T>
hipError_t launch_of(const RouteParams& P, int n_cus, hipStream_t stream) {
    const int n = P.n;
    if (P.t >= (int64_t)(n <= 128 ? 4 : 32) * n_cus && n <= 256 && P.top_k <= 16 && P.groups <= 16)
        return n <= 64 ? launch<T, 4, 16>(P, stream) : n <= 128 ? launch<T, 8, 16>(P, stream) : launch<T, 16, 16>(P, stream);
    return n <= 64    ? launch<T, 1, 64>(P, stream)
           : n <= 128 ? launch<T, 2, 64>(P, stream)
           : n <= 256 ? launch<T, 4, 64>(P, stream)
           : n <= 512 ? launch<T, 8, 64>(P, stream)
                      : launch<T, 16, 64>(P, stream);
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
    // (four tokens to a workgroup of 256 threads, of which a launch has fewer than 2^32)
    if (t > 0x3fffffc || stride > 0x3fffffff) return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: %lld tokens, rows %lld apart", what, (long long)t, (long long)stride);
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
    const RouteParams P{logits, stride, bias, t, n, top_k, groups, top_groups, group_best, renormalize != 0, scoring == IZWI_MOE_SIGMOID, scale, ids, weights, 0, 0, 0};
    const hipError_t e = launch_of<T>(P, n_cus, (hipStream_t)stream_);
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
