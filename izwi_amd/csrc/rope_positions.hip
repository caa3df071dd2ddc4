// Rotary positions of packed tokens: (a, b) -> (a cos - b sin, a sin + b cos) for the pairs of a head's first rotary_dim elements, angle
// position * frequency, optionally behind the head's RMSNorm; and the frequencies of models whose context is stretched.
//
// Angles are taken in 64 bits (position 10^6 in 32 bits would be off by 0.03), reduced by multiples of a quarter turn there, and cosine and sine
// worked out in 64 bits, too: times the factor they are rounded to 32 bits once.  (As 32-bit functions of a fraction of a turn in 32 bits
// they left f32 results 1.4 times as far off.  The f64 instructions are a few more and take no longer.)
//
// Bound by memory where there is much to do: 16384 tokens of 32 and 8 heads of 128, f32, 126 us, 5.3 TB/s (a copy of 1 GiB reaches 5.2; part of
// this fits the last-level cache); 2051 tokens bf16 with the norm, parts of q|k|v rows, 12.0 us, 3.5 TB/s.  By the launch and one chain
// of loads, angles (f64) and stores where there is little: one token 3.2 us, 777 of 24 heads of 64 4.3.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/izwi_decode_ops.h"
#include "qmm_internal.h"
#include "qmm_lanes.h"

namespace {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

struct RopeParams {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_stride, k_stride, q_out_stride, k_out_stride; // elements from a token to the next
    const int32_t* positions;
    const double* frequencies; // [rotary / 2]
    const void* weight;        // [2 d]: q's, then k's; NULL: no norm
    double factor;
    float eps;
    int64_t tokens;
    int q_heads, heads, d, rotary; // heads: q's and k's
};

constexpr int kMostPairs = 512;

// Cosine and sine of position * frequency, times the factor.  What is left of the angle, n quarter turns less (pi / 2 as two numbers; the first fma
// is exact), is at most pi / 4, where the series' next terms are below 2^-36 of the sum.
__device__ __forceinline__ void turn_of(const RopeParams& P, int position, int pair, float& c, float& s) {
    const double angle = (double)position * P.frequencies[pair], n = __builtin_rint(angle * 0.63661977236758134308);
    const double r = __builtin_fma(n, -0x1.1a62633145c07p-54, __builtin_fma(n, -0x1.921fb54442d18p+0, angle)), r2 = r * r;
    double sine = __builtin_fma(r2, -1.0 / 39916800, 1.0 / 362880);
    sine = __builtin_fma(sine, r2, -1.0 / 5040);
    sine = __builtin_fma(sine, r2, 1.0 / 120);
    sine = __builtin_fma(sine, r2, -1.0 / 6);
    sine = __builtin_fma(sine * r2, r, r);
    double cosine = __builtin_fma(r2, 1.0 / 479001600, -1.0 / 3628800);
    cosine = __builtin_fma(cosine, r2, 1.0 / 40320);
    cosine = __builtin_fma(cosine, r2, -1.0 / 720);
    cosine = __builtin_fma(cosine, r2, 1.0 / 24);
    cosine = __builtin_fma(cosine, r2, -0.5);
    cosine = __builtin_fma(cosine, r2, 1.0);
    const int quarter = (int)(n - 4.0 * __builtin_floor(n * 0.25)); // 0 to 3
    const double x = quarter & 1 ? sine : cosine, y = quarter & 1 ? cosine : sine;
    c = (float)(((quarter + 1) & 2 ? -x : x) * P.factor), s = (float)((quarter & 2 ? -y : y) * P.factor);
}

// A workgroup per token (in turn), a wave per head in turn, a lane per pair of elements in turn.
template <typename T, bool INTER>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeParams P) {
    __shared__ float cosine[kMostPairs], sine[kMostPairs];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pairs = P.rotary / 2;
    for (int64_t token = blockIdx.x; token < P.tokens; token += gridDim.x) {
        const int position = P.positions[token];
        for (int i = threadIdx.x; i < pairs; i += 256) turn_of(P, position, i, cosine[i], sine[i]);
        __syncthreads();
        for (int head = wave; head < P.heads; head += 4) {
            const bool is_q = head < P.q_heads;
            const int at = is_q ? head : head - P.q_heads;
            const T* const from = static_cast<const T*>(is_q ? P.q : P.k) + token * (is_q ? P.q_stride : P.k_stride) + (int64_t)at * P.d;
            T* const to = static_cast<T*>(is_q ? P.q_out : P.k_out) + token * (is_q ? P.q_out_stride : P.k_out_stride) + (int64_t)at * P.d;
            const T* const weight = P.weight ? static_cast<const T*>(P.weight) + (is_q ? 0 : P.d) : nullptr;
            float by = 1.0f;
            if (weight) {
                float sum = 0.0f;
                for (int i = lane; i < P.d; i += 64) {
                    const float v = (float)from[i];
                    sum += v * v;
                }
                by = 1.0f / sqrtf(wave_sum(sum) / (float)P.d + P.eps);
                asm volatile("" ::: "memory"); // (in place, lanes read others' elements above)
                __builtin_amdgcn_wave_barrier();
            }
            for (int i = lane; i < P.d / 2; i += 64) {
                const bool turns = i < pairs;
                const int a = turns && !INTER ? i : 2 * i, b = turns && !INTER ? i + pairs : 2 * i + 1;
                float u = (float)from[a], v = (float)from[b];
                if (weight) u = u * by * (float)weight[a], v = v * by * (float)weight[b];
                const float c = turns ? cosine[i] : 1.0f, s = turns ? sine[i] : 0.0f;
                to[a] = (T)(turns ? u * c - v * s : u);
                to[b] = (T)(turns ? u * s + v * c : v);
            }
        }
        __syncthreads(); // (cosines and sines are read)
    }
}

// The same in pieces of 16 bytes: a lane has two pieces of a head, those whose elements turn against each other (halves) or two neighbours
// (interleaved, and what does not turn), LP lanes a head, 64 / LP heads at once; a wave has `passes` such sets of one token's heads, requests
// kAtOnce of them ahead of working out the angles, and every angle once (a token whose heads go to several waves has its angles worked out
// by each).  (Pairs of single elements, a workgroup a token: 2051 tokens 32 us instead of 12.)  Reading the angles back has two lanes on a
// bank (a lane's are 64 bytes on from its neighbour's): 44 % of the LDS's cycles in use, which are 4 % of a busy compute unit's.
constexpr int kAtOnce = 4, kPiecePairs = 256;

template <typename T, int V>
struct Piece {
    typedef T vec __attribute__((ext_vector_type(V)));
    vec v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const vec*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<vec*>(p) = v; }
};

// sum over LP neighbouring lanes, in all of them
__device__ __forceinline__ float sum_lanes(float v, int lp) {
    if (lp > 1) v += dpp_f<0xB1>(v);  // quad_perm [1,0,3,2]
    if (lp > 2) v += dpp_f<0x4E>(v);  // quad_perm [2,3,0,1]
    if (lp > 4) v += dpp_f<0x141>(v); // row_half_mirror
    if (lp > 8) v += dpp_f<0x128>(v); // row_ror:8
    if (lp > 16) v = qmm_add_lane16(v);
    if (lp > 32) v = qmm_add_lane32(v);
    return v;
}

template <typename T, bool INTER, bool NORM>
__global__ __launch_bounds__(256) void rope_pieces_kernel(RopeParams P, int lp, int per_head, int passes, int shares) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float2 turns_of[4][kPiecePairs];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave, token = unit / shares;
    if (token >= P.tokens) return; // whole waves
    const int share = (int)(unit - token * shares), first = share * passes;
    const int sub = lane & (lp - 1), group = lane / lp, at_once = 64 / lp, pairs = P.rotary / 2;
    // the lane's pieces of a head
    const int rotating = pairs / V; // lanes whose pieces turn
    const bool turns = sub < rotating;
    const int a = turns ? (INTER ? 2 * sub * V : sub * V) : P.rotary + 2 * (sub - rotating) * V;
    const int b = turns && !INTER ? a + pairs : a + V;
    const int n = min(passes, (P.heads + at_once - 1) / at_once - first);

    struct Rows {
        const T* from;
        T* to;
        bool is_q, there;
    };
    const auto rows = [&](int pass) {
        const int head = (first + pass) * at_once + group;
        Rows r;
        r.there = sub < per_head && head < P.heads && pass < n;
        r.is_q = head < P.q_heads;
        const int64_t at = (int64_t)(r.there ? (r.is_q ? head : head - P.q_heads) : 0) * P.d;
        r.from = static_cast<const T*>(r.is_q ? P.q : P.k) + token * (r.is_q ? P.q_stride : P.k_stride) + at;
        r.to = static_cast<T*>(r.is_q ? P.q_out : P.k_out) + token * (r.is_q ? P.q_out_stride : P.k_out_stride) + at;
        return r;
    };
    Piece<T, V> x[kAtOnce], y[kAtOnce], wx[kAtOnce], wy[kAtOnce];
    const auto request = [&](int pass0) {
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const Rows r = rows(pass0 + i);
            if (!r.there) continue;
            x[i].load(r.from + a), y[i].load(r.from + b);
            if constexpr (NORM) {
                const T* const w = static_cast<const T*>(P.weight) + (r.is_q ? 0 : P.d);
                wx[i].load(w + a), wy[i].load(w + b);
            }
        }
    };
    const int position = P.positions[token];
    request(0);
    for (int i = lane; i < pairs; i += 64) {
        float c, s;
        turn_of(P, position, i, c, s);
        turns_of[wave][i] = float2{c, s};
    }
    asm volatile("" ::: "memory"); // (a wave's LDS instructions run in their order)
    __builtin_amdgcn_wave_barrier();
    float c[V], s[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float2 t = turns_of[wave][turns ? sub * V + i : 0];
        c[i] = t.x, s[i] = t.y;
    }
    for (int pass0 = 0; pass0 < n; pass0 += kAtOnce) {
        if (pass0) request(pass0);
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const Rows r = rows(pass0 + i);
            float u[2 * V]; // the pieces, one behind the other
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < V; j++) {
                u[j] = r.there ? (float)x[i].v[j] : 0.0f, u[V + j] = r.there ? (float)y[i].v[j] : 0.0f;
                if constexpr (NORM) sum += u[j] * u[j] + u[V + j] * u[V + j];
            }
            if constexpr (NORM) {
                const float by = 1.0f / sqrtf(sum_lanes(sum, lp) / (float)P.d + P.eps);
                if (!r.there) continue;
#pragma unroll
                for (int j = 0; j < V; j++) u[j] = u[j] * by * (float)wx[i].v[j], u[V + j] = u[V + j] * by * (float)wy[i].v[j];
            }
            if (!r.there) continue;
            if (turns) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const int p = INTER ? 2 * j : j, q = INTER ? 2 * j + 1 : V + j;
                    const float e = u[p] * c[j] - u[q] * s[j], f = u[p] * s[j] + u[q] * c[j];
                    u[p] = e, u[q] = f;
                }
            }
            Piece<T, V> xo, yo;
#pragma unroll
            for (int j = 0; j < V; j++) xo.v[j] = (T)u[j], yo.v[j] = (T)u[V + j];
            xo.store(r.to + a), yo.store(r.to + b);
        }
    }
}

#define ROPE_TRY(expr)                                                                 \
    do {                                                                               \
        hipError_t e_ = (expr);                                                        \
        if (e_ != hipSuccess) {                                                        \
            (void)hipGetLastError();                                                   \
            return qmm_fail(IZWI_QMM_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
        }                                                                              \
    } while (0)

template <typename T>
int rope_positions_impl(const T* q, int64_t q_stride, const T* k, int64_t k_stride, const int32_t* positions, const double* frequencies, double factor,
                        int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t d, int64_t rotary, int interleaved, const T* weight, float eps, T* q_out,
                        int64_t q_out_stride, T* k_out, int64_t k_out_stride, void* stream_) {
    constexpr const char* what = "rope_positions";
    if (tokens < 0 || q_heads < 0 || k_heads < 0 || q_heads > 65535 || k_heads > 65535 || d <= 0 || d % 2 || d > 2 * kMostPairs || rotary <= 0 || rotary % 2 || rotary > d)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: bad shape (tokens %lld, heads %lld and %lld of %lld, of which %lld turn: even, at most %d)", what, (long long)tokens,
                        (long long)q_heads, (long long)k_heads, (long long)d, (long long)rotary, 2 * kMostPairs);
    if ((q_heads && (q_stride < q_heads * d || q_out_stride < q_heads * d)) || (k_heads && (k_stride < k_heads * d || k_out_stride < k_heads * d)))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: rows overlap (strides %lld, %lld, %lld, %lld)", what, (long long)q_stride, (long long)k_stride,
                        (long long)q_out_stride, (long long)k_out_stride);
    if (interleaved != 0 && interleaved != 1) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: layout %d (0 halves, 1 interleaved)", what, interleaved);
    if (!std::isfinite((float)factor) || !(eps >= 0.0f) || !std::isfinite(eps)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: factor %g, eps %g", what, factor, (double)eps);
    // (four tokens to a workgroup of 256 threads, of which a launch has fewer than 2^32)
    if (tokens > 0x3fffffc || q_stride > 0x3fffffff || k_stride > 0x3fffffff || q_out_stride > 0x3fffffff || k_out_stride > 0x3fffffff)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: %lld tokens", what, (long long)tokens);
    if (tokens == 0 || q_heads + k_heads == 0) return IZWI_QMM_OK;
    if (!positions || !frequencies || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: NULL buffer", what);
    const auto rows = [&](const void* at, int64_t stride, int64_t heads) { return QmmRows{at, tokens, stride * (int64_t)sizeof(T), heads * d * (int64_t)sizeof(T)}; };
    const QmmRows qi = rows(q, q_stride, q_heads), ki = rows(k, k_stride, k_heads), qo = rows(q_out, q_out_stride, q_heads), ko = rows(k_out, k_out_stride, k_heads);
    const auto same = [](const QmmRows& a, const QmmRows& b) { return a.at == b.at && a.stride == b.stride; };
    if ((!same(qi, qo) && !qmm_rows_apart(qi, qo)) || (!same(ki, ko) && !qmm_rows_apart(ki, ko)) || !qmm_rows_apart(qi, ko) || !qmm_rows_apart(ki, qo) || !qmm_rows_apart(qo, ko))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: an output shares memory with another tensor (it may be its own input)", what);
    for (const QmmRows& to : {qo, ko}) // (one row of the output's stride: between two of its rows there may be room)
        if (!qmm_rows_apart(to, {positions, 1, to.stride, tokens * 4}) || !qmm_rows_apart(to, {frequencies, 1, to.stride, rotary / 2 * 8}) ||
            !qmm_rows_apart(to, {weight, weight ? 1 : 0, to.stride, 2 * d * (int64_t)sizeof(T)}))
            return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: an output shares memory with positions, frequencies or weights", what);
    int device = 0, n_cus = 0;
    if (int rc = qmm_current_device(&device, &n_cus)) return rc;
    RopeParams P{q, k, q_out, k_out, q_stride, k_stride, q_out_stride, k_out_stride, positions, frequencies, weight, factor, eps, tokens, (int)q_heads,
                 (int)(q_heads + k_heads), (int)d, (int)rotary};
    hipStream_t stream = (hipStream_t)stream_;
    constexpr int V = 16 / (int)sizeof(T);
    const auto aligned = [](const void* p, int64_t a, int64_t b) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && a % V == 0 && b % V == 0; };
    const int per_head = (int)(d / (2 * V));
    if (d % (2 * V) == 0 && rotary % (2 * V) == 0 && per_head <= 64 && rotary <= 2 * kPiecePairs && (!q_heads || (aligned(q, q_stride, 0) && aligned(q_out, q_out_stride, 0))) &&
        (!k_heads || (aligned(k, k_stride, 0) && aligned(k_out, k_out_stride, 0))) && aligned(weight, 0, 0)) {
        int lp = 1;
        while (lp < per_head) lp *= 2;
        // a token's heads go to as many waves as make 16 for every compute unit
        const int sets = (P.heads + 64 / lp - 1) / (64 / lp);
        const int passes = (int)std::max<int64_t>(1, std::min<int64_t>(sets, tokens * sets / (16 * n_cus)));
        const int shares = (sets + passes - 1) / passes;
        const auto run = [&](auto kernel) { kernel<<<(unsigned)((tokens * shares + 3) / 4), 256, 0, stream>>>(P, lp, per_head, passes, shares); };
        if (weight) interleaved ? run(rope_pieces_kernel<T, true, true>) : run(rope_pieces_kernel<T, false, true>);
        else interleaved ? run(rope_pieces_kernel<T, true, false>) : run(rope_pieces_kernel<T, false, false>);
    } else {
        const unsigned grid = (unsigned)std::min<int64_t>(tokens, 1 << 20);
        interleaved ? rope_any_kernel<T, true><<<grid, 256, 0, stream>>>(P) : rope_any_kernel<T, false><<<grid, 256, 0, stream>>>(P);
    }
    ROPE_TRY(hipGetLastError());
    return IZWI_QMM_OK;
}

} // namespace

extern "C" {

#define ROPE_POSITIONS(NAME, C, T)                                                                                                                         \
    int NAME(const C* q, int64_t q_stride, const C* k, int64_t k_stride, const int32_t* positions, const double* frequencies, double attention_factor,    \
             int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t head_dim, int64_t rotary_dim, int interleaved, const C* qk_weight, float eps,       \
             C* q_out, int64_t q_out_stride, C* k_out, int64_t k_out_stride, void* stream) {                                                               \
        return qmm_guarded(#NAME, [&]() -> int {                                                                                                           \
            return rope_positions_impl<T>((const T*)q, q_stride, (const T*)k, k_stride, positions, frequencies, attention_factor, tokens, q_heads,         \
                                          k_heads, head_dim, rotary_dim, interleaved, (const T*)qk_weight, eps, (T*)q_out, q_out_stride, (T*)k_out,        \
                                          k_out_stride, stream);                                                                                           \
        });                                                                                                                                                \
    }
ROPE_POSITIONS(izwi_rope_positions_f32, float, float)
ROPE_POSITIONS(izwi_rope_positions_f16, uint16_t, f16_t)
ROPE_POSITIONS(izwi_rope_positions_bf16, uint16_t, bf16_t)

int izwi_rope_frequencies(int scaling, int64_t rotary_dim, double base, double factor, double original_len, double low, double high, double* frequencies,
                          double* attention_factor) {
    return qmm_guarded("izwi_rope_frequencies", [&]() -> int {
    constexpr const char* what = "rope_frequencies";
    if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > 2 * kMostPairs) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: rotary_dim %lld", what, (long long)rotary_dim);
    if (scaling < IZWI_ROPE_PLAIN || scaling > IZWI_ROPE_YARN) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: scaling %d", what, scaling);
    if (!(base > 1.0) || !std::isfinite(base)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: base %g", what, base);
    if (scaling != IZWI_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: factor %g", what, factor);
    const bool by_waves = scaling == IZWI_ROPE_LLAMA3 || scaling == IZWI_ROPE_YARN;
    if (by_waves && (!(original_len > 0.0) || !std::isfinite(original_len) || !(low > 0.0) || !(high > low) || !std::isfinite(high)))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: original length %g, turns %g to %g", what, original_len, low, high);
    if (scaling == IZWI_ROPE_NTK && rotary_dim == 2) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: a base of one pair cannot be stretched", what);
    if (!frequencies || !attention_factor) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: NULL buffer", what);
    const double n = (double)rotary_dim, two_pi = 6.283185307179586477;
    if (scaling == IZWI_ROPE_NTK) base *= std::pow(factor, n / (n - 2.0));
    // YaRN's ramp runs over the pairs, between those that turn `high` and `low` times in the original length
    const auto pair_of = [&](double turns) { return n * std::log(original_len / (turns * two_pi)) / (2.0 * std::log(base)); };
    double from = 0.0, to = 0.0;
    if (scaling == IZWI_ROPE_YARN) {
        from = std::max(std::floor(pair_of(high)), 0.0), to = std::min(std::ceil(pair_of(low)), n - 1.0);
        if (to <= from) to = from + 0.001;
    }
    for (int64_t i = 0; i < rotary_dim / 2; i++) {
        const double f = std::pow(base, -2.0 * (double)i / n);
        double stretched = 0.0; // the share of the stretched frequency
        if (scaling == IZWI_ROPE_LINEAR) stretched = 1.0;
        else if (scaling == IZWI_ROPE_LLAMA3) stretched = 1.0 - std::min(std::max((original_len * f / two_pi - low) / (high - low), 0.0), 1.0);
        else if (scaling == IZWI_ROPE_YARN) stretched = std::min(std::max(((double)i - from) / (to - from), 0.0), 1.0);
        frequencies[i] = stretched == 0.0 ? f : f * (1.0 - stretched) + f / factor * stretched;
    }
    *attention_factor = scaling == IZWI_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
    return IZWI_QMM_OK;
    });
}

} // extern "C"
