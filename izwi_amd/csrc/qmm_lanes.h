// Reductions over lanes on the vector ALU and the pieces of a running softmax, shared by the decode-step kernels
// (decode_ops.hip, kv_cache.hip, kv_attention.hip, beam_select.hip, prompt_attention.hip, rope_positions.hip,
// moe_route_scored.hip); unnamed namespace, one copy per including file.
#ifndef IZWI_QMM_LANES_H
#define IZWI_QMM_LANES_H

#include <hip/hip_runtime.h>

#include <type_traits>
#include <utility>

#include "qmm_internal.h"

namespace {

// Sum over the wave, in every lane: halves, rows of 16, then the lanes 8, 4, 2 and 1 away, on the vector ALU (six
// shuffles through LDS were a third of a microsecond of a one-token kernel)
template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = qmm_add_lane16(qmm_add_lane32(v));
    v += dpp_f<0x128>(v); // row_ror:8
    v += dpp_f<0x124>(v); // row_ror:4 (lanes 8 apart are equal by now)
    v += dpp_f<0x4E>(v);  // quad_perm [2,3,0,1]
    v += dpp_f<0xB1>(v);  // quad_perm [1,0,3,2]
    return v;
}

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)u, (int)u, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(u >> 32), (int)(u >> 32), CTRL, 0xf, 0xf, false);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// e^d for d <= 0 (or -infinity: 0) in f64 to 7e-16 of itself, e^0 = 1: 2^n 2^f with n + f = d log2(e), |f| <= 1/2, and 2^f as 1 + f times the
// polynomial of degree 9 that meets (2^f - 1) / f at its Chebyshev nodes (worked out with 60 digits).  (Three degrees less leave 4e-11, e^0
// among it: a beam with one token left had a log-probability of 8e-11 instead of 0, and beams that close changed places.  They are 1.8 us of
// 36.7 for 16 prompts of 8 beams over 151936 tokens.)
__device__ __forceinline__ double exp_of(double d) {
    // (1.5 * 2^52 leaves no place behind the point: the low word of the sum is n)
    const double y = __builtin_fmax(d * 1.4426950408889634, -1100.0), t = y + 0x1.8p52, f = y - (t - 0x1.8p52);
    double p = 0x1.e5e9f548e5725p-28;
    p = __builtin_fma(p, f, 0x1.b6571de2f2351p-24);
    p = __builtin_fma(p, f, 0x1.62bfe46117445p-20);
    p = __builtin_fma(p, f, 0x1.ffcb76789860fp-17);
    p = __builtin_fma(p, f, 0x1.4309130378460p-13);
    p = __builtin_fma(p, f, 0x1.5d87fe908f88ap-10);
    p = __builtin_fma(p, f, 0x1.3b2ab6fba385fp-7);
    p = __builtin_fma(p, f, 0x1.c6b08d7044119p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff82c590p-3);
    p = __builtin_fma(p, f, 0x1.62e42fefa39f7p-1);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)__double_as_longlong(t));
}

// e^x for x <= 0 on the hardware's exp2 (relative error about 2^-22; e^-inf = 0)
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// weight of a partial result with running maximum m when merged under the maximum mn
__device__ __forceinline__ float merge_weight(float m, float mn) { return m == -INFINITY ? 0.0f : exp_neg(m - mn); }

// sum over the 8 lanes of a row group, in every lane of the group (two quad permutes and a
// mirror of the half row: no LDS traffic)
__device__ __forceinline__ float sum8(float v) {
    v += dpp_f<0xB1>(v);  // quad_perm [1,0,3,2]
    v += dpp_f<0x4E>(v);  // quad_perm [2,3,0,1]
    v += dpp_f<0x141>(v); // row_half_mirror
    return v;
}

// Lane N of every sixteen, in all of them
template <int N>
__device__ __forceinline__ uint32_t of_lane(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x150 + N, 0xf, 0xf, true); // row_newbcast
}

// f(0), .., f(N - 1), as constants
template <class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

} // namespace

#endif // IZWI_QMM_LANES_H
