// Reductions over lanes on the vector ALU and the pieces of a running softmax, shared by the decode-step kernels
// (decode_ops.hip, kv_cache.hip, kv_attention.hip, beam_select.hip); unnamed namespace, one copy per including file.
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
