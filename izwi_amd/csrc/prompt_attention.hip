// Attention over whole prompts: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the positions j that query i sees, for packed
// sequences of different lengths, causal or not, with grouped heads.
//
// One pass over the keys with a running reference and sum.  A workgroup has kRows rows of one kv head, a row being a (token, query
// head) pair, the heads of a group next to each other: the group shares every tile of keys and values, and a tile of rows spans few
// tokens, so that little of a causal triangle is worked out in vain.  A wave has 32 of the rows as the columns of both products on
// the matrix cores:
//   S^T = K Q^T   keys from LDS as the left operand, queries in registers; a lane has one row's scores of 16 of 32 positions,
//   O^T = V^T P^T what the first product leaves in a lane is what the second one takes, so weights never leave the registers; values come
//                 from LDS through the transposing reads.
// Reference and sum of a row are two numbers of a lane, and rescaling O^T is a multiplication by a lane's own number.
//
// f32: queries, keys, values and weights go as three bf16 numbers each, which hold all 24 bits (down to 2^-100: the third has no bits
// below 2^-133), and the six products of weight 2^-16 and more are summed in f32; what is left out is at most 2^-22 of a product, of either sign.
//
// f16 and bf16: weights go as two numbers of the type (Elem), so that values take two products where queries and keys take one.
//
// Bound by the matrix cores and the power that they may draw in long prompts: 8192 tokens of 32 bf16 heads of 128 on 8, causal, 719 us, 765 TFLOP/s (1150 with
// the weights' second product; a library product of 8192^3 1372, both operands along k 1622): they are at work 65 % of the cycles, at a clock of 1.8 GHz; exponentials
// and rounding of one wave overlap the products of the other on its SIMD only in part.  By the same, and the beginnings and ends of workgroups, in shorter
// ones: nine of 775 to 1501 tokens 186 us, 551 TFLOP/s; four clips of 867 to 1500 f16, heads of 64, not causal, 53 us, 450 TFLOP/s (an exponential
// takes as long there as a quarter of the products of its score).  By memory where few rows meet many keys: 17 tokens behind 30011 33 us, 3.7
// TB/s, and 5 to join them.  By launch and latency below that: 37 f32 tokens 11.5 us, bf16 6.0.  f32: six products for queries and keys, and for weights and values,
// 3500 tokens of 16 heads on 8 332 us, 151 TFLOP/s; 2048 138, 125; 1100 67, 74; 300 25, 15, in parts and with a launch to join them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "../../include/izwi_decode_ops.h"
#include "qmm_internal.h"
#include "qmm_lanes.h"
#include "qmm_tile.h"

namespace {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

struct PromptParams {
    const void *q, *k, *v;
    void* out;
    int64_t q_stride, k_stride, v_stride, out_stride; // elements from a token to the next
    const int32_t *cu_q, *cu_k;                       // NULL: one sequence
    int64_t total_q, total_k;
    int batch, heads, kv_heads, group, causal;
    int tiles, splits; // workgroups: tiles of rows x splits of the positions x kv heads
    int by_length;     // workgroups begin in the order of the positions that they see
    float sign;        // of the scale, or 0: what queries are multiplied by
    float scale, scale_rest; // |scale| log2(e) as two f32 numbers
    float* sums;       // [row][split][D], rows as in out (splits > 1)
    float2* stats;     // [row][split]: reference (base 2) and sum
};

// ---- the element types ---------------------------------------------------------------------------------------------
// N: bf16 / f16 numbers that a query, key or value goes as; NW: those that a weight goes as; kLift: weights stand 2^kLift higher than they are
// (an f16 has its full 11 bits from 2^-14 on: under a lift of 2^7, from 2^-21 of the row's reference on).  f16 and bf16 weights go as two
// numbers, rounded and what that left: one alone is off by 2^-12, 2^-9 of the weight, which the sum of the weights does not share, so that
// results were as far off by it as by their own rounding (against 64 bits bf16 2.1e-3 of the result where the rounding alone leaves 1.6e-3,
// f16 2.7e-4, 2.1e-4), and the mean of equal values was another value.
template <typename T>
struct Elem;
template <>
struct Elem<bf16_t> {
    static constexpr int N = 1, NW = 2, kLift = 0;
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
    static __device__ __forceinline__ uint32_t rest(float a, float b, uint32_t of) { // what pack left of them (to 2^-18)
        return pack_bf16(a - __uint_as_float(of << 16), b - __uint_as_float(of & 0xffff0000u));
    }
    static constexpr uint32_t kExponent = 0x7f807f80u;
};
template <>
struct Elem<f16_t> {
    static constexpr int N = 1, NW = 2, kLift = 7;
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b}); }
    static __device__ __forceinline__ uint32_t rest(float a, float b, uint32_t of) { // (an fma by 1 takes the f16 as it is, without a conversion)
        const f16x2 h = __builtin_bit_cast(f16x2, of);
        return pack(__builtin_fmaf((float)h[0], -1.0f, a), __builtin_fmaf((float)h[1], -1.0f, b));
    }
    static constexpr uint32_t kExponent = 0x7c007c00u;
};
template <>
struct Elem<float> {
    static constexpr int N = 3, NW = 3, kLift = 0;
    static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) { return Elem<bf16_t>::mma(a, b, c); }
    static constexpr uint32_t kExponent = 0x7f807f80u;
};

// Two f32 numbers as three bf16 numbers each, without a loss: the top 8 bits, what is left rounded to 8, the rest, which has either sign then (cut
// off, too, the second number left rests of the value's own sign, and what the six products leave out was up to 2^-21 of each and always of
// its sign).  (An infinity leaves NaN.)
__device__ __forceinline__ void split3(float a, float b, uint32_t (&to)[3]) {
    constexpr uint32_t kTop = 0x07060302u; // the upper halves of two dwords
    const uint32_t a0 = __float_as_uint(a), b0 = __float_as_uint(b);
    const float a1 = a - __uint_as_float(a0 & 0xffff0000u), b1 = b - __uint_as_float(b0 & 0xffff0000u);
    to[0] = __builtin_amdgcn_perm(b0, a0, kTop);
    to[1] = pack_bf16(a1, b1);
    const float a2 = a1 - __uint_as_float(to[1] << 16), b2 = b1 - __uint_as_float(to[1] & 0xffff0000u);
    to[2] = __builtin_amdgcn_perm(__float_as_uint(b2), __float_as_uint(a2), kTop);
}

__device__ __forceinline__ void split8(const float (&v)[8], u32x4 (&to)[3]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t three[3];
        split3(v[2 * i], v[2 * i + 1], three);
#pragma unroll
        for (int n = 0; n < 3; n++) to[n][i] = three[n];
    }
}

// Of NL numbers by NR the products whose weight is 2^-16 or more, the small ones first: product i is that of number left(i) of one and right(i) of
// the other.  Products go round between results, so that none adds to what the one before it wrote.
template <int NL, int NR = NL>
struct Products {
    static constexpr int kCount = NL == 1 ? NR : 6;
    static constexpr int left(int i) { return NL == 1 ? 0 : (i < 3 ? 2 - i : i < 5 ? 4 - i : 0); }
    static constexpr int right(int i) { return NL == 1 ? NR - 1 - i : (i < 3 ? i : i < 5 ? i - 3 : 0); }
};

// ---- a tile of keys or values in LDS -------------------------------------------------------------------------------
// Rows of D 16-bit numbers in pieces of 16 bytes, piece c of row r at place c ^ turn(r): so that 32 rows' pieces c (keys), and 64
// bytes of eight neighbouring rows (values), lie on different banks.
template <int D>
__device__ __forceinline__ int turn(int row) {
    return D == 64 ? ((row >> 1 & 1) << 2 | (row >> 2 & 3)) : ((row & 3) << 2 | (row >> 2 & 3));
}

// The sequence that a tile of rows belongs to.  Sequence b has the tiles from (its first row among all) / rows + b on, as many as it needs or
// one more, so that its place is found by its offset alone: 64 at a time, by the lanes.
struct Sequence {
    int64_t q0, k0; // its first tokens
    int len_q, len_k, row0; // row0: the tile's first row within it
};
__device__ __forceinline__ int bounded(const int32_t* cu, int i, int64_t total) { return (int)min((int64_t)max(cu[i], 0), total); }
__device__ __forceinline__ bool find_sequence(const PromptParams& P, int rows, int tile, int lane, Sequence& s) {
    if (!P.cu_q) {
        s = Sequence{0, 0, (int)P.total_q, (int)P.total_k, tile * rows};
        return (int64_t)tile * rows < P.total_q * P.group;
    }
    int from = 0, n = P.batch; // it is among from .. from + n - 1
    for (;;) {
        const int step = (n + 63) / 64, b = min(from + lane * step, P.batch - 1);
        const int q0 = bounded(P.cu_q, b, P.total_q), slot = q0 * P.group / rows + b; // (below 2^31: checked on the host)
        if (step > 1) {
            const int found = __popcll(__ballot(lane * step < n && slot <= tile));
            if (found == 0) return false;
            from += (found - 1) * step, n = min(step, n - (found - 1) * step);
            continue;
        }
        const int q1 = bounded(P.cu_q, b + 1, P.total_q), k0 = bounded(P.cu_k, b, P.total_k), k1 = bounded(P.cu_k, b + 1, P.total_k);
        const int found = __popcll(__ballot(lane < n && slot <= tile));
        if (found == 0) return false;
        const int l = found - 1;
        s.q0 = __builtin_amdgcn_readlane(q0, l), s.k0 = __builtin_amdgcn_readlane(k0, l);
        s.len_q = max(__builtin_amdgcn_readlane(q1, l) - (int)s.q0, 0), s.len_k = max(__builtin_amdgcn_readlane(k1, l) - (int)s.k0, 0);
        const int64_t row0 = (int64_t)(tile - __builtin_amdgcn_readlane(slot, l)) * rows;
        s.row0 = (int)min(row0, (int64_t)0x7fffffff);
        return row0 >= 0 && row0 < (int64_t)s.len_q * P.group; // (below 0 where offsets fall)
    }
}

// The same for at most 64 sequences, in the order of the positions that a tile sees, the most first: in that of the offsets the last ones begun
// may be long ones of a long sequence.  A tile's level is that number in whole tiles (causal; else the sequence's); `above` counts the
// tiles of higher levels, and unit u lies in the level where the count passes it.
__device__ __forceinline__ bool find_by_length(const PromptParams& P, int rows, int u, int lane, Sequence& s) {
    const int b = min(lane, P.batch - 1);
    const int q0 = bounded(P.cu_q, b, P.total_q), q1 = bounded(P.cu_q, b + 1, P.total_q), k0 = bounded(P.cu_k, b, P.total_k), k1 = bounded(P.cu_k, b + 1, P.total_k);
    const int len_q = max(q1 - q0, 0), len_k = max(k1 - k0, 0), n = lane < P.batch ? (len_q * P.group + rows - 1) / rows : 0;
    const int top = len_k / max(rows / P.group, 1); // the last tile's level; the one `e` before it is `e` lower (causal)
    const auto sum = [](int v) { return __builtin_amdgcn_readfirstlane((int)wave_sum((float)v)); }; // (exact: below 2^24)
    const auto above = [&](int level) { return sum(P.causal ? min(max(top - level, 0), n) : top > level ? n : 0); };
    if (u >= sum(n)) return false;
    int least = P.causal ? top - n : top - 1, most = top; // above(least) is all of a sequence's, above(most) none
    for (int i = 1; i < 64; i <<= 1) least = min(least, __shfl_xor(least, i)), most = max(most, __shfl_xor(most, i));
    least = __builtin_amdgcn_readfirstlane(least), most = __builtin_amdgcn_readfirstlane(most);
    while (most - least > 1) {
        const int middle = least + (most - least) / 2;
        if (above(middle) > u) least = middle;
        else most = middle;
    }
    // above(most) <= u < above(least)
    int at = u - above(most);
    const int here = P.causal ? (top - most >= 0 && top - most < n ? 1 : 0) : top == most ? n : 0;
    uint64_t left = __ballot(here > 0);
    int l = 0;
    for (;; left &= left - 1) { // (at is below the sum of `here`)
        l = __ffsll((unsigned long long)left) - 1;
        const int of = __builtin_amdgcn_readlane(here, l);
        if (at < of) break;
        at -= of;
    }
    const int tile = P.causal ? __builtin_amdgcn_readlane(n, l) - 1 - (__builtin_amdgcn_readlane(top, l) - most) : __builtin_amdgcn_readlane(n, l) - 1 - at;
    s.q0 = __builtin_amdgcn_readlane(q0, l), s.k0 = __builtin_amdgcn_readlane(k0, l);
    s.len_q = __builtin_amdgcn_readlane(len_q, l), s.len_k = __builtin_amdgcn_readlane(len_k, l);
    s.row0 = tile * rows;
    return true;
}

// v of the lane 32 away, the larger of both
__device__ __forceinline__ float max_lane32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 2^d, d <= 0, for what is summed already: 0 below 2^-126, as a weight is (bounded by that, it left 10^37 under a weight of zero a share of 0.1)
__device__ __forceinline__ float rescale(float d) { return __builtin_amdgcn_exp2f(d); }
// v times such a factor; of an infinity, which no factor changes, itself
template <typename V>
__device__ __forceinline__ V rescaled(V v, float by) {
    V r = v * by;
    if (by == 0.0f)
#pragma unroll
        for (int i = 0; i < (int)(sizeof(V) / 4); i++) r[i] = __builtin_isinf(v[i]) ? v[i] : r[i];
    return r;
}

constexpr float kSlack = 8.0f; // a reference stands until a score passes it by this (base 2): weights stay below 2^8

// WR sets of waves have 32 rows each, WZ sets KT positions each of a tile, DZ sets a part each of the head's elements: of heads of 256 one wave would hold
// twice the registers; two add up their scores through LDS and weigh their own halves of the values.
template <typename T, int D, int WR, int WZ, int DZ, int KT, bool SPLIT>
__global__ __launch_bounds__(64 * WR * WZ * DZ, Elem<T>::N == 1 || D == 64 ? 2 : 1) void prompt_attention_kernel(PromptParams P) {
    using E = Elem<T>;
    constexpr int N = E::N, NW = E::NW, W = WR * WZ * DZ, kRows = 32 * WR, KS = KT * WZ, DW = D / DZ, KK = DW / 16, PT = KT / 32, DT = DW / 32;
    constexpr bool kDirect = N == 1;          // keys and values go straight from memory into LDS
    constexpr int kPlane = KS * D * 2;        // bytes of a tile of 16-bit numbers
    constexpr int kTile = 2 * N * kPlane;     // keys, then values
    constexpr bool kDouble = !kDirect && DZ == 1 && WZ == 1; // a second tile is taken apart beside the first one's products
    constexpr int kTiles = kTile * (kDirect || kDouble ? 2 : 1), kScores = DZ > 1 ? 2 * W * PT * 16 * 256 : 0;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[]; // tiles (two where direct), partial scores of two tiles, a word
    uint32_t* odd_values = reinterpret_cast<uint32_t*>(smem + kTiles + kScores);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = lane & 31, h = lane >> 5, wr = wave % WR, dz = wave / WR % DZ, wz = wave / (WR * DZ);
    // the kv head runs fastest: workgroups of a kv head stay on one XCD, whose L2 then holds its keys and values; the last tiles of a
    // sequence, which see the most positions, begin first
    const int kv = blockIdx.x % P.kv_heads;
    const int unit = blockIdx.x / P.kv_heads, split = SPLIT ? unit % P.splits : 0;
    Sequence s;
    if (!SPLIT && P.by_length ? !find_by_length(P, kRows, unit, lane, s) : !find_sequence(P, kRows, P.tiles - 1 - (SPLIT ? unit / P.splits : unit), lane, s))
        return; // the whole workgroup

    const int rows = s.len_q * P.group; // of the sequence and kv head (fits: checked on the host)
    const int row = min(s.row0 + wr * 32 + x, rows - 1), token = row / P.group, head = kv * P.group + row % P.group;
    const int past = s.len_k - s.len_q;
    // positions up to `limit` count; of the workgroup's rows the first sees the fewest, the last the most
    const int limit = P.causal ? token + past : s.len_k - 1;
    const int last_token = min(s.row0 + kRows - 1, rows - 1) / P.group;
    const int fewest = P.causal ? max(s.row0 / P.group + past + 1, 0) : s.len_k;
    const int most = P.causal ? min(max(last_token + past + 1, 0), s.len_k) : s.len_k;
    const int n_tiles = (most + KS - 1) / KS;
    const int share = SPLIT ? (n_tiles + P.splits - 1) / P.splits : n_tiles;
    const int first = SPLIT ? min(split * share, n_tiles) : 0, end = min(first + share, n_tiles);

    const uint8_t* const k_rows = reinterpret_cast<const uint8_t*>(static_cast<const T*>(P.k) + s.k0 * P.k_stride + (int64_t)kv * D);
    const uint8_t* const v_rows = reinterpret_cast<const uint8_t*>(static_cast<const T*>(P.v) + s.k0 * P.v_stride + (int64_t)kv * D);
    const int64_t k_step = P.k_stride * (int)sizeof(T), v_step = P.v_stride * (int)sizeof(T);

    // A tile on its way into LDS.  Positions behind the last repeat it (they are masked).
    constexpr int kPer = KS * D / 8 / (64 * W); // pieces of 8 values that a thread has of the keys, and of the values
    static_assert(kPer * 8 * 64 * W == KS * D);
    [[maybe_unused]] f32x4 ahead[kDirect ? 1 : 2][kDirect ? 1 : kPer][2];
    const auto request = [&](int tile, int stage) {
        const int most_row = min(KS, s.len_k - tile * KS) - 1;
        const uint8_t* const kb = k_rows + (int64_t)tile * KS * k_step;
        const uint8_t* const vb = v_rows + (int64_t)tile * KS * v_step;
        if constexpr (kDirect) {
            const uint32_t base = (uint32_t)(uintptr_t)smem + stage * kTile;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const int piece = (i * W + wave) * 64 + lane, r = piece / (D / 8), c = (piece % (D / 8)) ^ turn<D>(r);
                const uint32_t at = min(r, most_row);
                load_to_lds(kb, at * (uint32_t)k_step + 16 * c, base + (i * W + wave) * 1024);
                load_to_lds(vb, at * (uint32_t)v_step + 16 * c, base + kPlane + (i * W + wave) * 1024);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const int piece = i * (64 * W) + threadIdx.x, r = min(piece / (D / 8), most_row), c = piece % (D / 8);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    ahead[0][i][j] = *reinterpret_cast<const f32x4*>(kb + r * k_step + 32 * c + 16 * j);
                    ahead[1][i][j] = *reinterpret_cast<const f32x4*>(vb + r * v_step + 32 * c + 16 * j);
                }
            }
        }
    };
    const auto deliver = [&](uint8_t* to, int w, int i) { // piece i of the keys (w = 0) or values requested into registers, as three planes
        if constexpr (!kDirect) {
            const int piece = i * (64 * W) + threadIdx.x, r = piece / (D / 8), c = (piece % (D / 8)) ^ turn<D>(r);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = ahead[w][i][j >> 2][j & 3];
            u32x4 o[3];
            split8(v, o);
#pragma unroll
            for (int n = 0; n < 3; n++) *reinterpret_cast<u32x4*>(to + (w * 3 + n) * kPlane + r * (2 * D) + 16 * c) = o[n];
        }
    };
    const auto deliver_all = [&](uint8_t* to) {
#pragma unroll
        for (int i = 0; i < 2 * kPer; i++) deliver(to, i / kPer, i % kPer);
    };

    if (first < end) request(first, 0); // (ahead of the queries: both ways to memory at once)

    // queries: lane (x, h) has of row x the elements 16 kk + 8 h .. + 7 of the wave's part of the head
    u32x4 q[KK][N];
    {
        const T* from = static_cast<const T*>(P.q) + (s.q0 + token) * P.q_stride + (int64_t)head * D + dz * DW + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if constexpr (N == 1) {
                typedef T vec __attribute__((ext_vector_type(8)));
                const vec v = *reinterpret_cast<const vec*>(from + 16 * kk);
                vec r;
#pragma unroll
                for (int i = 0; i < 8; i++) r[i] = (T)((float)v[i] * P.sign); // exact
                q[kk][0] = __builtin_bit_cast(u32x4, r);
            } else {
                float v[8];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(from + 16 * kk + 4 * i) * P.sign;
#pragma unroll
                    for (int j = 0; j < 4; j++) v[4 * i + j] = a[j];
                }
                split8(v, q[kk]);
            }
        }
    }

    // where a lane reads: keys of position x, piece 2 kk + h; values of positions 4 h + 0..3 (+ 8) through the transposing read, for
    // which the lanes of a sixteen name four rows of four pieces of 8 bytes
    const int k_at = (wz * KT + x) * (2 * D) + dz * (2 * DW) + ((h ^ turn<D>(x)) << 4);
    const int i16 = lane & 15, v_row = 4 * h + (i16 >> 2), v_piece = (lane >> 4 & 1) * 2 + (i16 >> 1 & 1);
    const int v_at0 = (wz * KT + v_row) * (2 * D) + dz * (2 * DW) + ((v_piece ^ turn<D>(v_row)) << 4) + (i16 & 1) * 8;
    const int v_at1 = (wz * KT + v_row + 8) * (2 * D) + dz * (2 * DW) + ((v_piece ^ turn<D>(v_row + 8)) << 4) + (i16 & 1) * 8;

    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    float ref = -INFINITY, sum[2] = {}; // ref: base 2; sum: of this lane's positions, in two parts
    constexpr bool kWide = E::kLift == 0; // values may be as large as f32 is
    constexpr float kShrink = kWide ? 0x1p-32f : 1.0f;
    [[maybe_unused]] float shrink = 1.0f; // of all weights, in the second pass (below)
    if (threadIdx.x == 0) *odd_values = 0;

    // Scores, weights and the weighted values of a tile that has landed.  MASKED: some row of the workgroup does not see all of its
    // positions.
    [[maybe_unused]] int turns = 0;
    // `there`: where the tile behind it, which waits in registers, goes meanwhile; `behind`: the one to be requested then (MORE)
    const auto weigh = [&](auto masked, auto more, const uint8_t* here, int p0, uint8_t* there = nullptr, int behind = 0) {
        constexpr bool MASKED = decltype(masked)::value, MORE = decltype(more)::value;
        // lane (x, h), register r of sub-tile pt: row x, position p0 + 32 pt + 8 (r / 4) + 4 h + r % 4
        f32x16 p[PT];
#pragma unroll
        for (int pt = 0; pt < PT; pt++) {
            f32x16 part[N > 1 ? 2 : 1];
#pragma unroll
            for (int i = 0; i < (N > 1 ? 2 : 1); i++)
#pragma unroll
                for (int r = 0; r < 16; r++) part[i][r] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                u32x4 a[N];
#pragma unroll
                for (int n = 0; n < N; n++) a[n] = *reinterpret_cast<const u32x4*>(here + n * kPlane + pt * 32 * (2 * D) + (k_at ^ (kk << 5)));
#pragma unroll
                for (int i = 0; i < Products<N>::kCount; i++)
                    part[N > 1 ? i & 1 : 0] = E::mma(a[Products<N>::left(i)], q[kk][Products<N>::right(i)], part[N > 1 ? i & 1 : 0]);
                if constexpr (MORE) { // (vector instructions beside the products)
                    static_assert(PT == 1 && KK % (2 * kPer) == 0);
                    constexpr int kEvery = KK / (2 * kPer);
                    if (kk % kEvery == kEvery - 1) deliver(there, kk / kEvery / kPer, kk / kEvery % kPer);
                }
            }
            p[pt] = part[0];
            if constexpr (N > 1) p[pt] += part[1];
        }
        if constexpr (MORE) {
#pragma unroll
            for (int i = 0; i < Products<N>::kCount * KK; i++) { // (four behind each product: 244 us without, 235 with it, 2048 tokens of 32 heads on 8)
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            }
            if (behind < end) request(behind, 0);
        }
        if constexpr (N == 1) { // eight operands on their way ahead of the first product (two: D = 256 2600 tokens 138 us instead of 134, 37 of D = 128 6.3, 6.0)
            constexpr int kReads = PT * KK, kAhead = kReads < 8 ? kReads : 8;
            __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
            for (int i = 0; i < kReads; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (i + kAhead < kReads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
        if constexpr (DZ > 1) { // (two places in turn: a wave may still read the last tile's)
            static_assert(DZ == 2);
            f32x4* const scores = reinterpret_cast<f32x4*>(smem + kTiles) + turns * (W * PT * 4 * 64) + lane;
            turns ^= 1;
#pragma unroll
            for (int pt = 0; pt < PT; pt++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    scores[((wave * PT + pt) * 4 + i) * 64] = f32x4{p[pt][4 * i], p[pt][4 * i + 1], p[pt][4 * i + 2], p[pt][4 * i + 3]};
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const int other = wave + (dz ? -WR : WR);
#pragma unroll
            for (int pt = 0; pt < PT; pt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const f32x4 v = scores[((other * PT + pt) * 4 + i) * 64];
#pragma unroll
                    for (int j = 0; j < 4; j++) p[pt][4 * i + j] += v[j]; // (the same sum in both)
                }
        }
        if constexpr (MASKED) {
#pragma unroll
            for (int pt = 0; pt < PT; pt++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (p0 + 32 * pt + 8 * (r >> 2) + 4 * h + (r & 3) > limit) p[pt][r] = -INFINITY;
        }
        float top = p[0][0];
#pragma unroll
        for (int pt = 0; pt < PT; pt++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, p[pt][r]);
        top = max_lane32(top) * P.scale;
        const bool passed = top > ref + kSlack; // (from -infinity: at the first score)
        if (__any(passed)) {                    // a row's own reference moves only by its own scores: no other row has a say in its result
            const float next = passed ? top : ref, by = ref == -INFINITY ? 1.0f : rescale(ref - next); // (zeros so far, and what is no number)
            sum[0] *= by, sum[1] *= by;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= by;
            ref = next;
        }
        const float from = ref == -INFINITY ? 0.0f : ref - E::kLift;
#pragma unroll
        for (int pt = 0; pt < PT; pt++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float e = __builtin_fmaf(p[pt][r], P.scale, -from);
                if constexpr (N == 3) e = p[pt][r] == -INFINITY ? e : __builtin_fmaf(p[pt][r], P.scale_rest, e); // (the rest may be negative)
                p[pt][r] = __builtin_amdgcn_exp2f(e);
                if constexpr (MASKED && kWide) p[pt][r] *= shrink;
                sum[r & 1] += p[pt][r];
            }

        // sixteen positions at a time: the lane's eight are 4 h + 0..3 and 8 + 4 h + 0..3 of them
#pragma unroll
        for (int t = 0; t < KT / 16; t++) {
            u32x4 w[NW];
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = p[t >> 1][8 * (t & 1) + i];
            if constexpr (N == 1) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[0][i] = E::pack(v[2 * i], v[2 * i + 1]), w[1][i] = E::rest(v[2 * i], v[2 * i + 1], w[0][i]);
            } else {
                split8(v, w);
            }
            u32x4 a[DT][N];
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const uint8_t* const plane = here + (N + n) * kPlane + t * 16 * (2 * D);
                    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(plane + (v_at0 ^ (d << 6)))));
                    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(plane + (v_at1 ^ (d << 6)))));
                    a[d][n] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                }
#pragma unroll
            for (int i = 0; i < Products<N, NW>::kCount; i++)
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] = E::mma(a[d][Products<N, NW>::left(i)], w[Products<N, NW>::right(i)], o[d]);
        }
        if constexpr (N == 1) { // the next sixteen positions' operands beside these
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * DT, 0);
#pragma unroll
            for (int t = 0; t < KT / 16; t++)
#pragma unroll
                for (int d = 0; d < NW * DT; d++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (t + 1 < KT / 16) __builtin_amdgcn_sched_group_barrier(0x100, 2 / NW, 0);
                }
        }
    };

    const auto arrive = [&](int tile) { // the tile is in LDS, the one behind it on its way
        uint8_t* const here = smem + (kDirect || kDouble ? (tile - first & 1) * kTile : 0);
        if constexpr (kDirect) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (tile + 1 < end) request(tile + 1, tile + 1 - first & 1);
        } else if constexpr (kDouble) {
            if (tile == first) {
                deliver_all(here);
                if (tile + 1 < end) request(tile + 1, 0);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        } else {
            __syncthreads(); // the tile before is read
            deliver_all(here);
            if (tile + 1 < end) request(tile + 1, 0);
            __syncthreads();
        }
        return here;
    };
    // A value that is no number must not reach the rows that do not see it, and a weight of zero would not keep it out; nor would what is left of a
    // weight, zero or below it, leave an infinity that a row does see what it is.  Results that hold one are worked out once more, with
    // care: the tile goes on with a zero in its place, and the rows that see such a value remember it, a bit for each of the lane's elements: up
    // is an infinity, down a negative one, both NaN (f32: any).  And as finite values may have left f32 on their way, all weights are 2^-32 of what
    // they were then: exact, but for those below 2^-94 of the reference.  (A look at the values of every tile that some row does not see all of took
    // 1200 of the 11600 cycles of 37 bf16 tokens.)
    uint64_t up = 0, down = 0;
    static_assert(DT * 16 <= 64);
    for (bool care = false;;) {
        int tile = first;
        if constexpr (!kDouble) // every row sees all of these
            for (const int whole = care ? first : min(end, fewest / KS); tile < whole; tile++) weigh(std::false_type{}, std::false_type{}, arrive(tile), 0);
        for (; tile < end; tile++) {
            uint8_t* const here = arrive(tile);
            const int p0 = tile * KS;
            constexpr uint32_t kLow = E::kExponent & 0xffffu, kHigh = E::kExponent & 0xffff0000u;
            constexpr int kPieces = N * kPlane / 16 / (64 * W);
            u32x4* const values = reinterpret_cast<u32x4*>(here + N * kPlane) + threadIdx.x;
            if (care) { // is there one in this tile?  (What the word held before differs from `tile + 2`; the barrier of the next tile is behind its reads.)
                bool odd = false;
#pragma unroll 1
                for (int i = 0; i < kPieces; i++) {
                    const u32x4 v = values[i * 64 * W];
#pragma unroll
                    for (int j = 0; j < 4; j++) odd |= (v[j] & kLow) == kLow || (v[j] & kHigh) == kHigh;
                }
                if (__any(odd) && lane == 0) *odd_values = tile + 2;
                __syncthreads();
            }
            if (care && *odd_values == (uint32_t)tile + 2) {
#pragma unroll 1
                for (int j = wz * KT; j < min((wz + 1) * KT, s.len_k - p0); j++) {
                    const bool sees = p0 + j <= limit;
#pragma unroll 1
                    for (int e = 0; e < DT * 4; e++) // four of the lane's elements, 16 (e / 4) + 4 (e % 4) of o and on
#pragma unroll
                        for (int n = 0; n < N; n++) {
                            const int c = (dz * (DW / 8) + e) ^ turn<D>(j);
                            const u32x2 four = *reinterpret_cast<const u32x2*>(here + (N + n) * kPlane + j * (2 * D) + 16 * c + 8 * h);
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const uint32_t bits = four[r >> 1] >> (16 * (r & 1)) & 0xffffu;
                                const bool odd = sees && (bits & kLow) == kLow, nan = N > 1 || (bits & 0x7fffu) != kLow;
                                up |= (uint64_t)(odd && (nan || !(bits >> 15))) << (4 * e + r);
                                down |= (uint64_t)(odd && (nan || bits >> 15)) << (4 * e + r);
                            }
                        }
                }
                __syncthreads();
#pragma unroll 1
                for (int i = 0; i < kPieces; i++) {
                    u32x4 v = values[i * 64 * W];
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] &= ((v[j] & kLow) == kLow ? 0u : 0xffffu) | ((v[j] & kHigh) == kHigh ? 0u : 0xffff0000u);
                    values[i * 64 * W] = v;
                }
                __syncthreads();
            }
            if (kDouble && tile + 1 < end) weigh(std::true_type{}, std::integral_constant<bool, kDouble>{}, here, p0, smem + (tile + 1 - first & 1) * kTile, tile + 2);
            else weigh(std::true_type{}, std::false_type{}, here, p0 + wz * KT);
        }
        if (care) break;
        float zero = 0.0f; // NaN where a result is no number
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) zero = __builtin_fmaf(o[d][r], 0.0f, zero);
        if (__any(zero != 0.0f) && lane == 0) *odd_values = 1;
        __syncthreads();
        if (*odd_values == 0) break;
        care = true, shrink = kShrink;
        if (first < end) request(first, 0);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
        ref = -INFINITY, sum[0] = sum[1] = 0.0f;
    }

    sum[0] += sum[1];
    if constexpr (WZ > 1) { // the sets' results meet in LDS
        constexpr int kNumbers = DT * 16 + 6;
        static_assert(DZ == 1 && (WZ - 1) * WR * kNumbers * 256 <= kTiles);
        float* const meet = reinterpret_cast<float*>(smem) + lane;
        __syncthreads();
        if (wz > 0) {
            float* const to = meet + ((wz - 1) * WR + wr) * kNumbers * 64;
            to[0] = ref, to[64] = sum[0];
#pragma unroll
            for (int i = 0; i < 4; i++) to[(2 + i) * 64] = __uint_as_float((uint32_t)((i < 2 ? up : down) >> (32 * (i & 1))));
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) to[(6 + 16 * d + r) * 64] = o[d][r];
        }
        __syncthreads();
        if (wz > 0) return;
        float refs[WZ], all = ref;
        refs[0] = ref;
#pragma unroll
        for (int z = 1; z < WZ; z++) refs[z] = meet[((z - 1) * WR + wr) * kNumbers * 64], all = fmaxf(all, refs[z]);
#pragma unroll
        for (int z = 0; z < WZ; z++) {
            const float by = refs[z] == -INFINITY ? 1.0f : rescale(refs[z] - all);
            const float* const in = meet + ((z - 1) * WR + wr) * kNumbers * 64;
            sum[0] = z == 0 ? sum[0] * by : sum[0] + in[64] * by;
            if (z > 0)
#pragma unroll
                for (int i = 0; i < 4; i++) (i < 2 ? up : down) |= (uint64_t)__float_as_uint(in[(2 + i) * 64]) << (32 * (i & 1));
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] = z == 0 ? o[d][r] * by : o[d][r] + in[(6 + 16 * d + r) * 64] * by;
        }
        ref = all;
    }
    if (__any((up | down) != 0))
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                o[d][r] += up >> (16 * d + r) & 1 ? INFINITY : 0.0f;
                o[d][r] += down >> (16 * d + r) & 1 ? -INFINITY : 0.0f;
            }
    // rows behind the sequence's last stay as they are
    if (s.row0 + wr * 32 + x >= rows) return;
    const float total = qmm_add_lane32(sum[0]);
    const int64_t out_row = (s.q0 + token) * P.heads + head;
    if constexpr (SPLIT) {
        // (a sum below zero: the split has no position that the row sees; sums divided by it: their mean is no larger than the values are)
        if (h == 0 && dz == 0) P.stats[out_row * P.splits + split] = float2{ref, first < end && limit >= first * KS ? total / shrink : -1.0f};
        const float mean = total == 0.0f ? 1.0f : 1.0f / total;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= mean;
        float* to = P.sums + (out_row * P.splits + split) * D + dz * DW + 4 * h;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<f32x4*>(to + 32 * d + 8 * i) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        return;
    }
    const bool none = limit < 0 || s.len_k == 0;
    const float inv = none ? 0.0f : 1.0f / total;
    T* const to = static_cast<T*>(P.out) + (s.q0 + token) * P.out_stride + (int64_t)head * D + dz * DW;
#pragma unroll
    for (int d = 0; d < DT; d++) {
        float v[16];
#pragma unroll
        for (int r = 0; r < 16; r++) v[r] = none ? 0.0f : o[d][r] * inv;
        if constexpr (N == 3) {
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<f32x4*>(to + 32 * d + 8 * i + 4 * h) = f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        } else {
            // halves trade: the lower lanes get the eight values of piece 0 (2), the upper ones those of piece 1 (3)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                u32x4 piece;
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const auto r = __builtin_amdgcn_permlane32_swap(E::pack(v[4 * i + 2 * j], v[4 * i + 2 * j + 1]), E::pack(v[4 * i + 4 + 2 * j], v[4 * i + 5 + 2 * j]), false, false);
                    piece[j] = r[0], piece[2 + j] = r[1];
                }
                *reinterpret_cast<u32x4*>(to + 32 * d + 8 * (i + h)) = piece;
            }
        }
    }
}

// A row's splits joined: by a wave where there are at most eight (FEW), else by a workgroup, D / 4 threads to a split.  Every lane works out
// the weights itself from statistics that are requested together with the sums.  (One split after the other by a wave: 544 rows of 32
// splits 19.6 us.)
template <typename T, int D, bool FEW>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptParams P, int64_t rows) {
    constexpr int E = FEW ? D / 64 : 4, kPer = 64 * 4 * (FEW ? 1 : 4) / D, A = FEW ? 8 : 4; // elements a thread, splits at once, requests at once
    typedef float vec __attribute__((ext_vector_type(E)));
    const int lane = threadIdx.x & 63;
    const int64_t row = FEW ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= rows) return;
    const int64_t token = row / P.heads;
    const float2* const stats = P.stats + row * P.splits;
    const int at = FEW ? lane : threadIdx.x % (D / 4), mine = FEW ? 0 : threadIdx.x / (D / 4), step = FEW ? 1 : kPer;
    const float* const sums = P.sums + row * P.splits * D + at * E;
    if (P.cu_q) { // rows behind the last sequence, or between two, have no sums
        bool inside = false;
        for (int b0 = 0; b0 < P.batch && !inside; b0 += 64) {
            const int b = min(b0 + lane, P.batch - 1);
            inside = __any(token >= bounded(P.cu_q, b, P.total_q) && token < bounded(P.cu_q, b + 1, P.total_q));
        }
        if (!inside) return; // (the same in the whole workgroup)
    }
    // (a reference of -infinity: no score is above it, the sum is zero or no number; a sum below zero: no position that the row sees)
    vec v[A], a = 0.0f;
    float2 st[A];
    const auto take = [&](int i0) {
#pragma unroll
        for (int j = 0; j < A; j++) {
            const int i = min(i0 + j * step, P.splits - 1);
            st[j] = stats[i];
            v[j] = *reinterpret_cast<const vec*>(sums + (int64_t)i * D);
        }
    };
    take(mine);
    float ref = -INFINITY, sum = 0.0f; // of all parts
    bool any = false;
    const auto weight = [&](float2 one) { return one.y * (one.x == -INFINITY ? 1.0f : rescale(one.x - ref)); };
    if constexpr (FEW) {
#pragma unroll
        for (int j = 0; j < A; j++) ref = fmaxf(ref, st[j].y < 0.0f ? -INFINITY : st[j].x);
#pragma unroll
        for (int j = 0; j < A; j++)
            if (j < P.splits && !(st[j].y < 0.0f)) any = true, sum += weight(st[j]);
    } else {
        for (int i = lane; i < P.splits; i += 64) {
            const float2 one = stats[i];
            ref = fmaxf(ref, one.y < 0.0f ? -INFINITY : one.x);
        }
        ref = qmm_max_lane_rows(ref);
        ref = fmaxf(ref, dpp_f<0x128>(ref)); // row_ror:8, then 4, 2, 1
        ref = fmaxf(ref, dpp_f<0x124>(ref));
        ref = fmaxf(ref, dpp_f<0x4E>(ref));
        ref = fmaxf(ref, dpp_f<0xB1>(ref));
        for (int i = lane; i < P.splits; i += 64) {
            const float2 one = stats[i];
            if (!(one.y < 0.0f)) any = true, sum += weight(one);
        }
        any = __any(any), sum = wave_sum(sum);
    }
    for (int i0 = mine; i0 < P.splits;) {
#pragma unroll
        for (int j = 0; j < A; j++)
            if (i0 + j * step < P.splits && !(st[j].y < 0.0f)) a += rescaled(v[j], weight(st[j]) / sum);
        i0 += A * step;
        if (i0 < P.splits) take(i0);
    }
    T* const to = static_cast<T*>(P.out) + token * P.out_stride + (row % P.heads) * D + at * E;
    if constexpr (FEW) {
#pragma unroll
        for (int e = 0; e < E; e++) to[e] = (T)(any ? a[e] : 0.0f);
    } else {
        __shared__ vec part[kPer][D / 4];
        part[mine][at] = a;
        __syncthreads();
        if (threadIdx.x >= D / 4) return;
        a = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; i++) a += part[i][at];
#pragma unroll
        for (int e = 0; e < E; e++) to[e] = (T)(any ? a[e] : 0.0f);
    }
}

#define PROMPT_TRY(expr)                                                               \
    do {                                                                               \
        hipError_t e_ = (expr);                                                        \
        if (e_ != hipSuccess) {                                                        \
            (void)hipGetLastError();                                                   \
            return qmm_fail(IZWI_QMM_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
        }                                                                              \
    } while (0)

// Tiles of `rows` rows, as far as the host can tell (of several sequences the last tiles may be partly filled).
int64_t row_tiles(const PromptParams& P, int rows) { return P.cu_q ? P.total_q * P.group / rows + P.batch : (P.total_q * P.group + rows - 1) / rows; }

// Parts that the keys are split into where workgroups are few: two tiles of `step` positions a part at the least, as a second launch has to join
// them: f16 and bf16 from eight tiles on (16 tokens of 16 heads on 8 behind 240: in one part 8.8 us, in two 10.8; behind 500: 13.0,
// 13.3, in four 11.7; behind 1000 18.8, 15.8, 12.6, in eight 11.1; of 32 on 8 and 16 on 2 alike), f32, whose tiles take three times as long, from four (behind 240: in one
// part 30.6 us, in two 21.0, in four 14.8).
// A causal f32 prompt in the larger workgroups: their lengths differ, so that one or two parts each are better rounded up to half as many again as
// there are compute units (16 heads on 8: D = 128 800 tokens in two parts 57, in four 45; 1000 69, in three 55; D = 256 400 47, in four 45; 600 in
// one part 87, in three 55; 900 128, in two 93; 1200 169, 142; 2048 299, 330; not causal 600 88, in two 109; six causal ones of 128 26, 42).
template <typename T>
int splits_of(int64_t wgs, int64_t max_k, int step, int n_cus, bool unequal = false) {
    const int64_t tiles = (max_k + step - 1) / step;
    const int64_t parts = sizeof(T) == 4 && unequal && n_cus / wgs <= 2 ? (6 * n_cus / wgs + 3) / 4 : n_cus / wgs;
    return tiles < (sizeof(T) == 4 ? 4 : 8) ? 1 : (int)std::max<int64_t>(1, std::min(parts, tiles / 2));
}

// f32 in the larger workgroups, one to a compute unit, of about equal lengths, that come in one part: in two to eight where a last turn that is nearly
// empty costs more than the join, by an estimate in us from what a tile (heads of 128 3.3, of 256 4.2) and a part's sums take.  16 heads on 8,
// not causal, us in one part and so: D = 128 1100 tokens 109, 97; 1400 151, 141; 2500 476, 358; 3500 661, 664; 8 heads on 8 2200 208, 159; 5000 933, 658; 32 on
// 8 550 60, 63; 1250 248, 208; ten sequences of up to 128 behind 500 73, 48; D = 256 1200 337, 250; 17 of up to 28 behind 13484 1850, 1045; 2048, whose turns are full, 547 (in three parts 621).
// As many as leave the stream's buffer within 256 MiB, sums and statistics (it grows to one and a half times what is asked for).
constexpr int64_t kMostScratch = (1 << 28) / 3 * 2;
int parts_by_turns(int64_t likely, int64_t most, int64_t tiles, int64_t rows, int d, int n_cus) { // (workgroups that have rows: the device knows)
    const double tile = d == 256 ? 4.2 : 3.3, join = (double)rows * d * 8 / 4e6; // of a part
    const auto turns = [&](int64_t wgs) { return (double)((wgs + n_cus - 1) / n_cus); };
    int best = 1;
    double least = 0.0;
    for (int parts = 1; parts <= std::max<int64_t>(1, std::min<int64_t>(8, tiles / 2)) && parts * rows * (d * 4 + 8) <= kMostScratch; parts++) {
        const double t = (2 * turns(likely * parts) + turns(most * parts)) / 3 * (double)((tiles + parts - 1) / parts) * tile + (parts > 1 ? 4.0 + join * parts : 0.0);
        if (parts == 1 || t < least) least = t, best = parts;
    }
    return best;
}

template <typename T, int D, int WR, int WZ, int DZ, int KT>
hipError_t launch(PromptParams P, int64_t max_k, int device, int n_cus, hipStream_t stream) {
    constexpr int N = Elem<T>::N, KS = KT * WZ;
    constexpr size_t lds = (size_t)2 * N * KS * D * 2 * (N == 1 || (DZ == 1 && WZ == 1) ? 2 : 1) + (DZ > 1 ? 2 * 64 * WR * WZ * DZ * KT / 32 * 16 * 4 : 0) + 16;
    static_assert(lds <= 160 * 1024);
    const int64_t wgs = row_tiles(P, 32 * WR) * P.kv_heads;
    P.tiles = (int)(wgs / P.kv_heads);
    // (f32 heads of 64 go to the larger workgroups for one tile, or where these are as many as the compute units, of causal calls twice as many: too
    // few or too many to be split)
    constexpr bool kSplits = sizeof(T) != 4 || D != 64 || WZ != 1;
    P.splits = kSplits ? splits_of<T>(wgs, max_k, KS, n_cus, P.causal && WZ == 1 && P.batch == 1) : 1;
    if constexpr (sizeof(T) == 4 && D >= 128 && WZ == 1)
        if (P.splits == 1 && P.batch <= 256 && (!P.causal || P.total_k >= 4 * P.total_q)) { // (the join looks through the offsets, 64 at a time)
            const int64_t likely = ((P.total_q * P.group + 32 * WR - 1) / (32 * WR) + (P.batch - 1) / 2) * P.kv_heads; // (the bound has a tile more a sequence)
            P.splits = parts_by_turns(likely, P.batch > 1 ? wgs : likely, (max_k + KS - 1) / KS, P.total_q * P.heads, D, n_cus);
        }
    // Sequences of several tiles on a few workgroups a compute unit: by length (unsplit).  Us by the offsets and so: f32 six causal prompts up to 700 85 to
    // 96, 75; bf16 D = 256 twelve up to 1000 122, 112; D = 64 five up to 2500 67, 61, four not causal up to 1500 60, 59; 16 heads on 2 twelve up to 900 60, 54; but where
    // workgroups are many, the last ones matter less than that those of one sequence find its keys in the L2 (30 up to 1501 of 32 heads 380, 401),
    // and many short sequences are over too soon (64 up to 100 19.6, 21.4).
    P.by_length = P.splits == 1 && P.batch > 1 && P.batch <= 64 && wgs > n_cus && wgs <= 8 * (int64_t)n_cus && P.total_q * P.group >= 4 * 128 * (int64_t)P.batch;
    const int64_t rows = P.total_q * P.heads;
    if (P.splits > 1) {
        void* scratch = nullptr;
        const hipError_t e = qmm_get_scratch(device, stream, (size_t)rows * P.splits * (D * sizeof(float) + sizeof(float2)), &scratch);
        if (e != hipSuccess) return e;
        P.sums = static_cast<float*>(scratch);
        P.stats = reinterpret_cast<float2*>(P.sums + (size_t)rows * P.splits * D);
    }
    const auto run = [&](auto split) {
        constexpr auto kernel = prompt_attention_kernel<T, D, WR, WZ, DZ, KT, decltype(split)::value>;
        if (lds > 64 * 1024) { // (once per kernel and device: the call takes as long as the checks in front of it)
            static std::atomic<uint64_t> allowed{0};
            const uint64_t bit = device < 64 ? 1ull << device : 0;
            if (!(allowed.load(std::memory_order_relaxed) & bit)) {
                const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
                if (e != hipSuccess) return e;
                allowed.fetch_or(bit, std::memory_order_relaxed);
            }
        }
        kernel<<<(unsigned)(wgs * P.splits), 64 * WR * WZ * DZ, lds, stream>>>(P);
        return hipGetLastError();
    };
    if constexpr (kSplits)
        if (P.splits > 1) {
            const hipError_t e = run(std::true_type{});
            if (e != hipSuccess) return e;
            if (P.splits <= 8) prompt_join_kernel<T, D, true><<<(unsigned)((rows + 3) / 4), 256, 0, stream>>>(P, rows);
            else prompt_join_kernel<T, D, false><<<(unsigned)rows, 256, 0, stream>>>(P, rows);
            return hipGetLastError();
        }
    return run(std::false_type{});
}
// Which workgroups.  f16 and bf16: four waves of 32 rows on 64 keys at a time (two on halves of the head each for D = 256, 32 keys), or where
// those would not fill the compute units, two waves of rows on 32 keys and two on the 32 behind them (D = 256: half the rows): causal
// prompts, whose workgroups are of unequal length, change over later.  16 bf16 heads on 8, us of the larger and the smaller workgroups: D = 128
// causal 700 tokens 28, 15; 2600 63, 52; 3500 93, 90; not causal 700 27, 15; 1500 37, 39; 2000 53, 56; D = 64 causal 2600 45, 34; 3500
// 62, 54; not causal 2600 66, 59; 3500 93, 101; D = 256 causal 2048 105, 84; 2600 134, 140; not causal 700 42, 29; 1500 75, 107 (of as many rows in 32 heads
// on 8, 8 on 8 and 16 on 2, twenty-two of each, the side taken is the slower one by 3 % at most).  More than 64 rows on very many keys read them too
// often with the smaller ones (17 tokens of 32 heads behind 30011 34, 38; 250 of 16 behind 8000 39, 42, behind 2000 25, 22).  Up to 64 keys the
// second pair would have few (37 tokens 6.5, 7.1).
// f32: the larger ones, whose next tile is taken apart beside the products, and the smaller where those leave compute units without work.  16
// heads on 8, us of the larger and the smaller: D = 128 few rows and many tiles each (4 tokens behind 1087 of 10 sequences 46.7, 36.5), two to
// four tiles (37 tokens 12.4, 11.6; 100 of 6 sequences 23, 16; one tile 8.8, 11.2; seven 28, 31), several causal prompts that are about as many
// larger workgroups as compute units, of unequal length and not in parts (700 and 700 tokens 73, 52; four of 400 45, 41; 1000 and 900 101, 82; six of
// 300 38.5, 40.6; of 8 heads on 8 and 16 on 2 alike, of 32 on 8 450, 150 and 250 50, 44; 500 and 450 55, 52), but not those behind a
// past and one prompt only where its tiles are few for its rows: these come in parts, whose join goes by the rows (1100 tokens 64, 75; 2048 137, 144; 3500
// 332, 408; behind 3000 250, 393; four of 300 behind 1000 110, 152; not causal 1100 98, 149; 8 heads on 8 2200 99, 139; but of 32 on 8 550 45, 42.5; 1024
// 86, 80); D = 64 causal 1200 tokens 64, 43; 3500 197, 174; 6000 433, 461; 100 of 30 15.7, 17.9; not causal
// 1200 64, 62; 2048 113, 113; one tile (9 of 13) 5.6, 6.6.
template <typename T, int D>
hipError_t launch_of(const PromptParams& P, int64_t max_k, int device, int n_cus, hipStream_t stream) {
    const int64_t all = P.total_q * P.group, wgs = std::max<int64_t>((all + 127) / 128, P.batch) * P.kv_heads, rows = all / P.batch; // rows: of a sequence, on average
    constexpr int DZ = D == 256 ? 2 : 1;
    if constexpr (sizeof(T) == 4 && D == 256) {
        return launch<T, D, 2, 1, DZ, 32>(P, max_k, device, n_cus, stream);
    } else if constexpr (sizeof(T) == 4) {
        const int64_t tiles = (max_k + 31) / 32;
        const int64_t large = row_tiles(P, 128) * P.kv_heads; // workgroups
        const bool small = D == 64 ? tiles > 1 && large < (P.causal ? 2 : 1) * (int64_t)n_cus
                                   : (rows <= 64 && tiles >= 4 * splits_of<T>(wgs, max_k, 32, n_cus)) || (tiles > 1 && tiles <= 4 && 2 * large <= n_cus) ||
                                         (P.causal && (P.batch > 1 ? P.total_k <= 2 * P.total_q : large > 6 * tiles) && tiles >= 12 && 2 * large > n_cus && 4 * large <= 5 * n_cus);
        return small ? launch<T, D, 2, 2, DZ, 32>(P, max_k, device, n_cus, stream) : launch<T, D, 4, 1, DZ, 32>(P, max_k, device, n_cus, stream);
    } else {
        const int quarters = P.causal ? (D == 64 ? 8 : D == 128 ? 7 : 4) : (D == 64 ? 6 : 2); // of a workgroup per compute unit
        const bool small = 4 * wgs <= quarters * n_cus && (D == 256 || max_k > 64) && (rows <= 64 || max_k < 8192);
        if constexpr (D == 256) return small ? launch<T, D, 2, 1, DZ, 32>(P, max_k, device, n_cus, stream) : launch<T, D, 4, 1, DZ, 32>(P, max_k, device, n_cus, stream);
        else return small ? launch<T, D, 2, 2, DZ, 32>(P, max_k, device, n_cus, stream) : launch<T, D, 4, 1, DZ, 64>(P, max_k, device, n_cus, stream);
    }
}

template <typename T>
int prompt_attention_impl(const T* q, int64_t q_stride, const T* k, int64_t k_stride, const T* v, int64_t v_stride, const int32_t* cu_q,
                          const int32_t* cu_k, int64_t batch, int64_t total_q, int64_t total_k, int64_t max_k, int64_t heads, int64_t kv_heads, int64_t d,
                          int causal, float scale, T* out, int64_t out_stride, void* stream_) {
    constexpr const char* what = "prompt_attention";
    if (d != 64 && d != 128 && d != 256)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: head_dim %lld (64, 128 and 256 are built)", what, (long long)d);
    if (batch < 0 || total_q < 0 || total_k < 0 || max_k < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 65535 || batch > 0xfffff)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: bad shape (batch %lld, tokens %lld on %lld, heads %lld on %lld)", what, (long long)batch,
                        (long long)total_q, (long long)total_k, (long long)heads, (long long)kv_heads);
    if ((cu_q == nullptr) != (cu_k == nullptr) || (!cu_q && batch != 1))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: offsets of queries and keys come together, and only one sequence (not %lld) has none", what, (long long)batch);
    if (q_stride < heads * d || out_stride < heads * d || k_stride < kv_heads * d || v_stride < kv_heads * d)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: rows overlap (strides %lld, %lld, %lld, %lld)", what, (long long)q_stride, (long long)k_stride,
                        (long long)v_stride, (long long)out_stride);
    if (!std::isfinite(scale) || std::fabs(scale) > 0x1p126f) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: scale %g", what, (double)scale); // (log2(e) as much is a float, too)
    constexpr int kPiece = 16 / (int)sizeof(T);
    if (q_stride % kPiece || k_stride % kPiece || v_stride % kPiece || out_stride % kPiece ||
        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out)) & 15))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: rows must begin on 16 bytes", what);
    if (total_q * heads > 0x3fffffff || total_k > 0x3fffffff || k_stride > (1 << 23) || v_stride > (1 << 23) || q_stride > 0x3fffffff ||
        out_stride > 0x3fffffff)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: %lld tokens of %lld heads on %lld, rows %lld and %lld apart", what, (long long)total_q,
                        (long long)heads, (long long)total_k, (long long)k_stride, (long long)v_stride);
    if (batch == 0 || total_q == 0) return IZWI_QMM_OK;
    if (!q || !out || (total_k && (!k || !v))) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: NULL buffer", what);
    const auto rows = [&](const void* at, int64_t n, int64_t stride, int64_t of_heads) { return QmmRows{at, n, stride * (int64_t)sizeof(T), of_heads * d * (int64_t)sizeof(T)}; };
    const QmmRows to = rows(out, total_q, out_stride, heads);
    if (!qmm_rows_apart(to, rows(q, total_q, q_stride, heads)) || !qmm_rows_apart(to, rows(k, total_k, k_stride, kv_heads)) || !qmm_rows_apart(to, rows(v, total_k, v_stride, kv_heads)))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: out shares memory with q, k or v", what);
    const int64_t offsets = cu_q ? 1 : 0; // (as one row of out's stride: between two of its rows there may be room)
    if (!qmm_rows_apart(to, {cu_q, offsets, to.stride, (batch + 1) * 4}) || !qmm_rows_apart(to, {cu_k, offsets, to.stride, (batch + 1) * 4}))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: out shares memory with the offsets", what);
    if ((total_q * (heads / kv_heads) / 32 + batch) * kv_heads > 0x3fffff)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: %lld sequences on %lld kv heads", what, (long long)batch, (long long)kv_heads);
    int device = 0, n_cus = 0;
    if (int rc = qmm_current_device(&device, &n_cus)) return rc;
    PromptParams P{};
    P.q = q, P.k = k, P.v = v, P.out = out;
    P.q_stride = q_stride, P.k_stride = k_stride, P.v_stride = v_stride, P.out_stride = out_stride;
    P.cu_q = cu_q, P.cu_k = cu_k, P.total_q = total_q, P.total_k = total_k;
    P.batch = (int)batch, P.heads = (int)heads, P.kv_heads = (int)kv_heads, P.group = (int)(heads / kv_heads), P.causal = causal != 0;
    const double by = std::fabs((double)scale) * 1.4426950408889634074;
    P.sign = scale == 0.0f ? 0.0f : scale < 0.0f ? -1.0f : 1.0f;
    P.scale = scale == 0.0f ? 1.0f : (float)by, P.scale_rest = scale == 0.0f ? 0.0f : (float)(by - (double)P.scale);
    max_k = std::min(max_k, total_k);
    hipStream_t stream = (hipStream_t)stream_;
    QmmCallScope call;
    PROMPT_TRY((d == 64    ? launch_of<T, 64>(P, max_k, device, n_cus, stream)
                : d == 128 ? launch_of<T, 128>(P, max_k, device, n_cus, stream)
                           : launch_of<T, 256>(P, max_k, device, n_cus, stream)));
    return IZWI_QMM_OK;
}

} // namespace

extern "C" {

#define PROMPT_ATTENTION(NAME, C, T)                                                                                                                     \
    int NAME(const C* q, int64_t q_stride, const C* k, int64_t k_stride, const C* v, int64_t v_stride, const int32_t* cu_q, const int32_t* cu_k,         \
             int64_t batch, int64_t total_q, int64_t total_k, int64_t max_k, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int causal,      \
             float scale, C* out, int64_t out_stride, void* stream) {                                                                                    \
        return qmm_guarded(#NAME, [&]() -> int {                                                                                                         \
            return prompt_attention_impl<T>((const T*)q, q_stride, (const T*)k, k_stride, (const T*)v, v_stride, cu_q, cu_k, batch, total_q, total_k,    \
                                            max_k, num_heads, num_kv_heads, head_dim, causal, scale, (T*)out, out_stride, stream);                       \
        });                                                                                                                                              \
    }
PROMPT_ATTENTION(izwi_qmm_prompt_attention_f32, float, float)
PROMPT_ATTENTION(izwi_qmm_prompt_attention_f16, uint16_t, f16_t)
PROMPT_ATTENTION(izwi_qmm_prompt_attention_bf16, uint16_t, bf16_t)

} // extern "C"
