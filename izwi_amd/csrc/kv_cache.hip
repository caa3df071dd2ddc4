// Writing the quantized key / value cache and reading it back (layout: kv_cache.h).
//
// A block of 32 values becomes an f16 scale and 32 quants, by the arithmetic of the GGUF formats in f32:
//   Q8_0  d = max|v| / 127,            quant = round(v * (1 / d)), halves away from zero
//   Q4_0  d = (first v of max|v|) / -8, quant = min(15, floor(v * (1 / d) + 8.5)) - 8
// and a value read back is f32(f16(d)) * quant, one rounding if it is stored as f16.  A block whose scale has no f16
// (an infinity or NaN among its values, or one beyond the range) reads as NaN throughout rather than as a number that it
// never held; one whose scale is zero in f16 reads as zeros.
//
// Every byte is touched once: bound by memory (12800 tokens of 8 heads of 128, f32 to Q8_0 and back: 24 us to write, 5.6 TB/s, 26 to
// read, 6.2 TB/s), small calls by the launch.  Beside the loads, the two IEEE divisions of a block count: they are worked
// out by one lane per block and handed round (with every lane of a value block dividing, writing took 27 us).
#include "kv_cache.h"

#include <type_traits>
#include <utility>

#include "qmm_lanes.h"

namespace {

typedef _Float16 f16_t;

struct KvRowsParams {
    const void* k_in;
    const void* v_in;
    void* k_out;
    void* v_out;
    int64_t k_stride, v_stride; // elements between the rows of two tokens
    KvPlanes cache;
    const int32_t* starts; // [batch]
    const int32_t* counts; // [batch], or NULL: every token counts
    const uint8_t* lineage; // [slots][padded], or NULL
    int beams;
    unsigned tokens, kv_heads, groups, items, rows; // groups of sixteen positions that `tokens` tokens may touch; items = batch * groups * kv_heads, rows = batch * tokens * kv_heads
    int first_slot;
    int64_t capacity;
    unsigned k_blocks; // workgroups that take keys; the others take values
};

// largest over the lanes x, 16 + x, 32 + x, 48 + x; over the sixteen lanes of a row
__device__ __forceinline__ unsigned umax_rows(unsigned v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max((unsigned)a[0], (unsigned)a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((unsigned)b[0], (unsigned)b[1]);
}
template <int CTRL>
__device__ __forceinline__ unsigned umax_dpp(unsigned v, unsigned of) {
    return max(v, (unsigned)__builtin_amdgcn_update_dpp((int)of, (int)of, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ unsigned umax8(unsigned v) {
    v = umax_dpp<0xB1>(v, v);        // quad_perm [1,0,3,2]
    v = umax_dpp<0x4E>(v, v);        // quad_perm [2,3,0,1]
    return umax_dpp<0x141>(v, v);    // row_half_mirror
}
__device__ __forceinline__ unsigned umax16(unsigned v) {
    v = umax8(v);
    return umax_dpp<0x140>(v, v);    // row_mirror
}
enum Lanes { kLanes4, kLanes8, kLanes16 }; // that hold a block: x, 16 + x, 32 + x, 48 + x; eight neighbours; sixteen neighbours
template <Lanes L>
__device__ __forceinline__ unsigned umax_over(unsigned v) {
    return L == kLanes4 ? umax_rows(v) : L == kLanes8 ? umax8(v) : umax16(v);
}

// The scale of a block whose largest magnitude has these bits (and, for Q4_0, this sign), and what its values are multiplied by;
// `bad`: a block without a scale, whose values do not count.
template <int QT>
__device__ __forceinline__ f16_t block_scale(unsigned amax, unsigned sign, float& inv, bool& bad) {
    const float d = QT == IZWI_KV_Q8_0 ? __fdiv_rn(__uint_as_float(amax), 127.0f) : __uint_as_float(amax | (sign << 31)) * -0.125f;
    const f16_t h = (f16_t)d;
    bad = amax >= 0x7f800000u || (float)h == INFINITY || (float)h == -INFINITY;
    inv = bad || h == (f16_t)0.0f ? 0.0f : __fdiv_rn(1.0f, d);
    return bad ? (f16_t)NAN : h;
}
// (a scale of zero multiplies by zero: quants of zero)
template <int QT>
__device__ __forceinline__ unsigned block_quant(float v, float inv) {
    const float scaled = __fmul_rn(v, inv);
    return QT == IZWI_KV_Q8_0 ? (unsigned)(qmm_round_clamp_i8(scaled) + 128) : (unsigned)min(15, (int)__fadd_rn(scaled, 8.5f));
}

// Of N values per lane, value n's largest over the sixteen lanes of a row, in lane x = n (and n + 8 where N = 8): halves of the values
// change lanes instead of every value going round, three instructions for two values a step.
template <int N>
__device__ __forceinline__ unsigned umax_scatter(const unsigned (&of)[N], int x) {
    static_assert(N == 8 || N == 16);
    unsigned v[N];
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = of[i];
    const auto step = [&](auto width, auto ctrl) { // values i and i + width: lanes with that bit keep the second
        constexpr int W = decltype(width)::value;
        const bool up = x & W;
#pragma unroll
        for (int i = 0; i < W; i++) {
            const unsigned keep = up ? v[i + W] : v[i], give = up ? v[i] : v[i + W];
            v[i] = umax_dpp<decltype(ctrl)::value>(keep, give);
        }
    };
    if constexpr (N == 16) {
        step(std::integral_constant<int, 8>{}, std::integral_constant<int, 0x128>{}); // row_ror:8
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = umax_dpp<0x128>(v[i], v[i]);
    }
    // (the lane 4 away in either direction: within a half row, mirrored twice)
    const bool up = x & 4;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const unsigned keep = up ? v[i + 4] : v[i], give = up ? v[i] : v[i + 4];
        const unsigned turned = (unsigned)__builtin_amdgcn_update_dpp((int)give, (int)give, 0x141, 0xf, 0xf, false); // row_half_mirror: lane x ^ 7
        v[i] = umax_dpp<0x1B>(keep, turned);                                                                          // quad_perm [3,2,1,0]: x ^ 3
    }
    step(std::integral_constant<int, 2>{}, std::integral_constant<int, 0x4E>{});
    step(std::integral_constant<int, 1>{}, std::integral_constant<int, 0xB1>{});
    return v[0];
}

// The N values of this lane out of a block that several lanes hold in the order of `lane`: the block's scale, and the quants as the cache stores them (q + 128, q + 8).  Magnitudes are compared as bits, so that a
// NaN is the largest of all.
template <int QT, int N, Lanes L>
__device__ __forceinline__ f16_t quantize_block(const float (&v)[N], int lane, unsigned (&q)[N]) {
    unsigned best = 0, sign = 0; // the lane's first value of largest magnitude
#pragma unroll
    for (int i = 0; i < N; i++) {
        const unsigned bits = __float_as_uint(v[i]), mag = bits & 0x7fffffffu;
        if (mag > best) best = mag, sign = bits >> 31;
    }
    const unsigned amax = umax_over<L>(best);
    unsigned key = 0;
    if constexpr (QT == IZWI_KV_Q4_0) key = umax_over<L>(best == amax ? ((unsigned)(16 - lane) << 1) | sign : 0u); // the lowest lane that holds the maximum decides the sign
    float inv;
    bool bad;
    const f16_t d = block_scale<QT>(amax, key & 1, inv, bad);
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = block_quant<QT>(bad ? 0.0f : v[i], inv);
    return d;
}

template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_values(const T* p, float (&v)[N]) {
    if constexpr (VEC) {
        typedef T vec __attribute__((ext_vector_type(N)));
        const vec t = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (float)p[i];
    }
}

template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_values(T* p, const float (&v)[N]) {
    if constexpr (VEC) {
        typedef T vec __attribute__((ext_vector_type(N)));
        vec t;
#pragma unroll
        for (int i = 0; i < N; i++) t[i] = (T)v[i];
        *reinterpret_cast<vec*>(p) = t;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = (T)v[i];
    }
}

// A wave has sixteen positions of one head, aligned as the cache's groups are, so that what it writes there (or reads) is whole pieces
// side by side: 16 bytes a lane.  (With a lane per four values and no such groups, writing 12800 tokens of 8 heads of 128 took 48 us
// and reading them 42.)
struct KvGroup {
    unsigned seq, head;
    int64_t pos0, start; // the group's first position, the sequence's
    int64_t begin;       // the sequence's slot and head in the planes
    int64_t slot;
    int64_t count;
    __device__ __forceinline__ bool token(int64_t capacity, int64_t pos, int64_t& t) const { // of this call, at this position
        t = pos - start;
        return t >= 0 && t < count && pos >= 0 && pos < capacity;
    }
};
__device__ __forceinline__ bool kv_group(const KvRowsParams& P, unsigned block, KvGroup& it) {
    const unsigned item = block * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= P.items) return false;
    const unsigned row = item / P.kv_heads, group = row % P.groups;
    it.head = item - row * P.kv_heads, it.seq = row / P.groups;
    it.start = P.starts[it.seq];
    it.count = P.counts ? min((int64_t)P.counts[it.seq], (int64_t)P.tokens) : (int64_t)P.tokens;
    it.pos0 = (it.start >> 4 << 4) + 16 * (int64_t)group;
    it.slot = (int64_t)P.first_slot + it.seq;
    it.begin = (it.slot * P.cache.kv_heads + it.head) * P.cache.padded;
    return true;
}

// Keys: lane (x, g) has of position x the values 8 g .. 8 g + 7 of every block.  Values: lane (x, g) has of positions 4 g .. 4 g + 3 the
// values 2 x and 2 x + 1 of every block.
template <typename T, int QT, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_append_kernel(KvRowsParams P) {
    using Row = KvRow<QT, D>;
    constexpr int NB = Row::kBlocks;
    const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
    const bool keys = blockIdx.x < P.k_blocks;
    KvGroup it;
    if (!kv_group(P, keys ? blockIdx.x : blockIdx.x - P.k_blocks, it)) return;
    if (it.pos0 + 16 <= it.start || it.pos0 >= it.start + it.count || it.pos0 >= P.capacity || it.pos0 < 0) return;
    if (keys) {
        int64_t t;
        const bool mine = it.token(P.capacity, it.pos0 + x, t);
        if (!mine) t = max((int64_t)0, min(it.count - 1, t)); // (the exchanges between lanes need every lane)
        const T* src = static_cast<const T*>(P.k_in) + ((int64_t)it.seq * P.tokens + t) * P.k_stride + it.head * D + 8 * g;
        float v[NB][8];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) load_values<T, 4, VEC>(src + 32 * b + 4 * h, *reinterpret_cast<float(*)[4]>(&v[b][4 * h]));
        f16_t d[NB];
        uint32_t w[Row::kBytes / 16];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            unsigned q[8];
            d[b] = quantize_block<QT, 8, kLanes4>(v[b], g, q);
            if constexpr (QT == IZWI_KV_Q8_0) {
                w[2 * b] = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
                w[2 * b + 1] = q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24;
            } else {
                w[b] = q[0] | q[2] << 4 | q[4] << 8 | q[6] << 12 | q[1] << 16 | q[3] << 20 | q[5] << 24 | q[7] << 28;
            }
        }
        if (!mine) return;
        uint8_t* dst = P.cache.kq + (it.begin + it.pos0) * Row::kBytes + lane * Row::kPiece;
        constexpr int W = Row::kPiece / 4;
        typedef uint32_t vec __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int i = 0; i < NB / Row::kPer; i++) {
            vec t;
#pragma unroll
            for (int n = 0; n < W; n++) t[n] = w[i * W + n];
            *reinterpret_cast<vec*>(dst + 64 * Row::kPiece * i) = t;
        }
        if (g == 0) {
            typedef f16_t scales __attribute__((ext_vector_type(NB)));
            scales t;
#pragma unroll
            for (int b = 0; b < NB; b++) t[b] = d[b];
            *reinterpret_cast<scales*>(P.cache.ks + (it.begin + it.pos0 + x) * NB) = t;
        }
        return;
    }
    bool mine[4];
    float v[4][NB][2];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        int64_t t;
        mine[i] = it.token(P.capacity, it.pos0 + 4 * g + i, t);
        t = mine[i] ? t : max((int64_t)0, min(it.count - 1, t));
        const T* src = static_cast<const T*>(P.v_in) + ((int64_t)it.seq * P.tokens + t) * P.v_stride + it.head * D + 2 * x;
#pragma unroll
        for (int b = 0; b < NB; b++) load_values<T, 2, VEC>(src + 32 * b, v[i][b]);
    }
    // a round of up to sixteen blocks (positions of the four, blocks of a row): lane x works out the scale of block x of the round for all
    constexpr int R = 4 * NB < 16 ? 4 * NB : 16, I = R / NB; // blocks, positions of a round
    uint16_t half[4][Row::kLane / 2] = {};
    f16_t d[4 / I]; // of block x % R of the rounds
#pragma unroll
    for (int i0 = 0; i0 < 4; i0 += I) {
        unsigned amax[R], sign[R];
#pragma unroll
        for (int n = 0; n < R; n++) {
            const unsigned u0 = __float_as_uint(v[i0 + n / NB][n % NB][0]), u1 = __float_as_uint(v[i0 + n / NB][n % NB][1]);
            const bool second = (u1 & 0x7fffffffu) > (u0 & 0x7fffffffu);
            amax[n] = (second ? u1 : u0) & 0x7fffffffu, sign[n] = (second ? u1 : u0) >> 31;
        }
        const unsigned mine_max = umax_scatter<R>(amax, x);
        unsigned key = 0;
        if constexpr (QT == IZWI_KV_Q4_0) { // the lowest lane that holds the maximum decides the sign
            unsigned keys[R];
            each<R>([&](auto n) { keys[n] = amax[n] == of_lane<n>(mine_max) ? (unsigned)(16 - x) << 1 | sign[n] : 0u; });
            key = umax_scatter<R>(keys, x);
        }
        float inv;
        bool bad;
        d[i0 / I] = block_scale<QT>(mine_max, key & 1, inv, bad);
        const unsigned mine_inv = __float_as_uint(inv), mine_bad = bad;
        each<R>([&](auto n) {
            const float by = __uint_as_float(of_lane<n>(mine_inv));
            const bool none = of_lane<n>(mine_bad);
            const int i = i0 + n / NB, b = n % NB;
            const unsigned q0 = block_quant<QT>(none ? 0.0f : v[i][b][0], by), q1 = block_quant<QT>(none ? 0.0f : v[i][b][1], by);
            if constexpr (QT == IZWI_KV_Q8_0) half[i][b] = (uint16_t)(q0 | q1 << 8);
            else half[i][b / 2] |= (uint16_t)((q0 | q1 << 4) << (8 * (b & 1)));
        });
    }
    const int64_t pos = it.pos0 + 4 * g;
    uint8_t* plane = P.cache.vq + it.begin * Row::kBytes;
    f16_t* scales = P.cache.vs + it.begin * NB;
    if (mine[0] && mine[1] && mine[2] && mine[3]) {
        constexpr int W = Row::kValuePiece / 4;
        typedef uint32_t vec __attribute__((ext_vector_type(W)));
        uint32_t w[Row::kLane];
#pragma unroll
        for (int n = 0; n < Row::kLane; n++) {
            constexpr int J = Row::kLane / 2;
            w[n] = half[2 * (n / J)][n % J] | (uint32_t)half[2 * (n / J) + 1][n % J] << 16;
        }
#pragma unroll
        for (int i = 0; i < Row::kLane / W; i++) {
            vec t;
#pragma unroll
            for (int n = 0; n < W; n++) t[n] = w[i * W + n];
            *reinterpret_cast<vec*>(plane + Row::value(pos, x, 0) + 16 * Row::kValuePiece * i) = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (mine[i])
#pragma unroll
                for (int j = 0; j < Row::kLane / 2; j++) *reinterpret_cast<uint16_t*>(plane + Row::value(pos + i, x, j)) = half[i][j];
    }
    if (x < R)
#pragma unroll
        for (int i0 = 0; i0 < 4; i0 += I) {
            const int i = i0 + x / NB;
            if (!(i == 0 ? mine[0] : i == 1 ? mine[1] : i == 2 ? mine[2] : mine[3])) continue;
            scales[Row::value_scale(pos + i, x % NB)] = d[i0 / I];
        }
}

// The same lanes the other way; what the cache does not have reads as zeros.
template <typename T, int QT, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(KvRowsParams P) {
    using Row = KvRow<QT, D>;
    constexpr int NB = Row::kBlocks, kBias = QT == IZWI_KV_Q8_0 ? 128 : 8;
    const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
    const bool keys = blockIdx.x < P.k_blocks;
    KvGroup it;
    if (!kv_group(P, keys ? blockIdx.x : blockIdx.x - P.k_blocks, it)) return;
    if (it.pos0 + 16 <= it.start || it.pos0 >= it.start + (int64_t)P.tokens) return;
    // where position `pos` of the sequence stands in the planes, and whether there is one
    const auto place = [&](int64_t pos, bool there, int64_t& begin) {
        begin = it.begin;
        if (P.lineage && there) {
            const int beam = P.lineage[it.slot * P.cache.padded + pos];
            there = beam < P.beams;
            if (there) begin += (it.slot / P.beams * P.beams + beam - it.slot) * P.cache.kv_heads * P.cache.padded;
        }
        return there;
    };
    if (keys) {
        const int64_t pos = it.pos0 + x;
        int64_t t, begin;
        const bool there = place(pos, it.token(P.capacity, pos, t), begin);
        if (t < 0 || t >= (int64_t)P.tokens) return;
        uint32_t w[Row::kBytes / 16];
        f16_t d[NB] = {};
        if (there) {
            const uint8_t* src = P.cache.kq + begin * Row::kBytes + Row::key(pos, 0, g);
#pragma unroll
            for (int i = 0; i < NB / Row::kPer; i++)
                __builtin_memcpy(w + i * (Row::kPiece / 4), __builtin_assume_aligned(src + 64 * Row::kPiece * i, Row::kPiece), Row::kPiece);
            __builtin_memcpy(d, __builtin_assume_aligned(P.cache.ks + (begin + pos) * NB, 2 * NB), 2 * NB);
        }
        T* dst = static_cast<T*>(P.k_out) + (((int64_t)it.seq * P.tokens + t) * P.kv_heads + it.head) * D + 8 * g;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int j = 4 * h + i, n = (j >> 1) + 4 * (j & 1);
                    const int q = QT == IZWI_KV_Q8_0 ? (int)(w[2 * b + h] >> (8 * i) & 255) : (int)(w[b] >> (4 * n) & 15);
                    v[i] = there ? (float)d[b] * (float)(q - kBias) : 0.0f;
                }
                store_values<T, 4, VEC>(dst + 32 * b + 4 * h, v);
            }
        return;
    }
    const int64_t quad = it.pos0 + 4 * g;
    uint16_t half[4][Row::kLane / 2];
    f16_t d[4][NB];
    bool there[4];
    int64_t t[4], begin[4];
    bool all = !P.lineage;
#pragma unroll
    for (int i = 0; i < 4; i++) there[i] = place(quad + i, it.token(P.capacity, quad + i, t[i]), begin[i]), all &= there[i];
    if (all) {
        uint32_t w[Row::kLane];
        constexpr int J = Row::kLane / 2, W = Row::kValuePiece / 4;
        const uint8_t* src = P.cache.vq + it.begin * Row::kBytes + Row::value(quad, x, 0);
#pragma unroll
        for (int i = 0; i < Row::kLane / W; i++)
            __builtin_memcpy(w + i * W, __builtin_assume_aligned(src + 16 * Row::kValuePiece * i, Row::kValuePiece), Row::kValuePiece);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < J; j++) half[i][j] = (uint16_t)(w[(i >> 1) * J + j] >> (16 * (i & 1)));
        f16_t pairs[2][NB][2];
        __builtin_memcpy(pairs, __builtin_assume_aligned(P.cache.vs + it.begin * NB + Row::value_scale(quad, 0), 8 * NB), 8 * NB);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int b = 0; b < NB; b++) d[i][b] = pairs[i >> 1][b][i & 1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (!there[i]) continue;
#pragma unroll
            for (int j = 0; j < Row::kLane / 2; j++)
                half[i][j] = *reinterpret_cast<const uint16_t*>(P.cache.vq + begin[i] * Row::kBytes + Row::value(quad + i, x, j));
#pragma unroll
            for (int b = 0; b < NB; b++) d[i][b] = P.cache.vs[begin[i] * NB + Row::value_scale(quad + i, b)];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (t[i] < 0 || t[i] >= (int64_t)P.tokens) continue;
        T* dst = static_cast<T*>(P.v_out) + (((int64_t)it.seq * P.tokens + t[i]) * P.kv_heads + it.head) * D + 2 * x;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int q = QT == IZWI_KV_Q8_0 ? half[i][b] : half[i][b / 2] >> (8 * (b & 1)) & 255;
            const int q0 = QT == IZWI_KV_Q8_0 ? q & 255 : q & 15, q1 = QT == IZWI_KV_Q8_0 ? q >> 8 : q >> 4;
            const float v[2] = {there[i] ? (float)d[i][b] * (float)(q0 - kBias) : 0.0f, there[i] ? (float)d[i][b] * (float)(q1 - kBias) : 0.0f};
            store_values<T, 2, VEC>(dst + 32 * b, v);
        }
    }
}

// Few rows: a lane per four values of keys, sixteen lanes per row of values, a row at a time.
// Where the row of `item` stands: its sequence, token and head, and whether the cache has (or gets) it
struct KvItem {
    unsigned row, head;
    int64_t begin, pos; // the first position of its slot and head in the planes, its own from there
    bool there;
};
template <bool READ>
__device__ __forceinline__ KvItem kv_item(const KvRowsParams& P, unsigned item) {
    KvItem it;
    it.row = item / P.kv_heads, it.head = item - it.row * P.kv_heads;
    const unsigned b = it.row / P.tokens, t = it.row - b * P.tokens;
    const int64_t pos = (int64_t)P.starts[b] + t;
    it.there = pos >= 0 && pos < P.capacity && (!P.counts || (int64_t)t < P.counts[b]);
    int64_t slot = (int64_t)P.first_slot + b;
    if constexpr (READ) {
        if (P.lineage && it.there) {
            const int beam = P.lineage[slot * P.cache.padded + pos];
            it.there = beam < P.beams;
            if (it.there) slot = slot / P.beams * P.beams + beam;
        }
    }
    it.begin = (slot * P.cache.kv_heads + it.head) * P.cache.padded, it.pos = it.there ? pos : 0;
    return it;
}

// Keys: a lane takes four values of a row, 8 lanes a block.  Values: lane x of 16 takes the pairs 2 x, 2 x + 1 of every
// block.  (Lanes behind the last item repeat it and store nothing: the exchanges between lanes need them.)
template <typename T, int QT, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_append_rows_kernel(KvRowsParams P) {
    using Row = KvRow<QT, D>;
    if (blockIdx.x < P.k_blocks) {
        constexpr int kLanes = D / 4;
        const unsigned thread = blockIdx.x * 256 + threadIdx.x, asked = thread / kLanes, item = min(asked, P.rows - 1);
        const int e = (threadIdx.x % kLanes) * 4, b = e / 32, g = (e & 31) >> 3, second = (e >> 2) & 1;
        const KvItem it = kv_item<false>(P, item);
        float v[4];
        load_values<T, 4, VEC>(static_cast<const T*>(P.k_in) + it.row * P.k_stride + it.head * D + e, v);
        unsigned q[4];
        const f16_t d = quantize_block<QT, 4, kLanes8>(v, threadIdx.x & 7, q);
        uint8_t* dst = P.cache.kq + it.begin * Row::kBytes + Row::key(it.pos, b, g);
        const bool mine = asked < P.rows && it.there;
        if constexpr (QT == IZWI_KV_Q8_0) {
            if (mine) *reinterpret_cast<uint32_t*>(dst + 4 * second) = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
        } else {
            // values 0 2 1 3 of this half of the unit: nibbles 2 s, 2 s + 1 and, 16 bits up, the odd ones
            unsigned bits = (q[0] | q[2] << 4 | q[1] << 16 | q[3] << 20) << (8 * second);
            bits |= (unsigned)__builtin_amdgcn_update_dpp((int)bits, (int)bits, 0xB1, 0xf, 0xf, false);
            if (mine && !second) *reinterpret_cast<uint32_t*>(dst) = bits;
        }
        if (mine && (threadIdx.x & 7) == 0) P.cache.ks[(it.begin + it.pos) * Row::kBlocks + b] = d;
        return;
    }
    const unsigned thread = (blockIdx.x - P.k_blocks) * 256 + threadIdx.x, asked = thread / 16, item = min(asked, P.rows - 1);
    const int x = threadIdx.x & 15;
    const KvItem it = kv_item<false>(P, item);
    const T* src = static_cast<const T*>(P.v_in) + it.row * P.v_stride + it.head * D + 2 * x;
    float v[Row::kBlocks][2];
    uint16_t half[Row::kLane / 2] = {};
    f16_t d[Row::kBlocks];
#pragma unroll
    for (int b = 0; b < Row::kBlocks; b++) load_values<T, 2, VEC>(src + 32 * b, v[b]);
#pragma unroll
    for (int b = 0; b < Row::kBlocks; b++) {
        unsigned q[2];
        d[b] = quantize_block<QT, 2, kLanes16>(v[b], x, q);
        if constexpr (QT == IZWI_KV_Q8_0) half[b] = (uint16_t)(q[0] | q[1] << 8);
        else half[b / 2] |= (uint16_t)((q[0] | q[1] << 4) << (8 * (b & 1)));
    }
    if (asked >= P.rows || !it.there) return;
#pragma unroll
    for (int j = 0; j < Row::kLane / 2; j++) *reinterpret_cast<uint16_t*>(P.cache.vq + it.begin * Row::kBytes + Row::value(it.pos, x, j)) = half[j];
#pragma unroll
    for (int b = 0; b < Row::kBlocks; b++)
        if (x == b) P.cache.vs[it.begin * Row::kBlocks + Row::value_scale(it.pos, b)] = d[b];
}

// The same lanes the other way; what the cache does not have reads as zeros.
template <typename T, int QT, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_read_rows_kernel(KvRowsParams P) {
    using Row = KvRow<QT, D>;
    constexpr int kBias = QT == IZWI_KV_Q8_0 ? 128 : 8;
    if (blockIdx.x < P.k_blocks) {
        constexpr int kLanes = D / 4;
        const unsigned thread = blockIdx.x * 256 + threadIdx.x, item = thread / kLanes;
        if (item >= P.rows) return;
        const int e = (threadIdx.x % kLanes) * 4, b = e / 32, g = (e & 31) >> 3, second = (e >> 2) & 1;
        const KvItem it = kv_item<true>(P, item);
        float v[4] = {};
        if (it.there) {
            const uint32_t* unit = reinterpret_cast<const uint32_t*>(P.cache.kq + it.begin * Row::kBytes + Row::key(it.pos, b, g));
            const float d = (float)P.cache.ks[(it.begin + it.pos) * Row::kBlocks + b];
            const uint32_t w = QT == IZWI_KV_Q8_0 ? unit[second] : unit[0] >> (8 * second);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int q = QT == IZWI_KV_Q8_0 ? (int)(w >> (8 * i) & 255) : (int)(w >> (16 * (i & 1) + 4 * (i >> 1)) & 15);
                v[i] = d * (float)(q - kBias);
            }
        }
        store_values<T, 4, VEC>(static_cast<T*>(P.k_out) + ((int64_t)it.row * P.kv_heads + it.head) * D + e, v);
        return;
    }
    const unsigned thread = (blockIdx.x - P.k_blocks) * 256 + threadIdx.x, item = thread / 16;
    if (item >= P.rows) return;
    const int x = threadIdx.x & 15;
    const KvItem it = kv_item<true>(P, item);
    T* dst = static_cast<T*>(P.v_out) + ((int64_t)it.row * P.kv_heads + it.head) * D + 2 * x;
    uint16_t half[Row::kLane / 2];
    f16_t d[Row::kBlocks];
#pragma unroll
    for (int j = 0; j < Row::kLane / 2; j++) half[j] = *reinterpret_cast<const uint16_t*>(P.cache.vq + it.begin * Row::kBytes + Row::value(it.pos, x, j));
#pragma unroll
    for (int b = 0; b < Row::kBlocks; b++) d[b] = P.cache.vs[it.begin * Row::kBlocks + Row::value_scale(it.pos, b)];
#pragma unroll
    for (int b = 0; b < Row::kBlocks; b++) {
        const int q = QT == IZWI_KV_Q8_0 ? half[b] : half[b / 2] >> (8 * (b & 1)) & 255;
        const int q0 = QT == IZWI_KV_Q8_0 ? q & 255 : q & 15, q1 = QT == IZWI_KV_Q8_0 ? q >> 8 : q >> 4;
        const float v[2] = {it.there ? (float)d[b] * (float)(q0 - kBias) : 0.0f, it.there ? (float)d[b] * (float)(q1 - kBias) : 0.0f};
        store_values<T, 2, VEC>(dst + 32 * b, v);
    }
}

// The row at a time where sixteen positions would be half empty or more, and for calls that are too small to fill the card with
// waves of sixteen.  Both sides, 8 heads of 128, Q8_0 and f32: one token of one sequence 2.7 us instead of 4.6 to write, 2.2 instead of 3.1
// to read; 8 tokens of 256 sequences 8.3 instead of 11.7, and 9.0 instead of 12; 16 of 256: 13.5 instead of 12.6, and 14 instead of 13.  256
// tokens of one sequence 3.5 instead of 3.9 to write, 2048 of one 8.3 instead of 5.7; 16 of 64 sequences 4.5 instead of 5.9 to read, 256
// of 8: 7.8 instead of 6.9.
constexpr unsigned kFewTokens = 8;
template <bool READ>
bool by_row(const KvRowsParams& P, int64_t d) {
    const int64_t values = P.rows * d;
    return values <= (READ ? 1 << 20 : 1 << 18) || (P.tokens <= kFewTokens && values <= 1 << 30);
}

template <typename T, int QT, int D, bool READ>
hipError_t launch_rows(const KvRowsParams& P0, bool vec, hipStream_t stream) {
    KvRowsParams P = P0;
    if (by_row<READ>(P, D)) {
        P.k_blocks = (unsigned)(((uint64_t)P.rows * (D / 4) + 255) / 256);
        const unsigned blocks = P.k_blocks + (unsigned)(((uint64_t)P.rows * 16 + 255) / 256);
        if constexpr (READ) {
            if (vec) kv_read_rows_kernel<T, QT, D, true><<<blocks, 256, 0, stream>>>(P);
            else kv_read_rows_kernel<T, QT, D, false><<<blocks, 256, 0, stream>>>(P);
        } else {
            if (vec) kv_append_rows_kernel<T, QT, D, true><<<blocks, 256, 0, stream>>>(P);
            else kv_append_rows_kernel<T, QT, D, false><<<blocks, 256, 0, stream>>>(P);
        }
        return hipGetLastError();
    }
    P.k_blocks = (P.items + 3) / 4;
    const unsigned blocks = 2 * P.k_blocks;
    if constexpr (READ) {
        if (vec) kv_read_kernel<T, QT, D, true><<<blocks, 256, 0, stream>>>(P);
        else kv_read_kernel<T, QT, D, false><<<blocks, 256, 0, stream>>>(P);
    } else {
        if (vec) kv_append_kernel<T, QT, D, true><<<blocks, 256, 0, stream>>>(P);
        else kv_append_kernel<T, QT, D, false><<<blocks, 256, 0, stream>>>(P);
    }
    return hipGetLastError();
}
template <typename T, bool READ>
hipError_t launch_rows_of(int type, int64_t d, const KvRowsParams& P, bool vec, hipStream_t stream) {
    if (type == IZWI_KV_Q8_0)
        return d == 64    ? launch_rows<T, IZWI_KV_Q8_0, 64, READ>(P, vec, stream)
               : d == 128 ? launch_rows<T, IZWI_KV_Q8_0, 128, READ>(P, vec, stream)
                          : launch_rows<T, IZWI_KV_Q8_0, 256, READ>(P, vec, stream);
    return d == 64    ? launch_rows<T, IZWI_KV_Q4_0, 64, READ>(P, vec, stream)
           : d == 128 ? launch_rows<T, IZWI_KV_Q4_0, 128, READ>(P, vec, stream)
                      : launch_rows<T, IZWI_KV_Q4_0, 256, READ>(P, vec, stream);
}

int check_rows(const char* what, const int32_t* starts, int64_t batch, int64_t tokens, int64_t first_slot, int64_t slots, int64_t kv_heads,
               int64_t d, const void* cache, const void* k, const void* v) {
    if (batch < 0 || tokens < 0 || first_slot < 0 || batch > slots || first_slot > slots - batch || tokens > 0x7fffffff)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: sequences %lld of %lld tokens at slot %lld of %lld", what, (long long)batch, (long long)tokens,
                        (long long)first_slot, (long long)slots);
    if (batch && tokens && batch * ((tokens + 30) / 16) > 0xffffff / kv_heads) // (threads stay below 2^32)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: more than 2^24 groups of sixteen rows in a call", what);
    if (!cache || !kv_aligned(cache, 16)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: the cache must be a 16-byte aligned buffer", what);
    if (batch && tokens && (!starts || !k || !v)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: NULL buffer", what);
    return IZWI_QMM_OK;
}

template <typename T>
int kv_append_impl(int type, const T* k, const T* v, int64_t k_stride, int64_t v_stride, const int32_t* starts, const int32_t* counts, int64_t batch,
                   int64_t tokens, int64_t first_slot, int64_t slots, int64_t kv_heads, int64_t capacity, int64_t d, void* cache, void* stream) {
    constexpr const char* what = "decode_kv_append";
    if (int rc = kv_check_shape(what, type, slots, kv_heads, capacity, d)) return rc;
    if (int rc = check_rows(what, starts, batch, tokens, first_slot, slots, kv_heads, d, cache, k, v)) return rc;
    if (k_stride < kv_heads * d || v_stride < kv_heads * d)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: row strides %lld and %lld for rows of %lld values", what, (long long)k_stride, (long long)v_stride,
                        (long long)(kv_heads * d));
    if (!batch || !tokens) return IZWI_QMM_OK;
    int device = 0, n_cus = 0;
    if (int rc = qmm_current_device(&device, &n_cus)) return rc;
    KvRowsParams P{};
    P.k_in = k, P.v_in = v, P.k_stride = k_stride, P.v_stride = v_stride;
    P.cache = kv_planes(type, cache, slots, kv_heads, capacity, d);
    P.starts = starts, P.counts = counts, P.tokens = (unsigned)tokens, P.kv_heads = (unsigned)kv_heads;
    P.groups = (unsigned)((tokens + 30) / 16), P.items = (unsigned)(batch * P.groups * kv_heads);
    P.rows = (unsigned)(batch * tokens * kv_heads), P.first_slot = (int)first_slot, P.capacity = capacity;
    // (four values a load of the keys, two of the values)
    const bool vec = kv_aligned(k, 4 * sizeof(T)) && k_stride % 4 == 0 && kv_aligned(v, 2 * sizeof(T)) && v_stride % 2 == 0;
    KV_TRY((launch_rows_of<T, false>(type, d, P, vec, (hipStream_t)stream)));
    return IZWI_QMM_OK;
}

template <typename T>
int kv_read_impl(int type, const void* cache, int64_t slots, int64_t kv_heads, int64_t capacity, int64_t d, const uint8_t* lineage, int64_t beams,
                 const int32_t* starts, const int32_t* counts, int64_t batch, int64_t tokens, int64_t first_slot, T* k, T* v, void* stream) {
    constexpr const char* what = "decode_kv_read";
    if (int rc = kv_check_shape(what, type, slots, kv_heads, capacity, d)) return rc;
    if (int rc = check_rows(what, starts, batch, tokens, first_slot, slots, kv_heads, d, cache, k, v)) return rc;
    if (lineage && (beams <= 0 || beams > 255 || slots % beams))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: lineage of %lld beams in %lld slots", what, (long long)beams, (long long)slots);
    if (!batch || !tokens) return IZWI_QMM_OK;
    int device = 0, n_cus = 0;
    if (int rc = qmm_current_device(&device, &n_cus)) return rc;
    KvRowsParams P{};
    P.k_out = k, P.v_out = v;
    P.cache = kv_planes(type, cache, slots, kv_heads, capacity, d);
    P.lineage = lineage, P.beams = lineage ? (int)beams : 1;
    P.starts = starts, P.counts = counts, P.tokens = (unsigned)tokens, P.kv_heads = (unsigned)kv_heads;
    P.groups = (unsigned)((tokens + 30) / 16), P.items = (unsigned)(batch * P.groups * kv_heads);
    P.rows = (unsigned)(batch * tokens * kv_heads), P.first_slot = (int)first_slot, P.capacity = capacity;
    const bool vec = kv_aligned(k, 4 * sizeof(T)) && kv_aligned(v, 2 * sizeof(T));
    KV_TRY((launch_rows_of<T, true>(type, d, P, vec, (hipStream_t)stream)));
    return IZWI_QMM_OK;
}

} // namespace

extern "C" {

uint64_t izwi_decode_kv_cache_bytes(int type, int64_t slots, int64_t kv_heads, int64_t capacity, int64_t head_dim) {
    if (kv_check_shape("decode_kv_cache_bytes", type, slots, kv_heads, capacity, head_dim)) return 0;
    const int64_t rows = slots * kv_heads * kv_padded(capacity);
    return 2 * (uint64_t)(kv_plane_bytes(rows, kv_row_bytes(type, head_dim)) + kv_plane_bytes(rows, head_dim / 16));
}

int izwi_decode_kv_append_f32(int type, const float* k, const float* v, int64_t k_stride, int64_t v_stride, const int32_t* starts,
                              const int32_t* counts, int64_t batch, int64_t tokens, int64_t first_slot, int64_t slots, int64_t num_kv_heads,
                              int64_t kv_capacity, int64_t head_dim, void* cache, void* stream) {
    return qmm_guarded("izwi_decode_kv_append_f32", [&]() -> int {
    return kv_append_impl<float>(type, k, v, k_stride, v_stride, starts, counts, batch, tokens, first_slot, slots, num_kv_heads, kv_capacity, head_dim,
                                 cache, stream);
    });
}
int izwi_decode_kv_append_f16(int type, const uint16_t* k, const uint16_t* v, int64_t k_stride, int64_t v_stride, const int32_t* starts,
                              const int32_t* counts, int64_t batch, int64_t tokens, int64_t first_slot, int64_t slots, int64_t num_kv_heads,
                              int64_t kv_capacity, int64_t head_dim, void* cache, void* stream) {
    return qmm_guarded("izwi_decode_kv_append_f16", [&]() -> int {
    return kv_append_impl<f16_t>(type, (const f16_t*)k, (const f16_t*)v, k_stride, v_stride, starts, counts, batch, tokens, first_slot, slots,
                                 num_kv_heads, kv_capacity, head_dim, cache, stream);
    });
}

int izwi_decode_kv_read_f32(int type, const void* cache, int64_t slots, int64_t num_kv_heads, int64_t kv_capacity, int64_t head_dim,
                            const uint8_t* lineage, int64_t beams, const int32_t* starts, const int32_t* counts, int64_t batch, int64_t tokens,
                            int64_t first_slot, float* k, float* v, void* stream) {
    return qmm_guarded("izwi_decode_kv_read_f32", [&]() -> int {
    return kv_read_impl<float>(type, cache, slots, num_kv_heads, kv_capacity, head_dim, lineage, beams, starts, counts, batch, tokens, first_slot, k, v,
                               stream);
    });
}
int izwi_decode_kv_read_f16(int type, const void* cache, int64_t slots, int64_t num_kv_heads, int64_t kv_capacity, int64_t head_dim,
                            const uint8_t* lineage, int64_t beams, const int32_t* starts, const int32_t* counts, int64_t batch, int64_t tokens,
                            int64_t first_slot, uint16_t* k, uint16_t* v, void* stream) {
    return qmm_guarded("izwi_decode_kv_read_f16", [&]() -> int {
    return kv_read_impl<f16_t>(type, cache, slots, num_kv_heads, kv_capacity, head_dim, lineage, beams, starts, counts, batch, tokens, first_slot,
                               (f16_t*)k, (f16_t*)v, stream);
    });
}

} // extern "C"
