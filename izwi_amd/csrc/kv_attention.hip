// Attention of one new token per sequence over the quantized cache (layout: kv_cache.h): positions that the sequences of a
// prompt share, then each sequence's own.
//
// One pass over the positions with a running maximum and sum per query row.  A workgroup has a tile of query rows (heads of one kv
// head, of all sequences of a prompt where the positions are shared) and a split of the positions; its waves take 32 positions
// in turn and meet in LDS, the splits in a second small kernel.  Both products run on the matrix cores, 16 x 16 x 32 in f16 with f32
// sums, and both with the query row as the column: what a lane holds of the scores (row x, positions 4 g .. 4 g + 3 of 16) is
// what it feeds to the second product, and a row's statistics stay in its lanes.
//  * Quants are exact in f16 (one byte permute and one subtraction for two of them).  A block of 32 is the depth of one matrix
//    instruction, so the keys' scales multiply finished sums in f32.  The values' scales run along the positions, over which the
//    second product sums: they multiply the weights, once for each block of 32 elements of the head.
//  * f32 queries and the weights go as two f16 numbers each, 22 bits: with the quants exact, two matrix products instead of one.
//    Queries are scaled by a power of two per row.  Weights stand under a reference that keeps the largest between 2^12 and 2^15.5 (it moves
//    when a score rises by a factor of 11: rarely, so most tiles pay for no rescaling): a weight is right to 2^-22 of itself or 2^-37 of the
//    largest, where the second number ends, whichever is more, so that many positions far below a few that dominate keep their sum.  (With the
//    largest between 2^5 and 2^15, which moves even less, 2^15 positions that have 2^-13 to 2^-27 of four others' weight each came out up to
//    28 % of their sum wrong, now 0.3 %, 2^-22 of the whole; moving costs some 2 % where many rows share positions.)  The values' scales stand under the power
//    of two that takes the largest of their block of the head and of the 32 positions to below 1, where those between 2^-12 and 1 of the last one
//    keep it: a scale is exact down to 2^-14 of the largest there, and off by 2^-25 of it below that.  (A power of two that never fell again let a single
//    large value cost all that follow their bits; looking for one costs 1 % where little is to do: 300 positions 6.8 us, not 6.7.)  Weight times scale is a product of f16 pairs whose loss
//    a fused multiply-add returns exactly: packed, half the instructions of f32 products split afterwards.
//    f16 queries are themselves.  (Weights of f16 results as single f16 numbers, rounded to f16 and once more under the scale, left 2.8e-4 of a
//    result where its own rounding leaves 2.1e-4, and far more where values cancel.)
//
// Bound by memory where few rows share positions: 32 sequences of 4001 positions of 32 heads on 8, D = 128, Q8_0, 40 us in a graph, 5.5 TB/s.
// By the issue of vector instructions around the matrix products where many do (per tile of 32 positions and 32 f32 rows about 500 beside 64
// matrix instructions, as fast with one wave on a SIMD as with two): 64 rows a kv head on 131072 positions 108 to 115 us, 2.6 TB/s and
// 310 TFLOP/s; 256 f16 rows a kv head on 8192 positions and 250 own of each sequence, Q4_0, 34 us, 250 TFLOP/s.  By two launches and the way to
// memory and back where there is little to do: 8 beams behind 1501 positions 9.3 us; by one and a workgroup's chain of loads: 300 positions of one
// sequence 6.8.
// Two row tiles a workgroup halve the conversions (65 -> 53 us at 64 rows a kv head on 60000 positions); four do not fit the registers.
#include "kv_cache.h"

#include <algorithm>
#include <cmath>

#include "qmm_lanes.h"

namespace {

typedef _Float16 f16_t;

typedef f16_t h2 __attribute__((ext_vector_type(2)));
typedef f16_t h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

// n / d for 0 <= n < 2^31 as a product: with s = ceil(log2 d) and m = floor(2^(31 + s) / d) + 1, the error of m n / 2^(31 + s) is
// below 1 / d.  (The compiler's divisions by arguments were most of the 1500 cycles before a workgroup's first load.)
struct Divisor {
    uint32_t d, m, s;
    Divisor() = default;
    explicit Divisor(int64_t by) : d((uint32_t)by), s(0) {
        while ((int64_t(1) << s) < by) s++;
        m = (uint32_t)(((uint64_t(1) << (31 + s)) / (uint64_t)by + 1));
    }
    __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n << 1, m) >> s); }
};

struct AttendParams {
    const void* q;
    void* out;
    int64_t q_stride;
    KvPlanes prefix, own;
    const int32_t* prefix_lens; // [prompts]
    const int32_t* lens;        // [batch]
    const uint8_t* lineage;
    int batch, beams, heads, kv_heads, group;
    int max_prefix, max_len; // 0: no such positions
    float scale;
    // workgroups: prefix_wgs of prefix_units (prompt, kv head, split) times prefix_z tiles of rows, then the same of (sequence, ..)
    int prefix_splits, prefix_units, prefix_z, prefix_wgs, own_splits, own_units, own_z, own_solo;
    Divisor by_group, by_kv_heads, by_beams, by_prefix_splits, by_own_splits, by_prefix_z, by_own_z;
    int parts;     // partial results of a row: prefix_splits + own_splits
    float* sums;   // [batch * heads][parts][D]
    float2* stats; // [batch * heads][parts]: reference (a power of two's exponent), sum of weights; (-infinity, 0) without a position, NaN with a score that is none
};

__device__ __forceinline__ int clamped_len(const int32_t* lens, int i, int most) { return most ? max(0, min(lens[i], most)) : 0; }

template <int N>
struct Words {
    uint32_t w[N];
    __device__ __forceinline__ void load(const void* p) {
        __builtin_memcpy(w, __builtin_assume_aligned(p, N % 4 == 0 ? 16 : 4 * N), 4 * N);
    }
};

// Two unsigned quants under the exponent of 1024, less 1024 and the bias: exact
__device__ __forceinline__ h2 as_h2(uint32_t w) { return __builtin_bit_cast(h2, w); }
__device__ __forceinline__ h2 bytes_less_128(uint32_t w) { return as_h2(w) + h2{(f16_t)-1152.0f, (f16_t)-1152.0f}; }
__device__ __forceinline__ h2 low_nibbles(uint32_t w, uint32_t e) { // of bits 0-3 and 16-19
    return as_h2((w & 0x000f000fu) | e) + h2{(f16_t)-1032.0f, (f16_t)-1032.0f};
}
__device__ __forceinline__ h2 high_nibbles(uint32_t w, uint32_t e) { // of bits 4-7 and 20-23: 1024 + 16 n, so a sixteenth less 64 + 8
    return __builtin_elementwise_fma(as_h2((w & 0x00f000f0u) | e), h2{(f16_t)0.0625f, (f16_t)0.0625f}, h2{(f16_t)-72.0f, (f16_t)-72.0f});
}
typedef unsigned short u2 __attribute__((ext_vector_type(2)));
template <int QT> // of two scales, as bits; those of Q8_0 have no sign
__device__ __forceinline__ u2 magnitudes(uint32_t w) { return __builtin_bit_cast(u2, QT == IZWI_KV_Q8_0 ? w : w & 0x7fff7fffu); }
__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) { return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]}; }

// The exponent of 1024 for bytes, or for the halves of a word, in a vector register: mask and exponent of a nibble are one instruction only if
// no more than one of them is a scalar
template <int QT>
__device__ __forceinline__ uint32_t exponents() {
    uint32_t e = QT == IZWI_KV_Q8_0 ? 0x64646464u : 0x64006400u;
    if constexpr (QT != IZWI_KV_Q8_0) asm volatile("" : "+v"(e));
    return e;
}
// The eight keys' values of a unit
template <int QT>
__device__ __forceinline__ h8 key_unit(const uint32_t* w, uint32_t e) {
    if constexpr (QT == IZWI_KV_Q8_0) {
        return join(bytes_less_128(__builtin_amdgcn_perm(e, w[0], 0x04010400u)), bytes_less_128(__builtin_amdgcn_perm(e, w[0], 0x04030402u)),
                    bytes_less_128(__builtin_amdgcn_perm(e, w[1], 0x04010400u)), bytes_less_128(__builtin_amdgcn_perm(e, w[1], 0x04030402u)));
    } else {
        const uint32_t u = w[0] >> 8;
        return join(low_nibbles(w[0], e), high_nibbles(w[0], e), low_nibbles(u, e), high_nibbles(u, e));
    }
}

// Of block b the values 2 x (first) and 2 x + 1 at eight positions: v[h] are the lane's quants of four positions, dwords of two
template <int QT, int N>
__device__ __forceinline__ void value_pair(const Words<N> (&v)[2], int b, uint32_t e, h8& first, h8& second) {
    h2 lo[4], hi[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if constexpr (QT == IZWI_KV_Q8_0) {
            const uint32_t w = v[r >> 1].w[(r & 1) * (N / 2) + b];
            lo[r] = bytes_less_128(__builtin_amdgcn_perm(e, w, 0x04020400u));
            hi[r] = bytes_less_128(__builtin_amdgcn_perm(e, w, 0x04030401u));
        } else {
            const uint32_t w = v[r >> 1].w[(r & 1) * (N / 2) + b / 2] >> (8 * (b & 1));
            lo[r] = low_nibbles(w, e);
            hi[r] = high_nibbles(w, e);
        }
    }
    first = join(lo[0], lo[1], lo[2], lo[3]);
    second = join(hi[0], hi[1], hi[2], hi[3]);
}

constexpr int kWaves = 4; // of a workgroup
constexpr float kRise = 3.5f, kHead = 12.0f; // powers of two, see above

template <typename T, int QT, int D, int RT, bool SHARED, bool LIN, bool SOLO = false>
__device__ __forceinline__ void attend_rows(const AttendParams& P, int id, float* lds) {
    using Row = KvRow<QT, D>;
    constexpr int NB = Row::kBlocks, KW = Row::kBytes / 16, VW = Row::kLane, ROWS = 16 * RT;
    // TWO: two tiles in registers.  Not where they do not fit beside the rest: with heads of 256 the second one leaves a SIMD one wave instead
    // of two or moves values to and fro (88 sequences of 64 heads on 8, f16 and Q4_0, 818 positions and 29 own: 49 us with it, 38 without; f32 and
    // Q8_0 57 and 53).
    constexpr bool SPLIT = sizeof(T) == 4, TWO = RT == 1 && !LIN && D <= 128;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = lane & 15, g = lane >> 4;
    // SOLO: every wave has a unit of its own, and nothing to meet for
    constexpr int kStep = SOLO ? 1 : kWaves;

    // what this workgroup (wave) works on
    const int Z = SHARED ? P.prefix_z : P.own_z, splits = SHARED ? P.prefix_splits : P.own_splits;
    int unit, z;
    if constexpr (SOLO) {
        const int n = id * kWaves + wave;
        unit = P.by_own_z.of(n), z = n - unit * Z;
    } else { // tiles of the same positions on one XCD
        const int eighth = (SHARED ? P.by_prefix_z : P.by_own_z).of(id >> 3);
        unit = eighth * 8 + (id & 7), z = (id >> 3) - eighth * Z;
    }
    if (unit >= (SHARED ? P.prefix_units : P.own_units)) return;
    const int of_split = (SHARED ? P.by_prefix_splits : P.by_own_splits).of(unit), split = unit - of_split * splits;
    const int seq = P.by_kv_heads.of(of_split), kvh = of_split - seq * P.kv_heads;
    const KvPlanes& C = SHARED ? P.prefix : P.own;
    const int len = SHARED ? clamped_len(P.prefix_lens, seq, P.max_prefix) : clamped_len(P.lens, seq, P.max_len);
    const int n_rows = SHARED ? P.beams * P.group : P.group, b0 = SHARED ? seq * P.beams : seq;
    const int part = SHARED ? split : P.prefix_splits + split;
    const int tiles = (len + 31) / 32, share = (SHARED ? P.by_prefix_splits : P.by_own_splits).of(tiles + splits - 1), first = split * share, last = min(tiles, first + share);
    auto row_index = [&](int r) { // of out, sums and stats
        const int n = z * ROWS + r, s = P.by_group.of(n);
        return (int64_t)(b0 + s) * P.heads + kvh * P.group + (n - s * P.group);
    };
    const int rows_here = min(ROWS, n_rows - z * ROWS);
    if (first >= last) { // nothing to add
        const int me = SOLO ? lane : threadIdx.x;
        if (P.parts == 1) {
            for (int i = me; i < rows_here * D; i += 64 * kStep) static_cast<T*>(P.out)[row_index(i / D) * D + i % D] = (T)0.0f;
        } else if (me < rows_here) {
            P.stats[row_index(me) * P.parts + part] = make_float2(-INFINITY, 0.0f);
        }
        return;
    }

    // A tile of 32 positions as this lane holds it: its key row and the values of its four positions, of each half; of the scales,
    // of keys words of one position, SL lanes a position (lane (h * 4 + i) * SL .. of the sixteen has those of position 16 h + 4 g + i), of
    // values a word per block for two positions, VL lanes a pair (lane (h * 2 + i) * VL .. has those of positions 16 h + 4 g + 2 i and the next)
    constexpr int SW = NB > 4 ? NB / 4 : 1, SL = NB / 2 / SW, VL = NB / SW;
    struct Keys {
        Words<KW> k[2];
        Words<SW> s;
    };
    struct Values {
        Words<VW> v[2];
        Words<LIN ? VW : 1> w[2]; // (LIN) those of the odd positions; v has the even ones'
    };
    struct Scales {
        Words<SW> s;
        Words<LIN ? SW : 1> w;  // (LIN) that of the odd position; s has the even one's
        uint32_t beam, beams[2]; // (LIN) of the two positions whose scales are here, of its four positions of each half
    };
    const int64_t begin = ((int64_t)(LIN ? P.by_beams.of(seq) * P.beams : seq) * C.kv_heads + kvh) * C.padded, step = C.kv_heads * C.padded;
    const int s_index = x / SL & 7, s_pos = 16 * (s_index >> 2) + 4 * g + (s_index & 3);
    const int v_index = x / VL & 3, v_pos = 16 * (v_index >> 1) + 4 * g + 2 * (v_index & 1);
    const uint8_t* lineage = LIN ? P.lineage + (int64_t)seq * C.padded : nullptr;
    uint32_t kb[2] = {}, vb[2] = {}, sb = 0, wb = 0; // (LIN) beams of the lane's key rows, of its positions, of its keys' and values' scales in the tile loaded next
    auto load_lineage = [&](int tile) {
        if constexpr (LIN) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                kb[t] = lineage[tile * 32 + 16 * t + x];
                vb[t] = *reinterpret_cast<const uint32_t*>(lineage + tile * 32 + 16 * t + 4 * g);
            }
            sb = lineage[tile * 32 + s_pos];
            wb = *reinterpret_cast<const uint16_t*>(lineage + tile * 32 + v_pos);
        }
    };
    auto beam_at = [&](uint32_t beam) -> int64_t { return LIN ? (int64_t)(beam < (uint32_t)P.beams ? beam : 0) * step : 0; };
    // (without lineage: uniform bases, 32-bit offsets of the lane)
    auto load_keys = [&](Keys& t, Scales& sc, int tile) {
        const int64_t at = begin + (int64_t)tile * 32;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint8_t* p = C.kq + (at + 16 * h) * Row::kBytes + (unsigned)(lane * Row::kPiece);
            if constexpr (LIN) p += beam_at(kb[h]) * Row::kBytes;
#pragma unroll
            for (int i = 0; i < Row::kBlocks / Row::kPer; i++)
                reinterpret_cast<Words<Row::kPiece / 4>*>(t.k[h].w)[i].load(p + 64 * Row::kPiece * i);
        }
        t.s.load(C.ks + (at + (LIN ? beam_at(sb) : 0)) * NB + (unsigned)(s_pos * NB + x % SL * (2 * SW)));
        const f16_t* vs = C.vs + at * NB + (unsigned)(v_pos * NB + x % VL * (2 * SW));
        if constexpr (LIN) {
            sc.s.load(vs + beam_at(wb & 255) * NB);
            sc.w.load(vs + beam_at(wb >> 8) * NB);
            sc.beam = wb, sc.beams[0] = vb[0], sc.beams[1] = vb[1];
        } else {
            sc.s.load(vs);
        }
    };
    auto load_values = [&](Values& t, const Scales& sc, int tile) {
        constexpr int U = Row::kValuePiece, W = U / 4;
        const int64_t at = begin + (int64_t)tile * 32;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint8_t* p = C.vq + (at + 16 * h) * Row::kBytes + (unsigned)(g * 4 * Row::kBytes + x * U);
            if constexpr (!LIN) {
#pragma unroll
                for (int i = 0; i < VW / W; i++) reinterpret_cast<Words<W>*>(t.v[h].w)[i].load(p + 16 * U * i);
            } else { // every position from its own beam, a pair of positions at a time
                constexpr int PW = VW / 2 < W ? VW / 2 : W; // words of a load
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint8_t* pi = p + beam_at(sc.beams[h] >> (8 * i) & 255) * Row::kBytes;
                    uint32_t* w = (i & 1 ? t.w[h].w : t.v[h].w) + (i >> 1) * (VW / 2);
#pragma unroll
                    for (int n = 0; n < VW / 2 / PW; n++) {
                        const int word = (i >> 1) * (VW / 2) + n * PW;
                        reinterpret_cast<Words<PW>*>(w)[n].load(pi + word / W * (16 * U) + word % W * 4);
                    }
                }
            }
        }
    };
    Keys keys[TWO ? 2 : 1];
    Values vals[TWO ? 2 : 1];
    Scales scales[2];
    int tile = first + (SOLO ? 0 : wave);
    const bool any = tile < last;
    if (any) {
        load_lineage(tile);
        load_keys(keys[0], scales[0], tile);
        load_values(vals[0], scales[0], tile);
        load_lineage(min(tile + kStep, last - 1));
    }

    // The queries: lane (x, g) holds of row x the values 8 g .. of every block.  f32 ones are scaled by a power of two to
    // below 2^14 and split.  The sign of the scale goes to them, so that the largest score is the largest product.
    h8 qh[RT][NB], ql[SPLIT ? RT : 1][SPLIT ? NB : 1];
    // What makes scores (in powers of two) of products.  A product of numbers is below 2^47 (queries 2^16, quants 2^7, scales 2^16, a head 2^8) and
    // two that differ do by 2^-48 or more, so a factor above 2^80 makes a weight of one of the largest and zero of the others whatever it is: with
    // 2^80 instead no score is beyond f32.
    constexpr float kMostFactor = 0x1p80f;
    float factor[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const T* q;
        {
            const int n = z * ROWS + min(16 * rt + x, rows_here - 1), s = P.by_group.of(n);
            q = static_cast<const T*>(P.q) + (b0 + s) * P.q_stride + (int64_t)(kvh * P.group + (n - s * P.group)) * D + 8 * g;
        }
        float f[NB][8], by = P.scale < 0.0f ? -1.0f : 1.0f;
        factor[rt] = fmaxf(fabsf(P.scale) * 1.44269504088896340736f, 1e-37f);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 8; j++) f[b][j] = (float)q[32 * b + j];
        float most = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(f[b][j]));
        if constexpr (!SPLIT) { // an infinity among the queries leaves no number (f32: infinity less infinity in the split)
            if (most == INFINITY) by = NAN;
        } else {
            most = qmm_max_lane_rows(most);
            // (an infinity or a subnormal gets some power or other)
            const int up = max(-113, min(113, 140 - (int)(__float_as_uint(most) >> 23)));
            by *= __uint_as_float((uint32_t)(127 + up) << 23);
            factor[rt] = fmaxf(factor[rt] * __uint_as_float((uint32_t)(127 - up) << 23), 1e-37f);
        }
        factor[rt] = fminf(factor[rt], kMostFactor);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            h8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = f[b][j] * by;
                hi[j] = (f16_t)y;
                lo[j] = (f16_t)(y - (float)hi[j]);
            }
            qh[rt][b] = hi;
            if constexpr (SPLIT) ql[rt][b] = lo;
        }
    }

    // of the lane's row: the maximum that the reference stands on, the product that makes a new one, the reference, this lane's sum of weights
    float top[RT], bar[RT], ref[RT], l[RT];
    f4 o[RT][2 * NB];
    // Of each block of the head: what its value scales are multiplied by, the power of two that takes the largest of a tile to below 1 (2^15 at
    // most).  A lane has it for the blocks of its value scales, and as f16 bits which scales need another: at or above 1 / it, or (less one) below
    // 2^-12 of that.
    float up[SW];
    uint32_t over[SW], under[SW];
    auto two_to = [](int n) { return __uint_as_float((uint32_t)(127 + n) << 23); };
    auto set_up = [&](int i, int n) { // 2^n
        up[i] = two_to(n);
        over[i] = __builtin_bit_cast(uint16_t, (f16_t)two_to(-n)); // (2^16: infinity's)
        under[i] = max(1u, (uint32_t)__builtin_bit_cast(uint16_t, (f16_t)two_to(-12 - n))) - 1;
    };
    auto up_of = [&](auto b) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(up[b % SW]), b / SW)); };
#pragma unroll
    for (int i = 0; i < SW; i++) set_up(i, 15);
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        top[rt] = bar[rt] = ref[rt] = -INFINITY, l[rt] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) o[rt][i] = f4{0, 0, 0, 0};
    }
    float s[RT][8];
    const uint32_t e1024 = exponents<QT>();
    // products of queries and keys, a block of the head at a time under its scale
    auto scores = [&](const Keys& t) {
        float d[2 * SW]; // the lane's scales, to be handed round
#pragma unroll
        for (int i = 0; i < 2 * SW; i++) d[i] = (float)as_h2(t.s.w[i / 2])[i & 1];
        each<NB>([&](auto b) {
            h8 a[2];
#pragma unroll
            for (int h = 0; h < 2; h++) a[h] = key_unit<QT>(t.k[h].w + b * (Row::kUnit / 4), e1024);
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                f4 acc[2];
#pragma unroll
                for (int h = 0; h < 2; h++) acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[h], qh[rt][b], f4{0, 0, 0, 0}, 0, 0, 0);
                if constexpr (SPLIT)
#pragma unroll
                    for (int h = 0; h < 2; h++) acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[h], ql[rt][b], acc[h], 0, 0, 0);
                each<8>([&](auto j) {
                    const float by = __uint_as_float(of_lane<j * SL + b / 2 / SW>(__float_as_uint(d[b / 2 % SW * 2 + (b & 1)])));
                    s[rt][j] = b == 0 ? by * acc[j >> 2][j & 3] : __builtin_fmaf(by, acc[j >> 2][j & 3], s[rt][j]);
                });
            }
        });
    };
    auto weights = [&](Scales& t, int at) {
        // positions behind the end, or of no beam: no weight, and a scale that is a number
        if (LIN || at * 32 + 32 > len) {
            asm volatile(""); // (a branch: without it every tile pays for the selections)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                bool gone = at * 32 + 16 * (j >> 2) + 4 * g + (j & 3) >= len;
                if constexpr (LIN) gone |= (t.beams[j >> 2] >> (8 * (j & 3)) & 255) >= (uint32_t)P.beams;
#pragma unroll
                for (int rt = 0; rt < RT; rt++) s[rt][j] = gone ? -INFINITY : s[rt][j];
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                bool gone = at * 32 + v_pos + i >= len;
                if constexpr (LIN) gone |= (t.beam >> (8 * i) & 255) >= (uint32_t)P.beams;
#pragma unroll
                for (int n = 0; n < SW; n++) {
                    if constexpr (LIN) if (i == 0) t.s.w[n] = (t.s.w[n] & 0xffffu) | (t.w.w[n] & 0xffff0000u);
                    t.s.w[n] &= gone ? 0xffffu << (16 * (1 - i)) : ~0u;
                }
            }
        }
        // does a row's maximum rise, or do the values' scales leave the range of their power of two?
        bool rise[RT], any_rise = false, odd = false;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float m = s[rt][0];
#pragma unroll
            for (int j = 1; j < 8; j++) m = fmaxf(m, s[rt][j]);
            rise[rt] = m > bar[rt], any_rise |= rise[rt];
        }
#pragma unroll
        for (int i = 0; i < SW; i++) {
            const u2 size = magnitudes<QT>(t.s.w[i]), less_one = size - u2{1, 1}; // (a scale of zero is not a small one)
            odd |= max((uint32_t)size[0], (uint32_t)size[1]) >= over[i] || min((uint32_t)less_one[0], (uint32_t)less_one[1]) < under[i];
        }
        if (__any(any_rise || odd)) {
            bool begun = false; // (before a row has a reference there is nothing to rescale)
#pragma unroll
            for (int rt = 0; rt < RT; rt++) begun |= ref[rt] != -INFINITY;
            begun = __any(begun);
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                if (!__any(rise[rt])) continue;
                float m = s[rt][0];
#pragma unroll
                for (int j = 1; j < 8; j++) m = fmaxf(m, s[rt][j]);
                top[rt] = fmaxf(top[rt], qmm_max_lane_rows(m) * factor[rt]);
                bar[rt] = (top[rt] + (kRise - fabsf(top[rt]) * 0x1p-22f)) / factor[rt]; // (less what rounding may add)
                // (from 2^24 on scores are whole numbers two or more apart, and a reference rounded further up would take a weight beyond f16)
                const float to = fabsf(top[rt]) < 0x1p24f ? top[rt] - kHead : top[rt], by = ref[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ref[rt] - to);
                ref[rt] = to, l[rt] *= by;
                if (begun)
#pragma unroll
                    for (int i = 0; i < 2 * NB; i++) o[rt][i] *= by;
            }
            if (__any(odd)) {
                float down[SW]; // of what is there
#pragma unroll
                for (int i = 0; i < SW; i++) {
                    const h2 two = __builtin_bit_cast(h2, magnitudes<QT>(t.s.w[i]));
                    float d = fmaxf(0.0f, fmaxf((float)two[0], (float)two[1])); // (passes over the NaN of a block that holds one)
                    d = fmaxf(d, dpp_f<0x128>(d)); // over the lanes x that have this block: row_ror 8, 4 (and 2)
                    d = fmaxf(d, dpp_f<0x124>(d));
                    if constexpr (VL == 2) d = fmaxf(d, dpp_f<0x122>(d));
                    d = qmm_max_lane_rows(d);
                    const int was = (int)(__float_as_uint(up[i]) >> 23) - 127, e = (int)(__float_as_uint(d) >> 23) - 127;
                    const int n = d == 0.0f ? was : min(15, -1 - e);
                    down[i] = two_to(n - was);
                    set_up(i, n);
                }
                if (begun)
                    each<NB>([&](auto b) {
                        const float by = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(down[b % SW]), b / SW));
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) o[rt][2 * b] *= by, o[rt][2 * b + 1] *= by;
                    });
            }
        }
        // weights
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float from = ref[rt] == -INFINITY ? 0.0f : -ref[rt];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // (not fused: where scores are so large that the reference is rounded, the largest product has to round like it)
                s[rt][j] = __builtin_amdgcn_exp2f(s[rt][j] * factor[rt] + from);
                l[rt] += s[rt][j];
            }
        }
    };
    // products of weights (under the values' scales) and values
    auto products = [&](Values& t, const Scales& sc) {
        if constexpr (LIN)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < VW; i++) t.v[h].w[i] = (t.v[h].w[i] & 0xffffu) | (t.w[h].w[i] & 0xffff0000u);
        uint32_t scale[SW];
#pragma unroll
        for (int i = 0; i < SW; i++) scale[i] = __builtin_bit_cast(uint32_t, as_h2(sc.s.w[i]) * h2{(f16_t)up[i], (f16_t)up[i]});
        h2 ph[RT][4], pl[RT][4];
        float less = -1.0f; // (unknown to the compiler: a fused multiply-add takes an f16 as it is, a subtraction does not)
        asm("" : "+s"(less));
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float a = s[rt][2 * r], c = s[rt][2 * r + 1];
                // (as it stands in its register, or each half is rounded again for the difference)
                uint32_t w = __builtin_bit_cast(uint32_t, h2{(f16_t)a, (f16_t)c});
                asm("" : "+v"(w));
                const h2 p = as_h2(w);
                ph[rt][r] = p;
                // (and the differences as f32, or each goes through an instruction of half the rate that rounds it at once)
                float da = __builtin_fmaf((float)p[0], less, a), dc = __builtin_fmaf((float)p[1], less, c);
                asm("" : "+v"(da), "+v"(dc));
                pl[rt][r] = h2{(f16_t)da, (f16_t)dc};
            }
        each<NB>([&](auto b) {
            h2 d[4];
            each<4>([&](auto r) { d[r] = as_h2(of_lane<r * VL + b / SW>(scale[b % SW])); });
            h8 va, vc;
            value_pair<QT>(t.v, b, e1024, va, vc);
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                h2 w[4], e[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    w[r] = ph[rt][r] * d[r];
                    // what the product lost, and the weight's second part
                    e[r] = __builtin_elementwise_fma(pl[rt][r], d[r], __builtin_elementwise_fma(ph[rt][r], d[r], -w[r]));
                }
                const h8 wh = join(w[0], w[1], w[2], w[3]), wl = join(e[0], e[1], e[2], e[3]);
                o[rt][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, wh, o[rt][2 * b], 0, 0, 0);
                o[rt][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, wh, o[rt][2 * b + 1], 0, 0, 0);
                o[rt][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, wl, o[rt][2 * b], 0, 0, 0);
                o[rt][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, wl, o[rt][2 * b + 1], 0, 0, 0);
            }
        });
    };
    if (any) {
        if constexpr (TWO) { // two sets of registers in turns: a tile is requested before the one in front of it is worked on
            for (;;) {
                load_keys(keys[1], scales[1], min(tile + kStep, last - 1));
                load_values(vals[1], scales[1], min(tile + kStep, last - 1));
                load_lineage(min(tile + 2 * kStep, last - 1));
                scores(keys[0]);
                weights(scales[0], tile);
                products(vals[0], scales[0]);
                tile += kStep;
                if (tile >= last) break;
                load_keys(keys[0], scales[0], min(tile + kStep, last - 1));
                load_values(vals[0], scales[0], min(tile + kStep, last - 1));
                load_lineage(min(tile + 2 * kStep, last - 1));
                scores(keys[1]);
                weights(scales[1], tile);
                products(vals[1], scales[1]);
                tile += kStep;
                if (tile >= last) break;
            }
        } else { // one set: keys are requested when the last ones have been used, so are values
            for (; tile < last; tile += kStep) {
                const int next = min(tile + kStep, last - 1);
                scores(keys[0]);
                load_keys(keys[0], scales[1], next);
                load_lineage(min(tile + 2 * kStep, last - 1));
                weights(scales[0], tile);
                products(vals[0], scales[0]);
                load_values(vals[0], scales[1], next);
                scales[0] = scales[1];
            }
        }
    }
    // What is known of a row's scores when all is read: the reference, and the sum of weights.  No position: -infinity and zero.  A score that
    // is NaN: both NaN, because the maximum passes over it and the reference of scores that are all NaN would stay at "no position".
    const auto statistics = [](float reference, float sum) { return make_float2(sum != sum ? sum : reference, sum); };
    if constexpr (SOLO) { // lane (x, g) has of row x and block b the values 8 g .. 8 g + 7
        static_assert(RT == 1);
        const float sum = qmm_add_lane32(qmm_add_lane16(l[0])), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        float down[NB];
        each<NB>([&](auto b) { down[b] = 1.0f / up_of(b); });
        if (x >= rows_here) return;
        const int64_t row = row_index(x);
        if (P.parts > 1 && g == 0) P.stats[row * P.parts + part] = statistics(ref[0], sum);
        each<NB>([&](auto b) {
            const f4 a = o[0][2 * b], c = o[0][2 * b + 1];
            const float v[8] = {a[0], c[0], a[1], c[1], a[2], c[2], a[3], c[3]}, by = down[b];
            if (P.parts > 1) {
                float* dst = P.sums + (row * P.parts + part) * D + 32 * b + 8 * g;
#pragma unroll
                for (int i = 0; i < 8; i++) dst[i] = v[i] * by;
            } else {
                T* dst = static_cast<T*>(P.out) + row * D + 32 * b + 8 * g;
#pragma unroll
                for (int i = 0; i < 8; i++) dst[i] = (T)(v[i] * (by * inv));
            }
        });
        return;
    }
    // the waves' results meet in LDS; lane (x, g) has of block b the values 8 g .. 8 g + 7 of row x
    float2* stat = reinterpret_cast<float2*>(lds + kWaves * ROWS * (D + 4));
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        float* dst = lds + (wave * ROWS + 16 * rt + x) * (D + 4) + 8 * g;
        each<NB>([&](auto b) {
            const float by = 1.0f / up_of(b);
            const f4 a = o[rt][2 * b] * by, c = o[rt][2 * b + 1] * by;
            *reinterpret_cast<f4*>(dst + 32 * b) = f4{a[0], c[0], a[1], c[1]};
            *reinterpret_cast<f4*>(dst + 32 * b + 4) = f4{a[2], c[2], a[3], c[3]};
        });
        const float sum = qmm_add_lane32(qmm_add_lane16(l[rt]));
        if (g == 0) stat[wave * ROWS + 16 * rt + x] = statistics(ref[rt], sum);
    }
    __syncthreads();
    // a thread per row turns the references into the waves' weights and leaves where the row goes
    f4* weight = reinterpret_cast<f4*>(stat + kWaves * ROWS); // a row's waves
    float* total = reinterpret_cast<float*>(weight + ROWS);
    int64_t* where = reinterpret_cast<int64_t*>(total + ROWS);
    static_assert(kWaves == 4);
    if ((int)threadIdx.x < rows_here) {
        const int r = threadIdx.x;
        float2 st[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; w++) st[w] = stat[w * ROWS + r];
        const float to = fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x));
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float by = st[w].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st[w].x - to);
            sum += by == 0.0f ? 0.0f : st[w].y * by;
            weight[r][w] = by;
        }
        const int64_t row = row_index(r);
        where[r] = row;
        if (P.parts > 1) P.stats[row * P.parts + part] = statistics(to, sum);
        else total[r] = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
    __syncthreads();
    constexpr int kTurns = ROWS * (D / 4) / (64 * kWaves);
#pragma unroll
    for (int turn = 0; turn < kTurns; turn++) {
        const int i = threadIdx.x + turn * (64 * kWaves), r = i / (D / 4), d = i % (D / 4) * 4;
        if (r >= rows_here) break;
        const int64_t row = where[r];
        const f4 by = weight[r];
        f4 v[kWaves], a = f4{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; w++) v[w] = *reinterpret_cast<const f4*>(lds + (w * ROWS + r) * (D + 4) + d);
#pragma unroll
        for (int w = 0; w < kWaves; w++) // (a wave without a position left zeros)
            a += v[w] * by[w];
        if (P.parts > 1) {
            *reinterpret_cast<f4*>(P.sums + (row * P.parts + part) * D + d) = a;
        } else {
            T* out = static_cast<T*>(P.out) + row * D + d;
            const float inv = total[r];
#pragma unroll
            for (int j = 0; j < 4; j++) out[j] = (T)(a[j] * inv);
        }
    }
}

// RT: tiles of 16 query rows that a workgroup has of a prompt; the own positions of a sequence go by one.
template <typename T, int QT, int D, int RT, bool LIN>
__global__ __launch_bounds__(64 * kWaves, D <= 128 ? 2 : 1) void attend_kernel(AttendParams P) {
    extern __shared__ __attribute__((aligned(16))) float lds[]; // see the end of attend_rows
    const int id = blockIdx.x;
    if (id < P.prefix_wgs) attend_rows<T, QT, D, RT, true, false>(P, id, lds);
    else if (P.own_solo) attend_rows<T, QT, D, 1, false, LIN, true>(P, id - P.prefix_wgs, lds);
    else attend_rows<T, QT, D, 1, false, LIN>(P, id - P.prefix_wgs, lds);
}

// A row's parts joined: by a wave where there are at most eight (FEW), by the four waves of a workgroup in turn where there are more.
// Statistics and sums are requested together, eight parts a wave at a time; what a part did not write (no position of the row) is in its
// place and not looked at.  (Scores that are NaN: see `statistics` above; a sum of zero is a row without positions.)
template <typename T, int D, bool FEW>
__global__ __launch_bounds__(256) void attend_join_kernel(const float* __restrict__ sums, const float2* __restrict__ stats, T* __restrict__ out, int parts,
                                                          int64_t rows) {
    constexpr int N = D / 64, A = 8, STEP = FEW ? 1 : 4;
    typedef float vec __attribute__((ext_vector_type(N)));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = FEW ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (FEW && row >= rows) return;
    stats += row * parts, sums += row * parts * D + lane * N;
    float to = -INFINITY, sum = 0.0f; // of this wave's parts so far
    vec a = 0.0f;
    for (int p0 = FEW ? 0 : wave; p0 < parts; p0 += STEP * A) {
        vec v[A];
        const int mine = p0 + STEP * (lane & (A - 1)); // lane i of eight: the statistics of part i
        const float2 st = stats[min(mine, parts - 1)];
#pragma unroll
        for (int i = 0; i < A; i++) v[i] = *reinterpret_cast<const vec*>(sums + (int64_t)min(p0 + STEP * i, parts - 1) * D);
        const float ref = mine < parts ? st.x : -INFINITY;
        const unsigned there = (unsigned)__ballot(ref != -INFINITY); // parts that wrote sums: also under a weight of zero, a NaN is not lost
        float most = ref;
        most = fmaxf(most, dpp_f<0xB1>(most));
        most = fmaxf(most, dpp_f<0x4E>(most));
        most = fmaxf(most, dpp_f<0x141>(most)); // over the eight
        const float next = fmaxf(to, most);
        const float by = ref == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ref - next), old = to == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(to - next);
        sum = sum * old + sum8(by == 0.0f ? 0.0f : st.y * by);
        a *= old;
#pragma unroll
        for (int i = 0; i < A; i++) // (no branch: it would take the load with it, one after the other)
            a += (there >> i & 1 ? v[i] : vec(0.0f)) * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(by), i));
        to = next;
    }
    if constexpr (FEW) {
        T* dst = out + row * D + lane * N;
#pragma unroll
        for (int i = 0; i < N; i++) dst[i] = (T)(sum == 0.0f ? 0.0f : a[i] / sum);
        return;
    }
    __shared__ float red[4][D + 2];
#pragma unroll
    for (int i = 0; i < N; i++) red[wave][lane * N + i] = a[i];
    if (lane == 0) red[wave][D] = sum, red[wave][D + 1] = to;
    __syncthreads();
    if (threadIdx.x < D) {
        float most = -INFINITY, total = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) most = fmaxf(most, red[w][D + 1]);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float by = red[w][D + 1] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(red[w][D + 1] - most);
            total += red[w][D] * by, v += red[w][threadIdx.x] * by;
        }
        out[row * D + threadIdx.x] = (T)(total == 0.0f ? 0.0f : v / total);
    }
}

template <typename T, int QT, int D>
hipError_t launch_attend_of(const AttendParams& P, int rt, hipStream_t stream) {
    const unsigned wgs = (unsigned)(P.prefix_wgs + (P.own_solo ? ((int64_t)P.own_units * P.own_z + kWaves - 1) / kWaves : (int64_t)(P.own_units + 7) / 8 * 8 * P.own_z));
    const size_t lds = (size_t)16 * rt * (kWaves * ((D + 4) * sizeof(float) + sizeof(float2)) + sizeof(f4) + sizeof(float) + sizeof(int64_t));
    const auto run = [&](auto kernel) {
        if (lds > 64 * 1024) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
            if (e != hipSuccess) return e;
        }
        kernel<<<wgs, 64 * kWaves, lds, stream>>>(P);
        return hipGetLastError();
    };
    hipError_t e;
    constexpr int R2 = D <= 128 ? 2 : 1;
    if (P.lineage) e = rt == 1 ? run(attend_kernel<T, QT, D, 1, true>) : run(attend_kernel<T, QT, D, R2, true>);
    else e = rt == 1 ? run(attend_kernel<T, QT, D, 1, false>) : run(attend_kernel<T, QT, D, R2, false>);
    if (e != hipSuccess || P.parts == 1) return e;
    const int64_t rows = (int64_t)P.batch * P.heads;
    if (P.parts <= 8) attend_join_kernel<T, D, true><<<(unsigned)((rows + 3) / 4), 256, 0, stream>>>(P.sums, P.stats, static_cast<T*>(P.out), P.parts, rows);
    else attend_join_kernel<T, D, false><<<(unsigned)rows, 256, 0, stream>>>(P.sums, P.stats, static_cast<T*>(P.out), P.parts, rows);
    return hipGetLastError();
}
template <typename T>
hipError_t launch_attend(int type, int64_t d, const AttendParams& P, int rt, hipStream_t stream) {
    if (type == IZWI_KV_Q8_0)
        return d == 64    ? launch_attend_of<T, IZWI_KV_Q8_0, 64>(P, rt, stream)
               : d == 128 ? launch_attend_of<T, IZWI_KV_Q8_0, 128>(P, rt, stream)
                          : launch_attend_of<T, IZWI_KV_Q8_0, 256>(P, rt, stream);
    return d == 64    ? launch_attend_of<T, IZWI_KV_Q4_0, 64>(P, rt, stream)
           : d == 128 ? launch_attend_of<T, IZWI_KV_Q4_0, 128>(P, rt, stream)
                      : launch_attend_of<T, IZWI_KV_Q4_0, 256>(P, rt, stream);
}

template <typename T>
int shared_attention_impl(int type, const T* q, int64_t q_stride, int64_t batch, int64_t beams, int64_t heads, int64_t kv_heads, int64_t d,
                          const void* prefix, int64_t prefix_slots, int64_t prefix_capacity, const int32_t* prefix_lens, int64_t max_prefix,
                          const void* cache, int64_t slots, int64_t capacity, const int32_t* lens, int64_t max_len, const uint8_t* lineage, float scale,
                          T* out, void* stream_) {
    constexpr const char* what = "decode_shared_attention";
    if (batch < 0 || beams <= 0 || batch % beams || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 65535 || batch > 0xfffff ||
        q_stride < heads * d)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: bad shape (batch %lld, beams %lld, heads %lld on %lld, row stride %lld)", what, (long long)batch,
                        (long long)beams, (long long)heads, (long long)kv_heads, (long long)q_stride);
    // (the format and the head size are checked where neither cache is given, too)
    if (int rc = kv_check_shape(what, type, prefix ? prefix_slots : 1, kv_heads, prefix ? prefix_capacity : 1, d)) return rc;
    if (int rc = kv_check_shape(what, type, cache ? slots : 1, kv_heads, cache ? capacity : 1, d)) return rc;
    if (prefix && (prefix_slots < batch / beams || max_prefix < 0 || max_prefix > prefix_capacity))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: %lld prompts of up to %lld positions in %lld slots of %lld", what, (long long)(batch / beams),
                        (long long)max_prefix, (long long)prefix_slots, (long long)prefix_capacity);
    if (cache && (slots < batch || max_len < 0 || max_len > capacity))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: %lld sequences of up to %lld positions in %lld slots of %lld", what, (long long)batch,
                        (long long)max_len, (long long)slots, (long long)capacity);
    if (batch > 0x7fffff / heads) // (threads stay below 2^32)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: %lld sequences of %lld heads", what, (long long)batch, (long long)heads);
    if (lineage && (beams > 255 || !cache))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: lineage of %lld beams (at most 255, of a cache)", what, (long long)beams);
    if (!std::isfinite(scale)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: scale %g", what, (double)scale);
    if (batch == 0) return IZWI_QMM_OK;
    if (!prefix && !cache) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: neither a prefix nor a cache", what);
    if (!q || !out || (prefix && !prefix_lens) || (cache && !lens)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: NULL buffer", what);
    if (kv_overlap(q, ((batch - 1) * q_stride + heads * d) * (int64_t)sizeof(T), out, batch * heads * d * (int64_t)sizeof(T)))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: out shares memory with q", what);
    if (!kv_aligned(prefix, 16) || !kv_aligned(cache, 16)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: caches must be 16-byte aligned", what);
    int device = 0, n_cus = 0;
    if (int rc = qmm_current_device(&device, &n_cus)) return rc;
    AttendParams P{};
    P.q = q, P.out = out, P.q_stride = q_stride;
    P.prefix = kv_planes(type, prefix, prefix_slots, kv_heads, prefix_capacity, d);
    P.own = kv_planes(type, cache, slots, kv_heads, capacity, d);
    P.prefix_lens = prefix_lens, P.lens = lens, P.lineage = lineage;
    P.batch = (int)batch, P.beams = (int)beams, P.heads = (int)heads, P.kv_heads = (int)kv_heads, P.group = (int)(heads / kv_heads);
    P.max_prefix = prefix ? (int)max_prefix : 0, P.max_len = cache ? (int)max_len : 0;
    P.scale = scale;
    hipStream_t stream = (hipStream_t)stream_;
    // Workgroups of four waves, about one per compute unit, each with the positions of a split in turns of 32 per wave (two per compute unit
    // take 2 us more nearly everywhere, for more to join: 8 sequences of 800 positions 8.5 us -> 9.5, 32 of 2000 25.4 -> 27.6, 16 beams on 32000 34 -> 38).
    constexpr int waves = kWaves;
    const auto turns = [&](int64_t n_seq, int most, int rows, int rt) { // of a wave, with one workgroup per compute unit
        const int64_t base = n_seq * kv_heads * ((rows + 16 * rt - 1) / (16 * rt)), tiles = (most + 31) / 32;
        const int64_t splits = std::max<int64_t>(1, std::min((n_cus + base - 1) / base, (tiles + waves - 1) / waves));
        return tiles / (splits * waves);
    };
    // Few positions of one kind stay with one workgroup per sequence and kv head: nothing is left to join, and the host has a launch less (16
    // heads on 8, in a graph: 200 positions 5.9 us instead of 7.1, 380 6.8 instead of 7.2; but 600 8.5 instead of 7.4).
    constexpr int kOneLaunchTiles = 12;
    const bool alone = P.max_prefix == 0 || P.max_len == 0;
    const auto units = [&](int64_t n_seq, int most, int rows, int rt, int& splits, int& n_units, int& z) {
        splits = n_units = 0, z = 1;
        if (most == 0) return;
        z = (rows + 16 * rt - 1) / (16 * rt);
        const int64_t base = n_seq * kv_heads * z, tiles = (most + 31) / 32;
        if (alone && tiles <= kOneLaunchTiles) { // no second kernel
            splits = 1, n_units = (int)base / z;
            return;
        }
        const int64_t s = std::max<int64_t>(1, std::min((n_cus + base - 1) / base, (tiles + waves - 1) / waves)), share = (tiles + s - 1) / s;
        splits = (int)((tiles + share - 1) / share);
        n_units = (int)(n_seq * kv_heads * splits);
    };
    // two tiles of query rows to a workgroup where there are two and the waves have enough to do all the same (32 heads on 8, 16 beams: 60000
    // positions 65 -> 53 us, 32000 40 -> 34; but 2000 10.1 -> 12.9, 8 beams on 1000 8.4 -> 10.8; 4 prompts of 4000, just below the bound, 24.6 -> 22.9)
    const int prompt_rows = (int)(beams * P.group);
    const int rt = d <= 128 && prompt_rows > 16 && turns(batch / beams, P.max_prefix, prompt_rows, 2) >= 8 ? 2 : 1;
    units(batch / beams, P.max_prefix, prompt_rows, rt, P.prefix_splits, P.prefix_units, P.prefix_z);
    units(batch, P.max_len, P.group, 1, P.own_splits, P.own_units, P.own_z);
    // A wave to each where that still fills the compute units, the better the shorter they are: a workgroup's prologue, its meeting in LDS and
    // its idle waves cost more than the positions of a short sequence (371 sequences of up to 14 own positions behind 570, 32 heads on 8: 50 ->
    // 35 us; but 132 of up to 355: 24.5 -> 30).
    P.own_solo = P.own_splits == 1 && (int64_t)P.own_units * P.own_z >= kWaves * n_cus * std::max<int64_t>(1, (P.max_len + 31) / 32 / 4);
    P.prefix_wgs = (P.prefix_units + 7) / 8 * 8 * P.prefix_z;
    P.parts = P.prefix_splits + P.own_splits;
    if (P.parts == 0) { // bounds of zero: zeros
        P.parts = P.own_splits = 1, P.own_units = (int)(batch * kv_heads);
        P.own_z = (P.group + 15) / 16;
    }
    P.by_group = Divisor(P.group), P.by_kv_heads = Divisor(kv_heads), P.by_beams = Divisor(beams);
    P.by_prefix_splits = Divisor(std::max(1, P.prefix_splits)), P.by_own_splits = Divisor(std::max(1, P.own_splits));
    P.by_prefix_z = Divisor(P.prefix_z), P.by_own_z = Divisor(P.own_z);
    QmmCallScope call;
    if (P.parts > 1) {
        const size_t rows = (size_t)batch * heads * P.parts;
        void* scratch = nullptr;
        KV_TRY(qmm_get_scratch(device, stream, rows * (d * sizeof(float) + sizeof(float2)), &scratch));
        P.sums = static_cast<float*>(scratch);
        P.stats = reinterpret_cast<float2*>(P.sums + rows * d);
    }
    KV_TRY(launch_attend<T>(type, d, P, rt, stream));
    return IZWI_QMM_OK;
}

} // namespace

extern "C" {

int izwi_decode_shared_attention_f32(int type, const float* q, int64_t q_stride, int64_t batch, int64_t beams, int64_t num_heads,
                                     int64_t num_kv_heads, int64_t head_dim, const void* prefix, int64_t prefix_slots, int64_t prefix_capacity,
                                     const int32_t* prefix_lens, int64_t max_prefix_len, const void* cache, int64_t slots, int64_t kv_capacity,
                                     const int32_t* lens, int64_t max_len, const uint8_t* lineage, float scale, float* out, void* stream) {
    return qmm_guarded("izwi_decode_shared_attention_f32", [&]() -> int {
    return shared_attention_impl<float>(type, q, q_stride, batch, beams, num_heads, num_kv_heads, head_dim, prefix, prefix_slots, prefix_capacity,
                                        prefix_lens, max_prefix_len, cache, slots, kv_capacity, lens, max_len, lineage, scale, out, stream);
    });
}
int izwi_decode_shared_attention_f16(int type, const uint16_t* q, int64_t q_stride, int64_t batch, int64_t beams, int64_t num_heads,
                                     int64_t num_kv_heads, int64_t head_dim, const void* prefix, int64_t prefix_slots, int64_t prefix_capacity,
                                     const int32_t* prefix_lens, int64_t max_prefix_len, const void* cache, int64_t slots, int64_t kv_capacity,
                                     const int32_t* lens, int64_t max_len, const uint8_t* lineage, float scale, uint16_t* out, void* stream) {
    return qmm_guarded("izwi_decode_shared_attention_f16", [&]() -> int {
    return shared_attention_impl<f16_t>(type, (const f16_t*)q, q_stride, batch, beams, num_heads, num_kv_heads, head_dim, prefix, prefix_slots,
                                        prefix_capacity, prefix_lens, max_prefix_len, cache, slots, kv_capacity, lens, max_len, lineage, scale,
                                        (f16_t*)out, stream);
    });
}

} // extern "C"
