// Writing the quantized key / value cache and reading it back (layout: kv_cache.h).
//
// A block of 32 values becomes an f16 scale and 32 quants, by the arithmetic of the GGUF formats in f32:
//   Q8_0  d = max|v| / 127,            quant = round(v * (1 / d)), halves away from zero
//   Q4_0  d = (first v of max|v|) / -8, quant = min(15, floor(v * (1 / d) + 8.5)) - 8
// and a value read back is f32(f16(d)) * quant, one rounding if it is stored as f16.  A block whose scale has no f16
// (an infinity or NaN among its values, or one beyond the range) reads as NaN throughout rather than as a number that it
// never held; one whose scale is zero in f16 reads as zeros.
//
// Both kernels touch every byte once and are bound by memory, small calls by the launch.
#include "kv_cache.h"

#include <type_traits>

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
    unsigned tokens, kv_heads, items; // items = batch * tokens * kv_heads
    int first_slot;
    int64_t capacity;
    unsigned k_blocks; // workgroups that take keys; the others take values
};

__device__ __forceinline__ unsigned umax8(unsigned v) { // over 8 lanes, in every one
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xf, 0xf, false));
    return max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xf, 0xf, false));
}
__device__ __forceinline__ unsigned umax16(unsigned v) {
    v = umax8(v);
    return max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xf, 0xf, false)); // row_mirror
}
template <int LANES>
__device__ __forceinline__ unsigned umax_over(unsigned v) {
    return LANES == 8 ? umax8(v) : umax16(v);
}

// The N values of this lane out of a block that LANES lanes hold in order: the block's scale, and the quants as the cache
// stores them (q + 128, q + 8).  Magnitudes are compared as bits, so that a NaN is the largest of all.
template <int QT, int N, int LANES>
__device__ __forceinline__ f16_t quantize_block(const float (&v)[N], int lane, unsigned (&q)[N]) {
    unsigned best = 0, sign = 0; // the lane's first value of largest magnitude
#pragma unroll
    for (int i = 0; i < N; i++) {
        const unsigned bits = __float_as_uint(v[i]), mag = bits & 0x7fffffffu;
        if (mag > best) best = mag, sign = bits >> 31;
    }
    const unsigned amax = umax_over<LANES>(best);
    float d;
    if constexpr (QT == IZWI_KV_Q8_0) {
        d = __fdiv_rn(__uint_as_float(amax), 127.0f);
    } else {
        // the lowest lane that holds the maximum decides the sign
        const unsigned key = umax_over<LANES>(best == amax ? ((unsigned)(LANES - lane) << 1) | sign : 0u);
        d = __uint_as_float(amax | (key << 31)) * -0.125f;
    }
    f16_t h = (f16_t)d;
    const bool bad = amax >= 0x7f800000u || (float)h == INFINITY || (float)h == -INFINITY;
    const bool dead = bad || h == (f16_t)0.0f;
    const float inv = dead ? 0.0f : __fdiv_rn(1.0f, d);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float scaled = __fmul_rn(bad ? 0.0f : v[i], inv);
        if constexpr (QT == IZWI_KV_Q8_0) q[i] = (unsigned)(qmm_round_clamp_i8(scaled) + 128);
        else q[i] = dead ? 8u : (unsigned)min(15, (int)__fadd_rn(scaled, 8.5f));
    }
    return bad ? (f16_t)NAN : h;
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

// where the row of `item` stands: its sequence, token and head, and whether the cache has (or gets) it
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
__global__ __launch_bounds__(256) void kv_append_kernel(KvRowsParams P) {
    using Row = KvRow<QT, D>;
    if (blockIdx.x < P.k_blocks) {
        constexpr int kLanes = D / 4;
        const unsigned thread = blockIdx.x * 256 + threadIdx.x, asked = thread / kLanes, item = min(asked, P.items - 1);
        const int e = (threadIdx.x % kLanes) * 4, b = e / 32, g = (e & 31) >> 3, second = (e >> 2) & 1;
        const KvItem it = kv_item<false>(P, item);
        float v[4];
        load_values<T, 4, VEC>(static_cast<const T*>(P.k_in) + it.row * P.k_stride + it.head * D + e, v);
        unsigned q[4];
        const f16_t d = quantize_block<QT, 4, 8>(v, threadIdx.x & 7, q);
        uint8_t* dst = P.cache.kq + it.begin * Row::kBytes + Row::key(it.pos, b, g);
        const bool mine = asked < P.items && it.there;
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
    const unsigned thread = (blockIdx.x - P.k_blocks) * 256 + threadIdx.x, asked = thread / 16, item = min(asked, P.items - 1);
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
        d[b] = quantize_block<QT, 2, 16>(v[b], x, q);
        if constexpr (QT == IZWI_KV_Q8_0) half[b] = (uint16_t)(q[0] | q[1] << 8);
        else half[b / 2] |= (uint16_t)((q[0] | q[1] << 4) << (8 * (b & 1)));
    }
    if (asked >= P.items || !it.there) return;
#pragma unroll
    for (int j = 0; j < Row::kLane / 2; j++) *reinterpret_cast<uint16_t*>(P.cache.vq + it.begin * Row::kBytes + Row::value(it.pos, x, j)) = half[j];
#pragma unroll
    for (int b = 0; b < Row::kBlocks; b++)
        if (x == b) P.cache.vs[it.begin * Row::kBlocks + Row::value_scale(it.pos, b)] = d[b];
}

// The same lanes the other way; what the cache does not have reads as zeros.
template <typename T, int QT, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(KvRowsParams P) {
    using Row = KvRow<QT, D>;
    constexpr int kBias = QT == IZWI_KV_Q8_0 ? 128 : 8;
    auto store = [](T* dst, const float* v, auto count) {
        constexpr int N = decltype(count)::value;
        if constexpr (VEC) {
            typedef T vec __attribute__((ext_vector_type(N)));
            vec t;
#pragma unroll
            for (int i = 0; i < N; i++) t[i] = (T)v[i];
            *reinterpret_cast<vec*>(dst) = t;
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) dst[i] = (T)v[i];
        }
    };
    if (blockIdx.x < P.k_blocks) {
        constexpr int kLanes = D / 4;
        const unsigned thread = blockIdx.x * 256 + threadIdx.x, item = thread / kLanes;
        if (item >= P.items) return;
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
        store(static_cast<T*>(P.k_out) + ((int64_t)it.row * P.kv_heads + it.head) * D + e, v, std::integral_constant<int, 4>{});
        return;
    }
    const unsigned thread = (blockIdx.x - P.k_blocks) * 256 + threadIdx.x, item = thread / 16;
    if (item >= P.items) return;
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
        store(dst + 32 * b, v, std::integral_constant<int, 2>{});
    }
}

template <typename T, int QT, int D, bool READ>
hipError_t launch_rows(const KvRowsParams& P0, bool vec, hipStream_t stream) {
    KvRowsParams P = P0;
    const uint64_t k_threads = (uint64_t)P.items * (D / 4), v_threads = (uint64_t)P.items * 16;
    P.k_blocks = (unsigned)((k_threads + 255) / 256);
    const unsigned blocks = P.k_blocks + (unsigned)((v_threads + 255) / 256);
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
    if (batch && tokens && (batch * tokens > 0x7fffffff / kv_heads || batch * tokens * kv_heads > 0x7fffffffLL * 256 / (d / 4 + 16) - 512))
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: more than 2^31 rows in a call", what);
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
    P.items = (unsigned)(batch * tokens * kv_heads), P.first_slot = (int)first_slot, P.capacity = capacity;
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
    P.items = (unsigned)(batch * tokens * kv_heads), P.first_slot = (int)first_slot, P.capacity = capacity;
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
