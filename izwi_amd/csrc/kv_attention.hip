// Attention of one new token per sequence over the quantized cache (layout: kv_cache.h): positions that the sequences of a
// prompt share, then each sequence's own.
#include "kv_cache.h"
#include "qmm_lanes.h"

namespace {

typedef _Float16 f16_t;

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
};

__device__ __forceinline__ int clamped_len(const int32_t* lens, int i, int most) { return most ? max(0, min(lens[i], most)) : 0; }

// One workgroup per sequence and query head, sixteen lanes a position.
template <typename T, int QT, int D>
__global__ __launch_bounds__(256) void attend_kernel(AttendParams P) {
    using Row = KvRow<QT, D>;
    constexpr int NB = Row::kBlocks, NU = (NB + 3) / 4;
    constexpr float kBias = QT == IZWI_KV_Q8_0 ? 128.0f : 8.0f;
    __shared__ float red[16][D + 2];
    const int b = blockIdx.x, h = blockIdx.y, kvh = h / P.group, prompt = b / P.beams;
    const int x = threadIdx.x & 15, slot16 = threadIdx.x >> 4, g = x & 3;
    const T* q = static_cast<const T*>(P.q) + b * P.q_stride + (int64_t)h * D;
    float qr[NU][8];
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
        for (int j = 0; j < 8; j++) qr[u][j] = (x >> 2) + 4 * u < NB ? (float)q[32 * ((x >> 2) + 4 * u) + 8 * g + j] : 0.0f;
    float m = -INFINITY, l = 0.0f, acc[NB][2] = {};
    const int np = clamped_len(P.prefix_lens, prompt, P.max_prefix), ns = clamped_len(P.lens, b, P.max_len);
    for (int p = slot16; p < np + ns; p += 16) {
        const bool shared = p < np;
        const KvPlanes& C = shared ? P.prefix : P.own;
        const int at = shared ? p : p - np;
        int slot = shared ? prompt : b;
        if (!shared && P.lineage) {
            const int beam = P.lineage[(int64_t)b * C.padded + at];
            if (beam >= P.beams) continue;
            slot = prompt * P.beams + beam;
        }
        const int64_t row = ((int64_t)slot * C.kv_heads + kvh) * C.padded + at;
        float dot = 0.0f;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const int blk = (x >> 2) + 4 * u;
            if (blk < NB) {
                const uint8_t* unit = C.kq + row * Row::kBytes + Row::unit(blk, g);
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int n = (j >> 1) + 4 * (j & 1);
                    const float k = QT == IZWI_KV_Q8_0 ? (float)unit[j] : (float)(unit[n >> 1] >> (4 * (n & 1)) & 15);
                    part += qr[u][j] * (k - kBias);
                }
                dot += part * (float)C.ks[row * NB + blk];
            }
        }
        dot = sum8(dot);
        dot += dpp_f<0x140>(dot);
        const float s = dot * P.scale, mn = fmaxf(m, s), alpha = merge_weight(m, mn), pe = exp_neg(s - mn);
        m = mn, l = l * alpha + pe;
        const uint8_t* vr = C.vq + row * Row::kBytes + x * Row::kLaneBytes;
#pragma unroll
        for (int blk = 0; blk < NB; blk++) {
            const float d = (float)C.vs[row * NB + blk];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float v = QT == IZWI_KV_Q8_0 ? (float)vr[2 * blk + i] : (float)(vr[blk] >> (4 * i) & 15);
                acc[blk][i] = acc[blk][i] * alpha + pe * (d * (v - kBias));
            }
        }
    }
#pragma unroll
    for (int blk = 0; blk < NB; blk++) red[slot16][32 * blk + 2 * x] = acc[blk][0], red[slot16][32 * blk + 2 * x + 1] = acc[blk][1];
    if (x == 0) red[slot16][D] = m, red[slot16][D + 1] = l;
    __syncthreads();
    if (threadIdx.x < D) {
        float mn = -INFINITY, a = 0.0f, sum = 0.0f;
        for (int i = 0; i < 16; i++) mn = fmaxf(mn, red[i][D]);
        for (int i = 0; i < 16; i++) {
            const float w = merge_weight(red[i][D], mn);
            a += red[i][threadIdx.x] * w, sum += red[i][D + 1] * w;
        }
        static_cast<T*>(P.out)[((int64_t)b * P.heads + h) * D + threadIdx.x] = (T)(sum != 0.0f ? a / sum : 0.0f);
    }
}

template <typename T>
hipError_t launch_attend(int type, int64_t d, const AttendParams& P, hipStream_t stream) {
    const dim3 grid(P.batch, P.heads);
    if (type == IZWI_KV_Q8_0) {
        if (d == 64) attend_kernel<T, IZWI_KV_Q8_0, 64><<<grid, 256, 0, stream>>>(P);
        else if (d == 128) attend_kernel<T, IZWI_KV_Q8_0, 128><<<grid, 256, 0, stream>>>(P);
        else attend_kernel<T, IZWI_KV_Q8_0, 256><<<grid, 256, 0, stream>>>(P);
    } else {
        if (d == 64) attend_kernel<T, IZWI_KV_Q4_0, 64><<<grid, 256, 0, stream>>>(P);
        else if (d == 128) attend_kernel<T, IZWI_KV_Q4_0, 128><<<grid, 256, 0, stream>>>(P);
        else attend_kernel<T, IZWI_KV_Q4_0, 256><<<grid, 256, 0, stream>>>(P);
    }
    return hipGetLastError();
}

template <typename T>
int shared_attention_impl(int type, const T* q, int64_t q_stride, int64_t batch, int64_t beams, int64_t heads, int64_t kv_heads, int64_t d,
                          const void* prefix, int64_t prefix_slots, int64_t prefix_capacity, const int32_t* prefix_lens, int64_t max_prefix,
                          const void* cache, int64_t slots, int64_t capacity, const int32_t* lens, int64_t max_len, const uint8_t* lineage, float scale,
                          T* out, void* stream) {
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
    if (lineage && (beams > 255 || !cache))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: lineage of %lld beams (at most 255, of a cache)", what, (long long)beams);
    if (batch == 0) return IZWI_QMM_OK;
    if (!q || !out || (prefix && !prefix_lens) || (cache && !lens)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: NULL buffer", what);
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
    KV_TRY(launch_attend<T>(type, d, P, (hipStream_t)stream));
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
