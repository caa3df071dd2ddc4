// One step of beam search: the best `beams` of beams * vocab candidates scores[w] + logits[w][t] - logsumexp(logits[w]),
// and the beams' lineage that follows.
//
// Two launches.  The first reads the logits once: a workgroup takes a chunk of a beam's row, keeps it in registers, and leaves its
// maximum, its sum of exponentials under that maximum and its best `beams` logits, largest first.  No more of a chunk can be
// among the best of its prompt.  The second, a workgroup per prompt, joins the chunks' sums, turns what is left into scores, picks
// the best and reorders the lineage.
//
// Sums and scores are f64: neighbours among 10^6 candidates lie closer than an f32 sum is exact, and which one is picked is
// a whole number.  Within a beam the order is the logits' own, in f32.
#include "kv_cache.h"
#include "qmm_lanes.h"

namespace {

constexpr int kMaxBeams = 64;

struct BeamParams {
    const float* logits;
    const float* scores;
    const uint8_t* finished;
    int32_t* tokens;
    int32_t* parents;
    float* scores_out;
    uint8_t* finished_out;
    const uint8_t* lineage;
    uint8_t* lineage_out;
    const int32_t* lens;
    double2* sums;  // [prompts * beams][chunks]: maximum, sum of exponentials
    uint64_t* keys; // [prompts * beams][chunks][beams]: order of the logit, then ~token; 0: none
    int beams, vocab, chunks;
    int64_t eos;
    int64_t padded; // bytes of a lineage row
};

// NaN as -infinity, +infinity as the largest float, -0 as 0
__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : fminf(v, 3.402823466e38f) + 0.0f; }
// floats, doubles (no NaN) in the order of unsigned numbers, and back
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t u = __float_as_uint(v);
    return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o ^ ((int32_t)o < 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t order_of(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return u ^ ((int64_t)u < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double double_of(uint64_t o) {
    return __longlong_as_double((long long)(o ^ ((int64_t)o < 0 ? 1ull << 63 : ~0ull)));
}

// The largest T that `k` lanes' values reach, bit by bit (0 where fewer lanes hold a value)
template <typename U>
__device__ __forceinline__ U kth_of_lanes(U v, int k) {
    U t = 0;
#pragma unroll
    for (int bit = 8 * (int)sizeof(U) - 1; bit >= 0; bit--) {
        const U trial = t | (U)1 << bit;
        if (__popcll(__ballot(v >= trial)) >= k) t = trial;
    }
    return t;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

constexpr int kChunkThreads = 256, kPer = 16, kChunk = kChunkThreads * kPer;

__global__ __launch_bounds__(kChunkThreads) void beam_chunk_kernel(BeamParams P) {
    __shared__ float top[4];
    __shared__ double sum[4];
    __shared__ uint32_t threshold[4];
    __shared__ uint64_t found[kChunk];
    __shared__ uint64_t best[4];
    __shared__ unsigned n_found;
    const int row = blockIdx.y, chunk = blockIdx.x, begin = chunk * kChunk, n = min(kChunk, P.vocab - begin);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t* keys = P.keys + ((int64_t)row * P.chunks + chunk) * P.beams;
    if (P.finished && P.finished[row]) return; // the second launch looks at neither
    const float score = clean(P.scores[row]);
    if (score == -INFINITY) { // every candidate of the beam is -infinity: the lowest tokens
        if (tid < P.beams) keys[tid] = tid < n ? (uint64_t)order_of(-INFINITY) << 32 | ~(uint32_t)(begin + tid) : 0;
        return;
    }
    const float* x = P.logits + (int64_t)row * P.vocab + begin;
    float v[kPer], m = -INFINITY;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) v[i] = x[min(i * kChunkThreads + tid, n - 1)];
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        v[i] = clean(v[i]);
        if (i * kChunkThreads + tid < n) m = fmaxf(m, v[i]), most = max(most, order_of(v[i]));
    }
    const float wm = wave_max(m);
    const uint32_t kth = kth_of_lanes<uint32_t>(most, P.beams);
    if (lane == 0) top[wave] = wm, threshold[wave] = kth;
    if (tid == 0) n_found = 0;
    __syncthreads();
    m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    const uint32_t t = max(max(threshold[0], threshold[1]), max(threshold[2], threshold[3]));
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        if (i * kChunkThreads + tid >= n) break;
        if (v[i] != -INFINITY) s += exp((double)v[i] - (double)m);
        if (order_of(v[i]) >= t) found[atomicAdd(&n_found, 1u)] = (uint64_t)order_of(v[i]) << 32 | ~(uint32_t)(begin + i * kChunkThreads + tid);
    }
    s = wave_sum(s);
    if (lane == 0) sum[wave] = s;
    __syncthreads();
    if (tid == 0) P.sums[(int64_t)row * P.chunks + chunk] = make_double2((double)m, sum[0] + sum[1] + sum[2] + sum[3]);
    const int got = (int)n_found; // (in any order; the keys are all different)
    if (got <= 4 * kChunkThreads) {
        for (int i = tid; i < got; i += kChunkThreads) {
            const uint64_t key = found[i];
            int rank = 0;
            for (int j = 0; j < got; j++) rank += found[j] > key;
            if (rank < P.beams) keys[rank] = key;
        }
        if (tid >= got && tid < P.beams) keys[tid] = 0;
        return;
    }
    // a chunk of few different values: the largest, again and again
    uint64_t last = ~0ull;
    for (int k = 0; k < P.beams; k++) {
        uint64_t mine = 0;
        for (int i = tid; i < got; i += kChunkThreads)
            if (found[i] < last) mine = max(mine, found[i]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mine = max(mine, (uint64_t)__shfl_xor((unsigned long long)mine, o));
        __syncthreads();
        if (lane == 0) best[wave] = mine;
        __syncthreads();
        last = max(max(best[0], best[1]), max(best[2], best[3]));
        if (tid == 0) keys[k] = last;
    }
}

constexpr int kPickThreads = 1024, kPickRoom = 4096;

struct Candidate {
    uint64_t score; // order of the score
    uint32_t flat;  // beam * vocab + token
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) { return a.score > b.score || (a.score == b.score && a.flat < b.flat); }

__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamParams P) {
    __shared__ double offset[kMaxBeams]; // of a beam's logits: score - logsumexp
    __shared__ uint8_t ended[kMaxBeams];
    __shared__ uint64_t thresholds[kPickThreads / 64];
    __shared__ __attribute__((aligned(16))) uint32_t room[3 * kPickRoom]; // what passes the threshold, then pieces of the lineage
    __shared__ uint64_t best_score[kPickThreads / 64];
    __shared__ uint32_t best_flat[kPickThreads / 64];
    __shared__ uint32_t picked[kMaxBeams];
    __shared__ uint64_t picked_score[kMaxBeams];
    __shared__ unsigned n_found;
    uint64_t* found_score = reinterpret_cast<uint64_t*>(room);
    uint32_t* found_flat = room + 2 * kPickRoom;
    const int prompt = blockIdx.x, W = P.beams, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row0 = (int64_t)prompt * W;
    for (int w = wave; w < W; w += kPickThreads / 64) {
        const float score = clean(P.scores[row0 + w]);
        const bool end = P.finished && P.finished[row0 + w];
        double o = score;
        if (!end && score != -INFINITY) {
            const double2* part = P.sums + (row0 + w) * P.chunks;
            double m = -INFINITY, s = 0.0;
            for (int c = lane; c < P.chunks; c += 64) m = fmax(m, part[c].x);
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) m = fmax(m, __shfl_xor(m, d));
            if (m != -INFINITY)
                for (int c = lane; c < P.chunks; c += 64) s += part[c].y == 0.0 ? 0.0 : part[c].y * exp(part[c].x - m);
            s = wave_sum(s);
            o = m == -INFINITY ? -INFINITY : (double)score - m - log(s);
        }
        if (lane == 0) offset[w] = o, ended[w] = end;
    }
    if (tid == 0) n_found = 0;
    __syncthreads();
    const int per_beam = P.chunks * W, total = W * per_beam;
    // candidate i: score order 0 for none
    auto candidate = [&](int i) {
        const int w = i / per_beam, j = i - w * per_beam;
        Candidate c{0, 0xffffffffu};
        if (ended[w]) {
            if (j == 0) c.score = order_of(offset[w]), c.flat = (uint32_t)w * P.vocab + (uint32_t)P.eos;
            return c;
        }
        const uint64_t key = P.keys[(row0 + w) * per_beam + j];
        if (key) {
            const float logit = value_of((uint32_t)(key >> 32));
            c.score = order_of(offset[w] == -INFINITY || logit == -INFINITY ? (double)-INFINITY : offset[w] + (double)logit);
            c.flat = (uint32_t)w * P.vocab + ~(uint32_t)key;
        }
        return c;
    };
    uint64_t most = 0;
    for (int i = tid; i < total; i += kPickThreads) most = max(most, candidate(i).score);
    const uint64_t kth = kth_of_lanes<uint64_t>(most, W);
    if (lane == 0) thresholds[wave] = kth;
    __syncthreads();
    uint64_t t = 1;
    for (int i = 0; i < kPickThreads / 64; i++) t = max(t, thresholds[i]);
    for (int i = tid; i < total; i += kPickThreads) {
        const Candidate c = candidate(i);
        if (c.score >= t) {
            const unsigned at = atomicAdd(&n_found, 1u);
            if (at < kPickRoom) found_score[at] = c.score, found_flat[at] = c.flat;
        }
    }
    __syncthreads();
    const int got = (int)n_found;
    if (got <= kPickRoom) {
        for (int i = tid; i < got; i += kPickThreads) {
            const Candidate c{found_score[i], found_flat[i]};
            int rank = 0;
            for (int j = 0; j < got; j++) rank += before(Candidate{found_score[j], found_flat[j]}, c);
            if (rank < W) picked[rank] = c.flat, picked_score[rank] = c.score;
        }
    } else { // many equal scores: the best, again and again
        Candidate last{~0ull, 0};
        for (int k = 0; k < W; k++) {
            Candidate mine{0, 0xffffffffu};
            for (int i = tid; i < total; i += kPickThreads) {
                const Candidate c = candidate(i);
                if (before(last, c) && before(c, mine)) mine = c;
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const Candidate c{(uint64_t)__shfl_xor((unsigned long long)mine.score, o), (uint32_t)__shfl_xor((int)mine.flat, o)};
                if (before(c, mine)) mine = c;
            }
            __syncthreads();
            if (lane == 0) best_score[wave] = mine.score, best_flat[wave] = mine.flat;
            __syncthreads();
            last = Candidate{best_score[0], best_flat[0]};
            for (int i = 1; i < kPickThreads / 64; i++) {
                const Candidate c{best_score[i], best_flat[i]};
                if (before(c, last)) last = c;
            }
            if (tid == 0) picked[k] = last.flat, picked_score[k] = last.score;
        }
    }
    __syncthreads();
    if (tid < W) {
        const uint32_t parent = picked[tid] / (uint32_t)P.vocab, token = picked[tid] - parent * (uint32_t)P.vocab;
        P.tokens[row0 + tid] = (int32_t)token;
        P.parents[row0 + tid] = (int32_t)parent;
        P.scores_out[row0 + tid] = (float)double_of(picked_score[tid]);
        if (P.finished_out) P.finished_out[row0 + tid] = ended[parent] || (int64_t)token == P.eos;
    }
    if (!P.lineage_out) return;
    // the rows in pieces that fit the LDS, read whole before they are written (lineage_out may be lineage)
    const uint32_t* in = reinterpret_cast<const uint32_t*>(P.lineage + row0 * P.padded);
    uint32_t* out = reinterpret_cast<uint32_t*>(P.lineage_out + row0 * P.padded);
    const int words = (int)(P.padded / 4), piece = min(words, 3 * kPickRoom / W);
    for (int from = 0; from < words; from += piece) {
        const int width = min(piece, words - from), all = W * width;
        __syncthreads();
        for (int i = tid; i < all; i += kPickThreads) room[i] = in[(int64_t)(i / width) * words + from + i % width];
        __syncthreads();
        for (int i = tid; i < all; i += kPickThreads) {
            const int beam = i / width, word = from + i % width, parent = (int)(picked[beam] / (uint32_t)P.vocab);
            uint32_t four = room[parent * width + i % width];
            const int at = P.lens[row0 + parent];
            if (at >= 0 && at >> 2 == word) four = (four & ~(255u << (8 * (at & 3)))) | (uint32_t)beam << (8 * (at & 3));
            out[(int64_t)beam * words + word] = four;
        }
    }
}

} // namespace

extern "C" {

int izwi_decode_beam_select_f32(const float* logits, int64_t prompts, int64_t beams, int64_t vocab, const float* scores, const uint8_t* finished,
                                int64_t eos_token, int32_t* tokens, int32_t* parents, float* scores_out, uint8_t* finished_out, const uint8_t* lineage,
                                int64_t lineage_capacity, const int32_t* lens, uint8_t* lineage_out, void* stream_) {
    return qmm_guarded("izwi_decode_beam_select_f32", [&]() -> int {
    constexpr const char* what = "decode_beam_select";
    if (prompts < 0 || beams <= 0 || vocab <= 0)
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: bad shape [%lld, %lld, %lld]", what, (long long)prompts, (long long)beams, (long long)vocab);
    if (beams > kMaxBeams || vocab > 0x7fffffffLL / beams || prompts > 65535 / beams)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: %lld prompts of %lld beams over %lld tokens (at most 65535 beams, %d a prompt, and 2^31 candidates)", what,
                        (long long)prompts, (long long)beams, (long long)vocab, kMaxBeams);
    if (eos_token < -1 || eos_token >= vocab || (finished && eos_token < 0))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: end token %lld of %lld%s", what, (long long)eos_token, (long long)vocab,
                        finished ? " (finished beams need one)" : "");
    if ((lineage != nullptr) != (lineage_out != nullptr) || (lineage && (!lens || lineage_capacity <= 0 || lineage_capacity > 0x3fffffff)))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: lineage comes with its successor, the lengths and a capacity (%lld)", what, (long long)lineage_capacity);
    if (prompts == 0) return IZWI_QMM_OK;
    if (!logits || !scores || !tokens || !parents || !scores_out) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: NULL buffer", what);
    if (!kv_aligned(lineage, 4) || !kv_aligned(lineage_out, 4)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: lineage must be 4-byte aligned", what);
    QmmCallScope call;
    int device = 0, n_cus = 0;
    if (int rc = qmm_current_device(&device, &n_cus)) return rc;
    hipStream_t stream = (hipStream_t)stream_;
    BeamParams P{logits, scores, finished, tokens, parents, scores_out, finished_out, lineage, lineage_out, lens, nullptr, nullptr, (int)beams, (int)vocab,
                 0, eos_token, kv_padded(lineage_capacity)};
    P.chunks = (int)((vocab + kChunk - 1) / kChunk);
    const size_t parts = (size_t)prompts * beams * P.chunks;
    void* scratch = nullptr;
    KV_TRY(qmm_get_scratch(device, stream, parts * (sizeof(double2) + (size_t)beams * sizeof(uint64_t)), &scratch));
    P.sums = static_cast<double2*>(scratch);
    P.keys = reinterpret_cast<uint64_t*>(P.sums + parts);
    beam_chunk_kernel<<<dim3((unsigned)P.chunks, (unsigned)(prompts * beams)), kChunkThreads, 0, stream>>>(P);
    KV_TRY(hipGetLastError());
    beam_pick_kernel<<<(unsigned)prompts, kPickThreads, 0, stream>>>(P);
    KV_TRY(hipGetLastError());
    return IZWI_QMM_OK;
    });
}

} // extern "C"
