// One step of beam search: the best `beams` of beams * vocab candidates scores[w] + logits[w][t] - logsumexp(logits[w]),
// and the beams' lineage that follows.
//
// Two launches (few logits: one).  The first reads the logits once: a workgroup takes a chunk of a beam's row, keeps it in registers, and leaves its
// maximum, its sum of exponentials under that maximum and its best `beams` logits, largest first.  No more of a chunk can be
// among the best of its prompt.  The second, a workgroup per prompt, joins the chunks' sums, turns what is left into scores, picks
// the best and reorders the lineage.
//
// Sums and scores are f64: neighbours among 10^6 candidates lie closer than an f32 sum is exact, and which one is picked is
// a whole number.  Within a beam the order is the logits' own, in f32.
//
// Many logits are bound by the issue of vector instructions, half of them the exponentials in f64 (16 prompts of 8 beams over 151936
// tokens, 78 MB: 28 us, 2.8 TB/s, and 9 for the second launch); fewer by the launches and each one's chain of
// loads and barriers (4 beams of 151936: 5.7 and 5.6 us).
#include "kv_cache.h"
#include "qmm_lanes.h"
#include "qmm_records.h"

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

// NaN as -infinity, +infinity as the largest float (fmaxf and fminf pass over a NaN)
__device__ __forceinline__ float clean(float v) { return fminf(fmaxf(v, -INFINITY), 3.402823466e38f); }
// floats, doubles (no NaN) in the order of unsigned numbers, and back
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f); // (-0 as 0)
    return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o ^ ((int32_t)o < 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t order_of(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0); // (a finished beam's score may be -0)
    return u ^ ((int64_t)u < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double double_of(uint64_t o) {
    return __longlong_as_double((long long)(o ^ ((int64_t)o < 0 ? 1ull << 63 : ~0ull)));
}

// Of the numbers whose last LOW bits are zero the largest that `k` lanes' values reach, bit by bit (0 where fewer lanes hold a value).
template <int LOW>
__device__ __forceinline__ uint32_t kth_of_lanes(uint32_t v, int k) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= LOW; bit--) {
        const uint32_t trial = t | 1u << bit;
        if (__popcll(__ballot(v >= trial)) >= k) t = trial;
    }
    return t;
}

// in every lane
__device__ __forceinline__ double wave_sum(double v) {
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    v += dpp_d<0x140>(v);
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float wave_max(float v) { return qmm_max_lane_rows(row16_max(v)); }

constexpr int kChunkThreads = 256, kChunkRoom = 1024;
struct ChunkShared {
    uint64_t found[kChunkRoom];
    double sum[4];
    uint64_t best[4];
    float top[4];
    uint32_t threshold[4];
    unsigned n_found;
};

// A chunk of a beam's row by 256 threads (tid; PER logits each): its maximum, sum and best candidates.  Every thread of the workgroup
// calls it (barriers); without `on` it does nothing.
template <int PER>
__device__ __forceinline__ void beam_chunk(const BeamParams& P, int row, int chunk, bool on, ChunkShared& S, int tid) {
    constexpr int kChunk = kChunkThreads * PER;
    const int begin = chunk * kChunk, n = min(kChunk, P.vocab - begin), lane = tid & 63, wave = tid >> 6;
    uint64_t* keys = P.keys + ((int64_t)row * P.chunks + chunk) * P.beams;
    const float* x = P.logits + (int64_t)row * P.vocab + begin;
    float v[PER], m = -INFINITY;
    if (on) {
        if (n == kChunk) {
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] = x[tid + i * kChunkThreads];
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] = x[min(i * kChunkThreads + tid, n - 1)];
        }
        if (P.finished && P.finished[row]) on = false; // its candidate comes from neither
    }
    if (on && clean(P.scores[row]) == -INFINITY) { // every candidate of the beam is -infinity: the lowest tokens
        if (tid < P.beams) keys[tid] = tid < n ? (uint64_t)order_of(-INFINITY) << 32 | ~(uint32_t)(begin + tid) : 0;
        on = false;
    }
    if (tid == 0) S.n_found = 0;
    if (on) {
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = clean(v[i]);
        if (n != kChunk) {
            asm volatile(""); // (a branch)
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] = i * kChunkThreads + tid < n ? v[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < PER; i++) m = fmaxf(m, v[i]);
        // the largest value that as many lanes reach as there are beams: that many of the chunk's logits are no smaller
        // (to 12 bits of the mantissa: a threshold that lets a few more through, in fewer steps)
        const uint32_t kth = kth_of_lanes<11>(tid < n ? order_of(m) : 0, P.beams);
        m = wave_max(m);
        if (lane == 0) S.top[wave] = m, S.threshold[wave] = kth;
    }
    __syncthreads();
    const auto key_of = [&](int i) { return (uint64_t)order_of(v[i]) << 32 | ~(uint32_t)(begin + i * kChunkThreads + tid); };
    if (on) {
        m = fmaxf(fmaxf(S.top[0], S.top[1]), fmaxf(S.top[2], S.top[3]));
        const uint32_t t = max(max(S.threshold[0], S.threshold[1]), max(S.threshold[2], S.threshold[3]));
        // (the number of that order; an order below -infinity's is no float's)
        const float least = t <= order_of(-INFINITY) ? -INFINITY : value_of(t);
        // (Few pass, one or two lanes of a wave at a time: the counter's address is hidden from the compiler, which would otherwise work out one
        // addition for all of them in some 25 instructions.  What is behind the end is -infinity.)
        unsigned hidden = 0;
        asm("" : "+v"(hidden));
        const bool ends = n != kChunk && least == -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (v[i] >= least) {
                if (ends && i * kChunkThreads + tid >= n) continue;
                const unsigned at = atomicAdd(&S.n_found + hidden, 1u);
                if (at < kChunkRoom) S.found[at] = key_of(i);
            }
        double s = 0.0, s2 = 0.0; // (what is behind the end is -infinity: nothing)
        const double md = m;
#pragma unroll
        for (int i = 0; i < PER; i += 2) s += exp_of((double)v[i] - md), s2 += exp_of((double)v[i + 1] - md);
        s = wave_sum(m == -INFINITY ? 0.0 : s + s2); // (no number: nothing)
        if (lane == 0) S.sum[wave] = s;
    }
    __syncthreads();
    const int got = on ? (int)S.n_found : 0; // (in any order; the keys are all different)
    if (on) {
        if (tid == 0) P.sums[(int64_t)row * P.chunks + chunk] = make_double2((double)m, S.sum[0] + S.sum[1] + S.sum[2] + S.sum[3]);
        if (got <= kChunkRoom) {
            for (int i = tid; i < got; i += kChunkThreads) {
                const uint64_t key = S.found[i];
                int rank = 0;
                for (int j = 0; j < got; j++) rank += S.found[j] > key;
                if (rank < P.beams) keys[rank] = key;
            }
            if (tid >= got && tid < P.beams) keys[tid] = 0;
        }
    }
    if (!__syncthreads_or(got > kChunkRoom)) return;
    // a chunk of few different values: the largest, again and again
    uint64_t last = ~0ull;
    for (int k = 0; k < P.beams; k++) {
        uint64_t mine = 0;
        if (on) {
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (i * kChunkThreads + tid < n && key_of(i) < last) mine = max(mine, key_of(i));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mine = max(mine, (uint64_t)__shfl_xor((unsigned long long)mine, o));
        __syncthreads();
        if (lane == 0) S.best[wave] = mine;
        __syncthreads();
        last = max(max(S.best[0], S.best[1]), max(S.best[2], S.best[3]));
        if (tid == 0 && got > kChunkRoom) keys[k] = last;
    }
    __syncthreads();
}

template <int PER>
__global__ __launch_bounds__(kChunkThreads) void beam_chunk_kernel(BeamParams P) {
    __shared__ ChunkShared S;
    beam_chunk<PER>(P, blockIdx.y, blockIdx.x, true, S, threadIdx.x);
}

constexpr int kPickThreads = 1024, kPickRoom = 4096, kPickKept = 4; // candidates that a thread keeps in registers
constexpr int kAheadWords = 4096;                                   // of the lineage, read before they are needed

struct Candidate {
    uint64_t score; // order of the score
    uint32_t flat;  // beam * vocab + token
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) { return a.score > b.score || (a.score == b.score && a.flat < b.flat); }

// PER > 0: the chunks too, four at most
template <int PER>
__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamParams P) {
    __shared__ double offset[kMaxBeams]; // of a beam's logits: score - logsumexp
    __shared__ uint8_t ended[kMaxBeams];
    __shared__ uint32_t thresholds[kPickThreads / 64];
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
    const int per_beam = P.chunks * W, total = W * per_beam;
    // a lineage that fits is on its way from the start
    const int words = (int)(P.padded / 4);
    const bool ahead = P.lineage_out && (int64_t)W * words <= kAheadWords;
    const uint32_t* in = reinterpret_cast<const uint32_t*>(P.lineage + row0 * P.padded);
    uint32_t early[kAheadWords / kPickThreads];
    int len = 0;
    if (ahead) {
#pragma unroll
        for (int i = 0; i < kAheadWords / kPickThreads; i++) early[i] = in[min(tid + i * kPickThreads, W * words - 1)];
        len = P.lens[row0 + min(tid, W - 1)];
    }
    if constexpr (PER > 0) {
        static_assert(4 * sizeof(ChunkShared) <= sizeof(room));
        ChunkShared* S = reinterpret_cast<ChunkShared*>(room);
        const int group = tid / kChunkThreads, c = min(group, W * P.chunks - 1), w = c / P.chunks;
        beam_chunk<PER>(P, (int)row0 + w, c - w * P.chunks, group < W * P.chunks, S[group], tid % kChunkThreads);
        __syncthreads();
    }
    // the first candidates are requested before the sums are joined
    uint64_t kept[kPickKept];
    const uint64_t* all_keys = P.keys + row0 * per_beam;
#pragma unroll
    for (int c = 0; c < kPickKept; c++) kept[c] = all_keys[min(tid + c * kPickThreads, total - 1)];
    for (int w = wave; w < W; w += kPickThreads / 64) {
        const float score = clean(P.scores[row0 + w]);
        const bool end = P.finished && P.finished[row0 + w];
        double o = score;
        if (!end && score != -INFINITY) {
            const double2* part = P.sums + (row0 + w) * P.chunks;
            float m = -INFINITY; // (the chunks' maxima are floats)
            double s = 0.0;
            const double2 one = part[min(lane, P.chunks - 1)];
            for (int c = lane; c < P.chunks; c += 64) m = fmaxf(m, (float)(c == lane ? one : part[c]).x);
            m = wave_max(m);
            for (int c = lane; c < P.chunks; c += 64) {
                const double2 p = c == lane ? one : part[c];
                if (p.y != 0.0) s += p.y * exp_of(p.x - (double)m);
            }
            s = wave_sum(s);
            o = m == -INFINITY ? -INFINITY : (double)score - (double)m - log(s);
        }
        if (lane == 0) offset[w] = o, ended[w] = end;
    }
    if (tid == 0) n_found = 0;
    __syncthreads();
    // candidate i (score order 0: none) from its key
    auto candidate = [&](int i, uint64_t key) {
        Candidate c{0, 0xffffffffu};
        if (i >= total) return c;
        const int w = i / per_beam;
        if (ended[w]) {
            if (i == w * per_beam) c.score = order_of(offset[w]), c.flat = (uint32_t)w * P.vocab + (uint32_t)P.eos;
        } else if (key) {
            const float logit = value_of((uint32_t)(key >> 32));
            c.score = order_of(offset[w] == -INFINITY || logit == -INFINITY ? (double)-INFINITY : offset[w] + (double)logit);
            c.flat = (uint32_t)w * P.vocab + ~(uint32_t)key;
        }
        return c;
    };
    // scores rounded to f32 keep their order: the threshold is found among those
    const auto coarse = [&](const Candidate& c) { return c.score ? order_of((float)double_of(c.score)) : 0u; };
    Candidate mine[kPickKept];
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < kPickKept; c++) mine[c] = candidate(tid + c * kPickThreads, kept[c]), most = max(most, coarse(mine[c]));
    for (int i = tid + kPickKept * kPickThreads; i < total; i += kPickThreads) most = max(most, coarse(candidate(i, all_keys[i])));
    const uint32_t kth = kth_of_lanes<0>(most, W);
    if (lane == 0) thresholds[wave] = kth;
    __syncthreads();
    uint32_t t = 1;
#pragma unroll
    for (int i = 0; i < kPickThreads / 64; i++) t = max(t, thresholds[i]);
    const auto keep = [&](const Candidate& c) {
        if (coarse(c) < t) return;
        const unsigned at = atomicAdd(&n_found, 1u);
        if (at < kPickRoom) found_score[at] = c.score, found_flat[at] = c.flat;
    };
#pragma unroll
    for (int c = 0; c < kPickKept; c++) keep(mine[c]);
    for (int i = tid + kPickKept * kPickThreads; i < total; i += kPickThreads) keep(candidate(i, all_keys[i]));
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
                const Candidate c = candidate(i, all_keys[i]);
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
    uint32_t* out = reinterpret_cast<uint32_t*>(P.lineage_out + row0 * P.padded);
    // word `word` of the new beam's row: its parent's, with the beam itself at the parent's length
    const auto successor = [&](uint32_t four, int beam, int word, int at) {
        return at >= 0 && at >> 2 == word ? (four & ~(255u << (8 * (at & 3)))) | (uint32_t)beam << (8 * (at & 3)) : four;
    };
    if (ahead) {
        __syncthreads(); // (room has been read)
#pragma unroll
        for (int i = 0; i < kAheadWords / kPickThreads; i++)
            if (tid + i * kPickThreads < W * words) room[tid + i * kPickThreads] = early[i];
        if (tid < W) room[kAheadWords + tid] = (uint32_t)len;
        __syncthreads();
#pragma unroll
        for (int n = 0; n < kAheadWords / kPickThreads; n++) {
            const int i = tid + n * kPickThreads;
            if (i >= W * words) break;
            const int beam = i / words, word = i - beam * words, parent = (int)(picked[beam] / (uint32_t)P.vocab);
            out[i] = successor(room[parent * words + word], beam, word, (int)room[kAheadWords + parent]);
        }
        return;
    }
    // longer ones in pieces that fit the LDS, read whole before they are written (lineage_out may be lineage)
    const int piece = min(words, 3 * kPickRoom / W);
    for (int from = 0; from < words; from += piece) {
        const int width = min(piece, words - from), all = W * width;
        __syncthreads();
        for (int i = tid; i < all; i += kPickThreads) room[i] = in[(int64_t)(i / width) * words + from + i % width];
        __syncthreads();
        for (int i = tid; i < all; i += kPickThreads) {
            const int beam = i / width, word = from + i % width, parent = (int)(picked[beam] / (uint32_t)P.vocab);
            out[(int64_t)beam * words + word] = successor(room[parent * width + i % width], beam, word, P.lens[row0 + parent]);
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
    if (lineage && lineage != lineage_out) {
        const int64_t bytes = prompts * beams * kv_padded(lineage_capacity);
        if (kv_overlap(lineage, bytes, lineage_out, bytes)) return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: lineage and its successor overlap", what);
    }
    QmmCallScope call;
    int device = 0, n_cus = 0;
    if (int rc = qmm_current_device(&device, &n_cus)) return rc;
    hipStream_t stream = (hipStream_t)stream_;
    BeamParams P{logits, scores, finished, tokens, parents, scores_out, finished_out, lineage, lineage_out, lens, nullptr, nullptr, (int)beams, (int)vocab,
                 0, eos_token, kv_padded(lineage_capacity)};
    // 4096 logits to a workgroup, 2048 where that leaves fewer than two workgroups to a compute unit and the second launch few lists to look
    // through (4 prompts of 4 beams of 32000: 9.8 us in a graph instead of 10.3, 1 of 8: 12.0 instead of 11.5).  Up to four chunks of 2048 of
    // a prompt are taken by the second launch itself, side by side: one launch in all, 3 us less for the host (in a graph, where that counts for
    // nothing, 2 beams of 2051 take 9.3 us instead of 8.7, a second turn of four chunks 5 us more).
    const int64_t chunks = beams * ((vocab + 4095) / 4096);
    const bool one_launch = beams * ((vocab + 2047) / 2048) <= 4, small = one_launch || (chunks <= 32 && prompts * chunks < 2 * n_cus);
    const int chunk = small ? 2048 : 4096;
    P.chunks = (int)((vocab + chunk - 1) / chunk);
    const size_t parts = (size_t)prompts * beams * P.chunks;
    void* scratch = nullptr;
    KV_TRY(qmm_get_scratch(device, stream, parts * (sizeof(double2) + (size_t)beams * sizeof(uint64_t)), &scratch));
    P.sums = static_cast<double2*>(scratch);
    P.keys = reinterpret_cast<uint64_t*>(P.sums + parts);
    if (one_launch) {
        beam_pick_kernel<8><<<(unsigned)prompts, kPickThreads, 0, stream>>>(P);
        KV_TRY(hipGetLastError());
        return IZWI_QMM_OK;
    }
    const dim3 grid((unsigned)P.chunks, (unsigned)(prompts * beams));
    if (small) beam_chunk_kernel<8><<<grid, kChunkThreads, 0, stream>>>(P);
    else beam_chunk_kernel<16><<<grid, kChunkThreads, 0, stream>>>(P);
    KV_TRY(hipGetLastError());
    beam_pick_kernel<0><<<(unsigned)prompts, kPickThreads, 0, stream>>>(P);
    KV_TRY(hipGetLastError());
    return IZWI_QMM_OK;
    });
}

} // extern "C"
