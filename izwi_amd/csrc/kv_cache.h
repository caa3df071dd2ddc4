// The quantized key / value cache: layout and the helpers that its writer, its reader and the attention over it share.
//
// A cache holds, for every (slot, kv head), `capacity` positions (rounded up to 32) of a key row and a value row of D
// values, quantized in blocks of 32 along the row: an f16 scale per block and a quant of 8 (Q8_0) or 4 (Q4_0) bits per
// value.  Four planes one behind the other: key quants, key scales, value quants, value scales.  Key scales are
// [slot][kv head][position][D / 32], value scales [slot][kv head][position / 2][D / 32][2].  The quants of a (slot, kv head) stand where the lanes of a wave want them as matrix-core operands, so that
// a load brings 16 bytes to every lane from neighbouring addresses and no value moves between lanes.  (With rows of positions
// instead, the lanes' 16-byte pieces of the keys are 128 bytes apart and each is an access to the L1 of its own: 662 accesses per 32
// positions, which bound the attention of sixteen rows a kv head.)
//  * keys: lane (x, g) of the wave (x of sixteen, g of four) multiplies of position 16 t + x the values 8 g .. 8 g + 7 of
//    every block, a unit of 8 bytes (Q8_0) or 4 (Q4_0).  Units that fill 16 bytes are neighbours (a piece): [16 positions][piece][g][x].
//  * values: lane (x, g) takes of positions 4 g .. 4 g + 3 of 16 the values 2 x and 2 x + 1 of every block.  A dword holds
//    16 bits of an even position, then 16 bits of the next: two values (Q8_0: of block j) or four (Q4_0: of blocks 2 j and 2 j + 1).
//    [4 positions][pieces of 16 bytes][x].
// Q8_0 quants are stored + 128, Q4_0 ones + 8: an unsigned byte or nibble under the exponent of 1024 is an f16, and one
// subtraction (exact) leaves the quant.  The eight nibbles of a key unit go in the order 0 2 4 6 1 3 5 7: bits 0-3 and
// 16-19 of the unit, shifted right by 4 r, are the values 2 r and 2 r + 1, a register of the operand.
#ifndef IZWI_KV_CACHE_H
#define IZWI_KV_CACHE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/izwi_decode_ops.h"
#include "qmm_internal.h"

namespace {

constexpr int kKvBlock = 32, kKvPad = 32;

struct KvPlanes {
    uint8_t *kq, *vq;
    _Float16 *ks, *vs;
    int64_t kv_heads, padded; // (slot, head) begins at position (slot * kv_heads + head) * padded of every plane
};
inline int64_t kv_padded(int64_t capacity) { return (capacity + kKvPad - 1) / kKvPad * kKvPad; }
inline int64_t kv_row_bytes(int type, int64_t d) { return type == IZWI_KV_Q8_0 ? d : d / 2; }
inline int64_t kv_plane_bytes(int64_t rows, int64_t row_bytes) { return (rows * row_bytes + 255) / 256 * 256; }
inline KvPlanes kv_planes(int type, const void* cache, int64_t slots, int64_t kv_heads, int64_t capacity, int64_t d) {
    KvPlanes p{};
    p.kv_heads = kv_heads, p.padded = kv_padded(capacity);
    const int64_t rows = slots * kv_heads * p.padded;
    uint8_t* at = static_cast<uint8_t*>(const_cast<void*>(cache));
    if (!at) return p;
    const int64_t quants = kv_plane_bytes(rows, kv_row_bytes(type, d)), scales = kv_plane_bytes(rows, d / 16);
    p.kq = at, p.ks = reinterpret_cast<_Float16*>(at + quants);
    p.vq = at + quants + scales, p.vs = reinterpret_cast<_Float16*>(at + 2 * quants + scales);
    return p;
}
// A cache that exists: a format and a head size that are built, sizes whose bytes are counted in 63 bits.  Zero or a status.
inline int kv_check_shape(const char* what, int type, int64_t slots, int64_t kv_heads, int64_t capacity, int64_t d) {
    if (type != IZWI_KV_Q8_0 && type != IZWI_KV_Q4_0)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: cache type %d (Q4_0 = 2 and Q8_0 = 8 are built)", what, type);
    if (d != 64 && d != 128 && d != 256)
        return qmm_fail(IZWI_QMM_ERR_UNSUPPORTED, "%s: head_dim %lld (64, 128 and 256 are built)", what, (long long)d);
    if (slots <= 0 || kv_heads <= 0 || capacity <= 0 || slots > 0xfffff || kv_heads > 0xffff || capacity > 0x3fffffff ||
        slots * kv_heads > (int64_t(1) << 50) / (kv_padded(capacity) * d))
        return qmm_fail(IZWI_QMM_ERR_INVALID, "%s: bad cache shape (slots %lld, kv heads %lld, capacity %lld)", what, (long long)slots,
                        (long long)kv_heads, (long long)capacity);
    return IZWI_QMM_OK;
}
inline bool kv_aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
inline bool kv_overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}

#define KV_TRY(expr)                                                                      \
    do {                                                                                  \
        hipError_t e_ = (expr);                                                           \
        if (e_ != hipSuccess) {                                                           \
            (void)hipGetLastError();                                                      \
            return qmm_fail(IZWI_QMM_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_));    \
        }                                                                                 \
    } while (0)

template <int QT, int D>
struct KvRow {
    static constexpr int kBlocks = D / kKvBlock;
    static constexpr int kBytes = QT == IZWI_KV_Q8_0 ? D : D / 2; // of a position's keys, or values
    static constexpr int kUnit = QT == IZWI_KV_Q8_0 ? 8 : 4;
    static constexpr int kPer = 16 / kUnit < kBlocks ? 16 / kUnit : kBlocks, kPiece = kPer * kUnit; // units, bytes of a key piece
    static constexpr int kLane = kBytes / 16;                        // bytes of a position's values that lane x takes
    static constexpr int kValuePiece = 4 * kLane < 16 ? 4 * kLane : 16; // of four positions' values
    // scales from the first position of the slot and head to that of block b of the values
    static __host__ __device__ constexpr int64_t value_scale(int64_t pos, int b) { return ((pos >> 1) * kBlocks + b) * 2 + (pos & 1); }
    // bytes from there to the unit of block b, lane group g of the keys, and to
    // the 16 bits j of lane x of the values
    static __host__ __device__ constexpr int64_t key(int64_t pos, int b, int g) {
        return (pos >> 4) * (16 * kBytes) + (b / kPer) * (64 * kPiece) + (g * 16 + (int)(pos & 15)) * kPiece + (b % kPer) * kUnit;
    }
    static __host__ __device__ constexpr int64_t value(int64_t pos, int x, int j) {
        const int at = (int)(pos >> 1 & 1) * (2 * kLane) + 4 * j + 2 * (int)(pos & 1);
        return (pos >> 2) * (4 * kBytes) + (at / kValuePiece) * (16 * kValuePiece) + x * kValuePiece + at % kValuePiece;
    }
};

} // namespace

#endif // IZWI_KV_CACHE_H
