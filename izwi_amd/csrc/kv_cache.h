// The quantized key / value cache: layout and the helpers that its writer, its reader and the attention over it share.
//
// A cache holds, for every (slot, kv head), `capacity` positions (rounded up to 32) of a key row and a value row of D
// values, quantized in blocks of 32 along the row: an f16 scale per block and a quant of 8 (Q8_0) or 4 (Q4_0) bits per
// value.  Four planes one behind the other, [slot][kv head][position][row bytes] each: key quants, key scales, value
// quants, value scales; a position's scales are its D / 32 halves in order.
//
// The quants of a row stand where the matrix-core operands of the attention want them, so that it loads whole pieces
// and never moves a value between lanes:
//  * keys: lane group g (of four) multiplies the values 8 g .. 8 g + 7 of every block: these are one unit of 8 bytes (Q8_0) or
//    4 (Q4_0), and the units that one lane takes are neighbours, up to 16 bytes of them.
//  * values: lane x (of sixteen) takes the values 2 x and 2 x + 1 of every block: its D / 16 quants are neighbours.
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
    int64_t kv_heads, padded; // row (slot, head, position) = (slot * kv_heads + head) * padded + position of every plane
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
    static constexpr int kBytes = QT == IZWI_KV_Q8_0 ? D : D / 2;
    static constexpr int kUnit = QT == IZWI_KV_Q8_0 ? 8 : 4;
    static constexpr int kPer = 16 / kUnit < kBlocks ? 16 / kUnit : kBlocks; // units of a lane that are neighbours
    static constexpr int kLaneBytes = kBytes / 16;                          // of a value row, per lane x
    // where the unit of block b, lane group g of a key row begins
    static __host__ __device__ constexpr int unit(int b, int g) { return ((b / kPer) * 4 + g) * kPer * kUnit + (b % kPer) * kUnit; }
};

} // namespace

#endif // IZWI_KV_CACHE_H
