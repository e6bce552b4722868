// kv_cache.h - the K/V cache types behind rmi_kv_*, rmi_attn_prep_axes and rmi_gqa_tree_decode: row addresses, the
// quantiser of one 32-dim block and the constants of the code formats.
//
// I8 and I4 scales carry four significant bits and codes at most seven, so code * scale has at most eleven: every value
// of a quantised cache is an fp16 number, subnormals included (the scale grid's step is 2^-17, fp16's 2^-24).  The
// attention then runs on fp16 operands without a rounding of its own, and a cache read back to fp16 loses nothing.  The
// price is the scale rounded up to four bits: 6 % of the step on average (0.09 bits) against a 16-bit scale, at one byte
// a block instead of two.
#pragma once

#include <cfloat>

#include "rmi_common.h"

namespace rmi {

constexpr int kKvF16 = RMI_KV_F16, kKvI8 = RMI_KV_I8, kKvI4 = RMI_KV_I4;
constexpr int kKvBlock = 32;   // dims that share a scale

__host__ __device__ constexpr int kv_qmax(int type) { return type == kKvI8 ? 127 : 7; }
__host__ __device__ constexpr int kv_bias(int type) { return type == kKvI8 ? 128 : 8; }
__host__ __device__ constexpr uint32_t kv_top_scale(int type) { return type == kKvI8 ? 192u : 224u; }   // 512 / 8192
// code bytes of one (position, head) row
__host__ __device__ constexpr int kv_row_bytes(int type, int head_dim) {
    return type == kKvF16 ? 2 * head_dim : type == kKvI8 ? head_dim : head_dim / 2;
}

inline bool kv_type_ok(int type) { return type == kKvF16 || type == kKvI8 || type == kKvI4; }
constexpr int kKvMaxCtx = 1 << 30;   // positions and a step past them fit an int
inline bool kv_shape_ok(int max_ctx, int n_kv, int head_dim) {
    return max_ctx > 0 && max_ctx <= kKvMaxCtx && n_kv > 0 && n_kv <= 65535 && (head_dim == 128 || head_dim == 256);
}

// one row of a cache; offsets are 64-bit (a long cache passes 2^32 bytes)
template <int T>
struct KvRow {
    size_t code;    // byte offset of the row's codes (F16: of its halves)
    size_t scale;   // byte offset of its scale bytes
};
template <int T>
__device__ __forceinline__ KvRow<T> kv_row(int p, int kv, int n_kv, int max_ctx, int head_dim) {
    KvRow<T> r;
    if constexpr (T == kKvF16) {
        r.code = (static_cast<size_t>(p) * n_kv + kv) * (2 * head_dim);
        r.scale = 0;
    } else {
        const size_t row = static_cast<size_t>(kv) * max_ctx + p;
        r.code = row * kv_row_bytes(T, head_dim);
        r.scale = static_cast<size_t>(n_kv) * max_ctx * kv_row_bytes(T, head_dim) + row * (head_dim / kKvBlock);
    }
    return r;
}

__device__ __forceinline__ float kv_scale_value(uint32_t byte) { return half_bits_to_float(byte << 7); }

// The scale byte of a block whose largest |x| has the bits amax_bits (an integer maximum, so that a NaN is kept): the
// smallest grid number s with Q s >= amax.  amax / Q is rounded up to the grid; where the division rounded down onto the
// grid, Q s (exact) is below amax and the next number is taken.
template <int T>
__device__ __forceinline__ uint32_t kv_scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 0xffu;   // fp16 0x7f80: NaN
    constexpr float kQ = static_cast<float>(kv_qmax(T));
    const float amax = __uint_as_float(amax_bits);
    const float t = amax / kQ;
    uint32_t b;
    if (t < 0x1p-14f) b = static_cast<uint32_t>(__builtin_ceilf(t * 0x1p17f));
    else b = ((__float_as_uint(t) + 0xfffffu) >> 20) - (112u << 3);
    b = b < kv_top_scale(T) ? b : kv_top_scale(T);
    if (b < kv_top_scale(T) && kQ * kv_scale_value(b) < amax) ++b;
    return b;
}

// 1 / s in two parts (inv + rest, exact to 2^-46)
__device__ __forceinline__ float kv_inverse_rest(float s, float inv) { return __builtin_fmaf(-inv, s, 1.0f) * inv; }

// code + bias, in the result's low byte: x / s to the nearest integer, half to even, as if divided exactly.  The two-part
// inverse gives x / s rounded to fp32 once, y.  Where y is no half-integer, rounding y is rounding x / s; where it is one, the
// remainder x - y s (exact: y s has 12 bits) tells whether x / s is.  For x that are fp16 numbers (X16) it always is: x / s is
// a multiple of 2^-12 of itself over a divisor of at most 15, so nothing but a tie comes near one.
template <int T, bool X16 = false>
__device__ __forceinline__ uint32_t kv_code(float x, float s, float inv, float rest) {
    constexpr float kQ = static_cast<float>(kv_qmax(T));
    float y = __builtin_fmaf(x, inv, x * rest);
    if constexpr (!X16) {
        if (__builtin_amdgcn_fractf(fabsf(y)) == 0.5f) {
            const float r = __builtin_fmaf(-y, s, x);
            y += r > 0.0f ? 0.25f : r < 0.0f ? -0.25f : 0.0f;
        }
    }
    const float k = __builtin_amdgcn_fmed3f(y, -kQ, kQ) + (8388608.0f + kv_bias(T));   // rounds to an integer, half to even
    return s > 0.0f ? __float_as_uint(k) : static_cast<uint32_t>(kv_bias(T));          // an empty block, or a NaN scale: 0
}

// where code + bias of dim d goes in the word of its eight dims (I4)
__device__ __forceinline__ int kv_i4_shift(int d) { return 4 * ((d & 7) >> 1) + 16 * (d & 1); }

}  // namespace rmi
