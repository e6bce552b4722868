// kv_operand.h - cache rows of any type as fp16 MFMA operands: codes to fp16, loads of a lane's dims, fp32 values in two parts,
// and what is done about values that are not finite.  Shared by the attention kernels.
#pragma once

#include "kv_cache.h"

namespace rmi {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));   // rows of a caller's stride

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
__device__ __forceinline__ half2v h2(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ uint32_t u2(half2v h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ half8 h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(half8, u32x4{a, b, c, d});
}

// Codes become fp16 by one fused multiply-add a pair: the code is put into the mantissa of a power of two (I8: 1024 + u,
// I4: 64 + u), and fma(x, s / 16, -bias s / 16) is code * s / 16 exactly (u is code + 128 or code + 8; a sixteenth keeps the
// addend an fp16 number up to the largest scale, and every value above fp16's smallest step).  The sixteenths come out of
// the scores' factor and the joined rows' weights.
template <int T>
constexpr float kSixteen = T == kKvF16 ? 1.0f : 16.0f;

struct Scale2 {
    half2v s, c;
};
// the scales of a pair's two values, from their scale bytes (I8 and I4)
template <int T>
__device__ __forceinline__ Scale2 scale2(uint32_t lo, uint32_t hi) {
    constexpr _Float16 kBias = static_cast<_Float16>(T == kKvI8 ? -1152.0f : -72.0f), kPart = static_cast<_Float16>(0.0625f);
    Scale2 r;
    r.s = h2((lo << 7) | (hi << 23)) * half2v{kPart, kPart};
    r.c = r.s * half2v{kBias, kBias};
    return r;
}
// The first scale byte whose addend is past fp16's largest number (199 for I8, 231 for I4): a block with it or a larger one has
// no finite value here.  The quantiser writes none but 255, the NaN's; unwritten memory holds any.
template <int T>
constexpr uint32_t kOddScale = kv_top_scale(T) + 7;
// what every value of such a block is (NaN); zero for the others
template <int T>
__device__ __forceinline__ float odd_value(uint32_t byte) { return byte < kOddScale<T> ? 0.0f : __builtin_nanf(""); }
__device__ __forceinline__ uint32_t fma2(uint32_t x, const Scale2& s) { return u2(__builtin_elementwise_fma(h2(x), s.s, s.c)); }

// (w & mask) | magic in one instruction: with both as literals the compiler takes two
__device__ __forceinline__ uint32_t nibbles(uint32_t w) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(0x00f000f0u), "v"(0x54005400u));
    return r;
}
// pair k of a word of eight I4 codes, at bits 4..7 of both halves
__device__ __forceinline__ uint32_t nibble_pair(uint32_t w, int k) { return nibbles(k == 0 ? w << 4 : w >> (4 * (k - 1))); }
constexpr uint32_t kMagic8 = 0x64646464u;   // high byte of the fp16 numbers 1024 + 0..255

typedef __amdgpu_buffer_rsrc_t Rsrc;

// 16 neighbouring dims of a position
template <int T>
struct Dims16 {
    uint32_t w[T == kKvF16 ? 8 : T == kKvI8 ? 4 : 2];
};
template <int T>
__device__ __forceinline__ Dims16<T> load16(Rsrc r, int lane_at, int at) {
    Dims16<T> x;
    if constexpr (T == kKvI4) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, lane_at, at, 0);
        x.w[0] = v[0], x.w[1] = v[1];
    } else {
#pragma unroll
        for (int i = 0; i < (T == kKvF16 ? 2 : 1); ++i) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, lane_at + 16 * i, at, 0);
            x.w[4 * i] = v[0], x.w[4 * i + 1] = v[1], x.w[4 * i + 2] = v[2], x.w[4 * i + 3] = v[3];
        }
    }
    return x;
}
// dims 8 hf + 0..7 of them as an MFMA operand
template <int T>
__device__ __forceinline__ half8 operand(const Dims16<T>& x, int hf, const Scale2& s) {
    if constexpr (T == kKvF16) {
        return h8(x.w[4 * hf], x.w[4 * hf + 1], x.w[4 * hf + 2], x.w[4 * hf + 3]);
    } else {
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kKvI8) r[i] = fma2(perm(kMagic8, x.w[2 * hf + (i >> 1)], i & 1 ? 0x04030402u : 0x04010400u), s);
            else r[i] = fma2(nibble_pair(x.w[hf], i), s);
        }
        return h8(r[0], r[1], r[2], r[3]);
    }
}

// A lane's VD dims of a position: in runs of 16 bytes at most, lane l's k-th run at byte kRun * (16 k + l), so that 16 lanes
// read whole lines
template <int T, int VD>
struct DimsV {
    static constexpr int kBytes = T == kKvF16 ? 2 * VD : T == kKvI8 ? VD : VD / 2, kRun = kBytes < 16 ? kBytes : 16;
    static constexpr int kRunDims = VD * kRun / kBytes;
    static __device__ __forceinline__ int dim(int l16, int e) { return kRunDims * (16 * (e / kRunDims) + l16) + e % kRunDims; }
    uint32_t w[kBytes / 4];
};
template <int T, int VD>
__device__ __forceinline__ DimsV<T, VD> load_dims(Rsrc r, int lane_at, int at) {
    DimsV<T, VD> x;
    constexpr int kB = DimsV<T, VD>::kBytes;
    if constexpr (kB >= 16) {
#pragma unroll
        for (int i = 0; i < kB / 16; ++i) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, lane_at + 256 * i, at, 0);
            x.w[4 * i] = v[0], x.w[4 * i + 1] = v[1], x.w[4 * i + 2] = v[2], x.w[4 * i + 3] = v[3];
        }
    } else if constexpr (kB == 8) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, lane_at, at, 0);
        x.w[0] = v[0], x.w[1] = v[1];
    } else {
        x.w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, lane_at, at, 0);
    }
    return x;
}
// dims 2 e and 2 e + 1 of two positions a, b as halves (a, b), scaled by s = the scales of a and b
template <int T, int VD>
__device__ __forceinline__ void v_pair(const DimsV<T, VD>& a, const DimsV<T, VD>& b, int e, const Scale2& s, uint32_t& even, uint32_t& odd) {
    if constexpr (T == kKvF16) {
        even = perm(b.w[e], a.w[e], 0x05040100u);
        odd = perm(b.w[e], a.w[e], 0x07060302u);
    } else if constexpr (T == kKvI8) {
        const uint32_t m = perm(b.w[e >> 1], a.w[e >> 1], e & 1 ? 0x07030602u : 0x05010400u);   // a0 b0 a1 b1
        even = fma2(perm(kMagic8, m, 0x04010400u), s);
        odd = fma2(perm(kMagic8, m, 0x04030402u), s);
    } else {
        // even dims are in a word's low half, odd ones in the high half
        even = fma2(nibble_pair(perm(b.w[e >> 2], a.w[e >> 2], 0x05040100u), e & 3), s);
        odd = fma2(nibble_pair(perm(b.w[e >> 2], a.w[e >> 2], 0x07060302u), e & 3), s);
    }
}

__device__ __forceinline__ floatx4 mfma(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// fp16 high part of eight fp32 values, and what is left of them
__device__ __forceinline__ void split8(const float (&x)[8], half8& hi, half8& lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const _Float16 h = static_cast<_Float16>(x[j]);
        hi[j] = h;
        lo[j] = static_cast<_Float16>(x[j] - static_cast<float>(h));
    }
}

__device__ __forceinline__ bool finite16(uint32_t w) {   // both halves
    return (w & 0x7c00u) != 0x7c00u && (w & 0x7c000000u) != 0x7c000000u;
}
// the larger magnitudes of two words of fp16, half by half, as bits
__device__ __forceinline__ uint32_t max_magnitude(uint32_t m, uint32_t w) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
// a word of fp16 V without its infinities and NaN
__device__ __forceinline__ uint32_t zero_odd(uint32_t w) {
    if ((w & 0x7c00u) == 0x7c00u) w &= 0xffff0000u;
    if ((w & 0x7c000000u) == 0x7c000000u) w &= 0xffffu;
    return w;
}

// the power of two that brings a row's largest |q| to [2^13, 2^14), as its exponent
__device__ __forceinline__ int q_shift(float amax) {
    if (!(amax > 0.0f && amax <= FLT_MAX)) return 0;
    return min(14 - __builtin_amdgcn_frexp_expf(amax), 126);
}

}  // namespace rmi
