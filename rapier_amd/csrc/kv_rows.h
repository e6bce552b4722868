// kv_rows.h - rows of fp32 / fp16 in and out of cache rows of any type: the parts that the calls on contiguous caches and on pages
// share.  A page is a cache of page_size positions.
#pragma once

#include <type_traits>

#include "kv_cache.h"

namespace rmi {

struct F8 {
    float v[8];
};

template <bool SRC16, bool VEC>
__device__ __forceinline__ F8 load8(const void* src, size_t e) {
    F8 x;
    if constexpr (SRC16) {
        const auto* p = static_cast<const uint16_t*>(src) + e;
        if constexpr (VEC) {
            const uint4 w = *reinterpret_cast<const uint4*>(p);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x.v[2 * i] = half_bits_to_float(ws[i]);
                x.v[2 * i + 1] = half_bits_to_float(ws[i] >> 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = half_bits_to_float(p[i]);
        }
    } else {
        const auto* p = static_cast<const float*>(src) + e;
        if constexpr (VEC) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            x = {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = p[i];
        }
    }
    return x;
}

__device__ __forceinline__ uint32_t half_bits(float v) {
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v)));
}

template <bool OUT16, bool VEC>
__device__ __forceinline__ void store8(void* out, size_t e, const F8& x) {
    if constexpr (OUT16) {
        auto* p = static_cast<uint16_t*>(out) + e;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = half_bits(x.v[2 * i]) | (half_bits(x.v[2 * i + 1]) << 16);
        if constexpr (VEC) {
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
        }
    } else {
        auto* p = static_cast<float*>(out) + e;
        if constexpr (VEC) {
            reinterpret_cast<float4*>(p)[0] = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = x.v[i];
        }
    }
}

// orders a wave's own LDS accesses
__device__ __forceinline__ void wave_lds_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ double group_sum64(double v) {
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) v += __shfl_xor(v, k, 64);
    return v;
}

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));   // rows of a caller's stride
typedef float float2u __attribute__((ext_vector_type(2), aligned(4)));

template <int N>
__device__ __forceinline__ void load_dims(float (&x)[N], const float* p) {
    if constexpr (N == 4) {
        const float4u v = *reinterpret_cast<const float4u*>(p);
        x[0] = v[0], x[1] = v[1], x[2] = v[2], x[3] = v[3];
    } else {
        const float2u v = *reinterpret_cast<const float2u*>(p);
        x[0] = v[0], x[1] = v[1];
    }
}

// the wave's row (lane: dims N lane + 0 .. N - 1) into position p of a cache
template <int T, int HD>
__device__ __forceinline__ void store_row(const float (&x)[HD / 64], uint8_t* cache, int p, int kv, int n_kv, int max_ctx,
                                          int lane) {
    constexpr int N = HD / 64;
    const KvRow<T> at = kv_row<T>(p, kv, n_kv, max_ctx, HD);
    const int d = N * lane;
    if constexpr (T == kKvF16) {
        uint32_t w[N / 2];
#pragma unroll
        for (int j = 0; j < N; j += 2) w[j / 2] = half_bits(x[j]) | (half_bits(x[j + 1]) << 16);
        if constexpr (N == 4) *reinterpret_cast<uint2*>(cache + at.code + 2 * d) = make_uint2(w[0], w[N / 2 - 1]);
        else *reinterpret_cast<uint32_t*>(cache + at.code + 2 * d) = w[0];
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
        if constexpr (N == 2) m = max(m, xor_lane<8>(m));
        m = max(m, xor_lane<4>(m));
        m = max(m, xor_lane<2>(m));
        m = max(m, xor_lane<1>(m));
        const uint32_t sb = kv_scale_byte<T>(m);
        const float s = kv_scale_value(sb), inv = 1.0f / s, rest = kv_inverse_rest(s, inv);
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t c = kv_code<T>(x[j], s, inv, rest) & (T == kKvI8 ? 0xffu : 0xfu);
            w |= c << (T == kKvI8 ? 8 * j : kv_i4_shift(d + j));
        }
        if constexpr (T == kKvI8) {
            if constexpr (N == 4) *reinterpret_cast<uint32_t*>(cache + at.code + d) = w;
            else *reinterpret_cast<uint16_t*>(cache + at.code + d) = static_cast<uint16_t>(w);
        } else {
            w |= xor_lane<1>(w);
            if constexpr (N == 2) w |= xor_lane<2>(w);
            if ((d & 7) == 0) *reinterpret_cast<uint32_t*>(cache + at.code + d / 2) = w;
        }
        if ((d & 31) == 0) cache[at.scale + d / 32] = static_cast<uint8_t>(sb);
    }
}

// eight dims 8 g .. of a cache row
template <int T>
__device__ __forceinline__ F8 read_unit(const uint8_t* __restrict__ cache, const KvRow<T>& at, int g) {
    F8 x;
    if constexpr (T == kKvF16) {
        x = load8<true, true>(cache + at.code, 8 * g);
    } else {
        const float s = kv_scale_value(cache[at.scale + (g >> 2)]);
        if constexpr (T == kKvI8) {
            const uint2 w = *reinterpret_cast<const uint2*>(cache + at.code + 8 * g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = ((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xffu;
                x.v[i] = static_cast<float>(static_cast<int>(b) - kv_bias(T)) * s;
            }
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(cache + at.code + 4 * g);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x.v[i] = static_cast<float>(static_cast<int>((w >> kv_i4_shift(i)) & 15u) - kv_bias(T)) * s;
        }
    }
    return x;
}

// calls f with the type as a constant
template <typename F>
int with_type(int type, F&& f) {
    if (type == kKvI8) return f(std::integral_constant<int, kKvI8>{});
    if (type == kKvI4) return f(std::integral_constant<int, kKvI4>{});
    return f(std::integral_constant<int, kKvF16>{});
}

}  // namespace rmi
