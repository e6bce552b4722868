// kv_cache.hip - K/V caches in 16, 8 or 4 bits (types and quantiser: kv_cache.h) for gfx950:
//   kv_write     fp32 / fp16 rows -> cache rows; a lane owns eight dims, four lanes a scale block
//   kv_read      cache rows -> fp32 / fp16 rows
//   kv_compact   the accepted path's rows of a drafted tree to the front of the draft, for all caches of a model at once
//   prep_axes    per-head RMSNorm, rotary embedding with three position axes, and the K / V write of new tokens
// No counterpart in the reference, whose cache is fp16 (store_kv2_kernel, qw:340-345) and whose draft is one token.
#include "kv_rows.h"
#include "overlap.h"
#include "rope.h"

#include <algorithm>
#include <cmath>

namespace rmi {
namespace {

// ---- rows in and out ---------------------------------------------------------------------------------------------------
// Both are copies with a little arithmetic, bound by the memory they touch.  The unit is eight dims: 16 bytes of fp16,
// 8 bytes of I8 codes, one word of I4 codes.

constexpr int kRowThreads = 256;

// eight dims x to unit (row, kv, g) of the cache; the lanes of a row's 16 neighbouring units call together
template <int T, bool SRC16>
__device__ __forceinline__ void write_unit(uint8_t* __restrict__ cache, const F8& x, int p, int kv, int g, int n_kv, int head_dim, int max_ctx) {
    const KvRow<T> at = kv_row<T>(p, kv, n_kv, max_ctx, head_dim);
    if constexpr (T == kKvF16) {
        store8<true, true>(cache + at.code, 8 * g, x);
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x.v[i]) & 0x7fffffffu);
        m = max(m, xor_lane<1>(m));
        m = max(m, xor_lane<2>(m));
        const uint32_t sb = kv_scale_byte<T>(m);
        const float s = kv_scale_value(sb), inv = 1.0f / s;
        const float rest = kv_inverse_rest(s, inv);
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = kv_code<T, SRC16>(x.v[i], s, inv, rest);
        if constexpr (T == kKvI8) {
            // the low bytes of four words: pairs, then pairs of pairs
            auto pack = [](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                return __builtin_amdgcn_perm(__builtin_amdgcn_perm(a3, a2, 0x0c0c0400u), __builtin_amdgcn_perm(a1, a0, 0x0c0c0400u), 0x05040100u);
            };
            *reinterpret_cast<uint2*>(cache + at.code + 8 * g) = make_uint2(pack(c[0], c[1], c[2], c[3]), pack(c[4], c[5], c[6], c[7]));
        } else {
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) w |= (c[i] & 15u) << kv_i4_shift(i);
            *reinterpret_cast<uint32_t*>(cache + at.code + 4 * g) = w;
        }
        uint32_t w = sb | (xor_lane<4>(sb) << 8);   // in the lanes of block 0 of four
        w |= xor_lane<8>(w) << 16;
        if ((g & 15) == 0) *reinterpret_cast<uint32_t*>(cache + at.scale + (g >> 2)) = w;
    }
}

// Workgroup (rows, KV head), a row's heads side by side (together they read whole rows): the head's rows are neighbours in
// the cache, and no lane divides.  A lane takes units of two rows, both loads out before the first is used.  fp16 to I4,
// 65501 rows of 1024 dims: 43 us, 3.9 TB/s (the rows read back: 27 us, 6.3 TB/s).
constexpr int kWriteUnits = 2;

template <int T, bool SRC16, bool VEC>
__global__ __launch_bounds__(kRowThreads) void kv_write_kernel(const void* __restrict__ src, int src_stride,
                                                               uint8_t* __restrict__ cache, int first, int n, int n_kv,
                                                               int head_dim, int max_ctx) {
    const int shift = head_dim == 256 ? 5 : 4, up = kRowThreads >> shift;   // units per row 2^shift, rows a unit of the lane is further
    const int rows = blockIdx.x / n_kv, kv = blockIdx.x - rows * n_kv;
    const int g = static_cast<int>(threadIdx.x) & ((1 << shift) - 1);   // eight dims 8 g ..
    const int row0 = rows * (kWriteUnits * up) + (static_cast<int>(threadIdx.x) >> shift);
    F8 x[kWriteUnits];
#pragma unroll
    for (int k = 0; k < kWriteUnits; ++k)
        x[k] = load8<SRC16, VEC>(src, static_cast<size_t>(min(row0 + k * up, n - 1)) * src_stride + kv * head_dim + 8 * g);
#pragma unroll
    for (int k = 0; k < kWriteUnits; ++k)   // a row's lanes stay or go together
        if (row0 + k * up < n) write_unit<T, SRC16>(cache, x[k], first + row0 + k * up, kv, g, n_kv, head_dim, max_ctx);
}

template <int T, bool OUT16, bool VEC>
__global__ __launch_bounds__(kRowThreads) void kv_read_kernel(const uint8_t* __restrict__ cache, void* __restrict__ out,
                                                              int out_stride, int first, int n, int n_kv, int head_dim,
                                                              int max_ctx) {
    const int shift = head_dim == 256 ? 5 : 4;
    const int rows = blockIdx.x / n_kv, kv = blockIdx.x - rows * n_kv;
    const int g = static_cast<int>(threadIdx.x) & ((1 << shift) - 1);
    const int row = rows * (kRowThreads >> shift) + (static_cast<int>(threadIdx.x) >> shift);
    if (row >= n) return;
    const KvRow<T> at = kv_row<T>(first + row, kv, n_kv, max_ctx, head_dim);
    const F8 x = read_unit<T>(cache, at, g);
    store8<OUT16, VEC>(out, static_cast<size_t>(row) * out_stride + kv * head_dim + 8 * g, x);
}

// ---- the accepted path's rows --------------------------------------------------------------------------------------------
// Workgroup (cache, head): up to 64 rows of up to 512 bytes are read into registers, a barrier, then written, so a source
// row that is another's destination is read before it goes.  Latency-bound (pos, path, one read, one write): 3.5 us for 5 rows
// of 16 caches, 3.8 for 31 of two.
constexpr int kMaxPath = 64;
constexpr int kMaxCaches = 64;
constexpr int kMoves = kMaxPath * 32 / 256;   // 16-byte pieces per lane

struct CachePtrs {
    uint8_t* p[kMaxCaches];
};

template <int T>
__global__ __launch_bounds__(256) void kv_compact_kernel(CachePtrs caches, const int* __restrict__ pos,
                                                         const int* __restrict__ path, const int* __restrict__ count,
                                                         int max_path, int n_kv, int head_dim, int max_ctx) {
    __shared__ int from[kMaxPath];
    uint8_t* cache = caches.p[blockIdx.x];
    const int kv = blockIdx.y, tid = threadIdx.x;
    const int base = pos[0], n = min(max(count[0], 0), max_path);
    if (tid < n) {
        const long long s = static_cast<long long>(base) + path[tid], d = static_cast<long long>(base) + tid;
        from[tid] = s >= 0 && s < max_ctx && d >= 0 && d < max_ctx ? static_cast<int>(s) : -1;
    }
    __syncthreads();
    const int per = kv_row_bytes(T, head_dim) / 16, sper = T == kKvF16 ? 0 : head_dim / 128;   // pieces, scale words
    uint4 x[kMoves];
    uint32_t sc = 0;
#pragma unroll
    for (int k = 0; k < kMoves; ++k) {
        const int i = tid + 256 * k, r = i / per;
        x[k] = make_uint4(0, 0, 0, 0);
        if (r < n && from[r] >= 0)
            x[k] = *reinterpret_cast<const uint4*>(cache + kv_row<T>(from[r], kv, n_kv, max_ctx, head_dim).code + 16 * (i - r * per));
    }
    const int sr = T == kKvF16 ? n : tid / sper;
    if (sr < n && from[sr] >= 0)
        sc = *reinterpret_cast<const uint32_t*>(cache + kv_row<T>(from[sr], kv, n_kv, max_ctx, head_dim).scale + 4 * (tid - sr * sper));
    // every load has returned before any lane passes the barrier
#pragma unroll
    for (int k = 0; k < kMoves; ++k) asm volatile("" : "+v"(x[k].x), "+v"(x[k].y), "+v"(x[k].z), "+v"(x[k].w));
    asm volatile("" : "+v"(sc));
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMoves; ++k) {
        const int i = tid + 256 * k, r = i / per;
        if (r < n && from[r] >= 0)
            *reinterpret_cast<uint4*>(cache + kv_row<T>(base + r, kv, n_kv, max_ctx, head_dim).code + 16 * (i - r * per)) = x[k];
    }
    if (sr < n && from[sr] >= 0)
        *reinterpret_cast<uint32_t*>(cache + kv_row<T>(base + sr, kv, n_kv, max_ctx, head_dim).scale + 4 * (tid - sr * sper)) = sc;
}

// ---- norm, rotation, cache write ------------------------------------------------------------------------------------------
// Workgroup (token, part): the token's (cos, sin) per pair once into LDS, then a wave per head row, a lane HD / 64 neighbouring
// dims; a row's loads go out before the work on the row before it.  q: attn_prep's arithmetic and bits.  K: the same steps in
// fp64, rounded to fp32 once, so what the cache holds does not hang on the order of a sum.  The rotation's partner comes
// through the wave's LDS row; a scale block is 8 (HD 256) or 16 lanes.
constexpr int kPrepWaves = 4;

struct PrepArgs {
    const float* q3;
    int q3_stride;
    const float *qn, *kn;
    uint8_t *kc, *vc;
    const int *pos, *axis_pos;
    float* qout;
    int n_head, n_kv, n_rot, max_ctx, ntok, per_wave;
    float theta, eps;
    Yarn yarn;
    rmi_rope_axes axes;
};

__device__ __forceinline__ int rope_axis(const rmi_rope_axes& a, int i) {
    if (a.interleaved) {
        const int m = i % 3;
        return m == 1 && i < 3 * a.section[1] ? 1 : m == 2 && i < 3 * a.section[2] ? 2 : 0;
    }
    return i < a.section[0] ? 0 : i < a.section[0] + a.section[1] ? 1 : 2;
}

// the sum of the squares of a row, as attn_prep takes it: per 64 dims a butterfly over the dim's bits from 32 down (its first
// step contracted: fma(x_d, x_d, x_{d + 32}^2) for d < 32), the 64-dim sums in order.  A dim's low bits are its place in
// the lane.
template <int N>
__device__ __forceinline__ float square_sum(const float (&x)[N]) {
    constexpr int L = 32 / N;   // lanes between d and d + 32
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = __builtin_fmaf(x[j], x[j], xor_lane<L>(x[j] * x[j]));
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if constexpr (L > 8) v[j] += xor_lane<8>(v[j]);
        if constexpr (L > 4) v[j] += xor_lane<4>(v[j]);
        v[j] += xor_lane<2>(v[j]);
        v[j] += xor_lane<1>(v[j]);
    }
    const float s = N == 4 ? (v[0] + v[2]) + (v[1] + v[N - 1]) : v[0] + v[1];
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 64 / (2 * L); ++k) t += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s), 2 * L * k));
    return t;
}

template <int KT, int VT, int HD>
__global__ __launch_bounds__(64 * kPrepWaves) void prep_axes_kernel(PrepArgs a) {
    constexpr int N = HD / 64;
    __shared__ double cs[HD / 2][2];
    __shared__ float2 csf[HD / 2];   // rounded, for q
    __shared__ __attribute__((aligned(16))) double rows[kPrepWaves][HD];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), d0 = N * lane;
    const int base = a.pos[0], half = a.n_rot / 2;
    const float* src = a.q3 + static_cast<size_t>(t) * a.q3_stride;
    const int items = a.n_head + 2 * a.n_kv, first = (blockIdx.y * kPrepWaves + wv) * a.per_wave;
    const int end = min(first + a.per_wave, items);
    float nx[N], wq[N], wk[N];   // nx: the next row
    auto load = [&](int it) {
        it = min(it, items - 1);
        load_dims(nx, (it < a.n_head ? src + it * 2 * HD : src + 2 * a.n_head * HD + (it - a.n_head) * HD) + d0);   // [q | gate] .., k, v
    };
    load(first);
    load_dims(wq, a.qn + d0);
    load_dims(wk, a.kn + d0);
    if (base < -t || base >= a.max_ctx - t) return;   // uniform: a slot outside the cache stores nothing
    const int p = base + t;
    if (tid < half) {
        const int ap = a.axis_pos ? a.axis_pos[static_cast<size_t>(rope_axis(a.axes, tid)) * a.ntok + t] : p;
        double c, s;
        rope_cos_sin_d(ap, rope_freq(tid, a.n_rot, a.theta), tid, a.yarn, &c, &s);
        cs[tid][0] = c;
        cs[tid][1] = s;
        csf[tid] = make_float2(static_cast<float>(c), static_cast<float>(s));
    }
    __syncthreads();
    for (int it = first; it < end; ++it) {
        float x[N];
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = nx[j];
        if (it + 1 < end) load(it + 1);
        if (it >= a.n_head + a.n_kv) {
            store_row<VT, HD>(x, a.vc, p, it - a.n_head - a.n_kv, a.n_kv, a.max_ctx, lane);
        } else if (it < a.n_head) {
            float* xs = reinterpret_cast<float*>(rows[wv]);
            const float inv = rsqrtf(square_sum<N>(x) / static_cast<float>(HD) + a.eps);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[j] = x[j] * inv * wq[j];
                xs[d0 + j] = x[j];
            }
            wave_lds_sync();
            if (d0 < a.n_rot) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int d = d0 + j;
                    if (d >= a.n_rot) break;
                    const float2 e = csf[d < half ? d : d - half];
                    x[j] = d < half ? rope_lo(x[j], xs[d + half], e.x, e.y) : rope_hi(xs[d - half], x[j], e.x, e.y);
                }
            }
            wave_lds_sync();   // the next row overwrites the exchange
            float* to = a.qout + (static_cast<size_t>(t) * a.n_head + it) * HD + d0;
            if constexpr (N == 4) *reinterpret_cast<float4u*>(to) = float4u{x[0], x[1], x[2], x[N - 1]};
            else *reinterpret_cast<float2u*>(to) = float2u{x[0], x[1]};
        } else {
            double* xs = rows[wv];
            double y[N], ss = 0.0;
#pragma unroll
            for (int j = 0; j < N; ++j) ss += static_cast<double>(x[j]) * static_cast<double>(x[j]);
            const double inv = 1.0 / sqrt(group_sum64(ss) / HD + static_cast<double>(a.eps));
#pragma unroll
            for (int j = 0; j < N; ++j) {
                y[j] = static_cast<double>(x[j]) * inv * static_cast<double>(wk[j]);
                xs[d0 + j] = y[j];
            }
            wave_lds_sync();
            if (d0 < a.n_rot) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int d = d0 + j;
                    if (d >= a.n_rot) break;
                    const int i = d < half ? d : d - half;
                    y[j] = d < half ? y[j] * cs[i][0] - xs[d + half] * cs[i][1] : xs[d - half] * cs[i][1] + y[j] * cs[i][0];
                }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = static_cast<float>(y[j]);
            wave_lds_sync();
            store_row<KT, HD>(x, a.kc, p, it - a.n_head, a.n_kv, a.max_ctx, lane);
        }
    }
}

constexpr long long kMaxBlocks = 0xffffffffLL / kRowThreads;   // a launch's work-items along an axis are a 32-bit number
static_assert(kRowThreads == 64 * kPrepWaves);

bool aligned_to(const void* p, size_t n) { return p && (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// whether rows outside share bytes with the cache's of positions [first, first + n)
bool on_cache_rows(int type, const void* rows, int rows16, int stride, const void* cache, int first, int n, int n_kv, int head_dim, int max_ctx) {
    const long long el = rows16 ? 2 : 4, heads = n_kv, ctx = max_ctx, per = kv_row_bytes(type, head_dim), sper = head_dim / kKvBlock;
    const RowSet out{rows, n, stride * el, heads * head_dim * el};
    const auto* c = static_cast<const uint8_t*>(cache);
    if (type == kKvF16) return rows_overlap(out, block_of(c + heads * per * first, heads * per * n));
    return rows_overlap(out, {c + per * first, heads, ctx * per, per * n}) ||
           rows_overlap(out, {c + heads * ctx * per + sper * first, heads, ctx * sper, sper * n});
}

int row_args(const char* what, int type, const void* cache, const void* rows, int rows16, int stride, int first, int n,
             int n_kv, int head_dim, int max_ctx) {
    if (!kv_type_ok(type)) return fail(RMI_ERR_UNSUPPORTED, what);
    if (!kv_shape_ok(max_ctx, n_kv, head_dim) || first < 0 || n < 0 || n > max_ctx || first > max_ctx - n ||
        static_cast<long long>(n_kv) * head_dim > stride)
        return fail(RMI_ERR_SHAPE, what);
    if (!aligned16(cache) || !aligned_to(rows, rows16 ? 2 : 4)) return fail(RMI_ERR_POINTER, what);
    return RMI_OK;
}

}  // namespace
}  // namespace rmi

using namespace rmi;

extern "C" size_t rmi_kv_cache_bytes(int type, int max_ctx, int n_kv, int head_dim) {
    if (!kv_type_ok(type) || !kv_shape_ok(max_ctx, n_kv, head_dim)) {
        set_error("kv_cache_bytes: type F16, I8 or I4, positive max_ctx and n_kv, head_dim 128 or 256");
        return 0;
    }
    const size_t rows = static_cast<size_t>(max_ctx) * n_kv;
    return rows * kv_row_bytes(type, head_dim) + (type == kKvF16 ? 0 : rows * (head_dim / kKvBlock));
}

extern "C" int rmi_kv_write(int type, const void* src, int src_f16, int src_stride, void* cache, int first, int n,
                            int n_kv, int head_dim, int max_ctx, void* stream) {
    RMI_TRY(row_args("kv_write: invalid arguments", type, cache, src, src_f16, src_stride, first, n, n_kv, head_dim, max_ctx));
    if (n == 0) return RMI_OK;
    const int per = kWriteUnits * kRowThreads / (head_dim / 8);   // rows a workgroup
    const long long blocks = (static_cast<long long>(n) + per - 1) / per * n_kv;
    if (blocks > kMaxBlocks) return fail(RMI_ERR_SHAPE, "kv_write: too many rows for one call");
    if (on_cache_rows(type, src, src_f16, src_stride, cache, first, n, n_kv, head_dim, max_ctx))
        return fail(RMI_ERR_POINTER, "kv_write: the source lies on the rows it goes to");
    const bool vec = aligned16(src) && src_stride % (src_f16 ? 8 : 4) == 0;   // 16-byte loads, else one by one
    auto* out = static_cast<uint8_t*>(cache);
    return with_type(type, [&](auto t) {
        auto go = [&](auto* kernel) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), src,
                               src_stride, out, first, n, n_kv, head_dim, max_ctx);
            return launch_status("kv_write");
        };
        constexpr int T = decltype(t)::value;
        if (src_f16) return vec ? go(&kv_write_kernel<T, true, true>) : go(&kv_write_kernel<T, true, false>);
        return vec ? go(&kv_write_kernel<T, false, true>) : go(&kv_write_kernel<T, false, false>);
    });
}

extern "C" int rmi_kv_read(int type, const void* cache, void* out, int out_f16, int out_stride, int first, int n,
                           int n_kv, int head_dim, int max_ctx, void* stream) {
    RMI_TRY(row_args("kv_read: invalid arguments", type, cache, out, out_f16, out_stride, first, n, n_kv, head_dim, max_ctx));
    if (n == 0) return RMI_OK;
    const int per = kRowThreads / (head_dim / 8);
    const long long blocks = (static_cast<long long>(n) + per - 1) / per * n_kv;
    if (blocks > kMaxBlocks) return fail(RMI_ERR_SHAPE, "kv_read: too many rows for one call");
    if (on_cache_rows(type, out, out_f16, out_stride, cache, first, n, n_kv, head_dim, max_ctx))
        return fail(RMI_ERR_POINTER, "kv_read: the output lies on the rows it comes from");
    const bool vec = aligned16(out) && out_stride % (out_f16 ? 8 : 4) == 0;
    const auto* in = static_cast<const uint8_t*>(cache);
    return with_type(type, [&](auto t) {
        auto go = [&](auto* kernel) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), in,
                               out, out_stride, first, n, n_kv, head_dim, max_ctx);
            return launch_status("kv_read");
        };
        constexpr int T = decltype(t)::value;
        if (out_f16) return vec ? go(&kv_read_kernel<T, true, true>) : go(&kv_read_kernel<T, true, false>);
        return vec ? go(&kv_read_kernel<T, false, true>) : go(&kv_read_kernel<T, false, false>);
    });
}

extern "C" int rmi_kv_compact(int type, void* const* caches, int n_caches, const int* pos, const int* path,
                              const int* count, int max_path, int n_kv, int head_dim, int max_ctx, void* stream) {
    if (!kv_type_ok(type)) return fail(RMI_ERR_UNSUPPORTED, "kv_compact: unknown cache type");
    if (!kv_shape_ok(max_ctx, n_kv, head_dim) || n_caches < 1 || n_caches > kMaxCaches || max_path < 1 || max_path > kMaxPath)
        return fail(RMI_ERR_SHAPE, "kv_compact: invalid arguments");
    if (!caches || !aligned4(pos) || !aligned4(path) || !aligned4(count))
        return fail(RMI_ERR_POINTER, "kv_compact: invalid arguments");
    CachePtrs ptrs{};
    const size_t bytes = rmi_kv_cache_bytes(type, max_ctx, n_kv, head_dim);
    for (int i = 0; i < n_caches; ++i) {
        if (!aligned16(caches[i])) return fail(RMI_ERR_POINTER, "kv_compact: null or misaligned cache");
        ptrs.p[i] = static_cast<uint8_t*>(caches[i]);
        for (int j = 0; j < i; ++j)   // two workgroups would move the same rows
            if (rows_overlap(block_of(caches[i], bytes), block_of(caches[j], bytes)))
                return fail(RMI_ERR_POINTER, "kv_compact: caches overlap");
    }
    return with_type(type, [&](auto t) {
        hipLaunchKernelGGL((kv_compact_kernel<decltype(t)::value>), dim3(n_caches, n_kv), dim3(256), 0,
                           static_cast<hipStream_t>(stream), ptrs, pos, path, count, max_path, n_kv, head_dim, max_ctx);
        return launch_status("kv_compact");
    });
}

extern "C" int rmi_attn_prep_axes(const float* q3, int q3_stride, const float* qn, const float* kn, int ktype,
                                  void* kcache, int vtype, void* vcache, const int* pos, const int* axis_pos, float* qout,
                                  int n_head, int n_kv, int head_dim, int n_rot, const rmi_rope_params* rope,
                                  const rmi_rope_axes* axes, float eps, int ntok, int max_ctx, void* stream) {
    const char* what = "attn_prep_axes: invalid arguments";
    if (!kv_type_ok(ktype) || !kv_type_ok(vtype)) return fail(RMI_ERR_UNSUPPORTED, "attn_prep_axes: unknown cache type");
    if (!kv_shape_ok(max_ctx, n_kv, head_dim) || n_head <= 0 || n_head > 65535 || n_head % n_kv || n_rot < 0 || n_rot > head_dim || n_rot % 2 ||
        ntok < 1 || ntok > max_ctx || ntok > kMaxBlocks || !rope || !(rope->freq_base > 1.0f) || !axes ||
        2LL * n_head * head_dim + 2LL * n_kv * head_dim > 0x7fffffffLL)
        return fail(RMI_ERR_SHAPE, what);
    const int* s = axes->section;
    const int half = n_rot / 2;
    if (s[0] < 0 || s[1] < 0 || s[2] < 0 || s[0] > half || s[1] > half || s[2] > half || s[0] + s[1] + s[2] != half)
        return fail(RMI_ERR_SHAPE, "attn_prep_axes: the axes' sections must add up to n_rot / 2");
    // dealt out in turn, the last pairs of axes 1 and 2 are 3 s - 2 and 3 s - 1
    if (axes->interleaved && ((s[1] > 0 && 3 * s[1] - 2 >= half) || (s[2] > 0 && 3 * s[2] - 1 >= half)))
        return fail(RMI_ERR_SHAPE, "attn_prep_axes: an interleaved axis has more pairs than its turns");
    if (!aligned4(q3) || !aligned4(qn) || !aligned4(kn) || !aligned16(kcache) || !aligned16(vcache) || !aligned4(pos) ||
        (axis_pos && !aligned4(axis_pos)) || !aligned4(qout))
        return fail(RMI_ERR_POINTER, what);
    const RowSet read{q3, ntok, 4LL * q3_stride, 4LL * (2 * n_head + 2 * n_kv) * head_dim};
    const RowSet written[] = {block_of(kcache, rmi_kv_cache_bytes(ktype, max_ctx, n_kv, head_dim)),
                              block_of(vcache, rmi_kv_cache_bytes(vtype, max_ctx, n_kv, head_dim)),
                              block_of(qout, static_cast<size_t>(ntok) * n_head * head_dim * 4)};
    if (rows_overlap(written[0], written[1])) return fail(RMI_ERR_POINTER, "attn_prep_axes: the caches overlap");
    if (rows_overlap(written[2], written[0]) || rows_overlap(written[2], written[1]))
        return fail(RMI_ERR_POINTER, "attn_prep_axes: qout lies on a cache");
    for (const RowSet& w : written)
        if (rows_overlap(read, w)) return fail(RMI_ERR_POINTER, "attn_prep_axes: qout or a cache lies on the rows of q3");
    PrepArgs a{};
    if (!yarn_setup(*rope, n_rot, &a.yarn)) return fail(RMI_ERR_SHAPE, "attn_prep_axes: invalid YaRN parameters");
    a.q3 = q3;
    a.q3_stride = q3_stride;
    a.qn = qn;
    a.kn = kn;
    a.kc = static_cast<uint8_t*>(kcache);
    a.vc = static_cast<uint8_t*>(vcache);
    a.pos = pos;
    a.axis_pos = axis_pos;
    a.qout = qout;
    a.n_head = n_head;
    a.n_kv = n_kv;
    a.n_rot = n_rot;
    a.max_ctx = max_ctx;
    a.ntok = ntok;
    a.theta = rope->freq_base;
    a.eps = eps;
    a.axes = *axes;
    const int items = n_head + 2 * n_kv;
    // rows a wave: as many as leave about a thousand workgroups (they share a token's angles), one for few tokens (latency).
    // 999 tokens, 24 rows each: 1 / 3 / 6 rows a wave 19.6 / 15.9 / 14.4 us
    a.per_wave = std::min((items + kPrepWaves - 1) / kPrepWaves, static_cast<int>((static_cast<long long>(items) * ntok + 4095) / 4096));
    const int parts = (items + kPrepWaves * a.per_wave - 1) / (kPrepWaves * a.per_wave);
    return with_type(ktype, [&](auto k) {
        return with_type(vtype, [&](auto v) {
            auto go = [&](auto* kernel) {
                hipLaunchKernelGGL(kernel, dim3(ntok, parts), dim3(64 * kPrepWaves), 0, static_cast<hipStream_t>(stream), a);
                return launch_status("attn_prep_axes");
            };
            constexpr int KT = decltype(k)::value, VT = decltype(v)::value;
            return head_dim == 256 ? go(&prep_axes_kernel<KT, VT, 256>) : go(&prep_axes_kernel<KT, VT, 128>);
        });
    });
}
