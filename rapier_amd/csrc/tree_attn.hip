// tree_attn.hip - attention of a tree (or chain) of drafted tokens over a K/V cache in 16, 8 or 4 bits, for gfx950
// (rmi_gqa_tree_decode; caches: kv_cache.h).  No counterpart in the reference, whose draft is one token (gqa_head_kernel,
// qw:384-442, per column).
//
//   partial   workgroup (chunk of 128 nsub positions, KV head, group of 16 query rows); row r = token r / G, head r % G of
//             the KV head's G.  Each of the four waves streams a quarter of the chunk in steps of 32 positions with a
//             running maximum, sum and output per row, and the four are joined at the end: one record (m, l, o) a row.
//   merge     workgroup (token, head): joins the chunks' records, gates, writes fp32 and Q8_1.
//
// Both products run on v_mfma_f32_16x16x32_f16 (lane: l16 = l % 16, g4 = l / 16; A rows, B and D columns are l16; A and B
// hold k = 8 g4 + 0..7; D rows are 4 g4 + 0..3).  The cache's values are fp16 numbers in every type; the fp32 operand
// (q, p) goes as fp16 high + low part, 22 bits, in two products, so the result keeps fp32's accuracy.
//   scores    D[position][row] += K[position][dims] . q[row][dims]: lane (l16, g4) takes 16 neighbouring dims of position
//             l16 at a time, 64 i + 16 g4 + [0, 16), as two operands of eight, straight from the cache.
//   P V       D[row][dim] += P[row][positions] V[positions][dim]: the score lane (row l16, positions 4 g4 + r of two tiles)
//             holds P in the A layout already, k slot j being position 4 g4 + j or 16 + 4 g4 + j - 4.  V comes by lane
//             (l16, g4) as HD / 16 neighbouring dims of those eight positions; operand e gathers dim e of the eight.
// The scores' exponent is base 2 (q is scaled by log2 e once).
//
// What a token does not see has no part in it: scores are masked before the maximum, and in the steps that reach into the
// draft a V that is not finite is taken out of the product and added to the rows that see it alone (an infinity times a
// masked zero would be NaN).
#include <algorithm>
#include <cmath>

#include "kv_cache.h"

namespace rmi {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;          // query rows of a group
constexpr int kWaves = 4;
constexpr int kStep = 32;          // positions of a step
constexpr int kUnit = kWaves * kStep;
constexpr int kMaxChunks = 2048;
constexpr int kMaxTree = 64, kMaxChain = 1024;

struct TreeArgs {
    const float* q;
    const uint8_t *kc, *vc;
    const int* pos;
    const uint64_t* masks;
    float *wo, *wml;   // records: o [chunk][kv][row][HD], (m, l) [chunk][kv][row][2]
    int n_head, n_kv, ntok, rows, rows_pad, groups, npairs, nsub, max_ctx;
    float scale;
};

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
__device__ __forceinline__ half2v h2(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ uint32_t u2(half2v h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ half8 h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(half8, u32x4{a, b, c, d});
}

constexpr uint32_t kMagic = 0x64646464u;   // high byte of the fp16 numbers 1024 + 0..255
__device__ __forceinline__ half2v bias2(int type) {
    const _Float16 b = static_cast<_Float16>(1024 + kv_bias(type));
    return half2v{b, b};
}
// two scales (bytes 0 and 1 of w, spread to the halves) as fp16
__device__ __forceinline__ half2v scale2(uint32_t lo, uint32_t hi) { return h2((lo << 7) | (hi << 23)); }

// 16 neighbouring dims of one position's K
template <int T>
struct Dims16 {
    uint32_t w[T == kKvF16 ? 8 : T == kKvI8 ? 4 : 2];
};
template <int T>
__device__ __forceinline__ Dims16<T> load_k16(const uint8_t* p) {
    Dims16<T> x;
    if constexpr (T == kKvI4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        x.w[0] = v.x, x.w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < (T == kKvF16 ? 2 : 1); ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            x.w[4 * i] = v.x, x.w[4 * i + 1] = v.y, x.w[4 * i + 2] = v.z, x.w[4 * i + 3] = v.w;
        }
    }
    return x;
}
// dims 8 hf + 0..7 of them as an MFMA operand
template <int T>
__device__ __forceinline__ half8 k_operand(const Dims16<T>& x, int hf, half2v s) {
    if constexpr (T == kKvF16) {
        return h8(x.w[4 * hf], x.w[4 * hf + 1], x.w[4 * hf + 2], x.w[4 * hf + 3]);
    } else if constexpr (T == kKvI8) {
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = perm(kMagic, x.w[2 * hf + (i >> 1)], i & 1 ? 0x04030402u : 0x04010400u);
            r[i] = u2((h2(c) - bias2(T)) * s);
        }
        return h8(r[0], r[1], r[2], r[3]);
    } else {
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = ((x.w[hf] >> (4 * i)) & 0x000f000fu) | 0x64006400u;
            r[i] = u2((h2(c) - bias2(T)) * s);
        }
        return h8(r[0], r[1], r[2], r[3]);
    }
}

// VD neighbouring dims of one position's V
template <int T, int VD>
struct DimsV {
    static constexpr int kBytes = T == kKvF16 ? 2 * VD : T == kKvI8 ? VD : VD / 2;
    uint32_t w[kBytes / 4];
};
template <int T, int VD>
__device__ __forceinline__ DimsV<T, VD> load_v(const uint8_t* p) {
    DimsV<T, VD> x;
    constexpr int kB = DimsV<T, VD>::kBytes;
    if constexpr (kB >= 16) {
#pragma unroll
        for (int i = 0; i < kB / 16; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            x.w[4 * i] = v.x, x.w[4 * i + 1] = v.y, x.w[4 * i + 2] = v.z, x.w[4 * i + 3] = v.w;
        }
    } else if constexpr (kB == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        x.w[0] = v.x, x.w[1] = v.y;
    } else {
        x.w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    return x;
}
// dims 2 e and 2 e + 1 of two positions a, b as halves (a, b), scaled by s = (scale of a, scale of b)
template <int T, int VD>
__device__ __forceinline__ void v_pair(const DimsV<T, VD>& a, const DimsV<T, VD>& b, int e, half2v s, uint32_t& even, uint32_t& odd) {
    if constexpr (T == kKvF16) {
        even = perm(b.w[e], a.w[e], 0x05040100u);
        odd = perm(b.w[e], a.w[e], 0x07060302u);
    } else if constexpr (T == kKvI8) {
        const uint32_t m = perm(b.w[e >> 1], a.w[e >> 1], e & 1 ? 0x07030602u : 0x05010400u);   // a0 b0 a1 b1
        even = u2((h2(perm(kMagic, m, 0x04010400u)) - bias2(T)) * s);
        odd = u2((h2(perm(kMagic, m, 0x04030402u)) - bias2(T)) * s);
    } else {
        // even dims are in a word's low half, odd ones in the high half
        const uint32_t lo = perm(b.w[e >> 2], a.w[e >> 2], 0x05040100u), hi = perm(b.w[e >> 2], a.w[e >> 2], 0x07060302u);
        const int k = 4 * (e & 3);
        even = u2((h2(((lo >> k) & 0x000f000fu) | 0x64006400u) - bias2(T)) * s);
        odd = u2((h2(((hi >> k) & 0x000f000fu) | 0x64006400u) - bias2(T)) * s);
    }
}

__device__ __forceinline__ floatx4 mfma(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// fp16 high and low parts of eight fp32 values
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

template <int KT, int VT, int HD>
__global__ __launch_bounds__(64 * kWaves, 1) void tree_partial_kernel(TreeArgs a) {
    constexpr int NI = HD / 64;        // K: 16-dim pieces a lane takes of a position
    constexpr int VD = HD / 16;        // V: dims a lane takes of a position
    constexpr int NB = HD / kKvBlock;  // scale bytes of a row
    constexpr int kKB = kv_row_bytes(KT, HD), kVB = kv_row_bytes(VT, HD);
    __shared__ __attribute__((aligned(16))) float ob[kWaves / 2][kRows][HD];   // joins; V of a step that is not finite
    __shared__ float pb[kWaves][kRows][kStep];
    __shared__ float stat[kWaves][2][kRows];

    // the groups of a (chunk, head) pair are consecutive workgroups of one XCD (workgroups go to the XCDs round robin),
    // so the pair's rows come from HBM once
    const int k8 = static_cast<int>(blockIdx.x >> 3), q8 = k8 / a.groups;
    const int group = k8 - q8 * a.groups, pair = 8 * q8 + static_cast<int>(blockIdx.x & 7);
    if (pair >= a.npairs) return;
    const int chunk = pair / a.n_kv, kv = pair - chunk * a.n_kv;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l16 = lane & 15, g4 = lane >> 4;
    const int G = a.n_head / a.n_kv;
    const int base = a.pos[0];
    if (base < 0 || base > a.max_ctx - a.ntok) return;   // uniform: a slot outside the cache
    const int row = kRows * group + l16, rowc = min(row, a.rows - 1), tok = rowc / G;
    // the last position any row of the group sees
    const int last = a.masks ? base + a.ntok - 1 : base + min(kRows * group + kRows - 1, a.rows - 1) / G;
    const int wlen = kStep * a.nsub, cbase = chunk * kWaves * wlen;
    if (cbase > last) return;   // uniform; the merge does not read this record
    uint64_t mask = 0;   // of the row's token: bit j = draft slot base + j
    if (a.masks && row < a.rows) mask = a.masks[tok];
    const int lim = row >= a.rows ? -1 : a.masks ? base - 1 : base + tok;   // the row sees every position up to here

    half8 qh[NI][2], ql[NI][2];
    {
        const float* qr = a.q + (static_cast<size_t>(tok) * a.n_head + kv * G + (rowc - tok * G)) * HD + 16 * g4;
        const float c = a.scale * 1.44269504088896340736f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const float4 u = reinterpret_cast<const float4*>(qr + 64 * i + 8 * hf)[0];
                const float4 v = reinterpret_cast<const float4*>(qr + 64 * i + 8 * hf)[1];
                const float x[8] = {u.x * c, u.y * c, u.z * c, u.w * c, v.x * c, v.y * c, v.z * c, v.w * c};
                split8(x, qh[i][hf], ql[i][hf]);
            }
    }

    // the head's rows: position p at kp + p * kstride
    const size_t kstride = KT == kKvF16 ? static_cast<size_t>(a.n_kv) * kKB : kKB;
    const size_t vstride = VT == kKvF16 ? static_cast<size_t>(a.n_kv) * kVB : kVB;
    const uint8_t* kp = a.kc + kv_row<KT>(0, kv, a.n_kv, a.max_ctx, HD).code + g4 * (kKB / (HD / 16));
    const uint8_t* vp = a.vc + kv_row<VT>(0, kv, a.n_kv, a.max_ctx, HD).code + l16 * DimsV<VT, VD>::kBytes;
    const uint8_t* ks = a.kc + kv_row<KT>(0, kv, a.n_kv, a.max_ctx, HD).scale;
    const uint8_t* vs = a.vc + kv_row<VT>(0, kv, a.n_kv, a.max_ctx, HD).scale + VD * l16 / kKvBlock;

    Dims16<KT> kx[2][NI];
    uint32_t ksc[2][2];
    DimsV<VT, VD> vx[8];
    uint32_t vsc[8];
    const int wbase = cbase + wv * wlen;
    const int nsteps = wbase > last ? 0 : min(a.nsub, (last - wbase) / kStep + 1);
    auto load_k = [&](int sb) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const size_t p = min(sb + 16 * t + l16, last);   // rows past the last are masked
#pragma unroll
            for (int i = 0; i < NI; ++i) kx[t][i] = load_k16<KT>(kp + p * kstride + i * (kKB / NI));
            if constexpr (KT != kKvF16) {
                if constexpr (NB == 8) {
                    const uint2 s = *reinterpret_cast<const uint2*>(ks + p * NB);
                    ksc[t][0] = s.x, ksc[t][1] = s.y;
                } else {
                    ksc[t][0] = *reinterpret_cast<const uint32_t*>(ks + p * NB);
                }
            }
        }
    };
    auto load_vs = [&](int sb) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const size_t p = min(sb + 4 * g4 + (j < 4 ? j : 12 + j), last);
            vx[j] = load_v<VT, VD>(vp + p * vstride);
            if constexpr (VT != kKvF16) vsc[j] = vs[p * NB];
        }
    };

    floatx4 o[VD];
#pragma unroll
    for (int e = 0; e < VD; ++e) o[e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l_run = 0.0f;   // l_run: this lane's positions only

    if (nsteps > 0) {
        load_k(wbase);
        load_vs(wbase);
    }
    for (int st = 0; st < nsteps; ++st) {
        const int sb = wbase + st * kStep;
        float sc[8];   // j: position sb + 4 g4 + j, or 16 further from j = 4 on
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            floatx4 dh = {0.0f, 0.0f, 0.0f, 0.0f}, dl = dh;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                half2v s = {};
                if constexpr (KT != kKvF16) {   // block 2 i + g4 / 2
                    const uint32_t b = (ksc[t][i >> 1] >> (16 * (i & 1) + 8 * (g4 >> 1))) & 0xffu;
                    s = scale2(b, b);
                }
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const half8 kk = k_operand<KT>(kx[t][i], hf, s);
                    dh = mfma(kk, qh[i][hf], dh);
                    dl = mfma(kk, ql[i][hf], dl);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[4 * t + r] = dh[r] + dl[r];
        }
        const bool more = st + 1 < nsteps;
        if (more) load_k(sb + kStep);
        const bool tail = sb + kStep > base;   // uniform: the step reaches into the draft
        uint32_t seen = 0xffu;
        if (tail || row >= a.rows) {
            seen = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int p = sb + 4 * g4 + (j < 4 ? j : 12 + j);
                bool ok = p <= lim;
                if (mask && p >= base && p - base < a.ntok) ok = ok || ((mask >> (p - base)) & 1);
                if (ok) seen |= 1u << j;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sc[j] = seen >> j & 1 ? sc[j] : -INFINITY;
        }
        float mloc = sc[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mloc = fmaxf(mloc, sc[j]);
        mloc = fmaxf(mloc, xor_lane<16>(mloc));
        mloc = fmaxf(mloc, xor_lane<32>(mloc));
        const float m_new = fmaxf(m_run, mloc);
        const float m_ref = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: exp2(-inf) = 0, no NaN
        const float alpha = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_ref);
        float p[8], lsum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = __builtin_amdgcn_exp2f(sc[j] - m_ref);
            lsum += p[j];
        }
        l_run = l_run * alpha + lsum;
        m_run = m_new;
        if (__ballot(alpha != 1.0f)) {   // uniform: some row's maximum moved
            float al[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) al[r] = __shfl(alpha, 4 * g4 + r, 64);
#pragma unroll
            for (int e = 0; e < VD; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[e][r] *= al[r];
        }
        half8 ph, pl;
        split8(p, ph, pl);
        half2v vsp[4];
        if constexpr (VT != kKvF16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) vsp[j] = scale2(vsc[2 * j], vsc[2 * j + 1]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) vsp[j] = half2v{};
        }
        if (tail) {
            // V rows that are not finite (of tokens that others do not see, or never written): zeroed in the product and
            // added by hand to the rows that see them
            bool odd = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (VT != kKvF16) {
                    odd = odd || !finite16(u2(vsp[j]));
                } else {
#pragma unroll
                    for (int e = 0; e < VD / 2; ++e) odd = odd || !finite16(vx[2 * j].w[e]) || !finite16(vx[2 * j + 1].w[e]);
                }
            }
            if (__ballot(odd)) {
                float* pw = &pb[wv][0][0];   // [row][position in the step], -1 where not seen
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    pw[l16 * kStep + 4 * g4 + (j < 4 ? j : 12 + j)] = seen >> j & 1 ? p[j] : -1.0f;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // this lane's dims of its position j, one lane group after another
                    for (int g = 0; g < 4; ++g) {
#pragma unroll
                        for (int e = 0; e < VD; ++e) {
                            float v;
                            if constexpr (VT == kKvF16) v = half_bits_to_float(vx[j].w[e >> 1] >> (16 * (e & 1)));
                            else v = static_cast<float>(vsp[j >> 1][j & 1]);   // a NaN scale: every value of the block
                            v = __shfl(v, 16 * g + l16, 64);
                            if (!(fabsf(v) <= FLT_MAX)) {
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    const float w = pw[(4 * g4 + r) * kStep + 4 * g + (j < 4 ? j : 12 + j)];
                                    if (w >= 0.0f || w != w) o[e][r] = __builtin_fmaf(w, v, o[e][r]);
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if constexpr (VT == kKvF16) {
#pragma unroll
                        for (int e = 0; e < VD / 2; ++e) {
                            uint32_t& w = vx[j].w[e];
                            if ((w & 0x7c00u) == 0x7c00u) w &= 0xffff0000u;
                            if ((w & 0x7c000000u) == 0x7c000000u) w &= 0xffffu;
                        }
                    } else if (!finite16(u2(vsp[j >> 1]) >> (16 * (j & 1)) & 0xffffu)) {
                        vsp[j >> 1][j & 1] = static_cast<_Float16>(0.0f);
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        }
#pragma unroll
        for (int e = 0; e < VD / 2; ++e) {
            uint32_t ev[4], od[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v_pair<VT, VD>(vx[2 * j], vx[2 * j + 1], e, vsp[j], ev[j], od[j]);
            const half8 b0 = h8(ev[0], ev[1], ev[2], ev[3]), b1 = h8(od[0], od[1], od[2], od[3]);
            o[2 * e] = mfma(ph, b0, o[2 * e]);
            o[2 * e] = mfma(pl, b0, o[2 * e]);
            o[2 * e + 1] = mfma(ph, b1, o[2 * e + 1]);
            o[2 * e + 1] = mfma(pl, b1, o[2 * e + 1]);
        }
        if (more) load_vs(sb + kStep);
    }

    // join the waves: (0 + 1) + (2 + 3), scaled to the common maximum
    l_run += xor_lane<16>(l_run);
    l_run += xor_lane<32>(l_run);
    if (g4 == 0) {
        stat[wv][0][l16] = m_run;
        stat[wv][1][l16] = l_run;
    }
    __syncthreads();
    float f[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int rr = 4 * g4 + r;
        const float mm = fmaxf(fmaxf(stat[0][0][rr], stat[1][0][rr]), fmaxf(stat[2][0][rr], stat[3][0][rr]));
        f[r] = __builtin_amdgcn_exp2f(stat[wv][0][rr] - (mm == -INFINITY ? 0.0f : mm));
    }
#pragma unroll
    for (int e = 0; e < VD; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[e][r] *= f[r];
    if (wv & 1) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < VD; ++e) ob[wv >> 1][4 * g4 + r][VD * l16 + e] = o[e][r];
    }
    __syncthreads();
    if (!(wv & 1)) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < VD; ++e) {
                float& w = ob[wv >> 1][4 * g4 + r][VD * l16 + e];
                w = o[e][r] + w;
            }
    }
    __syncthreads();
    const size_t rec = (static_cast<size_t>(chunk) * a.n_kv + kv) * a.rows_pad + kRows * group;
    for (int i = threadIdx.x; i < kRows * HD / 4; i += 64 * kWaves) {
        const float4 x = reinterpret_cast<const float4*>(&ob[0][0][0])[i], y = reinterpret_cast<const float4*>(&ob[1][0][0])[i];
        reinterpret_cast<float4*>(a.wo + rec * HD)[i] = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
    }
    if (threadIdx.x < kRows) {
        const int r = threadIdx.x;
        const float mm = fmaxf(fmaxf(stat[0][0][r], stat[1][0][r]), fmaxf(stat[2][0][r], stat[3][0][r]));
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) l = __builtin_fmaf(stat[w][1][r], __builtin_amdgcn_exp2f(stat[w][0][r] - ref), l);
        a.wml[2 * (rec + r)] = mm;
        a.wml[2 * (rec + r) + 1] = l;
    }
}

// ---- merge -------------------------------------------------------------------------------------------------------------
// Workgroup (token, head): the chunks' (m, l) give weights 2^(m - M) and L; lane groups of HD / 4 lanes sum every n-th
// chunk's o (four dims a lane), the groups are added in order; gate, fp32, Q8_1.  A row that sees nothing has M = -inf.
constexpr int kMergeThreads = 256;

template <int HD>
__global__ __launch_bounds__(kMergeThreads) void tree_merge_kernel(TreeArgs a, const float* __restrict__ gsrc, int gstride,
                                                                   float* __restrict__ y, int y_stride,
                                                                   uint8_t* __restrict__ q8, int q8_stride) {
    constexpr int L4 = HD / 4, NG = kMergeThreads / L4;
    __shared__ float wts[kMaxChunks];
    __shared__ float red[2][kMergeThreads / 64];
    __shared__ __attribute__((aligned(16))) float part[NG][HD];
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int G = a.n_head / a.n_kv, kv = h / G, row = t * G + (h - kv * G);
    const int base = a.pos[0];
    if (base < 0 || base > a.max_ctx - a.ntok) return;   // uniform: a slot outside the cache
    const int last = base + (a.masks ? a.ntok - 1 : t);
    const int nchunk = last / (kUnit * a.nsub) + 1;
    const size_t cstride = static_cast<size_t>(a.n_kv) * a.rows_pad, r0 = static_cast<size_t>(kv) * a.rows_pad + row;
    float m = -INFINITY;
    for (int c = tid; c < nchunk; c += kMergeThreads) m = fmaxf(m, a.wml[2 * (r0 + c * cstride)]);
    m = group_max<64>(m);
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    for (int c = tid; c < nchunk; c += kMergeThreads) {
        const float2 ml = *reinterpret_cast<const float2*>(a.wml + 2 * (r0 + c * cstride));
        const float w = __builtin_amdgcn_exp2f(ml.x - ref);
        wts[c] = w;
        l = __builtin_fmaf(ml.y, w, l);
    }
    l = group_sum<64>(l);
    if ((tid & 63) == 0) red[1][tid >> 6] = l;
    __syncthreads();
    l = ((red[1][0] + red[1][1]) + red[1][2]) + red[1][3];
    const int g = tid / L4, d = 4 * (tid % L4);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c = g; c < nchunk; c += NG) {
        const float4 x = *reinterpret_cast<const float4*>(a.wo + (r0 + c * cstride) * HD + d);
        const float w = wts[c];
        o.x = __builtin_fmaf(w, x.x, o.x);
        o.y = __builtin_fmaf(w, x.y, o.y);
        o.z = __builtin_fmaf(w, x.z, o.z);
        o.w = __builtin_fmaf(w, x.w, o.w);
    }
    *reinterpret_cast<float4*>(&part[g][d]) = o;
    __syncthreads();
    if (tid >= HD) return;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < NG; ++i) v += part[i][tid];
    v = m == -INFINITY ? 0.0f : v / l;
    if (gsrc) {
        const float x = gsrc[static_cast<size_t>(t) * gstride + h * 2 * HD + HD + tid];
        v *= 1.0f / (1.0f + expf(-x));
    }
    if (y) y[static_cast<size_t>(t) * y_stride + h * HD + tid] = v;
    if (q8) q8_1_store_lane(v, q8 + static_cast<size_t>(t) * q8_stride + (h * (HD / 32) + tid / 32) * kQ8_1Bytes);
}

bool tree_shape_ok(int max_ctx, int n_head, int n_kv, int head_dim, int ntok) {
    return kv_shape_ok(max_ctx, n_kv, head_dim) && n_head > 0 && n_head <= 65535 && n_head % n_kv == 0 && n_head / n_kv <= 64 &&
           ntok >= 1 && ntok <= kMaxChain;
}
int tree_rows(int n_head, int n_kv, int ntok) { return ntok * (n_head / n_kv); }
int tree_groups(int rows) { return (rows + kRows - 1) / kRows; }
long long tree_chunks(int max_ctx, int nsub) {
    const long long len = static_cast<long long>(kUnit) * nsub;
    return (max_ctx + len - 1) / len;
}

}  // namespace
}  // namespace rmi

using namespace rmi;

extern "C" int rmi_gqa_tree_nsub(int ctx, int n_head, int n_kv, int head_dim, int ntok) {
    if (!tree_shape_ok(ctx, n_head, n_kv, head_dim, ntok)) {
        set_error("gqa_tree_nsub: invalid shape");
        return 0;
    }
    // two workgroups a compute unit
    const long long groups = tree_groups(tree_rows(n_head, n_kv, ntok)), units = (ctx + kUnit - 1) / kUnit;
    const long long want = (units * n_kv * groups + 511) / 512;
    return static_cast<int>(std::max(std::max(1LL, (units + kMaxChunks - 1) / kMaxChunks), std::min(units, want)));
}

extern "C" size_t rmi_gqa_tree_workspace_bytes(int max_ctx, int n_head, int n_kv, int head_dim, int ntok, int nsub) {
    if (!tree_shape_ok(max_ctx, n_head, n_kv, head_dim, ntok) || nsub < 1 || tree_chunks(max_ctx, nsub) > kMaxChunks) {
        set_error("gqa_tree_workspace_bytes: invalid shape");
        return 0;
    }
    const size_t rows = static_cast<size_t>(tree_groups(tree_rows(n_head, n_kv, ntok))) * kRows;
    return static_cast<size_t>(tree_chunks(max_ctx, nsub)) * n_kv * rows * (head_dim + 2) * sizeof(float);
}

extern "C" int rmi_gqa_tree_decode(const float* q, int ktype, const void* kcache, int vtype, const void* vcache,
                                   const int* pos, const uint64_t* masks, const float* gate_src, int gate_stride, float* y,
                                   int y_stride, uint8_t* q8, int q8_stride, void* workspace, int n_head, int n_kv,
                                   int head_dim, int ntok, int max_ctx, int nsub, float scale, void* stream) {
    if (!kv_type_ok(ktype) || !kv_type_ok(vtype) || (ktype != vtype && !(ktype == kKvI8 && vtype == kKvI4)))
        return fail(RMI_ERR_UNSUPPORTED, "gqa_tree_decode: cache types F16 / F16, I8 / I8, I4 / I4 or I8 / I4");
    if (!tree_shape_ok(max_ctx, n_head, n_kv, head_dim, ntok) || ntok > max_ctx || (masks && ntok > kMaxTree) || nsub < 1 ||
        tree_chunks(max_ctx, nsub) > kMaxChunks)
        return fail(RMI_ERR_SHAPE, "gqa_tree_decode: invalid arguments");
    if (!aligned16(q) || !aligned16(kcache) || !aligned16(vcache) || !aligned4(pos) || !aligned16(workspace) ||
        (masks && (reinterpret_cast<uintptr_t>(masks) & 7u)) || (gate_src && !aligned4(gate_src)) || (!y && !q8) ||
        (y && !aligned4(y)) || (q8 && (!aligned4(q8) || q8_stride % 4)))
        return fail(RMI_ERR_POINTER, "gqa_tree_decode: null or misaligned pointer");
    TreeArgs a{};
    a.q = q;
    a.kc = static_cast<const uint8_t*>(kcache);
    a.vc = static_cast<const uint8_t*>(vcache);
    a.pos = pos;
    a.masks = masks;
    a.n_head = n_head;
    a.n_kv = n_kv;
    a.ntok = ntok;
    a.rows = tree_rows(n_head, n_kv, ntok);
    a.groups = tree_groups(a.rows);
    a.rows_pad = a.groups * kRows;
    a.nsub = static_cast<int>(std::min<long long>(nsub, (static_cast<long long>(max_ctx) + kUnit - 1) / kUnit));
    a.max_ctx = max_ctx;
    a.scale = scale;
    const long long pairs = tree_chunks(max_ctx, nsub) * n_kv, blocks = (pairs + 7) / 8 * 8 * a.groups;
    if (blocks > 0x7fffffffLL) return fail(RMI_ERR_SHAPE, "gqa_tree_decode: too many workgroups");
    a.npairs = static_cast<int>(pairs);
    a.wo = static_cast<float*>(workspace);
    a.wml = a.wo + static_cast<size_t>(pairs) * a.rows_pad * head_dim;
    auto* s = static_cast<hipStream_t>(stream);
    auto go = [&](auto* kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves), 0, s, a); };
    if (head_dim == 256) {
        if (ktype == kKvF16) go(&tree_partial_kernel<kKvF16, kKvF16, 256>);
        else if (ktype == kKvI4) go(&tree_partial_kernel<kKvI4, kKvI4, 256>);
        else if (vtype == kKvI8) go(&tree_partial_kernel<kKvI8, kKvI8, 256>);
        else go(&tree_partial_kernel<kKvI8, kKvI4, 256>);
        hipLaunchKernelGGL((tree_merge_kernel<256>), dim3(ntok, n_head), dim3(kMergeThreads), 0, s, a, gate_src, gate_stride, y,
                           y_stride, q8, q8_stride);
    } else {
        if (ktype == kKvF16) go(&tree_partial_kernel<kKvF16, kKvF16, 128>);
        else if (ktype == kKvI4) go(&tree_partial_kernel<kKvI4, kKvI4, 128>);
        else if (vtype == kKvI8) go(&tree_partial_kernel<kKvI8, kKvI8, 128>);
        else go(&tree_partial_kernel<kKvI8, kKvI4, 128>);
        hipLaunchKernelGGL((tree_merge_kernel<128>), dim3(ntok, n_head), dim3(kMergeThreads), 0, s, a, gate_src, gate_stride, y,
                           y_stride, q8, q8_stride);
    }
    return launch_status("gqa_tree_decode");
}
