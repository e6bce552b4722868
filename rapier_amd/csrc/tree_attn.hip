// tree_attn.hip - attention of a tree (or chain) of drafted tokens over a K/V cache in 16, 8 or 4 bits, for gfx950
// (rmi_gqa_tree_decode; caches: kv_cache.h).  No counterpart in the reference, whose draft is one token (gqa_head_kernel,
// qw:384-442, per column).
//
//   partial   workgroup (chunk of 128 nsub positions, KV head, group of query rows); row r = token r / G, head r % G of the
//             KV head's G.  Each wave streams its part of the chunk in steps of 32 positions with a running maximum, sum and
//             output per row; the waves' parts are joined at the end, one record (m, l, o) a row.
//   merge     workgroup (token, head, 64 dims): joins the chunks' records, gates, writes fp32 and Q8_1.  A call of one chunk
//             needs none: the partial launch writes the result.
//
// Both products run on fp16 MFMAs.  The cache's values are fp16 numbers in every type; the fp32 operand (q, p) goes as fp16
// high + low part, 22 bits, so the result keeps fp32's accuracy.  fp16's subnormals would cut the low parts short: a row's q
// is scaled by a power of two to [2^13, 2^14) and p by 2^8.  The scores' exponent is base 2.
//
// What a token does not see has no part in it: scores are masked before the maximum, and in the steps that reach into the
// draft a V that is not finite is taken out of the product and added to the rows that see it alone (an infinity times a
// masked zero would be NaN).
#include <algorithm>
#include <cmath>

#include "kv_operand.h"
#include "overlap.h"

namespace rmi {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kStep = 32;          // positions of a step
constexpr int kUnit = kWaves * kStep;
constexpr int kMaxChunks = 2048;   // a chunk's weight in the merge's LDS; named in the messages
constexpr int kMaxTree = 64, kMaxChain = 1024;
constexpr float kPScale = 8.0f;    // p goes as 2^8 p
constexpr float kLazy = 7.0f;      // a maximum moves once a score passes it by more than 2^7 (2^15 p is an fp16 number)

struct TreeArgs {
    const float* q;
    const uint8_t *kc, *vc;
    const int* pos;
    const uint64_t* masks;
    float *wo, *wml;   // records: o [chunk][kv][row][HD], (m, l) [chunk][kv][row][2]
    const float* gate;
    float* y;
    uint8_t* q8;
    int n_head, n_kv, ntok, rows, rows_pad, groups, npairs, nsub, max_ctx, gate_stride, y_stride, q8_stride, direct;
    float scale;
};

// `rows` rows from p as a buffer: a row past them reads as zeros, so a step past the last position loads nothing.  The length
// is told to be scalar: clamping takes a vector instruction, and each load would loop over its lanes' descriptors.
__device__ __forceinline__ Rsrc rows_buffer(const uint8_t* p, int rows, size_t stride) {
    const int n = __builtin_amdgcn_readfirstlane(min(max(rows, 0), kStep));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, static_cast<int>(n * stride), 0x00027000);
}

// what a workgroup works on; false where it has nothing to do (uniform)
struct Work {
    int chunk, kv, row0, base, last;   // row0: its first row, last: the last position any of its rows sees
};
template <int ROWS>
__device__ __forceinline__ bool tree_share(const TreeArgs& a, Work& w) {
    w.base = a.pos[0];   // in flight over what does not depend on it
    // the groups of a (chunk, head) pair are consecutive workgroups of one XCD (workgroups go to the XCDs round robin),
    // so the pair's rows come from HBM once
    const int k8 = static_cast<int>(blockIdx.x >> 3), q8 = k8 / a.groups;
    const int pair = 8 * q8 + static_cast<int>(blockIdx.x & 7);
    if (pair >= a.npairs) return false;
    w.chunk = pair / a.n_kv;
    w.kv = pair - w.chunk * a.n_kv;
    w.row0 = ROWS * (k8 - q8 * a.groups);
    return true;
}
template <int ROWS>
__device__ __forceinline__ bool tree_reach(const TreeArgs& a, Work& w) {
    if (w.base < 0 || w.base > a.max_ctx - a.ntok) return false;   // a slot outside the cache
    const int G = a.n_head / a.n_kv;
    w.last = w.base + (a.masks ? a.ntok - 1 : min(w.row0 + ROWS - 1, a.rows - 1) / G);
    return w.chunk * kUnit * a.nsub <= w.last;   // else the merge does not read this record
}

// which of a step's positions (first + 0..31, bit by bit) row `row` of token tok sees: lim is the last of its unbroken run
__device__ __forceinline__ bool sees(int p, int lim, uint64_t mask, int base, int ntok) {
    return p <= lim || (mask && p >= base && p - base < ntok && ((mask >> (p - base)) & 1));
}

// A row's o / l; zero where its token sees nothing.  A maximum of -inf alone does not say so: seen scores that are all NaN or
// -inf leave it too, and those rows are NaN (l is NaN, or 0 / 0).
__device__ __forceinline__ float normed(const TreeArgs& a, int t, float o, float m, float l) {
    if (m == -INFINITY && a.masks && a.pos[0] == 0 && !(a.masks[t] & (~0ull >> (64 - a.ntok)))) return 0.0f;
    return o / l;
}

// Four dims of a row's result from its joined sums: gate, fp32, Q8_1.  The lanes of a row's 32-dim block are eight
// neighbours.
template <int HD>
__device__ __forceinline__ void finish4(const TreeArgs& a, int t, int h, int d, float (&o)[4], float m, float l, const float (&gate)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        o[k] = normed(a, t, o[k], m, l);
        if (a.gate) o[k] *= 1.0f / (1.0f + expf(-gate[k]));
    }
    if (a.y) *reinterpret_cast<float4u*>(a.y + static_cast<size_t>(t) * a.y_stride + h * HD + d) = float4u{o[0], o[1], o[2], o[3]};
    if (a.q8) {   // q8_1_store_lane's block and bits: its lane's element is 4 (lane % 8) + k here
        float amax = fmaxf(fmaxf(fabsf(o[0]), fabsf(o[1])), fmaxf(fabsf(o[2]), fabsf(o[3])));
        amax = fmaxf(amax, xor_lane<4>(amax));
        amax = fmaxf(amax, xor_lane<2>(amax));
        amax = fmaxf(amax, xor_lane<1>(amax));
        float s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            s[k] = o[k] + xor_lane<4>(o[k]);
            s[k] += xor_lane<2>(s[k]);
            s[k] += xor_lane<1>(s[k]);
        }
        const float total = (s[0] + s[2]) + (s[1] + s[3]), dq = amax / 127.0f;
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w |= (static_cast<uint32_t>(amax == 0.0f ? 0 : static_cast<int>(roundf(o[k] / dq))) & 0xffu) << (8 * k);
        uint8_t* block = a.q8 + static_cast<size_t>(t) * a.q8_stride + (h * (HD / 32) + d / 32) * kQ8_1Bytes;
        *reinterpret_cast<uint32_t*>(block + 4 + (d & 31)) = w;
        if ((d & 31) == 0) *reinterpret_cast<uint32_t*>(block) = float_to_half_sat(dq) | (float_to_half_sat(total) << 16);
    }
}
template <int HD>
__device__ __forceinline__ void load_gate(const TreeArgs& a, int t, int h, int d, float (&g)[4]) {
    float4u x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.gate) x = *reinterpret_cast<const float4u*>(a.gate + static_cast<size_t>(t) * a.gate_stride + h * 2 * HD + HD + d);
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = x[k];
}

// Joins the waves' parts of RB row blocks from their LDS slabs [wave][row of the block][HD] and either writes records or,
// for a call of one chunk, the result: fac[wave][row] is a part's weight, top[row] and sum[row] the joined m and l.  Wave w
// holds part w / RB of row block w % RB.
template <int HD, int WAVES, int RB, int BLOCK>
__device__ __forceinline__ void join_rows(const TreeArgs& a, const Work& w, const float (&slab)[WAVES][BLOCK][HD],
                                          const float (&fac)[WAVES][BLOCK], const float (&top)[RB][BLOCK],
                                          const float (&sum)[RB][BLOCK]) {
    constexpr int PB = WAVES / RB, N = RB * BLOCK * HD / (4 * 64 * WAVES);   // N rounds of four dims a lane
    const int G = a.n_head / a.n_kv;
    const int d = 4 * (static_cast<int>(threadIdx.x) % (HD / 4)), r0 = static_cast<int>(threadIdx.x) / (HD / 4);
    constexpr int kUp = 4 * 64 * WAVES / HD;   // rows a round is further
    float g[N][4];
    if (a.direct && a.gate) {   // all gates in flight together
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = min(w.row0 + r0 + i * kUp, a.rows - 1), t = row / G;
            load_gate<HD>(a, t, w.kv * G + row - t * G, d, g[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + i * kUp, rb = r / BLOCK, rk = r % BLOCK, row = w.row0 + r;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < PB; ++p) {
            const float4 x = *reinterpret_cast<const float4*>(&slab[rb + RB * p][rk][d]);
            const float f = fac[rb + RB * p][rk];
            v[0] = __builtin_fmaf(x.x, f, v[0]);
            v[1] = __builtin_fmaf(x.y, f, v[1]);
            v[2] = __builtin_fmaf(x.z, f, v[2]);
            v[3] = __builtin_fmaf(x.w, f, v[3]);
        }
        if (row < a.rows) {
            if (a.direct) {
                const int t = row / G;
                finish4<HD>(a, t, w.kv * G + row - t * G, d, v, top[rb][rk], sum[rb][rk], g[i]);
            } else {
                const size_t rec = (static_cast<size_t>(w.chunk) * a.n_kv + w.kv) * a.rows_pad + row;
                *reinterpret_cast<float4*>(a.wo + rec * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
                if (d == 0) *reinterpret_cast<float2*>(a.wml + 2 * rec) = make_float2(top[rb][rk], sum[rb][rk]);
            }
        }
    }
}

// the parts' weights and the joined sum of every row, from stat[wave][m, l][row of the block]
// (times `unit`, what the parts' o is short of)
template <int WAVES, int RB, int BLOCK>
__device__ __forceinline__ void join_stats(float unit, const float (&stat)[WAVES][2][BLOCK], float (&fac)[WAVES][BLOCK], float (&top)[RB][BLOCK],
                                           float (&sum)[RB][BLOCK]) {
    constexpr int PB = WAVES / RB;
    const int i = threadIdx.x;
    if (i >= RB * BLOCK) return;
    const int rb = i / BLOCK, r = i % BLOCK;
    float m = stat[rb][0][r];
#pragma unroll
    for (int p = 1; p < PB; ++p) m = fmaxf(m, stat[rb + RB * p][0][r]);
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
#pragma unroll
    for (int p = 0; p < PB; ++p) {
        const float f = __builtin_amdgcn_exp2f(stat[rb + RB * p][0][r] - ref);
        fac[rb + RB * p][r] = f * unit;
        l = __builtin_fmaf(stat[rb + RB * p][1][r], f, l);
    }
    top[rb][r] = m;
    sum[rb][r] = l;
}

// ---- few query rows: v_mfma_f32_16x16x32_f16 from the cache ---------------------------------------------------------------
// Lane: l16 = l % 16, g4 = l / 16; A rows, B and D columns are l16; A and B hold k = 8 g4 + 0..7; D rows are 4 g4 + 0..3.
//   scores    D[position][n] += K[position][dims] . q_n[dims]; lane (l16, g4) takes 32 neighbouring dims of position l16,
//             128 k + 32 g4 + [0, 32), as four operands of eight, straight from the cache: one load and one scale of I4.
//             (F16 would read in whole lines with other dims, 5 % over 64K, but then its bits would not be the others'.)
//   P V       D[m][dim] += P_m[positions] V[positions][dim].  The score lane (row, positions 4 g4 + r of two tiles) holds P in
//             the A layout already, k slot j being position 4 g4 + j or 16 + 4 g4 + j - 4.  V comes by lane (l16, g4) as
//             HD / 16 dims of those eight positions (DimsV); operand e gathers the lane's dim e.
// Up to 8 rows, column (row) n < 8 is the high part of row n and n >= 8 the low part of row n - 8: one product gives both.  Up
// to 16 rows the parts are two products, with q's operands in LDS (the registers hold o and the step's K and V).
// The waves take quarters of the chunk.  K of the next step is loaded when this step's scores are done, V when its product is:
// each has half a step to arrive.  (Two steps ahead, in alternating registers, cost more than it hid: 30 us for 23.)
// One token of 16 heads behind 65501 positions: F16 50 us with its join (5.3 TB/s), I8 33 (4.2), I4 23 (3.1).  Seven of them
// are the beginning (position, first loads, q's parts) and the end; past that F16 and I8 are bound by the memory.  I4 has one wave a SIMD,
// whose vector units are busy for 51 % of its life (5928 instructions for eight steps, a beginning and an end) and which waits
// 26 % of it; I8 keys with I4 values 25 us.
template <int KT, int VT, int HD, int ROWS>
__global__ __launch_bounds__(kThreads, KT == kKvF16 ? 1 : 2) void tree_few_kernel(TreeArgs a) {
    constexpr bool PACKED = ROWS == 8;
    constexpr int NI = HD / 64;        // K: 16-dim pieces a lane takes of a position, two to a 32-dim run
    constexpr int VD = HD / 16;        // V: dims a lane takes of a position
    constexpr int NB = HD / kKvBlock;  // scale bytes of a row
    constexpr int kKB = kv_row_bytes(KT, HD), kVB = kv_row_bytes(VT, HD);
    __shared__ __attribute__((aligned(16))) float slab[kWaves][ROWS][HD];   // the rows that are joined
    // until then q's operands [piece][half][part][lane]
    auto& qs = *reinterpret_cast<half8(*)[NI][2][2][64]>(&slab[0][0][0]);
    static_assert(PACKED || sizeof(qs) <= sizeof(slab), "q's operands fit");
    __shared__ float pb[kWaves][ROWS][kStep];   // a step's p where a V is not finite
    __shared__ float stat[kWaves][2][ROWS], fac[kWaves][ROWS], top[1][ROWS], sum[1][ROWS];

    Work w;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
    if (!tree_share<ROWS>(a, w)) return;
    const int G = a.n_head / a.n_kv, kv = w.kv;
    const int slot = PACKED ? l16 & 7 : l16, row = w.row0 + slot, rowc = min(row, a.rows - 1), tok = rowc / G;
    const bool low = PACKED && l16 >= 8;
    // the query rows and masks do not depend on the position: in flight together with it
    const float* qr = a.q + (static_cast<size_t>(tok) * a.n_head + kv * G + (rowc - tok * G)) * HD + 32 * g4;
    float qx[NI][16];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const float4 u = reinterpret_cast<const float4*>(qr + 128 * (i >> 1) + 16 * (i & 1))[f];
            qx[i][4 * f] = u.x, qx[i][4 * f + 1] = u.y, qx[i][4 * f + 2] = u.z, qx[i][4 * f + 3] = u.w;
        }
    uint64_t mask = 0;   // of the row's token: bit j = draft slot base + j
    if (a.masks && row < a.rows) mask = a.masks[tok];
    if (!tree_reach<ROWS>(a, w)) return;
    const int base = w.base, last = w.last;
    const int wlen = kStep * a.nsub, wbase = (w.chunk * kWaves + wv) * wlen;
    const int nsteps = wbase > last ? 0 : min(a.nsub, (last - wbase) / kStep + 1);
    const int lim = row >= a.rows ? -1 : a.masks ? base - 1 : base + tok;   // the row sees every position up to here

    // the head's rows, kstride apart; a lane's place in a step's
    const size_t kstride = KT == kKvF16 ? static_cast<size_t>(a.n_kv) * kKB : kKB;
    const size_t vstride = VT == kKvF16 ? static_cast<size_t>(a.n_kv) * kVB : kVB;
    const KvRow<KT> k0 = kv_row<KT>(0, kv, a.n_kv, a.max_ctx, HD);
    const KvRow<VT> v0 = kv_row<VT>(0, kv, a.n_kv, a.max_ctx, HD);
    const uint8_t *kp = a.kc + k0.code, *ks = a.kc + k0.scale, *vp = a.vc + v0.code, *vs = a.vc + v0.scale;
    const int kat = static_cast<int>(l16 * kstride) + g4 * (kKB / (HD / 32)), vat = static_cast<int>(4 * g4 * vstride) + l16 * DimsV<VT, VD>::kRun;
    const int vsat = 4 * g4 * NB + VD * l16 / kKvBlock;

    Dims16<KT> kx[2][NI];
    uint32_t ksc[2][2];
    DimsV<VT, VD> vx[8];
    uint32_t vsc[8];
    auto load_k = [&](int sb, bool wanted) {   // rows past the last read as zeros
        const int n = wanted ? last + 1 - sb : 0;
        const Rsrc r = rows_buffer(kp + sb * kstride, n, kstride);
        const Rsrc rs = rows_buffer(ks + static_cast<size_t>(sb) * NB, n, NB);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < NI; i += 2) {
                if constexpr (KT == kKvI4) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, kat + i * (kKB / NI), static_cast<int>(16 * t * kstride), 0);
                    kx[t][i].w[0] = v[0], kx[t][i].w[1] = v[1], kx[t][i + 1].w[0] = v[2], kx[t][i + 1].w[1] = v[3];
                } else {
                    kx[t][i] = load16<KT>(r, kat + i * (kKB / NI), static_cast<int>(16 * t * kstride));
                    kx[t][i + 1] = load16<KT>(r, kat + i * (kKB / NI) + kKB / (HD / 16), static_cast<int>(16 * t * kstride));
                }
            }
            if constexpr (KT != kKvF16) {
                if constexpr (NB == 8) {
                    const auto s = __builtin_amdgcn_raw_buffer_load_b64(rs, l16 * NB, 16 * t * NB, 0);
                    ksc[t][0] = s[0], ksc[t][1] = s[1];
                } else {
                    ksc[t][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, l16 * NB, 16 * t * NB, 0);
                }
            }
        }
    };
    auto load_vs = [&](int sb, bool wanted) {
        const int n = wanted ? last + 1 - sb : 0;
        const Rsrc r = rows_buffer(vp + sb * vstride, n, vstride);
        const Rsrc rs = rows_buffer(vs + static_cast<size_t>(sb) * NB, n, NB);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int p = j < 4 ? j : 12 + j;
            vx[j] = load_dims<VT, VD>(r, vat, static_cast<int>(p * vstride));
            if constexpr (VT != kKvF16) vsc[j] = __builtin_amdgcn_raw_buffer_load_b8(rs, vsat + p * NB, 0, 0);
        }
    };
    load_k(wbase, nsteps > 0);
    __builtin_amdgcn_sched_barrier(0);   // in this order, as in the loop: a wait for K then leaves V in flight
    load_vs(wbase, nsteps > 0);

    half8 qb[PACKED ? NI : 1][2];
    float post;   // score = product * post, in base 2
    {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(qx[i][e]));
        m = fmaxf(m, xor_lane<16>(m));
        m = fmaxf(m, xor_lane<32>(m));
        const int sh = q_shift(m);
        const float f = ldexpf(1.0f, sh);
        post = a.scale * (1.44269504088896340736f * kSixteen<KT>) * ldexpf(1.0f, -sh);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
            {
                float x[8];
                half8 hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = qx[i][8 * hf + e] * f;
                split8(x, hi, lo);
                if constexpr (PACKED) {
                    qb[i][hf] = low ? lo : hi;
                } else if (i == wv) {   // every wave has the group's rows: each writes a piece
                    qs[i][hf][0][lane] = hi;
                    qs[i][hf][1][lane] = lo;
                }
            }
    }

    if constexpr (!PACKED) {
        static_assert(PACKED || NI <= kWaves, "a piece a wave");
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();   // __syncthreads would also wait for the first K and V
        asm volatile("" ::: "memory");
    }
    floatx4 o[VD];
#pragma unroll
    for (int e = 0; e < VD; ++e) o[e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l_run = 0.0f;   // l_run: this lane's positions only

    for (int st = 0; st < nsteps; ++st) {
        const int sb = wbase + st * kStep;
        float sc[8];   // j: position sb + 4 g4 + j, or 16 + 4 g4 + j - 4 further
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f}, acl = acc;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                Scale2 s = {};
                if constexpr (KT != kKvF16) {   // block 4 (i / 2) + g4
                    const uint32_t b = (ksc[t][i >> 1] >> (8 * g4)) & 0xffu;
                    s = scale2<KT>(b, b);
                }
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const half8 kk = operand<KT>(kx[t][i], hf, s);
                    if constexpr (PACKED) {
                        acc = mfma(kk, qb[i][hf], acc);
                    } else {
                        acc = mfma(kk, qs[i][hf][0][lane], acc);
                        acl = mfma(kk, qs[i][hf][1][lane], acl);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[4 * t + r] = (acc[r] + (PACKED ? xor_lane<8>(acc[r]) : acl[r])) * post;
        }
        // the loads are not under a branch: behind one, every wait would be for all that might be out
        const bool more = st + 1 < nsteps;
        load_k(sb + kStep, more);
        const bool tail = sb + kStep > base;   // uniform: the step reaches into the draft
        uint32_t seen = 0xffu;
        if (tail || row >= a.rows) {
            seen = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (sees(sb + 4 * g4 + (j < 4 ? j : 12 + j), lim, mask, base, a.ntok)) seen |= 1u << j;
                else sc[j] = -INFINITY;
            }
        }
        float mloc = sc[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mloc = fmaxf(mloc, sc[j]);
        mloc = fmaxf(mloc, xor_lane<16>(mloc));
        mloc = fmaxf(mloc, xor_lane<32>(mloc));
        const float m_new = mloc > m_run + kLazy ? mloc : m_run;
        const float m_ref = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: exp2(-inf) = 0, no NaN
        const float alpha = m_run == m_new || m_run == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_ref);   // -inf: o is 0
        float p[8], lsum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = __builtin_amdgcn_exp2f(sc[j] - m_ref + kPScale);
            lsum += p[j];
        }
        l_run = l_run * alpha + lsum;
        m_run = m_new;
        if (__ballot(alpha != 1.0f)) {   // uniform: some row's maximum moved
            float al[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) al[r] = __shfl(alpha, PACKED ? 4 * (g4 & 1) + r : 4 * g4 + r, 64);
#pragma unroll
            for (int e = 0; e < VD; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[e][r] *= al[r];
        }
        half8 ph, pl;
        split8(p, ph, pl);
        if (low) ph = pl;
        Scale2 vsp[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (VT != kKvF16) vsp[j] = scale2<VT>(vsc[2 * j], vsc[2 * j + 1]);
            else vsp[j] = Scale2{};
        }
        if (tail) {
            uint32_t big = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (VT != kKvF16) {
                    big = max_magnitude(big, u2(vsp[j].c));   // not finite wherever s is not
                } else {
#pragma unroll
                    for (int e = 0; e < VD / 2; ++e) big = max_magnitude(max_magnitude(big, vx[2 * j].w[e]), vx[2 * j + 1].w[e]);
                }
            }
            if (__ballot(!finite16(big))) {
                float(*pw)[kStep] = pb[wv];   // [row][position], -1: not seen
                if (!low)
#pragma unroll
                    for (int j = 0; j < 8; ++j) pw[slot][4 * g4 + (j < 4 ? j : 12 + j)] = seen >> j & 1 ? p[j] : -1.0f;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                for (int pp = 0; pp < kStep; ++pp) {
                    const size_t p1 = min(sb + pp, last);
#pragma unroll
                    for (int e = 0; e < VD; ++e) {
                        float v;
                        if constexpr (VT == kKvF16) v = half_bits_to_float(reinterpret_cast<const uint16_t*>(vp + p1 * vstride)[DimsV<VT, VD>::dim(l16, e)]);
                        else v = odd_value<VT>(vs[p1 * NB + VD * l16 / kKvBlock]);
                        if (fabsf(v) <= FLT_MAX) continue;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float x = !PACKED ? pw[4 * g4 + r][pp] : g4 < 2 ? pw[4 * (g4 & 1) + r][pp] : -1.0f;   // the high rows
                            if (!(x < 0.0f)) o[e][r] = __builtin_fmaf(x, v, o[e][r]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if constexpr (VT == kKvF16) {
#pragma unroll
                        for (int e = 0; e < VD / 2; ++e) vx[j].w[e] = zero_odd(vx[j].w[e]);
                    } else if ((j & 1) == 0) {
                        uint32_t s = u2(vsp[j >> 1].s), c = u2(vsp[j >> 1].c);
                        if ((c & 0x7c00u) == 0x7c00u) s &= 0xffff0000u, c &= 0xffff0000u;
                        if ((c & 0x7c000000u) == 0x7c000000u) s &= 0xffffu, c &= 0xffffu;
                        vsp[j >> 1] = {h2(s), h2(c)};
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < VD / 2; ++e) {
            uint32_t ev[4], od[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v_pair<VT, VD>(vx[2 * j], vx[2 * j + 1], e, vsp[j], ev[j], od[j]);
            const half8 b0 = h8(ev[0], ev[1], ev[2], ev[3]), b1 = h8(od[0], od[1], od[2], od[3]);
            o[2 * e] = mfma(ph, b0, o[2 * e]);
            o[2 * e + 1] = mfma(ph, b1, o[2 * e + 1]);
            if constexpr (!PACKED) {
                o[2 * e] = mfma(pl, b0, o[2 * e]);
                o[2 * e + 1] = mfma(pl, b1, o[2 * e + 1]);
            }
        }
        load_vs(sb + kStep, more);
    }

    l_run += xor_lane<16>(l_run);
    l_run += xor_lane<32>(l_run);
    if (g4 == 0 && !low) {
        stat[wv][0][slot] = m_run;
        stat[wv][1][slot] = l_run;
    }
    if constexpr (!PACKED) __syncthreads();   // q's operands are read
    if constexpr (PACKED) {
        // high rows + low rows, two registers at a time: a swap of a's upper and b's lower lanes, then one add, leaves a's sums
        // in the lower lanes (row 4 g4 + r) and b's in the upper (row 4 (g4 - 2) + r + 1)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            float v[VD];
#pragma unroll
            for (int e = 0; e < VD; ++e) {
                const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[e][r]), __float_as_uint(o[e][r + 1]), false, false);
                v[e] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            }
            float* to = slab[wv][4 * (g4 & 1) + r + (g4 >> 1)];
#pragma unroll
            for (int e = 0; e < VD; e += 4) *reinterpret_cast<float4*>(to + DimsV<VT, VD>::dim(l16, e)) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < VD; e += 4)
                *reinterpret_cast<float4*>(&slab[wv][4 * g4 + r][DimsV<VT, VD>::dim(l16, e)]) = make_float4(o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]);
    }
    __syncthreads();
    join_stats<kWaves, 1, ROWS>(kSixteen<VT>, stat, fac, top, sum);
    __syncthreads();
    join_rows<HD, kWaves, 1, ROWS>(a, w, slab, fac, top, sum);
}

// ---- more rows: the tile in LDS ---------------------------------------------------------------------------------------------
// Eight waves, two to a SIMD: RB hold different 16 rows (q in high and low parts and o in registers), 8 / RB different parts
// of the chunk.  The RB waves of a part share its tile of 32 positions in LDS as fp16, [position][dim] for K and V alike, so
// each cache value is turned into fp16 once for 16 RB rows: a thread takes 16 dims of a position per unit, the next tile's
// loads in flight over this tile's products.
//   scores    A = K tile rows (16-byte reads), B = q rows: D[position][row], as above with one register set per part.
//   P V       A = P, B = V columns by transposed reads (ds_read_b64_tr_b16: the 16 lanes of a g4 give the addresses of four
//             positions x 16 dims and get a dim's four positions each), k slots as above.
// Row strides of 16 and 32 bytes past a power of two spread a read's rows over the banks.
// 999 tokens x 16 heads behind 8001 positions, I8 / I4: 286 us with the join's 16, 278 GFLOP of the two products each at 83 % of
// the rate of a large matrix product; 64 rows a workgroup in place of 128 362 us.
constexpr int kTileWaves = 8;
constexpr int kTileThreads = 64 * kTileWaves;
constexpr int kRowBlock = 16;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int HD, int RB>
struct TilePool {
    static constexpr int kParts = kTileWaves / RB;
    static constexpr int kKRow = 2 * HD + 16, kVRow = 2 * HD + 32;     // bytes
    static constexpr int kBytes = kStep * (kKRow + kVRow);             // one tile
    static constexpr int kBufs = kParts == 4 ? 1 : 2;                  // two tiles a part where they fit
    static constexpr int kPool = kParts * kBufs * kBytes;
    static_assert(kParts == 1 || kPool >= kTileWaves * kRowBlock * HD * 4, "the parts' rows are joined in the tiles' place");
};

// The order of N groups of R LDS reads and M products in a block: AHEAD groups' reads, then a group's reads for a group's
// products.  Left alone the compiler reads two operands ahead and waits out the latency at each.
template <int N, int R, int M, int AHEAD>
__device__ __forceinline__ void interleave() {
    constexpr int kAhead = N < AHEAD ? N : AHEAD;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead * R, 0);   // LDS reads
#pragma unroll
    for (int i = 0; i < N - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);        // MFMAs
        __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, M * kAhead, 0);
}

template <int KT, int VT, int HD, int RB>
__global__ __launch_bounds__(kTileThreads, 2) void tree_tile_kernel(TreeArgs a) {
    using Pool = TilePool<HD, RB>;
    constexpr int PB = Pool::kParts, BUFS = Pool::kBufs;
    constexpr int NC = HD / 32;                                  // 32-dim pieces of a row
    constexpr int NE = HD / 16;                                  // 16-dim columns of o
    constexpr int NB = HD / kKvBlock;
    constexpr int kUnits = kStep * NE;                           // 16-dim units of a tile
    constexpr int U = kUnits > 64 * RB ? kUnits / (64 * RB) : 1;   // of them a thread's, of K and of V
    constexpr int kKB = kv_row_bytes(KT, HD), kVB = kv_row_bytes(VT, HD);
    __shared__ __attribute__((aligned(16))) uint8_t pool[Pool::kPool];
    __shared__ float pb[kTileWaves][kRowBlock][kStep];           // a step's p where a V is not finite
    __shared__ int odd_step[PB][BUFS];                           // the last step whose V had one
    __shared__ float stat[kTileWaves][2][kRowBlock], fac[kTileWaves][kRowBlock], top[RB][kRowBlock], sum[RB][kRowBlock];   // PB > 1

    Work w;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
    if (!tree_share<kRowBlock * RB>(a, w)) return;
    const int G = a.n_head / a.n_kv, kv = w.kv;
    const int rb = wv % RB, part = wv / RB, tt = rb * 64 + lane;   // tt: thread within the part
    const int row0 = w.row0 + kRowBlock * rb, row = row0 + l16, rowc = min(row, a.rows - 1), tok = rowc / G;
    // the query rows and masks do not depend on the position: in flight together with it
    const float* qr = a.q + (static_cast<size_t>(tok) * a.n_head + kv * G + (rowc - tok * G)) * HD + 8 * g4;
    float4 qx[NC][2];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int f = 0; f < 2; ++f) qx[c][f] = reinterpret_cast<const float4*>(qr + 32 * c)[f];
    uint64_t mask = 0;
    if (a.masks && row < a.rows) mask = a.masks[tok];
    if (!tree_reach<kRowBlock * RB>(a, w)) return;
    if (threadIdx.x < PB * BUFS) odd_step[threadIdx.x / BUFS][threadIdx.x % BUFS] = -1;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();   // __syncthreads would also wait for the query rows
    const int base = w.base;
    // the last position the wave's rows see (w.last: any of the workgroup's)
    const int last = row0 >= a.rows ? -1 : a.masks ? w.last : base + min(row0 + kRowBlock - 1, a.rows - 1) / G;
    const int psteps = kUnit * a.nsub / (kStep * PB), cbase = w.chunk * kUnit * a.nsub, pbase = cbase + part * psteps * kStep;
    const int nsteps = min(psteps, (w.last - cbase) / kStep + 1);   // of the first part: the others run along
    const int lim = row >= a.rows ? -1 : a.masks ? base - 1 : base + tok;

    const size_t kstride = KT == kKvF16 ? static_cast<size_t>(a.n_kv) * kKB : kKB;
    const size_t vstride = VT == kKvF16 ? static_cast<size_t>(a.n_kv) * kVB : kVB;
    const KvRow<KT> k0 = kv_row<KT>(0, kv, a.n_kv, a.max_ctx, HD);
    const KvRow<VT> v0 = kv_row<VT>(0, kv, a.n_kv, a.max_ctx, HD);
    const uint8_t *kp = a.kc + k0.code, *ks = a.kc + k0.scale, *vp = a.vc + v0.code, *vs = a.vc + v0.scale;
    // the thread's first unit; the next ones are kUp positions further
    constexpr int kUp = 64 * RB / NE;
    const int unit = tt % NE, pos0 = tt / NE;
    const int kat = static_cast<int>(pos0 * kstride) + unit * (kKB / NE), vat = static_cast<int>(pos0 * vstride) + unit * (kVB / NE);
    const int sat = pos0 * NB + unit / 2;

    Dims16<KT> kx[U];
    Dims16<VT> vx[U];
    uint32_t ksc[U], vsc[U];
    auto load = [&](int sb) {   // rows past the last read as zeros
        const int n = w.last + 1 - sb;
        const Rsrc rk = rows_buffer(kp + sb * kstride, n, kstride), rks = rows_buffer(ks + static_cast<size_t>(sb) * NB, n, NB);
        const Rsrc rv = rows_buffer(vp + sb * vstride, n, vstride), rvs = rows_buffer(vs + static_cast<size_t>(sb) * NB, n, NB);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kUnits < 64 * RB && tt >= kUnits) break;
            kx[u] = load16<KT>(rk, kat, static_cast<int>(u * kUp * kstride));
            vx[u] = load16<VT>(rv, vat, static_cast<int>(u * kUp * vstride));
            if constexpr (KT != kKvF16) ksc[u] = __builtin_amdgcn_raw_buffer_load_b8(rks, sat + u * kUp * NB, 0, 0);
            if constexpr (VT != kKvF16) vsc[u] = __builtin_amdgcn_raw_buffer_load_b8(rvs, sat + u * kUp * NB, 0, 0);
        }
    };
    uint8_t* tiles = pool + part * (BUFS * Pool::kBytes);
    auto store = [&](int buf, int st) {
        const bool tail = pbase + (st + 1) * kStep > base;   // uniform in the part
        uint8_t* kt = tiles + buf * Pool::kBytes + unit * 32;
        uint8_t* vt = kt + kStep * Pool::kKRow;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kUnits < 64 * RB && tt >= kUnits) break;
            const int p = pos0 + u * kUp;
            Scale2 sk = {}, sv = {};
            if constexpr (KT != kKvF16) sk = scale2<KT>(ksc[u], ksc[u]);
            if constexpr (VT != kKvF16) sv = scale2<VT>(vsc[u], vsc[u]);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                *reinterpret_cast<half8*>(kt + p * Pool::kKRow + 16 * hf) = operand<KT>(kx[u], hf, sk);
                u32x4 v = __builtin_bit_cast(u32x4, operand<VT>(vx[u], hf, sv));
                if (tail && !(finite16(v[0]) && finite16(v[1]) && finite16(v[2]) && finite16(v[3]))) {
                    v = u32x4{zero_odd(v[0]), zero_odd(v[1]), zero_odd(v[2]), zero_odd(v[3])};
                    odd_step[part][buf] = st;   // every writer stores the same
                }
                *reinterpret_cast<u32x4*>(vt + p * Pool::kVRow + 16 * hf) = v;
            }
        }
    };
    load(pbase);

    half8 qh[NC], ql[NC];
    float post;   // score = product * post, in base 2
    {
        float m = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int f = 0; f < 2; ++f)
                m = fmaxf(m, fmaxf(fmaxf(fabsf(qx[c][f].x), fabsf(qx[c][f].y)), fmaxf(fabsf(qx[c][f].z), fabsf(qx[c][f].w))));
        m = fmaxf(m, xor_lane<16>(m));
        m = fmaxf(m, xor_lane<32>(m));
        const int sh = q_shift(m);
        const float f = ldexpf(1.0f, sh);
        post = a.scale * (1.44269504088896340736f * kSixteen<KT>) * ldexpf(1.0f, -sh);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float x[8] = {qx[c][0].x * f, qx[c][0].y * f, qx[c][0].z * f, qx[c][0].w * f,
                                qx[c][1].x * f, qx[c][1].y * f, qx[c][1].z * f, qx[c][1].w * f};
            split8(x, qh[c], ql[c]);
        }
    }
    floatx4 o[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) o[e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l_run = 0.0f;   // l_run: this lane's positions only

    store(0, 0);
    __syncthreads();
    for (int st = 0; st < nsteps; ++st) {
        const int sb = pbase + st * kStep, buf = BUFS == 2 ? st & 1 : 0;
        const bool more = st + 1 < nsteps;
        if (more) load(sb + kStep);
        if (sb <= last) {   // uniform in the wave
            const uint8_t* kt = tiles + buf * Pool::kBytes + l16 * Pool::kKRow + 16 * g4;
            float sc[8];   // j: position sb + 4 g4 + j, or 16 + 4 g4 + j - 4 further
            floatx4 dh[2], dl[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                dh[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                dl[t] = dh[t];
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const half8 kk = *reinterpret_cast<const half8*>(kt + 16 * t * Pool::kKRow + 64 * c);
                    dh[t] = mfma(kk, qh[c], dh[t]);
                    dl[t] = mfma(kk, ql[c], dl[t]);
                }
            }
            interleave<2 * NC, 1, 2, 4>();
#pragma unroll
            for (int j = 0; j < 8; ++j) sc[j] = (dh[j >> 2][j & 3] + dl[j >> 2][j & 3]) * post;
            const bool tail = sb + kStep > base;   // uniform: the step reaches into the draft
            uint32_t seen = 0xffu;
            if (tail || row >= a.rows) {
                seen = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (sees(sb + 4 * g4 + (j < 4 ? j : 12 + j), lim, mask, base, a.ntok)) seen |= 1u << j;
                    else sc[j] = -INFINITY;
                }
            }
            float mloc = sc[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mloc = fmaxf(mloc, sc[j]);
            mloc = fmaxf(mloc, xor_lane<16>(mloc));
            mloc = fmaxf(mloc, xor_lane<32>(mloc));
            const float m_new = mloc > m_run + kLazy ? mloc : m_run;
            const float m_ref = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: exp2(-inf) = 0, no NaN
            const float alpha = m_run == m_new || m_run == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_ref);   // -inf: o is 0
            float p[8], lsum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = __builtin_amdgcn_exp2f(sc[j] - m_ref + kPScale);
                lsum += p[j];
            }
            l_run = l_run * alpha + lsum;
            m_run = m_new;
            if (__ballot(alpha != 1.0f)) {   // uniform: some row's maximum moved
                float al[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) al[r] = __shfl(alpha, 4 * g4 + r, 64);
#pragma unroll
                for (int e = 0; e < NE; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[e][r] *= al[r];
            }
            half8 ph, pl;
            split8(p, ph, pl);
            // the lane's address of the transposed reads: position 4 g4 + l16 / 4, dims 4 (l16 % 4) ..
            const uint8_t* vr = tiles + buf * Pool::kBytes + kStep * Pool::kKRow + (4 * g4 + (l16 >> 2)) * Pool::kVRow + 8 * (l16 & 3);
            auto column = [&](int e) {   // dims 16 e + l16 of the lane's eight positions
                const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*) (vr + 32 * e));
                const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*) (vr + 16 * Pool::kVRow + 32 * e));
                const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
                return h8(x.x, x.y, y.x, y.y);
            };
            if (tail && odd_step[part][buf] == st) {   // uniform: some V is not finite (zero in the tile)
                float(*pw)[kStep] = pb[wv];   // [row][position], -1: not seen
#pragma unroll
                for (int j = 0; j < 8; ++j) pw[l16][4 * g4 + (j < 4 ? j : 12 + j)] = seen >> j & 1 ? p[j] : -1.0f;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                for (int pp = 0; pp < kStep; ++pp) {
                    float x[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] = pw[4 * g4 + r][pp];
                    const KvRow<VT> vrow = kv_row<VT>(min(sb + pp, w.last), kv, a.n_kv, a.max_ctx, HD);
#pragma unroll
                    for (int e = 0; e < NE; ++e) {
                        const int d = 16 * e + l16;
                        float v;
                        if constexpr (VT == kKvF16) v = half_bits_to_float(reinterpret_cast<const uint16_t*>(a.vc + vrow.code)[d]);
                        else v = odd_value<VT>(a.vc[vrow.scale + d / kKvBlock]);
                        if (fabsf(v) <= FLT_MAX) continue;
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!(x[r] < 0.0f)) o[e][r] = __builtin_fmaf(x[r], v, o[e][r]);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < NE; e += 2) {
                const half8 v0 = column(e), v1 = column(e + 1);
                o[e] = mfma(ph, v0, o[e]);
                o[e + 1] = mfma(ph, v1, o[e + 1]);
                o[e] = mfma(pl, v0, o[e]);
                o[e + 1] = mfma(pl, v1, o[e + 1]);
            }
            interleave<NE / 2, 4, 4, 2>();
        }
        if (BUFS == 1) __syncthreads();   // the tile is read
        if (more) store(BUFS == 2 ? buf ^ 1 : 0, st + 1);
        __syncthreads();
    }

    l_run += xor_lane<16>(l_run);
    l_run += xor_lane<32>(l_run);
    if constexpr (PB > 1) {
        if (g4 == 0) {
            stat[wv][0][l16] = m_run;
            stat[wv][1][l16] = l_run;
        }
        auto& slab = *reinterpret_cast<float(*)[kTileWaves][kRowBlock][HD]>(pool);   // the tiles are read
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < NE; ++e) slab[wv][4 * g4 + r][16 * e + l16] = o[e][r];
        __syncthreads();
        join_stats<kTileWaves, RB, kRowBlock>(kSixteen<VT>, stat, fac, top, sum);
        __syncthreads();
        join_rows<HD, kTileWaves, RB, kRowBlock>(a, w, slab, fac, top, sum);
    } else {
        // one part: the wave's rows straight from its registers, 16 dims of four rows an instruction
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int rw = row0 + 4 * g4 + r, t = min(rw, a.rows - 1) / G, h = kv * G + min(rw, a.rows - 1) - t * G;
            const float m = __shfl(m_run, 4 * g4 + r, 64), l = __shfl(l_run, 4 * g4 + r, 64);
            if (!a.direct) {
                const size_t rec = (static_cast<size_t>(w.chunk) * a.n_kv + kv) * a.rows_pad + rw;
                if (rw < a.rows) {
#pragma unroll
                    for (int e = 0; e < NE; ++e) a.wo[rec * HD + 16 * e + l16] = o[e][r] * kSixteen<VT>;
                    if (l16 == 0) *reinterpret_cast<float2*>(a.wml + 2 * rec) = make_float2(m, l);
                }
                continue;
            }
            float g[NE];
#pragma unroll
            for (int e = 0; e < NE; ++e) g[e] = a.gate ? a.gate[static_cast<size_t>(t) * a.gate_stride + h * 2 * HD + HD + 16 * e + l16] : 0.0f;
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                float v = normed(a, t, o[e][r] * kSixteen<VT>, m, l);
                if (a.gate) v *= 1.0f / (1.0f + expf(-g[e]));
                o[e][r] = v;
                if (a.y && rw < a.rows) a.y[static_cast<size_t>(t) * a.y_stride + h * HD + 16 * e + l16] = v;
            }
            if (!a.q8) continue;
#pragma unroll
            for (int e = 0; e < NE; e += 2) {   // q8_1_store_lane's block and bits: its lane's element is 16 (e % 2) + l16 here
                const float u = o[e][r], v = o[e + 1][r];
                const float amax = group_max<16>(fmaxf(fabsf(u), fabsf(v))), total = group_sum<16>(u + v), dq = amax / 127.0f;
                uint8_t* block = a.q8 + static_cast<size_t>(t) * a.q8_stride + (h * (HD / 32) + e / 2) * kQ8_1Bytes;
                if (rw < a.rows) {
                    block[4 + l16] = static_cast<uint8_t>(static_cast<int8_t>(amax == 0.0f ? 0 : static_cast<int>(roundf(u / dq))));
                    block[20 + l16] = static_cast<uint8_t>(static_cast<int8_t>(amax == 0.0f ? 0 : static_cast<int>(roundf(v / dq))));
                    if (l16 == 0) *reinterpret_cast<uint32_t*>(block) = float_to_half_sat(dq) | (float_to_half_sat(total) << 16);
                }
            }
        }
    }
}

// ---- merge -------------------------------------------------------------------------------------------------------------
// Workgroup (token, head, 64 dims): every lane has the (m, l) of a chunk and its group's first o in flight together; weights
// 2^(m - M) to LDS, wave g sums chunks g, g + 4, ... in order, then the four waves in order; gate, fp32, Q8_1.  64 chunks of one
// token 3.9 us, a chain of waits (position, records, two barriers).  A whole row a workgroup: 10.6 us in place of 11.2 for 32 chunks of 64 tokens,
// which are joined in groups of 16 rows, over few chunks, instead.
constexpr int kMergeDims = 64, kMergeBatch = 16;

template <int HD>
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(TreeArgs a) {
    __shared__ float wts[kMaxChunks];
    __shared__ float red[2][kWaves];
    __shared__ float part[kWaves][kMergeDims];
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, g = tid >> 6;
    const int d = kMergeDims * blockIdx.z + lane;
    const int G = a.n_head / a.n_kv, kv = h / G, row = t * G + (h - kv * G);
    // the first records and o values do not wait for the position: every chunk of the cache has a place (what a chunk past
    // the last position holds is not used), and indexes are clamped (a load under a branch gets a wait of its own)
    const int all = a.npairs / a.n_kv;
    const size_t cstride = static_cast<size_t>(a.n_kv) * a.rows_pad, r0 = static_cast<size_t>(kv) * a.rows_pad + row;
    const float2* ml = reinterpret_cast<const float2*>(a.wml) + r0;
    const float* ro = a.wo + r0 * HD + d;
    const float2 first = ml[min(tid, all - 1) * cstride];
    float oa[kMergeBatch];   // chunks g + 4 k
#pragma unroll
    for (int k = 0; k < kMergeBatch; ++k) oa[k] = ro[min(g + 4 * k, all - 1) * cstride * HD];
    float gate = 0.0f;
    if (a.gate) gate = a.gate[static_cast<size_t>(t) * a.gate_stride + h * 2 * HD + HD + d];
    const int base = a.pos[0];
    if (base < 0 || base > a.max_ctx - a.ntok) return;   // uniform: a slot outside the cache
    const int nchunk = (base + (a.masks ? a.ntok - 1 : t)) / (kUnit * a.nsub) + 1;
    float m = tid < nchunk ? first.x : -INFINITY;
    for (int c = tid + kThreads; c < nchunk; c += kThreads) m = fmaxf(m, ml[c * cstride].x);
    m = group_max<64>(m);
    if (lane == 0) red[0][g] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    for (int c = tid; c < nchunk; c += kThreads) {
        const float2 x = c == tid ? first : ml[c * cstride];
        const float wt = __builtin_amdgcn_exp2f(x.x - ref);
        wts[c] = wt;
        l = __builtin_fmaf(x.y, wt, l);
    }
    l = group_sum<64>(l);
    if (lane == 0) red[1][g] = l;
    __syncthreads();
    l = ((red[1][0] + red[1][1]) + red[1][2]) + red[1][3];
    float o = 0.0f;
    for (int c0 = 0; 4 * c0 < nchunk; c0 += kMergeBatch) {
        const bool more = 4 * (c0 + kMergeBatch) < nchunk;
        float nx[kMergeBatch];
        if (more) {
#pragma unroll
            for (int k = 0; k < kMergeBatch; ++k) nx[k] = ro[min(g + 4 * (c0 + kMergeBatch + k), nchunk - 1) * cstride * HD];
        }
#pragma unroll
        for (int k = 0; k < kMergeBatch; ++k) {
            const int c = g + 4 * (c0 + k);
            if (c < nchunk) o = __builtin_fmaf(wts[c], oa[k], o);
        }
        if (more) {
#pragma unroll
            for (int k = 0; k < kMergeBatch; ++k) oa[k] = nx[k];
        }
    }
    part[g][lane] = o;
    __syncthreads();
    if (g != 0) return;
    float v = ((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane];
    v = normed(a, t, v, m, l);
    if (a.gate) v *= 1.0f / (1.0f + expf(-gate));
    if (a.y) a.y[static_cast<size_t>(t) * a.y_stride + h * HD + d] = v;
    if (a.q8) q8_1_store_lane(v, a.q8 + static_cast<size_t>(t) * a.q8_stride + (h * (HD / 32) + d / 32) * kQ8_1Bytes);
}

// The same for a few chunks, where the work is a pass over the records: HD / 4 lanes a row, four dims a lane, no LDS.  999 tokens,
// two chunks: 16 us, 4.1 TB/s.
constexpr int kFlatChunks = 8;

template <int HD>
__global__ __launch_bounds__(kThreads) void tree_merge_flat_kernel(TreeArgs a) {
    constexpr int L4 = HD / 4;
    const int i = blockIdx.x * (kThreads / L4) + static_cast<int>(threadIdx.x) / L4, d = 4 * (static_cast<int>(threadIdx.x) % L4);
    if (i >= a.ntok * a.n_head) return;
    const int t = i / a.n_head, h = i - t * a.n_head;
    const int G = a.n_head / a.n_kv, kv = h / G, row = t * G + (h - kv * G);
    float g[4];
    load_gate<HD>(a, t, h, d, g);
    const int base = a.pos[0];
    if (base < 0 || base > a.max_ctx - a.ntok) return;   // uniform: a slot outside the cache
    const int nchunk = (base + (a.masks ? a.ntok - 1 : t)) / (kUnit * a.nsub) + 1;
    const size_t cstride = static_cast<size_t>(a.n_kv) * a.rows_pad, r0 = static_cast<size_t>(kv) * a.rows_pad + row;
    const float2* ml = reinterpret_cast<const float2*>(a.wml) + r0;
    const float* ro = a.wo + r0 * HD + d;
    float m = -INFINITY, l = 0.0f;
    for (int c = 0; c < nchunk; ++c) m = fmaxf(m, ml[c * cstride].x);
    const float ref = m == -INFINITY ? 0.0f : m;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < nchunk; ++c) {
        const float2 x = ml[c * cstride];
        const float4 v = *reinterpret_cast<const float4*>(ro + c * cstride * HD);
        const float w = __builtin_amdgcn_exp2f(x.x - ref);
        l = __builtin_fmaf(x.y, w, l);
        o[0] = __builtin_fmaf(w, v.x, o[0]);
        o[1] = __builtin_fmaf(w, v.y, o[1]);
        o[2] = __builtin_fmaf(w, v.z, o[2]);
        o[3] = __builtin_fmaf(w, v.w, o[3]);
    }
    finish4<HD>(a, t, h, d, o, m, l, g);
}

bool tree_shape_ok(int max_ctx, int n_head, int n_kv, int head_dim, int ntok) {
    return kv_shape_ok(max_ctx, n_kv, head_dim) && n_head > 0 && n_head <= 65535 && n_head % n_kv == 0 && n_head / n_kv <= 64 &&
           ntok >= 1 && ntok <= kMaxChain;
}

// The form of a call: query rows per KV head, 16-row blocks side by side in a workgroup (0: the form of few rows), rows a
// workgroup holds, workgroups per (chunk, KV head).  Up to 16 rows the form of few rows; more rows are groups of it where the
// split asks for that (RMI_TREE_SHORT: rmi_gqa_tree_nsub), else tiles, which turn K and V to fp16 once for all of a workgroup's
// rows.  17 to 32 rows of I8 and I4 stay groups of few (64K, 8 tokens x 4 heads: 45.7 / 38.9 us, tiles 47.3 / 40.2; I8 / I4 41), F16 takes
// tiles over long chunks (60 us, groups of few 83: they load K and V twice).
constexpr int kLongSub = 6;
constexpr int kShort = RMI_TREE_SHORT;
struct Form {
    int rows, rb, held, groups;
};
Form tree_form(int n_head, int n_kv, int ntok, int split, bool f16) {
    Form f;
    f.rows = ntok * (n_head / n_kv);
    f.rb = f.rows <= 16 || (split & kShort) ? 0 : f.rows <= 32 ? (f16 && split >= kLongSub ? 2 : 0) : f.rows <= 64 ? 4 : 8;
    f.held = f.rb ? kRowBlock * f.rb : f.rows <= 8 ? 8 : 16;
    f.groups = (f.rows + f.held - 1) / f.held;
    return f;
}
// the chunk's length in a split, in units; 0: not one
int split_nsub(int split) { return split < 1 || split >= 2 * kShort ? 0 : split & (kShort - 1); }
long long tree_chunks(int max_ctx, int nsub) {
    const long long len = static_cast<long long>(kUnit) * nsub;
    return (max_ctx + len - 1) / len;
}

template <int KT, int VT, int HD>
void launch_partial(const TreeArgs& a, const Form& f, unsigned blocks, hipStream_t s) {
    auto go = [&](auto* kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, s, a); };
    if (f.held == 8) go(&tree_few_kernel<KT, VT, HD, 8>, kThreads);
    else if (f.held == 16) go(&tree_few_kernel<KT, VT, HD, 16>, kThreads);
    else if (f.rb == 2) {
        if constexpr (KT == kKvF16) go(&tree_tile_kernel<KT, VT, HD, 2>, kTileThreads);
    } else if (f.rb == 4) go(&tree_tile_kernel<KT, VT, HD, 4>, kTileThreads);
    else go(&tree_tile_kernel<KT, VT, HD, 8>, kTileThreads);
}

template <int HD>
void launch_tree(const TreeArgs& a, int ktype, int vtype, const Form& f, unsigned blocks, hipStream_t s) {
    if (ktype == kKvF16) launch_partial<kKvF16, kKvF16, HD>(a, f, blocks, s);
    else if (ktype == kKvI4) launch_partial<kKvI4, kKvI4, HD>(a, f, blocks, s);
    else if (vtype == kKvI8) launch_partial<kKvI8, kKvI8, HD>(a, f, blocks, s);
    else launch_partial<kKvI8, kKvI4, HD>(a, f, blocks, s);
    if (a.npairs / a.n_kv > kFlatChunks)
        hipLaunchKernelGGL((tree_merge_kernel<HD>), dim3(a.ntok, a.n_head, HD / kMergeDims), dim3(kThreads), 0, s, a);
    else if (!a.direct)
        hipLaunchKernelGGL((tree_merge_flat_kernel<HD>), dim3((a.ntok * a.n_head + 1024 / HD - 1) / (1024 / HD)), dim3(kThreads), 0, s, a);
}

}  // namespace
}  // namespace rmi

using namespace rmi;

extern "C" int rmi_gqa_tree_nsub(int ctx, int n_head, int n_kv, int head_dim, int ntok) {
    if (!tree_shape_ok(ctx, n_head, n_kv, head_dim, ntok)) {
        set_error("gqa_tree_nsub: invalid shape");
        return 0;
    }
    // One workgroup for each of 256 compute units: as many chunks as leave an XCD's 32 units a (chunk, head, group) each, since
    // a 33rd is done after or beside another.  I8, 12 tokens x 4 heads behind 16K: 33 an XCD 32.0 us, 24 23.7; 1 token at
    // 64K with two workgroups a unit 32.8 us, one 32.8 (I4 23.7 / 22.9, F16 55 / 51).
    const long long units = (ctx + kUnit - 1) / kUnit;
    auto nsub_for = [&](int groups) {
        const int pairs = 8 * std::max(1, 32 / groups), chunks = std::max(1, pairs / n_kv);
        return (units + chunks - 1) / chunks;
    };
    // More than 16 rows as groups of few while a wave of theirs has at most 8 steps, where a workgroup's beginning and end
    // and the records of many chunks weigh more than turning K and V to fp16 once: 16 tokens x 4 heads, groups / tiles: I8 4K
    // 16.9 / 21.3 us, 8K 20.0 / 22.6, 16K 24.9 / 25.8; 64 tokens 4K 26.5 / 33.7, 32 tokens 16K (16 steps) 40 / 36;
    // F16 16 tokens 4K 18.1 / 21.2, 16K 32.1 / 27.0, 64 tokens 4K 32.6 / 32.0; I4 16 tokens 4K 16.5 / 21.3, 16K 25.8 / 29.0.
    // The rule does not know the cache's type: 16 tokens of F16 behind 16K are a sixth faster with the tiles' split (2), which a
    // caller may give.
    constexpr int kFewSteps = 8;
    const Form few = tree_form(n_head, n_kv, ntok, kShort + 1, false), tile = tree_form(n_head, n_kv, ntok, kLongSub, true);
    long long nsub = nsub_for(few.groups);
    const bool in_groups = few.rows > 16 && few.groups <= 32 && nsub <= kFewSteps;
    if (few.rows > 16 && !in_groups) nsub = std::max<long long>(tile.rb == 2 ? kLongSub : 1, nsub_for(tile.groups));
    nsub = std::max({1LL, (units + kMaxChunks - 1) / kMaxChunks, nsub});
    return static_cast<int>(nsub) | (in_groups ? kShort : 0);
}

extern "C" size_t rmi_gqa_tree_workspace_bytes(int max_ctx, int n_head, int n_kv, int head_dim, int ntok, int nsub) {
    const int split = nsub;
    nsub = split_nsub(split);
    if (!tree_shape_ok(max_ctx, n_head, n_kv, head_dim, ntok) || nsub < 1) {
        set_error("gqa_tree_workspace_bytes: invalid shape");
        return 0;
    }
    if (tree_chunks(max_ctx, nsub) > kMaxChunks) {
        set_error("gqa_tree_workspace_bytes: more than 2048 chunks of 128 nsub positions in max_ctx: a larger nsub");
        return 0;
    }
    const Form f = tree_form(n_head, n_kv, ntok, split, false);   // 17 to 32 rows take the same space in both forms
    return static_cast<size_t>(tree_chunks(max_ctx, nsub)) * n_kv * (static_cast<size_t>(f.groups) * f.held) * (head_dim + 2) * sizeof(float);
}

extern "C" int rmi_gqa_tree_decode(const float* q, int ktype, const void* kcache, int vtype, const void* vcache,
                                   const int* pos, const uint64_t* masks, const float* gate_src, int gate_stride, float* y,
                                   int y_stride, uint8_t* q8, int q8_stride, void* workspace, int n_head, int n_kv,
                                   int head_dim, int ntok, int max_ctx, int nsub, float scale, void* stream) {
    if (!kv_type_ok(ktype) || !kv_type_ok(vtype) || (ktype != vtype && !(ktype == kKvI8 && vtype == kKvI4)))
        return fail(RMI_ERR_UNSUPPORTED, "gqa_tree_decode: cache types F16 / F16, I8 / I8, I4 / I4 or I8 / I4");
    const int split = nsub;
    nsub = split_nsub(split);
    if (!tree_shape_ok(max_ctx, n_head, n_kv, head_dim, ntok) || ntok > max_ctx || (masks && ntok > kMaxTree) || nsub < 1)
        return fail(RMI_ERR_SHAPE, "gqa_tree_decode: invalid arguments");
    if (tree_chunks(max_ctx, nsub) > kMaxChunks)
        return fail(RMI_ERR_SHAPE, "gqa_tree_decode: more than 2048 chunks of 128 nsub positions in max_ctx: a larger nsub");
    if (!aligned16(q) || !aligned16(kcache) || !aligned16(vcache) || !aligned4(pos) || !aligned16(workspace) ||
        (masks && (reinterpret_cast<uintptr_t>(masks) & 7u)) || (gate_src && !aligned4(gate_src)) || (!y && !q8) ||
        (y && !aligned4(y)) || (q8 && (!aligned4(q8) || q8_stride % 4)))
        return fail(RMI_ERR_POINTER, "gqa_tree_decode: null or misaligned pointer");
    const int width = n_head * head_dim;
    if (ntok > 1 && ((y && y_stride < width) || (q8 && q8_stride < width / 32 * static_cast<int>(kQ8_1Bytes))))
        return fail(RMI_ERR_SHAPE, "gqa_tree_decode: output rows overlap");
    // y may be q itself: a row's workgroup alone reads its q, and before it writes
    const RowSet in[] = {block_of(q, static_cast<size_t>(ntok) * width * 4), block_of(kcache, rmi_kv_cache_bytes(ktype, max_ctx, n_kv, head_dim)),
                         block_of(vcache, rmi_kv_cache_bytes(vtype, max_ctx, n_kv, head_dim))};
    const RowSet out[] = {block_of(workspace, rmi_gqa_tree_workspace_bytes(max_ctx, n_head, n_kv, head_dim, ntok, split)),
                          {q8, q8 ? ntok : 0, q8_stride, width / 32 * kQ8_1Bytes},
                          {y, y ? ntok : 0, 4LL * y_stride, 4LL * width}};
    const bool in_place = y == q && (ntok == 1 || y_stride == width);
    for (const RowSet& o : out) {
        for (const RowSet& i : in)
            if (o.n && !(in_place && o.p == y && i.p == q) && rows_overlap(o, i))
                return fail(RMI_ERR_POINTER, "gqa_tree_decode: an output or the workspace lies on what the call reads");
        // a token's gates from the first to the last, then head by head: a row of q8 may fit between two
        if (gate_src && o.n && rows_overlap(o, {gate_src + head_dim, ntok, 4LL * gate_stride, 4LL * (2 * width - head_dim)}))
            for (int h = 0; h < n_head; ++h)
                if (rows_overlap(o, {gate_src + static_cast<size_t>(2 * h + 1) * head_dim, ntok, 4LL * gate_stride, 4LL * head_dim}))
                    return fail(RMI_ERR_POINTER, "gqa_tree_decode: an output or the workspace lies on the gates");
        for (const RowSet* other = out; other != &o; ++other)
            if (o.n && other->n && rows_overlap(o, *other))
                return fail(RMI_ERR_POINTER, "gqa_tree_decode: an output or the workspace lies on another");
    }
    const Form f = tree_form(n_head, n_kv, ntok, split, ktype == kKvF16);
    TreeArgs a{};
    a.q = q;
    a.kc = static_cast<const uint8_t*>(kcache);
    a.vc = static_cast<const uint8_t*>(vcache);
    a.pos = pos;
    a.masks = masks;
    a.gate = gate_src;
    a.y = y;
    a.q8 = q8;
    a.n_head = n_head;
    a.n_kv = n_kv;
    a.ntok = ntok;
    a.rows = f.rows;
    a.groups = f.groups;
    a.rows_pad = f.groups * f.held;
    a.nsub = static_cast<int>(std::min<long long>(nsub, (static_cast<long long>(max_ctx) + kUnit - 1) / kUnit));
    a.max_ctx = max_ctx;
    a.gate_stride = gate_stride;
    a.y_stride = y_stride;
    a.q8_stride = q8_stride;
    a.scale = scale;
    const long long chunks = tree_chunks(max_ctx, nsub), pairs = chunks * n_kv, blocks = (pairs + 7) / 8 * 8 * f.groups;
    if (blocks > 0xffffffffLL / kTileThreads) return fail(RMI_ERR_SHAPE, "gqa_tree_decode: too many workgroups");
    a.npairs = static_cast<int>(pairs);
    a.direct = chunks == 1;
    a.wo = static_cast<float*>(workspace);
    a.wml = a.wo + static_cast<size_t>(pairs) * a.rows_pad * head_dim;
    auto* s = static_cast<hipStream_t>(stream);
    if (head_dim == 256) launch_tree<256>(a, ktype, vtype, f, static_cast<unsigned>(blocks), s);
    else launch_tree<128>(a, ktype, vtype, f, static_cast<unsigned>(blocks), s);
    return launch_status("gqa_tree_decode");
}
