// batch_attn.hip - causal attention for a batch of requests of different lengths, for gfx950:
//   gqa_paged_attn    new tokens of each request over its pages (kv_pages.h), F16 / I8 / I4; q and y in fp16 or bf16
//   gqa_prompt_attn   whole prompts packed row by row, q, k, v and y in fp16 or bf16, no cache
// No counterpart in the reference, which serves one request (gqa_head_kernel, qw:384-442; its ingest's score pass, qw:444-559).
//
// Query row r of a request and KV head is token r / G, head r % G of the head's G.  Token t of n new ones is at position
// len - n + t and sees the positions up to its own.  Kernels:
//   few     up to 16 rows a request, 32 of a quantised cache (decode, drafts): workgroup (request, KV head, chunk of positions), K
//           and V straight from the pages into matrix operands; bound by the cache
//   tile    more rows: workgroup (128 or 256 rows, KV head, chunk), K and V tiles in LDS
//   parts   prompts of few tiles: workgroup (32 rows, KV head), its waves taking steps of the positions in turn
//   join    the chunks' records (m, l, o) of a row, where the context is split
// A paged call with requests of both kinds launches the first two; each takes its own requests.
#include "kv_operand.h"
#include "kv_pages.h"
#include "overlap.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace rmi {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kFewRows = 16;
constexpr int kWaveRows = 32;      // of a wave of the form of more rows
constexpr int kTileRows = 128;     // rows of four such waves, the unit of a split
constexpr int kChunkUnit = 128;    // a chunk is a whole number of them
constexpr int kMaxChunks = 1024;   // named in the messages
constexpr float kPScale = 8.0f;    // p goes as 2^8 p in fp16, whose subnormals then begin 2^-22 below a row's maximum (bf16 has no need)
constexpr float kLazy = 7.0f;      // a maximum moves once a score passes it by more than 2^7 (2^15 p is an fp16 number)

struct BatchArgs {
    const uint8_t *q, *k, *v;   // q rows; pools, or k and v rows
    const int *table, *row_start, *kv_len;
    const float* gate;
    uint8_t *y, *q8;
    float *wo, *wml;   // records: o [chunk][row][head][HD], (m, l) [chunk][row][head][2]
    int q_stride, k_stride, v_stride, gate_stride, y_stride, q8_stride;   // elements (q8: bytes)
    int table_stride, n_req, ntok, max_new, max_ctx, n_head, n_kv, shift, n_pages;
    int chunk, chunks, levels, few, bf16;   // levels: the most tiles of a prompt; few: the rows that the form of few rows takes
    float post;   // score = q.k * post, in base 2
};

// ---- requests --------------------------------------------------------------------------------------------------------------
typedef const __attribute__((address_space(4))) int* ConstInts;   // read through the scalar cache
__device__ __forceinline__ int word(const int* p, size_t i) { return reinterpret_cast<ConstInts>(reinterpret_cast<uintptr_t>(p))[i]; }

struct Req {
    int start, n, len;   // rows [start, start + n) of the call, positions
};
// request i's rows, cut to those of the call; none where it is past the call's bounds
__device__ __forceinline__ Req request(const BatchArgs& a, int i, int first, int end) {
    Req r;
    r.start = min(max(first, 0), a.ntok);
    r.n = min(max(end, r.start), a.ntok) - r.start;
    r.len = a.kv_len ? word(a.kv_len, i) : r.n;
    if (r.n > a.max_new || r.len > a.max_ctx) r.n = 0;
    r.len = max(r.len, 0);
    return r;
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {   // a scalar
    const uint32_t upto = wave_scan(v, [](uint32_t x, uint32_t y) { return x + y; });
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
}

// The workgroup's tile by its rank among all of the call.  A request's tile at `level` is its rows 128 level ..; tiles go by level,
// the highest first, since the work grows with it (the prefix a tile sees): the longest start first and the short ones fill the
// end.  count(i): request i's number of tiles, i < 64 ceil(n_req / 64).  False: the call has no such tile.
template <typename F>
__device__ __forceinline__ bool tile_of_rank(const BatchArgs& a, F&& count, uint32_t rank, int* req, int* level) {
    const int lane = threadIdx.x & 63;
    auto above = [&](int l) {   // tiles at level l and higher
        uint32_t s = 0;
        for (int i = lane; i < a.n_req; i += 64) s += static_cast<uint32_t>(max(count(i) - l, 0));
        return wave_sum(s);
    };
    if (rank >= above(0)) return false;
    int lo = 0, hi = a.levels;   // above(lo) > rank, above(hi) <= rank (nothing is at the bound)
    uint32_t below = 0;          // above(hi)
    if (a.n_req == 1) {
        const int n = __builtin_amdgcn_readfirstlane(count(0));
        *req = 0;
        *level = n - 1 - static_cast<int>(rank);
        return true;
    }
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const uint32_t f = above(mid);
        if (f > rank) lo = mid;
        else hi = mid, below = f;
    }
    uint32_t k = rank - below;   // which of the level's requests, in order
    for (int i0 = 0; i0 < a.n_req; i0 += 64) {
        const uint64_t has = __ballot(i0 + lane < a.n_req && count(min(i0 + lane, a.n_req - 1)) > lo);
        const uint32_t n = __popcll(has);
        if (k < n) {
            uint64_t m = has;
            while (k--) m &= m - 1;
            *req = i0 + __builtin_ctzll(m);
            *level = lo;
            return true;
        }
        k -= n;
    }
    return false;
}

// tile_of_rank for tiles of ROWS rows, in a workgroup of THREADS; counts: kMaxReq words of LDS, free again afterwards
template <int ROWS, int THREADS>
__device__ __forceinline__ bool find_tile(const BatchArgs& a, int* counts, uint32_t rank, int G, int* req, int* level) {
    const int tid = threadIdx.x, lane = tid & 63;
    auto tiles_of = [&](int k) {
        const int rows = request(a, k, a.row_start[k], a.row_start[k + 1]).n * G;
        return (rows + ROWS - 1) / ROWS;
    };
    bool has;
    if (a.n_req <= 64) {   // a request a lane
        const int mine = tiles_of(min(lane, a.n_req - 1));
        has = tile_of_rank(a, [&](int) { return mine; }, rank, req, level);
    } else {
        for (int k = tid; k < a.n_req; k += THREADS) counts[k] = tiles_of(k);
        __syncthreads();
        has = tile_of_rank(a, [&](int k) { return counts[k]; }, rank, req, level);
        __syncthreads();   // read before the first tile overwrites them
    }
    *req = __builtin_amdgcn_readfirstlane(*req);
    *level = __builtin_amdgcn_readfirstlane(*level);
    return has;
}

// A paged call's work by its rank: the requests' items one behind another, count(request) of each, so that the workgroups that have
// work are the first ones, as many to each XCD (they go there in turn), and a round of one for each compute unit is one.  (Launched
// as every request's items to the longest one's, 32 requests of one token behind 1 K to 4 K positions took 78 us in chunks of 1792,
// so 70; two of 40 tokens behind 30 K and 15 K, I8, in chunks of 768, 128 and 83.)  False: the call has no such item.
template <typename F>
__device__ __forceinline__ bool item_of_rank(const BatchArgs& a, uint32_t rank, F&& count, int* req, int* item) {
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < a.n_req; i0 += 64) {
        const int i = min(i0 + lane, a.n_req - 1);
        const uint32_t n = i0 + lane < a.n_req ? count(request(a, i, a.row_start[i], a.row_start[i + 1])) : 0;
        const uint32_t upto = wave_scan(n, [](uint32_t x, uint32_t y) { return x + y; });
        const uint64_t past = __ballot(upto > rank);
        if (past) {
            const int l = __builtin_ctzll(past);
            *req = i0 + l;
            *item = static_cast<int>(rank) - __builtin_amdgcn_readlane(static_cast<int>(upto - n), l);
            return true;
        }
        rank -= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
    }
    return false;
}
// chunks of a request's positions, one at least (its rows are written there)
__device__ __forceinline__ int chunks_in(const BatchArgs& a, int len) { return max((len + a.chunk - 1) / a.chunk, 1); }

// ---- 16-bit rows -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { return u2(__builtin_convertvector(floatx2{a, b}, half2v)); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, bf16x2));
}
__device__ __forceinline__ uint32_t pack16(int bf16, float a, float b) { return bf16 ? pack_bf16(a, b) : pack_f16(a, b); }

// bf16 pairs as fp16, times 2^sh
__device__ __forceinline__ uint32_t bf16_to_f16(uint32_t w, int sh) {
    return pack_f16(ldexpf(__uint_as_float(w << 16), sh), ldexpf(__uint_as_float(w & 0xffff0000u), sh));
}

template <bool BF>
__device__ __forceinline__ floatx16 mfma32(u32x4 a, u32x4 b, floatx16 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mfma16(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// ---- results ---------------------------------------------------------------------------------------------------------------
constexpr float kLog2e = 1.44269504088896340736f;
// v sigmoid(g): |g| 2^-23 relative from the exponent's rounding, two more roundings
__device__ __forceinline__ float gated(float v, float g) { return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g)); }

// the Q8_1 block and bits of q8_1_store_lane from a lane's four values of a 32-dim row block whose eight lanes are neighbours
__device__ __forceinline__ void store_q8_quads(const float (&o)[4], uint8_t* block, int d) {
    float amax = fmaxf(fmaxf(fabsf(o[0]), fabsf(o[1])), fmaxf(fabsf(o[2]), fabsf(o[3])));
    amax = group_max<8>(amax);
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
    for (int k = 0; k < 4; ++k) w |= (static_cast<uint32_t>(amax == 0.0f ? 0 : static_cast<int>(roundf(o[k] / dq))) & 0xffu) << (8 * k);
    *reinterpret_cast<uint32_t*>(block + 4 + (d & 31)) = w;
    if ((d & 31) == 0) *reinterpret_cast<uint32_t*>(block) = float_to_half_sat(dq) | (float_to_half_sat(total) << 16);
}

template <int HD>
__device__ __forceinline__ void load_gate(const BatchArgs& a, int t, int h, int d, float (&g)[4]) {
    float4u x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.gate) x = *reinterpret_cast<const float4u*>(a.gate + static_cast<ptrdiff_t>(t) * a.gate_stride + h * 2 * HD + HD + d);
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = x[k];
}

// a row's sums over its weights' sum; zeros where the token sees nothing
__device__ __forceinline__ void normed4(float (&o)[4], float l, bool none) {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = none ? 0.0f : o[k] / l;
}

// four dims of a row's result; the lanes of a 32-dim block are eight neighbours
template <int HD>
__device__ __forceinline__ void finish4(const BatchArgs& a, int t, int h, int d, float (&o)[4], const float (&gate)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (a.gate) o[k] = gated(o[k], gate[k]);
    if (a.y)
        *reinterpret_cast<uint2*>(a.y + 2 * (static_cast<ptrdiff_t>(t) * a.y_stride + h * HD + d)) =
            make_uint2(pack16(a.bf16, o[0], o[1]), pack16(a.bf16, o[2], o[3]));
    if (a.q8) store_q8_quads(o, a.q8 + static_cast<ptrdiff_t>(t) * a.q8_stride + (h * (HD / 32) + d / 32) * kQ8_1Bytes, d);
}

// ---- few rows --------------------------------------------------------------------------------------------------------------
// v_mfma_f32_16x16x32_f16 straight from the pages.  Lane: l16 = l % 16, g4 = l / 16; A rows, B and D columns are l16; A and B hold
// k = 8 g4 + 0..7; D rows are 4 g4 + 0..3.
//   scores    D[position][row] += K[position][dims] . q_row[dims]; lane (l16, g4) takes 32 neighbouring dims of position l16,
//             128 k + 32 g4 + [0, 32), as four operands of eight
//   P V       D[row][dim] += P_row[positions] V[positions][dim].  The score lane (row, positions 4 g4 + r of two 16s) holds P in the
//             A layout already, k slot j being position 4 g4 + j or 16 + 4 g4 + j - 4.  V comes by lane as HD / 16 dims of those
//             eight positions (DimsV); operand e gathers the lane's dim e.
// The waves take steps of 32 positions in turn.  A step's positions lie in one or two pages: each half has its own buffer, whose
// length ends at the last position (rows past it read as zeros) and is zero for a page that is not one.  K of the next step is
// loaded when this step's scores are done, V when its product is.
// RB blocks of 16 rows share a step's operands (few_rows says when).
// Bound by the cache, which is read once: 32 requests of one token behind 1 K to 4 K positions F16 (16 heads, 4 KV heads of 256 dims)
// 65 us, 5.2 TB/s, one behind 65501 positions I8 25 us, 5.5 TB/s (a large copy 5.12).  Of small calls, and of a round's every
// workgroup, 5 us go into starts: lengths, then page ids, then codes, each a wait for memory.  F16 holds two waves' registers in one (at
// two waves a SIMD the loads ahead no longer fit: slower).
struct Half {
    Rsrc kr, ks, vr, vs;
};

template <int KT, int VT, int HD, int RB>
__global__ __launch_bounds__(kThreads, KT == kKvF16 || RB == 2 ? 1 : 2) void batch_few_kernel(BatchArgs a) {
    constexpr int NI = HD / 64;        // K: 16-dim pieces a lane takes of a position, two to a 32-dim run
    constexpr int VD = HD / 16;        // V: dims a lane takes of a position
    constexpr int NB = HD / kKvBlock;  // scale bytes of a row
    constexpr int ROWS = kFewRows * RB;
    constexpr int kKB = kv_row_bytes(KT, HD), kVB = kv_row_bytes(VT, HD);
    __shared__ __attribute__((aligned(16))) float slab[kWaves][ROWS][HD];   // the rows that are joined
    __shared__ float pb[kWaves][ROWS][32];   // a step's p where a V is not finite
    __shared__ float stat[kWaves][2][ROWS], fac[kWaves][ROWS], sum[2][ROWS];

    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
    const int kv = blockIdx.x % a.n_kv, G = a.n_head / a.n_kv;
    int i = 0, chunk = 0;
    auto count = [&](const Req& r) { return r.n > 0 && r.n * G <= ROWS ? chunks_in(a, r.len) : 0; };
    if (!item_of_rank(a, blockIdx.x / a.n_kv, count, &i, &chunk)) return;   // uniform
    const Req rq = request(a, i, word(a.row_start, i), word(a.row_start, i + 1));
    const int rows = rq.n * G, base = rq.len - rq.n, last = rq.len - 1, c0 = chunk * a.chunk;
    const bool second = RB == 2 && rows > kFewRows;   // uniform: the second 16 rows are there
    u32x4 qb[RB][NI][2];
    int lim[RB];   // row 16 b + l16 sees every position up to here
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int row = kFewRows * b + l16, rowc = min(row, rows - 1), tok = rowc / G;
        const uint16_t* qr = reinterpret_cast<const uint16_t*>(a.q) + (static_cast<ptrdiff_t>(rq.start + tok) * a.q_stride + (kv * G + rowc - tok * G) * HD) + 32 * g4;
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) qb[b][k][hf] = *reinterpret_cast<const u32x4*>(qr + 128 * (k >> 1) + 16 * (k & 1) + 8 * hf);
        lim[b] = row >= rows ? -1 : base + tok;
    }
    const int end = min(last + 1, c0 + a.chunk);
    const int total = max(end - c0 + 31, 0) / 32, nsteps = max(total - wv + kWaves - 1, 0) / kWaves;

    const int size = 1 << a.shift;
    const size_t kpage = kv_page_bytes(KT, size, a.n_kv, HD), vpage = kv_page_bytes(VT, size, a.n_kv, HD);
    const size_t kstride = KT == kKvF16 ? static_cast<size_t>(a.n_kv) * kKB : kKB;
    const size_t vstride = VT == kKvF16 ? static_cast<size_t>(a.n_kv) * kVB : kVB;
    const KvRow<KT> k0 = kv_row<KT>(0, kv, a.n_kv, size, HD);
    const KvRow<VT> v0 = kv_row<VT>(0, kv, a.n_kv, size, HD);
    const int* const ids = a.table + static_cast<size_t>(i) * a.table_stride;
    auto page_at = [&](int p) {   // -1: not a page
        const int at = min(p, last) >> a.shift;
        const int id = p <= last && at < a.table_stride ? word(ids, at) : -1;
        return id >= 0 && id < a.n_pages ? id : -1;
    };
    // a half step's 16 rows from position p on
    auto half_of = [&](int p, int id, bool k) {
        const int off = p & (size - 1);
        const int n = id < 0 ? 0 : min(max(end - p, 0), 16);
        const uint8_t* pool = k ? a.k + static_cast<size_t>(max(id, 0)) * kpage + k0.code + off * kstride
                                : a.v + static_cast<size_t>(max(id, 0)) * vpage + v0.code + off * vstride;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(pool), 0, __builtin_amdgcn_readfirstlane(static_cast<int>(n * (k ? kstride : vstride))), 0x00027000);
    };
    auto scales_of = [&](int p, int id, bool k) {
        const int off = p & (size - 1);
        const int n = id < 0 ? 0 : min(max(end - p, 0), 16);
        const uint8_t* pool = k ? a.k + static_cast<size_t>(max(id, 0)) * kpage + k0.scale : a.v + static_cast<size_t>(max(id, 0)) * vpage + v0.scale;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(pool) + off * NB, 0, __builtin_amdgcn_readfirstlane(n * NB), 0x00027000);
    };
    const int kat = static_cast<int>(l16 * kstride) + g4 * (kKB / (HD / 32)), vat = static_cast<int>(4 * g4 * vstride) + l16 * DimsV<VT, VD>::kRun;
    const int vsat = 4 * g4 * NB + VD * l16 / kKvBlock;

    Dims16<KT> kx[2][NI];
    uint32_t ksc[2][2];
    DimsV<VT, VD> vx[8];
    uint32_t vsc[8];
    auto load_k = [&](int sb, const int (&id)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Rsrc r = half_of(sb + 16 * t, id[t], true);
#pragma unroll
            for (int k = 0; k < NI; k += 2) {
                if constexpr (KT == kKvI4) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, kat + k * (kKB / NI), 0, 0);
                    kx[t][k].w[0] = v[0], kx[t][k].w[1] = v[1], kx[t][k + 1].w[0] = v[2], kx[t][k + 1].w[1] = v[3];
                } else {
                    kx[t][k] = load16<KT>(r, kat + k * (kKB / NI), 0);
                    kx[t][k + 1] = load16<KT>(r, kat + k * (kKB / NI) + kKB / (HD / 16), 0);
                }
            }
            if constexpr (KT != kKvF16) {
                const Rsrc rs = scales_of(sb + 16 * t, id[t], true);
                if constexpr (NB == 8) {
                    const auto s = __builtin_amdgcn_raw_buffer_load_b64(rs, l16 * NB, 0, 0);
                    ksc[t][0] = s[0], ksc[t][1] = s[1];
                } else {
                    ksc[t][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, l16 * NB, 0, 0);
                }
            }
        }
    };
    auto load_v = [&](int sb, const int (&id)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Rsrc r = half_of(sb + 16 * t, id[t], false);
#pragma unroll
            for (int j = 0; j < 4; ++j) vx[4 * t + j] = load_dims<VT, VD>(r, vat, static_cast<int>(j * vstride));
            if constexpr (VT != kKvF16) {
                const Rsrc rs = scales_of(sb + 16 * t, id[t], false);
#pragma unroll
                for (int j = 0; j < 4; ++j) vsc[4 * t + j] = __builtin_amdgcn_raw_buffer_load_b8(rs, vsat + j * NB, 0, 0);
            }
        }
    };
    int sb = c0 + 32 * wv;
    int id[2] = {page_at(sb), page_at(sb + 16)};
    load_k(sb, id);
    __builtin_amdgcn_sched_barrier(0);   // in this order, as in the loop: a wait for K then leaves V in flight
    load_v(sb, id);
    int nid[2] = {page_at(sb + 32 * kWaves), page_at(sb + 32 * kWaves + 16)};

    float post[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        post[b] = a.post * kSixteen<KT>;
        if (a.bf16) {   // uniform: q as fp16, a row's largest brought to [2^13, 2^14)
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < NI; ++k)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int e = 0; e < 4; ++e) m = max_magnitude(m, qb[b][k][hf][e]);
            float top = __uint_as_float(max(m << 16, m & 0xffff0000u));
            top = fmaxf(top, xor_lane<16>(top));
            top = fmaxf(top, xor_lane<32>(top));
            const int sh = q_shift(top);
            post[b] *= ldexpf(1.0f, -sh);
#pragma unroll
            for (int k = 0; k < NI; ++k)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int e = 0; e < 4; ++e) qb[b][k][hf][e] = bf16_to_f16(qb[b][k][hf][e], sh);
        }
    }
    floatx4 o[RB][VD];
    float m_run[RB], l_run[RB];   // l_run: this lane's positions only
#pragma unroll
    for (int b = 0; b < RB; ++b) {
#pragma unroll
        for (int e = 0; e < VD; ++e) o[b][e] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        m_run[b] = -INFINITY;
        l_run[b] = 0.0f;
    }

    for (int st = 0; st < nsteps; ++st) {
        float sc[RB][8];   // j: position sb + 4 g4 + j, or 16 + 4 g4 + j - 4 further
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            floatx4 acc[RB];
#pragma unroll
            for (int b = 0; b < RB; ++b) acc[b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < NI; ++k) {
                Scale2 s = {};
                if constexpr (KT != kKvF16) {   // block 4 (k / 2) + g4
                    const uint32_t byte = (ksc[t][k >> 1] >> (8 * g4)) & 0xffu;
                    s = scale2<KT>(byte, byte);
                }
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const half8 kk = operand<KT>(kx[t][k], hf, s);
#pragma unroll
                    for (int b = 0; b < RB; ++b) acc[b] = mfma16(kk, __builtin_bit_cast(half8, qb[b][k][hf]), acc[b]);
                }
            }
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[b][4 * t + r] = acc[b][r] * post[b];
        }
        const int bad = (id[0] < 0 && sb < end ? 1 : 0) | (id[1] < 0 && sb + 16 < end ? 2 : 0);   // uniform
        // the loads are not under a branch: behind one, every wait would be for all that might be out
        const int next = sb + 32 * kWaves;
        load_k(next, nid);
        const bool tail = sb + 31 > base;   // uniform: not every row sees the whole step
        half8 ph[RB];
        uint32_t seen[RB];
        float p[RB][8];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            if (bad)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (bad >> (j >> 2) & 1) sc[b][j] = __builtin_nanf("");
            seen[b] = 0xffu;
            if (tail || kFewRows * (b + 1) > rows) {
                seen[b] = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (sb + 4 * g4 + (j < 4 ? j : 12 + j) <= lim[b]) seen[b] |= 1u << j;
                    else sc[b][j] = -INFINITY;
                }
            }
            float mloc = sc[b][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mloc = fmaxf(mloc, sc[b][j]);
            mloc = fmaxf(mloc, xor_lane<16>(mloc));
            mloc = fmaxf(mloc, xor_lane<32>(mloc));
            const float m_new = mloc > m_run[b] + kLazy ? mloc : m_run[b];
            const float m_ref = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: exp2(-inf) = 0, no NaN
            const float alpha = m_run[b] == m_new || m_run[b] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run[b] - m_ref);   // -inf: o is 0
            float lsum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[b][j] = __builtin_amdgcn_exp2f(sc[b][j] - m_ref + kPScale);
                lsum += p[b][j];
            }
            l_run[b] = l_run[b] * alpha + lsum;
            m_run[b] = m_new;
            if (__ballot(alpha != 1.0f)) {   // uniform: some row's maximum moved
                float al[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) al[r] = __shfl(alpha, 4 * g4 + r, 64);
#pragma unroll
                for (int e = 0; e < VD; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[b][e][r] *= al[r];
            }
            ph[b] = h8(pack_f16(p[b][0], p[b][1]), pack_f16(p[b][2], p[b][3]), pack_f16(p[b][4], p[b][5]), pack_f16(p[b][6], p[b][7]));
        }
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
                float(*pw)[32] = pb[wv];   // [row][position], -1: not seen
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int j = 0; j < 8; ++j) pw[kFewRows * b + l16][4 * g4 + (j < 4 ? j : 12 + j)] = seen[b] >> j & 1 ? p[b][j] : -1.0f;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                for (int pp = 0; pp < 32; ++pp) {
                    const int p1 = sb + pp, pid = pp < 16 ? id[0] : id[1];
                    if (p1 >= end || pid < 0) continue;   // uniform; not read: zeros
                    const KvRow<VT> at = kv_row<VT>(p1 & (size - 1), kv, a.n_kv, size, HD);
                    const uint8_t* page = a.v + static_cast<size_t>(pid) * vpage;
#pragma unroll
                    for (int e = 0; e < VD; ++e) {
                        float v;
                        if constexpr (VT == kKvF16) v = half_bits_to_float(reinterpret_cast<const uint16_t*>(page + at.code)[DimsV<VT, VD>::dim(l16, e)]);
                        else v = odd_value<VT>(page[at.scale + VD * l16 / kKvBlock]);
                        if (fabsf(v) <= FLT_MAX) continue;
#pragma unroll
                        for (int b = 0; b < RB; ++b)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float x = pw[kFewRows * b + 4 * g4 + r][pp];
                                if (!(x < 0.0f)) o[b][e][r] = __builtin_fmaf(x, v, o[b][e][r]);
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
            const half8 v0 = h8(ev[0], ev[1], ev[2], ev[3]), v1 = h8(od[0], od[1], od[2], od[3]);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                o[b][2 * e] = mfma16(ph[b], v0, o[b][2 * e]);
                o[b][2 * e + 1] = mfma16(ph[b], v1, o[b][2 * e + 1]);
            }
        }
        load_v(next, nid);
        sb = next;
        id[0] = nid[0], id[1] = nid[1];
        nid[0] = page_at(sb + 32 * kWaves), nid[1] = page_at(sb + 32 * kWaves + 16);
    }

#pragma unroll
    for (int b = 0; b < RB; ++b) {
        if (b == 1 && !second) break;
        l_run[b] += xor_lane<16>(l_run[b]);
        l_run[b] += xor_lane<32>(l_run[b]);
        if (g4 == 0) {
            stat[wv][0][kFewRows * b + l16] = m_run[b];
            stat[wv][1][kFewRows * b + l16] = l_run[b];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < VD; e += 4)
                *reinterpret_cast<float4*>(&slab[wv][kFewRows * b + 4 * g4 + r][DimsV<VT, VD>::dim(l16, e)]) =
                    make_float4(o[b][e][r], o[b][e + 1][r], o[b][e + 2][r], o[b][e + 3][r]);
    }
    __syncthreads();
    if (threadIdx.x < (second ? ROWS : kFewRows)) {   // the parts' weights and the joined sum of every row
        const int r = threadIdx.x;
        float m = stat[0][0][r];
#pragma unroll
        for (int p = 1; p < kWaves; ++p) m = fmaxf(m, stat[p][0][r]);
        const float ref = m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
#pragma unroll
        for (int p = 0; p < kWaves; ++p) {
            const float f = __builtin_amdgcn_exp2f(stat[p][0][r] - ref);
            fac[p][r] = f * kSixteen<VT>;
            l = __builtin_fmaf(stat[p][1][r], f, l);
        }
        sum[0][r] = m;
        sum[1][r] = l;
    }
    __syncthreads();
    constexpr int L4 = HD / 4, kUp = kThreads / L4;   // four dims a lane, kUp rows a round
    const int d = 4 * (static_cast<int>(threadIdx.x) % L4);
    for (int r = static_cast<int>(threadIdx.x) / L4; r < rows; r += kUp) {
        const int t = r / G, h = kv * G + r - t * G, at = rq.start + t;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f}, g[4];
        if (a.chunks == 1) load_gate<HD>(a, at, h, d, g);
#pragma unroll
        for (int p = 0; p < kWaves; ++p) {
            const float4 x = *reinterpret_cast<const float4*>(&slab[p][r][d]);
            const float f = fac[p][r];
            v[0] = __builtin_fmaf(x.x, f, v[0]);
            v[1] = __builtin_fmaf(x.y, f, v[1]);
            v[2] = __builtin_fmaf(x.z, f, v[2]);
            v[3] = __builtin_fmaf(x.w, f, v[3]);
        }
        if (a.chunks == 1) {
            normed4(v, sum[1][r], base + t < 0);
            finish4<HD>(a, at, h, d, v, g);
        } else {
            const size_t rec = (static_cast<size_t>(chunk) * a.ntok + at) * a.n_head + h;
            *reinterpret_cast<float4*>(a.wo + rec * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
            if (d == 0) *reinterpret_cast<float2*>(a.wml + 2 * rec) = make_float2(sum[0][r], sum[1][r]);
        }
    }
}

// ---- more rows: tiles in LDS -------------------------------------------------------------------------------------------------
// WAVES waves of 32 query rows over steps of STEP positions, v_mfma_f32_32x32x16: lane l32 = l % 32, h = l / 32; A rows, B and D
// columns are l32; A and B hold k = 8 h + 0..7; D register r is row 8 (r / 4) + 4 h + r % 4.
//   scores    D[position][row] += K[position][dims] . q_row[dims]: a lane has half of its row's scores, so a row's maximum and sum
//             take one exchange with lane l ^ 32, and what scales a row is a lane's own value
//   P V       D[dim][row] += V^T[dim][positions] P^T[positions][row].  P's registers are the B operand as they are: k slot
//             (h, e) of 16 positions is position 8 (e / 4) + 4 h + e % 4, and V's transposed reads (ds_read_b64_tr_b16: 16 lanes
//             give the addresses of 4 positions x 16 dims and get a dim's four positions each) take the same order.
// q and o stay in registers.  16-bit K and V go from memory into LDS without passing registers, the next step's over this step's
// products; codes go there as they are, two steps ahead, and are turned to fp16 tiles by the next step.  Turning codes on their way
// from memory held up every wave: 999 tokens behind 8 K of I8 / I4 249 us, 179 so.
// Bound by the matrix cores and LDS together: a step of 256 rows x 32 positions is 2048 cycles of products and 256 KB of operands, 2048
// cycles at 128 bytes each, with the softmax beside them, and takes some 3400: one prompt of 8001 tokens x 16 heads of 256 dims
// 457 to 502 us, 1.05 to 1.15 PFLOP/s (a large library product 1.18), the matrix cores busy for 58 % of it.  Codes cost 7 % more over F16 pages (999
// tokens behind 7 K: 159 us with the join, I8 170, I4 163).
// LDS rows have no padding (the direct loads write 1024 bytes in a row); instead their 16-byte (K) or 32-byte (V) pieces are permuted by the row, so that the lanes of a read fall on different banks:
// K piece c of row p is at c ^ (p % 16), V piece c at c ^ {0, 3, 5, 6}[p % 4].
constexpr int kPaged = 1, kRowsF16 = 2, kRowsBF16 = 3;   // where K and V come from

// 16 bytes a lane from base + off into LDS: lane l's at `to` + 16 l (base and to uniform).  Written out because the compiler, where
// it knows of such a load, waits for all of them before any read of LDS; the loop waits for its own, a step later.  Nothing else
// here uses m0.
__device__ __forceinline__ void load_lds(const uint8_t* base, uint32_t off, uint32_t to) {
    const uint64_t b = reinterpret_cast<uintptr_t>(base);
    const uint64_t u = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b))) |
                       static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b >> 32)))) << 32;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(static_cast<int>(to))), "v"(off),
                 "s"(u)
                 : "memory");
}
// the same for four bytes a lane, each lane's from a place of its own
__device__ __forceinline__ void load_lds4(const uint8_t* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(static_cast<int>(to))), "v"(from) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*) p));
}

// N products, product k of the operand that read(k) brings from LDS, with AHEAD operands on their way: left alone the compiler
// reads an operand, waits for it and multiplies.  `ready` holds the first ones.
template <int AHEAD, int N, typename READ, typename PRODUCT>
__device__ __forceinline__ void stream(u32x4 (&ready)[AHEAD], READ&& read, PRODUCT&& product) {
    static_assert(N >= AHEAD, "");
#pragma unroll
    for (int k = 0; k < N; ++k) {
        product(k, ready[k % AHEAD]);
        if (k + AHEAD < N) ready[k % AHEAD] = read(k + AHEAD);
        __builtin_amdgcn_sched_barrier(0x6);   // vector and scalar arithmetic alone may pass
    }
}

// the same value, of which the compiler does not know that a loop leaves it as it is: what is made of it then is made anew in each
// round, by an instruction or two, and not kept in registers that there are none of
template <bool ON>
__device__ __forceinline__ int fresh(int x) {
    if constexpr (ON) asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ int v_swizzle(int p) { return (0x6530 >> (4 * (p & 3))) & 7; }

template <int HD>
struct TileShape {
    static constexpr int kStep = HD == 256 ? 32 : 64;
    static constexpr int kRow = 2 * HD;               // bytes of a row in LDS
    static constexpr int kHalf = kStep * kRow;        // of K or V of a step
    static constexpr int kTile = 2 * kHalf;
};

// ---- a step of 32 query rows -------------------------------------------------------------------------------------------------
// where a V row's values are, for the few that are read past the tile
struct VRow {
    const uint8_t* p;
    size_t scale;   // codes: from p to the row's scale bytes
    bool ok;        // there is one
};

// Scores, softmax and P V of the positions sb .. sb + STEP - 1 in the tiles kt and vt for the wave's 32 rows.  lim: the last position
// that the lane's row sees, last: that any row of the workgroup sees; cut: uniform, some row does not see the whole step; bad: 16-position
// pieces without a page.  scored() is called when the last product of the scores is issued, v_ready() when K is read, has_odd() tells (uniformly) whether a value that is not finite was
// taken out of vt, v_row(position) where it is.  FRESH: no addresses kept in registers.  V_EARLY: the first of V over the softmax.
template <bool BF, int HD, int VT, bool FRESH, bool V_EARLY, typename SCORED, typename READY, typename ODD, typename ROWS>
__device__ __forceinline__ void tile_step(const uint8_t* kt, const uint8_t* vt, int kat, int vat, const u32x4 (&q)[HD / 16], floatx16 (&o)[HD / 32],
                                          float& m_run, float& l_run, float post, int sb, int last, int lim, int h, uint32_t bad, bool cut,
                                          SCORED&& scored, READY&& v_ready, ODD&& has_odd, ROWS&& v_row) {
    constexpr int STEP = TileShape<HD>::kStep, ROW = TileShape<HD>::kRow, NS = STEP / 32, NK = HD / 16, ND = HD / 32;
    constexpr int AHEAD = HD == 256 ? 2 : 4;   // operands from LDS on their way
    floatx16 s[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] = 0.0f;
    const int ka = fresh<FRESH>(kat), va = fresh<FRESH>(vat);
    auto k_piece = [&](int n) {   // dims 16 k .. of positions 32 j ..
        const int j = n / NK, k = n % NK;
        return *reinterpret_cast<const u32x4*>(kt + 32 * j * ROW + (ka ^ ((k & 7) << 5)) + (k >> 3) * 256);
    };
    auto v_piece = [&](int n) {   // 16 positions 16 k .. of dims 32 d ..
        const int k = n / ND, d = n % ND;
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const uint8_t* at = vt + 16 * k * ROW + (va ^ ((d & 3) << 6)) + (d >> 2) * 256;
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*) at));
        const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*) (at + 8 * ROW)));
        return u32x4{x.x, x.y, y.x, y.y};
    };
    // the matrix cores go to the wave that has its operands, so that the two waves of a SIMD take turns at them and at the softmax
    u32x4 ready[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) ready[n] = k_piece(n);
    __builtin_amdgcn_sched_barrier(0x6);
    __builtin_amdgcn_s_setprio(1);
    stream<AHEAD, NS * NK>(ready, k_piece, [&](int n, u32x4 x) { s[n / NK] = mfma32<BF>(x, q[n % NK], s[n / NK]); });
    __builtin_amdgcn_s_setprio(0);
    scored();
    auto v_first = [&] {
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) ready[n] = v_piece(n);
        __builtin_amdgcn_sched_barrier(0x6);
    };
    if constexpr (V_EARLY) {
        v_ready();
        v_first();
    }
    if (bad)
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (bad >> (2 * j + (r >> 3)) & 1) s[j][r] = __builtin_nanf("");
    if (cut)
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (sb + 32 * j + 8 * (r >> 2) + 4 * h + (r & 3) > lim) s[j][r] = -INFINITY;
    float top = s[0][0];
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[j][r]);
    top = fmaxf(top, xor_lane<32>(top)) * post;   // post > 0
    const float m_new = top > m_run + kLazy ? top : m_run;
    const float m_ref = m_new == -INFINITY ? 0.0f : m_new;   // nothing seen yet: exp2(-inf) = 0, no NaN
    const float alpha = m_run == m_new || m_run == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_ref);   // -inf: o is 0
    m_run = m_new;
    const float shift = (BF ? 0.0f : kPScale) - m_ref;
    float sum = 0.0f;
    u32x4 p[2 * NS];
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], post, shift)), y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r + 1], post, shift));
            sum += x + y;
            p[2 * j + (r >> 3)][(r & 7) >> 1] = BF ? pack_bf16(x, y) : pack_f16(x, y);
        }
    l_run = __builtin_fmaf(l_run, alpha, sum);
    if (__ballot(alpha != 1.0f)) {   // uniform: some row's maximum moved
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
    if constexpr (!V_EARLY) v_ready();
    if (has_odd()) {   // uniform
        for (int pp = 0; pp < STEP; ++pp) {
            const int at = sb + pp;
            if (at > last) break;
            // the row's p of this position, from the half that has it
            const int j = pp >> 5, r = 4 * ((pp >> 3) & 3) + (pp & 3);
            float x = 0.0f;
#pragma unroll
            for (int jj = 0; jj < NS; ++jj)
#pragma unroll
                for (int rr = 0; rr < 16; ++rr)
                    if (j == jj && r == rr) x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[jj][rr], post, shift));
            const float other = xor_lane<32>(x);
            if (((pp >> 2) & 1) != h) x = other;
            const int hh = fresh<true>(h);   // with the barriers below: no address or load of another dim takes a register here
            const VRow row = v_row(at);
            if (!row.ok) continue;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
#pragma unroll
                for (int r2 = 0; r2 < 16; ++r2) {
                    const int dim = 32 * d + 8 * (r2 >> 2) + 4 * hh + (r2 & 3);
                    float v;
                    if constexpr (VT != kKvF16) v = odd_value<VT>(row.p[row.scale + d]);
                    else if constexpr (BF) v = __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row.p)[dim]) << 16);
                    else v = half_bits_to_float(reinterpret_cast<const uint16_t*>(row.p)[dim]);
                    if (!(fabsf(v) <= FLT_MAX) && at <= lim) o[d][r2] = __builtin_fmaf(x, v, o[d][r2]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if constexpr (!V_EARLY) v_first();
    __builtin_amdgcn_s_setprio(1);
    stream<AHEAD, 2 * NS * ND>(ready, v_piece, [&](int n, u32x4 x) { o[n % ND] = mfma32<BF>(x, p[n / ND], o[n % ND]); });
    __builtin_amdgcn_s_setprio(0);
}

// what is not finite leaves the 16 bytes at `at`; whether there was any
template <bool BF>
__device__ __forceinline__ bool clear_odd(u32x4* at) {
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
    u32x4 w = *at;
    bool found = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if ((w[e] & E) == E) w[e] &= 0xffff0000u, found = true;
        if ((w[e] & (E << 16)) == (E << 16)) w[e] &= 0xffffu, found = true;
    }
    if (found) *at = w;
    return found;
}

template <int SRC, int KT, int VT, int HD, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void batch_tile_kernel(BatchArgs a) {
    using S = TileShape<HD>;
    constexpr int THREADS = 64 * WAVES, ROWS = kWaveRows * WAVES;   // query rows of a workgroup
    constexpr bool BF = SRC == kRowsBF16, PAGED = SRC == kPaged;
    constexpr bool CODES = KT != kKvF16;             // K and V are codes to be turned to fp16 (both or neither)
    constexpr int LEAD = CODES ? 2 : 1;              // steps that loads are ahead
    constexpr int STEP = S::kStep, ROW = S::kRow;
    constexpr int NK = HD / 16, ND = HD / 32;
    // the waves that load 16-bit rows, and rows of a step of each.  Eight waves: the first four, whose loads hold them up for 500 cycles
    // and more, so that the other wave of a SIMD is ahead of them and one is at its products while the other is at its softmax (8001
    // tokens 505 us with two workgroups of four waves, 485 so)
    constexpr int LOADERS = 4, WR = STEP / LOADERS;
    constexpr int PER = 1024 / ROW, NL = WR / PER;   // rows a direct load, loads a wave
    constexpr int NG = STEP / 16;                    // 16-position pieces, each in one page
    constexpr int NB = HD / kKvBlock;
    constexpr int kKB = kv_row_bytes(KT, HD), kVB = kv_row_bytes(VT, HD);
    constexpr int RAW = STEP * (kKB + kVB + 2 * NB);   // a step's codes and scales
    __shared__ __attribute__((aligned(16))) uint8_t pool[2 * S::kTile + (CODES ? 2 * RAW : 0)];
    __shared__ int odd[2];   // a tile's V had a value that is not finite
    static_assert(sizeof(pool) >= kMaxReq * sizeof(int), "the requests' tiles are counted in the tiles' place");

    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
    const int G = a.n_head / a.n_kv;
    // KV heads innermost: workgroups go to the XCDs round robin, so a head's tiles meet its K and V in one or two L2s
    const int kv = blockIdx.x % a.n_kv;
    const uint32_t rank = blockIdx.x / a.n_kv;
    int i = 0, level = 0, chunk = 0;
    if (tid < 2) odd[tid] = 0;
    if constexpr (PAGED) {
        auto tiles = [&](int n) { return (n * G + ROWS - 1) / ROWS; };
        int item = 0;
        if (!item_of_rank(a, rank, [&](const Req& r) { return r.n * G > a.few ? tiles(r.n) * chunks_in(a, r.len) : 0; }, &i, &item)) return;   // uniform
        const int n = tiles(request(a, i, word(a.row_start, i), word(a.row_start, i + 1)).n);
        chunk = item / n;
        level = n - 1 - item % n;
    } else {
        if (!find_tile<ROWS, THREADS>(a, reinterpret_cast<int*>(pool), rank, G, &i, &level)) return;   // uniform
    }
    const Req rq = request(a, i, word(a.row_start, i), word(a.row_start, i + 1));
    const int rows = rq.n * G, base = rq.len - rq.n, c0 = chunk * a.chunk;
    const int first = base + level * ROWS / G, last = base + min(level * ROWS + ROWS - 1, rows - 1) / G;   // of the workgroup's tokens
    if (chunk > 0 && c0 > last) return;
    const int row0 = level * ROWS + kWaveRows * wv, row = row0 + l32, rowc = min(row, rows - 1), tok = rowc / G;
    const int head = kv * G + rowc - tok * G;
    const int lim = row < rows ? base + tok : -1;   // the row sees every position up to here
    const int wfirst = base + min(row0, rows - 1) / G, wlast = row0 < rows ? base + min(row0 + kWaveRows - 1, rows - 1) / G : -1;
    const int end = min(last + 1, c0 + a.chunk), nsteps = max(end - c0 + STEP - 1, 0) / STEP;

    u32x4 q[NK];
    {
        const uint16_t* qr = reinterpret_cast<const uint16_t*>(a.q) + (static_cast<ptrdiff_t>(rq.start + tok) * a.q_stride + head * HD) + 8 * h;
#pragma unroll
        for (int k = 0; k < NK; ++k) q[k] = *reinterpret_cast<const u32x4*>(qr + 16 * k);
    }

    const int size = 1 << a.shift;
    const size_t kpage = kv_page_bytes(KT, size, a.n_kv, HD), vpage = kv_page_bytes(VT, size, a.n_kv, HD);
    // bytes from a position's row to the next
    const size_t kstride = !PAGED ? 2 * static_cast<size_t>(a.k_stride) : !CODES ? static_cast<size_t>(a.n_kv) * kKB : kKB;
    const size_t vstride = !PAGED ? 2 * static_cast<size_t>(a.v_stride) : !CODES ? static_cast<size_t>(a.n_kv) * kVB : kVB;
    const int* const ids = a.table + static_cast<size_t>(i) * a.table_stride;
    int id[NG];              // pages of the step that is loaded next
    int asked[NG];           // what the table says of the one after
    uint32_t next_bad = 0;   // of its 16-position pieces: not a page
    // A step's page ids, by scalar loads, which come back in any order: a read of LDS beside them would wait for them, so they are
    // asked for where none is on its way, before the softmax
    auto ask_pages = [&](int sb) {
        if constexpr (PAGED) {
#pragma unroll
            for (int g = 0; g < NG; ++g) asked[g] = word(ids, max(min(min(sb + 16 * g, last) >> a.shift, a.table_stride - 1), 0));
        }
    };
    auto find_pages = [&](int sb) {
        next_bad = 0;
        if constexpr (PAGED) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int p = sb + 16 * g, x = asked[g];
                const bool ok = p <= last && p >> a.shift < a.table_stride && x >= 0 && x < a.n_pages;
                if (p <= last && !ok) next_bad |= 1u << g;
                id[g] = ok ? x : 0;
            }
        }
    };
    // Rows of 16-bit values straight into LDS: a load's lane l writes piece l % PIECES of its row l / PIECES.  Both permutations are
    // exclusive ors and linear in the row, so the n-th load's piece is the first's with a constant.
    constexpr int PIECES = ROW / 16;
    const int p0 = WR * wv, lr = lane / PIECES;
    const uint32_t k_piece0 = 16 * (lane % PIECES ^ ((p0 + lr) & 15)), v_piece0 = 16 * (lane % PIECES ^ (v_swizzle(lr) << 1));
    const uint32_t k_line = static_cast<uint32_t>(lr) * static_cast<uint32_t>(kstride), v_line = static_cast<uint32_t>(lr) * static_cast<uint32_t>(vstride);
    auto direct = [&](const uint8_t* src, size_t page_bytes, size_t stride, size_t at0, int sb, uint32_t to, bool k) {
        const uint32_t piece0 = fresh<PAGED>(k ? k_piece0 : v_piece0);
        const uint8_t* from;
        int over = 0;   // how many of the wave's rows lie behind the call's (prompts: the last step of the last rows)
        if constexpr (PAGED) {
            int page = id[0];
#pragma unroll
            for (int g = 1; g < NG; ++g) page = p0 / 16 == g ? id[g] : page;
            from = src + static_cast<size_t>(page) * page_bytes + at0 + ((sb + p0) & (size - 1)) * stride;
        } else {
            const int r = min(rq.start + sb + p0, a.ntok - 1);
            over = r + WR - a.ntok;
            from = src + static_cast<size_t>(r) * stride + at0;
        }
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            const uint32_t piece = piece0 ^ (k ? 16 * (n * PER & 15) : 32 * v_swizzle(n * PER));
            const uint32_t lds = to + (p0 + n * PER) * ROW;
            if (over <= 0) load_lds(from + n * PER * stride, (k ? k_line : v_line) + piece, lds);
            else load_lds(from, static_cast<uint32_t>(min(n * PER + lr, WR - 1 - over)) * static_cast<uint32_t>(stride) + piece, lds);
        }
    };
    const size_t k_at = PAGED ? kv_row<KT>(0, kv, a.n_kv, size, HD).code : static_cast<size_t>(kv) * ROW;
    const size_t v_at = PAGED ? kv_row<VT>(0, kv, a.n_kv, size, HD).code : static_cast<size_t>(kv) * ROW;
    const uint32_t pool0 = lds_address(pool);
    // Codes and their scales into LDS as they are: rows of a page lie one behind another, so a wave's 1024 bytes are in a row.
    // The loading waves take K's and V's codes in turn, two of them the scales.
    auto raw_codes = [&](const uint8_t* src, size_t page_bytes, size_t at0, auto type, int sb, uint32_t to, int turn) {
        constexpr int B = kv_row_bytes(decltype(type)::value, HD), R = 1024 / B;   // rows a load
        static_assert(R <= 16, "within a page's 16");
        if (turn >= STEP / R) return;   // uniform
        const int p = turn * R;
        int page = id[0];
#pragma unroll
        for (int g = 1; g < NG; ++g) page = p / 16 == g ? id[g] : page;
        load_lds(src + static_cast<size_t>(page) * page_bytes + at0 + static_cast<size_t>((sb + p) & (size - 1)) * B, 16 * lane, to + 1024 * turn);
    };
    auto raw_scales = [&](const uint8_t* src, size_t page_bytes, size_t at0, int sb, uint32_t to) {
        const uint32_t l = static_cast<uint32_t>(fresh<PAGED>(lane)), p = 4 * l / NB;   // the lane's four bytes
        int page = id[0];
#pragma unroll
        for (int g = 1; g < NG; ++g) page = p / 16 == g ? id[g] : page;
        load_lds4(src + static_cast<size_t>(page) * page_bytes + at0 + static_cast<size_t>((sb + static_cast<int>(p)) & (size - 1)) * NB + (4 * l) % NB, to);
    };
    // a step's rows on their way, to tile or raw buffer `buf`
    auto load = [&](int buf, int sb) {
        if (wv >= LOADERS) return;   // uniform
        if constexpr (CODES) {
            const uint32_t to = pool0 + 2 * S::kTile + buf * RAW;
#pragma unroll
            for (int n = 0; n < S::kHalf / 2 / (1024 * LOADERS); ++n) {   // as many as rows of eight bits take
                raw_codes(a.k, kpage, k_at, std::integral_constant<int, KT>{}, sb, to, wv + n * LOADERS);
                raw_codes(a.v, vpage, v_at, std::integral_constant<int, VT>{}, sb, to + STEP * kKB, wv + n * LOADERS);
            }
            if (wv == 0) raw_scales(a.k, kpage, kv_row<KT>(0, kv, a.n_kv, size, HD).scale, sb, to + STEP * (kKB + kVB));
            if (wv == 1) raw_scales(a.v, vpage, kv_row<VT>(0, kv, a.n_kv, size, HD).scale, sb, to + STEP * (kKB + kVB + NB));
        } else {
            const uint32_t to = pool0 + buf * S::kTile;
            direct(a.k, kpage, kstride, k_at, sb, to, true);
            direct(a.v, vpage, vstride, v_at, sb, to + S::kHalf, false);
        }
    };
    // raw buffer `buf` to tile `buf`: a thread turns 16 dims of K and of V of a position at a time, both read before either is turned
    auto codes16 = [](auto type, const uint8_t* codes, int at) {
        constexpr int T = decltype(type)::value;
        Dims16<T> x;
        if constexpr (T == kKvI8) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(codes + 16 * at);
            x.w[0] = v[0], x.w[1] = v[1], x.w[2] = v[2], x.w[3] = v[3];
        } else if constexpr (T == kKvI4) {
            const uint2 v = *reinterpret_cast<const uint2*>(codes + 8 * at);
            x.w[0] = v.x, x.w[1] = v.y;
        }
        return x;
    };
    auto swap_halves = [](auto& x, bool yes) {
        constexpr int W = sizeof(x.w) / sizeof(x.w[0]) / 2;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const uint32_t lo = x.w[e], hi = x.w[e + W];
            x.w[e] = yes ? hi : lo;
            x.w[e + W] = yes ? lo : hi;
        }
    };
    auto turn = [&](int buf) {
        if constexpr (CODES) {
            constexpr int UP = THREADS / (HD / 16);   // positions to a thread's next unit
            const uint8_t* const raw = pool + 2 * S::kTile + buf * RAW;
            const uint8_t* const scales = raw + STEP * (kKB + kVB);
            uint8_t* const to = pool + buf * S::kTile;
            const uint32_t t = static_cast<uint32_t>(fresh<true>(tid)), pos = t / (HD / 16), col = t % (HD / 16);
#pragma unroll
            for (int u = 0; u < STEP / UP; ++u) {
                const uint32_t p = pos + u * UP, n = t + u * THREADS;   // unit n = p HD / 16 + col
                Dims16<KT> k = codes16(std::integral_constant<int, KT>{}, raw, n);
                const uint32_t ks = scales[n / 2];
                Dims16<VT> v = codes16(std::integral_constant<int, VT>{}, raw + STEP * kKB, n);
                const uint32_t vs = scales[STEP * NB + n / 2];
                const Scale2 k2 = scale2<KT>(ks, ks), v2 = scale2<VT>(vs, vs);
                uint8_t* const row = to + p * ROW;
                // columns from the ninth on write their second half first: a row's 16 lanes would meet on half of the banks
                const uint32_t other = col & 8;
                const uint32_t at_k = (16 * ((2 * col) ^ (p & 15))) ^ (2 * other), at_v = (32 * (col ^ v_swizzle(p))) ^ (2 * other);
                swap_halves(k, other != 0);
                swap_halves(v, other != 0);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) *reinterpret_cast<half8*>(row + (at_k ^ (16 * hf))) = operand<KT>(k, hf, k2);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) *reinterpret_cast<half8*>(row + S::kHalf + (at_v ^ (16 * hf))) = operand<VT>(v, hf, v2);
            }
        }
    };

    ask_pages(c0);
    find_pages(c0);
    if (nsteps > 0) load(0, c0);
    uint32_t bad = next_bad, bad2 = 0;   // of this step and the next
    ask_pages(c0 + STEP);
    if constexpr (CODES) {   // codes come two steps ahead
        find_pages(c0 + STEP);
        if (nsteps > 1) load(1, c0 + STEP);
        bad2 = next_bad;
        ask_pages(c0 + 2 * STEP);
    }
    // q is here before the loop: inside it, a wait for q would be one for the tiles on their way
#pragma unroll
    for (int k = 0; k < NK; ++k) asm volatile("" : "+v"(q[k]));

    floatx16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;   // l_run: the lane's half of the row's positions
    float post = a.post * kSixteen<KT>;
    if (PAGED && a.bf16) {   // uniform: q as fp16, a row's largest brought to [2^13, 2^14)
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = max_magnitude(m, q[k][e]);
        float top = __uint_as_float(max(m << 16, m & 0xffff0000u));
        top = fmaxf(top, xor_lane<32>(top));
        const int sh = q_shift(top);
        post *= ldexpf(1.0f, -sh);
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) q[k][e] = bf16_to_f16(q[k][e], sh);
    }

    // the lane's addresses in a tile: K piece h of row l32, V piece of position 4 h + (l % 16) / 4
    const int kat = l32 * ROW + ((h ^ (l32 & 15)) << 4);
    const int vp = 4 * h + ((lane & 15) >> 2);
    const int vat = vp * ROW + ((((lane >> 4) & 1) ^ v_swizzle(vp)) << 5) + 8 * (lane & 3);
    auto v_row = [&](int at) {
        VRow r = {a.v, 0, true};
        if constexpr (PAGED) {
            const int page = word(ids, min(at >> a.shift, a.table_stride - 1));
            const KvRow<VT> row = kv_row<VT>(at & (size - 1), kv, a.n_kv, size, HD);
            r.ok = page >= 0 && page < a.n_pages;
            r.p += static_cast<size_t>(r.ok ? page : 0) * vpage + row.code;
            r.scale = row.scale - row.code;
        } else {
            r.p += (static_cast<size_t>(rq.start) + at) * vstride + v_at;
        }
        return r;
    };

    if constexpr (CODES) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        turn(0);
    }
    for (int st = 0; st < nsteps; ++st) {
        const int sb = c0 + st * STEP, buf = st & 1;
        const uint8_t* const tile = pool + buf * S::kTile;
        const bool more = st + 1 < nsteps;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();   // this step's tile is there, and the other one is read
        asm volatile("" ::: "memory");
        const uint32_t step_bad = bad;
        auto load_ahead = [&] {
            find_pages(sb + LEAD * STEP);
            if (st + LEAD < nsteps) load(CODES ? buf : buf ^ 1, sb + LEAD * STEP);
            bad = CODES ? bad2 : next_bad;
            bad2 = next_bad;
        };
        if (!CODES) load_ahead();
        // half of the waves turn the next step's codes before their products, half after: a SIMD has one of each
        if (CODES && more && wv >= WAVES / 2) turn(buf ^ 1);
        const bool tail = sb + STEP - 1 > first;   // uniform: not every row sees the whole step
        if (tail) {
            // what is not finite leaves V's tile, so that a product with a masked zero is zero, and is added by itself to the rows
            // that see it
            uint8_t* const vt = pool + buf * S::kTile + S::kHalf;
            bool found = false;
#pragma unroll
            for (int n = 0; n < S::kHalf / (16 * THREADS); ++n) found |= clear_odd<BF>(reinterpret_cast<u32x4*>(vt + 16 * (tid + n * THREADS)));
            if (found) odd[buf] = st + 1;   // every writer stores the same
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
        auto scored = [&] {
            if (CODES) load_ahead();   // at the step's start it held up the waves that turn codes then: 900 cycles became 1340
            ask_pages(sb + (LEAD + 1) * STEP);
        };
        if (sb > wlast) scored();   // uniform in the wave (with `else` for the next line the compiler spills half of o)
        if (sb <= wlast)
            tile_step<BF, HD, VT, PAGED, HD == 128>(tile, tile + S::kHalf, kat, vat, q, o, m_run, l_run, post, sb, last, lim, h, step_bad,
                                                    sb + STEP - 1 > wfirst || row0 + kWaveRows > rows, scored, [] {},
                                                    [&] { return tail && odd[buf] == st + 1; }, v_row);
        if (CODES && more && wv < WAVES / 2) turn(buf ^ 1);
    }

    l_run += xor_lane<32>(l_run);
    if (row >= rows) return;
    const int t = rq.start + tok;
    if (a.chunks > 1) {
        const size_t rec = (static_cast<size_t>(chunk) * a.ntok + t) * a.n_head + head;
        float* const to = a.wo + rec * HD + 4 * h;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<float4*>(to + 32 * d + 2 * r) =
                    make_float4(o[d][r] * kSixteen<VT>, o[d][r + 1] * kSixteen<VT>, o[d][r + 2] * kSixteen<VT>, o[d][r + 3] * kSixteen<VT>);
        if (h == 0) *reinterpret_cast<float2*>(a.wml + 2 * rec) = make_float2(m_run, l_run);
        return;
    }
    // the lane's half of its row, from its registers.  Gates four 32-dim blocks ahead: one block's at a time would wait for memory
    // eight times over (3 us each way at a workgroup's end)
    const float unit = kSixteen<VT> / l_run;
    constexpr int BLOCKS = 4;
    const float* const from = a.gate ? a.gate + static_cast<ptrdiff_t>(t) * a.gate_stride + head * 2 * HD + HD + 4 * h : nullptr;
    float4u g[BLOCKS][4];
    auto block = [&](int d) {
#pragma unroll
        for (int e = 0; e < 4; ++e) g[d % BLOCKS][e] = *reinterpret_cast<const float4u*>(from + 32 * d + 8 * e);
    };
    if (from) {
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d) block(d);
    }
    uint16_t* const to = reinterpret_cast<uint16_t*>(a.y) + static_cast<ptrdiff_t>(t) * a.y_stride + head * HD + 4 * h;
    uint8_t* const to8 = a.q8 + static_cast<ptrdiff_t>(t) * a.q8_stride + head * ND * kQ8_1Bytes;
    const bool out_bf = PAGED ? a.bf16 : BF;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        float v[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = lim < 0 ? 0.0f : o[d][r] * unit;
        if (from) {
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] = gated(v[r], g[d % BLOCKS][r >> 2][r & 3]);
            if (d + BLOCKS < ND) block(d + BLOCKS);
        }
        if (a.y)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<uint2*>(to + 32 * d + 2 * r) = make_uint2(pack16(out_bf, v[r], v[r + 1]), pack16(out_bf, v[r + 2], v[r + 3]));
        if (a.q8) {   // q8_1_store_lane's block and bits: a lane has elements 8 (r / 4) + 4 h + r % 4
            float amax = 0.0f, s[8];
#pragma unroll
            for (int r = 0; r < 16; ++r) amax = fmaxf(amax, fabsf(v[r]));
            amax = fmaxf(amax, xor_lane<32>(amax));
#pragma unroll
            for (int r = 0; r < 8; ++r) s[r] = v[r] + v[r + 8];   // element ^ 16
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[r] += s[r + 4];               // ^ 8
                s[r] += xor_lane<32>(s[r]);     // ^ 4
            }
            const float total = (s[0] + s[2]) + (s[1] + s[3]), dq = amax / 127.0f;
            uint8_t* const blk = to8 + d * kQ8_1Bytes;
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                uint32_t w = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w |= (static_cast<uint32_t>(amax == 0.0f ? 0 : static_cast<int>(roundf(v[r + e] / dq))) & 0xffu) << (8 * e);
                *reinterpret_cast<uint32_t*>(blk + 4 + 2 * r + 4 * h) = w;
            }
            if (h == 0) *reinterpret_cast<uint32_t*>(blk) = float_to_half_sat(dq) | (float_to_half_sat(total) << 16);
        }
    }
}

// ---- few tiles: 32 rows a workgroup, the positions in four parts --------------------------------------------------------------
// Short prompts: tiles of 128 rows would leave compute units empty and each wave alone with a long chain of steps.  Here a workgroup
// has 32 rows, its waves take steps of the positions in turn, each with K and V tiles of its own in LDS (no barriers), and their
// parts are joined at the end.  A wave loads K of its next step when this step's scores are done and V when its product is.
// 500 tokens x 16 heads 24 us, tiles of 128 rows 31.6.
template <bool BF, int HD>
__global__ __launch_bounds__(kThreads, 1) void batch_parts_kernel(BatchArgs a) {
    using S = TileShape<HD>;
    constexpr int STEP = S::kStep, ROW = S::kRow, NK = HD / 16, ND = HD / 32, PER = 1024 / ROW, NL = STEP / PER, PIECES = ROW / 16;
    constexpr int ROWS = kWaveRows;
    __shared__ __attribute__((aligned(16))) uint8_t pool[kWaves * S::kTile];
    __shared__ float stat[kWaves][2][ROWS];
    static_assert(sizeof(pool) >= kWaves * ROWS * HD * sizeof(float), "the parts' rows are joined in the tiles' place");
    static_assert(sizeof(pool) >= kMaxReq * sizeof(int), "the requests' tiles are counted in the tiles' place");

    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
    const int G = a.n_head / a.n_kv, kv = blockIdx.x % a.n_kv;
    int i = 0, level = 0;
    if (!find_tile<ROWS, kThreads>(a, reinterpret_cast<int*>(pool), blockIdx.x / a.n_kv, G, &i, &level)) return;   // uniform
    const Req rq = request(a, i, word(a.row_start, i), word(a.row_start, i + 1));
    const int rows = rq.n * G, row0 = level * ROWS, row = row0 + l32, rowc = min(row, rows - 1), tok = rowc / G, head = kv * G + rowc - tok * G;
    const int first = row0 / G, last = min(row0 + ROWS - 1, rows - 1) / G, lim = row < rows ? tok : -1;
    const int nsteps = (last + STEP) / STEP;   // of all waves

    u32x4 q[NK];
    {
        const uint16_t* qr = reinterpret_cast<const uint16_t*>(a.q) + (static_cast<ptrdiff_t>(rq.start + tok) * a.q_stride + head * HD) + 8 * h;
#pragma unroll
        for (int k = 0; k < NK; ++k) q[k] = *reinterpret_cast<const u32x4*>(qr + 16 * k);
    }
    const size_t kstride = 2 * static_cast<size_t>(a.k_stride), vstride = 2 * static_cast<size_t>(a.v_stride);
    uint8_t* const kt = pool + wv * S::kTile;
    uint8_t* const vt = kt + S::kHalf;
    const uint32_t klds = lds_address(kt), vlds = lds_address(vt);
    const int lr = lane / PIECES;   // as in the tiles above, with all of a step's rows a wave's
    const uint32_t k_piece0 = 16 * (lane % PIECES ^ (lr & 15)), v_piece0 = 16 * (lane % PIECES ^ (v_swizzle(lr) << 1));
    auto load = [&](const uint8_t* src, size_t stride, int sb, uint32_t to, uint32_t piece0, bool k) {
        const int r = min(rq.start + sb, a.ntok - 1), over = r + STEP - a.ntok;
        const uint8_t* from = src + static_cast<size_t>(r) * stride + static_cast<size_t>(kv) * ROW;
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            const uint32_t piece = piece0 ^ (k ? 16 * (n * PER & 15) : 32 * v_swizzle(n * PER));
            if (over <= 0) load_lds(from + n * PER * stride, static_cast<uint32_t>(lr) * static_cast<uint32_t>(stride) + piece, to + 1024 * n);
            else load_lds(from, static_cast<uint32_t>(min(n * PER + lr, STEP - 1 - over)) * static_cast<uint32_t>(stride) + piece, to + 1024 * n);
        }
    };
    auto load_k = [&](int sb) { load(a.k, kstride, sb, klds, k_piece0, true); };
    auto load_v = [&](int sb) { load(a.v, vstride, sb, vlds, v_piece0, false); };
    if (wv < nsteps) {
        load_k(wv * STEP);
        load_v(wv * STEP);
    }
#pragma unroll
    for (int k = 0; k < NK; ++k) asm volatile("" : "+v"(q[k]));   // here before the loop

    floatx16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;
    const int kat = l32 * ROW + ((h ^ (l32 & 15)) << 4), vp = 4 * h + ((lane & 15) >> 2);
    const int vat = vp * ROW + ((((lane >> 4) & 1) ^ v_swizzle(vp)) << 5) + 8 * (lane & 3);
    const bool short_rows = row0 + ROWS > rows;
    auto v_row = [&](int at) { return VRow{a.v + (static_cast<size_t>(rq.start) + at) * vstride + static_cast<size_t>(kv) * ROW, 0, true}; };
    for (int st = wv; st < nsteps; st += kWaves) {   // uniform in the wave
        const int sb = st * STEP;
        const bool more = st + kWaves < nsteps, tail = sb + STEP - 1 > first;
        bool odd = false;
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");   // K; V's loads came after
        tile_step<BF, HD, kKvF16, false, false>(
            kt, vt, kat, vat, q, o, m_run, l_run, a.post, sb, last, lim, h, 0, tail || short_rows, [] {},
            [&] {
                if (more) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K is read
                    load_k(sb + kWaves * STEP);
                    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");   // V; the next K came after
                } else {
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                }
                if (tail) {   // as in the tiles above
                    bool found = false;
#pragma unroll 4
                    for (int n = 0; n < S::kHalf / 1024; ++n) found |= clear_odd<BF>(reinterpret_cast<u32x4*>(vt + 16 * (lane + 64 * n)));
                    odd = __ballot(found) != 0;
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                }
            },
            [&] { return odd; }, v_row);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // V is read
            load_v(sb + kWaves * STEP);
        }
    }

    l_run += xor_lane<32>(l_run);
    if (h == 0) {
        stat[wv][0][l32] = m_run;
        stat[wv][1][l32] = l_run;
    }
    // a thread's pieces of the joined rows: four dims of every UP-th row; their gates on the way
    constexpr int L4 = HD / 4, UP = kThreads / L4, NR = ROWS / UP;
    const int piece = tid % L4, r0 = tid / L4;
    float g[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int rw = min(row0 + r0 + n * UP, rows - 1), t = rw / G;
        load_gate<HD>(a, rq.start + t, kv * G + rw - t * G, 4 * piece, g[n]);
    }
    __syncthreads();   // the tiles are read
    float* const slab = reinterpret_cast<float*>(pool);   // [part][row][HD], a row's pieces of four permuted by exclusive or with the row
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<float4*>(slab + (wv * ROWS + l32) * HD + 4 * ((8 * d + r / 2 + h) ^ l32)) = make_float4(o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int r = r0 + n * UP, rw = row0 + r;
        if (rw >= rows) break;   // the lanes of a block of eight stay together
        float m = stat[0][0][r];
#pragma unroll
        for (int p = 1; p < kWaves; ++p) m = fmaxf(m, stat[p][0][r]);
        const float ref = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < kWaves; ++p) {
            const float f = __builtin_amdgcn_exp2f(stat[p][0][r] - ref);
            const float4 x = *reinterpret_cast<const float4*>(slab + (p * ROWS + r) * HD + 4 * (piece ^ r));
            l = __builtin_fmaf(stat[p][1][r], f, l);
            v[0] = __builtin_fmaf(x.x, f, v[0]);
            v[1] = __builtin_fmaf(x.y, f, v[1]);
            v[2] = __builtin_fmaf(x.z, f, v[2]);
            v[3] = __builtin_fmaf(x.w, f, v[3]);
        }
        const int t = rw / G;
        normed4(v, l, false);
        finish4<HD>(a, rq.start + t, kv * G + rw - t * G, 4 * piece, v, g[n]);
    }
}

// ---- join ------------------------------------------------------------------------------------------------------------------
// the request of a call's row t: the last whose rows begin at or before it (the first if none does), 64 starts at a time
__device__ __forceinline__ int request_of_row(const BatchArgs& a, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.n_req;   // among requests [lo, lo + n)
    while (n > 1) {
        const int step = (n + 63) / 64, at = lo + lane * step;
        const bool in = lane * step < n && a.row_start[min(at, a.n_req - 1)] <= t;
        const int k = max(static_cast<int>(__popcll(__ballot(in))) - 1, 0);   // starts ascend; the count is unsigned, and there may be none
        n = min(step, n - k * step);
        lo += k * step;
    }
    return lo;
}

// A row's chunks; false: the row is not written (no request's, or past the call's bounds)
__device__ __forceinline__ bool row_chunks(const BatchArgs& a, int t, int* chunks, bool* none) {
    const int i = __builtin_amdgcn_readfirstlane(request_of_row(a, t));
    const Req r = request(a, i, word(a.row_start, i), word(a.row_start, i + 1));
    if (t < r.start || t >= r.start + r.n) return false;
    const int p = r.len - r.n + (t - r.start);
    // the form of few rows works on chunks up to the request's last position, tiles on those up to their last token's
    *chunks = p < 0 ? 1 : p / a.chunk + 1;
    *none = p < 0;
    return true;
}

// Few chunks: a wave a row of 256 dims or two of 128, four dims a lane.  Bound by its bytes: 999 tokens, 16 heads of 256 dims, four
// chunks, 95 MB with gates and outputs, 19.8 us (4.8 TB/s).
constexpr int kFlatChunks = 8;

template <int HD>
__global__ __launch_bounds__(kThreads) void batch_join_flat_kernel(BatchArgs a) {
    constexpr int L4 = HD / 4, ROWS = 64 / L4;   // lanes a row, rows a wave
    const int lane = threadIdx.x & 63, wave = blockIdx.x * kWaves + static_cast<int>(threadIdx.x >> 6);
    // a wave's rows are heads of one token (ROWS divides their number or the last wave of a token has fewer)
    const int per = (a.n_head + ROWS - 1) / ROWS, t = __builtin_amdgcn_readfirstlane(wave / per), h = (wave - t * per) * ROWS + lane / L4, d = 4 * (lane % L4);
    if (t >= a.ntok) return;
    int n;
    bool none;
    if (!row_chunks(a, t, &n, &none) || h >= a.n_head) return;
    float g[4];
    load_gate<HD>(a, t, h, d, g);
    const size_t stride = static_cast<size_t>(a.ntok) * a.n_head, r0 = static_cast<size_t>(t) * a.n_head + h;
    float m = -INFINITY, l = 0.0f;
    for (int c = 0; c < n; ++c) m = fmaxf(m, a.wml[2 * (r0 + c * stride)]);
    const float ref = m == -INFINITY ? 0.0f : m;
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < n; ++c) {
        const float2 x = *reinterpret_cast<const float2*>(a.wml + 2 * (r0 + c * stride));
        const float4 v = *reinterpret_cast<const float4*>(a.wo + (r0 + c * stride) * HD + d);
        const float w = __builtin_amdgcn_exp2f(x.x - ref);
        l = __builtin_fmaf(x.y, w, l);
        o[0] = __builtin_fmaf(w, v.x, o[0]);
        o[1] = __builtin_fmaf(w, v.y, o[1]);
        o[2] = __builtin_fmaf(w, v.z, o[2]);
        o[3] = __builtin_fmaf(w, v.w, o[3]);
    }
    normed4(o, l, none);
    finish4<HD>(a, t, h, d, o, g);
}

// Many chunks: workgroup (row, 64 dims); weights to LDS, wave w sums chunks w, w + 4, ... in order, then the waves in order.  One token
// of 16 heads over 64 chunks 4.6 us.
constexpr int kJoinBatch = 16;

template <int HD>
__global__ __launch_bounds__(kThreads) void batch_join_kernel(BatchArgs a) {
    __shared__ float wts[kMaxChunks];
    __shared__ float red[2][kWaves];
    __shared__ float part[kWaves][64];
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, d = 64 * blockIdx.z + lane;
    const size_t stride = static_cast<size_t>(a.ntok) * a.n_head, r0 = static_cast<size_t>(t) * a.n_head + h;
    const float2* ml = reinterpret_cast<const float2*>(a.wml) + r0;
    const float* ro = a.wo + r0 * HD + d;
    // the first records do not wait for the request: every chunk has a place in the workspace (what one past the row's last holds
    // is not used)
    const float2 first = ml[min(tid, a.chunks - 1) * stride];
    float oa[kJoinBatch];   // chunks w + 4 k
#pragma unroll
    for (int k = 0; k < kJoinBatch; ++k) oa[k] = ro[min(w + 4 * k, a.chunks - 1) * stride * HD];
    float gate = 0.0f;
    if (a.gate) gate = a.gate[static_cast<ptrdiff_t>(t) * a.gate_stride + h * 2 * HD + HD + d];
    int n;
    bool none;
    if (!row_chunks(a, t, &n, &none)) return;   // uniform
    float m = tid < n ? first.x : -INFINITY;
    for (int c = tid + kThreads; c < n; c += kThreads) m = fmaxf(m, ml[c * stride].x);
    m = group_max<64>(m);
    if (lane == 0) red[0][w] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    for (int c = tid; c < n; c += kThreads) {
        const float2 x = c == tid ? first : ml[c * stride];
        const float f = __builtin_amdgcn_exp2f(x.x - ref);
        wts[c] = f;
        l = __builtin_fmaf(x.y, f, l);
    }
    l = group_sum<64>(l);
    if (lane == 0) red[1][w] = l;
    __syncthreads();
    l = ((red[1][0] + red[1][1]) + red[1][2]) + red[1][3];
    float o = 0.0f;
    for (int c0 = 0; 4 * c0 < n; c0 += kJoinBatch) {
        const bool more = 4 * (c0 + kJoinBatch) < n;
        float nx[kJoinBatch];
        if (more) {
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) nx[k] = ro[min(w + 4 * (c0 + kJoinBatch + k), n - 1) * stride * HD];
        }
#pragma unroll
        for (int k = 0; k < kJoinBatch; ++k) {
            const int c = w + 4 * (c0 + k);
            if (c < n) o = __builtin_fmaf(wts[c], oa[k], o);
        }
        if (more) {
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) oa[k] = nx[k];
        }
    }
    part[w][lane] = o;
    __syncthreads();
    if (w != 0) return;
    float v = ((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane];
    v = none ? 0.0f : v / l;
    if (a.gate) v = gated(v, gate);
    if (a.y) reinterpret_cast<uint16_t*>(a.y)[static_cast<ptrdiff_t>(t) * a.y_stride + h * HD + d] = static_cast<uint16_t>(pack16(a.bf16, v, 0.0f));
    if (a.q8) q8_1_store_lane(v, a.q8 + static_cast<ptrdiff_t>(t) * a.q8_stride + (h * (HD / 32) + d / 32) * kQ8_1Bytes);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
bool heads_ok(int n_head, int n_kv, int head_dim) {
    return n_kv > 0 && n_head > 0 && n_head <= 65535 && n_head % n_kv == 0 && n_head / n_kv <= 64 && (head_dim == 128 || head_dim == 256);
}
bool batch_ok(int n_req, int ntok, int max_new) { return n_req >= 1 && n_req <= kMaxReq && ntok >= 1 && max_new >= 1 && ntok <= 1 << 24; }
int chunks_of(int max_ctx, int split) { return static_cast<int>((static_cast<long long>(max_ctx) + split - 1) / split); }
bool split_ok(int max_ctx, int split) { return split >= kChunkUnit && split % kChunkUnit == 0 && chunks_of(max_ctx, split) <= kMaxChunks; }

// tiles of `held` rows: the most that a request of max_new tokens has, and that n_req requests of ntok tokens in all have
int most_levels(int ntok, int max_new, int G, int held) {
    return static_cast<int>((static_cast<long long>(std::min(max_new, ntok)) * G + held - 1) / held);
}
long long most_tiles(int n_req, int ntok, int max_new, int G, int held) {
    return std::min(static_cast<long long>(ntok) * G / held + n_req, static_cast<long long>(most_levels(ntok, max_new, G, held)) * n_req);
}

// The rows of a request that the form of few rows takes in a call: 32, two blocks of 16, where no request has more and the cache is
// quantised (a code is turned once for both blocks), else 16.  16 requests of 5 tokens behind 4096 positions (16 heads, 4 KV heads of
// 256 dims) I8 33 us with two blocks and 68 in tiles, I4 32 and 66; 200 of 5 behind 500 I8 74 and 117; F16 in tiles 50, with two
// blocks 54.  Beside longer requests two blocks would cost single tokens a workgroup: their records leave one to a compute unit.
int few_rows(bool quantised, int ntok, int max_new, int G) {
    const long long most = static_cast<long long>(std::min(max_new, ntok)) * G;
    return quantised && most > kFewRows && most <= 2 * kFewRows ? 2 * kFewRows : kFewRows;
}

struct Outputs {
    const float* gate;
    int gate_stride;
    void* y;
    int y_stride;
    uint8_t* q8;
    int q8_stride;
};

int check_outputs(const char* what, const Outputs& o, int ntok, int n_head, int head_dim) {
    const int width = n_head * head_dim;
    if ((o.gate && !aligned4(o.gate)) || (!o.y && !o.q8) || (o.y && ((reinterpret_cast<uintptr_t>(o.y) & 7u) || o.y_stride % 4)) ||
        (o.q8 && (!aligned4(o.q8) || o.q8_stride % 4)))
        return fail(RMI_ERR_POINTER, what);
    if (ntok > 1 && ((o.y && o.y_stride < width) || (o.q8 && o.q8_stride < width / 32 * kQ8_1Bytes))) return fail(RMI_ERR_SHAPE, what);
    return RMI_OK;
}

// whether an output or the workspace shares bytes with what the call reads (in) or with another of them
bool outputs_overlap(const Outputs& o, int ntok, int n_head, int head_dim, const void* ws, size_t ws_bytes, const RowSet* in, int n_in) {
    const int width = n_head * head_dim;
    const RowSet out[] = {block_of(ws, ws ? ws_bytes : 0), {o.q8, o.q8 ? ntok : 0, o.q8_stride, width / 32 * kQ8_1Bytes}, {o.y, o.y ? ntok : 0, 2LL * o.y_stride, 2LL * width}};
    for (int k = 0; k < 3; ++k) {
        if (!out[k].n || !out[k].bytes) continue;
        for (int i = 0; i < n_in; ++i)
            if (in[i].n && in[i].bytes && rows_overlap(out[k], in[i])) return true;
        for (int j = 0; j < k; ++j)
            if (out[j].n && out[j].bytes && rows_overlap(out[k], out[j])) return true;
        // a token's gates from the first to the last, then head by head: a row may fit between two
        if (o.gate && rows_overlap(out[k], {o.gate + head_dim, ntok, 4LL * o.gate_stride, 4LL * (2 * width - head_dim)}))
            for (int h = 0; h < n_head; ++h)
                if (rows_overlap(out[k], {o.gate + static_cast<size_t>(2 * h + 1) * head_dim, ntok, 4LL * o.gate_stride, 4LL * head_dim})) return true;
    }
    return false;
}

void set_outputs(BatchArgs* a, const Outputs& o) {
    a->gate = o.gate;
    a->gate_stride = o.gate_stride;
    a->y = static_cast<uint8_t*>(o.y);
    a->y_stride = o.y_stride;
    a->q8 = o.q8;
    a->q8_stride = o.q8_stride;
}

constexpr int kMaxStride = 1 << 25;   // the 64 rows of a step are within 32 bits of its first, in bytes

constexpr long long kMostBlocks = 0xffffffffLL / kThreads;

// waves of a paged tile's workgroup
constexpr int tile_waves(int ktype) { return ktype == kKvF16 ? 4 : 8; }

template <int KT, int VT, int HD>
void launch_paged(const BatchArgs& a, bool tiles, long long few_blocks, long long tile_blocks, hipStream_t s) {
    constexpr int W = tile_waves(KT);
    if (tiles) hipLaunchKernelGGL((batch_tile_kernel<kPaged, KT, VT, HD, W>), dim3(static_cast<unsigned>(tile_blocks)), dim3(64 * W), 0, s, a);
    auto* few = &batch_few_kernel<KT, VT, HD, 1>;
    if constexpr (KT != kKvF16)
        if (a.few > kFewRows) few = &batch_few_kernel<KT, VT, HD, 2>;
    hipLaunchKernelGGL(few, dim3(static_cast<unsigned>(few_blocks)), dim3(kThreads), 0, s, a);
    if (a.chunks > kFlatChunks) {
        hipLaunchKernelGGL((batch_join_kernel<HD>), dim3(a.ntok, a.n_head, HD / 64), dim3(kThreads), 0, s, a);
    } else if (a.chunks > 1) {
        const int rows = 256 / HD, per = (a.n_head + rows - 1) / rows;
        hipLaunchKernelGGL((batch_join_flat_kernel<HD>), dim3(static_cast<unsigned>((static_cast<long long>(a.ntok) * per + kWaves - 1) / kWaves)), dim3(kThreads), 0, s, a);
    }
}

template <int HD>
void launch_paged(const BatchArgs& a, int ktype, int vtype, bool tiles, long long few_blocks, long long tile_blocks, hipStream_t s) {
    if (ktype == kKvF16) launch_paged<kKvF16, kKvF16, HD>(a, tiles, few_blocks, tile_blocks, s);
    else if (ktype == kKvI4) launch_paged<kKvI4, kKvI4, HD>(a, tiles, few_blocks, tile_blocks, s);
    else if (vtype == kKvI8) launch_paged<kKvI8, kKvI8, HD>(a, tiles, few_blocks, tile_blocks, s);
    else launch_paged<kKvI8, kKvI4, HD>(a, tiles, few_blocks, tile_blocks, s);
}

// The chunk of a call with more rows, from what its parts cost (us; 256 dims, 32 positions a step): a workgroup's beginning and end
// 4.5, a step 1.3 alone on its compute unit and 2.2 beside another, so that a round of up to 256 workgroups takes 4.5 + 1.3 steps and
// one of up to 512 4.5 + 2.2 steps; the join 5 and its records at 4 TB/s.  Measured against the chunks around it, F16: 999 tokens
// behind 8001 positions 2048 (182 / 159 / 184 us at 1024 / 2048 / 4096), behind 65501 16384 (1530 at 15872, five chunks and two
// rounds, 1050 at 16384), 300 behind 2000 512 (41 / 40 / 55 at 256 / 512 / 1024), 16 requests of 5 behind 4096 512 (62 / 50 / 55),
// 8 of 200 behind 1000 one chunk (62 / 54 at 512 / 1024).
long long tile_chunk(long long total_ctx, int max_ctx, int n_req, int ntok, int max_new, int G, int n_head, int n_kv, int head_dim) {
    const int new_each = std::min(max_new, ntok);
    // as if all tokens were in requests of the longest kind
    const double tiles = std::max(1.0, std::floor(static_cast<double>(ntok) / new_each + 0.5)) * most_levels(ntok, new_each, G, kTileRows) * n_kv;
    // contexts: the requests' average, or the longest where most tokens are one request's
    const bool one = n_req == 1 || ntok < 2LL * new_each;
    const double len = one ? max_ctx : std::min(static_cast<double>(max_ctx), static_cast<double>(total_ctx) / n_req), step = 32.0 * 256 / head_dim;
    double best = 0.0;
    long long chunk = 0;
    for (int k = 1, before = 0; k <= 512; ++k) {
        const int c = static_cast<int>((static_cast<long long>(max_ctx) + static_cast<long long>(k) * kChunkUnit - 1) / (static_cast<long long>(k) * kChunkUnit)) * kChunkUnit;
        if (c == before) continue;
        before = c;
        const int chunks = chunks_of(max_ctx, c);
        const double groups = tiles * (one ? chunks : std::min<double>(chunks, len / c + (chunks > 1 ? 0.5 : 0.0))), steps = std::ceil(std::min<double>(c, max_ctx) / step);
        const double round = 4.5 + (groups <= 256 ? 1.3 : 2.2) * steps, rounds = std::max(1.0, std::ceil(groups * (one ? 1.0 : 1.06) / 512));   // ragged: some more than the average says
        const double cost = round * rounds + (chunks > 1 ? 5.0 + static_cast<double>(chunks) * ntok * n_head * head_dim * 4 / 4e6 : 0.0);
        if (chunk == 0 || cost < best) best = cost, chunk = c;
    }
    return chunk;
}

}  // namespace
}  // namespace rmi

using namespace rmi;

extern "C" int rmi_gqa_paged_split(long long total_ctx, int max_ctx, int n_req, int ntok, int max_new, int n_head, int n_kv, int head_dim) {
    if (!heads_ok(n_head, n_kv, head_dim) || !batch_ok(n_req, ntok, max_new) || max_ctx < 1 || max_ctx > kKvMaxCtx || total_ctx < 1) {
        set_error("gqa_paged_split: invalid shape");
        return 0;
    }
    const int G = n_head / n_kv;
    long long chunk;
    if (static_cast<long long>(std::min(max_new, ntok)) * G <= few_rows(true, ntok, max_new, G)) {   // F16's tiles of 17 to 32 rows take these chunks within 10 % of their best
        // Few rows: one round of workgroups, one for each of 256 compute units, since past the memory's rate it is their beginnings,
        // ends and records that cost.  A request of any length has half a chunk too many on average; eight workgroups are left for
        // more.  More rounds where one would leave a chunk much longer than its share.
        const long long total = std::min<long long>(total_ctx, static_cast<long long>(max_ctx) * n_req);
        long long rounds = 1, slots;
        do {
            slots = 512 * rounds - static_cast<long long>(n_req - 1) * n_kv - (n_req > 1 ? 16 : 0);   // halves
            chunk = slots > 0 ? (2 * total * n_kv + slots - 1) / slots : max_ctx;
        } while (++rounds <= 8 && 256 * chunk > 2 * total * n_kv);
    } else {
        chunk = tile_chunk(total_ctx, max_ctx, n_req, ntok, max_new, G, n_head, n_kv, head_dim);
    }
    chunk = std::max<long long>(chunk, (static_cast<long long>(max_ctx) + kMaxChunks - 1) / kMaxChunks);
    chunk = std::min<long long>(std::max(chunk, 1LL), max_ctx);
    return static_cast<int>((chunk + kChunkUnit - 1) / kChunkUnit * kChunkUnit);
}

extern "C" size_t rmi_gqa_paged_workspace_bytes(int ntok, int max_ctx, int n_head, int head_dim, int split) {
    if (ntok < 1 || ntok > 1 << 24 || max_ctx < 1 || max_ctx > kKvMaxCtx || n_head < 1 || n_head > 65535 || (head_dim != 128 && head_dim != 256) ||
        !split_ok(max_ctx, split)) {
        set_error("gqa_paged_workspace_bytes: invalid shape, or a split that is no multiple of 128 or leaves more than 1024 chunks");
        return 0;
    }
    const int chunks = chunks_of(max_ctx, split);
    return chunks == 1 ? 16 : static_cast<size_t>(chunks) * ntok * n_head * (head_dim + 2) * sizeof(float);
}

extern "C" int rmi_gqa_paged_attn(int qtype, const void* q, int ktype, const void* kpool, int vtype, const void* vpool, const int* table,
                                  int table_stride, const int* row_start, const int* kv_len, const float* gate_src, int gate_stride, void* y,
                                  int y_stride, uint8_t* q8, int q8_stride, void* workspace, int n_req, int ntok, int max_new, int max_ctx,
                                  int n_head, int n_kv, int head_dim, int page_size, int n_pages, int split, float scale, void* stream) {
    if (!kv_type_ok(ktype) || !kv_type_ok(vtype) || (ktype != vtype && !(ktype == kKvI8 && vtype == kKvI4)))
        return fail(RMI_ERR_UNSUPPORTED, "gqa_paged_attn: cache types F16 / F16, I8 / I8, I4 / I4 or I8 / I4");
    if (qtype != RMI_ROWS_F16 && qtype != RMI_ROWS_BF16) return fail(RMI_ERR_UNSUPPORTED, "gqa_paged_attn: rows of F16 or BF16");
    if (!heads_ok(n_head, n_kv, head_dim) || !batch_ok(n_req, ntok, max_new) || !pool_ok(page_size, n_pages) || table_stride < 1 ||
        static_cast<long long>(n_req) * table_stride > 0x7fffffffLL || max_ctx < 1 || max_ctx > kKvMaxCtx || !(scale > 0.0f && scale <= FLT_MAX))
        return fail(RMI_ERR_SHAPE, "gqa_paged_attn: invalid arguments");
    if (!split_ok(max_ctx, split)) return fail(RMI_ERR_SHAPE, "gqa_paged_attn: a split is a multiple of 128 that leaves at most 1024 chunks of max_ctx");
    const size_t ws_bytes = rmi_gqa_paged_workspace_bytes(ntok, max_ctx, n_head, head_dim, split);
    const int chunks = chunks_of(max_ctx, split);
    if (!aligned16(q) || !aligned16(kpool) || !aligned16(vpool) || !aligned4(table) || !aligned4(row_start) || !aligned4(kv_len) ||
        (chunks > 1 && !aligned16(workspace)))
        return fail(RMI_ERR_POINTER, "gqa_paged_attn: null or misaligned pointer");
    const Outputs out{gate_src, gate_stride, y, y_stride, q8, q8_stride};
    RMI_TRY(check_outputs("gqa_paged_attn: no output, or misaligned or overlapping output rows", out, ntok, n_head, head_dim));
    const RowSet in[] = {block_of(q, static_cast<size_t>(ntok) * n_head * head_dim * 2), block_of(kpool, n_pages * kv_page_bytes(ktype, page_size, n_kv, head_dim)),
                         block_of(vpool, n_pages * kv_page_bytes(vtype, page_size, n_kv, head_dim)),
                         block_of(table, static_cast<size_t>(n_req) * table_stride * 4), block_of(row_start, (n_req + 1) * 4ul), block_of(kv_len, n_req * 4ul)};
    if (outputs_overlap(out, ntok, n_head, head_dim, chunks > 1 ? workspace : nullptr, ws_bytes, in, 6))
        return fail(RMI_ERR_POINTER, "gqa_paged_attn: an output or the workspace lies on another argument");
    BatchArgs a{};
    const int G = n_head / n_kv;
    a.q = static_cast<const uint8_t*>(q);
    a.k = static_cast<const uint8_t*>(kpool);
    a.v = static_cast<const uint8_t*>(vpool);
    a.table = table;
    a.row_start = row_start;
    a.kv_len = kv_len;
    set_outputs(&a, out);
    a.q_stride = n_head * head_dim;
    a.table_stride = table_stride;
    a.n_req = n_req;
    a.ntok = ntok;
    a.max_new = max_new;
    a.max_ctx = max_ctx;
    a.n_head = n_head;
    a.n_kv = n_kv;
    a.shift = page_shift_of(page_size);
    a.n_pages = n_pages;
    a.chunk = std::min(split, (max_ctx + kChunkUnit - 1) / kChunkUnit * kChunkUnit);   // a length and a chunk fit an int
    a.chunks = chunks;
    a.wo = static_cast<float*>(workspace);
    a.wml = a.wo + static_cast<size_t>(chunks) * ntok * n_head * head_dim;
    const int held = kWaveRows * tile_waves(ktype);
    a.bf16 = qtype == RMI_ROWS_BF16;
    a.post = scale * kLog2e;
    a.few = few_rows(ktype != kKvF16, ntok, max_new, G);
    const bool tiles = static_cast<long long>(std::min(max_new, ntok)) * G > a.few;
    const long long few = static_cast<long long>(n_req) * n_kv * chunks, tile = most_tiles(n_req, ntok, max_new, G, held) * n_kv * chunks;
    if (few > kMostBlocks || (tiles && tile > kMostBlocks / 2) || static_cast<long long>(ntok) * n_head > kMostBlocks)
        return fail(RMI_ERR_SHAPE, "gqa_paged_attn: too many workgroups");
    auto* s = static_cast<hipStream_t>(stream);
    if (head_dim == 256) launch_paged<256>(a, ktype, vtype, tiles, few, tile, s);
    else launch_paged<128>(a, ktype, vtype, tiles, few, tile, s);
    return launch_status("gqa_paged_attn");
}

extern "C" int rmi_gqa_prompt_attn(int type, const void* q, int q_stride, const void* k, int k_stride, const void* v, int v_stride,
                                   const int* row_start, const float* gate_src, int gate_stride, void* y, int y_stride, uint8_t* q8,
                                   int q8_stride, int n_req, int ntok, int max_len, int n_head, int n_kv, int head_dim, float scale,
                                   void* stream) {
    if (type != RMI_ROWS_F16 && type != RMI_ROWS_BF16) return fail(RMI_ERR_UNSUPPORTED, "gqa_prompt_attn: rows of F16 or BF16");
    if (!heads_ok(n_head, n_kv, head_dim) || !batch_ok(n_req, ntok, max_len) || !(scale > 0.0f && scale <= FLT_MAX) || q_stride % 8 || k_stride % 8 ||
        v_stride % 8 || k_stride > kMaxStride || v_stride > kMaxStride || (ntok > 1 && (q_stride < n_head * head_dim || k_stride < n_kv * head_dim || v_stride < n_kv * head_dim)))
        return fail(RMI_ERR_SHAPE, "gqa_prompt_attn: invalid arguments (strides are multiples of 8 elements, k's and v's up to 2^25)");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned4(row_start))
        return fail(RMI_ERR_POINTER, "gqa_prompt_attn: null or misaligned pointer");
    const Outputs out{gate_src, gate_stride, y, y_stride, q8, q8_stride};
    RMI_TRY(check_outputs("gqa_prompt_attn: no output, or misaligned or overlapping output rows", out, ntok, n_head, head_dim));
    const RowSet in[] = {{q, ntok, 2LL * q_stride, 2LL * n_head * head_dim}, {k, ntok, 2LL * k_stride, 2LL * n_kv * head_dim},
                         {v, ntok, 2LL * v_stride, 2LL * n_kv * head_dim}, block_of(row_start, (n_req + 1) * 4ul)};
    if (outputs_overlap(out, ntok, n_head, head_dim, nullptr, 0, in, 4))
        return fail(RMI_ERR_POINTER, "gqa_prompt_attn: an output lies on another argument");
    BatchArgs a{};
    const int G = n_head / n_kv;
    a.q = static_cast<const uint8_t*>(q);
    a.k = static_cast<const uint8_t*>(k);
    a.v = static_cast<const uint8_t*>(v);
    a.row_start = row_start;
    set_outputs(&a, out);
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.n_req = n_req;
    a.ntok = ntok;
    a.max_new = max_len;
    a.max_ctx = ntok;
    a.n_head = n_head;
    a.n_kv = n_kv;
    a.chunk = (ntok + kChunkUnit - 1) / kChunkUnit * kChunkUnit;
    a.chunks = 1;
    a.bf16 = type == RMI_ROWS_BF16;
    a.post = scale * kLog2e;
    // Three forms.  Eight waves over 256 rows, which share a tile's K and V, for long prompts from about two rounds of workgroups on:
    // one prompt of 8001 tokens (504 tiles, 16 heads, 4 KV heads of 256 dims) 505 us with 128 rows, 485 with 256; of 4000 (252) 190 /
    // 196; 40 of 200 (664, up to 13 levels) 103 / 110.  32 rows with the positions in four parts where prompts are long enough for
    // steps to part and tiles few: one prompt of 128 / 500 / 750 tokens (64 / 252 / 376 tiles of 32) 14.0 / 24.1 / 36 us, tiles of 128
    // rows 17.5 / 31.6 / 41; but 20 prompts of 25 tokens on average (260 tiles, 3 levels) 26.5 / 16.6 and ten of 100 (540 tiles) 40 /
    // 23.5.  128 rows else.
    const int most_rows = 8 * kWaveRows;
    const bool wide = most_levels(ntok, max_len, G, most_rows) >= 64 && most_tiles(n_req, ntok, max_len, G, most_rows) * n_kv >= 480;
    const bool parts = !wide && most_levels(ntok, max_len, G, 4 * kWaveRows) >= 4 && most_tiles(n_req, ntok, max_len, G, kWaveRows) * n_kv <= 400;
    const int held = parts ? kWaveRows : (wide ? 8 : 4) * kWaveRows;
    a.levels = most_levels(ntok, max_len, G, held);
    const long long blocks = most_tiles(n_req, ntok, max_len, G, held) * n_kv;
    if (blocks > kMostBlocks / (wide ? 2 : 1)) return fail(RMI_ERR_SHAPE, "gqa_prompt_attn: too many workgroups");
    auto go = [&](auto* kernel, int waves) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * waves), 0, static_cast<hipStream_t>(stream), a);
        return launch_status("gqa_prompt_attn");
    };
    auto with = [&](auto bf, auto hd) {
        constexpr int HD = decltype(hd)::value;
        constexpr bool BF = decltype(bf)::value;
        constexpr int SRC = BF ? kRowsBF16 : kRowsF16;
        if (parts) return go(&batch_parts_kernel<BF, HD>, kWaves);
        if (wide) return go(&batch_tile_kernel<SRC, kKvF16, kKvF16, HD, 8>, 8);
        return go(&batch_tile_kernel<SRC, kKvF16, kKvF16, HD, 4>, 4);
    };
    auto of_type = [&](auto bf) { return head_dim == 256 ? with(bf, std::integral_constant<int, 256>{}) : with(bf, std::integral_constant<int, 128>{}); };
    return a.bf16 ? of_type(std::true_type{}) : of_type(std::false_type{});
}
