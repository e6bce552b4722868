// kv_pages.hip - caches in pages for several requests at once (layout: kv_pages.h), for gfx950:
//   page_plan        row starts, lengths, slots and positions of a batch's new tokens and the pages they need, from the lengths
//   page_trim        the pages past the lengths that requests keep, back to the free list
//   kv_page_read     rows of slots -> fp32 / fp16 rows
//   attn_prep_paged  per-head RMSNorm, rotary embedding, q in 16 bits, K / V to their slots
// No counterpart in the reference, whose engine serves one request from one contiguous fp16 cache (qw:340-345, 1532-1548).
#include "kv_pages.h"

#include <algorithm>
#include <cmath>

#include "kv_rows.h"
#include "overlap.h"
#include "rope.h"
#include "turns.h"

namespace rmi {
namespace {

// ---- plan and trim -----------------------------------------------------------------------------------------------------
// Both are two prefix sums over the requests and a copy.  Every workgroup takes the sums of all requests for itself (16 KB of
// lengths at most, from the L2), so one launch does and no workgroup waits for another; tokens and pages are then dealt out over
// all of them, each finding its request by bisection of the sums in LDS.  Latency-bound: loads, two sums with their barriers, a bisection, a
// load; a plan of 32 requests of one token 4.4 us, of 999 with 121 K tokens 9.3 us; a trim 2.5 and 4.4.
constexpr int kPlanThreads = 256;
constexpr uint32_t kSat = 1u << 30;   // sums stop here: min(a + b, kSat) is associative, and lengths may be anything
constexpr uint32_t kRefused = 1u << 31;

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kSat); }
__device__ __forceinline__ int pages_of(int n, int shift) { return static_cast<int>((static_cast<uint32_t>(n) + (1u << shift) - 1) >> shift); }

// a[0 .. n) becomes its exclusive prefix sums (saturated), a[n] the whole; sums: a word a wave
__device__ __forceinline__ void scan_requests(uint32_t* a, int n, uint32_t* sums) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int per = (n + kPlanThreads - 1) / kPlanThreads, first = tid * per, end = min(first + per, n);
    uint32_t mine = 0;
    for (int i = first; i < end; ++i) mine = sat_add(mine, a[i]);
    const uint32_t upto = wave_scan(mine, sat_add);
    if (lane == 63) sums[wv] = upto;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64 - 1; ++w) before = sat_add(before, w < wv ? sums[w] : 0);
    const uint32_t prev = __shfl_up(upto, 1, 64);
    if (lane > 0) before = sat_add(before, prev);
    for (int i = first; i < end; ++i) {
        const uint32_t v = a[i];
        a[i] = before;
        before = sat_add(before, v);
    }
    if (first < n && end == n) a[n] = before;
    __syncthreads();
}

// the last i < n with a[i] (without its flag) <= x
__device__ __forceinline__ int request_of(const uint32_t* a, int n, uint32_t x) {
    int lo = 0, hi = n;   // a[lo] <= x < a[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((a[mid] & ~kRefused) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct PlanArgs {
    const int *past, *count, *free_pages, *n_free;
    int *table, *row_start, *kv_len, *slot, *pos, *n_left, *status;
    int n_req, shift, n_pages, table_stride, max_tok;
};

__global__ __launch_bounds__(kPlanThreads) void page_plan_kernel(PlanArgs a) {
    __shared__ uint32_t rows[kMaxReq + 1], offs[kMaxReq + 1];   // row starts; pages taken before, with kRefused
    __shared__ int pasts[kMaxReq];
    __shared__ uint32_t sums[kPlanThreads / 64], taken;
    constexpr int E = kMaxReq / kPlanThreads;   // requests a thread has, 256 apart
    const int tid = threadIdx.x, n = a.n_req;
    int past[E], count[E];   // in flight together
#pragma unroll
    for (int k = 0; k < E; ++k)
        if (k * kPlanThreads < n) {   // uniform
            const int i = min(k * kPlanThreads + tid, n - 1);
            past[k] = a.past[i];
            count[k] = a.count[i];
        }
    const int n_free = min(max(a.n_free[0], 0), a.n_pages);
    const long long room = min(static_cast<long long>(a.table_stride) << a.shift, static_cast<long long>(kSat));
    const uint32_t max_tok = static_cast<uint32_t>(a.max_tok);
    // f(request, its past and count) for each of the thread's
    auto each = [&](auto f) {
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (k * kPlanThreads + tid < n) f(k * kPlanThreads + tid, past[k], count[k]);
    };
    auto fits = [&](int i, int p, int c) { return p >= 0 && c >= 0 && static_cast<long long>(p) + c <= room && rows[i] + static_cast<uint32_t>(c) <= max_tok; };
    auto need = [&](int p, int c) { return static_cast<uint32_t>(pages_of(p + c, a.shift) - pages_of(p, a.shift)); };
    if (tid == 0) taken = 0;
    each([&](int i, int p, int c) {
        rows[i] = static_cast<uint32_t>(min(max(c, 0), static_cast<int>(kSat)));
        pasts[i] = p;
    });
    __syncthreads();
    scan_requests(rows, n, sums);
    each([&](int i, int p, int c) { offs[i] = fits(i, p, c) ? need(p, c) : 0; });
    __syncthreads();
    scan_requests(offs, n, sums);
    const uint32_t wanted = offs[n];
    each([&](int i, int p, int c) {
        const bool good = fits(i, p, c);
        const uint32_t before = offs[i], pages = good ? need(p, c) : 0;
        const bool ok = good && (pages == 0 || before + pages <= static_cast<uint32_t>(n_free));
        if (!ok) offs[i] = before | kRefused;   // only this thread reads it before the barrier
        else if (pages) atomicMax(&taken, before + pages);
        if (blockIdx.x == 0) {
            a.row_start[i] = static_cast<int>(min(rows[i], max_tok));
            a.kv_len[i] = ok ? p + c : 0;
            a.status[i] = ok ? RMI_PAGES_OK : good ? RMI_PAGES_NONE_LEFT : RMI_PAGES_BAD_LENGTH;
        }
    });
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        a.row_start[n] = static_cast<int>(min(rows[n], max_tok));
        a.n_left[0] = n_free - static_cast<int>(taken);   // those admitted come first among those that need pages
    }
    const uint32_t used = min(rows[n], max_tok), step = gridDim.x * kPlanThreads;
    for (uint32_t t = blockIdx.x * kPlanThreads + tid; t < max_tok; t += step) {
        int slot = -1, p = 0;
        if (t < used) {
            const int i = request_of(rows, n, t);
            const uint32_t off = offs[i];
            p = static_cast<int>(static_cast<uint32_t>(pasts[i]) + (t - rows[i]));   // anything if the lengths are bad
            if (!(off & kRefused)) {
                const int held = pages_of(pasts[i], a.shift), at = p >> a.shift;
                const int page = at < held ? a.table[static_cast<size_t>(i) * a.table_stride + at]
                                           : a.free_pages[n_free - 1 - static_cast<int>(off) - (at - held)];
                if (page >= 0 && page < a.n_pages) slot = (page << a.shift) | (p & ((1 << a.shift) - 1));
            }
        }
        a.slot[t] = slot;
        a.pos[t] = p;
    }
    const uint32_t pages = min(wanted, static_cast<uint32_t>(n_free));
    for (uint32_t k = blockIdx.x * kPlanThreads + tid; k < pages; k += step) {
        const int i = request_of(offs, n, k);
        const uint32_t off = offs[i];
        if (!(off & kRefused))
            a.table[static_cast<size_t>(i) * a.table_stride + pages_of(pasts[i], a.shift) + (k - off)] = a.free_pages[n_free - 1 - static_cast<int>(k)];
    }
}

struct TrimArgs {
    const int *len, *keep, *table, *n_free;
    int *free_pages, *n_out;
    int n_req, shift, n_pages, table_stride;
};

__global__ __launch_bounds__(kPlanThreads) void page_trim_kernel(TrimArgs a) {
    __shared__ uint32_t offs[kMaxReq + 1];
    __shared__ uint32_t sums[kPlanThreads / 64];
    const int tid = threadIdx.x, n = a.n_req;
    const int n_free = min(max(a.n_free[0], 0), a.n_pages);
#pragma unroll 4
    for (int i = tid; i < n; i += kPlanThreads) {
        const int len = a.len[i], keep = a.keep[i];
        const int end = min(pages_of(len, a.shift), a.table_stride), first = pages_of(keep, a.shift);
        offs[i] = keep >= 0 && keep <= len && first < end ? static_cast<uint32_t>(end - first) : 0;
    }
    __syncthreads();
    scan_requests(offs, n, sums);
    const uint32_t back = min(offs[n], static_cast<uint32_t>(a.n_pages - n_free));
    if (blockIdx.x == 0 && tid == 0) a.n_out[0] = n_free + static_cast<int>(back);
    for (uint32_t k = blockIdx.x * kPlanThreads + tid; k < back; k += gridDim.x * kPlanThreads) {
        const int i = request_of(offs, n, k);
        a.free_pages[n_free + k] = a.table[static_cast<size_t>(i) * a.table_stride + pages_of(a.keep[i], a.shift) + (k - offs[i])];
    }
}

// ---- rows of slots -------------------------------------------------------------------------------------------------------
// kv_read's unit (eight dims a lane), each row at its own slot: 1999 rows of 4 x 256 dims F16 4.3 us, of which 2 are the beginning and
// end of a launch (16.4 MB with the outputs)
constexpr int kReadThreads = 256;

template <int T, bool OUT16, bool VEC>
__global__ __launch_bounds__(kReadThreads) void kv_page_read_kernel(const uint8_t* __restrict__ pool, const int* __restrict__ slots,
                                                                    void* __restrict__ out, int out_stride, int n, int n_kv, int head_dim,
                                                                    int shift, int n_pages) {
    const int s = head_dim == 256 ? 5 : 4;
    const int rows = blockIdx.x / n_kv, kv = blockIdx.x - rows * n_kv;
    const int g = static_cast<int>(threadIdx.x) & ((1 << s) - 1);
    const int row = rows * (kReadThreads >> s) + (static_cast<int>(threadIdx.x) >> s);
    if (row >= n) return;
    const int slot = slots[row], page = slot >> shift, size = 1 << shift;
    F8 x = {};
    if (slot >= 0 && page < n_pages) {
        const uint8_t* at = pool + static_cast<size_t>(page) * kv_page_bytes(T, size, n_kv, head_dim);
        x = read_unit<T>(at, kv_row<T>(slot & (size - 1), kv, n_kv, size, head_dim), g);
    }
    store8<OUT16, VEC>(out, static_cast<size_t>(row) * out_stride + kv * head_dim + 8 * g, x);
}

// ---- norm, rotation, rows to their slots ---------------------------------------------------------------------------------
// Workgroup (token, part): the token's (cos, sin) per pair once into LDS, then a wave per head row, a lane HD / 64 neighbouring
// dims; a row's loads go out before the work on the row before it.  The frequencies are the host's (2 pi left out, YaRN's ramp in
// them), so that an angle is one fp64 product, its fraction, and two polynomials; pow and sincos on the device were half of
// attn_prep_axes' time.  q is normed and rotated in fp32 and rounded to 16 bits; K in fp64, rounded to fp32 once, so that what a
// cache holds does not hang on the order of a sum (a code at a border would).  Bound by the rows: 1999 tokens of 16 + 4 heads of 256
// dims, 74 MB, 17.8 us (4.2 TB/s); 32 tokens, a wave a row, 4.6 us of waits: slot, row, weights, then the angles' barrier.
constexpr int kPrepWaves = 4;
constexpr int kMaxPairs = 128;

struct PagedPrepArgs {
    const float* q3;
    const float *qn, *kn;
    uint8_t *kp, *vp;
    const int *slot, *pos;
    uint16_t* qout;
    int q3_stride, n_head, n_kv, n_rot, shift, n_pages, per_wave, neighbours, bf16;
    float eps;
    double size;              // of cos and sin
    double turns[kMaxPairs];  // of pair i in one position
};

__device__ __forceinline__ uint32_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }

template <int KT, int VT, int HD>
__global__ __launch_bounds__(64 * kPrepWaves) void prep_paged_kernel(PagedPrepArgs a) {
    constexpr int N = HD / 64;
    __shared__ double cs[HD / 2][2];
    __shared__ float2 csf[HD / 2];   // rounded, for q
    __shared__ __attribute__((aligned(16))) double rows[kPrepWaves][HD];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), d0 = N * lane;
    const int half = a.n_rot / 2;
    const float* src = a.q3 + static_cast<ptrdiff_t>(t) * a.q3_stride;
    const int items = a.n_head + 2 * a.n_kv, first = (blockIdx.y * kPrepWaves + wv) * a.per_wave;
    const int end = min(first + a.per_wave, items);
    float nx[N], wq[N], wk[N];   // nx: the next row
    auto load = [&](int it) {
        it = min(it, items - 1);
        load_dims(nx, (it < a.n_head ? src + it * 2 * HD : src + 2 * a.n_head * HD + (it - a.n_head) * HD) + d0);   // [q | gate] .., k, v
    };
    const int slot = a.slot[t], p = a.pos[t];
    load(first);
    load_dims(wq, a.qn ? a.qn + d0 : src);   // not used where there is no norm
    load_dims(wk, a.kn ? a.kn + d0 : src);
    const int page = slot >> a.shift, size = 1 << a.shift, off = slot & (size - 1);
    if (slot < 0 || page >= a.n_pages) return;   // uniform: a row that goes nowhere
    uint8_t* const kp = a.kp + static_cast<size_t>(page) * kv_page_bytes(KT, size, a.n_kv, HD);
    uint8_t* const vp = a.vp + static_cast<size_t>(page) * kv_page_bytes(VT, size, a.n_kv, HD);
    if (tid < half) {
        const double turn = static_cast<double>(p) * a.turns[tid];
        double c, s;
        cos_sin_turns(turn - __builtin_rint(turn), &c, &s);
        c *= a.size;
        s *= a.size;
        cs[tid][0] = c;
        cs[tid][1] = s;
        csf[tid] = make_float2(static_cast<float>(c), static_cast<float>(s));
    }
    __syncthreads();
    // the pair of dim d and whether d is its first; the partner of half pairs comes through LDS, a neighbour is in the lane
    auto pair_of = [&](int d) { return a.neighbours ? d >> 1 : d < half ? d : d - half; };
    auto is_first = [&](int d) { return a.neighbours ? (d & 1) == 0 : d < half; };
    for (int it = first; it < end; ++it) {
        float x[N];
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = nx[j];
        if (it + 1 < end) load(it + 1);
        if (it >= a.n_head + a.n_kv) {
            store_row<VT, HD>(x, vp, off, it - a.n_head - a.n_kv, a.n_kv, size, lane);
        } else if (it < a.n_head) {
            float* xs = reinterpret_cast<float*>(rows[wv]);
            if (a.qn) {
                float ss = 0.0f;
#pragma unroll
                for (int j = 0; j < N; ++j) ss = __builtin_fmaf(x[j], x[j], ss);
                const float inv = rsqrtf(group_sum<64>(ss) / static_cast<float>(HD) + a.eps);
#pragma unroll
                for (int j = 0; j < N; ++j) x[j] = x[j] * inv * wq[j];
            }
            if (!a.neighbours) {
#pragma unroll
                for (int j = 0; j < N; ++j) xs[d0 + j] = x[j];
                wave_lds_sync();
            }
            if (d0 < a.n_rot) {
                float y[N];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int d = d0 + j;
                    y[j] = x[j];
                    if (d >= a.n_rot) break;
                    const float2 e = csf[pair_of(d)];
                    const float o = a.neighbours ? x[j ^ 1] : xs[d < half ? d + half : d - half];
                    y[j] = is_first(d) ? rope_lo(x[j], o, e.x, e.y) : rope_hi(o, x[j], e.x, e.y);
                }
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (d0 + j < a.n_rot) x[j] = y[j];
            }
            if (!a.neighbours) wave_lds_sync();   // the next row overwrites the exchange
            uint16_t* to = a.qout + (static_cast<size_t>(t) * a.n_head + it) * HD + d0;
            uint32_t w[N / 2];
#pragma unroll
            for (int j = 0; j < N; j += 2)
                w[j / 2] = a.bf16 ? bf16_bits(x[j]) | (bf16_bits(x[j + 1]) << 16) : half_bits(x[j]) | (half_bits(x[j + 1]) << 16);
            if constexpr (N == 4) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[N / 2 - 1]);
            else *reinterpret_cast<uint32_t*>(to) = w[0];
        } else {
            double* xs = rows[wv];
            double y[N];
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = static_cast<double>(x[j]);
            if (a.kn) {
                double ss = 0.0;
#pragma unroll
                for (int j = 0; j < N; ++j) ss += y[j] * y[j];
                const double inv = 1.0 / sqrt(group_sum64(ss) / HD + static_cast<double>(a.eps));
#pragma unroll
                for (int j = 0; j < N; ++j) y[j] = y[j] * inv * static_cast<double>(wk[j]);
            }
            if (!a.neighbours) {
#pragma unroll
                for (int j = 0; j < N; ++j) xs[d0 + j] = y[j];
                wave_lds_sync();
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int d = d0 + j;
                double z = y[j];
                if (d < a.n_rot) {
                    const int i = pair_of(d);
                    const double o = a.neighbours ? y[j ^ 1] : xs[d < half ? d + half : d - half];
                    z = is_first(d) ? y[j] * cs[i][0] - o * cs[i][1] : o * cs[i][1] + y[j] * cs[i][0];
                }
                x[j] = static_cast<float>(z);
                asm("" : "+v"(x[j]));   // else the compiler makes one rounding of this and fp16's
            }
            if (!a.neighbours) wave_lds_sync();
            store_row<KT, HD>(x, kp, off, it - a.n_head, a.n_kv, size, lane);
        }
    }
}

// The turns of each pair in one position, from the rotation's parameters: base^(-2 i / n_rot) by products of one power in the host's
// 80-bit numbers, 128 of which lose less than fp64 does by one rounding (a pow for each pair takes the host longer).
bool rope_turns(const rmi_rope_params& r, int n_rot, double* turns, double* size) {
    Yarn y;
    if (!yarn_setup(r, n_rot, &y)) return false;
    const long double ratio = n_rot > 2 ? std::pow(static_cast<long double>(r.freq_base), -2.0L / n_rot) : 1.0L;
    long double power = 1.0L;
    for (int i = 0; i < n_rot / 2; ++i, power *= ratio) {
        double f = static_cast<double>(power);
        if (y.on) {
            const double ramp = (1.0 - std::fmin(1.0, std::fmax(0.0, (i - y.low) / std::fmax(0.001, y.high - y.low)))) * y.ext;
            f = f / y.factor * (1.0 - ramp) + f * ramp;
        }
        turns[i] = f / 6.28318530717958647692;
    }
    *size = y.on ? y.mscale : 1.0;
    return true;
}

// whether any of the outputs shares bytes with an input or with another output
bool apart(const RowSet* in, int n_in, const RowSet* out, int n_out) {
    for (int o = 0; o < n_out; ++o) {
        if (!out[o].n || !out[o].bytes) continue;
        for (int i = 0; i < n_in; ++i)
            if (in[i].n && in[i].bytes && rows_overlap(out[o], in[i])) return false;
        for (int k = 0; k < o; ++k)
            if (out[k].n && out[k].bytes && rows_overlap(out[o], out[k])) return false;
    }
    return true;
}
RowSet ints(const int* p, long long n) { return block_of(p, static_cast<size_t>(n) * 4); }

bool table_ok(int n_req, int table_stride) {
    return n_req >= 1 && n_req <= kMaxReq && table_stride >= 1 && static_cast<long long>(n_req) * table_stride <= 0x7fffffffLL;
}

}  // namespace
}  // namespace rmi

using namespace rmi;

extern "C" int rmi_page_plan(const int* past, const int* count, int n_req, int page_size, int n_pages, const int* free_pages,
                             const int* n_free, int* table, int table_stride, int max_tok, int* row_start, int* kv_len, int* slot,
                             int* pos, int* n_left, int* status, void* stream) {
    if (!pool_ok(page_size, n_pages) || !table_ok(n_req, table_stride) || max_tok < 1 || max_tok > static_cast<int>(kSat))
        return fail(RMI_ERR_SHAPE, "page_plan: 1..4096 requests, pages of 16, 32, 64, 128 or 256 positions, max_tok 1..2^30");
    if (!aligned4(past) || !aligned4(count) || !aligned4(free_pages) || !aligned4(n_free) || !aligned4(table) || !aligned4(row_start) ||
        !aligned4(kv_len) || !aligned4(slot) || !aligned4(pos) || !aligned4(n_left) || !aligned4(status))
        return fail(RMI_ERR_POINTER, "page_plan: null or misaligned pointer");
    const RowSet in[] = {ints(past, n_req), ints(count, n_req), ints(free_pages, n_pages), ints(n_free, 1)};
    const RowSet out[] = {ints(table, static_cast<long long>(n_req) * table_stride), ints(row_start, n_req + 1LL), ints(kv_len, n_req),
                          ints(slot, max_tok), ints(pos, max_tok), ints(n_left, 1), ints(status, n_req)};
    if (!apart(in, 4, out, 7)) return fail(RMI_ERR_POINTER, "page_plan: an output lies on another argument");
    const PlanArgs a{past, count, free_pages, n_free, table, row_start, kv_len, slot, pos, n_left, status,
                     n_req, page_shift_of(page_size), n_pages, table_stride, max_tok};
    // a token a thread up to four workgroups a compute unit: each repeats the sums, but a thread's tokens wait for one another.
    // 999 requests with 121 K tokens, four tokens a thread 13.2 us, one 9.5
    const int blocks = std::min(1024, (max_tok + kPlanThreads - 1) / kPlanThreads);
    hipLaunchKernelGGL(page_plan_kernel, dim3(blocks), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), a);
    return launch_status("page_plan");
}

extern "C" int rmi_page_trim(const int* len, const int* keep, int n_req, int page_size, int n_pages, const int* table,
                             int table_stride, const int* n_free, int* free_pages, int* n_out, void* stream) {
    if (!pool_ok(page_size, n_pages) || !table_ok(n_req, table_stride))
        return fail(RMI_ERR_SHAPE, "page_trim: 1..4096 requests, pages of 16, 32, 64, 128 or 256 positions");
    if (!aligned4(len) || !aligned4(keep) || !aligned4(table) || !aligned4(n_free) || !aligned4(free_pages) || !aligned4(n_out))
        return fail(RMI_ERR_POINTER, "page_trim: null or misaligned pointer");
    const RowSet in[] = {ints(len, n_req), ints(keep, n_req), ints(table, static_cast<long long>(n_req) * table_stride), ints(n_free, 1)};
    const RowSet out[] = {ints(free_pages, n_pages), ints(n_out, 1)};
    if (!apart(in, 4, out, 2)) return fail(RMI_ERR_POINTER, "page_trim: an output lies on another argument");
    const TrimArgs a{len, keep, table, n_free, free_pages, n_out, n_req, page_shift_of(page_size), n_pages, table_stride};
    const long long most = std::min<long long>(n_pages, static_cast<long long>(n_req) * table_stride);
    const int blocks = static_cast<int>(std::min<long long>(256, (most + 4 * kPlanThreads - 1) / (4 * kPlanThreads)));
    hipLaunchKernelGGL(page_trim_kernel, dim3(blocks), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), a);
    return launch_status("page_trim");
}

extern "C" int rmi_kv_page_read(int type, const void* pool, const int* slot, void* out, int out_f16, int out_stride, int n,
                                int n_kv, int head_dim, int page_size, int n_pages, void* stream) {
    if (!kv_type_ok(type)) return fail(RMI_ERR_UNSUPPORTED, "kv_page_read: unknown cache type");
    if (!pool_ok(page_size, n_pages) || !kv_shape_ok(page_size, n_kv, head_dim) || n < 0 ||
        static_cast<long long>(n_kv) * head_dim > out_stride)
        return fail(RMI_ERR_SHAPE, "kv_page_read: invalid arguments");
    if (n == 0) return RMI_OK;
    const int per = kReadThreads / (head_dim / 8);
    const long long blocks = (static_cast<long long>(n) + per - 1) / per * n_kv;
    if (blocks > 0xffffffffLL / kReadThreads) return fail(RMI_ERR_SHAPE, "kv_page_read: too many rows for one call");
    if (!aligned16(pool) || !aligned4(slot) || !out || (reinterpret_cast<uintptr_t>(out) & (out_f16 ? 1u : 3u)))
        return fail(RMI_ERR_POINTER, "kv_page_read: null or misaligned pointer");
    const long long el = out_f16 ? 2 : 4;
    const RowSet in[] = {block_of(pool, n_pages * kv_page_bytes(type, page_size, n_kv, head_dim)), ints(slot, n)};
    const RowSet to[] = {{out, n, out_stride * el, static_cast<long long>(n_kv) * head_dim * el}};
    if (!apart(in, 2, to, 1)) return fail(RMI_ERR_POINTER, "kv_page_read: the output lies on what the call reads");
    const bool vec = aligned16(out) && out_stride % (out_f16 ? 8 : 4) == 0;
    return with_type(type, [&](auto t) {
        auto go = [&](auto* kernel) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kReadThreads), 0, static_cast<hipStream_t>(stream),
                               static_cast<const uint8_t*>(pool), slot, out, out_stride, n, n_kv, head_dim, page_shift_of(page_size), n_pages);
            return launch_status("kv_page_read");
        };
        constexpr int T = decltype(t)::value;
        if (out_f16) return vec ? go(&kv_page_read_kernel<T, true, true>) : go(&kv_page_read_kernel<T, true, false>);
        return vec ? go(&kv_page_read_kernel<T, false, true>) : go(&kv_page_read_kernel<T, false, false>);
    });
}

extern "C" int rmi_attn_prep_paged(const float* q3, int q3_stride, const float* qn, const float* kn, int ktype, void* kpool, int vtype,
                                   void* vpool, const int* slot, const int* pos, int qtype, void* qout, int n_head, int n_kv,
                                   int head_dim, int n_rot, const rmi_rope_params* rope, int pairs, float eps, int ntok, int page_size,
                                   int n_pages, void* stream) {
    if (!kv_type_ok(ktype) || !kv_type_ok(vtype)) return fail(RMI_ERR_UNSUPPORTED, "attn_prep_paged: unknown cache type");
    if (qtype != RMI_ROWS_F16 && qtype != RMI_ROWS_BF16) return fail(RMI_ERR_UNSUPPORTED, "attn_prep_paged: q in F16 or BF16");
    if (!pool_ok(page_size, n_pages) || !kv_shape_ok(page_size, n_kv, head_dim) || n_head <= 0 || n_head > 65535 || n_head % n_kv ||
        n_rot < 0 || n_rot > head_dim || n_rot % 2 || ntok < 1 || ntok > 0x7fffffff / (64 * kPrepWaves) || !rope ||
        !(rope->freq_base > 1.0f) || (pairs != RMI_ROPE_HALF && pairs != RMI_ROPE_NEIGHBOURS) ||
        2LL * n_head * head_dim + 2LL * n_kv * head_dim > 0x7fffffffLL)
        return fail(RMI_ERR_SHAPE, "attn_prep_paged: invalid arguments");
    if (!aligned4(q3) || (qn && !aligned4(qn)) || (kn && !aligned4(kn)) || !aligned16(kpool) || !aligned16(vpool) || !aligned4(slot) ||
        !aligned4(pos) || !aligned16(qout))
        return fail(RMI_ERR_POINTER, "attn_prep_paged: null or misaligned pointer");
    const size_t pools[] = {n_pages * kv_page_bytes(ktype, page_size, n_kv, head_dim), n_pages * kv_page_bytes(vtype, page_size, n_kv, head_dim)};
    const RowSet in[] = {{q3, ntok, 4LL * q3_stride, 4LL * (2 * n_head + 2 * n_kv) * head_dim}, block_of(qn, qn ? head_dim * 4 : 0),
                         block_of(kn, kn ? head_dim * 4 : 0), ints(slot, ntok), ints(pos, ntok)};
    const RowSet out[] = {block_of(kpool, pools[0]), block_of(vpool, pools[1]), block_of(qout, static_cast<size_t>(ntok) * n_head * head_dim * 2)};
    if (!apart(in, 5, out, 3)) return fail(RMI_ERR_POINTER, "attn_prep_paged: a pool or qout lies on another argument");
    PagedPrepArgs a{};
    if (!rope_turns(*rope, n_rot, a.turns, &a.size)) return fail(RMI_ERR_SHAPE, "attn_prep_paged: invalid YaRN parameters");
    a.q3 = q3;
    a.qn = qn;
    a.kn = kn;
    a.kp = static_cast<uint8_t*>(kpool);
    a.vp = static_cast<uint8_t*>(vpool);
    a.slot = slot;
    a.pos = pos;
    a.qout = static_cast<uint16_t*>(qout);
    a.q3_stride = q3_stride;
    a.n_head = n_head;
    a.n_kv = n_kv;
    a.n_rot = n_rot;
    a.shift = page_shift_of(page_size);
    a.n_pages = n_pages;
    a.neighbours = pairs == RMI_ROPE_NEIGHBOURS;
    a.bf16 = qtype == RMI_ROWS_BF16;
    a.eps = eps;
    const int items = n_head + 2 * n_kv;
    // rows a wave: as many as leave about a thousand workgroups (they share a token's angles), one for few tokens (latency)
    a.per_wave = std::min((items + kPrepWaves - 1) / kPrepWaves, static_cast<int>((static_cast<long long>(items) * ntok + 4095) / 4096));
    const int parts = (items + kPrepWaves * a.per_wave - 1) / (kPrepWaves * a.per_wave);
    return with_type(ktype, [&](auto k) {
        return with_type(vtype, [&](auto v) {
            auto go = [&](auto* kernel) {
                hipLaunchKernelGGL(kernel, dim3(ntok, parts), dim3(64 * kPrepWaves), 0, static_cast<hipStream_t>(stream), a);
                return launch_status("attn_prep_paged");
            };
            constexpr int KT = decltype(k)::value, VT = decltype(v)::value;
            return head_dim == 256 ? go(&prep_paged_kernel<KT, VT, 256>) : go(&prep_paged_kernel<KT, VT, 128>);
        });
    });
}
