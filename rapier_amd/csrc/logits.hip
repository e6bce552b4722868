// logits.hip - what a sampler wants done to logits before argmax / top-k, for the columns of a tree's nodes: additive
// biases, penalties for repeated tokens and a grammar's mask (no counterpart in the reference, whose server gets the raw
// logits, qw:2513-2531).
//
// One launch, no workspace: a workgroup owns 1024 neighbouring logits and counts the history's tokens among them in LDS
// (integer adds, so the order does not matter).  A column's text is the shared history plus its path in the draft, and a
// window that reaches over the path's tokens drops as many of the history's oldest: both are at most 64 single tokens per
// column, kept as a short list of those in the slice and added to the counts for that column alone.  Every workgroup reads
// the whole history (four ids a lane and load, from the L2): one column of 248320 logits takes 4.8 us behind 4001 tokens and
// 8.1 behind 20001, bound by the chain length - ids - counts - logits at the first and by those reads at the second.
#include "overlap.h"
#include "rmi_common.h"

#include <cmath>

namespace rmi {
namespace {

constexpr int kSlice = 1024;
constexpr int kThreads = 256;   // four neighbouring logits each
constexpr int kMaxDraft = 64;

typedef int int4u __attribute__((ext_vector_type(4), aligned(4)));   // a window begins anywhere

struct LogitsArgs {
    const float* logits;
    float* out;
    int n, ncols, col_stride, out_stride, per_wg;   // per_wg: columns a workgroup handles
    const int *history, *history_len;
    int max_history;
    const int* draft;
    const uint64_t* masks;
    int ndraft;
    rmi_penalties pen;
    const int* bias_ids;
    const float* bias_vals;
    int n_bias;
    const uint32_t* allow;
    int allow_stride;
};

template <bool VEC>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a) {
    __shared__ __attribute__((aligned(16))) int cnt[kSlice];
    __shared__ __attribute__((aligned(16))) int bidx[kSlice];
    __shared__ int adj[2 * kMaxDraft];   // offset in the slice, or -1: history tokens that a window drops, then draft tokens
    __shared__ int any;
    const int tid = threadIdx.x, v0 = blockIdx.x * kSlice, o0 = 4 * tid, v = v0 + o0;
    const int c0 = blockIdx.y * a.per_wg, c1 = min(c0 + a.per_wg, a.ncols);
    // a column's four logits and the grammar's word, a column ahead
    float nx[4];
    uint32_t nok = 0xfu;
    auto load = [&](int c) {
        const float* in = a.logits + static_cast<size_t>(c) * a.col_stride + v;
        if (VEC && v + 3 < a.n) {
            const float4 f = *reinterpret_cast<const float4*>(in);
            nx[0] = f.x, nx[1] = f.y, nx[2] = f.z, nx[3] = f.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) nx[i] = v + i < a.n ? in[i] : 0.0f;
        }
        if (a.allow && v < a.n) nok = a.allow[static_cast<size_t>(c) * a.allow_stride + (v >> 5)] >> (v & 31);
    };
    load(c0);
    *reinterpret_cast<int4*>(cnt + o0) = make_int4(0, 0, 0, 0);
    *reinterpret_cast<int4*>(bidx + o0) = make_int4(-1, -1, -1, -1);
    if (tid == 0) any = 0;
    const int len = a.history_len ? min(max(a.history_len[0], 0), a.max_history) : 0;
    const int window = a.pen.window > 0 ? a.pen.window : 0x7fffffff;
    const int start = len > window ? len - window : 0;
    __syncthreads();
    if (tid < 2 * kMaxDraft) {
        int off = -1;
        const int k = tid < kMaxDraft ? tid : tid - kMaxDraft;
        if (k < a.ndraft) {
            const int* from = tid < kMaxDraft ? (start + k < len ? a.history + start + k : nullptr) : a.draft + k;
            if (from) off = static_cast<int>(static_cast<unsigned>(from[0]) - static_cast<unsigned>(v0));
        }
        const bool in = static_cast<unsigned>(off) < kSlice;
        adj[tid] = in ? off : -1;
        if (in) any = 1;   // every writer stores the same value
    }
    auto count = [&](int id) {
        const unsigned off = static_cast<unsigned>(id) - static_cast<unsigned>(v0);
        if (off < kSlice) atomicAdd(&cnt[off], 1);
    };
    const int* hist = a.history + start;
    const int nh = len - start, whole = nh & ~3;
#pragma unroll 4
    for (int i = 4 * tid; i < whole; i += 4 * kThreads) {
        const int4u h = *reinterpret_cast<const int4u*>(hist + i);
        count(h[0]);
        count(h[1]);
        count(h[2]);
        count(h[3]);
    }
    if (tid < nh - whole) count(hist[whole + tid]);
    for (int i = tid; i < a.n_bias; i += kThreads) {
        const unsigned off = static_cast<unsigned>(a.bias_ids[i]) - static_cast<unsigned>(v0);
        if (off < kSlice) atomicMax(&bidx[off], i);
    }
    __syncthreads();
    const int4 bi = *reinterpret_cast<const int4*>(bidx + o0);
    float bias[4];
    bias[0] = bi.x >= 0 ? a.bias_vals[bi.x] : 0.0f;
    bias[1] = bi.y >= 0 ? a.bias_vals[bi.y] : 0.0f;
    bias[2] = bi.z >= 0 ? a.bias_vals[bi.z] : 0.0f;
    bias[3] = bi.w >= 0 ? a.bias_vals[bi.w] : 0.0f;
    const bool biased[4] = {bi.x >= 0, bi.y >= 0, bi.z >= 0, bi.w >= 0};
    const bool adjust = any != 0;   // uniform
    for (int c = c0; c < c1; ++c) {
        float x[4] = {nx[0], nx[1], nx[2], nx[3]};
        const uint32_t ok = nok;
        if (c + 1 < c1) load(c + 1);
        int delta = 0, doff = -1;
        if (adjust) {
            if (tid < 2 * kMaxDraft) {
                const uint64_t mask = a.masks[c] & (a.ndraft >= 64 ? ~0ull : (1ull << a.ndraft) - 1);
                const int np = __popcll(mask);
                const long long total = static_cast<long long>(len) + np;
                const long long begin = total > window ? total - window : 0;   // the window's first place in the text
                doff = adj[tid];
                if (tid < kMaxDraft) {
                    delta = start + tid < begin ? -1 : 0;
                } else {
                    const int j = tid - kMaxDraft;
                    const long long place = static_cast<long long>(len) + __popcll(mask & ((1ull << j) - 1));
                    delta = (mask >> j & 1) && place >= begin ? 1 : 0;
                }
                if (doff < 0) delta = 0;
                if (delta) atomicAdd(&cnt[doff], delta);
            }
            __syncthreads();
        }
        const int4 m4 = *reinterpret_cast<const int4*>(cnt + o0);
        const int m[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (biased[i]) x[i] += bias[i];
            if (m[i] > 0) {
                x[i] = x[i] > 0.0f ? x[i] / a.pen.repetition : x[i] * a.pen.repetition;
                x[i] -= static_cast<float>(m[i]) * a.pen.frequency + a.pen.presence;
            }
            if (!(ok >> i & 1u)) x[i] = -INFINITY;
        }
        float* out = a.out + static_cast<size_t>(c) * a.out_stride + v;
        if (VEC && v + 3 < a.n) {
            *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (v + i < a.n) out[i] = x[i];
        }
        if (adjust) {
            __syncthreads();   // every count is read
            if (delta) atomicAdd(&cnt[doff], -delta);
            __syncthreads();
        }
    }
}

}  // namespace
}  // namespace rmi

using namespace rmi;

extern "C" int rmi_logits_process(const float* logits, int n, int ncols, int col_stride, float* out, int out_stride,
                                  const int* history, const int* history_len, int max_history, const int* draft,
                                  const uint64_t* masks, int ndraft, const rmi_penalties* penalties, const int* bias_ids,
                                  const float* bias_vals, int n_bias, const uint32_t* allow, int allow_stride,
                                  void* stream) {
    if (n <= 0 || n > 0x7fffffff - kSlice || ncols < 1 || ncols > 64 || (ncols > 1 && (col_stride < n || out_stride < n)) || max_history < 0 || ndraft < 0 ||
        ndraft > kMaxDraft || n_bias < 0 || !penalties || !(penalties->repetition > 0.0f) ||
        (allow && ncols > 1 && allow_stride < (n - 1) / 32 + 1) || (out == logits && ncols > 1 && out_stride != col_stride))
        return fail(RMI_ERR_SHAPE, "logits_process: invalid arguments");
    const bool hist = max_history > 0;
    if (!aligned4(logits) || !aligned4(out) || (hist && (!aligned4(history) || !aligned4(history_len))) ||
        (ndraft > 0 && (!aligned4(draft) || !masks || (reinterpret_cast<uintptr_t>(masks) & 7u))) ||
        (n_bias > 0 && (!aligned4(bias_ids) || !aligned4(bias_vals))) || (allow && !aligned4(allow)))
        return fail(RMI_ERR_POINTER, "logits_process: null or misaligned pointer");
    if (out != logits && rows_overlap({logits, ncols, 4LL * col_stride, 4LL * n}, {out, ncols, 4LL * out_stride, 4LL * n}))
        return fail(RMI_ERR_POINTER, "logits_process: the output lies on other logits' places");
    LogitsArgs a{};
    a.logits = logits;
    a.out = out;
    a.n = n;
    a.ncols = ncols;
    a.col_stride = col_stride;
    a.out_stride = out_stride;
    a.history = history;
    a.history_len = hist ? history_len : nullptr;
    a.max_history = max_history;
    a.draft = draft;
    a.masks = masks;
    a.ndraft = ndraft;
    a.pen = *penalties;
    a.bias_ids = bias_ids;
    a.bias_vals = bias_vals;
    a.n_bias = n_bias;
    a.allow = allow;
    a.allow_stride = allow_stride;
    // columns a workgroup: they share its counts, but about 2000 workgroups are needed to hide a column's latency.  248320
    // logits, history 1999, 1 / 2 / 4 / 8 columns a workgroup: 16 columns 11.9 / 9.7 / 10.6 / 14.1 us (3.3 TB/s at the
    // rule's 2), 64 columns 43.8 / 34.8 / 31.1 / 29.7 (4.3 TB/s at 8)
    const int slices = (n + kSlice - 1) / kSlice;
    a.per_wg = static_cast<int>((static_cast<long long>(ncols) * slices + 2047) / 2048);
    a.per_wg = a.per_wg < ncols ? a.per_wg : ncols;
    const bool vec = aligned16(logits) && aligned16(out) && (ncols == 1 || (col_stride % 4 == 0 && out_stride % 4 == 0));
    auto go = [&](auto* kernel) {
        hipLaunchKernelGGL(kernel, dim3(slices, (ncols + a.per_wg - 1) / a.per_wg), dim3(kThreads), 0,
                           static_cast<hipStream_t>(stream), a);
        return launch_status("logits_process");
    };
    return vec ? go(&logits_kernel<true>) : go(&logits_kernel<false>);
}
