// kv_pages.h - caches in pages, shared by the calls on them.  A page is a cache (kv_cache.h) of page_size positions, a pool
// n_pages of them; slot s is position s % page_size of page s / page_size.  Everything that a device word says is checked
// there: no page id, slot or length leads outside a pool, a table or the rows of a call.
#pragma once

#include "kv_cache.h"

namespace rmi {

constexpr int kMaxReq = 4096;   // requests of a batch: their row starts fit LDS

inline bool page_size_ok(int n) { return n == 16 || n == 32 || n == 64 || n == 128 || n == 256; }
inline int page_shift_of(int n) { return __builtin_ctz(static_cast<unsigned>(n)); }
inline bool pool_ok(int page_size, int n_pages) {
    return page_size_ok(page_size) && n_pages > 0 && n_pages <= 0x7fffffff / page_size;   // a slot fits an int
}
__host__ __device__ constexpr size_t kv_page_bytes(int type, int page_size, int n_kv, int head_dim) {
    return static_cast<size_t>(page_size) * n_kv * (kv_row_bytes(type, head_dim) + (type == kKvF16 ? 0 : head_dim / kKvBlock));
}

// v of lane l - 1, - 2, ... of a row of 16, or of the last lane of the rows before; 0 where there is none
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_before(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
}
// inclusive prefix sums over a wave, by an addition that may saturate: within rows of 16 lanes by row shifts, then the last lanes
// of rows 0 and 2 to the next row, then lane 31 to rows 2 and 3.  All lanes are active.
template <typename F>
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, F&& add) {
    v = add(v, lane_before<0x111, 0xf>(v));
    v = add(v, lane_before<0x112, 0xf>(v));
    v = add(v, lane_before<0x114, 0xf>(v));
    v = add(v, lane_before<0x118, 0xf>(v));
    v = add(v, lane_before<0x142, 0xa>(v));
    v = add(v, lane_before<0x143, 0xc>(v));
    return v;
}

}  // namespace rmi
