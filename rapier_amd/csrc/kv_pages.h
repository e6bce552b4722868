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

}  // namespace rmi
