// overlap.h - whether two arguments of a call share bytes (host only, exact for strided rows): workgroups that write what
// others read give results that hang on their order.
#pragma once

#include <cstddef>
#include <cstdint>
#include <utility>

namespace rmi {

// n rows of `bytes` from p, `stride` bytes apart
struct RowSet {
    const void* p;
    long long n, stride, bytes;
};
inline RowSet block_of(const void* p, size_t bytes) { return {p, 1, 0, static_cast<long long>(bytes)}; }

// Row by row of the smaller set, each against the other set by one division; sets that lie apart by their ends alone.
inline bool rows_overlap(RowSet a, RowSet b) {
    auto begin = [](RowSet& r) {   // of the rows in ascending order
        long long p = static_cast<long long>(reinterpret_cast<uintptr_t>(r.p));
        if (r.stride < 0) p += (r.n - 1) * r.stride, r.stride = -r.stride;
        if (r.stride == 0) r.n = 1;
        return p;
    };
    long long pa = begin(a), pb = begin(b);
    if (a.n > b.n) std::swap(a, b), std::swap(pa, pb);
    if (pb + (b.n - 1) * b.stride + b.bytes <= pa || pa + (a.n - 1) * a.stride + a.bytes <= pb) return false;
    for (long long i = 0; i < a.n; ++i) {
        const long long first = pa + i * a.stride, end = first + a.bytes;
        const long long d = first - pb - b.bytes;   // b's row k ends behind `first` where k stride > d
        const long long k = d < 0 ? 0 : b.n == 1 ? 1 : d / b.stride + 1;
        if (k < b.n && pb + k * b.stride < end) return true;
    }
    return false;
}

}  // namespace rmi
