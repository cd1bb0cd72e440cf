// Rows at any address.  A row is brought into shared memory as the aligned 16-byte granules that cover it; thread c's
// 16 bytes lie at the same offset, 0 to 15, in granules c and c + 1 for every thread, and come out with a few selects and
// a funnel shift.  Results are laid down in shared memory in the row's own order and leave as aligned granules the same
// way, the first and last by value.  A granule at a row's end may hold values of its neighbours, which are not used; one
// that reaches beyond the buffer's first or last value is read value by value (granule.h), so nothing outside the buffer
// (from its first row's first value to its last row's last one) is read.
#pragma once

#include "granule.h"
#include "row_ops.cuh"

namespace peer {

constexpr int RING_COLUMNS = 16, RING_THREADS = 512;      // columns per thread, threads of a block at most
inline int ring_warps(int64_t D) { return static_cast<int>((D + 32 * RING_COLUMNS - 1) / (32 * RING_COLUMNS)); }

// 16, 8 or 4 bytes of this thread's shared memory
template <typename V> __device__ __forceinline__ V shared_at(uint32_t at);
template <> __device__ __forceinline__ uint4 shared_at<uint4>(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
template <> __device__ __forceinline__ uint2 shared_at<uint2>(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
template <> __device__ __forceinline__ uint32_t shared_at<uint32_t>(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ void store_shared(uint32_t at, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void store_shared(uint32_t at, const uint2& v) {
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void store_shared(uint32_t at, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
// the first `bytes` (0 to 16) of a granule, zeros behind them
__device__ __forceinline__ void copy_async_filled(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// 16 bytes at offset `shift` (0 to 15) of two granules
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, uint32_t shift) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (shift & 8u) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (shift & 4u) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const uint32_t bits = (shift & 3u) * 8u;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                      __funnelshift_r(w[3], w[4], bits));
}
// 16 bytes at offset `shift` of the 32 at `at`
__device__ __forceinline__ uint4 shared_shifted(uint32_t at, uint32_t shift) {
    return shifted(shared_at<uint4>(at), shared_at<uint4>(at + 16), shift);
}
// 8 or 4 bytes at any shared address
template <typename V> __device__ __forceinline__ V shared_unaligned(uint32_t at);
template <> __device__ __forceinline__ uint2 shared_unaligned<uint2>(uint32_t at) {
    const uint32_t a = at & ~3u, bits = (at & 3u) * 8u;
    const uint32_t w0 = shared_at<uint32_t>(a), w1 = shared_at<uint32_t>(a + 4), w2 = shared_at<uint32_t>(a + 8);
    return make_uint2(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits));
}
template <> __device__ __forceinline__ uint32_t shared_unaligned<uint32_t>(uint32_t at) {
    const uint32_t a = at & ~3u;
    return __funnelshift_r(shared_at<uint32_t>(a), shared_at<uint32_t>(a + 4), (at & 3u) * 8u);
}
// granules that cover `bytes` at an address of offset `shift`
__device__ __forceinline__ int granules(uint32_t shift, int bytes) { return (static_cast<int>(shift) + bytes + 15) >> 4; }
__device__ __forceinline__ uint32_t offset16(const void* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u; }

// A granule that reaches beyond its buffer [begin, end), value by value, zeros in place of what lies outside.  Rare (the first
// and last rows of a buffer at an odd address), so it is kept out of line: beside the loads of whole granules its branches
// would keep them from being in flight together.
template <typename T>
__device__ __noinline__ uint4 partial_granule(const void* g, const void* begin, const void* end) {
    const GranulePart part = granule_part(reinterpret_cast<uintptr_t>(g), reinterpret_cast<uintptr_t>(begin), reinterpret_cast<uintptr_t>(end));
    alignas(16) T v[16 / sizeof(T)];
#pragma unroll
    for (int q = 0; q < static_cast<int>(16 / sizeof(T)); ++q) {
        const int byte = q * static_cast<int>(sizeof(T));
        v[q] = byte >= part.first && byte < part.last ? __ldg(static_cast<const T*>(g) + q) : T{};
    }
    return *reinterpret_cast<const uint4*>(v);
}

// a group's threads bring the granules of one row, and zeros in the one behind them (a thread's 16 bytes may reach there).
// Behind the row's own end nothing is read.  HEAD: the row may be the buffer's first, and its first granule reach out in front.
template <bool HEAD>
__device__ __forceinline__ void fetch_row(uint32_t dst, const void* row, int bytes, int gt, int threads, const void* begin) {
    const uint32_t shift = offset16(row);
    const char* first = static_cast<const char*>(row) - shift;
    const int n = granules(shift, bytes), end = static_cast<int>(shift) + bytes;
    int c = gt;
    if (HEAD && gt == 0 && first < static_cast<const char*>(begin)) {
        store_shared(dst, partial_granule<uint8_t>(first, begin, static_cast<const char*>(row) + bytes));
        c += threads;
    }
    for (; c <= n; c += threads) copy_async_filled(dst + c * 16, c < n ? first + c * 16 : first, max(min(16, end - c * 16), 0));
}
// Only the first row's granules reach out in front of the buffer, so only a ring's first fetch asks: rows closer together than
// a granule (`stride` bytes) at an odd address go by value.
inline bool first_row_alone(const void* begin, int64_t stride, int64_t rows) { return rows <= 1 || stride >= 16 || aligned16(begin); }
// a row laid down at `src` (16 bytes in front of it are the group's too) to its place in memory; U: a value
template <typename U>
__device__ __forceinline__ void store_row(void* row, uint32_t src, int bytes, int gt, int threads) {
    const uint32_t shift = offset16(row);
    char* first = static_cast<char*>(row) - shift;
    const int n = granules(shift, bytes);
    for (int c = gt; c < n; c += threads) {
        const uint4 v = shared_shifted(src + c * 16 - (shift ? 16u : 0u), (16u - shift) & 15u);
        const int from = c * 16 - static_cast<int>(shift);           // of the row's bytes
        if (from >= 0 && from + 16 <= bytes) {
            *reinterpret_cast<uint4*>(first + c * 16) = v;
        } else {
            const U* e = reinterpret_cast<const U*>(&v);
#pragma unroll
            for (int q = 0; q < static_cast<int>(16 / sizeof(U)); ++q) {
                const int at = from + q * static_cast<int>(sizeof(U));
                if (at >= 0 && at < bytes) *reinterpret_cast<U*>(static_cast<char*>(row) + at) = e[q];
            }
        }
    }
}

// The same without shared memory, for a thread that takes 16 / sizeof(T) values of a row of D from value `at` on, where `at`
// may lie up to that many in front of the row or behind it: the one or two granules that hold them, zeros for one that holds
// none of the row's values, and the values' offset in them.  `load_granules` is for rows 16 bytes and more away from the ends of
// their buffer; its loads have no branch between them.  `load_edge_granules` takes any row.
struct Granules { uint4 lo, hi; uint32_t shift; };
template <typename T>
__device__ __forceinline__ Granules load_granules(const T* row, int64_t at, int64_t D) {
    const GranuleWants w = granule_wants(reinterpret_cast<uintptr_t>(row), at, D, sizeof(T));
    const uint4* first = reinterpret_cast<const uint4*>(w.first);
    Granules g;
    g.shift = w.shift;
    g.lo = w.lo ? __ldg(first) : make_uint4(0u, 0u, 0u, 0u);
    g.hi = w.hi ? __ldg(first + 1) : make_uint4(0u, 0u, 0u, 0u);
    return g;
}
template <typename T>
__device__ __forceinline__ Granules load_edge_granules(const T* row, int64_t at, int64_t D, const void* begin, const void* end) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(begin), e = reinterpret_cast<uintptr_t>(end);
    const GranuleWants w = granule_wants(reinterpret_cast<uintptr_t>(row), at, D, sizeof(T));
    const uint4* first = reinterpret_cast<const uint4*>(w.first);
    Granules g{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u), w.shift};
    if (w.lo) g.lo = granule_inside(w.first, b, e) ? __ldg(first) : partial_granule<T>(first, begin, end);
    if (w.hi) g.hi = granule_inside(w.first + 16, b, e) ? __ldg(first + 1) : partial_granule<T>(first + 1, begin, end);
    return g;
}
// rows at either end of a buffer of n rows that lie within 16 bytes of it, for rows `stride` bytes apart
inline int64_t edge_rows(int64_t n, int64_t stride) { return stride >= 16 ? 1 : stride > 0 ? (16 + stride - 1) / stride : n; }
// values [at, at + 16 / sizeof(T)) to a row, the address of value `at` being a granule's
template <typename T>
__device__ __forceinline__ void store_granule(T* row, int64_t at, int64_t D, const uint4& v) {
    constexpr int N = 16 / sizeof(T);
    if (at >= 0 && at + N <= D) {
        *reinterpret_cast<uint4*>(row + at) = v;
    } else {
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (at + q >= 0 && at + q < D) row[at + q] = e[q];
    }
}

// bytes of shared memory that hold a row of `columns` values of `size` bytes wherever it begins
__host__ __device__ constexpr int row_room(int columns, int size) { return columns * size + 32; }

}  // namespace peer
