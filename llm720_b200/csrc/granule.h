// Which bytes of an aligned 16-byte granule belong to a buffer.  Rows at any address are read as granules; the ones at the
// buffer's two ends may reach beyond it, and of those only the buffer's own values are read.  Plain C++, so that the
// arithmetic can be run on the host.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define PEER_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define PEER_HOST_DEVICE inline
#endif

namespace peer {

struct GranulePart { int first, last; };      // bytes [first, last) of the granule, first == last: none
PEER_HOST_DEVICE bool granule_inside(uintptr_t granule, uintptr_t begin, uintptr_t end) {
    return granule >= begin && granule + 16 <= end;
}
PEER_HOST_DEVICE GranulePart granule_part(uintptr_t granule, uintptr_t begin, uintptr_t end) {
    if (granule + 16 <= begin || granule >= end) return {0, 0};
    return {granule < begin ? static_cast<int>(begin - granule) : 0, granule + 16 > end ? static_cast<int>(end - granule) : 16};
}

// The part of a row's copy that goes by pieces of 16 bytes: values [begin, end) of D, pieces being granules of the row that is
// written at `dst`, each read as the granules that hold it, `shift` bytes behind the first one's start.  Fewer than two pieces'
// values are left over at either end, those of a piece whose granules reach beyond the buffer [buf, buf_end) among them.
struct PieceRange { int begin, end; uint32_t shift; };
PEER_HOST_DEVICE PieceRange piece_range(uintptr_t row, uintptr_t dst, int D, int size, uintptr_t buf, uintptr_t buf_end) {
    const int N = 16 / size;
    PieceRange p;
    p.begin = static_cast<int>((16u - (static_cast<uint32_t>(dst) & 15u)) & 15u) / size;
    p.begin = p.begin < D ? p.begin : D;
    p.end = D - ((D - p.begin) & (N - 1));
    p.shift = (static_cast<uint32_t>(row) + static_cast<uint32_t>(p.begin * size)) & 15u;
    if (p.shift && p.begin < p.end) {
        // the first piece's first granule can only reach out in front, the last piece's second one only behind
        if (row + p.begin * size < buf + p.shift) p.begin += N;
        if (p.begin < p.end && row + p.end * size + 16 > buf_end + p.shift) p.end -= N;
    }
    return p;
}

// 16 / size values of a row of D from value `at` on (which may lie up to that many in front of the row or behind it): address of
// the first granule that may hold some, which of it and the next one do, and the values' offset from its start.
struct GranuleWants { uintptr_t first; bool lo, hi; uint32_t shift; };
PEER_HOST_DEVICE GranuleWants granule_wants(uintptr_t row, int64_t at, int64_t D, int size) {
    const uintptr_t a = row + at * size;
    const uint32_t shift = static_cast<uint32_t>(a & 15u);
    const int N = 16 / size, lead = static_cast<int>(shift) / size;       // values in front of these in the first granule
    const bool some = at < D;
    return {a - shift, some && at + N - lead > 0, some && lead > 0 && at + N - lead < D, shift};
}

}  // namespace peer
