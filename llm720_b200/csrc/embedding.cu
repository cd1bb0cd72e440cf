// Scaled embedding lookup and its gradient.
//
//   out[t]  = scale * W[id_t]                       (a row of zeros for an id outside the table)
//   dW[v]   = scale * sum over t with id_t = v of dy[t], rounded once; zero for rows no token names
//
// The lookup replaces the nn.Embedding read of the reference's model
// (llm/models/foundation.py:338) and of torch's backward pass to it.  The
// gradient sorts the positions by id (row_sort.cu), then adds each id's rows in
// the order of their positions, in fp32: nothing is accumulated in memory, so
// the sums have one order and every row of dW is written exactly once.
//
// The sorted positions are cut into tiles of equal length, whatever the ids'
// frequencies are (text: one id can hold a tenth of all tokens).  An id whose
// positions lie in one tile is finished there; one that crosses tiles leaves a
// partial row per tile, and the join kernel adds those in tile order.
#include <cstdio>

#include "kernels.h"
#include "row_ops.cuh"

namespace peer {
void set_global_error(const char* msg);

namespace {

constexpr int SUM_THREADS = 256;

template <typename T, int VEC> struct Load;
template <typename T> struct Load<T, 1> {
    __device__ static __forceinline__ void get(const T* p, float (&f)[1]) { f[0] = to_f32<T>(*p); }
    __device__ static __forceinline__ void put(T* p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }
};
template <> struct Load<float, 4> {
    __device__ static __forceinline__ void get(const float* p, float (&f)[4]) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p));
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
    __device__ static __forceinline__ void put(float* p, const float (&f)[4]) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
};
template <typename T> struct Load<T, 8> {
    __device__ static __forceinline__ void get(const T* p, float (&f)[8]) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = to_f32<T>(e[q]);
    }
    __device__ static __forceinline__ void put(T* p, const float (&f)[8]) {
        uint4 v;
        T* e = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int q = 0; q < 8; ++q) e[q] = from_f32<T>(f[q]);
        *reinterpret_cast<uint4*>(p) = v;
    }
};

__device__ __forceinline__ int64_t id_at(const void* ids, int id_bytes, int64_t i) {
    return id_bytes == 8 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// one warp per token
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_kernel(const void* __restrict__ ids, int id_bytes, int64_t n, const T* __restrict__ w,
                                                    int64_t vocab, int64_t D, float scale, T* __restrict__ out,
                                                    unsigned long long* dropped) {
    const int lane = threadIdx.x & 31;
    const int64_t stride = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
    for (int64_t t = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; t < n; t += stride) {
        const int64_t id = id_at(ids, id_bytes, t);
        const bool inside = id >= 0 && id < vocab;
        if (!inside && dropped && lane == 0) atomicAdd(dropped, 1ULL);
        const T* row = w + (inside ? id : 0) * D;
        for (int64_t c = static_cast<int64_t>(lane) * VEC; c < D; c += 32 * VEC) {
            float f[VEC];
            if (inside) {
                Load<T, VEC>::get(row + c, f);
#pragma unroll
                for (int q = 0; q < VEC; ++q) f[q] *= scale;
            } else {
#pragma unroll
                for (int q = 0; q < VEC; ++q) f[q] = 0.f;
            }
            Load<T, VEC>::put(out + t * D + c, f);
        }
    }
}

struct SumParams {
    const uint32_t* keys; const uint32_t* order;   // sorted ids (vocab = none) and their positions
    int64_t n; uint32_t vocab;
    const void* src; int64_t src_stride;           // rows that are added
    float scale;
    void* out; int64_t D;
    float* partial;                                // [tiles][2][D]
    int per_tile; int64_t tiles;
};

// block: one tile of sorted positions, SUM_THREADS * VEC columns
template <typename T, int VEC>
__global__ void __launch_bounds__(SUM_THREADS) row_sum_kernel(const SumParams p) {
    const int64_t c = (static_cast<int64_t>(blockIdx.y) * SUM_THREADS + threadIdx.x) * VEC;
    if (c >= p.D) return;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per_tile;
    const int64_t t1 = t0 + p.per_tile < p.n ? t0 + p.per_tile : p.n;
    uint32_t cur = p.keys[t0];
    if (cur == p.vocab) return;
    bool open_left = t0 > 0 && p.keys[t0 - 1] == cur;      // the id's positions begin in an earlier tile
    float acc[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
    for (int64_t j = t0; j <= t1; ++j) {
        const uint32_t key = j < p.n ? p.keys[j] : p.vocab;
        if (key != cur || j == t1) {
            const bool open_right = key == cur;
            if (open_left || open_right) {
                float* dst = p.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (open_left ? 0 : 1)) * p.D + c;
#pragma unroll
                for (int q = 0; q < VEC; ++q) dst[q] = acc[q];
            } else {
                float f[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) f[q] = acc[q] * p.scale;
                Load<T, VEC>::put(static_cast<T*>(p.out) + static_cast<int64_t>(cur) * p.D + c, f);
            }
            if (j == t1 || key == p.vocab) return;
            cur = key;
            open_left = false;
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
        }
        float f[VEC];
        Load<T, VEC>::get(static_cast<const T*>(p.src) + static_cast<int64_t>(p.order[j]) * p.src_stride + c, f);
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] += f[q];
    }
}

// first index in [0, n) whose key is not below `key`
__device__ __forceinline__ int64_t lower_bound(const uint32_t* __restrict__ keys, int64_t n, uint32_t key) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < key) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// the id whose positions begin in tile blockIdx.x and reach past its end: the sum of its partial rows
template <typename T>
__global__ void __launch_bounds__(SUM_THREADS) row_sum_join_kernel(const SumParams p) {
    const int64_t c = static_cast<int64_t>(blockIdx.y) * SUM_THREADS + threadIdx.x;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per_tile, t1 = t0 + p.per_tile;
    if (t1 >= p.n || c >= p.D) return;
    const uint32_t cur = p.keys[t1 - 1];
    if (cur == p.vocab || p.keys[t1] != cur) return;
    if (t0 > 0 && p.keys[t0] == cur && p.keys[t0 - 1] == cur) return;      // began in an earlier tile
    const int64_t last = (lower_bound(p.keys, p.n, cur + 1) - 1) / p.per_tile;
    float acc = p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + 1) * p.D + c];
    for (int64_t u = static_cast<int64_t>(blockIdx.x) + 1; u <= last; ++u) acc += p.partial[u * 2 * p.D + c];
    static_cast<T*>(p.out)[static_cast<int64_t>(cur) * p.D + c] = from_f32<T>(acc * p.scale);
}

// rows that no position names: zeros (one warp per row)
template <typename T>
__global__ void __launch_bounds__(256) row_zero_kernel(const SumParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t stride = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
    for (int64_t v = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; v < p.vocab; v += stride) {
        const int64_t at = lower_bound(p.keys, p.n, static_cast<uint32_t>(v));
        if (at < p.n && p.keys[at] == static_cast<uint32_t>(v)) continue;
        for (int64_t c = lane; c < p.D; c += 32) static_cast<T*>(p.out)[v * p.D + c] = from_f32<T>(0.f);
    }
}

int per_tile_for(int64_t n) { return n <= (1 << 15) ? 16 : 64; }

template <typename T>
cudaError_t embed_t(const void* ids, int id_bytes, int64_t n, const void* w, int64_t vocab, int64_t D, float scale, void* out,
                    int64_t* dropped, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int64_t blocks = (n + 7) / 8;
    const unsigned grid = static_cast<unsigned>(blocks < 148 * 32 ? blocks : 148 * 32);
    const bool vec = D % V == 0 && ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    auto* d = reinterpret_cast<unsigned long long*>(dropped);
    if (vec) embed_kernel<T, V><<<grid, 256, 0, s>>>(ids, id_bytes, n, static_cast<const T*>(w), vocab, D, scale, static_cast<T*>(out), d);
    else embed_kernel<T, 1><<<grid, 256, 0, s>>>(ids, id_bytes, n, static_cast<const T*>(w), vocab, D, scale, static_cast<T*>(out), d);
    return cudaGetLastError();
}

template <typename T>
cudaError_t sums_t(const SumParams& p, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = p.D % V == 0 && p.src_stride % V == 0 &&
                     ((reinterpret_cast<uintptr_t>(p.src) | reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0;
    const int64_t zb = (static_cast<int64_t>(p.vocab) + 7) / 8;
    row_zero_kernel<T><<<static_cast<unsigned>(zb < 148 * 16 ? zb : 148 * 16), 256, 0, s>>>(p);
    if (p.n > 0) {
        auto slabs = [&](int v) { return static_cast<unsigned>((p.D + SUM_THREADS * v - 1) / (SUM_THREADS * v)); };
        const unsigned tiles = static_cast<unsigned>(p.tiles);
        if (vec) row_sum_kernel<T, V><<<dim3(tiles, slabs(V)), SUM_THREADS, 0, s>>>(p);
        else row_sum_kernel<T, 1><<<dim3(tiles, slabs(1)), SUM_THREADS, 0, s>>>(p);
        if (p.tiles > 1) row_sum_join_kernel<T><<<dim3(tiles, slabs(1)), SUM_THREADS, 0, s>>>(p);
    }
    return cudaGetLastError();
}

int report(const char* name, cudaError_t e) {
    if (e == cudaSuccess) return PEER_OK;
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", name, cudaGetErrorString(e));
    set_global_error(buf);
    return PEER_ERR_CUDA;
}
int refuse(const char* msg) {
    set_global_error(msg);
    return PEER_ERR_INVALID_ARG;
}
constexpr int64_t INDEX_MAX = 0x7ffffffe;

}  // namespace
}  // namespace peer

using namespace peer;

extern "C" int peer_embedding(const void* ids, int32_t id_bytes, int64_t n_ids, const void* weight, int32_t dtype, int64_t vocab,
                              int64_t dim, float scale, void* out, int64_t* dropped, void* stream) {
    if (n_ids < 0 || vocab < 1 || vocab > INDEX_MAX || dim < 1 || dim > PEER_ROW_DIM_MAX)
        return refuse("peer_embedding: n_ids must not be negative, vocab lie in [1, 2^31 - 2], dim in [1, 2^20]");
    if (id_bytes != 4 && id_bytes != 8) return refuse("peer_embedding: ids are int32 or int64");
    if (n_ids == 0) return PEER_OK;
    if (!ids || !weight || !out) return refuse("peer_embedding: null pointer");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == PEER_DTYPE_F32) return report("peer_embedding", embed_t<float>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_embedding", embed_t<__nv_bfloat16>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    if (dtype == PEER_DTYPE_F16) return report("peer_embedding", embed_t<__half>(ids, id_bytes, n_ids, weight, vocab, dim, scale, out, dropped, s));
    return refuse("peer_embedding: dtype must be F32, BF16 or F16");
}

extern "C" int64_t peer_embedding_workspace(int64_t n_ids, int64_t dim) {
    if (n_ids <= 0 || dim < 1) return 0;
    const int per = per_tile_for(n_ids);
    const int64_t tiles = (n_ids + per - 1) / per;
    return row_sort_bytes(n_ids) + tiles * 2 * dim * static_cast<int64_t>(sizeof(float));
}

extern "C" int peer_embedding_backward(const void* ids, int32_t id_bytes, int64_t n_ids, const void* grad, int64_t grad_stride,
                                       int32_t dtype, int64_t vocab, int64_t dim, float scale, int64_t padding_idx,
                                       void* grad_weight, void* workspace, int64_t workspace_bytes, void* stream) {
    if (n_ids < 0 || n_ids > INDEX_MAX || vocab < 1 || vocab > INDEX_MAX || dim < 1 || dim > PEER_ROW_DIM_MAX || grad_stride < 0)
        return refuse("peer_embedding_backward: n_ids and vocab must lie below 2^31 - 1, dim in [1, 2^20]");
    if (id_bytes != 4 && id_bytes != 8) return refuse("peer_embedding_backward: ids are int32 or int64");
    if (dtype != PEER_DTYPE_F32 && dtype != PEER_DTYPE_BF16 && dtype != PEER_DTYPE_F16)
        return refuse("peer_embedding_backward: dtype must be F32, BF16 or F16");
    if (!grad_weight || (n_ids > 0 && (!ids || !grad))) return refuse("peer_embedding_backward: null pointer");
    if (n_ids > 0 && (!workspace || workspace_bytes < peer_embedding_workspace(n_ids, dim)))
        return refuse("peer_embedding_backward: workspace is missing or smaller than peer_embedding_workspace says");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    RowSortArgs a{};
    a.ids = ids; a.id_bytes = id_bytes; a.n = n_ids; a.vocab = vocab; a.skip = padding_idx;
    SumParams p{};
    p.n = n_ids; p.vocab = static_cast<uint32_t>(vocab); p.src = grad; p.src_stride = grad_stride; p.scale = scale;
    p.out = grad_weight; p.D = dim;
    if (n_ids > 0) {
        row_sort_layout(a, workspace);
        const cudaError_t e = launch_row_sort(a, s);
        if (e != cudaSuccess) return report("peer_embedding_backward", e);
        p.keys = a.sorted_keys; p.order = a.order;
        p.per_tile = per_tile_for(n_ids);
        p.tiles = (n_ids + p.per_tile - 1) / p.per_tile;
        p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + row_sort_bytes(n_ids));
    }
    if (dtype == PEER_DTYPE_F32) return report("peer_embedding_backward", sums_t<float>(p, s));
    if (dtype == PEER_DTYPE_BF16) return report("peer_embedding_backward", sums_t<__nv_bfloat16>(p, s));
    return report("peer_embedding_backward", sums_t<__half>(p, s));
}
